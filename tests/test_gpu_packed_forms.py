"""Attention over packed sequences on the GPU: values that are not finite, captured and replayed calls, streams, layouts, partial gradients, through the
compiled host path and the ctypes one."""
import math

import pytest
import torch

from oracle import packed_oracle as ref
from test_gpu_packed import i32, inputs, near, rand, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "ctypes"])
def host_path(request, monkeypatch):
    from lvar_amd import packed_ops
    if request.param == "ctypes":
        monkeypatch.setattr(packed_ops, "_native", lambda: None)
    return request.param


def by_rows(q, k, v, go, off, koff, causal):
    """Results and tolerances from the keys that each row sees, and nothing else."""
    q, k, v, go = (t.double() for t in (q, k, v, go))
    H, T, d = q.shape[1:]
    G = H // k.shape[1]
    out = {n: torch.zeros_like(q) for n in ("o", "dq", "t_o", "t_dq")}
    out.update({n: torch.zeros_like(k) for n in ("dk", "dv", "t_dk", "t_dv")})
    for b in range(len(off) - 1):
        n, m = off[b + 1] - off[b], koff[b + 1] - koff[b]
        for h in range(H):
            for i in range(n):
                seen = max(0, min(m, m - n + i + 1)) if causal else m
                if seen == 0:
                    continue
                at, keys = (0, h, slice(off[b] + i, off[b] + i + 1)), (0, h // G, slice(koff[b], koff[b] + seen))
                r = ref.sequence(q[at], k[keys], v[keys], 1 / math.sqrt(d), False, go[at])
                # (a key of infinite elements is seen with weight 0 or leaves nothing finite: either way it adds no error)
                some = torch.isfinite(k[keys]).all(-1)
                t = ref.sequence(q[at], k[keys][some], v[keys][some], 1 / math.sqrt(d), False, go[at])
                for name in ("o", "dq"):
                    out[name][at], out["t_" + name][at] = r[name], t["t_" + name]
                for name in ("dk", "dv"):
                    out[name][keys] += r[name]
                    out["t_" + name][keys] += (n * G + 8) * ref.F32 * r[name].abs()
                    out["t_" + name][keys] += torch.zeros(seen, d, dtype=torch.float64).masked_scatter(some[:, None].expand(seen, d), t["t_" + name])
    return out


BAD = [
    # lengths, key lengths, H, Hkv, d, causal
    ([150, 40], None, 2, 1, 64, True),
    ([100, 70], [130, 30], 2, 2, 128, True),
    ([90], None, 2, 1, 256, True),
    ([60, 60], [70, 90], 1, 1, 128, False),
    ([600], [70], 1, 1, 64, True),          # (rows that see nothing; several workgroups share the keys)
    ([300], None, 4, 1, 128, True),         # (so they do here)
    ([70, 3], [3300, 3000], 1, 1, 64, True),     # (several workgroups share the keys of a query tile)
    ([9], [3100], 2, 1, 256, True),
    ([33, 8], [900, 2900], 1, 1, 128, False),
]


@pytest.mark.parametrize("case", BAD, ids=str)
@pytest.mark.parametrize("where", ["q", "k", "v", "go"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_not_finite(case, where, value):
    """It reaches the rows that see it and their gradients, and nothing else."""
    from lvar_amd.packed_ops import packed_attn
    lens, klens, H, Hkv, d, causal = case
    q, k, v, off, koff = (x if not torch.is_tensor(x) else x.contiguous() for x in inputs(lens, klens, H, Hkv, d, seed=d))
    go = rand(*q.shape, seed=6)
    t = dict(q=q, k=k, v=v, go=go)[where]
    t[0, 0, min(lens[0], t.shape[2]) * 2 // 3, 5] = value
    t[0, -1, t.shape[2] - 2, d - 1] = value
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    o, _ = packed_attn(*leaves, i32(off), i32(koff), causal=causal)
    grads = torch.autograd.grad(o, leaves, go.cuda())
    r = by_rows(q, k, v, go, off, off if koff is None else koff, causal)
    for name, x in (("o", o), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        fine = torch.isfinite(r[name])
        assert bool((~torch.isfinite(x.cpu()))[~fine].all()), name + " hides a value that is not finite"
        near(x.cpu().float().masked_fill(~fine, 0), r[name].masked_fill(~fine, 0), r["t_" + name].masked_fill(~fine, 0), name)


def test_large_scores(host_path):
    """Scores of -2^20 and 2^20 (off by up to 2^-4, which the tolerance counts), and a row of scores of -infinity, which counts as one without a key."""
    from lvar_amd.packed_ops import packed_attn
    q, k, v = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16), torch.ones(1, 1, 4, 64, dtype=torch.bfloat16), rand(1, 1, 4, 64, seed=1)
    q[0, 0, :, 0] = torch.tensor([-2.0 ** 23, 2.0 ** 23, -1.0, 1.0])
    off = [0, 1, 2, 3, 4]
    for value in (None, math.inf):
        if value:
            k[0, 0, 2, 0] = value
        o, (M, L) = packed_attn(q.cuda(), k.cuda(), v.cuda(), i32(off), scale=0.125)
        r = ref.packed_attn(q, k, v, off, scale=0.125)
        some = [0, 1, 3] if value else [0, 1, 2, 3]
        for name, x in (("o", o), ("M", M), ("L", L)):
            near(x[:, :, some], r[name][:, :, some], r["t_" + name][:, :, some], name)
    assert bool((o[0, 0, 2] == 0).all()) and M[0, 0, 2, 0] == -math.inf and L[0, 0, 2, 0] == 1


def run(q, k, v, off, koff, go, **kw):
    from lvar_amd.packed_ops import packed_attn
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    o, (M, L) = packed_attn(*leaves, off, koff, **kw)
    return [o.detach(), M, L, *torch.autograd.grad(o, leaves, go)]


SETS = [([300, 0, 41, 500], None, 4, 2, 128, True), ([1000, 400], [60, 10], 4, 4, 64, False), ([260], None, 8, 1, 256, True), ([20, 1400], [1700, 4700], 2, 1, 128, True)]


@pytest.mark.parametrize("case", SETS, ids=str)
def test_the_same_bits(case, host_path):
    lens, klens, H, Hkv, d, causal = case
    q, k, v, off, koff = (x.cuda() if torch.is_tensor(x) else x for x in inputs(lens, klens, H, Hkv, d, lead=2, tail=3, seed=1))
    go = rand(*q.shape, seed=3).cuda()
    off, koff = i32(off), i32(koff)
    want = run(q, k, v, off, koff, go, causal=causal)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, off, koff, go, causal=causal), want))


@pytest.mark.parametrize("case", SETS[:2], ids=str)
def test_layouts(case, host_path):
    """Orders of axes, odd strides, misaligned bases, broadcast heads and gradients: the bits of packed tensors."""
    lens, klens, H, Hkv, d, causal = case
    q, k, v, off, koff = (x.cuda().contiguous() if torch.is_tensor(x) else x for x in inputs(lens, klens, H, Hkv, d, seed=4))
    go = rand(*q.shape, seed=3).cuda()
    off, koff = i32(off), i32(koff)
    want = run(q, k, v, off, koff, go, causal=causal)

    def wide(t, pad, shift):   # rows of d + pad elements, the base shifted
        x = torch.empty(t.numel() // d * (d + pad) + 64, dtype=t.dtype, device="cuda")
        x = x[shift:].as_strided(t.shape, (0, t.shape[2] * (d + pad), d + pad, 1))
        return x.copy_(t)
    tokens_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    forms = [lambda t: wide(t, 8, 0), lambda t: wide(t, 8, 3), lambda t: wide(t, 3, 0), tokens_first, lambda t: wide(t, 24, 8),
             lambda t: t.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)]
    for i, f in enumerate(forms):
        g = forms[(i + 1) % len(forms)]
        got = run(f(q), f(k), g(v), off, koff, g(go), causal=causal)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    # one token's gradient for all
    one = go[:, :, :1].expand_as(go)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, off, koff, one, causal=causal), run(q, k, v, off, koff, one.contiguous(), causal=causal)))
    # one key head for all: its gradient is the sum, formed by the caller's expand
    k1, v1 = k[:, :1].detach().requires_grad_(), v[:, :1].detach().requires_grad_()
    got = run(q, k1.expand_as(k), v1.expand_as(v), off, koff, go, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(got, run(q, k[:, :1].expand_as(k).contiguous(), v[:, :1].expand_as(v).contiguous(), off, koff, go, causal=causal)))


@pytest.mark.parametrize("case", SETS, ids=str)
def test_partial_gradients(case, host_path):
    from lvar_amd.packed_ops import packed_attn
    lens, klens, H, Hkv, d, causal = case
    q, k, v, off, koff = (x.cuda() if torch.is_tensor(x) else x for x in inputs(lens, klens, H, Hkv, d, seed=4))
    go = rand(*q.shape, seed=3).cuda()
    off, koff = i32(off), i32(koff)
    want = run(q, k, v, off, koff, go, causal=causal)[3:]
    for which in range(1, 7):
        leaves = [x.detach().requires_grad_(bool(which >> i & 1)) for i, x in enumerate((q, k, v))]
        o, (M, L) = packed_attn(*leaves, off, koff, causal=causal)
        some = [i for i in range(3) if which >> i & 1]
        for got, i in zip(torch.autograd.grad(o, [leaves[i] for i in some], go), some):
            assert torch.equal(got, want[i])


def test_no_tokens(host_path):
    from lvar_amd.packed_ops import packed_attn
    z = lambda h, t: torch.randn(1, h, t, 64, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    for T, Tk in ((0, 0), (0, 9), (5, 0)):
        leaves = [z(2, T).requires_grad_(), z(1, Tk).requires_grad_(), z(1, Tk).requires_grad_()]
        for causal in (True, False):
            o, (M, L) = packed_attn(*leaves, i32([0, 0, T]), i32([0, Tk, Tk]), causal=causal)
            assert o.shape == (1, 2, T, 64) and bool((o == 0).all()) and bool((M == -math.inf).all()) and bool((L == 1).all())
            for g, x in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), leaves):
                assert g.shape == x.shape and bool((g == 0).all())


def test_gradients_of_many_sequences(host_path):
    """More borders than a wave has lanes, empty ones among them."""
    lens = [(i * 37) % 90 for i in range(100)]
    klens = [(i * 53) % 70 for i in range(100)]
    for kl, causal in ((None, True), (klens, False), (klens, True)):
        q, k, v, off, koff = inputs(lens, kl, 2, 1, 64, lead=1, tail=2, seed=9)
        go = rand(*q.shape, seed=3)
        got = run(q.cuda(), k.cuda(), v.cuda(), i32(off), i32(koff), go.cuda(), causal=causal)
        r = ref.packed_attn(q, k, v, off, koff, causal=causal, go=go)
        for name, x in zip(("o", "M", "L", "dq", "dk", "dv"), got):
            near(x, r[name], r["t_" + name], name)


def test_in_a_graph(host_path):
    """Forward and backward captured twice on leaves of their own, replayed in turn with other lengths and values, beside eager work."""
    H, Hkv, d, T = 4, 1, 64, 700
    off = i32([0, 100, 400, 700])
    make = lambda: [rand(1, h, T, d, seed=i).cuda() for i, h in enumerate((H, Hkv, Hkv, H))]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*make()[:3], off, None, make()[3])
    torch.cuda.current_stream().wait_stream(side)
    graphs, held, outs = [], [], []
    for _ in range(2):
        x = make()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(*x[:3], off, None, x[3]))
        graphs.append(g)
        held.append(x)
    for r in range(5):
        off.copy_(torch.tensor([[0, 100, 400, 700], [0, 0, 0, 700], [3, 50, 51, 699], [0, 700, 700, 700], [0, 300, 600, 650]][r], dtype=torch.int32))
        for j, x in enumerate(held):
            for i, t in enumerate(x):
                t.copy_(rand(*t.shape, seed=100 * r + 10 * j + i))
        want = [run(*x[:3], off, None, x[3]) for x in held]
        torch.cuda.synchronize()
        for j in (r % 2, 1 - r % 2):
            graphs[j].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[j], want[j])), (r, j)


def test_two_streams(host_path):
    sets = []
    for i in range(2):
        q, k, v, off, _ = inputs([900, 300 + i], None, 4, 1, 128, seed=i)
        sets.append([*(t.cuda() for t in (q, k, v)), i32(off), None, rand(*q.shape, seed=7).cuda()])
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(4):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(run(*s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for x in g:
            assert all(torch.equal(a, b) for a, b in zip(x, w))


def test_what_it_refuses(host_path):
    from lvar_amd.packed_ops import ShapeError, packed_attn
    x = lambda h, t=8, d=64: torch.zeros(1, h, t, d, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    off = i32([0, 3, 8])
    for args in [(x(4), x(3), x(3), off), (x(4), x(2), x(1), off), (x(4), x(2, 9), x(2, 9), off), (x(4, 8, 96), x(2, 8, 96), x(2, 8, 96), off),
                 (x(4).expand(2, 4, 8, 64), x(2), x(2), off), (x(4), x(2), x(2), off[:1]), (x(4), x(2), x(2), off[None]), (x(4), x(2), x(2), off.cpu()),
                 (x(4), x(2), x(2), off, off[:2]), (x(4)[0], x(2), x(2), off), (x(4), x(2, 8, 128), x(2, 8, 128), off)]:
        with pytest.raises(ShapeError):
            packed_attn(*args)
    for args in [(x(4).float(), x(2), x(2), off), (x(4), x(2), x(2), off.long()), (x(4), x(2), x(2), off, off.float())]:
        with pytest.raises(TypeError):
            packed_attn(*args)
    with pytest.raises(RuntimeError, match="HIP device"):
        packed_attn(x(4), x(2).cpu(), x(2), off)
    for scale in (0.0, -1.0, math.nan, math.inf, 1e-39):
        with pytest.raises(RuntimeError):
            packed_attn(x(4), x(2), x(2), off, scale=scale)
    q = x(4).requires_grad_()
    o, (M, L) = packed_attn(q, x(2), x(2), off)
    assert not M.requires_grad and not L.requires_grad
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(o, q, torch.ones_like(o), create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x(4), x(4))
        with pytest.raises(RuntimeError, match="forward"):
            packed_attn(dual, x(2), x(2), off)


def test_modes(host_path):
    from lvar_amd.packed_ops import packed_attn
    q, k, v, off, _ = inputs([70], None, 2, 1, 64, seed=2)
    q, k, v, off = q.cuda(), k.cuda(), v.cuda(), i32(off)
    want = packed_attn(q, k, v, off)[0]
    with torch.inference_mode():
        o, (M, L) = packed_attn(q, k, v, off)
        assert o.is_inference() and torch.equal(o, want)
    with torch.no_grad():
        assert not packed_attn(q.requires_grad_(), k, v, off)[0].requires_grad
    go = rand(*q.shape, seed=3).cuda()
    grads = run(q, k, v, off, None, go)[3:]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().cpu(), lambda t: t.cuda()):
        assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, off, None, go)[3:], grads))
    # a leaf that is written between forward and backward
    leaf = k.detach().clone().requires_grad_()
    o, _ = packed_attn(q, leaf, v, off)
    with torch.no_grad():
        leaf.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        o.backward(go)
    # kept for a second backward pass
    o, _ = packed_attn(q, k.requires_grad_(), v, off)
    a, b = (torch.autograd.grad(o, k, go, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(a, b) and torch.equal(a, grads[1])


def test_rows_far_apart(host_path):
    """Rows 2 MiB apart, and further, and heads beyond 32 bits of elements."""
    from lvar_amd.packed_ops import packed_attn
    H, T, d = 3, 12, 64
    big = torch.zeros(2 ** 32 + 2 ** 25, dtype=torch.bfloat16, device="cuda")
    small = [rand(1, H, T, d, seed=i).cuda() for i in range(4)]
    off = i32([0, 7, 12])
    want = run(*small[:3], off, None, small[3])
    for row in (1 << 20, 1 << 21):
        views = [big.as_strided((1, H, T, d), (0, 2 ** 31, row, 1), 4096 * i).copy_(t) for i, t in enumerate(small)]
        assert all(torch.equal(a, b) for a, b in zip(run(*views[:3], off, None, views[3]), want))
    with torch.no_grad():
        assert torch.equal(packed_attn(*views[:3], off)[0], want[0])


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit formula, from the kernel's gradients."""
    q, k, v, off, _ = inputs([90, 40], None, 4, 2, 64, seed=12)
    go = rand(*q.shape, seed=3)
    got = [x.double().cpu() for x in run(q.cuda(), k.cuda(), v.cuda(), i32(off), None, go.cuda())[3:]]
    r = ref.packed_attn(q, k, v, off, go=go)
    x = [t.double() for t in (q, k, v)]
    f = lambda x: float((go.double() * ref.packed_attn(*x, off)["o"]).sum())  # noqa: E731
    eps = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        step = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        up, down = ([t + s * eps * step if j == i else t for j, t in enumerate(x)] for s in (1, -1))
        slope = (f(up) - f(down)) / (2 * eps)
        # (the error of the difference itself: eps^2 of the third derivative, and 2^-52 of the sum over eps)
        tol = float((r["t_" + name] * step.abs()).sum()) + 1e-6 * float((r[name].abs() * step.abs()).sum())
        assert abs(float((got[i] * step).sum()) - slope) <= tol


def test_many_tokens(host_path):
    """2.2 million tokens of 20000 sequences that are alike: elements beyond 31 bits, heads that are copied because they span 2^31 bytes; every sequence
    has the bits of one alone."""
    H, n, B, d = 8, 110, 20000, 128
    one = [rand(1, h, n, d, seed=i).cuda() for i, h in enumerate((H, 1, 1, H))]
    want = run(*one[:3], i32([0, n]), None, one[3])
    many = [t.transpose(1, 2).repeat(1, B, 1, 1).transpose(1, 2) for t in one]      # [1,h,T,d], tokens first
    got = run(*many[:3], torch.arange(B + 1, dtype=torch.int32, device="cuda") * n, None, many[3])
    for a, b in zip(got, want):
        a = a.view(*a.shape[:2], B, n, a.shape[3]) if a.is_contiguous() else a.transpose(1, 2).view(1, B, n, a.shape[1], a.shape[3]).permute(0, 3, 1, 2, 4)
        assert bool((a == b[:, :, None]).all())


def test_workspace_that_is_too_small():
    """Where the keys of a query tile are shared, the entry point wants room for the parts."""
    import ctypes as C
    from lvar_amd import _lib
    lib = _lib.load()
    T, Tk, d = 64, 8192, 128
    sizes = (1, T, Tk, 1, 1, d, 0)
    need = lib.lvar_packed_attn_fwd_workspace_bytes(*sizes)
    assert need > 0
    q, k = rand(1, 1, T, d).cuda(), rand(1, 1, Tk, d, seed=1).cuda()
    o, st = torch.zeros_like(q), torch.zeros(2, T, device="cuda")
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    view = lambda t: _lib.LvarTensor(t.data_ptr(), 0, 0, d)  # noqa: E731
    ptr = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    off, koff = i32([0, T]), i32([0, Tk])
    call = lambda w, n: lib.lvar_packed_attn_fwd(view(q), view(k), view(k), view(o), ptr(off), ptr(koff), ptr(st[0]), ptr(st[1]), w, n, *sizes, 0.1,  # noqa: E731
                                                 C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert call(None, need) == -1 and call(ptr(ws), need - 1) == -1 and call(C.c_void_p(ws.data_ptr() + 8), need) == -1
    assert bool((o == 0).all())
    assert call(ptr(ws), need) == 0
    torch.cuda.synchronize()
    assert bool((o != 0).any())
