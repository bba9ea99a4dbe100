"""Norms with rotation, the paged cache and the attention over it on the GPU, against the 64-bit oracle.

Tolerances count roundings: a result is rounded once to bf16 (half a step, 2^-8 of the value); sums of n products in 32 bits are
off by at most about n * 2^-24 of the sum of magnitudes; the attention also rounds its probabilities to bf16 (2^-8 each)."""
import math

import pytest
import torch

from oracle import kv_cache_oracle as ref

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8          # half a step, relative
F32 = 2.0 ** -24
EPS = {"l2": 1e-12, "rms": 1e-6, None: 0.0}


def rand(*shape, seed=0, amp=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * amp).to(dtype)


def tables(rows, half, seed=5):
    a = torch.randn(rows, half, generator=torch.Generator().manual_seed(seed)) * 3
    return a.cos(), a.sin()


def weight(kind, heads, d, seed, dtype=torch.float32):
    if kind is None:
        return None
    shape = {"head": (heads, 1), "dim": (d,), "row": (1, d), "one": (1, 1), "full": (heads, d)}[kind]
    return 1 + 0.3 * torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def cu(t):
    return None if t is None else t.cuda()


def check_rows(got, want, what):
    """One rounding to bf16, and 32-bit arithmetic of a row (its sum of d squares, a root, a quotient, four products)."""
    assert got.dtype == torch.bfloat16 and got.is_contiguous()
    top = want.abs().amax(-1, keepdim=True)
    tol = BF16 * want.abs() + (want.shape[-1] + 16) * F32 * top + 1e-38
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err - tol).max()):.3g} over"


def projection(B, H, Hkv, L, d, seed, amp=1.0):
    """q, k, v as views on one fused projection"""
    x = rand(B, L, H + 2 * Hkv, d, seed=seed, amp=amp).transpose(1, 2)
    return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]


# ---- norm and rotation ----

NORM_CASES = [
    # B, H, Hkv, L, d, rot, norm, weight, interleaved, positions
    (1, 1, 1, 1, 16, 16, "l2", None, True, None),
    (2, 3, 1, 5, 32, 16, "rms", "dim", False, None),
    (2, 16, 16, 16, 128, 128, "l2", "head", True, None),
    (3, 6, 2, 37, 64, 64, "rms", "full", False, "batch"),
    (1, 5, 5, 101, 128, 64, None, "row", False, "flat"),
    (2, 4, 4, 33, 256, 256, "l2", "one", False, "batch64"),
    (2, 8, 2, 19, 128, 96, "rms", "dim", True, "flat64"),
    (1, 7, 7, 1500, 64, 32, "l2", "head", True, None),       # several heads per workgroup, ragged chunks of heads
    (4, 9, 3, 700, 128, 128, "rms", "full", False, "batch"),
    (2, 5, 1, 300, 256, 128, None, None, True, None),
    (1, 2, 2, 9, 64, 0, "rms", "dim", True, None),           # no rotation
]


def norm_inputs(case, weights=torch.float32):
    B, H, Hkv, L, d, rot, norm, wk, inter, pos = case
    q, k, _ = projection(B, H, Hkv, L, d, seed=L + d)
    rows = L + 3
    cos, sin = tables(rows, rot // 2) if rot else (None, None)
    positions = None
    if pos:
        g = torch.Generator().manual_seed(3)
        positions = torch.randint(-2, rows + 2, (B, L) if pos.startswith("batch") else (L,), generator=g)      # (clamped to the table)
        positions = positions if pos.endswith("64") else positions.int()
    w = [weight(wk, h, d, 7 + i, weights) for i, h in enumerate((H, Hkv))]
    return q, k, w, cos, sin, positions, rows


@pytest.mark.parametrize("case", NORM_CASES)
def test_norm_rope(case):
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, L, d, rot, norm, wk, inter, pos = case
    q, k, w, cos, sin, positions, rows = norm_inputs(case)
    got = kv.qk_norm_rope(q.cuda(), k.cuda(), cu(cos), cu(sin), cu(positions), cu(w[0]), cu(w[1]), norm=norm, interleaved=inter)
    at = ref.table_rows(B, L, rows, positions)
    for x, y, wx, name in ((q, got[0], w[0], "q"), (k, got[1], w[1], "k")):
        check_rows(y, ref.norm_rope(x, wx, cos, sin, at, norm, EPS[norm], inter), name)


@pytest.mark.parametrize("case", NORM_CASES)
@pytest.mark.parametrize("weights", [torch.float32, torch.bfloat16])
def test_norm_rope_gradients(case, weights):
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, L, d, rot, norm, wk, inter, pos = case
    q, k, w, cos, sin, positions, rows = norm_inputs(case, weights)
    leaves = [x.cuda().requires_grad_() if x is not None else None for x in (q, k, *w)]
    outs = kv.qk_norm_rope(leaves[0], leaves[1], cu(cos), cu(sin), cu(positions), leaves[2], leaves[3], norm=norm, interleaved=inter)
    # gradients as they come from a transposition: not contiguous
    gs = [rand(B, L, x.shape[1], d, seed=90 + i).transpose(1, 2) for i, x in enumerate((q, k))]
    some = [x for x in leaves if x is not None]
    grads = dict(zip(map(id, some), torch.autograd.grad(outs, some, [g.cuda() for g in gs])))
    at = ref.table_rows(B, L, rows, positions)
    for i, x in enumerate((q, k)):
        dx, dw = ref.norm_rope_grads(x, w[i], cos, sin, at, norm, EPS[norm], inter, gs[i])
        got = grads[id(leaves[i])]
        assert got.shape == x.shape and got.dtype == torch.bfloat16
        r = ref.factor(x.double(), norm, EPS[norm])
        size = r * (gs[i].double().norm(dim=-1, keepdim=True)) * (1.0 if w[i] is None else float(w[i].abs().max()))     # of what is subtracted
        tol = BF16 * dx.abs() + 4 * (d + 16) * F32 * size + 1e-38
        err = (got.double().cpu() - dx).abs()
        assert bool((err <= tol).all()), f"d{'qk'[i]}: {float((err - tol).max()):.3g} over"
        if w[i] is not None:
            dw_got = grads[id(leaves[2 + i])]
            assert dw_got.shape == w[i].shape and dw_got.dtype == w[i].dtype
            # sums of n products of size up to |g| |n|: magnitudes added up, the rounding of each of the two factors and of the sum's steps
            n = x.double() * r
            mag = gs[i].double().norm(dim=-1, keepdim=True) * n.abs()
            mag = mag.sum((0, 2))
            if w[i].dim() == 1:
                mag = mag.sum(0)
            else:
                for axis in (0, 1):
                    if w[i].shape[axis] == 1:
                        mag = mag.sum(axis, keepdim=True)
            tol = (d + 64) * F32 * mag + (BF16 * dw.abs() if weights == torch.bfloat16 else 0.0)
            err = (dw_got.double().cpu() - dw).abs()
            assert bool((err <= tol).all()), f"dw{'qk'[i]}: {float((err - tol).max()):.3g} over"


@pytest.mark.parametrize("kind", ["head", "full", "row", "dim", "one"])
@pytest.mark.parametrize("H,Hkv,L,d", [(3, 1, 1, 128), (2, 2, 16, 128), (5, 5, 64, 128), (4, 2, 65, 128), (3, 3, 30, 256), (2, 1, 37, 64), (6, 3, 250, 32), (1, 1, 90, 32)])
def test_norm_rope_gradients_of_few_tokens(kind, H, Hkv, L, d):
    """Around the sizes up to which the gradient of a weight is written without partial sums (8 tiles of 2048 / d tokens)."""
    test_norm_rope_gradients((2, H, Hkv, L, d, d, "rms" if L % 2 else "l2", kind, bool(L % 3), None), torch.float32 if H % 2 else torch.bfloat16)


def test_norm_rope_gradient_against_differences():
    """The gradient of the operator against central differences of the 64-bit forward pass."""
    from lvar_amd import kv_cache_ops as kv
    case = (2, 4, 2, 11, 64, 32, "l2", "head", False, None)
    q, k, w, cos, sin, _, rows = norm_inputs(case)
    leaves = [x.cuda().requires_grad_() for x in (q, k, *w)]
    outs = kv.qk_norm_rope(*leaves[:2], cos.cuda(), sin.cuda(), q_weight=leaves[2], k_weight=leaves[3], interleaved=False)
    gs = [rand(*x.shape, seed=4 + i) for i, x in enumerate((q, k))]
    grads = [g.double().cpu() for g in torch.autograd.grad(outs, leaves, [g.cuda() for g in gs])]
    at = ref.table_rows(2, 11, rows)
    f = lambda q, k, wq, wk: sum((g.double() * ref.norm_rope(x, y, cos, sin, at, "l2", 1e-12, False)).sum() for g, x, y in ((gs[0], q, wq), (gs[1], k, wk)))  # noqa: E731
    base = [x.detach().double().cpu() for x in leaves]
    for i in range(4):
        t = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        step = 1e-5
        up, down = [x + step * t if j == i else x for j, x in enumerate(base)], [x - step * t if j == i else x for j, x in enumerate(base)]
        diff = float((f(*up) - f(*down)) / (2 * step))
        # the operator's gradient is rounded to bf16, element by element
        assert abs(diff - float((grads[i] * t).sum())) <= BF16 * float((grads[i] * t).abs().sum()) + 1e-6


def test_norm_rope_rows_below_eps_and_zero_rows():
    from lvar_amd import kv_cache_ops as kv
    x = rand(1, 2, 4, 64, seed=1)
    x[0, 0, 1] = 0
    x[0, 1, 2] *= 1e-4
    g = rand(1, 2, 4, 64, seed=2)
    for norm, eps in (("l2", 0.25), ("rms", 1e-3), ("l2", 1e-12)):
        q = x.cuda().requires_grad_()
        o, _ = kv.qk_norm_rope(q, x.cuda(), norm=norm, eps=eps)
        dx, = torch.autograd.grad(o, q, g.cuda())
        at = ref.table_rows(1, 4, 1)
        check_rows(o.detach(), ref.norm_rope(x, None, None, None, at, norm, eps, True), "o")
        want, _ = ref.norm_rope_grads(x, None, None, None, at, norm, eps, True, g)
        size = ref.factor(x.double(), norm, eps) * g.double().norm(dim=-1, keepdim=True)
        assert bool(((dx.double().cpu() - want).abs() <= BF16 * want.abs() + 4 * 80 * F32 * size).all())


@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("interleaved", [True, False])
def test_norm_rope_of_extreme_values(norm, interleaved):
    """The largest bf16 values (whose squares are infinite in 32 bits: the factor is 0, as in eager fp32) and the smallest normal ones give finite results."""
    from lvar_amd import kv_cache_ops as kv
    cos, sin = (t.cuda() for t in tables(4, 32))
    for v in (torch.finfo(torch.bfloat16).max, 1e25, 2e-38):
        q = (torch.sign(rand(1, 2, 4, 64, seed=3)) * v).to(torch.bfloat16).cuda()
        for w in (None, torch.full((64,), 2.0, device="cuda")):
            got = kv.qk_norm_rope(q, q, cos, sin, q_weight=w, k_weight=w, norm=norm, interleaved=interleaved)
            assert all(bool(torch.isfinite(t).all()) for t in got)
            if v > 1:
                assert all(bool((t == 0).all()) for t in got)


def test_norm_rope_broadcast_inputs_and_one_output():
    """An expanded input gets the sum of its copies' gradients, an expanded weight a gradient per head; an output nobody used none."""
    from lvar_amd import kv_cache_ops as kv
    x = rand(1, 1, 6, 64, seed=1).cuda().requires_grad_()
    w = torch.full((1, 1), 1.5, device="cuda", requires_grad=True)
    q, wide = x.expand(2, 4, 6, 64), w.expand(4, 1)
    o, _ = kv.qk_norm_rope(q, rand(2, 4, 6, 64, seed=2).cuda(), q_weight=wide, norm="rms")
    g = rand(2, 4, 6, 64, seed=3)
    dx, dw, dwide = torch.autograd.grad(o, (x, w, wide), g.cuda())
    at = ref.table_rows(2, 6, 1)
    want, ww = ref.norm_rope_grads(q.detach().cpu(), wide.detach().cpu(), None, None, at, "rms", 1e-6, True, g)
    assert dwide.shape == (4, 1) and torch.allclose(dwide.double().cpu(), ww, rtol=1e-5, atol=1e-4)
    assert abs(float(dw) - float(ww.sum())) <= 1e-4 * float(ww.abs().sum())
    # eight bf16 gradients added up in bf16 by autograd's expand: a rounding of each, and of the sum
    assert bool(((dx.double().cpu() - want.sum((0, 1), keepdim=True)).abs() <= 2 * BF16 * want.abs().sum((0, 1), keepdim=True)).all())


@pytest.mark.parametrize("binding", [True, False])
def test_norm_rope_host_paths(binding, monkeypatch):
    """The compiled and the Python host path give the same bits and refuse a second derivative."""
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    q, k, _ = (t.cuda() for t in projection(2, 6, 2, 9, 64, seed=1))
    w = weight("full", 6, 64, 2).cuda().requires_grad_()
    cos, sin = (t.cuda() for t in tables(9, 16))
    q = q.requires_grad_()
    o = kv.qk_norm_rope(q, k, cos, sin, q_weight=w, norm="rms")
    assert o[0].requires_grad
    with torch.no_grad():
        assert all(torch.equal(x, y) for x, y in zip(o, kv.qk_norm_rope(q, k, cos, sin, q_weight=w, norm="rms")))
    g = [torch.ones_like(x) for x in o]
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(o, (q, w), g, create_graph=True)
    o = kv.qk_norm_rope(q, k, cos, sin, q_weight=w, norm="rms")
    dq, dw = torch.autograd.grad(o, (q, w), g)
    assert dq.stride() == torch.empty_like(q).stride()
    monkeypatch.setattr(kv, "_native", lambda: None)
    o2 = kv.qk_norm_rope(q, k, cos, sin, q_weight=w, norm="rms")
    dq2, dw2 = torch.autograd.grad(o2, (q, w), g)
    assert torch.equal(dq, dq2) and torch.equal(dw, dw2) and all(torch.equal(x, y) for x, y in zip(o, o2))


def test_norm_rope_leaves_nothing_for_empty_calls():
    from lvar_amd import kv_cache_ops as kv
    q = torch.zeros(2, 4, 0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    o, _ = kv.qk_norm_rope(q, q.detach()[:, :2], q_weight=w)
    assert o.shape == (2, 4, 0, 64)
    dq, dw = torch.autograd.grad(o, (q, w), torch.zeros_like(o))
    assert dq.shape == q.shape and float(dw.abs().sum()) == 0


# ---- writing and reading ----

def make_cache(P, H, page, d, dtype, seed, layout="heads"):
    """A cache full of leftovers: NaN and huge values where nobody has written."""
    from lvar_amd import kv_cache_ops as kv
    shape = (P, H, page, d) if layout == "heads" else (P, page, H, d)
    ts = []
    for i in range(2):
        g = torch.Generator().manual_seed(seed + i)
        if dtype == torch.bfloat16:
            x = torch.randn(shape, generator=g).to(torch.bfloat16)
            x[torch.rand(shape, generator=g) < 0.2] = math.nan
            x[torch.rand(shape, generator=g) < 0.1] = math.inf
        else:
            x = torch.randint(0, 256, shape, generator=g).to(torch.uint8).view(torch.float8_e4m3fn)
        ts.append(x if layout == "heads" else x.view(torch.uint8 if x.element_size() == 1 else torch.int16).transpose(1, 2).view(x.dtype))
    if dtype == torch.bfloat16:
        return kv.PagedKVCache(*ts)
    return kv.PagedKVCache(*ts, *(torch.randint(100, 140, (P, H, page), generator=torch.Generator().manual_seed(seed + 5 + i)).to(torch.uint8) for i in range(2)))


def to_gpu(cache):
    """(keeps the strides)"""
    out = []
    for t in cache:
        if t is None:
            out.append(None)
            continue
        n = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
        n.view(torch.uint8 if t.element_size() == 1 else torch.int16).copy_(t.view(torch.uint8 if t.element_size() == 1 else torch.int16))
        out.append(n)
    return type(cache)(*out)


def table_for(B, per, P, seed):
    return torch.randperm(P, generator=torch.Generator().manual_seed(seed))[:B * per].to(torch.int32).view(B, per).contiguous()


def same_bytes(a, b):
    view = torch.uint8 if a.element_size() == 1 else torch.int16
    return torch.equal(a.cpu().contiguous().view(view), b.contiguous().view(view))


APPEND_CASES = [
    # B, H, L, d, page, starts, counts, layout
    (1, 1, 1, 64, 16, [0], None, "heads"),
    (2, 3, 7, 128, 16, [13, 30], None, "heads"),           # across pages
    (3, 2, 40, 64, 32, [0, 5, 61], [40, 0, 17], "heads"),  # padded batch
    (2, 2, 33, 256, 64, [60, 127], None, "tokens"),
    (2, 16, 300, 128, 128, [1, 250], [-3, 500], "heads"),
    (2, 2, 50, 64, 16, [-10, 90], None, "heads"),          # partly outside the table, on both ends
]


@pytest.mark.parametrize("case", APPEND_CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_append_and_read(case, dtype):
    """Bit for bit, the rows nobody wrote as they were."""
    from lvar_amd import kv_cache_ops as kv
    B, H, L, d, page, starts, counts, layout = case
    per = -(-(min(max(starts), 60) + L) // page) if starts[0] < 0 else -(-(max(starts) + L) // page)
    P = B * per + 2
    cache = make_cache(P, H, page, d, dtype, 11, layout)
    table = table_for(B, per, P, 3)
    if per > 2:
        table[0, 1] = -1                                   # no page
        table[B - 1, 0] = P + 4
    _, k, v = projection(B, H, H, L, d, seed=17, amp=3.0)
    k = k.clone()
    k[:, :, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan]).to(torch.bfloat16)
    k[0, 0, -1] = 0
    v[0, 0, -1] *= 2.0 ** -120                             # the smallest scales
    start = torch.tensor(starts, dtype=torch.int32)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    g = to_gpu(cache)
    kv.kv_cache_append(g, k.cuda(), v.cuda(), table.cuda(), start.cuda(), cu(n))
    for pages, exps, x, got, got_e in ((cache.k, cache.k_exp, k, g.k, g.k_exp), (cache.v, cache.v_exp, v, g.v, g.v_exp)):
        want, want_e = ref.append(pages, exps, table, x, start, n)
        if want_e is not None:
            assert torch.equal(got_e.cpu(), want_e)
            a, b = got.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8)
            nan = (b & 127) == 127                          # (the sign of a NaN says nothing)
            assert torch.equal(a[~nan], b[~nan]) and bool(((a[nan] & 127) == 127).all())
        else:
            assert same_bytes(got, want)
    for lengths, first, most in (([per * page] * B, None, None), ([max(0, s) + L // 2 for s in starts], starts, L), ([0] * B, None, 5)):
        lens, first = torch.tensor(lengths, dtype=torch.int32), None if first is None else torch.tensor(first, dtype=torch.int32)
        rk, rv = kv.kv_cache_read(g, table.cuda(), lens.cuda(), most, cu(first))
        for pages, exps, got in ((g.k, g.k_exp, rk), (g.v, g.v_exp, rv)):
            want, _ = ref.read(pages.cpu(), None if exps is None else exps.cpu(), table, lens, per * page if most is None else most, first)
            assert torch.equal(torch.nan_to_num(got.double().cpu(), 7.0, 8.0, 9.0), torch.nan_to_num(want, 7.0, 8.0, 9.0))


def test_row_scales_at_their_borders():
    from lvar_amd import kv_cache_ops as kv
    g = torch.Generator().manual_seed(0)
    x = rand(1, 1, 256, 64, seed=2)
    top = torch.tensor([448.0, 450.0, 446.0, 224.0, 225.0, 1.0, 0.875, 0.878])      # the largest of a row: at, behind, before 1.75 * 2^n
    x = x / x.abs().amax(-1, keepdim=True)
    x = (x * (top.repeat(32) * torch.exp2(torch.randint(-20, 20, (256,), generator=g).float()))[None, None, :, None]).to(torch.bfloat16)
    x[0, 0, 5, :] = 3.3895313892515355e38                                          # the largest bf16
    x[0, 0, 6, :] = 1e-40                                                           # below the normal numbers
    cache = to_gpu(make_cache(4, 1, 64, 64, torch.float8_e4m3fn, 3))
    table = torch.arange(4, dtype=torch.int32).view(1, 4)
    kv.kv_cache_append(cache, x.cuda(), x.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    codes, byte = ref.quantise(x)
    assert torch.equal(cache.k_exp.cpu().view(-1), byte.view(-1))
    assert torch.equal(cache.k.cpu().view(torch.uint8).view(-1), codes.view(-1))


@pytest.mark.parametrize("norm,wk,inter,rot,d,H,Hkv,L", [("l2", "head", True, 128, 128, 16, 16, 36), ("rms", "dim", False, 64, 64, 6, 2, 1), ("rms", "full", True, 128, 256, 4, 4, 300),
                                                         (None, None, False, 0, 128, 8, 1, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_norm_rope_append(norm, wk, inter, rot, d, H, Hkv, L, dtype):
    from lvar_amd import kv_cache_ops as kv
    B, page = 3, 32
    starts, counts = [0, 21, 50], [L, max(1, L - 2), 0]
    per = -(-(50 + L) // page)
    P = B * per + 1
    q, k, v = projection(B, H, Hkv, L, d, seed=5)
    w = [weight(wk, h, d, 7 + i) for i, h in enumerate((H, Hkv))]
    cos, sin = tables(60 + L, rot // 2) if rot else (None, None)
    table = table_for(B, per, P, 1)
    start, n = torch.tensor(starts, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)
    cache = make_cache(P, Hkv, page, d, dtype, 4)
    g = to_gpu(cache)
    oq = kv.qk_norm_rope_append(g, q.cuda(), k.cuda(), v.cuda(), table.cuda(), start.cuda(), cu(cos), cu(sin), cu(n), None, cu(w[0]), cu(w[1]), norm, None, inter)
    at = ref.table_rows(B, L, 60 + L, None, start)
    check_rows(oq, ref.norm_rope(q, w[0], cos, sin, at, norm, EPS[norm], inter), "q")
    # values: as kv_cache_append writes them; keys: as qk_norm_rope makes them (same bits for bf16), rows nobody wrote as they were
    plain = to_gpu(cache)
    pos = (start[:, None] + torch.arange(L)).cuda()
    _, ok = kv.qk_norm_rope(q.cuda(), k.cuda(), cu(cos), cu(sin), pos, cu(w[0]), cu(w[1]), norm, None, inter)
    kv.kv_cache_append(plain, ok, v.cuda(), table.cuda(), start.cuda(), n.cuda())
    assert same_bytes(g.v, plain.v.cpu())
    if dtype == torch.bfloat16:
        assert same_bytes(g.k, plain.k.cpu())
        return
    assert torch.equal(g.v_exp, plain.v_exp)
    want_k = ref.norm_rope(k, w[1], cos, sin, at, norm, EPS[norm], inter)
    lens = start + n
    got, there = ref.read(g.k.cpu(), g.k_exp.cpu(), table, lens, L, start)
    scale = want_k.abs().amax(-1, keepdim=True) / 224                        # a row's power of two is at most top / 224
    tol = 2.0 ** -4 * want_k.abs() + scale * 2.0 ** -10 + (d + 16) * F32 * 448 * scale
    err = (got - want_k).abs()[there[:, None].expand(B, Hkv, L)]
    assert bool((err <= tol[there[:, None].expand(B, Hkv, L)]).all())


# ---- attention ----

def attn_case(B, H, Hkv, Lq, lengths, d, page, dtype, causal, counts=None, extra=1, seed=0, holes=False, layout="heads", scale=None, max_len=None):
    """Runs the operator on a cache whose other rows hold leftovers, and compares."""
    from lvar_amd import kv_cache_ops as kv
    n = max(max(lengths), 1)
    per = -(-n // page) + extra
    P = B * per + 2
    cache = make_cache(P, Hkv, page, d, dtype, seed, layout)
    table = table_for(B, per, P, seed)
    x = [rand(B, Hkv, n, d, seed=seed + 30 + i) for i in range(2)]
    lens = torch.tensor(lengths, dtype=torch.int32)
    pages = [ref.append(c, e, table, y, torch.zeros(B, dtype=torch.int32), lens) for c, e, y in ((cache.k, cache.k_exp, x[0]), (cache.v, cache.v_exp, x[1]))]
    cache = kv.PagedKVCache(pages[0][0], pages[1][0], pages[0][1], pages[1][1])
    if layout == "tokens":
        cache = cache._replace(k=cache.k.transpose(1, 2).contiguous().transpose(1, 2), v=cache.v.transpose(1, 2).contiguous().transpose(1, 2))
    for b in range(B):                                    # entries behind the last page of a sequence are leftovers as well
        table[b, -(-max(lengths[b], 0) // page):] = torch.tensor([-7, 2 ** 31 - 1, P])[b % 3]
    if holes:
        table[0, 0] = -1
        table[B - 1, max(0, (lengths[B - 1] - 1) // page)] = P
    q = rand(B, Lq, H, d, seed=seed + 50).transpose(1, 2)
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    g = to_gpu(cache)
    o, (M, L) = kv.paged_attn(q.cuda(), g, table.cuda(), lens.cuda(), scale, causal, cu(c), max_len)
    k, there = ref.read(cache.k, cache.k_exp, table, lens, n)
    v, _ = ref.read(cache.v, cache.v_exp, table, lens, n)
    seen = lens if max_len is None else lens.clamp(max=max_len)
    s = d ** -0.5 if scale is None else scale
    want, Mr, Lr, spread = ref.paged_attn(q, k, v, there, seen, s, causal, c)
    check_attn(o, M, L, want, Mr, Lr, spread, q, k, s, n)
    return o, M, L, (q.cuda(), g, table.cuda(), lens.cuda(), scale, causal, cu(c), max_len)


def check_attn(o, M, L, want, Mr, Lr, spread, q, k, scale, n):
    assert o.dtype == torch.bfloat16 and M.shape == Mr.shape and L.shape == Lr.shape and M.dtype == L.dtype == torch.float32
    o, M, L = o.double().cpu(), M.double().cpu(), L.double().cpu()
    empty = torch.isinf(Mr)
    assert torch.equal(torch.isinf(M), empty) and bool((M[empty] < 0).all()) and bool((L[empty] == 1).all()) and bool((o[empty.expand_as(o)] == 0).all())
    # a score: d products of 32 bits, scaled; its magnitudes add up to at most |q| |k|
    ds = (q.shape[-1] + 8) * F32 * scale * 1.4427 * float(q.double().norm(dim=-1).max()) * float(torch.nan_to_num(k).norm(dim=-1).max())
    full = ~empty
    assert bool(((M - Mr).abs()[full] <= ds + F32 * Mr.abs()[full]).all())
    # a term of the sum is off by the two scores' errors, its exponential by 2 steps, the sum by the number of its levels (here: at most n)
    dl = 2 * ds + (4 + min(n, 4096)) * F32
    assert bool(((L - Lr).abs()[full] <= dl * Lr[full]).all())
    tol = (BF16 + 2 * dl) * spread + BF16 * want.abs() + 1e-30
    err = (o - want).abs()
    assert bool((err <= tol).all()), f"{float((err - tol).max()):.3g} over, at {(err - tol).argmax()}"


ATTN_CASES = [
    # B, H, Hkv, Lq, lengths, d, page, causal, counts
    (1, 1, 1, 1, [1], 64, 16, False, None),
    (2, 4, 4, 1, [1, 0], 128, 16, True, None),                     # a sequence without a token
    (3, 8, 2, 1, [15, 16, 17], 128, 16, True, None),               # around the end of a page
    (3, 4, 1, 1, [31, 32, 33], 64, 32, False, None),
    (2, 16, 16, 16, [21, 21], 128, 64, False, None),               # scale 4 of an image
    (2, 3, 3, 36, [57, 50], 64, 64, False, [36, 20]),              # padded batch
    (4, 6, 2, 5, [200, 5, 3, 0], 128, 16, True, [5, 5, 5, 5]),     # fewer tokens than new ones: rows that see nothing
    (3, 8, 1, 7, [129, 300, 64], 256, 64, True, [7, 1, 0]),
    (2, 10, 2, 13, [700, 123], 128, 128, True, None),              # 65 rows: two row tiles
    (2, 4, 4, 64, [121, 185], 256, 16, False, None),
    (1, 7, 7, 1, [1025], 64, 1024, False, None),
    (2, 2, 1, 1, [3000, 511], 128, 16, True, None),                # cut into pieces and joined
    (3, 4, 2, 3, [2500, 127, 1281], 64, 32, True, [3, 2, 3]),
    (2, 5, 1, 8, [1111, 2222], 256, 64, False, None),
    (2, 12, 3, 61, [1501, 900], 128, 64, True, [61, 30]),
]


@pytest.mark.parametrize("case", ATTN_CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_paged_attn(case, dtype):
    B, H, Hkv, Lq, lengths, d, page, causal, counts = case
    attn_case(B, H, Hkv, Lq, lengths, d, page, dtype, causal, counts, seed=sum(lengths))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_paged_attn_forms(dtype):
    """Pages that are missing, another order of axes, a bound on the lengths, other scales, many sequences."""
    attn_case(2, 4, 2, 3, [150, 201], 128, 16, dtype, True, holes=True, seed=1)
    attn_case(2, 4, 2, 1, [40, 40], 64, 64, dtype, False, holes=True, seed=2)          # every page missing
    attn_case(2, 6, 3, 2, [333, 70], 128, 32, dtype, True, layout="tokens", seed=3)
    attn_case(2, 4, 4, 2, [1000, 90], 128, 32, dtype, False, max_len=700, seed=4)
    attn_case(2, 4, 4, 2, [1000, 90], 128, 32, dtype, False, max_len=200, seed=4)      # short enough not to be cut
    attn_case(1, 2, 1, 4, [900], 64, 16, dtype, True, scale=2.0, seed=5)
    attn_case(1, 2, 1, 4, [90], 64, 16, dtype, True, scale=1e-4, seed=6)
    attn_case(70, 2, 1, 1, [(i * 37) % 150 for i in range(70)], 64, 16, dtype, True, seed=7)      # more than a wave of sequences


def test_paged_attn_many_sequences_cut():
    """Over 64 sequences, long ones among short ones: the plan counts pieces across the lanes of two waves."""
    lengths = [20 + (i * 53) % 90 for i in range(130)]
    lengths[3] = lengths[64] = lengths[129] = 1900
    attn_case(130, 1, 1, 1, lengths, 64, 64, torch.bfloat16, True, extra=0, seed=8)


def test_paged_attn_growing_maxima_and_infinities():
    """Scores that keep growing along the cache; an infinite score; NaN in a key that is seen reaches its row."""
    from lvar_amd import kv_cache_ops as kv
    B, H, n, d = 1, 2, 640, 64
    q, k, v = rand(B, H, 2, d, seed=1), rand(B, H, n, d, seed=2), rand(B, H, n, d, seed=3)
    k = (k.float() * torch.linspace(0.1, 6, n)[:, None]).to(torch.bfloat16)
    cache = kv.PagedKVCache.alloc(10, H, d, 64)
    table, lens = torch.arange(10, dtype=torch.int32, device="cuda").view(1, 10), torch.tensor([n], dtype=torch.int32, device="cuda")
    kv.kv_cache_append(cache, k.cuda(), v.cuda(), table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    o, (M, L) = kv.paged_attn(q.cuda(), cache, table, lens, scale=1.0)
    there = torch.ones(1, n, dtype=torch.bool)
    check_attn(o, M, L, *ref.paged_attn(q, k.double(), v.double(), there, [n], 1.0), q, k.double(), 1.0, n)
    cache.k[2, 0, 5, 0] = math.nan
    o2, (M2, L2) = kv.paged_attn(q.cuda(), cache, table, lens, scale=1.0)
    assert bool(torch.isnan(o2[:, 0]).all()) and torch.equal(o2[:, 1], o[:, 1])
    o3, (M3, L3) = kv.paged_attn(torch.full_like(q, math.nan).cuda(), cache, table, lens)
    assert bool(torch.isnan(o3).all())


def test_paged_attn_of_nothing():
    from lvar_amd import kv_cache_ops as kv
    cache = kv.PagedKVCache.alloc(3, 2, 64, 16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.tensor([4, 0], dtype=torch.int32, device="cuda")
    o, (M, L) = kv.paged_attn(torch.zeros(2, 4, 0, 64, dtype=torch.bfloat16, device="cuda"), cache, table, lens)
    assert o.shape == (2, 4, 0, 64) and M.shape == (2, 4, 0, 1)
    k, v = kv.kv_cache_read(cache, table, lens, 0)
    assert k.shape == (2, 2, 0, 64)
    o, (M, L) = kv.paged_attn(rand(2, 4, 3, 64).cuda(), cache, table, lens, max_len=0)
    assert float(o.abs().sum()) == 0 and bool(torch.isinf(M).all()) and bool((L == 1).all())


def test_offsets_beyond_32_bits():
    """Pages behind the first 4 GiB of a cache, bf16 and 8-bit."""
    from lvar_amd import kv_cache_ops as kv
    H, page, d, n = 1, 1024, 256, 3000
    for dtype, P in ((torch.bfloat16, 10000), (torch.float8_e4m3fn, 20000)):
        k, v = (torch.empty((P, H, page, d), dtype=torch.uint8 if dtype != torch.bfloat16 else dtype, device="cuda") for _ in range(2))
        assert k.numel() * k.element_size() > 2 ** 32
        e = [None, None] if dtype == torch.bfloat16 else [torch.full((P, H, page), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
        cache = kv.PagedKVCache(k.view(dtype), v.view(dtype), *e)
        table = torch.tensor([[P - 1, 0, P - 2]], dtype=torch.int32, device="cuda")
        q, nk, nv = rand(1, 2, 1, d, seed=1), rand(1, H, n, d, seed=2), rand(1, H, n, d, seed=3)
        kv.kv_cache_append(cache, nk.cuda(), nv.cuda(), table, torch.zeros(1, dtype=torch.int32, device="cuda"))
        lens = torch.tensor([n], dtype=torch.int32, device="cuda")
        rk, rv = kv.kv_cache_read(cache, table, lens, n)
        want = [x.double() if dtype == torch.bfloat16 else ref.dequantise(*ref.quantise(x)) for x in (nk, nv)]
        assert torch.equal(rk.double().cpu(), want[0]) and torch.equal(rv.double().cpu(), want[1])
        o, (M, L) = kv.paged_attn(q.cuda(), cache, table, lens)
        check_attn(o, M, L, *ref.paged_attn(q, *want, torch.ones(1, n, dtype=torch.bool), [n], d ** -0.5), q, want[0], d ** -0.5, n)
        del cache, k, v, e, rk, rv
        torch.cuda.empty_cache()


def test_same_bits_again_and_beside_other_streams():
    """Twice the same call, from two streams at once: the same bits (each call has its own workspace)."""
    o, M, L, args = attn_case(2, 8, 2, 3, [2000, 700], 128, 16, torch.bfloat16, True, seed=9)
    from lvar_amd import kv_cache_ops as kv
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(kv.paged_attn(*args))
    torch.cuda.synchronize()
    for o2, (M2, L2) in got:
        assert torch.equal(o2, o) and torch.equal(M2, M) and torch.equal(L2, L)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_step_in_a_graph(dtype):
    """A decoding step (norm, rotation, append, attention) captured twice and replayed alternately, with lengths that change between the replays."""
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, d, page, P = 3, 8, 2, 128, 16, 120
    cos, sin = (t.cuda() for t in tables(700, d // 2))
    w = weight("dim", H, d, 3).cuda()
    table = table_for(B, P // B, P, 1).cuda()
    x = projection(B, H, Hkv, 1, d, seed=1)
    buf = [torch.empty_like(t, device="cuda") for t in x]
    start = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(cache):
        q = kv.qk_norm_rope_append(cache, *buf, table, start, cos, sin, q_weight=w, norm="rms", interleaved=False)
        return kv.paged_attn(q, cache, table, start + 1, causal=True)
    caches = [to_gpu(make_cache(P, Hkv, page, d, dtype, 5)) for _ in range(3)]
    step(to_gpu(make_cache(P, Hkv, page, d, dtype, 5)))       # (a cache of its own: the three hold the same)
    graphs, outs = [], []
    for c in caches[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c))
        graphs.append(g)
    for r in range(6):
        start.copy_(torch.tensor([r, 100 * r + 3, 620 - r], dtype=torch.int32))
        for i, t in enumerate(projection(B, H, Hkv, 1, d, seed=20 + r)):
            buf[i].copy_(t)
        o, (M, L) = step(caches[2])
        torch.cuda.synchronize()
        for i in (r % 2, 1 - r % 2):
            graphs[i].replay()
        for i in range(2):
            # (what the first sequences see of the cache: rows written by earlier steps, and leftovers that are the same in all three)
            same = lambda a, b: torch.equal(torch.nan_to_num(a.float(), 3.0, 4.0, 5.0), torch.nan_to_num(b.float(), 3.0, 4.0, 5.0))  # noqa: E731
            assert same(outs[i][0], o) and same(outs[i][1][0], M) and same(outs[i][1][1], L)


@pytest.mark.parametrize("binding", [True, False])
def test_gradients_with_hooks_on_saved_tensors(binding, monkeypatch):
    """Saved tensors that come back as packed copies (as save_on_cpu does), where tables, weights and positions were slices of wider memory."""
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    B, H, L, d = 2, 4, 37, 64
    wide = [rand(B, H, L, 2 * d, seed=i).cuda() for i in range(2)]
    cos, sin = (torch.cat([t, t], 1).cuda()[:, :d // 2] for t in tables(50, d // 2))
    positions = torch.randint(0, 50, (1, L), generator=torch.Generator().manual_seed(1)).cuda().expand(B, L)
    ws = [torch.cat([weight("full", H, d, 3 + i)] * 2, 1).cuda()[:, :d] for i in range(2)]
    g = [rand(B, H, L, d, seed=7 + i).cuda() for i in range(2)]

    def grads():
        q, k = (t.detach()[..., :d].requires_grad_() for t in wide)
        w = [t.detach().requires_grad_() for t in ws]
        return torch.autograd.grad(kv.qk_norm_rope(q, k, cos, sin, positions, *w), (q, k, *w), g)
    want = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().cpu().contiguous(), lambda t: t.cuda()):
        got = grads()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_in_a_graph():
    """Forward and backward captured on leaves of their own and replayed, beside eager work on other leaves."""
    from lvar_amd import kv_cache_ops as kv
    cos, sin = (t.cuda() for t in tables(40, 64))
    x = [rand(2, 4, 40, 128, seed=i).cuda() for i in range(2)]
    w0 = weight("head", 4, 128, 3).cuda()
    g0 = rand(2, 4, 40, 128, seed=9).cuda()

    def grads(leaves):
        o = kv.qk_norm_rope(leaves[0], leaves[1], cos, sin, q_weight=leaves[2], k_weight=leaves[3])
        return torch.autograd.grad(o, leaves, (g0, g0))
    make = lambda: [t.detach().clone().requires_grad_() for t in (*x, w0, w0)]  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(make())
    torch.cuda.current_stream().wait_stream(side)
    leaves = make()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads(leaves)
    for r in range(4):
        with torch.no_grad():
            leaves[0].copy_(rand(2, 4, 40, 128, seed=30 + r))
        eager = grads([t.detach().clone().requires_grad_() for t in leaves])
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


PADDED_CASES = [
    # B, H, Hkv, Lq, lengths, d, page, causal, counts: padding that leaves whole row tiles without a token, cut and uncut sequences
    (4, 8, 1, 64, [1500, 70, 40, 900], 128, 64, True, [64, 3, 0, 17]),
    (4, 8, 1, 64, [1500, 70, 40, 900], 64, 16, False, [1, 64, 64, 16]),
    (3, 4, 1, 50, [900, 2000, 10], 256, 32, True, [50, 1, 0]),
    (70, 4, 1, 40, [(i * 31) % 300 for i in range(70)], 64, 16, True, [(i * 7) % 45 - 2 for i in range(70)]),
    (330, 4, 2, 66, [(i * 37) % 41 for i in range(330)], 64, 16, False, [(i * 11) % 69 - 1 for i in range(330)]),   # more uncut tiles than workgroups of a round
]


@pytest.mark.parametrize("case", PADDED_CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_paged_attn_padded_batches(case, dtype):
    B, H, Hkv, Lq, lengths, d, page, causal, counts = case
    attn_case(B, H, Hkv, Lq, lengths, d, page, dtype, causal, counts, seed=7)


@pytest.mark.parametrize("Lq,H,Hkv,d,lengths", [(17, 2, 2, 64, [130, 64]), (33, 1, 1, 128, [700, 65]), (16, 3, 1, 128, [129, 48]), (129, 1, 1, 64, [300, 129]), (65, 2, 1, 256, [190, 1000]),
                                                (257, 1, 1, 128, [257, 900])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_paged_attn_row_tiles(Lq, H, Hkv, d, lengths, dtype):
    """Rows around the ends of tiles of 16, 32, 64 and 128."""
    for causal in (True, False):
        attn_case(2, H, Hkv, Lq, lengths, d, 16, dtype, causal, seed=Lq)


@pytest.mark.parametrize("Lq", [1, 20, 70])
def test_leftover_bytes_of_any_value(Lq):
    """Codes and scale bytes of rows nobody has written: every byte there is, NaN and infinities among them, on pages that are shared and on one that is missing."""
    from lvar_amd import kv_cache_ops as kv
    B, H, d, page, n = 2, 2, 128, 32, 330
    P, per = 30, 12
    g = torch.Generator().manual_seed(1)
    shape = (P, H, page, d)
    raw = [torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    exps = [torch.randint(0, 256, shape[:3], generator=g, dtype=torch.uint8) for _ in range(2)]
    cache = kv.PagedKVCache(*raw, *exps)
    table = table_for(B, per, P, 2)
    lens = torch.tensor([n, 97], dtype=torch.int32)
    x = [rand(B, H, n, d, seed=3 + i) for i in range(2)]
    pages = [ref.append(c, e, table, y, torch.zeros(B, dtype=torch.int32), lens) for c, e, y in ((cache.k, cache.k_exp, x[0]), (cache.v, cache.v_exp, x[1]))]
    cache = kv.PagedKVCache(pages[0][0], pages[1][0], pages[0][1], pages[1][1])
    table[1, 1] = -1
    q = rand(B, H, Lq, d, seed=9)
    k, there = ref.read(cache.k, cache.k_exp, table, lens, n)
    v, _ = ref.read(cache.v, cache.v_exp, table, lens, n)
    for causal in (False, True):
        o, (M, L) = kv.paged_attn(q.cuda(), to_gpu(cache), table.cuda(), lens.cuda(), causal=causal)
        check_attn(o, M, L, *ref.paged_attn(q, k, v, there, lens, d ** -0.5, causal), q, k, d ** -0.5, n)


def test_paged_attn_operands_of_other_layouts():
    """Queries with a head axis of stride 0 and as a slice of longer rows; one page table, one row, for all sequences; lengths as a slice."""
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, d, page, n = 3, 4, 2, 64, 16, 90
    cache = kv.PagedKVCache.alloc(8, Hkv, d, page)
    one = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    x = [rand(1, Hkv, n, d, seed=i).cuda() for i in range(2)]
    kv.kv_cache_append(cache, *x, one, torch.zeros(1, dtype=torch.int32, device="cuda"))
    table = one.expand(B, 6)
    lens = torch.tensor([[90, 0], [33, 0], [64, 0]], dtype=torch.int32, device="cuda")[:, 0]
    wide = rand(B, 1, 2, 2 * d, seed=5).cuda()
    q = wide[..., d:].expand(B, H, 2, d)
    o, (M, L) = kv.paged_attn(q, cache, table, lens, causal=True)
    o2, (M2, L2) = kv.paged_attn(q.contiguous(), cache, table.contiguous(), lens.contiguous(), causal=True)
    assert torch.equal(o, o2) and torch.equal(M, M2) and torch.equal(L, L2) and torch.equal(o[:, 0], o[:, 1])
    k, v = (t.double().cpu().expand(B, Hkv, n, d) for t in x)
    check_attn(o, M, L, *ref.paged_attn(q.cpu(), k, v, torch.ones(B, n, dtype=torch.bool), lens.cpu(), d ** -0.5, True), q.cpu(), k, d ** -0.5, n)


@pytest.mark.parametrize("Lq", [1, 24, 100])
def test_entry_point_without_workspace(Lq):
    """No workspace: no sequence is cut, the same result but for the order of the sums; a workspace that is too small is not used."""
    from lvar_amd import _lib, kv_cache_ops as kv
    o, M, L, args = attn_case(2, 4, 2, Lq, [1800, 300], 128, 32, torch.bfloat16, True, seed=3)
    q, cache, table, lens = args[:4]
    lib = _lib.load()
    need = lib.lvar_paged_attn_workspace_bytes(2, 4, 2, Lq, 1800, 128)
    assert need > 0
    small = torch.full((1024,), 7, dtype=torch.uint8, device="cuda")
    for ws, size in ((None, 0), (small.data_ptr(), 1024)):
        o2, M2, L2 = torch.full_like(o, 9), torch.full_like(M, 9), torch.full_like(L, 9)
        st = lib.lvar_paged_attn_fwd(kv._view(q), kv._cache_arg(cache, table, 2, q.device), lens.data_ptr(), None, o2.data_ptr(), M2.data_ptr(), L2.data_ptr(), ws, size,
                                     2, 4, Lq, 1 << 30, 1, 128 ** -0.5, kv._stream(q))
        assert st == 0
        # two roundings of the same sum; maxima are exact, the sums' terms differ by the reference that they count from
        assert torch.equal(M2, M) and torch.allclose(L2, L, rtol=2e-5) and float((o2.float() - o.float()).abs().max()) <= 2 * BF16 * float(o.float().abs().max())
    assert bool((small == 7).all())


def test_staged_tiles_first_called_under_capture():
    """Tiles of many rows raise their kernel's LDS limit on the first call; that call may be a captured one."""
    from lvar_amd import kv_cache_ops as kv
    cache = kv.PagedKVCache.alloc(40, 1, 256, 16)
    x = [rand(1, 1, 600, 256, seed=i).cuda() for i in range(2)]
    table, lens = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40), torch.tensor([600], dtype=torch.int32, device="cuda")
    kv.kv_cache_append(cache, *x, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = rand(1, 1, 77, 256, seed=4).cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, (M, L) = kv.paged_attn(q, cache, table, lens, causal=True)
    for r in range(3):
        q.copy_(rand(1, 1, 77, 256, seed=10 + r))
        e, (Me, Le) = kv.paged_attn(q, cache, table, lens, causal=True)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(o, e) and torch.equal(M, Me) and torch.equal(L, Le)


def test_two_appends_and_reads_on_two_streams():
    from lvar_amd import kv_cache_ops as kv
    B, H, d, n = 2, 4, 128, 500
    x = [rand(B, H, n, d, seed=i).cuda() for i in range(2)]
    table, start = table_for(B, 8, 16, 1).cuda(), torch.zeros(B, dtype=torch.int32, device="cuda")
    lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c = kv.PagedKVCache.alloc(16, H, d, 64, torch.float8_e4m3fn)
            kv.kv_cache_append(c, *x, table, start)
            got.append(kv.kv_cache_read(c, table, lens, n) + kv.paged_attn(x[0], c, table, lens)[:1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_cache_views_and_shared_pages(dtype):
    """Keys and values as views of one buffer [pages, 2, heads, page, d]; two sequences whose first pages are the same, one page named twice in a row."""
    from lvar_amd import kv_cache_ops as kv
    P, H, page, d, n = 9, 3, 16, 64, 40
    raw = torch.zeros(P, 2, H, page, d, dtype=torch.bfloat16 if dtype is torch.bfloat16 else torch.uint8, device="cuda")
    exps = torch.full((P, 2, H, page), 127, dtype=torch.uint8, device="cuda")
    buf = raw if dtype is torch.bfloat16 else raw.view(dtype)
    cache = kv.PagedKVCache(buf[:, 0], buf[:, 1], *(() if dtype is torch.bfloat16 else (exps[:, 0], exps[:, 1])))
    plain = kv.PagedKVCache.alloc(P, H, d, page, dtype)
    x = [rand(1, H, n, d, seed=i).cuda() for i in range(2)]
    first = torch.tensor([[4, 2, 7]], dtype=torch.int32, device="cuda")
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    for c in (cache, plain):
        kv.kv_cache_append(c, *x, first, start)
    assert all(torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, plain) if a is not None)
    table = torch.tensor([[4, 2, 7], [4, 2, 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([40, 48], dtype=torch.int32, device="cuda")
    for Lq in (1, 40):
        q = rand(2, 2 * H, Lq, d, seed=9).cuda()
        got, want = (kv.paged_attn(q, c, table, lens, causal=True) for c in (cache, plain))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1][0], want[1][0]) and torch.equal(got[1][1], want[1][1])
        k, v = (t.double().cpu() for t in kv.kv_cache_read(cache, table, lens))
        assert torch.equal(k[0, :, :32], k[1, :, :32]) and torch.equal(k[1, :, 16:32], k[1, :, 32:])
        check_attn(*[t for t in (got[0], *got[1])], *ref.paged_attn(q.cpu(), k, v, torch.arange(48)[None] < lens.cpu()[:, None], lens.cpu(), d ** -0.5, True), q.cpu(), k, d ** -0.5, 48)


def test_large_forms_of_the_norm():
    """Calls large enough for four heads per workgroup, in both pair orders, with heads that do not fill the last chunk."""
    from lvar_amd import kv_cache_ops as kv
    for d, H, Hkv, inter, norm in ((16, 14, 7, True, "l2"), (32, 6, 6, False, "rms"), (64, 10, 5, False, "l2"), (128, 7, 7, True, "rms"), (256, 5, 5, False, None)):
        L = 4 * 1024 * 256 // 4 // d * 4 // (H + Hkv) * 2 + 1
        q, k, _ = projection(1, H, Hkv, L, d, seed=d)
        w = [weight("full", h, d, 7 + i) for i, h in enumerate((H, Hkv))]
        cos, sin = tables(L, d // 2)
        got = kv.qk_norm_rope(q.cuda(), k.cuda(), cos.cuda(), sin.cuda(), None, w[0].cuda(), w[1].cuda(), norm, None, inter)
        at = ref.table_rows(1, L, L)
        for x, y, wx in ((q, got[0], w[0]), (k, got[1], w[1])):
            check_rows(y, ref.norm_rope(x, wx, cos, sin, at, norm, EPS[norm], inter), (d, norm))


# ---- together ----

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_image_schedule(dtype):
    """The scales of an image: every scale is normalised, rotated and appended in one launch and attends to all tokens so far; the paged
    attention and the dense attention on what is read back agree, and a block-sparse and a column-sum call take the same tensors."""
    from lvar_amd import kv_cache_ops as kv, sparse_attn_ops as ops
    B, H, d, page = 2, 4, 128, 64
    sides = (1, 2, 4, 6, 8, 12)
    total = sum(s * s for s in sides)
    per = -(-total // page)
    cache = kv.PagedKVCache.alloc(B * per, H, d, page, dtype)
    table = table_for(B, per, B * per, 2).cuda()
    cos, sin = (t.cuda() for t in tables(total, d // 2))
    w = (4 * weight("head", H, d, 1)).cuda()
    done = 0
    for side in sides:
        n = side * side
        q, k, v = (t.cuda() for t in projection(B, H, H, n, d, seed=side))
        start = torch.full((B,), done, dtype=torch.int32, device="cuda")
        q = kv.qk_norm_rope_append(cache, q, k, v, table, start, cos, sin, q_weight=w)
        done += n
        lens = torch.full((B,), done, dtype=torch.int32, device="cuda")
        o, (M, L) = kv.paged_attn(q, cache, table, lens, scale=1.0)
        ck, cv = kv.kv_cache_read(cache, table, lens, done)
        o2, (M2, L2) = ops.dense_attn(q, ck, cv, scale=1.0)
        kr, vr = ck.double().cpu(), cv.double().cpu()
        r = ref.paged_attn(q.cpu(), kr, vr, torch.ones(B, done, dtype=torch.bool), [done] * B, 1.0)
        check_attn(o, M, L, *r, q.cpu(), kr, 1.0, done)
        assert bool(((o.float() - o2.float()).abs() <= 2e-2 + 1e-2 * o2.float().abs()).all()) and float((M - M2).abs().max()) < 1e-3
    cs = ops.colsum(q, ck, 1.0, 192, lse=(M, L))
    assert cs.shape == (B, H, 1, total) and torch.allclose(cs.sum(-1), torch.full((B, H, 1), float(n), device="cuda"), rtol=1e-3)
    scores = ops.window_key_scores(q, ck, torch.arange(total - 16, total, device="cuda").expand(B, H, 16).contiguous())
    assert scores.shape == (B, H, total)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_host_paths_give_the_same(dtype, monkeypatch):
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, L, d, page, P = 2, 4, 2, 21, 128, 32, 20
    table = table_for(B, P // B, P, 1).cuda()
    start, lens = torch.tensor([250, 3], dtype=torch.int32, device="cuda"), torch.tensor([271, 24], dtype=torch.int32, device="cuda")
    cos, sin = (t.cuda() for t in tables(300, d // 2))
    q, k, v = (t.cuda() for t in projection(B, H, Hkv, L, d, seed=3))
    got = []
    for native in (kv._native, lambda: None):
        monkeypatch.setattr(kv, "_native", native)
        c = to_gpu(make_cache(P, Hkv, page, d, dtype, 5))
        kv.kv_cache_append(c, v, k, table, start)
        oq = kv.qk_norm_rope_append(c, q, k, v, table, start, cos, sin, counts=lens - start)
        o, (M, L_) = kv.paged_attn(oq, c, table, lens, causal=True, counts=lens - start)
        got.append((oq, *kv.kv_cache_read(c, table, lens, L, start), o, M, L_, *(t.view(torch.uint8) for t in c if t is not None)))
    for a, b in zip(*got):
        assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- refusals ----

@pytest.mark.parametrize("binding", [True, False])
def test_refusals_on_the_device(binding, monkeypatch):
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    x = rand(2, 2, 3, 64).cuda()
    c = kv.PagedKVCache.alloc(4, 2, 64, 16)
    c8 = kv.PagedKVCache.alloc(4, 2, 64, 16, torch.float8_e4m3fn)
    table, i = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cos, sin = (t.cuda() for t in tables(3, 32))

    def refused(error, f, *a, **kw):
        with pytest.raises(error):
            f(*a, **kw)
    S, T = kv.ShapeError, TypeError
    nr, ap, rd, at = kv.qk_norm_rope, kv.kv_cache_append, kv.kv_cache_read, kv.paged_attn
    # norm
    refused(S, nr, x, x[:, :, :2]), refused(S, nr, x[:, :1], x), refused(S, nr, x, x, norm="max"), refused(S, nr, x, x, eps=-1.0), refused(S, nr, x, x, eps=math.nan)
    refused(S, nr, x, x, cos), refused(S, nr, x, x, cos[:, :20], sin[:, :20]), refused(S, nr, x, x, cos[:2], sin[:2]), refused(T, nr, x, x, cos.double(), sin.double())
    refused(S, nr, x, x, cos.cpu(), sin.cpu()), refused(S, nr, x, x, torch.ones(3, 48, device="cuda"), torch.ones(3, 48, device="cuda"))
    refused(RuntimeError, nr, x, x, cos.clone().requires_grad_(), sin)
    refused(T, nr, x, x, cos, sin, torch.zeros(3, device="cuda")), refused(S, nr, x, x, cos, sin, torch.zeros(2, device="cuda", dtype=torch.int32))
    refused(S, nr, x, x, cos, sin, torch.zeros(3, dtype=torch.int32))
    refused(S, nr, x, x, q_weight=torch.ones(3, 64, device="cuda")), refused(S, nr, x, x, k_weight=torch.ones(2, device="cuda")), refused(T, nr, x, x, k_weight=torch.ones(64, device="cuda").half())
    refused(S, nr, x, x, k_weight=torch.ones(64)), refused(S, nr, rand(1, 1, 2, 48).cuda(), rand(1, 1, 2, 48).cuda()), refused(T, nr, x.half(), x.half())
    # cache
    refused(S, ap, c, x, x[:, :1], table, i), refused(S, ap, c, x[:, :1], x[:, :1], table, i), refused(S, ap, c, x, x, table[:1], i), refused(T, ap, c, x, x, table.long(), i)
    refused(T, ap, c, x, x, table, i.long()), refused(S, ap, c, x, x, table, i[:1]), refused(S, ap, c, x, x, table, None), refused(S, ap, c, x, x, table, i, i[:1])
    refused(S, ap, c, x, x, table.cpu(), i), refused(S, ap, c, x, x, table, i.cpu()), refused(S, ap, c._replace(v=c.v[:, :, :8]), x, x, table, i)
    refused(T, ap, c._replace(v=c8.v), x, x, table, i), refused(S, ap, c._replace(k_exp=c8.k_exp, v_exp=c8.v_exp), x, x, table, i)
    refused(S, ap, c8._replace(k_exp=None), x, x, table, i), refused(T, ap, c8._replace(k_exp=c8.k_exp.int(), v_exp=c8.v_exp.int()), x, x, table, i)
    refused(S, ap, kv.PagedKVCache(*(torch.zeros(4, 2, 24, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))), x, x, table, i)
    refused(S, ap, c._replace(v=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device="cuda").transpose(1, 2)), x, x, table, i)      # other strides than k
    refused(S, ap, kv.PagedKVCache(*(torch.zeros(4, 2, 16, 68, dtype=torch.bfloat16, device="cuda")[..., 4:] for _ in range(2))), x, x, table, i)   # rows not aligned
    refused(S, ap, kv.PagedKVCache(*(torch.zeros(4, 2, 1, 64, dtype=torch.bfloat16, device="cuda").expand(4, 2, 16, 64) for _ in range(2))), x, x, table, i)   # rows on top of each other
    refused(S, rd, c, table, None), refused(S, rd, c, table, i, -1), refused(T, rd, c, table, i.float()), refused(S, rd, c, table, i, 3, i[:1])
    # attention
    refused(S, at, x[:, :1], c, table, i), refused(S, at, rand(2, 2, 3, 128).cuda(), c, table, i), refused(S, at, x[:1], c, table, i), refused(S, at, x, c, table, None)
    refused(T, at, x.half(), c, table, i), refused(T, at, x, c, table, i.long()), refused(S, at, x, c, table, i, max_len=-1)
    refused(RuntimeError, at, x.clone().requires_grad_(), c, table, i), refused(Exception, at, x, c, table, i, -1.0)
    # more workgroups than a launch holds (the entry point says so before it launches anything)
    from lvar_amd import _lib
    many = kv._cache_arg(c, table, x.shape[0], x.device)
    many.kv_heads = 16384
    assert _lib.load().lvar_paged_attn_fwd(kv._view(x), many, i.data_ptr(), None, x.data_ptr(), x.data_ptr(), x.data_ptr(), None, 0, 4096, 16384, 1, 100, 0, 1.0, kv._stream(x)) == -1
    torch.cuda.synchronize()


# ---- derivatives, versions and values that are not there ----

def small_call(dtype=torch.bfloat16):
    """q, k, v, cache, table, start, lengths of a small step on the device"""
    from lvar_amd import kv_cache_ops as kv
    q, k, v = (t.cuda() for t in projection(2, 4, 2, 3, 64, seed=1))
    cache = kv.PagedKVCache.alloc(4, 2, 64, 16, dtype)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    return q, k, v, cache, table, torch.zeros(2, dtype=torch.int32, device="cuda"), torch.full((2,), 3, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("binding", [True, False])
def test_tangents_are_refused(binding, monkeypatch):
    """Tensors with a forward-mode tangent: no operator may hand back outputs that have lost it."""
    import torch.autograd.forward_ad as fw
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    q, k, v, cache, table, start, lens = small_call()
    w, (cos, sin) = torch.ones(64, device="cuda"), (t.cuda() for t in tables(3, 32))
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (lambda: kv.qk_norm_rope(dual(q), k), lambda: kv.qk_norm_rope(q, dual(k)), lambda: kv.qk_norm_rope(q, k, q_weight=dual(w)),
                  lambda: kv.qk_norm_rope(q, k, k_weight=dual(w)), lambda: kv.qk_norm_rope(q, k, dual(cos), sin), lambda: kv.qk_norm_rope(q, k, cos, dual(sin)),
                  lambda: kv.qk_norm_rope(dual(q).transpose(0, 1), k.transpose(0, 1)),
                  lambda: kv.kv_cache_append(cache, dual(k), v, table, start), lambda: kv.kv_cache_append(cache, k, dual(v), table, start),
                  lambda: kv.qk_norm_rope_append(cache, dual(q), k, v, table, start), lambda: kv.qk_norm_rope_append(cache, q, k, v, table, start, k_weight=dual(w)),
                  lambda: kv.qk_norm_rope_append(cache, q, k, v, table, start, cos, dual(sin)), lambda: kv.paged_attn(dual(q), cache, table, lens)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    f()
        leaf = q.detach().clone().requires_grad_()
        o, _ = kv.qk_norm_rope(leaf, k)
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(o, leaf, dual(torch.ones_like(o)))
        # plain tensors are taken as ever
        assert torch.equal(kv.qk_norm_rope(leaf, k)[0], kv.qk_norm_rope(q, k)[0])
        kv.kv_cache_append(cache, k, v, table, start)
    assert torch.equal(kv.kv_cache_read(cache, table, lens, 3)[0], k)


@pytest.mark.parametrize("Lq,H", [((1 << 26) + 37, 1), ((1 << 25) + 1, 2)])
def test_padding_of_more_than_31_bits_of_pieces(Lq, H):
    """2^26 rows of head_dim 256 behind one new token: 2^31 pieces of 16 bytes, all of them written."""
    from lvar_amd import _lib, kv_cache_ops as kv
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 36 GB")
    d = 256
    cache = kv.PagedKVCache.alloc(4, 1, d, 16)
    x = [rand(1, 1, 40, d, seed=i).cuda() for i in range(2)]
    table, zero = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), torch.zeros(1, dtype=torch.int32, device="cuda")
    kv.kv_cache_append(cache, *x, table, zero)
    lens, counts = zero + 40, zero + 1
    q = rand(1, 1, 1, d, seed=5).cuda()
    o, M, L = torch.full((H * Lq, d), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full((H * Lq,), 7.0, device="cuda"), torch.full((H * Lq,), 7.0, device="cuda")
    rows = _lib.LvarTensor(q.data_ptr(), 0, 0, 0)           # (every query is the same row)
    assert _lib.load().lvar_paged_attn_fwd(rows, kv._cache_arg(cache, table, 1, q.device), lens.data_ptr(), counts.data_ptr(), o.data_ptr(), M.data_ptr(), L.data_ptr(), None, 0,
                                           1, H, Lq, 64, 1, d ** -0.5, kv._stream(q)) == 0
    one, (M1, L1) = kv.paged_attn(q, cache, table, lens)
    o, M, L = o.view(H, Lq, d), M.view(H, Lq), L.view(H, Lq)
    for h in range(H):
        # both are rounded, and the call of many rows rounds its probabilities
        assert float((o[h, 0].float() - one[0, 0, 0].float()).abs().max()) <= 3 * BF16 * float(x[1].abs().max()) and float((M[h, 0] - M1.view(())).abs()) <= 2 * (d + 8) * F32 * float(M1.abs().max() + 10)
        assert all(bool((c == 0).all()) for c in o[h, 1:].split(1 << 22))
        assert bool((M[h, 1:] == -math.inf).all()) and bool((L[h, 1:] == 1).all())
    del o, M, L
    torch.cuda.empty_cache()


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_caches_that_need_a_gradient_are_refused(dtype, binding, monkeypatch):
    """Learned keys and values as pages: the operators have no gradient for them and say so, but take them where none is wanted."""
    import torch.autograd.forward_ad as fw
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    q, k, v, cache, table, start, lens = small_call(dtype)
    calls = (lambda c: kv.kv_cache_append(c, k, v, table, start), lambda c: kv.qk_norm_rope_append(c, q, k, v, table, start), lambda c: kv.kv_cache_read(c, table, lens, 3),
             lambda c: kv.paged_attn(q, c, table, lens))
    for name in ("k", "v"):
        learned = cache._replace(**{name: getattr(cache, name).detach().clone().requires_grad_()})
        for f in calls:
            with pytest.raises(RuntimeError, match="no backward"):
                f(learned)
            with torch.no_grad():
                f(learned)
        if dtype is torch.bfloat16:
            with fw.dual_level():
                dual = cache._replace(**{name: fw.make_dual(getattr(cache, name), torch.ones_like(cache.k))})
                for f in calls:
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        f(dual)


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_writing_a_cache_counts_as_a_change(dtype, binding, monkeypatch):
    """Autograd finds out that a cache it has saved was written; a cache made in inference mode has no counter."""
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    q, k, v, cache, table, start, lens = small_call(dtype)
    for f in (lambda c: kv.kv_cache_append(c, k, v, table, start), lambda c: kv.qk_norm_rope_append(c, q, k, v, table, start)):
        before = [t._version for t in cache if t is not None]
        if dtype is torch.bfloat16:
            x = torch.ones(64, dtype=dtype, device="cuda", requires_grad=True)
            y = (cache.k * x).sum()
        f(cache)
        assert all(t._version > n for t, n in zip((t for t in cache if t is not None), before))
        if dtype is torch.bfloat16:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
        before = [t._version for t in cache if t is not None]
        kv.kv_cache_read(cache, table, lens, 3), kv.paged_attn(q, cache, table, lens)
        assert [t._version for t in cache if t is not None] == before
        with torch.inference_mode():
            made = kv.PagedKVCache.alloc(4, 2, 64, 16, dtype)
            f(made)
        with torch.no_grad():
            f(made)
        assert torch.equal(made.k.view(torch.uint8), cache.k.view(torch.uint8))


@pytest.mark.parametrize("binding", [True, False])
def test_no_query_heads_are_refused(binding, monkeypatch):
    """0 is a multiple of the key heads, but a call without queries would hand back keys that nobody wrote."""
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    q, k, v, cache, table, start, lens = small_call()
    for f in (lambda: kv.qk_norm_rope(q[:, :0], k), lambda: kv.qk_norm_rope_append(cache, q[:, :0], k, v, table, start), lambda: kv.paged_attn(q[:, :0], cache, table, lens)):
        with pytest.raises(kv.ShapeError):
            f()


@pytest.mark.parametrize("binding", [True, False])
def test_eps_below_the_normal_numbers_is_refused(binding, monkeypatch):
    """Its reciprocal is no fp32 number (rows of zeros would come out as NaN); the least normal one is fine."""
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    q, k, v, cache, table, start, _ = small_call()
    q = q.clone()
    q[:, :, 1] = 0
    for norm in ("l2", "rms"):
        for eps in (1e-39, 1e-60, 5e-324, 1e39):
            for x in (q, q.detach().clone().requires_grad_()):
                with pytest.raises(kv.ShapeError):
                    kv.qk_norm_rope(x, k, norm=norm, eps=eps)
            with pytest.raises(kv.ShapeError):
                kv.qk_norm_rope_append(cache, q, k, v, table, start, norm=norm, eps=eps)
        x = q.detach().clone().requires_grad_()
        o, _ = kv.qk_norm_rope(x, k, norm=norm, eps=2.0 ** -126)
        assert bool(torch.isfinite(o).all()) and float(o[:, :, 1].abs().sum()) == 0


def leak_case(Lq, H, Hkv, d, lengths, dtype, page=16, counts=None):
    """Causal calls whose newest values hold infinities and NaN: column by column, rows that see one are not finite, all others are what they are without it."""
    from lvar_amd import kv_cache_ops as kv
    B, n = len(lengths), max(lengths)
    per = -(-n // page)
    table = table_for(B, per, B * per + 1, 3)
    x = [rand(B, Hkv, n, d, seed=20 + i) for i in range(2)]
    lens, zero = torch.tensor(lengths, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    new = [Lq] * B if counts is None else counts
    g = torch.Generator().manual_seed(Lq + d)
    bad = torch.zeros(B, Hkv, n, d, dtype=torch.bool)
    for b in range(B):
        first = max(0, lengths[b] - new[b])
        for j in {lengths[b] - 1, first + (lengths[b] - first) // 2, min(first + 1, lengths[b] - 1), max(0, lengths[b] - 33)}:
            for h in range(Hkv):
                bad[b, h, j, torch.randint(0, d, (3,), generator=g)] = True
    kinds = torch.tensor([math.inf, -math.inf, math.nan]).to(torch.bfloat16)
    spoiled = torch.where(bad, kinds[torch.randint(0, 3, bad.shape, generator=g)], x[1])
    caches = []
    for v in (torch.where(bad, torch.zeros((), dtype=torch.bfloat16), x[1]), spoiled):
        c = to_gpu(make_cache(B * per + 1, Hkv, page, d, dtype, 6))
        kv.kv_cache_append(c, x[0].cuda(), v.cuda(), table.cuda(), zero.cuda(), lens.cuda())
        caches.append(c)
    q = rand(B, H, Lq, d, seed=9)
    c = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    (o, (M, L)), (want, (Mw, Lw)) = (kv.paged_attn(q.cuda(), x, table.cuda(), lens.cuda(), causal=True, counts=cu(c)) for x in (caches[1], caches[0]))
    assert torch.equal(M, Mw) and torch.equal(L, Lw)
    # which (row, column) sees which value
    i = torch.arange(Lq)
    limit = torch.stack([torch.where(i < new[b], lengths[b] - new[b] + i + 1, 0) for b in range(B)])      # [B, Lq]
    sees = (torch.arange(n) < limit[..., None]).double()                                                  # [B, Lq, n]
    hit = torch.matmul(sees[:, None], bad.double()) > 0                                                   # [B, Hkv, Lq, d]
    hit = hit.repeat_interleave(H // Hkv, 1)
    assert bool(hit.any()) and not bool(hit.all())
    o, want = o.cpu(), want.cpu()
    assert bool(torch.isfinite(want).all())
    assert not bool(torch.isfinite(o[hit]).any()), "a row that sees a value which is not finite"
    assert torch.equal(o[~hit], want[~hit]), f"{int((~(o == want))[~hit].sum())} results of rows that do not see one"


LEAK_CASES = [
    # Lq, H, Hkv, d, lengths, counts
    (4, 2, 2, 64, [40, 4], None), (4, 2, 2, 128, [130, 70], None), (3, 2, 1, 256, [33, 300], None),          # up to 16 rows
    (29, 2, 2, 64, [64, 200], None), (13, 4, 2, 128, [13, 77], [13, 5]),                                     # up to 32
    (50, 2, 2, 64, [50, 190], None), (60, 2, 2, 128, [129, 61], [60, 31]),                                   # staged, 64 rows
    (70, 4, 2, 64, [500, 70], None), (200, 2, 1, 128, [200, 1300], None), (70, 1, 1, 256, [75, 600], None),  # several row tiles, cut
    (5, 2, 2, 128, [2500, 700], None), (5, 2, 2, 256, [1500, 64], None),                                     # cut and joined
]


@pytest.mark.parametrize("case", LEAK_CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_values_that_are_not_finite_stay_behind_the_causal_border(case, dtype):
    Lq, H, Hkv, d, lengths, counts = case
    leak_case(Lq, H, Hkv, d, lengths, dtype, counts=counts)


@pytest.mark.parametrize("Lq,d", [(1, 128), (2, 64), (9, 256), (40, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_values_that_are_not_finite_reach_who_sees_them(Lq, d, dtype):
    """Anywhere in the cache, beside pages that are missing and behind the causal border or not."""
    from lvar_amd import kv_cache_ops as kv
    n, page = 331, 16
    table = torch.arange(21, dtype=torch.int32).view(1, 21)
    k, v = (rand(1, 1, n, d, seed=i) for i in (1, 2))
    for spot in (0, 5, 40, 200, 319, 320, n - Lq, n - 1):
        for x in (math.inf, math.nan):
            w = v.clone()
            w[0, 0, spot, d // 3] = x
            c = to_gpu(make_cache(22, 1, page, d, dtype, 6))
            kv.kv_cache_append(c, k.cuda(), w.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
            holes = table.clone()
            holes[0, 1] = holes[0, min(spot // 16 ^ 1, 19)] = -1          # (of 16 keys beside it)
            seen = int(holes[0, spot // 16]) >= 0
            for causal in (False, True):
                o, _ = kv.paged_attn(rand(1, 2, Lq, d, seed=3).cuda(), c, holes.cuda(), torch.full((1,), n, dtype=torch.int32, device="cuda"), causal=causal)
                rows = torch.arange(n - Lq, n) >= spot if causal else torch.ones(Lq, dtype=torch.bool)
                want = torch.ones(Lq, d, dtype=torch.bool)
                want[:, d // 3] = ~(rows & seen)
                assert torch.equal(torch.isfinite(o[0]).cpu(), want.expand(2, Lq, d)), (spot, x, causal)
        # a key: whole rows
        w = k.clone()
        w[0, 0, spot, d // 3] = math.nan
        c = to_gpu(make_cache(22, 1, page, d, dtype, 6))
        kv.kv_cache_append(c, w.cuda(), v.cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
        o, _ = kv.paged_attn(rand(1, 2, Lq, d, seed=3).cuda(), c, table.cuda(), torch.full((1,), n, dtype=torch.int32, device="cuda"), causal=True)
        rows = torch.arange(n - Lq, n) < spot
        assert torch.equal(torch.isfinite(o[0]).cpu(), rows[:, None].expand(2, Lq, d)), (spot, "key")


@pytest.mark.parametrize("binding", [True, False])
def test_rows_at_odd_places(binding, monkeypatch):
    """Unit stride on d is all that a tensor needs: bases between 16-byte borders, and odd strides of axes of one element, which count as contiguous."""
    from lvar_amd import kv_cache_ops as kv
    if not binding:
        monkeypatch.setattr(kv, "_native", lambda: None)
    d = 64
    table, zero = torch.arange(2, dtype=torch.int32, device="cuda").view(1, 2), torch.zeros(1, dtype=torch.int32, device="cuda")
    flat = rand(4 * 300, seed=1).cuda()
    places = [lambda i: flat[i * 300 + 1:i * 300 + 1 + d].view(1, 1, 1, d),                                  # contiguous, 2 bytes behind a border
              lambda i: flat.as_strided((1, 1, 1, d), (131, 67, 3, 1), i * 304),                              # aligned, odd strides
              lambda i: flat.as_strided((1, 1, 3, d), (131, 67, 72, 1), i * 304)]
    for place in places:
        x = [place(i) for i in range(4)]
        y = [t.clone(memory_format=torch.contiguous_format) for t in x]
        got, want = [], []
        for ts, out in ((x, got), (y, want)):
            q, k, v, g = ts
            cache = kv.PagedKVCache.alloc(2, 1, d, 16)
            out += kv.qk_norm_rope(q, k)
            out.append(kv.qk_norm_rope_append(cache, q, k, v, table, zero))
            kv.kv_cache_append(cache, k, v, table, zero + 5)
            lens = zero + 5 + k.shape[2]
            out += [cache.k, cache.v, kv.paged_attn(q, cache, table, lens)[0]]
            a, b = (t.detach().requires_grad_() for t in (q, k))
            o = kv.qk_norm_rope(a, b)
            out += torch.autograd.grad(o, (a, b), (g, v))
        assert all(torch.equal(s, t) for s, t in zip(got, want))
