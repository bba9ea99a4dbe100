"""What a serving and a training program do with the operators around packed prompts and cache pages, one behind the other: eager against a plain
program in 64 bits, and captured in graphs whose inputs change between the replays."""
import math

import pytest
import torch

from oracle import kv_cache_oracle as kref
from oracle import packed_oracle as ref
from oracle import pages_oracle as pref
from test_gpu_packed import i32, rand

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -24


def grid_positions(lens, side=7):
    """Frame, row and column of each token, as numbers with fractions."""
    at = torch.cat([torch.arange(n) for n in lens]).double()
    return torch.stack([at // (side * side), at // side % side + 0.25, at % side * 0.5]).float()


def test_prompts_to_samples():
    """Rotate packed prompts by three axes, attend, put their keys into pages, fork each into samples, append a token, attend over the pages, keep a part
    of each, give the rest back."""
    from lvar_amd import kv_cache_ops as kv
    from lvar_amd.packed_ops import packed_attn
    lens, H, Hkv, d, page, S, n = [70, 33, 128], 4, 2, 64, 16, 3, 2
    T, B = sum(lens), S * (1 + n)
    off = [0, 70, 103, 231]
    x = rand(1, T, H + 2 * Hkv, d, seed=1).transpose(1, 2)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    pos, freqs = grid_positions(lens), kv.axis_freqs((16, 24, 24), device="cpu")
    gq, gk = kv.qk_norm_rope(q.cuda(), k.cuda(), positions=pos.cuda(), freqs=freqs.cuda(), norm="rms")
    o, _ = packed_attn(gq, gk, v.cuda(), i32(off))
    # (what follows is compared from the kernels' own bf16 queries and keys on)
    r = ref.packed_attn(gq, gk, v, off)
    assert bool(((o.double().cpu() - r["o"]).abs() <= r["t_o"]).all())
    angle = (pos.double()[:, :, None] * freqs[:, None]).sum(0)
    for got, t in ((gq, q), (gk, k)):
        want = kref.norm_rope(t, None, angle.cos(), angle.sin(), torch.arange(T)[None], "rms", 1e-6, True)
        assert bool(((got.double().cpu() - want).abs() <= BF16 * want.abs() + (d + 40) * F32 * want.abs().amax(-1, keepdim=True)).all())

    P, width = 80, 10
    cache = kv.PagedKVCache.alloc(P, Hkv, d, page_size=page)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    lengths = torch.tensor(lens + [0] * (S * n), dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(lengths)
    kv.kv_pages_alloc(refs, table, zero, (lengths + page - 1) // page)
    Lmax = max(lens)
    padded = [torch.zeros(S, Hkv, Lmax, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for b in range(S):
        for t, src in zip(padded, (gk, v.cuda())):
            t[b, :, :lens[b]] = src[0, :, off[b]:off[b + 1]]
    kv.kv_cache_append(cache, *padded, table[:S], zero[:S], counts=lengths[:S])
    source, target = i32([b for b in range(S) for _ in range(n)]), i32(range(S, B))
    kv.kv_cache_fork(cache, refs, table, source, target, lengths)
    lengths[S:] = lengths[source.long()]
    samples = table[S:]
    kv.kv_pages_alloc(refs, samples, (lengths[S:] + page - 1) // page, (lengths[S:] + page) // page)    # a page where none is started
    named = table[table >= 0].tolist()
    assert refs.tolist() == [named.count(p) for p in range(P)]
    new = [rand(S * n, h, 1, d, seed=20 + i).cuda() for i, h in enumerate((H, Hkv, Hkv))]
    kv.kv_cache_append(cache, new[1], new[2], samples, lengths[S:])
    o, _ = kv.paged_attn(new[0], cache, samples, lengths[S:] + 1)
    lines = []
    for i in range(S * n):
        b = i // n
        kk = torch.cat([gk[0, :, off[b]:off[b + 1]].cpu(), new[1][i].cpu()], 1)
        vv = torch.cat([v[0, :, off[b]:off[b + 1]], new[2][i].cpu()], 1)
        lines.append((kk, vv))
        for h in range(H):
            s = ref.sequence(new[0][i, h].double().cpu(), kk[h // 2].double(), vv[h // 2].double(), 1 / math.sqrt(d), False)
            assert bool(((o[i, h].double().cpu() - s["o"]).abs() <= s["t_o"]).all())
    # the prompts are as they were
    back, _ = kv.kv_cache_read(cache, table[:S], lengths[:S], max_len=Lmax)
    assert torch.equal(back, padded[0])
    # 20 tokens of every sample, other ones for every head, in pages of their own
    keep = torch.stack([torch.stack([torch.randperm(lens[i // n] + 1, generator=torch.Generator().manual_seed(i * 7 + h))[:20].sort().values for h in range(Hkv)])
                        for i in range(S * n)]).cuda()
    small = torch.full((S * n, 2), -1, dtype=torch.int32, device="cuda")
    kv.kv_pages_alloc(refs, small, zero[S:], zero[S:] + 2)
    kv.kv_cache_compact(cache, samples, keep, small)
    kv.kv_pages_free(refs, table)
    assert refs.sum() == S * n * 2 and bool((refs[small.flatten().long()] == 1).all()) and bool((table == -1).all())
    gk2, gv2 = kv.kv_cache_read(cache, small, zero[S:] + 20, max_len=20)
    for i, (kk, vv) in enumerate(lines):
        at = keep[i].cpu()[:, :, None].expand(Hkv, 20, d)
        assert torch.equal(gk2[i].cpu(), kk.gather(1, at)) and torch.equal(gv2[i].cpu(), vv.gather(1, at))


def test_a_training_step():
    """Norm, rotation by two axes and attention over packed sequences as one graph of autograd: the gradients of its inputs, against the chain in 64 bits
    from the kernels' own intermediate results on."""
    from lvar_amd import kv_cache_ops as kv
    from lvar_amd.packed_ops import packed_attn
    lens, H, Hkv, d = [50, 0, 77], 4, 2, 64
    off = [0, 50, 50, 127]
    T = 127
    x = rand(1, T, H + 2 * Hkv, d, seed=5)
    pos, freqs = grid_positions(lens)[1:], kv.axis_freqs((32, 32), device="cpu")
    leaf = x.cuda().requires_grad_()
    t = leaf.transpose(1, 2)
    gq, gk = kv.qk_norm_rope(t[:, :H], t[:, H:H + Hkv], positions=pos.cuda(), freqs=freqs.cuda(), norm="l2")
    gq.retain_grad(), gk.retain_grad()
    o, _ = packed_attn(gq, gk, t[:, H + Hkv:], i32(off), scale=8.0)
    go = rand(1, H, T, d, seed=6)
    o.backward(go.cuda())
    r = ref.packed_attn(gq, gk, x.transpose(1, 2)[:, H + Hkv:], off, scale=8.0, go=go)
    for name, got in (("dq", gq.grad), ("dk", gk.grad), ("dv", leaf.grad.transpose(1, 2)[:, H + Hkv:])):
        assert bool(((got.double().cpu() - r[name]).abs() <= r["t_" + name]).all()), name
    angle = (pos.double()[:, :, None] * freqs[:, None]).sum(0)
    xt = x.transpose(1, 2)
    for lo, hi, g in ((0, H, gq.grad), (H, H + Hkv, gk.grad)):
        want, _ = kref.norm_rope_grads(xt[:, lo:hi], None, angle.cos(), angle.sin(), torch.arange(T)[None], "l2", 1e-12, True, g.cpu())
        got = leaf.grad.transpose(1, 2)[:, lo:hi].double().cpu()
        assert bool(((got - want).abs() <= BF16 * want.abs() + (4 * d + 40) * F32 * want.abs().amax(-1, keepdim=True) + 1e-38).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_life_of_pages_in_a_graph(dtype):
    """A step that drops, forks, opens, rotates, appends, attends, compacts, captured twice on states of their own and replayed in turn with other lengths,
    beside the same step run eagerly."""
    from lvar_amd import kv_cache_ops as kv
    Hkv, H, d, page, P, S, n, width = 2, 4, 64, 16, 200, 3, 2, 9
    B = S * (1 + n)
    freqs = kv.axis_freqs((32, 32))
    source, target = i32([b for b in range(S) for _ in range(n)]), i32(range(S, B))
    g = torch.Generator().manual_seed(3)

    def state():
        order = torch.randperm(P, generator=torch.Generator().manual_seed(9))[:S * width].int().view(S, width).cuda()
        table = torch.full((B, width + 2), -1, dtype=torch.int32, device="cuda")
        table[:S, :width] = order
        refs = torch.zeros(P, dtype=torch.int32, device="cuda")
        refs[order.flatten().long()] = 1
        cache = kv.PagedKVCache.alloc(P, Hkv, d, page_size=page, dtype=dtype)
        full = [rand(S, Hkv, width * page, d, seed=40 + i).cuda() for i in range(2)]
        kv.kv_cache_append(cache, *full, order, torch.zeros(S, dtype=torch.int32, device="cuda"))
        return cache, table, refs, torch.full((S * n, 2), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    stay = i32([width] * S + [0] * (S * n))
    x = [torch.zeros(S * n, h, 3, d, dtype=torch.bfloat16, device="cuda") for h in (H, Hkv, Hkv)]
    pos = torch.zeros(S * n, 2, 3, dtype=torch.float32, device="cuda")
    keep = torch.zeros(S * n, Hkv, 20, dtype=torch.int64, device="cuda")
    two = i32([2] * (S * n))
    none = i32([0] * (S * n))

    def step(cache, table, refs, small):
        kv.kv_pages_free(refs, table, stay)
        kv.kv_pages_free(refs, small)
        kv.kv_cache_fork(cache, refs, table, source, target, lengths)
        have = lengths[S:]
        kv.kv_pages_alloc(refs, table[S:], (have + page - 1) // page, (have + 3 + page - 1) // page)
        q = kv.qk_norm_rope_append(cache, *x, table[S:], have, positions=pos, freqs=freqs)
        o, (M, L) = kv.paged_attn(q, cache, table[S:], have + 3, causal=True)
        kv.kv_pages_alloc(refs, small, none, two)
        kv.kv_cache_compact(cache, table[S:], keep, small)
        kk, vv = kv.kv_cache_read(cache, small, none + 20, max_len=20)
        return o, M, L, kk, vv, table.clone(), refs.clone()
    step(*state())
    graphs, outs = [], []
    states = [state() for _ in range(3)]
    for s in states[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s))
        graphs.append(graph)
    for r in range(5):
        have = torch.randint(1, width * page, (S,), generator=g).int()
        have[r % S] = (16, 1, 144, 15, 128)[r]
        lengths.copy_(torch.cat([have, have.repeat_interleave(n)]))
        for t in x:
            t.copy_(rand(*t.shape, seed=r))
        pos.copy_(torch.randn(pos.shape, generator=g) * 30)
        keep.copy_(torch.randint(0, 200, keep.shape, generator=g))
        want = step(*states[2])
        torch.cuda.synchronize()
        for j in (r % 2, 1 - r % 2):
            graphs[j].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[j], want)), (r, j)


def test_gradients_of_the_rotation_in_a_graph():
    """By several axes, with tables (a large call) and without."""
    from lvar_amd import kv_cache_ops as kv
    freqs = kv.axis_freqs((32, 32))
    for B, H, L in ((1, 3, 70), (4, 16, 3000)):
        pos = torch.zeros(2, L, device="cuda")
        w0 = torch.ones(H, 1, device="cuda")

        def grads(leaves, g):
            o = kv.qk_norm_rope(leaves[0], leaves[1], positions=pos, freqs=freqs, q_weight=leaves[2], k_weight=leaves[3])
            return [t.detach() for t in o] + list(torch.autograd.grad(o, leaves, (g, g)))
        make = lambda s: [rand(B, H, L, 64, seed=s + i).cuda().requires_grad_() for i in range(2)] + [w0.clone().requires_grad_() for _ in range(2)]  # noqa: E731
        go = rand(B, H, L, 64, seed=9).cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            grads(make(1), go)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs, leaves = [], [], [make(2), make(4)]
        for j in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(grads(leaves[j], go))
            graphs.append(graph)
        for r in range(4):
            pos.copy_(torch.randn(2, L, generator=torch.Generator().manual_seed(r)) * 100)
            with torch.no_grad():
                leaves[r % 2][0].copy_(rand(B, H, L, 64, seed=50 + r))
            want = [grads([t.detach().clone().requires_grad_() for t in x], go) for x in leaves]
            torch.cuda.synchronize()
            for j in (r % 2, 1 - r % 2):
                graphs[j].replay()
            torch.cuda.synchronize()
            for j in range(2):
                assert all(torch.equal(a, b) for a, b in zip(outs[j], want[j])), (B, r, j)


def test_two_streams():
    """Searches, forks and rotations of two programs at once: each has its own workspace."""
    from lvar_amd import kv_cache_ops as kv
    P, width, page = 30000, 40, 16

    def program(seed):
        cache = kv.PagedKVCache.alloc(P, 1, 64, page_size=page)
        table = torch.full((200, width), -1, dtype=torch.int32, device="cuda")
        refs = torch.zeros(P, dtype=torch.int32, device="cuda")
        refs[::3 + seed] = 1
        lengths = i32([(37 * b + seed) % (width * page) for b in range(200)])
        source, target = i32(range(100)), i32(range(100, 200))
        first = torch.zeros_like(lengths)
        torch.cuda.synchronize()

        def go():
            kv.kv_pages_alloc(refs, table[:100], first[:100], (lengths[:100] + page - 1) // page)
            kv.kv_cache_fork(cache, refs, table, source, target, lengths)
            out = table.clone(), refs.clone()
            kv.kv_pages_free(refs, table)
            return out
        return go
    programs = [program(0), program(1)]
    want = [p() for p in programs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in programs], [[], []]
    for _ in range(5):
        for i, (p, s) in enumerate(zip(programs, streams)):
            with torch.cuda.stream(s):
                got[i].append(p())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for x in g:
            assert all(torch.equal(a, b) for a, b in zip(x, w))


@pytest.fixture(params=["compiled", "ctypes"])
def host_path(request, monkeypatch):
    from lvar_amd import kv_cache_ops
    if request.param == "ctypes":
        monkeypatch.setattr(kv_cache_ops, "_native", lambda: None)


def test_refused_rotations(host_path):
    from lvar_amd import kv_cache_ops as kv
    x = lambda h=2, L=5, d=64: torch.zeros(2, h, L, d, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    f, p = kv.axis_freqs((32, 32)), torch.zeros(2, 5, device="cuda")
    cos = torch.ones(9, 32, device="cuda")
    for kw in [dict(freqs=f), dict(freqs=f, positions=p[0]), dict(freqs=f, positions=p[:, :4]), dict(freqs=f, positions=p.expand(3, 2, 5)), dict(freqs=f[:, :5], positions=p),
               dict(freqs=f[0], positions=p), dict(freqs=f.repeat(5, 1), positions=p.repeat(5, 1)), dict(freqs=f.repeat(1, 2), positions=p), dict(freqs=f.cpu(), positions=p),
               dict(freqs=f, positions=p.cpu()), dict(freqs=f, positions=p, cos=cos, sin=cos), dict(freqs=f[:0], positions=p[:0]), dict(freqs=f[:, :0], positions=p)]:
        with pytest.raises(kv.ShapeError):
            kv.qk_norm_rope(x(), x(), **kw)
    for kw in [dict(freqs=f.bfloat16(), positions=p), dict(freqs=f, positions=p.double()), dict(freqs=f, positions=p.bfloat16()), dict(freqs=f, positions=p.bool())]:
        with pytest.raises(TypeError):
            kv.qk_norm_rope(x(), x(), **kw)
    for kw in [dict(freqs=f.clone().requires_grad_(), positions=p), dict(freqs=f, positions=p.clone().requires_grad_())]:
        with pytest.raises(RuntimeError, match="no gradient"):
            kv.qk_norm_rope(x(), x(), **kw)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(p, p)
        with pytest.raises(RuntimeError, match="forward"):
            kv.qk_norm_rope(x(), x(), freqs=f, positions=dual)
    cache = kv.PagedKVCache.alloc(4, 2, 64, page_size=16)
    with pytest.raises(RuntimeError, match="no gradient|backward"):
        kv.qk_norm_rope_append(cache, x(), x(), x(), i32([[0], [1]]), i32([0, 0]), freqs=f.clone().requires_grad_(), positions=p)
    with pytest.raises(kv.ShapeError):
        kv.qk_norm_rope_append(cache, x(), x(), x(), i32([[0], [1]]), i32([0, 0]), freqs=f)
    for columns in ((), (3, 5), (-2, 4)):
        with pytest.raises(kv.ShapeError):
            kv.axis_freqs(columns)


def test_refused_pages(host_path):
    from lvar_amd import kv_cache_ops as kv
    cache = kv.PagedKVCache.alloc(6, 2, 64, page_size=16)
    refs, table, one = i32([0] * 6), i32([[0, 1], [2, 3]]), i32([0, 0])
    wide = i32([[0, 1, 2, 3], [2, 3, 4, 5]])
    for f in (lambda r, t, x=one: kv.kv_pages_alloc(r, t, x, x), lambda r, t, x=one: kv.kv_pages_free(r, t, x),
              lambda r, t, x=one: kv.kv_cache_fork(cache, r, t, one, one, x)):
        for r, t in ((refs[None], table), (refs, table[0]), (refs, wide[:, ::2]), (refs, table[:1].expand(2, 2)), (refs[::2], table), (refs, table[:0]), (refs, table[:, :0])):
            with pytest.raises(kv.ShapeError):
                f(r, t)
        for r, t in ((refs.long(), table), (refs, table.long())):
            with pytest.raises(TypeError):
                f(r, t)
        for r, t in ((refs.cpu(), table), (refs, table.cpu())):
            with pytest.raises(RuntimeError):
                f(r, t)
        with pytest.raises(kv.ShapeError):
            f(refs, table, i32([0, 0, 0]))
        with pytest.raises(TypeError):
            f(refs, table, one.long())
    with pytest.raises(kv.ShapeError):
        kv.kv_cache_fork(cache, refs[:5], table, one, one, one)
    with pytest.raises(kv.ShapeError):
        kv.kv_cache_fork(cache, refs, table, one, one[:1], one)
    with pytest.raises(kv.ShapeError):
        kv.kv_cache_fork(cache, refs, table, one[None], one[None], one)
    keep = torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda")
    for a in ((table, keep[0], table), (table, keep[:, :1], table), (table, keep, table[:1]), (table[:1], keep, table), (table, keep.cpu(), table), (table, keep, table, i32([1])),
              (table, keep, table[:, :0]), (wide[:, ::2], keep, table)):
        with pytest.raises(kv.ShapeError):
            kv.kv_cache_compact(cache, *a)
    for a in ((table, keep.short(), table), (table, keep.float(), table), (table.long(), keep, table), (table, keep, table.long()), (table, keep, table, one.long())):
        with pytest.raises(TypeError):
            kv.kv_cache_compact(cache, *a)
    grad = kv.PagedKVCache(cache.k.clone().requires_grad_(), cache.v)
    for f in (lambda: kv.kv_cache_fork(grad, refs, table, one, one, one), lambda: kv.kv_cache_compact(grad, table, keep, table)):
        with pytest.raises(RuntimeError, match="no backward"):
            f()
    assert table.tolist() == [[0, 1], [2, 3]] and refs.tolist() == [0] * 6


def test_what_autograd_saved_is_seen_to_change(host_path):
    """Tensors that are written in place count as written, as after an operator of torch's own; nothing to do is no write into others' memory."""
    from lvar_amd import kv_cache_ops as kv
    cache = kv.PagedKVCache.alloc(6, 2, 64, page_size=16)
    refs, table, one = i32([1, 1, 1, 0, 0, 0]), i32([[0, 1], [2, -1], [-1, -1]]), i32([0, 0, 0])
    versions = lambda: [t._version for t in (refs, table, cache.k, cache.v)]  # noqa: E731
    v = versions()
    kv.kv_cache_fork(cache, refs, table, i32([0]), i32([2]), i32([20, 0, 0]))
    assert all(a < b for a, b in zip(v, versions()))
    v = versions()
    kv.kv_pages_alloc(refs, table, one + 1, one + 2)
    assert versions()[0] > v[0] and versions()[1] > v[1]
    v = versions()
    kv.kv_pages_free(refs, table)
    assert versions()[0] > v[0] and versions()[1] > v[1]
    v = versions()
    kv.kv_cache_compact(cache, i32([[0]]), torch.zeros(1, 2, 1, dtype=torch.int32, device="cuda"), i32([[5]]))
    assert versions()[2] > v[2] and versions()[3] > v[3]
    with torch.inference_mode():
        t = table.clone()
        kv.kv_pages_free(refs.clone(), t)
        assert bool((t == -1).all())
    none = i32([])
    kv.kv_cache_fork(cache, refs, table, none, none, one)
    kv.kv_cache_compact(cache, i32([[0]]), torch.zeros(1, 2, 0, dtype=torch.int32, device="cuda"), i32([[5]]))


def test_strided_tables_and_caches(host_path):
    """Tables that are slices of wider ones, pools with a stride between heads, pages beyond 32 bits of bytes."""
    from lvar_amd import kv_cache_ops as kv
    P, page, d = 5, 16, 64
    big = torch.zeros(2 ** 31 + 2 ** 16, dtype=torch.bfloat16, device="cuda")
    views = [big.as_strided((P, 2, page, d), (2 ** 29, 8 * page * d, d, 1), i * 4 * page * d) for i in range(2)]
    for i, t in enumerate(views):
        t.copy_(rand(P, 2, page, d, seed=i))
    before = [t.clone() for t in views]
    cache = kv.PagedKVCache(*views)
    wide = torch.full((4, 9), -1, dtype=torch.int32, device="cuda")
    table = wide[:, 2:5]
    table[0, :2] = i32([3, 1])
    refs = i32([1, 1, 0, 1, 0])
    kv.kv_cache_fork(cache, refs, table, i32([0, 0]), i32([1, 3]), i32([21, 0, 0, 0]))
    assert wide.tolist() == [[-1, -1, 3, 1, -1] + [-1] * 4, [-1, -1, 3, 2, -1] + [-1] * 4, [-1] * 9, [-1, -1, 3, 4, -1] + [-1] * 4]
    assert refs.tolist() == [1, 1, 1, 3, 1]
    for t, x in zip(views, before):
        x[2, :, :5] = x[1, :, :5]
        x[4, :, :5] = x[1, :, :5]
        assert torch.equal(t, x)
    kv.kv_cache_compact(cache, table[:1], torch.tensor([[[20, 0], [3, 17]]], device="cuda"), i32([[0]]))
    for t, x in zip(views, before):
        x[0, 0, :2] = torch.stack([x[1, 0, 4], x[3, 0, 0]])
        x[0, 1, :2] = torch.stack([x[3, 1, 3], x[1, 1, 1]])
        assert torch.equal(t, x)
    assert pref.free([1, 1], [[0, 1]]) == ([0, 0], [[-1, -1]])
