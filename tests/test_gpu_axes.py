"""Norms with a rotation of several position axes on the GPU, against the 64-bit oracle.  Tolerances count roundings as for the rotation by
tables: half a step of bf16 for a result, 32-bit arithmetic of a row; sines and cosines of the reduced angle are off by a few steps of 32 bits."""
import pytest
import torch

from oracle import kv_cache_oracle as ref

pytestmark = pytest.mark.gpu

BF16, F32 = 2.0 ** -8, 2.0 ** -24
EPS = {"l2": 1e-12, "rms": 1e-6, None: 0.0}


@pytest.fixture(params=["compiled", "ctypes"])
def host_path(request, monkeypatch):
    from lvar_amd import kv_cache_ops
    if request.param == "ctypes":
        monkeypatch.setattr(kv_cache_ops, "_native", lambda: None)
    return request.param


def rand(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def weight(kind, heads, d, seed):
    if kind is None:
        return None
    shape = {"head": (heads, 1), "dim": (d,), "full": (heads, d)}[kind]
    return 1 + 0.3 * torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def cu(t):
    return None if t is None else t.cuda()


def turned(positions, freqs, B):
    """cos and sin [B * L, rot/2] in 64 bits, and the row of each token"""
    p = positions.double()
    p = p[None].expand(B, *p.shape) if p.dim() == 2 else p
    angle = (p[..., None] * freqs.double()[None, :, None, :]).sum(1)
    L = angle.shape[1]
    return angle.cos().flatten(0, 1), angle.sin().flatten(0, 1), torch.arange(B * L).view(B, L)


def near(got, want, what, grad=False):
    top = want.abs().amax(-1, keepdim=True)
    tol = BF16 * want.abs() + ((4 if grad else 1) * want.shape[-1] + 40) * F32 * top + 1e-38
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err - tol).max()):.3g} over"


CASES = [
    # B, H, Hkv, L, d, rot, axes, positions, per sequence, frequencies, norm, weight, interleaved
    (1, 1, 1, 1, 16, 16, 1, torch.int32, False, torch.float64, "l2", None, True),
    (2, 16, 16, 16, 128, 128, 2, torch.float32, False, torch.float64, "l2", "head", True),
    (1, 8, 2, 257, 128, 128, 3, torch.int64, False, torch.float32, "rms", "dim", False),
    (3, 5, 5, 33, 64, 32, 4, torch.int64, True, torch.float64, None, "full", False),
    (2, 4, 2, 70, 256, 256, 2, torch.float32, True, torch.float32, "rms", "full", True),
    (2, 3, 3, 9, 32, 32, 8, torch.int32, True, torch.float64, "l2", "dim", True),
    (1, 12, 4, 3000, 64, 64, 3, torch.int32, False, torch.float64, "rms", "head", False),    # several heads per workgroup
    (4, 9, 3, 700, 128, 96, 2, torch.float32, True, torch.float64, None, None, True),
]


def make(case):
    B, H, Hkv, L, d, rot, A, ptype, own, ftype, norm, wk, inter = case
    x = rand(B, L, H + 2 * Hkv, d, seed=L + d).transpose(1, 2)
    g = torch.Generator().manual_seed(A)
    shape = (B, A, L) if own else (A, L)
    p = torch.randn(shape, generator=g) * 50 if ptype == torch.float32 else torch.randint(-5, 200000, shape, generator=g).to(ptype)
    f = (torch.rand((A, rot // 2), generator=g, dtype=torch.float64) * torch.rand((A, 1), generator=g, dtype=torch.float64)).to(ftype)
    return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:], p, f, weight(wk, H, d, 7), weight(wk, Hkv, d, 8)


@pytest.mark.parametrize("case", CASES, ids=lambda c: str(c).replace("torch.", "").replace(" ", ""))
def test_forward_and_gradients(case, host_path):
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, L, d, rot, A, ptype, own, ftype, norm, wk, inter = case
    q, k, _, p, f, wq, wkk = make(case)
    leaves = [None if x is None else x.cuda().detach().requires_grad_() for x in (q, k, wq, wkk)]
    plain = kv.qk_norm_rope(*(x.detach() for x in leaves[:2]), positions=cu(p), freqs=cu(f), q_weight=cu(wq), k_weight=cu(wkk), norm=norm, interleaved=inter)
    outs = kv.qk_norm_rope(leaves[0], leaves[1], positions=cu(p), freqs=cu(f), q_weight=leaves[2], k_weight=leaves[3], norm=norm, interleaved=inter)
    assert torch.equal(plain[0], outs[0]) and torch.equal(plain[1], outs[1])
    gs = [rand(B, L, x.shape[1], d, seed=90 + i).transpose(1, 2) for i, x in enumerate((q, k))]
    some = [x for x in leaves if x is not None]
    grads = dict(zip(map(id, some), torch.autograd.grad(outs, some, [x.cuda() for x in gs])))
    cos, sin, at = turned(p, f, B)
    for i, (x, w, out) in enumerate(((q, wq, outs[0]), (k, wkk, outs[1]))):
        near(out.detach(), ref.norm_rope(x, w, cos, sin, at, norm, EPS[norm], inter), "qk"[i])
        dx, dw = ref.norm_rope_grads(x, w, cos, sin, at, norm, EPS[norm], inter, gs[i])
        near(grads[id(leaves[i])], dx, "d" + "qk"[i], grad=True)
        if w is not None:
            got = grads[id(leaves[2 + i])].double().cpu()
            mags = ref.norm_rope_grads(x, w, cos, sin, at, norm, EPS[norm], inter, gs[i])[1].abs()
            # n products of a normalised element (about 1, or 1 / sqrt(d)) and a gradient, in 32 bits
            n = B * L * (1 if w.dim() == 2 else x.shape[1]) * (d if w.shape[-1] == 1 else 1)
            size = float(x.double().abs().max()) if norm is None else 4.0
            assert bool(((got - dw).abs() <= F32 * mags + (n ** 0.5 * 8 + d + 40) * F32 * size * 8 * n ** 0.5).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("case", [CASES[1], CASES[3], CASES[4], CASES[7]], ids=lambda c: str(c).replace("torch.", "").replace(" ", ""))
def test_append(case, dtype, host_path):
    from lvar_amd import kv_cache_ops as kv
    B, H, Hkv, L, d, rot, A, ptype, own, ftype, norm, wk, inter = case
    q, k, v, p, f, wq, wkk = make(case)
    per = -(-(L + 9) // 32)
    cache = kv.PagedKVCache.alloc(B * per + 1, Hkv, d, page_size=32, dtype=dtype)
    table = torch.randperm(B * per + 1)[:B * per].int().view(B, per).cuda()
    start = torch.arange(B, dtype=torch.int32, device="cuda") * 3 % 9
    oq = kv.qk_norm_rope_append(cache, q.cuda(), k.cuda(), v.cuda(), table, start, positions=cu(p), freqs=cu(f), q_weight=cu(wq), k_weight=cu(wkk), norm=norm, interleaved=inter)
    cos, sin, at = turned(p, f, B)
    near(oq, ref.norm_rope(q, wq, cos, sin, at, norm, EPS[norm], inter), "q")
    gk, gv = kv.kv_cache_read(cache, table, start + L, max_len=L, start=start)
    want = ref.norm_rope(k, wkk, cos, sin, at, norm, EPS[norm], inter)
    if dtype == torch.bfloat16:
        near(gk, want, "k")
        assert torch.equal(gv.cpu(), v.contiguous())
    else:   # one rounding to e4m3: 2^-4 of the element, or half a step below its normal range
        for got, x in ((gk, want), (gv, v.double())):
            top = x.abs().amax(-1, keepdim=True)
            assert bool(((got.double().cpu() - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -17 * top + (d + 40) * F32 * top).all())


def test_the_same_as_tables(host_path):
    """One axis with whole positions is the rotation by tables, but for the rounding of the tables."""
    from lvar_amd import kv_cache_ops as kv
    q, k = rand(2, 4, 50, 128, seed=1).cuda(), rand(2, 2, 50, 128, seed=2).cuda()
    f = kv.axis_freqs((128,))
    assert f.dtype == torch.float64 and f.shape == (1, 64)
    angle = torch.arange(50, device="cuda", dtype=torch.float64)[:, None] * f
    a = kv.qk_norm_rope(q, k, angle.cos().float(), angle.sin().float())
    b = kv.qk_norm_rope(q, k, positions=torch.arange(50, device="cuda")[None], freqs=f)
    for x, y in zip(a, b):
        assert float((x.float() - y.float()).abs().max()) <= 2 * BF16 * float(x.float().abs().max())
        assert float((x != y).float().mean()) < 1e-3          # (a rounding that falls the other way)


def test_axis_freqs():
    from lvar_amd import kv_cache_ops as kv
    f = kv.axis_freqs((16, 0, 32), theta=100.0, device="cpu")
    assert f.shape == (3, 24) and not bool(f[1].any()) and not bool(f[0, 8:].any()) and not bool(f[2, :8].any())
    assert torch.allclose(f[0, :8], 100.0 ** (-torch.arange(8, dtype=torch.float64) / 8)) and torch.allclose(f[2, 8:], 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16))
    with pytest.raises(AssertionError):
        kv.axis_freqs((3,), device="cpu")


def test_far_positions(host_path):
    """Positions of 2^40 times a frequency of 1: 64 bits keep 2^-12 of a radian, 32 would keep nothing."""
    from lvar_amd import kv_cache_ops as kv
    q, k = rand(1, 2, 64, 64, seed=1), rand(1, 1, 64, 64, seed=2)
    p = (2 ** 40 + torch.arange(64) * 12345)[None]
    f = torch.ones(1, 32, dtype=torch.float64) * torch.linspace(0.1, 1, 32, dtype=torch.float64)
    got = kv.qk_norm_rope(q.cuda(), k.cuda(), positions=p.cuda(), freqs=f.cuda(), norm=None)
    cos, sin, at = turned(p, f, 1)
    for x, y in ((q, got[0]), (k, got[1])):
        want = ref.norm_rope(x, None, cos, sin, at, None, 0.0, True)
        # 2^40 turns are rounded to 2^-52 of themselves, twice on either side
        assert bool(((y.double().cpu() - want).abs() <= BF16 * want.abs() + (4 * 2.0 ** -12 + 64 * F32) * want.abs().amax(-1, keepdim=True)).all())
