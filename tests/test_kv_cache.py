"""Paged cache, norms and rotation without a GPU: the oracle against independent statements, refusals of the operators and of
the C entry points."""
import ctypes

import pytest
import torch

from oracle import kv_cache_oracle as ref


@pytest.fixture(scope="module")
def lib():
    import os
    from lvar_amd import _lib
    from lvar_amd.build import LIB_PATH, build_library
    if not os.path.exists(LIB_PATH):
        build_library()
    return _lib.load()


# ---- the oracle ----

@pytest.mark.parametrize("norm,eps", [("l2", 1e-12), ("l2", 0.5), ("rms", 1e-6), (None, 0.0)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shape", [(16,), (1, 16), (3, 1), (3, 16), None])
def test_gradient_formulas_against_differences(norm, eps, interleaved, shape):
    g = torch.Generator().manual_seed(1)
    B, H, L, d = 2, 3, 4, 16
    x = torch.randn(B, H, L, d, generator=g, dtype=torch.float64)
    if eps == 0.5:
        x[0, 0] *= 0.01                        # rows below the threshold of the l2 norm
    w = None if shape is None else torch.randn(shape, generator=g, dtype=torch.float64)
    angle = torch.randn(9, 8, generator=g, dtype=torch.float64)
    at = ref.table_rows(B, L, 9, torch.tensor([[0, 8, 3, 12], [2, 2, -1, 5]]))
    go = torch.randn(B, H, L, d, generator=g, dtype=torch.float64)
    f = lambda x, w: (go * ref.norm_rope(x, w, angle.cos(), angle.sin(), at, norm, eps, interleaved)).sum()  # noqa: E731
    dx, dw = ref.norm_rope_grads(x, w, angle.cos(), angle.sin(), at, norm, eps, interleaved, go)
    step = 1e-6                                # central differences in 64 bits: off by about step^2 and 2^-52 / step
    for _ in range(4):
        t = torch.randn(x.shape, generator=g, dtype=torch.float64)
        diff = (f(x + step * t, w) - f(x - step * t, w)) / (2 * step)
        assert abs(float(diff - (dx * t).sum())) < 1e-6 * max(1.0, float(dx.norm()))
        if w is not None:
            t = torch.randn(w.shape, generator=g, dtype=torch.float64)
            diff = (f(x, w + step * t) - f(x, w - step * t)) / (2 * step)
            assert dw.shape == w.shape and abs(float(diff - (dw * t).sum())) < 1e-6 * max(1.0, float(dw.norm()))


def test_codes_against_torch():
    """torch's own conversion to e4m3 rounds to nearest even as well."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(400, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (400, 1), generator=g).float())
    x[0] = 0
    x[1, 0] = 448.0 * 2.0 ** 5
    x[2, 0] = 449.0 * 2.0 ** 5
    codes, byte = ref.quantise(x)
    top, scale = x.abs().amax(-1), torch.exp2(byte.float() - 127)
    assert bool((top <= 448 * scale).all()) and bool(((top > 224 * scale) | (top == 0)).all())
    assert torch.equal(codes, (x / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8))
    y = ref.dequantise(codes, byte)
    assert torch.equal(y, y.to(torch.bfloat16).double())          # every value is a bf16 value
    assert bool(((y - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + scale.double()[:, None] * 2.0 ** -10).all())


# ---- refusals ----

def _cache(dtype=torch.bfloat16, P=4, H=2, page=16, d=64):
    from lvar_amd import kv_cache_ops as kv
    return kv.PagedKVCache.alloc(P, H, d, page, dtype, "cpu")


def test_operators_refuse_cpu_tensors_and_wrong_types():
    from lvar_amd import kv_cache_ops as kv
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        c = _cache(dtype)
        with pytest.raises(RuntimeError, match="no CPU path"):
            kv.kv_cache_append(c, x, x, table, i)
        with pytest.raises(RuntimeError, match="no CPU path"):
            kv.qk_norm_rope_append(c, x, x, x, table, i)
        with pytest.raises(RuntimeError, match="no CPU path"):
            kv.kv_cache_read(c, table, i)
        with pytest.raises(RuntimeError, match="no CPU path"):
            kv.paged_attn(x, c, table, i)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv.qk_norm_rope(x, x)
    with pytest.raises(TypeError):
        kv.qk_norm_rope(x.float(), x.float())
    with pytest.raises(TypeError):
        kv.PagedKVCache.alloc(1, 1, 64, 16, torch.float16, "cpu")
    grad = x.clone().requires_grad_()
    for call in (lambda: kv.kv_cache_append(_cache(), grad, x, table, i), lambda: kv.paged_attn(grad, _cache(), table, i),
                 lambda: kv.qk_norm_rope_append(_cache(), x, x, grad, table, i)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()


def _structs():
    from lvar_amd import _lib
    tensor = _lib.LvarTensor(0x1000, 128 * 16 * 128, 16 * 128, 128)
    cache = dict(k=0x1000, v=0x2000, k_exp=None, v_exp=None, stride_page=2 * 16 * 128, stride_head=16 * 128, stride_row=128, exp_stride_page=32,
                 exp_stride_head=16, page_table=0x3000, table_stride=8, num_pages=9, kv_heads=2, page_size=16, head_dim=128, max_pages=8)
    return _lib, tensor, cache


BAD_CACHES = [
    (dict(k=None), -1), (dict(v=0x1008), -1), (dict(page_table=None), -1), (dict(page_table=0x3002), -1), (dict(num_pages=0), -1), (dict(max_pages=0), -1),
    (dict(kv_heads=0), -1), (dict(page_size=0), -1), (dict(page_size=8), -2), (dict(page_size=48), -2), (dict(page_size=2048), -2), (dict(head_dim=96), -2),
    (dict(head_dim=16), -2), (dict(stride_row=127), -1), (dict(stride_row=132), -1), (dict(stride_head=4), -1), (dict(stride_page=-4096), -1),
    (dict(k_exp=0x4000), -1), (dict(k_exp=0x4001, v_exp=0x4000), -1), (dict(k_exp=0x4000, v_exp=0x4000, exp_stride_head=18), -1),
    (dict(k_exp=0x4000, v_exp=0x4000, stride_row=136), -1), (dict(stride_row=1 << 26), -1), (dict(max_pages=1 << 27), -1), (dict(table_stride=-1), -1),
]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_entry_points_refuse_bad_caches(lib, change, status):
    _lib, t, c = _structs()
    bad = _lib.LvarPagedCache(**{**c, **change})
    one = ctypes.c_void_p(0x5000)
    assert lib.lvar_kv_cache_append(t, t, t, None, None, bad, one, None, 1, 2, 3, None) == status
    assert lib.lvar_kv_cache_read(bad, None, one, one, one, 1, 3, None) == status
    assert lib.lvar_paged_attn_fwd(t, bad, one, None, one, one, one, None, 0, 1, 4, 3, 100, 0, 1.0, None) == status


def test_entry_points_refuse_bad_arguments(lib):
    _lib, t, c = _structs()
    good, one, odd = _lib.LvarPagedCache(**c), ctypes.c_void_p(0x5000), ctypes.c_void_p(0x5002)
    null, skew = _lib.LvarTensor(None, 0, 0, 0), _lib.LvarTensor(0x1008, 2048, 128, 128)
    how = lambda **kw: _fill(_lib.LvarNormRope(), **kw)  # noqa: E731
    H = dict(norm=1, eps=1e-6)
    table = dict(cos=0x6000, sin=0x7000, table_stride=64, table_rows=9, rot_dim=128)
    for kw, status in (({**H, "norm": 3}, -1), ({**H, "norm": -1}, -1), ({**H, "eps": -1.0}, -1), ({**H, "eps": float("nan")}, -1),
                       ({**H, **table, "sin": None}, -1), ({**H, **table, "rot_dim": 24}, -2), ({**H, **table, "rot_dim": 144}, -1), ({**H, **table, "rot_dim": 0}, -1),
                       ({**H, **table, "cos": 0x6004}, -1), ({**H, **table, "table_stride": 62}, -1), ({**H, **table, "table_rows": 0}, -1),
                       ({**H, **table, "positions": 0x6002}, -1), ({**H, **table, "positions": 0x6004, "positions64": 1}, -1),
                       ({**H, "q_weight": _lib.LvarWeight(0x8004, 128, 1, 0)}, -1), ({**H, "k_weight": _lib.LvarWeight(0x8000, 4, 1, 0)}, -1),
                       ({**H, "k_weight": _lib.LvarWeight(0x8000, 0, 2, 0)}, -1), ({**H, "k_weight": _lib.LvarWeight(0x8000, 0, 0, 2)}, -1),
                       ({**H, "q_weight": _lib.LvarWeight(0x8002, 1, 0, 0)}, -1)):
        assert lib.lvar_qk_norm_rope_fwd(t, t, how(**kw), one, one, 1, 4, 2, 3, 128, None) == status, kw
        assert lib.lvar_qk_norm_rope_bwd(t, t, how(**kw), one, one, t, t, None, None, None, 0, 1, 4, 2, 3, 128, None) == status, kw
        assert lib.lvar_kv_cache_append(t, t, t, ctypes.byref(how(**kw)), one, good, one, None, 1, 4, 3, None) == status, kw
    fwd = lambda q, k, oq, ok, *dims: lib.lvar_qk_norm_rope_fwd(q, k, how(**H), oq, ok, *dims, None)  # noqa: E731
    for dims, status in (((0, 4, 2, 3, 128), -1), ((1, 4, 3, 3, 128), -1), ((1, 4, 0, 3, 128), -1), ((1, 4, 2, 0, 128), -1), ((1, 4, 2, 3, 96), -2),
                         ((65536, 4, 2, 3, 128), -1), ((60000, 4, 2, 60000, 128), -1), ((1, 32768, 2, 3, 128), -1),
                         ((1, 1, 1, 1 << 30, 16), -1)):   # (2^32 threads, more than a launch holds)
        assert fwd(t, t, one, one, *dims) == status, dims
    assert fwd(null, t, one, one, 1, 4, 2, 3, 128) == -1 and fwd(t, skew, one, one, 1, 4, 2, 3, 128) == -1
    assert fwd(t, t, None, one, 1, 4, 2, 3, 128) == -1 and fwd(t, t, one, odd, 1, 4, 2, 3, 128) == -1
    # gradients: a weight gradient needs a weight and scratch
    bwd = lambda h, dqw, scratch, n: lib.lvar_qk_norm_rope_bwd(t, t, h, one, one, t, t, dqw, None, scratch, n, 1, 4, 2, 3, 128, None)  # noqa: E731
    assert bwd(how(**H), one, one, 1 << 40) == -1
    w = _lib.LvarWeight(0x8000, 0, 1, 0)
    assert bwd(how(**H, q_weight=w), one, None, 1 << 40) == -1 and bwd(how(**H, q_weight=w), one, ctypes.c_void_p(0x5008), 1 << 40) == -1
    # append: q, how and oq together; start
    app = lambda q, k, v, h, oq, start, B=1, L=3: lib.lvar_kv_cache_append(q, k, v, h, oq, good, start, None, B, 4, L, None)  # noqa: E731
    hp = ctypes.byref(how(**H))
    for args in ((t, t, t, hp, None, one), (t, t, t, None, one, one), (null, t, t, hp, one, one), (t, null, t, hp, one, one), (t, t, skew, hp, one, one),
                 (t, t, t, hp, one, None), (t, t, t, hp, one, odd), (t, t, t, hp, odd, one), (t, t, t, None, None, one, 0), (t, t, t, None, None, one, 1, 0)):
        assert app(*args) == -1
    # read
    for args in ((None, None, one, one, 1, 3), (None, one, None, one, 1, 3), (None, one, one, odd, 1, 3), (odd, one, one, one, 1, 3), (None, one, one, one, 0, 3),
                 (None, one, one, one, 1, 0), (None, one, one, one, 1, -3), (None, one, one, one, 1, 1 << 30)):
        assert lib.lvar_kv_cache_read(good, *args, None) == -1
    # attention
    att = lambda q=t, lengths=one, counts=None, o=one, M=one, L=one, B=1, H=4, Lq=3, n=100, scale=1.0: lib.lvar_paged_attn_fwd(  # noqa: E731
        q, good, lengths, counts, o, M, L, None, 0, B, H, Lq, n, 0, scale, None)
    for kw in (dict(q=null), dict(q=skew), dict(lengths=None), dict(lengths=odd), dict(counts=odd), dict(o=None), dict(o=odd), dict(M=None), dict(L=None), dict(B=0),
               dict(H=3), dict(H=0), dict(Lq=0), dict(n=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(B=65536)):
        assert att(**kw) == -1, kw
    assert lib.lvar_paged_attn_workspace_bytes(1, 4, 3, 1, 100, 128) == -1 and lib.lvar_paged_attn_workspace_bytes(1, 4, 2, 1, -1, 128) == -1
    assert lib.lvar_paged_attn_workspace_bytes(1, 4, 2, 1, 100, 96) == -2 and lib.lvar_qk_norm_rope_bwd_scratch_bytes(1, 4, 2, 3, 96) == -2
    assert lib.lvar_qk_norm_rope_bwd_scratch_bytes(1, 4, 2, 0, 128) == -1


def _fill(s, **kw):
    for n, v in kw.items():
        setattr(s, n, v)
    return s


def test_operators_refuse_tangents():
    """Ahead of everything else, so that it shows without a device too."""
    import torch.autograd.forward_ad as fw
    from lvar_amd import kv_cache_ops as kv
    x, w = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16), torch.ones(64)
    i, table, c = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32), _cache()
    cos = torch.ones(3, 32)
    with fw.dual_level():
        y, wy, cy = (fw.make_dual(t, torch.ones_like(t)) for t in (x, w, cos))
        for call in (lambda: kv.qk_norm_rope(y, x), lambda: kv.qk_norm_rope(x, y), lambda: kv.qk_norm_rope(x, x, k_weight=wy), lambda: kv.qk_norm_rope(x, x, cy, cos),
                     lambda: kv.kv_cache_append(c, x, y, table, i), lambda: kv.qk_norm_rope_append(c, y, x, x, table, i),
                     lambda: kv.qk_norm_rope_append(c, x, x, x, table, i, cos, cy), lambda: kv.paged_attn(y, c, table, i)):
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_operators_refuse_caches_that_need_a_gradient():
    from lvar_amd import kv_cache_ops as kv
    x, i, table = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int32)
    for name in ("k", "v"):
        c = _cache()
        c = c._replace(**{name: getattr(c, name).clone().requires_grad_()})
        for call in (lambda: kv.kv_cache_append(c, x, x, table, i), lambda: kv.qk_norm_rope_append(c, x, x, x, table, i), lambda: kv.kv_cache_read(c, table, i),
                     lambda: kv.paged_attn(x, c, table, i)):
            with pytest.raises(RuntimeError, match="no backward"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
                call()


def test_checks_refuse_no_heads():
    from lvar_amd import kv_cache_ops as kv
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    for q, k in ((x[:, :0], x), (x, x[:, :0]), (x[:, :0], x[:, :0])):
        with pytest.raises(kv.ShapeError):
            kv._norm_args(q, k, None, None, None, "l2", None)
    assert kv._norm_args(x[:0], x[:0], None, None, None, "l2", None) == (None, None, 1e-12)


def test_eps_is_zero_or_normal(lib):
    from lvar_amd import kv_cache_ops as kv
    _lib, t, _ = _structs()
    x, one = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16), ctypes.c_void_p(0x5000)
    for norm in ("l2", "rms", None):
        for eps in (1e-39, 5e-324, 1e39, -0.1, float("nan"), float("inf")):
            with pytest.raises(kv.ShapeError):
                kv._norm_args(x, x, None, None, None, norm, eps)
        assert kv._norm_args(x, x, None, None, None, norm, 2.0 ** -126)[2] == 2.0 ** -126 and kv._norm_args(x, x, None, None, None, norm, 0)[2] == 0.0
    for eps in (1e-39, 1e-45, float("inf"), -1e-6):
        assert lib.lvar_qk_norm_rope_fwd(t, t, _fill(_lib.LvarNormRope(), norm=1, eps=eps), one, one, 1, 4, 2, 3, 128, None) == -1
