"""The rotation by several axes on the GPU in the forms that a program may hand it: layouts of positions and frequencies, shared and own positions, rows that
are not finite, no tokens, the same bits every time."""
import math

import pytest
import torch

from test_gpu_packed import i32, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "ctypes"])
def host_path(request, monkeypatch):
    from lvar_amd import kv_cache_ops
    if request.param == "ctypes":
        monkeypatch.setattr(kv_cache_ops, "_native", lambda: None)


def grads(q, k, pos, freqs, g, **kw):
    from lvar_amd import kv_cache_ops as kv
    leaves = [t.detach().requires_grad_() for t in (q, k)]
    o = kv.qk_norm_rope(*leaves, positions=pos, freqs=freqs, **kw)
    return [t.detach() for t in o] + list(torch.autograd.grad(o, leaves, g))


@pytest.mark.parametrize("L", [1, 37, 2500])      # (with tables in the backward pass from 2^18 angles on)
@pytest.mark.parametrize("ptype", [torch.float32, torch.int32, torch.int64])
@pytest.mark.parametrize("ftype", [torch.float32, torch.float64])
def test_layouts(L, ptype, ftype, host_path):
    B, H, d, A = 3, 2, 128, 3
    q, k = (rand(B, H, L, d, seed=i).cuda() for i in range(2))
    g = [rand(B, H, L, d, seed=5 + i).cuda() for i in range(2)]
    pos = (torch.randn(A, L, generator=torch.Generator().manual_seed(L)) * 60).to(ptype).cuda()
    f = torch.rand(A, d // 2, generator=torch.Generator().manual_seed(2), dtype=torch.float64).to(ftype).cuda()
    want = grads(q, k, pos, f, g)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(grads(q, k, pos, f, g), want))
    wide = torch.zeros(A, d // 2 + 16, dtype=ftype, device="cuda")
    wide[:, :d // 2] = f
    shifted = torch.zeros(A * d // 2 + 1, dtype=ftype, device="cuda")[1:].view(A, d // 2).copy_(f)
    stepped = torch.zeros(A, 2 * L, dtype=ptype, device="cuda")[:, ::2].copy_(pos)
    own = pos[None].expand(B, A, L)
    for p, x in ((pos.t().contiguous().t(), f), (stepped, wide[:, :d // 2]), (own, shifted), (own.contiguous(), f.t().contiguous().t()),
                 (own.transpose(0, 2).contiguous().transpose(0, 2), f)):
        assert all(torch.equal(a, b) for a, b in zip(grads(q, k, p, x, g), want))
    # strided queries and gradients
    t = rand(B, L, 3 * H, d, seed=9).cuda().transpose(1, 2)
    a = grads(t[:, :H], t[:, H:2 * H], pos, f, [t[:, 2 * H:], g[1][:, :1].expand(B, H, L, d)])
    b = grads(t[:, :H].contiguous(), t[:, H:2 * H].contiguous(), pos, f, [t[:, 2 * H:].contiguous(), g[1][:, :1].expand(B, H, L, d).contiguous()])
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # one position for all tokens, one axis for all
    one = pos[:, :1].expand(A, L)
    assert all(torch.equal(x, y) for x, y in zip(grads(q, k, one, f, g), grads(q, k, one.contiguous(), f, g)))
    same = pos[:1].expand(A, L)
    assert all(torch.equal(x, y) for x, y in zip(grads(q, k, same, f, g), grads(q, k, same.contiguous(), f, g)))


def test_rows_that_are_not_finite(host_path):
    """A row, or a position, that is not finite stays with its token and head."""
    B, H, L, d = 2, 4, 50, 64
    pos = torch.randn(2, L, device="cuda")
    f = torch.rand(2, 32, dtype=torch.float64, device="cuda")
    for value in (math.inf, -math.inf, math.nan):
        q, k = (rand(B, H, L, d, seed=i).cuda() for i in range(2))
        g = [rand(B, H, L, d, seed=5 + i).cuda() for i in range(2)]
        want = grads(q, k, pos, f, g, norm="rms")
        q[1, 2, 7, 3] = value
        g[1][0, 1, 9, 60] = value
        p = pos.clone()
        p[1, 20] = value
        got = grads(q, k, p, f, g, norm="rms")
        for i, (a, b) in enumerate(zip(got, want)):
            where = torch.zeros(B, H, L, dtype=torch.bool, device="cuda")
            where[:, :, 20] = True
            if i in (0, 2):
                where[1, 2, 7] = True
            if i == 3:
                where[0, 1, 9] = True
            assert torch.equal(a[~where], b[~where]) and not bool(torch.isfinite(a[:, :, 20].float()).any())
            if i == 3:
                assert not bool(torch.isfinite(a[0, 1, 9].float()).all())


def test_no_tokens(host_path):
    from lvar_amd import kv_cache_ops as kv
    f = kv.axis_freqs((32, 32))
    for B, L in ((2, 0), (0, 3)):
        q = torch.zeros(B, 4, L, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        o = kv.qk_norm_rope(q, q, positions=torch.zeros(2, L, device="cuda"), freqs=f)
        assert o[0].shape == q.shape and torch.autograd.grad(o[0].sum() + o[1].sum(), q)[0].shape == q.shape
    cache = kv.PagedKVCache.alloc(2, 4, 64, page_size=16)
    q = torch.zeros(1, 4, 0, 64, device="cuda", dtype=torch.bfloat16)
    assert kv.qk_norm_rope_append(cache, q, q, q, i32([[0]]), i32([0]), positions=torch.zeros(2, 0, device="cuda"), freqs=f).shape == q.shape


def test_workspace():
    from lvar_amd import _lib
    lib = _lib.load()
    f = lib.lvar_qk_norm_axes_bwd_scratch_bytes
    assert f(1, 4, 2, 3, 128, 128, 0) >= lib.lvar_qk_norm_rope_bwd_scratch_bytes(1, 4, 2, 3, 128)
    # a large call has room for tables of sines and cosines, one set if the sequences share their positions
    less, more = f(8, 40, 40, 4096, 128, 128, 0), f(8, 40, 40, 4096, 128, 128, 1)
    assert less - lib.lvar_qk_norm_rope_bwd_scratch_bytes(8, 40, 40, 4096, 128) >= 4096 * 64 * 8 and more - less >= 7 * 4096 * 64 * 8
    assert f(1, 4, 2, 3, 128, 0, 0) == -1 and f(1, 4, 2, 3, 128, 144, 0) == -1


def test_one_turn_more():
    """Angles are reduced in 64 bits: whole turns, added by a second axis, change nothing that bf16 shows but roundings at ties."""
    from lvar_amd import kv_cache_ops as kv
    x = rand(1, 2, 40, 64, seed=1).cuda()
    f = torch.rand(1, 32, dtype=torch.float64, generator=torch.Generator().manual_seed(3)).cuda()
    pos = torch.arange(40, dtype=torch.float32, device="cuda")[None]
    a, _ = kv.qk_norm_rope(x, x, positions=pos, freqs=f)
    both = torch.cat([f, torch.full((1, 32), 2 * math.pi, dtype=torch.float64, device="cuda")])
    b, _ = kv.qk_norm_rope(x, x, positions=torch.cat([pos, torch.full((1, 40), 1000.0, device="cuda")]), freqs=both)
    # 1000 * 2 pi is off by 2^-53 of it, about 1e-12; a sum that falls on the other side of a tie is off by one step
    assert bool(((a.float() - b.float()).abs() <= 2 * 2.0 ** -8 * a.float().abs() + 1e-6).all())
    assert float((a != b).float().mean()) < 0.01
