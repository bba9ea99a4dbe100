"""What needs no device of the rotation by several axes and of the life of pages: refusals of the operators and of the entry points, workspaces,
the plain implementations themselves."""
import ctypes as C

import pytest
import torch

from oracle import pages_oracle as ref


@pytest.fixture(scope="module")
def lib():
    from lvar_amd import _lib
    return _lib.load()


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_operators_refuse_cpu_tensors():
    from lvar_amd import kv_cache_ops as kv
    x = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16)
    cache = kv.PagedKVCache(*(torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16) for _ in range(2)))
    refs, table, one = i32([0] * 4), i32([[0, 1]]), i32([0])
    f, p = torch.zeros(2, 32), torch.zeros(2, 3)
    for call in (lambda: kv.qk_norm_rope(x, x, freqs=f, positions=p), lambda: kv.qk_norm_rope_append(cache, x, x, x, table, one, freqs=f, positions=p),
                 lambda: kv.kv_pages_alloc(refs, table, one, one), lambda: kv.kv_pages_free(refs, table), lambda: kv.kv_cache_fork(cache, refs, table, one, one, one),
                 lambda: kv.kv_cache_compact(cache, table, torch.zeros(1, 2, 3, dtype=torch.int32), table)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_operators_refuse_tangents():
    import torch.autograd.forward_ad as fw
    from lvar_amd import kv_cache_ops as kv
    x, f, p = torch.zeros(1, 2, 3, 64, dtype=torch.bfloat16), torch.zeros(2, 32), torch.zeros(2, 3)
    with fw.dual_level():
        fd, pd = fw.make_dual(f, f), fw.make_dual(p, p)
        for kw in (dict(freqs=fd, positions=p), dict(freqs=f, positions=pd)):
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                kv.qk_norm_rope(x, x, **kw)


def test_axis_freqs():
    from lvar_amd import kv_cache_ops as kv
    f = kv.axis_freqs((4, 0, 6), theta=100.0, device="cpu")
    assert f.shape == (3, 5) and f.dtype == torch.float64
    want = torch.zeros(3, 5, dtype=torch.float64)
    want[0, :2] = torch.tensor([1.0, 0.1], dtype=torch.float64)
    want[2, 2:] = 100.0 ** (-2.0 * torch.arange(3, dtype=torch.float64) / 6)
    assert torch.allclose(f, want, rtol=1e-15, atol=0)
    for bad in ((), (3, 5), (-2, 4)):
        with pytest.raises(kv.ShapeError):
            kv.axis_freqs(bad, device="cpu")


AXES = dict(freqs=0x6000, freq_stride=64, freq_type=0, axes=2, rot_dim=128, interleaved=1, positions=0x7000, pos_stride_b=0, pos_stride_axis=3, pos_stride_row=1, position_type=2)


@pytest.mark.parametrize("change,status", [
    (dict(freqs=None), -1), (dict(freqs=0x6008), -1), (dict(positions=None), -1), (dict(positions=0x7002), -1), (dict(position_type=1, positions=0x7004), -1),
    (dict(position_type=3), -1), (dict(position_type=-1), -1), (dict(freq_type=2), -1), (dict(freq_stride=63), -1), (dict(freq_type=1, freq_stride=66), -1),
    (dict(axes=0), -1), (dict(axes=9), -1), (dict(rot_dim=0), -1), (dict(rot_dim=144), -1), (dict(rot_dim=24), -2), (dict(cos=0x9000), -1)])
def test_entry_points_refuse_axes(lib, change, status):
    from lvar_amd import _lib
    t, one = _lib.LvarTensor(0x1000, 2048, 512, 128), C.c_void_p(0x5000)
    cache = _lib.LvarPagedCache(0x1000, 0x2000, None, None, 4096, 2048, 128, 0, 0, 0x3000, 4, 8, 2, 16, 128, 4)
    how = _lib.LvarNormRope()
    how.norm, how.eps = 1, 1e-6
    if "cos" in change:      # a rotation by tables as well
        how.cos = how.sin = change["cos"]
        how.table_stride, how.table_rows, how.rot_dim = 64, 9, 128
    axes = _lib.LvarRopeAxes(**{**AXES, **{k: v for k, v in change.items() if k != "cos"}})
    assert lib.lvar_qk_norm_axes_fwd(t, t, how, axes, one, one, 1, 4, 2, 3, 128, None) == status
    assert lib.lvar_qk_norm_axes_bwd(t, t, how, axes, one, one, t, t, None, None, None, 0, 1, 4, 2, 3, 128, None) == status
    assert lib.lvar_kv_cache_append_axes(t, t, t, how, axes, one, cache, one, None, 1, 4, 3, None) == status


def test_workspace_of_the_rotation(lib):
    f = lib.lvar_qk_norm_axes_bwd_scratch_bytes
    assert f(0, 4, 2, 3, 128, 128, 0) == -1 and f(1, 4, 2, 3, 96, 64, 0) == -2


PAGES = dict(refs=0x4000, num_pages=8, table=0x3000, table_stride=4, rows=3, max_pages=4)


@pytest.mark.parametrize("change", [dict(refs=None), dict(refs=0x4002), dict(num_pages=0), dict(table=None), dict(table=0x3002), dict(table_stride=3), dict(rows=0), dict(rows=65536),
                                    dict(max_pages=0), dict(num_pages=(1 << 30) + 1), dict(table_stride=-4)])
def test_entry_points_refuse_tables(lib, change):
    from lvar_amd import _lib
    a = {**PAGES, **change}
    one, first = C.c_void_p(0x5000), [C.c_void_p(a["refs"]), a["num_pages"], C.c_void_p(a["table"]), a["table_stride"], a["rows"], a["max_pages"]]
    assert lib.lvar_kv_pages_alloc(*first, one, one, one, 1 << 40, None) == -1
    assert lib.lvar_kv_pages_free(*first, None, None) == -1
    cache = _lib.LvarPagedCache(0x1000, 0x2000, None, None, 4096, 2048, 128, 0, 0, 0x3000, a["table_stride"], a["num_pages"], 2, 16, 128, a["max_pages"])
    assert lib.lvar_kv_cache_fork(cache, first[0], first[2], a["rows"], one, one, one, 2, one, 1 << 40, None) == -1


def test_entry_points_refuse_pages(lib):
    from lvar_amd import _lib
    one, odd, z = C.c_void_p(0x5000), C.c_void_p(0x5002), None
    table = [C.c_void_p(0x4000), 8, C.c_void_p(0x3000), 4, 3, 4]
    for first, last in ((z, one), (one, z), (odd, one), (one, odd)):
        assert lib.lvar_kv_pages_alloc(*table, first, last, one, 1 << 40, None) == -1
    assert lib.lvar_kv_pages_free(*table, odd, None) == -1
    good = dict(k=0x1000, v=0x2000, k_exp=None, v_exp=None, stride_page=4096, stride_head=2048, stride_row=128, exp_stride_page=0, exp_stride_head=0, page_table=0x3000,
                table_stride=4, num_pages=8, kv_heads=2, page_size=16, head_dim=128, max_pages=4)
    cache = lambda **kw: _lib.LvarPagedCache(**{**good, **kw})  # noqa: E731
    fork = lambda c, a, n=2, ws=one, size=1 << 40: lib.lvar_kv_cache_fork(c, table[0], table[2], 3, *a, n, ws, size, None)  # noqa: E731
    for a in ((z, one, one), (one, z, one), (one, one, z), (odd, one, one), (one, odd, one), (one, one, odd)):
        assert fork(cache(), a) == -1
    for kw in (dict(n=0), dict(n=65536), dict(ws=z), dict(ws=odd), dict(size=7)):
        assert fork(cache(), (one, one, one), **kw) == -1
    compact = lambda c, out=one, stride=4, pages=4, keep=one, wide=0, counts=z, B=3, n=5: lib.lvar_kv_cache_compact(  # noqa: E731
        c, out, stride, pages, keep, wide, 10, 5, 1, counts, B, n, None)
    for kw in (dict(out=z), dict(out=odd), dict(stride=-1), dict(pages=0), dict(keep=z), dict(keep=odd), dict(keep=C.c_void_p(0x5004), wide=1), dict(counts=odd),
               dict(B=0), dict(n=0), dict(B=65536), dict(n=1 << 30)):
        assert compact(cache(), **kw) == -1, kw
    for kw, status in ((dict(page_size=24), -2), (dict(head_dim=96), -2), (dict(k=0x1008), -1), (dict(k_exp=0x8000), -1), (dict(num_pages=0), -1), (dict(stride_row=100), -1)):
        assert compact(cache(**kw)) == status and fork(cache(**kw), (one, one, one)) == status, kw
    # what does not fit LDS: what becomes of each fork, long lists of pages
    f = lib.lvar_kv_pages_scratch_bytes
    assert f(0, 100) == 0 and f(7, 100) == 28 and f(0, 100000) == 400000 and f(7, 100000) == 400028 and f(-1, 9) == -1 and f(1, 0) == -1


def test_plain_fork():
    refs, table, copies = ref.fork([1, 1, 0, 1, 0], [[0, 1], [-1, -1], [3, -1]], [0, 2, 1], [1, 0, 1], [20, 9, 3], 16)
    # (1, 1) is no pair; 0 is a target and a source, so that of 2 is left out; 0 goes to 1
    assert (refs, table, copies) == ([2, 1, 1, 1, 0], [[0, 1], [0, 2], [3, -1]], [(1, 2, 4)])
    assert ref.fork([1, 1, 0], [[0, 1], [-1, -1], [-1, -1]], [0, 2, 1], [1, 1, 0], [9, 0, 0], 16) == ([1, 1, 0], [[0, 1], [-1, -1], [-1, -1]], [])
    refs, table, copies = ref.fork([1, 1, 0, 1, 0], [[0, 1], [-1, -1], [3, -1]], [0], [1], [20, 9, 3], 16)
    assert (refs, table, copies) == ([2, 1, 1, 1, 0], [[0, 1], [0, 2], [3, -1]], [(1, 2, 4)])
