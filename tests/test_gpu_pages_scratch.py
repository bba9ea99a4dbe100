"""More forks than there are pages: every free page is dealt, and nothing is written behind the scratch that the entry point asks for."""
import ctypes as C

import pytest
import torch

from oracle import pages_oracle as ref
from test_gpu_pages import host_path, i32, pool, raw  # noqa: F401

pytestmark = pytest.mark.gpu

# forks, pages (a search keeps 4096 of them in LDS), entries of a row, pages in use
CASES = [(5000, 4096, 2, 30), (4097, 4096, 1, 1), (9000, 40, 3, 7), (4097, 4097, 2, 1), (65000, 4096, 1, 4000), (70, 33, 2, 3), (1030, 1025, 1, 5)]


def program(n, P, width, used):
    """Row 0 is a prompt that ends inside its last page; all other rows become samples of it."""
    table = [list(range(P - width, P))] + [[-1] * width for _ in range(n)]
    refs = [0] * P
    for page in [*range(used), *table[0]]:
        refs[page] = 1
    return table, refs, [0] * n, list(range(1, n + 1)), [16 * (width - 1) + 5] + [0] * n


def check(case, call):
    n, P, width, used = case
    table, refs, source, target, lengths = program(*case)
    cache = pool(P, 1, 16, 64, torch.bfloat16, seed=n)
    gt, gr, before = i32(table), i32(refs), raw(cache)
    call(cache, gr, gt, i32(source), i32(target), i32(lengths))
    refs, table, copies = ref.fork(refs, table, source, target, lengths, 16)
    assert gt.tolist() == table and gr.tolist() == refs
    for x, y in zip(before, raw(cache)):
        for old, new, k in copies:
            x[new, :, :k] = x[old, :, :k]
        assert torch.equal(x, y)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_more_forks_than_pages(case, host_path):  # noqa: F811
    from lvar_amd import kv_cache_ops as kv
    check(case, kv.kv_cache_fork)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_scratch_of_the_least_size(case):
    from lvar_amd import _lib, kv_cache_ops as kv
    lib = _lib.load()

    def call(cache, refs, table, source, target, lengths):
        n, need = source.numel(), lib.lvar_kv_pages_scratch_bytes(source.numel(), refs.numel())
        room = torch.full((need + (1 << 18),), 0x5A, dtype=torch.uint8, device="cuda")
        arg = kv._cache_arg(cache, table, table.shape[0], refs.device)
        arg.table_stride = table.shape[1]
        ptr = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        st = lib.lvar_kv_cache_fork(arg, ptr(refs), ptr(table), table.shape[0], ptr(source), ptr(target), ptr(lengths), n, ptr(room), need,
                                    C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert st == 0 and bool((room[need:] == 0x5A).all()), "written behind the scratch"

    check(case, call)
