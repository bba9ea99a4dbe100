"""Pages of a cache that are opened, dropped, forked and compacted, on the GPU, against lists on the CPU: whole numbers and bytes, equal."""
import random

import pytest
import torch

from oracle import pages_oracle as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["compiled", "ctypes"])
def host_path(request, monkeypatch):
    from lvar_amd import kv_cache_ops
    if request.param == "ctypes":
        monkeypatch.setattr(kv_cache_ops, "_native", lambda: None)
    return request.param


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(P, H, page, d, dtype, seed=0):
    """A cache of random bytes (every bit pattern of bf16 and e4m3, and exponents)."""
    from lvar_amd.kv_cache_ops import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    bits = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)  # noqa: E731
    if dtype == torch.bfloat16:
        return PagedKVCache(*(bits(P, H, page, 2 * d).view(torch.bfloat16).cuda() for _ in range(2)))
    return PagedKVCache(*(bits(P, H, page, d).view(dtype).cuda() for _ in range(2)), *(bits(P, H, page).cuda() for _ in range(2)))


def raw(cache):
    return [t.view(torch.uint8).cpu() if t.dtype != torch.bfloat16 else t.view(torch.int16).cpu() for t in cache if t is not None]


def tables(rows, width, P, seed, holes=True):
    """A table whose rows name pages of their own, with odd entries, and the counts."""
    r = random.Random(seed)
    pages = list(range(P))
    r.shuffle(pages)
    table, refs = [], [0] * P
    for b in range(rows):
        n = r.randrange(width + 1)
        row = [pages.pop() if pages else -1 for _ in range(n)] + [-1] * (width - n)
        if holes and n > 2:
            row[r.randrange(n)] = r.choice((-7, P, P + 5))
        for p in row:
            if 0 <= p < P:
                refs[p] += 1
        table.append(row)
    return table, refs


@pytest.mark.parametrize("rows,width,P", [(1, 1, 1), (3, 5, 7), (20, 9, 300), (200, 12, 1900), (7, 300, 4000), (64, 33, 2500), (5000, 3, 20000), (2, 9000, 20001)])
def test_free_and_alloc(rows, width, P, host_path):
    from lvar_amd import kv_cache_ops as kv
    table, refs = tables(rows, width, P, seed=rows)
    r = random.Random(P)
    keep = [r.randrange(-2, width + 3) for _ in range(rows)]
    gt, gr = i32(table), i32(refs)
    kv.kv_pages_free(gr, gt, i32(keep))
    refs, table = ref.free(refs, table, keep)
    assert gr.tolist() == refs and gt.tolist() == table
    for _ in range(2):
        first = [r.randrange(-3, width + 3) for _ in range(rows)]
        last = [r.choice((f, f + 1, f + r.randrange(width + 3), 2 ** 31 - 1, -2 ** 31)) for f in first]
        kv.kv_pages_alloc(gr, gt, i32(first), i32(last))
        refs, table = ref.alloc(refs, table, first, last)
        assert gr.tolist() == refs and gt.tolist() == table
    kv.kv_pages_free(gr, gt)
    refs, table = ref.free(refs, table)
    assert gr.tolist() == refs and gt.tolist() == table


def test_alloc_of_extreme_ranges(host_path):
    """first beyond the row and last below nothing: no entry, and no difference that leaves 32 bits."""
    from lvar_amd import kv_cache_ops as kv
    table, refs = i32([[5, 6], [7, 8], [1, 2]]), i32([0] * 9)
    kv.kv_pages_alloc(refs, table, i32([2 ** 31 - 1, -2 ** 31, 2]), i32([-2 ** 31, -2 ** 31, 2 ** 31 - 1]))
    assert table.tolist() == [[5, 6], [7, 8], [1, 2]] and refs.tolist() == [0] * 9


def test_alloc_wants_more_than_there_are(host_path):
    """2048 rows of 1.1 million entries each: what they want in all is beyond 31 bits."""
    from lvar_amd import kv_cache_ops as kv
    B, n, P = 2048, 1100000, 9000
    table = torch.full((B, n), -5, dtype=torch.int32, device="cuda")
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    refs[::3] = 1
    want = torch.nonzero(refs == 0).flatten().int()
    kv.kv_pages_alloc(refs, table, i32([0] * B), i32([n] * B))
    assert torch.equal(table[0, :want.numel()], want) and bool((table[0, want.numel():] == -1).all()) and bool((table[1:] == -1).all())
    assert bool((refs == 1).all())


FORKS = [
    # rows, entries, page, heads, head_dim, dtype
    (6, 4, 16, 1, 64, torch.bfloat16),
    (9, 5, 64, 3, 128, torch.bfloat16),
    (12, 3, 32, 2, 256, torch.float8_e4m3fn),
    (40, 6, 16, 5, 64, torch.float8_e4m3fn),
]


@pytest.mark.parametrize("case", FORKS, ids=str)
@pytest.mark.parametrize("scarce", [False, True])
def test_fork(case, scarce, host_path):
    from lvar_amd import kv_cache_ops as kv
    rows, width, page, H, d, dtype = case
    P = rows * width + 5
    table, refs = tables(rows, width, P, seed=rows + page)
    if scarce:   # two pages are free
        gone = [p for p in range(P) if refs[p] == 0][2:]
        for p in gone:
            refs[p] = 1
    cache = pool(P, H, page, d, dtype, seed=rows)
    r = random.Random(rows)
    lengths = [r.choice((0, 1, page - 1, page, page + 1, 2 * page, width * page, width * page + 9, -4, r.randrange(width * page))) for _ in range(rows)]
    half = rows // 2
    source = [r.randrange(half) for _ in range(half, rows)] + [-1, 0, rows, 1]      # the last ones are left out
    target = list(range(half, rows)) + [0, rows + 3, 1, 1]
    refs, table = ref.free(refs, table, [width] * half + [0] * (rows - half))
    gt, gr, before = i32(table), i32(refs), raw(cache)
    kv.kv_cache_fork(cache, gr, gt, i32(source), i32(target), i32(lengths))
    refs, table, copies = ref.fork(refs, table, source, target, lengths, page)
    assert gt.tolist() == table and gr.tolist() == refs
    for x, y in zip(before, raw(cache)):
        for old, new, n in copies:
            x[new, :, :n] = x[old, :, :n]
        assert torch.equal(x, y)


def test_many_forks(host_path):
    """More forks than the search keeps in LDS."""
    from lvar_amd import kv_cache_ops as kv
    n, P = 9000, 9100
    cache = pool(P, 1, 16, 64, torch.bfloat16)
    table = [[9050, -1]] + [[-1, -1]] * n
    refs = [0] * P
    refs[9050] = 1
    refs[::7] = [1] * len(refs[::7])
    gt, gr = i32(table), i32(refs)
    kv.kv_cache_fork(cache, gr, gt, i32([0] * n), i32(list(range(1, n + 1))), i32([5] * (n + 1)))
    refs, table, copies = ref.fork(refs, table, [0] * n, range(1, n + 1), [5] * (n + 1), 16)
    assert gt.tolist() == table and gr.tolist() == refs
    fresh = torch.tensor([c[1] for c in copies], device="cuda")
    assert bool((cache.v.view(torch.int16)[fresh, 0, :5] == cache.v.view(torch.int16)[9050, 0, :5]).all())


@pytest.mark.parametrize("rows", [6, 40, 400, 5000])
def test_forks_that_depend_on_each_other(rows, host_path):
    """Targets that are named twice, or sources themselves, are left out; nothing of their rows, pages and counts changes."""
    from lvar_amd import kv_cache_ops as kv
    r = random.Random(rows)
    P, width, page = 3 * rows + 7, 3, 16
    table, refs = tables(rows, width, P, seed=rows, holes=False)
    cache = pool(P, 1, page, 64, torch.bfloat16, seed=rows)
    lengths = [r.randrange(width * page + 9) for _ in range(rows)]
    pairs = [(0, 1), (1, 2), (2, 3), (0, 4), (3, 4), (5, 5)] if rows == 6 else [(r.randrange(rows), r.randrange(-1, rows + 1)) for _ in range(rows // 2)]
    source, target = zip(*pairs)
    gt, gr, before = i32(table), i32(refs), raw(cache)
    kv.kv_cache_fork(cache, gr, gt, i32(source), i32(target), i32(lengths))
    refs, table, copies = ref.fork(refs, table, source, target, lengths, page)
    assert gt.tolist() == table and gr.tolist() == refs and (rows > 6 or len(copies) <= 1)
    for x, y in zip(before, raw(cache)):
        for old, new, n in copies:
            x[new, :, :n] = x[old, :, :n]
        assert torch.equal(x, y)


COMPACT = [
    # B, heads, entries, page, head_dim, kept, dtype
    (1, 1, 1, 16, 64, 1, torch.bfloat16),
    (2, 3, 5, 16, 128, 37, torch.bfloat16),
    (3, 2, 3, 64, 256, 100, torch.float8_e4m3fn),
    (2, 5, 4, 32, 64, 70, torch.float8_e4m3fn),
]


@pytest.mark.parametrize("case", COMPACT, ids=str)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_compact(case, dtype, host_path):
    from lvar_amd import kv_cache_ops as kv
    B, H, width, page, d, n, kind = case
    out = -(-n // page) + 1
    P = B * (width + out) + 2
    cache = pool(P, H, page, d, kind, seed=n)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(n)).tolist()
    table = [order[b * width:(b + 1) * width] for b in range(B)]
    at = B * width
    out_table = [order[at + b * out:at + (b + 1) * out] for b in range(B)]
    if width > 2:
        table[0][1], table[-1][2] = -1, P + 3
        out_table[-1][0] = -2
    g = torch.Generator().manual_seed(n + 1)
    keep = torch.randint(-3, width * page + 5, (B, n, H), generator=g).to(dtype).transpose(1, 2)       # any order, twice, and outside
    if dtype == torch.int64:
        keep[0, 0, 0] = 2 ** 40
    for counts in (None, [n - 1, 0, n + 4][:B]):
        before = raw(cache)
        kv.kv_cache_compact(cache, i32(table), keep.cuda(), i32(out_table), counts=None if counts is None else i32(counts))
        for x, y, nothing in zip(before, raw(cache), (0, 0, 127, 127)):
            assert torch.equal(ref.compact(x, table, keep, out_table, counts, nothing), y)


def test_compact_of_broadcast_positions(host_path):
    from lvar_amd import kv_cache_ops as kv
    cache = pool(8, 4, 16, 64, torch.bfloat16)
    keep = torch.tensor([3, 9, 20])[None, None].expand(2, 4, 3)
    before = raw(cache)
    kv.kv_cache_compact(cache, i32([[0, 1], [2, 3]]), keep.cuda()[:1, :1].expand(2, 4, 3), i32([[4], [5]]))
    for x, y in zip(before, raw(cache)):
        assert torch.equal(ref.compact(x, [[0, 1], [2, 3]], keep, [[4], [5]]), y)
