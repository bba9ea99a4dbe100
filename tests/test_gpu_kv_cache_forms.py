"""Forms of the launches that sizes alone choose: several heads per workgroup, gradients over more tiles than workgroups, cut calls beyond one round, row tiles of
a prompt, probabilities in two terms.  Sizes follow from the rules that choose, and each test says so."""
import math

import pytest
import torch

import test_gpu_kv_cache as base
from oracle import kv_cache_oracle as ref
from oracle.paged_plan import Plan
from test_gpu_kv_cache import BF16, EPS, F32, attn_case, check_attn, check_rows, cu, make_cache, projection, rand, same_bytes, table_for, tables, to_gpu, weight

pytestmark = pytest.mark.gpu

both = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


# ---- norms ----

def tokens_for(chunks: int, d: int, workgroups: int) -> int:
    """Tokens that give `workgroups` workgroups and a few more, with a last tile that is not full."""
    rpb = 256 * 8 // d
    return (-(-workgroups // chunks) + 3) * rpb + rpb // 2 + 1


def four_heads(H: int, Hkv: int, d: int, append: bool, ready: bool = False) -> int:
    """Tokens from which on a workgroup takes four heads: four such workgroups per compute unit."""
    up = lambda n: -(-n // 4)  # noqa: E731
    chunks = (0 if ready else up(H)) + (2 if append else 1) * up(Hkv)
    L = tokens_for(chunks, d, 4 * cus())
    assert -(-L // (2048 // d)) * chunks >= 4 * cus()
    return L


@pytest.mark.parametrize("d,H,Hkv,wk,inter,norm", [(16, 14, 7, "full", True, "l2"), (32, 6, 6, "head", False, "rms"), (64, 10, 5, "dim", False, "l2"), (128, 7, 7, "head", True, "l2"),
                                                   (256, 6, 3, None, False, None)])
def test_norm_with_four_heads_per_workgroup(d, H, Hkv, wk, inter, norm):
    from lvar_amd import kv_cache_ops as kv
    L = four_heads(H, Hkv, d, False)
    q, k, _ = projection(1, H, Hkv, L, d, seed=d)
    w = [weight(wk, h, d, 7 + i) for i, h in enumerate((H, Hkv))]
    cos, sin = tables(L, d // 2)
    got = kv.qk_norm_rope(q.cuda(), k.cuda(), cos.cuda(), sin.cuda(), None, cu(w[0]), cu(w[1]), norm, None, inter)
    at = ref.table_rows(1, L, L)
    for x, y, wx in ((q, got[0], w[0]), (k, got[1], w[1])):
        check_rows(y, ref.norm_rope(x, wx, cos, sin, at, norm, EPS[norm], inter), (d, norm))


def long_append(d, H, Hkv, L, dtype, page=64):
    """A cache, its table and where two sequences go on, one of them padded, for L new tokens in all."""
    n = L // 2 + 1
    starts, counts = torch.tensor([37, 5], dtype=torch.int32), torch.tensor([n, n - 19], dtype=torch.int32)
    per = -(-(37 + n) // page)
    cache = make_cache(2 * per + 1, Hkv, page, d, dtype, 4)
    table = table_for(2, per, 2 * per + 1, 1)
    table[0, 1] = -1
    return n, starts, counts, cache, table, projection(2, H, Hkv, n, d, seed=5, amp=2.0)


@pytest.mark.parametrize("d,Hkv", [(64, 6), (128, 5), (256, 3)])
@both
def test_append_with_four_heads_per_workgroup(d, Hkv, dtype):
    from lvar_amd import kv_cache_ops as kv
    n, starts, counts, cache, table, (_, k, v) = long_append(d, Hkv, Hkv, four_heads(Hkv, Hkv, d, True, True), dtype)
    g = to_gpu(cache)
    kv.kv_cache_append(g, k.cuda(), v.cuda(), table.cuda(), starts.cuda(), counts.cuda())
    for pages, exps, x, got, got_e in ((cache.k, cache.k_exp, k, g.k, g.k_exp), (cache.v, cache.v_exp, v, g.v, g.v_exp)):
        want, want_e = ref.append(pages, exps, table, x, starts, counts)
        assert same_bytes(got, want) and (want_e is None or torch.equal(got_e.cpu(), want_e))


@pytest.mark.parametrize("d,H,Hkv,wk,inter,norm", [(64, 10, 5, "dim", False, "rms"), (128, 7, 7, "head", True, "l2"), (256, 6, 3, "full", True, "l2")])
@both
def test_norm_and_append_with_four_heads_per_workgroup(d, H, Hkv, wk, inter, norm, dtype):
    from lvar_amd import kv_cache_ops as kv
    n, starts, counts, cache, table, (q, k, v) = long_append(d, H, Hkv, four_heads(H, Hkv, d, True), dtype)
    w = [weight(wk, h, d, 7 + i) for i, h in enumerate((H, Hkv))]
    rows = n + 40
    cos, sin = tables(rows, d // 2)
    g = to_gpu(cache)
    oq = kv.qk_norm_rope_append(g, q.cuda(), k.cuda(), v.cuda(), table.cuda(), starts.cuda(), cos.cuda(), sin.cuda(), counts.cuda(), None, cu(w[0]), cu(w[1]), norm, None, inter)
    at = ref.table_rows(2, n, rows, None, starts)
    check_rows(oq, ref.norm_rope(q, w[0], cos, sin, at, norm, EPS[norm], inter), "q")
    want, want_e = ref.append(cache.v, cache.v_exp, table, v, starts, counts)
    assert same_bytes(g.v, want) and (want_e is None or torch.equal(g.v_exp.cpu(), want_e))
    # keys: one rounding from 32 bits, to bf16 or to e4m3 with a power of two of at most top / 224; rows nobody wrote as they were
    wanted = ref.norm_rope(k, w[1], cos, sin, at, norm, EPS[norm], inter)
    lens = starts + counts
    got, there = ref.read(g.k.cpu(), None if g.k_exp is None else g.k_exp.cpu(), table, lens, n, starts)
    there = there[:, None].expand(2, Hkv, n)
    top = wanted.abs().amax(-1, keepdim=True)
    tol = BF16 * wanted.abs() if dtype is torch.bfloat16 else 2.0 ** -4 * wanted.abs() + top / 224 * 2.0 ** -10
    tol = tol + (d + 16) * F32 * 2 * top
    assert bool(((got - wanted).abs() <= tol)[there].all())
    # (the rows that are written are those that zeros would be written to)
    mark, _ = ref.append(cache.k, cache.k_exp, table, torch.zeros_like(k), starts, counts)
    kept = (mark.view(torch.uint8 if mark.element_size() == 1 else torch.int16) != 0)
    view = torch.uint8 if mark.element_size() == 1 else torch.int16
    assert torch.equal(g.k.cpu().view(view)[kept], cache.k.view(view)[kept])


@pytest.mark.parametrize("kind", ["head", "full", "dim", "one"])
@pytest.mark.parametrize("d,H,Hkv,norm", [(64, 5, 5, "l2"), (256, 3, 1, "rms"), (16, 2, 2, "l2")])
def test_gradients_over_more_tiles_than_workgroups(kind, d, H, Hkv, norm):
    """Eight workgroups per compute unit take the tiles in turn; their partial sums are more than 256 rows, and more than 8 x 1024 numbers."""
    chunks = -(-H // 2) + -(-Hkv // 2)
    blocks = -(-8 * cus() // chunks)
    tokens = blocks * (2048 // d) * 2 + 77                 # two tiles for each, three for some
    assert blocks > 256 or cus() < 128
    L = tokens // 3 + 1
    base.test_norm_rope_gradients((3, H, Hkv, L, d, d, norm, kind, d != 64, None), torch.float32 if d != 16 else torch.bfloat16)


# ---- cut calls ----

def shared_case(B, H, Hkv, Lq, lengths, d, dtype, causal=False, counts=None, page=256, seed=0):
    """All sequences over the same pages (a cache of one), through the entry point with a workspace of its own, so that the plan it holds can be read.  The
    reference is a product of all rows at once."""
    from lvar_amd import _lib, kv_cache_ops as kv
    n = max(lengths)
    per = -(-n // page)
    cache = make_cache(per, Hkv, page, d, dtype, seed)
    table = torch.arange(per, dtype=torch.int32).view(1, per)
    x = [rand(1, Hkv, n, d, seed=seed + i) for i in (1, 2)]
    g = to_gpu(cache)
    kv.kv_cache_append(g, x[0].cuda(), x[1].cuda(), table.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    k, v = (t if dtype is torch.bfloat16 else ref.dequantise(*ref.quantise(t)) for t in x)
    q = rand(B, H, Lq, d, seed=seed + 9)
    lens, c = torch.tensor(lengths, dtype=torch.int32), None if counts is None else torch.tensor(counts, dtype=torch.int32)
    tables_ = table.cuda().expand(B, per)
    lib = _lib.load()
    o, M, L = torch.full((B, H, Lq, d), 7.0, dtype=torch.bfloat16, device="cuda"), *(torch.full((B, H, Lq, 1), 7.0, device="cuda") for _ in range(2))
    plan = Plan(lengths, counts, H, Hkv, Lq, d, dtype is not torch.bfloat16, per * page, cus())
    need = lib.lvar_paged_attn_workspace_bytes(B, H, Hkv, Lq, per * page, d)
    assert need == plan.ws_bytes > 0
    guard = 4096
    ws = torch.full((need + guard,), 0x5a, dtype=torch.uint8, device="cuda")
    qg, lg, cg = q.cuda(), lens.cuda(), cu(c)              # (named: they live until the call has run)
    st = lib.lvar_paged_attn_fwd(kv._view(qg), kv._cache_arg(g, tables_, B, qg.device), lg.data_ptr(), None if cg is None else cg.data_ptr(), o.data_ptr(), M.data_ptr(), L.data_ptr(),
                                 ws.data_ptr(), need, B, H, Lq, per * page, 1 if causal else 0, d ** -0.5, kv._stream(qg))
    assert st == 0
    torch.cuda.synchronize()
    assert bool((ws[need:] == 0x5a).all()), "written behind the workspace"
    head = ws[:8 * B].view(torch.int32).cpu().view(B, 2)
    assert head[:, 0].tolist() == plan.n and [s for s, m in zip(head[:, 1].tolist(), plan.n) if m > 1] == [s for s, m in zip(plan.first_slot, plan.n) if m > 1]
    # reference
    G = H // Hkv
    new = [Lq] * B if counts is None else [max(0, min(Lq, m)) for m in counts]
    i = torch.arange(Lq)
    limit = torch.stack([torch.where(i < new[b], (lengths[b] - new[b] + i + 1).clamp_min(0) if causal else torch.full_like(i, lengths[b]), 0) for b in range(B)])   # [B, Lq]
    got = [t.cpu() for t in (o, M, L)]
    for h in range(Hkv):
        rows = q[:, h * G:(h + 1) * G].double().reshape(B * G * Lq, d)
        lim = limit[:, None].expand(B, G, Lq).reshape(-1, 1)
        s = (rows @ k[0, h].double().T) * (d ** -0.5 * math.log2(math.e))
        s.masked_fill_(torch.arange(n) >= lim, -math.inf)
        Mr = s.amax(-1, keepdim=True)
        p = torch.exp2(s - torch.where(torch.isinf(Mr), 0.0, Mr))
        Lr = p.sum(-1, keepdim=True)
        none = Lr == 0
        Lr = torch.where(none, 1.0, Lr)
        p /= Lr
        shape = lambda t: t.view(B, G, Lq, -1)  # noqa: E731
        check_attn(*(t[:, h * G:(h + 1) * G] for t in got), shape(p @ v[0, h].double()), shape(Mr), shape(Lr), shape(p @ v[0, h].double().abs()), q, k, d ** -0.5, n)
    return plan


def ragged(B, most):
    return [max(1, int(most * (1 - (b * 0.618034) % 1))) for b in range(B)]


# (way that the plan takes on 256 compute units, then the call)
PLANS = [
    ("target", (61, 6, 3, 1, [3000] + ragged(60, 1100), 128, False, None)),   # up to 4 stages per compute unit
    ("wide", (64, 4, 2, 1, ragged(64, 8000), 128, True, None)),
    ("wider", (30, 12, 6, 1, ragged(30, 9000), 64, False, None)),
    ("target", (12, 8, 8, 1, ragged(12, 46000), 64, True, None)),             # more than 64 per compute unit
    ("finer", (130, 4, 4, 1, ragged(130, 8000), 64, True, None)),             # three waves of sequences, no round holds their pieces
    ("finer", (260, 5, 5, 1, ragged(260, 4500), 64, False, None)),
    ("one round", (16, 8, 8, 1, [2560] * 16, 128, False, None)),              # alike
    ("wide", (70, 2, 1, 12, ragged(70, 7000), 64, True, None)),               # 24 rows
    ("target", (70, 2, 1, 25, ragged(70, 2600), 128, True, [(7 * b) % 27 - 1 for b in range(70)])),    # staged
    ("wide", (90, 3, 1, 70, ragged(90, 4500), 128, True, [(11 * b) % 72 for b in range(90)])),         # staged, several row tiles, padded
    ("wide", (40, 2, 2, 90, ragged(40, 3000), 256, False, None)),
    ("wide", (48, 3, 3, 1, ragged(48, 2700), 256, True, None)),
]


@pytest.mark.parametrize("way,case", PLANS)
@both
def test_plans_beyond_one_round(way, case, dtype):
    B, H, Hkv, Lq, lengths, d, causal, counts = case
    plan = shared_case(B, H, Hkv, Lq, lengths, d, dtype, causal, counts, seed=B)
    assert plan.cut
    if cus() == 256 and dtype is torch.bfloat16:
        assert plan.way == way, (plan.way, plan.total, plan.target, plan.some, plan.many, plan.most)


@both
def test_plans_of_fine_pieces(dtype):
    """Short and long sequences such that no round holds the pieces: they are cut finely."""
    lengths = [257 + 128 * (b % 2) for b in range(600)] + [9000] * 8
    plan = shared_case(608, 1, 1, 1, lengths, 128, dtype, seed=3)
    assert plan.cut
    if cus() == 256:
        assert plan.way == "finer", (plan.way, plan.total, plan.pieces)


# ---- many row tiles, and keys that few rows see ----

@pytest.mark.parametrize("B,H,Hkv,Lq,lengths,d,causal,counts", [
    (1, 2, 1, 600, [600], 128, True, None), (2, 1, 1, 700, [700, 760], 64, True, [700, 333]), (1, 1, 1, 500, [501], 256, True, None),
    (1, 1, 1, 1300, [1300], 128, True, None), (1, 1, 1, 1100, [1500], 64, False, None), (1, 2, 2, 700, [300], 128, True, None),      # more new tokens than the cache holds
])
@both
def test_prompts(B, H, Hkv, Lq, lengths, d, causal, counts, dtype):
    """Row tiles whose limits lie far before the end of the sequence: pieces behind them are empty and are joined all the same."""
    attn_case(B, H, Hkv, Lq, lengths, d, 64, dtype, causal, counts, extra=0, seed=Lq)


# ---- probabilities ----

def test_probabilities_are_two_terms():
    """Up to 32 rows (in bf16, head_dim 256: none), what the probabilities lose on their way into the second product is 2^-16 of them, not 2^-8: keys whose values cancel,
    so that the rounding of the result does not hide it.  A rounding to one bf16 term, made here, breaks the bound."""
    from lvar_amd import kv_cache_ops as kv
    for d, rows, dtype in ((64, 1, torch.bfloat16), (128, 16, torch.bfloat16), (128, 20, torch.bfloat16), (64, 32, torch.bfloat16), (64, 1, torch.float8_e4m3fn), (128, 32, torch.float8_e4m3fn),
                           (256, 1, torch.float8_e4m3fn), (256, 16, torch.float8_e4m3fn)):
        B, n, page, scale = 12, 12, 16, 1.0
        stored = (lambda t: t.to(torch.bfloat16)) if dtype is torch.bfloat16 else (lambda t: ref.dequantise(*ref.quantise(t)).to(torch.bfloat16))
        g = torch.Generator().manual_seed(d + rows)
        k = torch.zeros(B, 1, n, d)
        k[..., 0] = torch.rand(B, 1, n, generator=g) * 1.5           # scores 0 .. 1.5: no probability stands out
        k, v = stored(k.to(torch.bfloat16)), torch.zeros(B, 1, n, d)
        q = torch.zeros(B, 1, 1, d, dtype=torch.bfloat16)
        q[..., 0] = 1
        s = k[:, 0, :, 0].double() * (scale * math.log2(math.e))
        p = torch.exp2(s - s.amax(-1, keepdim=True))
        v[:, :, :9] = torch.sign(torch.randn(B, 1, 9, d, generator=g))
        for j in (9, 10, 11):                                        # each takes away what is left but for its own rounding
            left = (p[:, None, :, None] * v.double()).sum(2)
            v[:, :, j] = stored((-left / p[:, None, j, None]).to(torch.bfloat16)).float()
        v = v.to(torch.bfloat16)
        cache = kv.PagedKVCache.alloc(B, 1, d, page, dtype)
        table, lens = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1), torch.full((B,), n, dtype=torch.int32, device="cuda")
        kv.kv_cache_append(cache, k.cuda(), v.cuda(), table, lens - n)
        rk, rv = kv.kv_cache_read(cache, table, lens, n)
        assert torch.equal(rk.cpu(), k) and torch.equal(rv.cpu(), v)
        o, (M, L) = kv.paged_attn(q.cuda().expand(B, 1, rows, d), cache, table, lens, scale=scale)
        sums = lambda w: (w[:, None, :, None] * v.double()).sum(2, keepdim=True) / p.sum(-1)[:, None, None, None]  # noqa: E731
        want, spread = sums(p), (p[:, None, :, None] * v.double().abs()).sum(2, keepdim=True) / p.sum(-1)[:, None, None, None]
        # scores exact up to the product with log2(e) (two roundings of at most 2.2), the hardware's exponential a step, 12 sums, the two terms 2^-16, the result's own half step
        tol = (2.0 ** -16 + (2 * 2.2 + 2 + 2 * 12) * F32) * spread + BF16 * want.abs() + 1e-30
        err = (o.double().cpu() - want).abs()
        assert bool((err <= tol).all()), f"{(d, rows, dtype)}: {float((err / tol).max()):.3g} of the bound"
        once = (sums(p.to(torch.bfloat16).double()) - want).abs()
        assert bool((once > 2 * tol).any()), "the case does not show a single rounding"
