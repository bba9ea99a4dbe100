"""The operators of whole prompts, as cases that can be timed: attention over packed sequences of different lengths (and its
gradients), norms with a rotation whose angle comes from several position axes (into tensors or into a paged cache, and its gradients),
and the life of the pages of a cache: dropping, forking and opening them, and keeping a chosen part of a sequence.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, angles in 64, rounded once at the end) or, with
``own`` set, through the entry points of ``lvar_amd.packed_ops`` and ``lvar_amd.kv_cache_ops``.  Sizes are those of the Infinity-2B
schedule (16 heads of 128, images of 64 x 64 tokens, 10521 tokens over all scales) and of VAR-d16 (heads of 64, 680 tokens) where a
comment says so, and generic sizes (32 query heads over 8 key/value heads, prompts of up to 32768 tokens) elsewhere; drawn cases
spread over the same ranges.

Lengths of ragged batches follow a fixed formula of the case, so that ``work`` can count them; everything else comes from
the seed.
"""
import math

import torch

own = False

LOG2E = 1.4426950408889634


def listed():
    return [
        # one short prompt before the first scale of an image (VAR-d16's heads): launch and latency
        dict(name="prompt_short", kind="attn", train=False, B=1, H=16, Hkv=16, d=64, Lmax=77, ragged=False, causal=True, keys=0),
        # sixteen prompts of very different lengths at once, grouped heads, rows of padding behind the last
        dict(name="prompts_ragged", kind="attn", train=False, B=16, H=32, Hkv=8, d=128, Lmax=4096, ragged=True, causal=True, keys=0),
        # one long prompt
        dict(name="prompt_long", kind="attn", train=False, B=1, H=32, Hkv=8, d=128, Lmax=32768, ragged=False, causal=True, keys=0),
        # a training step over packed texts, grouped heads: outputs and gradients of queries, keys and values
        dict(name="train_ragged", kind="attn", train=True, B=12, H=32, Hkv=8, d=128, Lmax=2047, ragged=True, causal=True, keys=0),
        # a training step of image tokens (four images of the last scale) that attend to packed texts of up to 300 tokens, heads of 64
        dict(name="train_image_to_text", kind="attn", train=True, B=4, H=16, Hkv=16, d=64, Lmax=4096, ragged=False, causal=False, keys=300),
        # scale 4 of an image: 16 tokens on a 64 x 64 grid, positions that are not whole numbers; launch and latency
        dict(name="axes_scale_4", kind="rope", how="step", B=2, H=16, Hkv=16, L=16, d=128, rot=128, axes=2, mixed=False, norm="l2", weight="head", interleaved=True, own_positions=False),
        # a training step over 8 frames of 64 x 64 tokens: time, row and column
        dict(name="axes_train_video", kind="rope", how="train", B=1, H=32, Hkv=8, L=32768, d=128, rot=128, axes=3, mixed=False, norm="rms", weight="dim", interleaved=False, own_positions=False),
        # the last scale of an image into an 8-bit cache
        dict(name="axes_append_scale_64_e4m3", kind="rope", how="append", B=2, H=16, Hkv=16, L=4096, d=128, rot=128, axes=2, mixed=False, norm="l2", weight="head", interleaved=True, own_positions=False, page=64, cache="e4m3"),
        # a prompt that becomes four images, which drop what they had: bookkeeping and a few rows, latency
        dict(name="fork_four", kind="fork", S=1, n=4, Hkv=16, d=128, page=64, Lmax=1000, grow=1, cache="bf16"),
        # 48 prompts of different lengths with four samples each
        dict(name="fork_48_prompts", kind="fork", S=48, n=4, Hkv=8, d=128, page=64, Lmax=2500, grow=2, cache="bf16"),
        # a tenth of the cache of an image is kept, other positions for every head
        dict(name="compact_image", kind="compact", B=2, Hkv=16, d=128, page=64, Lmax=10521, keep=1052, ragged=False, cache="bf16"),
        # the same of a batch in 8 bits, another number for every sequence
        dict(name="compact_ragged_e4m3", kind="compact", B=8, Hkv=8, d=128, page=64, Lmax=8191, keep=4001, ragged=True, cache="e4m3"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most=40):
    Hkv = rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
    return Hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 7, 8) if g * Hkv <= most]), Hkv


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "rope", "rope", "fork", "compact"))
    while True:
        H, Hkv = _heads(rng)
        d = rng.choice((64, 128, 128, 256))
        if kind == "attn":
            causal = rng.random() < 0.7
            c = dict(kind=kind, train=rng.random() < 0.5, B=_log_int(rng, 1, 64), H=H, Hkv=Hkv, d=d, Lmax=_log_int(rng, 1, 32768),
                     ragged=rng.random() < 0.6, causal=causal, keys=_log_int(rng, 1, 4096) if rng.random() < (0.2 if causal else 0.6) else 0)
            w = work(c)
            if sum(_lengths(c)[0]) * (H + 2 * Hkv) * d <= 3e8 and sum(_lengths(c)[1]) * Hkv * d <= 3e8 and w["flops"] <= 4e12:
                return c
        elif kind == "rope":
            how = rng.choice(("step", "train", "append"))
            if how != "append":
                d = rng.choice((d, 32, 16))
            axes = rng.choice((1, 2, 2, 3, 4))
            c = dict(kind=kind, how=how, B=_log_int(rng, 1, 64), H=H, Hkv=Hkv, L=_log_int(rng, 1, 32768), d=d, rot=max(16, d // rng.choice((1, 1, 2))),
                     axes=axes, mixed=rng.random() < 0.3, norm=rng.choice(("l2", "rms", "none")), weight=rng.choice(("none", "head", "dim", "full")),
                     interleaved=rng.random() < 0.5, own_positions=rng.random() < 0.4)
            if how == "append":
                c.update(page=rng.choice((16, 32, 64, 128, 256)), cache=rng.choice(("bf16", "e4m3")))
            if c["B"] * (H + 2 * Hkv) * c["L"] * d <= 3.2e8:
                return c
        elif kind == "fork":
            c = dict(kind=kind, S=_log_int(rng, 1, 64), n=_log_int(rng, 1, 16), Hkv=Hkv, d=d, page=rng.choice((16, 32, 64, 128, 256)),
                     Lmax=_log_int(rng, 1, 8192), grow=rng.choice((0, 1, 2, 5)), cache=rng.choice(("bf16", "bf16", "e4m3")))
            if _fork_pages(c) * c["page"] * Hkv * d <= 3e8:
                return c
        else:
            Lmax = _log_int(rng, 1, 32768)
            c = dict(kind=kind, B=_log_int(rng, 1, 32), Hkv=Hkv, d=d, page=rng.choice((16, 32, 64, 128, 256)), Lmax=Lmax,
                     keep=_log_int(rng, 1, Lmax), ragged=rng.random() < 0.5, cache=rng.choice(("bf16", "e4m3")))
            if c["B"] * 2 * (Lmax + c["page"]) * Hkv * d <= 6e8:
                return c


# ---- what a case is made of ----

def _lengths(c):
    """Queries and keys of every sequence (fixed by the case): some of a ragged batch have no token, some texts no key."""
    B = c["B"]
    q = [c["Lmax"]] * B
    if c["ragged"]:
        q = [0 if b % 8 == 5 else max(1, int(c["Lmax"] * (1.0 - (b * 0.618034) % 1.0))) for b in range(B)]
    if not c["keys"]:
        return q, q
    return q, [0 if b % 8 == 6 else max(1, int(c["keys"] * (1.0 - (b * 0.381966) % 1.0))) for b in range(B)]


def _pairs(c):
    """(query, key) pairs that count, per head."""
    total = 0
    for n, m in zip(*_lengths(c)):
        if c["causal"]:
            see = min(n, m)                      # the last `see` rows see m - see + 1 .. m keys
            total += see * (m - see) + see * (see + 1) // 2
        else:
            total += n * m
    return total


def _fork_lengths(c):
    return [max(1, int(c["Lmax"] * (1.0 - (s * 0.618034) % 1.0))) for s in range(c["S"])]


def _fork_pages(c):
    per = [-(-n // c["page"]) for n in _fork_lengths(c)]
    return sum(per) + c["S"] * c["n"] * (1 + c["grow"]) + 9


def _kept(c):
    return [max(1, c["keep"] - int(c["keep"] * ((b * 0.381966) % 1.0))) if c["ragged"] else c["keep"] for b in range(c["B"])]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _pages(c, shape, gen):
    s = {}
    for n in ("k", "v"):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
        if c["cache"] == "bf16":
            s[n + "_pages"], s[n + "_exp"] = x.mul_(0.5), None
        else:
            s[n + "_pages"] = x.mul_(64).to(torch.float8_e4m3fn)
            s[n + "_exp"] = torch.randint(118, 122, shape[:3], generator=gen, device="cuda", dtype=torch.uint8)
    return s


def _weight(c, heads, gen):
    if c["weight"] == "none":
        return None
    w = torch.randn({"head": (heads, 1), "dim": (c["d"],), "full": (heads, c["d"])}[c["weight"]], generator=gen, device="cuda")
    return torch.exp(1.4 + 0.3 * w) if c["norm"] == "l2" else 1.0 + 0.2 * w


def _positions(c, gen):
    """[axes, L] (or [B, axes, L]): a grid of tokens with the last axes fastest.  An image's grid is stretched over 64 x 64 (its positions
    are fractions), a video's counts on from a far frame, a text's starts again with every sequence."""
    L, A = c["L"], c["axes"]
    t = torch.arange(L, device="cuda")
    if A == 1:
        p = (t % max(1, (L * 2) // 3))[None].to(torch.int32)
    elif A == 2:
        side = max(1, math.isqrt(L))
        p = torch.stack((t // side, t % side)).float() * (64.0 / side)
    else:
        side = max(1, math.isqrt(max(1, L // 8)))
        far = 100000 + int(torch.randint(0, 1000, (1,), generator=gen, device="cuda"))
        axes = [t // (side * side) + far, (t // side) % side, t % side, (t * 7) % 31]
        p = torch.stack(axes[:A]).to(torch.int64)
    if c["own_positions"]:
        p = p[None] + torch.arange(c["B"], device="cuda")[:, None, None].to(p.dtype)
    return p


def _freqs(c, gen):
    """[axes, rot / 2] radians per unit of position: each axis its own columns, or all of them in every column (mixed)."""
    half, A = c["rot"] // 2, c["axes"]
    if c["mixed"]:
        f = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        return f * torch.rand((A, half), generator=gen, device="cuda", dtype=torch.float64)
    f = torch.zeros((A, half), dtype=torch.float64, device="cuda")
    cuts = [half * a // A for a in range(A + 1)]
    for a, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
        f[a, lo:hi] = 10000.0 ** (-torch.arange(hi - lo, device="cuda", dtype=torch.float64) / max(1, hi - lo))
    return f


def prepare(case, seed):
    c, dev = case, "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=c)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16)  # noqa: E731
    if c["kind"] == "attn":
        nq, nk = _lengths(c)
        H, Hkv, d = c["H"], c["Hkv"], c["d"]
        T = max(1, sum(nq)) + (5 if c["ragged"] else 0)         # rows of padding behind the last sequence
        s["offsets"], s["k_offsets"] = _i32(_offsets(nq)), None
        if c["keys"]:                                           # queries and keys from projections of their own
            s["q"] = normal(1, T, H, d).transpose(1, 2)
            kv = normal(1, max(1, sum(nk)), 2 * Hkv, d).transpose(1, 2)
            s["k"], s["v"], s["k_offsets"] = kv[:, :Hkv], kv[:, Hkv:], _i32(_offsets(nk))
        else:                                                   # views on one fused projection
            x = normal(1, T, H + 2 * Hkv, d).transpose(1, 2)
            s["q"], s["k"], s["v"] = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
        if c["train"]:
            s["go"] = normal(1, T, H, d).transpose(1, 2)
    elif c["kind"] == "rope":
        H, Hkv, d, B, L = c["H"], c["Hkv"], c["d"], c["B"], c["L"]
        x = normal(B, L, H + 2 * Hkv, d).mul_(0.5).transpose(1, 2)
        s["q"], s["k"], s["v"] = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
        s["positions"], s["freqs"] = _positions(c, gen), _freqs(c, gen)
        s["q_weight"], s["k_weight"] = _weight(c, H, gen), _weight(c, Hkv, gen)
        if c["how"] == "train":
            s["gq"], s["gk"] = normal(B, H, L, d), normal(B, Hkv, L, d)
        if c["how"] == "append":
            starts = [(7 * b) % 50 for b in range(B)]
            per = -(-(max(starts) + L) // c["page"])
            P = B * per + 3
            s.update(_pages(c, (P, Hkv, c["page"], d), gen))
            s["table"] = torch.randperm(P, generator=gen, device=dev)[: B * per].to(torch.int32).view(B, per)
            s["start"], s["lengths"] = _i32(starts), _i32([x + L for x in starts])
    elif c["kind"] == "fork":
        S, n, page = c["S"], c["n"], c["page"]
        lengths = _fork_lengths(c)
        used = [-(-x // page) for x in lengths]
        P, B, width = _fork_pages(c), S * (1 + n), max(used) + c["grow"] + 1
        s.update(_pages(c, (P, c["Hkv"], page, c["d"]), gen))
        s["table"] = torch.full((B, width), -1, dtype=torch.int32, device=dev)
        s["refs"] = torch.zeros(P, dtype=torch.int32, device=dev)
        order, at = torch.randperm(P, generator=gen, device=dev).to(torch.int32), 0
        for b, m in enumerate(used):
            s["table"][b, :m] = order[at:at + m]
            at += m
        s["refs"][order[:at].long()] = 1
        # rows 0 .. S-1 are the prompts, row S + s * n + i the i-th sample of prompt s
        source = [b for b in range(S) for _ in range(n)]
        s["source"], s["target"] = _i32(source), _i32(range(S, B))
        s["lengths"] = _i32(lengths + [lengths[b] for b in source])
        s["stay"] = _i32(used + [0] * (S * n))                  # pages that rows keep: the prompts all, the samples of the step before none
        full = [0] * S + [-(-lengths[b] // page) for b in source]
        s["first"], s["last"] = _i32(full), _i32([0] * S + [x + c["grow"] for x in full[S:]])
        s["tail"] = _i32([lengths[b] // page * page for b in source])
    else:
        B, page, n = c["B"], c["page"], c["keep"]
        per, out = -(-c["Lmax"] // page), -(-n // page)
        P = B * (per + out) + 3
        s.update(_pages(c, (P, c["Hkv"], page, c["d"]), gen))
        order = torch.randperm(P, generator=gen, device=dev).to(torch.int32)
        s["table"], s["out_table"] = order[: B * per].view(B, per), order[B * per: B * (per + out)].view(B, out)
        score = torch.rand((B, c["Hkv"], c["Lmax"]), generator=gen, device=dev)
        s["keep"] = torch.sort(torch.topk(score, n, dim=-1).indices, dim=-1).values
        s["counts"] = _i32(_kept(c))
    return s


# ---- plain forms: 32 bits, rounded once ----

def _plain_hidden(n, m, lo, hi, causal, dev):
    """True where row lo .. hi-1 of n queries does not see a key of m."""
    if not causal:
        return None
    i, j = torch.arange(lo, hi, device=dev), torch.arange(m, device=dev)
    return j[None, :] > (i + m - n)[:, None]


def _plain_rows(total, width):
    """Rows at a time, so that scores of `width` columns stay below 1.5 GB."""
    return max(1, min(total, int(4e8) // max(1, width)))


def _plain_sequence(q, k, v, scale, causal, go=None):
    """q [H,n,d], k and v [Hkv,m,d] fp32 -> o, M, L; with go also dq, dk, dv."""
    H, n, d = q.shape
    Hkv, m = k.shape[0], k.shape[1]
    G = H // Hkv
    o, M, L = torch.zeros_like(q), torch.full_like(q[..., :1], -math.inf), torch.ones_like(q[..., :1])
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    if m == 0 or n == 0:
        return (o, M, L) if go is None else (o, dq, dk, dv)
    for h in range(Hkv):
        heads = slice(h * G, (h + 1) * G)
        step = _plain_rows(n, m * G)
        for lo in range(0, n, step):
            hi = min(n, lo + step)
            x = torch.matmul(q[heads, lo:hi], k[h].T).mul_(scale * LOG2E)
            hidden = _plain_hidden(n, m, lo, hi, causal, q.device)
            if hidden is not None:
                x.masked_fill_(hidden, -math.inf)
            top = x.amax(-1, keepdim=True)
            x.sub_(torch.where(top == -math.inf, 0.0, top)).exp2_()
            total = x.sum(-1, keepdim=True)
            total = torch.where(total == 0, 1.0, total)
            x.div_(total)
            out = torch.matmul(x, v[h])
            o[heads, lo:hi], M[heads, lo:hi], L[heads, lo:hi] = out, top, total
            if go is not None:
                g = go[heads, lo:hi]
                dv[h] += torch.matmul(x.flatten(0, 1).T, g.flatten(0, 1))
                dx = torch.matmul(g, v[h].T).sub_((g * out).sum(-1, keepdim=True)).mul_(x).mul_(scale)
                dq[heads, lo:hi] = torch.matmul(dx, k[h])
                dk[h] += torch.matmul(dx.flatten(0, 1).T, q[heads, lo:hi].flatten(0, 1))
    return (o, M, L) if go is None else (o, dq, dk, dv)


def _plain_attn(s):
    c = s["case"]
    nq, nk = _lengths(c)
    aq, ak = _offsets(nq), _offsets(nk)
    bf = torch.bfloat16
    q, k, v = s["q"], s["k"], s["v"]
    o, M, L = torch.zeros_like(q), torch.full(q.shape[:3] + (1,), -math.inf, device=q.device), torch.ones(q.shape[:3] + (1,), device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(c["B"]):
        rows, cols = slice(aq[b], aq[b + 1]), slice(ak[b], ak[b + 1])
        go = s["go"][0, :, rows].float() if c["train"] else None
        r = _plain_sequence(q[0, :, rows].float(), k[0, :, cols].float(), v[0, :, cols].float(), 1.0 / math.sqrt(c["d"]), c["causal"], go)
        o[0, :, rows] = r[0].to(bf)
        if c["train"]:
            dq[0, :, rows], dk[0, :, cols], dv[0, :, cols] = r[1].to(bf), r[2].to(bf), r[3].to(bf)
        else:
            M[0, :, rows], L[0, :, rows] = r[1], r[2]
    return (o, dq, dk, dv) if c["train"] else (o, M, L)


def _plain_angles(s):
    """cos and sin [1 or B, 1, L, rot/2] in 32 bits of angles in 64."""
    p, f = s["positions"].double(), s["freqs"].double()
    angle = (p[..., None] * f[:, None, :]).sum(-3)
    angle = angle[None, None] if angle.dim() == 2 else angle[:, None]
    return angle.cos().float(), angle.sin().float()


def _plain_turn(x, cos, sin, interleaved):
    half = cos.shape[-1]
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, rest), -1)


def _plain_norm(x, w, norm):
    x = x.float()
    if norm == "l2":
        x = x / x.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
    elif norm == "rms":
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    return x if w is None else x * (w if w.dim() == 1 else w[:, None, :])


def _two_to(e):
    """2^e of whole e in -126 .. 127, exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _plain_codes(x):
    """e4m3 codes of fp32 rows and the byte of their power of two: the smallest 2^e with max|x| <= 448 * 2^e."""
    top = x.abs().amax(-1)
    m, ex = torch.frexp(top)
    e = torch.where(m <= 0.875, ex - 9, ex - 8).clamp(-126, 127)
    codes = (x * _two_to(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).to(torch.uint8)


def _plain_place(table, positions, page):
    """Page and slot of positions [B, n]."""
    return torch.gather(table.long(), 1, positions // page), positions % page


def _plain_write(s, name, x, positions):
    at, slot = _plain_place(s["table"], positions, s["case"]["page"])
    x, pages, exps = x.float().transpose(1, 2), s[name + "_pages"], s[name + "_exp"]
    if exps is None:
        pages[at, :, slot] = x.to(torch.bfloat16)
    else:
        codes, e = _plain_codes(x)
        pages.view(torch.uint8)[at, :, slot] = codes
        exps[at, :, slot] = e


def _plain_read(s, name, table, positions, there):
    """Tokens at positions [B, n] as bf16 [B,Hkv,n,d], zeros where not ``there``."""
    at, slot = _plain_place(table, positions.clamp_max(table.shape[1] * s["case"]["page"] - 1), s["case"]["page"])
    there, at = there & (at >= 0), at.clamp_min(0)
    pages, exps = s[name + "_pages"], s[name + "_exp"]
    if exps is None:
        x = pages[at, :, slot].float()
    else:
        x = pages.view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn).float() * _two_to(exps[at, :, slot].int() - 127)[..., None]
    return x.masked_fill(~there[:, :, None, None], 0.0).to(torch.bfloat16).transpose(1, 2).contiguous()


def _plain_rope(s):
    c = s["case"]
    bf = torch.bfloat16
    norm = None if c["norm"] == "none" else c["norm"]
    cos, sin = _plain_angles(s)
    if c["how"] != "train":
        q = _plain_turn(_plain_norm(s["q"], s["q_weight"], norm), cos, sin, c["interleaved"]).to(bf)
        k = _plain_turn(_plain_norm(s["k"], s["k_weight"], norm), cos, sin, c["interleaved"])
        if c["how"] == "step":
            return q, k.to(bf)
        positions = s["start"].long()[:, None] + torch.arange(c["L"], device=k.device)
        _plain_write(s, "k", k, positions)
        _plain_write(s, "v", s["v"], positions)
        there = torch.ones_like(positions, dtype=torch.bool)
        return q, _plain_read(s, "k", s["table"], positions, there), _plain_read(s, "v", s["table"], positions, there)
    leaves = [None if s[n] is None else s[n].detach().requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
    q = _plain_turn(_plain_norm(leaves[0], leaves[2], norm), cos, sin, c["interleaved"]).to(bf)
    k = _plain_turn(_plain_norm(leaves[1], leaves[3], norm), cos, sin, c["interleaved"]).to(bf)
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), [x for x in leaves if x is not None], (s["gq"], s["gk"]))


def _plain_fork(s):
    c, table, refs = s["case"], s["table"], s["refs"]
    page, width = c["page"], s["table"].shape[1]
    entry = torch.arange(width, device=table.device)

    def count(pages, one):
        refs.index_add_(0, pages.long(), torch.full_like(pages, one))

    # drop what the samples had
    gone = (entry[None, :] >= s["stay"][:, None]) & (table >= 0)
    count(table[gone], -1)
    table.masked_fill_(entry[None, :] >= s["stay"][:, None], -1)
    # share whole pages, copy the started one
    n = s["lengths"][s["source"].long()]
    whole, rest = n // page, n % page
    rows = torch.where(entry[None, :] < whole[:, None], table[s["source"].long()], -1)
    free = torch.nonzero(refs == 0).flatten().int()
    started = torch.nonzero(rest > 0).flatten()
    fresh = free[: started.numel()]
    count(rows[rows >= 0], 1)
    rows[started, whole[started].long()] = fresh
    refs[fresh.long()] = 1
    table[s["target"].long()] = rows
    old = table[s["source"].long()[started], whole[started].long()].long()
    live = torch.arange(page, device=table.device)[None, :] < rest[started][:, None]
    for name in ("k", "v"):
        for pool in (s[name + "_pages"], s[name + "_exp"]):
            if pool is not None:
                raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
                keep = live[:, None, :, None] if raw.dim() == 4 else live[:, None, :]
                raw[fresh.long()] = torch.where(keep, raw[old], raw[fresh.long()])
    # open the next pages
    free = torch.nonzero(refs == 0).flatten().int()
    opened = (entry[None, :] >= s["first"][:, None]) & (entry[None, :] < s["last"][:, None])
    fresh = free[: int(c["S"] * c["n"] * c["grow"])]
    table[opened] = fresh
    refs[fresh.long()] = 1
    if c["cache"] == "bf16":
        return table, refs, s["k_pages"], s["v_pages"]
    at = s["tail"].long()[:, None] + torch.arange(page, device=table.device)
    there = at < s["lengths"][c["S"]:].long()[:, None]
    return table, refs, _plain_read(s, "k", table[c["S"]:], at, there), _plain_read(s, "v", table[c["S"]:], at, there)


def _plain_compact(s):
    c = s["case"]
    B, Hkv, n = s["keep"].shape
    page, dev = c["page"], s["keep"].device
    head = torch.arange(Hkv, device=dev)[None, :, None]
    i = torch.arange(n, device=dev)
    from_page = torch.gather(s["table"].long()[:, None].expand(B, Hkv, -1), 2, s["keep"] // page)
    to_page = s["out_table"].long()[:, i // page][:, None].expand(B, Hkv, n)
    live = (i[None, :] < s["counts"][:, None])[:, None].expand(B, Hkv, n)
    to = (to_page[live], head.expand(B, Hkv, n)[live], (i % page).expand(B, Hkv, n)[live])
    frm = (from_page[live], to[1], (s["keep"] % page)[live])
    for name in ("k", "v"):
        for pool in (s[name + "_pages"], s[name + "_exp"]):
            if pool is not None:
                raw = pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool
                raw[to] = raw[frm]
    if c["cache"] == "bf16":
        return s["k_pages"], s["v_pages"]
    at = i[None, :].expand(B, n)
    there = at < s["counts"][:, None]
    return _plain_read(s, "k", s["out_table"], at, there), _plain_read(s, "v", s["out_table"], at, there)


def _own(s):
    from lvar_amd import kv_cache_ops as kv
    c = s["case"]
    if c["kind"] == "attn":
        from lvar_amd.packed_ops import packed_attn
        if not c["train"]:
            o, (M, L) = packed_attn(s["q"], s["k"], s["v"], s["offsets"], k_offsets=s["k_offsets"], causal=c["causal"])
            return o, M, L
        leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v")]
        o, _ = packed_attn(*leaves, s["offsets"], k_offsets=s["k_offsets"], causal=c["causal"])
        return (o.detach(),) + torch.autograd.grad(o, leaves, s["go"])
    if c["kind"] == "rope":
        how = dict(positions=s["positions"], freqs=s["freqs"], norm=None if c["norm"] == "none" else c["norm"], interleaved=c["interleaved"])
        if c["how"] == "train":
            leaves = [None if s[n] is None else s[n].detach().requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
            q, k = kv.qk_norm_rope(leaves[0], leaves[1], q_weight=leaves[2], k_weight=leaves[3], **how)
            return (q.detach(), k.detach()) + torch.autograd.grad((q, k), [x for x in leaves if x is not None], (s["gq"], s["gk"]))
        how.update(q_weight=s["q_weight"], k_weight=s["k_weight"])
        if c["how"] == "step":
            return kv.qk_norm_rope(s["q"], s["k"], **how)
        cache = kv.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
        q = kv.qk_norm_rope_append(cache, s["q"], s["k"], s["v"], s["table"], s["start"], **how)
        return (q,) + kv.kv_cache_read(cache, s["table"], s["lengths"], max_len=c["L"], start=s["start"])
    cache = kv.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
    if c["kind"] == "fork":
        kv.kv_pages_free(s["refs"], s["table"], s["stay"])
        kv.kv_cache_fork(cache, s["refs"], s["table"], s["source"], s["target"], s["lengths"])
        kv.kv_pages_alloc(s["refs"], s["table"], s["first"], s["last"])
        if c["cache"] == "bf16":
            return s["table"], s["refs"], s["k_pages"], s["v_pages"]
        S = c["S"]
        return (s["table"], s["refs"]) + kv.kv_cache_read(cache, s["table"][S:], s["lengths"][S:], max_len=c["page"], start=s["tail"])
    kv.kv_cache_compact(cache, s["table"], s["keep"], s["out_table"], counts=s["counts"])
    if c["cache"] == "bf16":
        return s["k_pages"], s["v_pages"]
    return kv.kv_cache_read(cache, s["out_table"], s["counts"], max_len=c["keep"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "rope": _plain_rope, "fork": _plain_fork, "compact": _plain_compact}[state["case"]["kind"]](state)


def work(case):
    """Every input read once, every output written once."""
    c = case
    if c["kind"] == "attn":
        nq, nk = _lengths(c)
        rows, cols, pairs = c["H"] * sum(nq) * c["d"], 2 * c["Hkv"] * sum(nk) * c["d"], _pairs(c)
        # forward q, k, v -> o (and its statistics); with gradients also do -> dq, dk, dv
        stats = 0 if c["train"] else 8 * c["H"] * sum(nq)
        return {"bytes": (8 * rows + 4 * cols if c["train"] else 4 * rows + 2 * cols) + stats, "flops": (14 if c["train"] else 4) * c["H"] * c["d"] * pairs}
    if c["kind"] == "rope":
        B, Hkv, L, d = c["B"], c["Hkv"], c["L"], c["d"]
        n, places = B * (c["H"] + Hkv) * L * d, 4 * c["axes"] * L * (B if c["own_positions"] else 1)
        if c["how"] == "append":
            q, kv, row = B * c["H"] * L * d, B * Hkv * L, 2 * d if c["cache"] == "bf16" else d + 1
            # q, k, v in, q out, k and v into the cache, out of it, and out packed
            return {"bytes": 4 * q + 2 * kv * (2 * d + 2 * row + 2 * d) + places, "flops": 10 * (q + 2 * kv * d)}
        return {"bytes": (10 if c["how"] == "train" else 4) * n + places, "flops": (30 if c["how"] == "train" else 10) * n}
    row = 2 * c["d"] if c["cache"] == "bf16" else c["d"] + 1
    if c["kind"] == "fork":
        rest = sum(n % c["page"] for n in _fork_lengths(c)) * c["n"]
        used = [-(-n // c["page"]) for n in _fork_lengths(c)]
        rows = 4 * c["S"] * (1 + c["n"]) * (max(used) + c["grow"] + 1)
        back = 0 if c["cache"] == "bf16" else 2 * c["Hkv"] * (rest * row + 2 * c["d"] * c["S"] * c["n"] * c["page"])
        # started pages in and out, the table and the counts read and written
        return {"bytes": 4 * c["Hkv"] * rest * row + 2 * rows + 8 * _fork_pages(c) + back, "flops": 0}
    kept = sum(_kept(c)) * c["Hkv"]
    back = 0 if c["cache"] == "bf16" else 2 * (kept * row + 2 * c["d"] * c["B"] * c["Hkv"] * c["keep"])
    return {"bytes": 4 * kept * row + 8 * kept + back, "flops": 0}


# ---- the definitions in 64 bits, apart from the above ----

def _exact_attn(s):
    c = s["case"]
    nq, nk = _lengths(c)
    H, G, d, dev = c["H"], c["H"] // c["Hkv"], c["d"], "cuda"
    f64 = torch.float64
    T, Tk = s["q"].shape[2], s["k"].shape[2]
    o, M, L = torch.zeros((1, H, T, d), dtype=f64, device=dev), torch.full((1, H, T, 1), -math.inf, dtype=f64, device=dev), torch.ones((1, H, T, 1), dtype=f64, device=dev)
    dq, dk, dv = torch.zeros_like(o), torch.zeros((1, c["Hkv"], Tk, d), dtype=f64, device=dev), torch.zeros((1, c["Hkv"], Tk, d), dtype=f64, device=dev)
    r = 1.0 / math.sqrt(d)
    q0 = k0 = 0
    for n, m in zip(nq, nk):
        for h in range(H if n and m else 0):
            k, v = s["k"][0, h // G, k0:k0 + m].double(), s["v"][0, h // G, k0:k0 + m].double()
            for lo in range(0, n, 2048):
                hi = min(n, lo + 2048)
                see = min(m, max(0, m - n + hi)) if c["causal"] else m       # no row of these sees more
                at = slice(q0 + lo, q0 + hi)
                q = s["q"][0, h, at].double()
                z = (q @ k[:see].T) * r
                if c["causal"]:
                    last = torch.arange(lo, hi, device=dev) + (m - n)
                    z[torch.arange(see, device=dev)[None] > last[:, None]] = -math.inf
                some = torch.isfinite(z).any(-1) if see else torch.zeros(hi - lo, dtype=torch.bool, device=dev)
                if not bool(some.any()):
                    continue
                top = torch.where(some, z.amax(-1), 0.0)
                p = torch.exp(z - top[:, None])
                total = p.sum(-1)
                p = torch.where(some[:, None], p / total[:, None], 0.0)
                M[0, h, at, 0] = torch.where(some, top * LOG2E, -math.inf)
                L[0, h, at, 0] = torch.where(some, total, 1.0)
                o[0, h, at] = p @ v[:see]
                if c["train"]:
                    g = s["go"][0, h, at].double()
                    dv[0, h // G, k0:k0 + see] += p.T @ g
                    dz = p * (g @ v[:see].T - (g * o[0, h, at]).sum(-1, keepdim=True)) * r
                    dq[0, h, at] = dz @ k[:see]
                    dk[0, h // G, k0:k0 + see] += dz.T @ q
        q0, k0 = q0 + n, k0 + m
    return (o, dq, dk, dv) if c["train"] else (o, M, L)


def _exact_rotate(u, c, s, interleaved):
    """Rotation of the first columns of u by angles with cosines c and sines s."""
    half = c.shape[-1]
    y = u.clone()
    ia = torch.arange(half, device=u.device) * 2 if interleaved else torch.arange(half, device=u.device)
    ib = ia + 1 if interleaved else ia + half
    z = torch.complex(u[..., ia], u[..., ib]) * torch.complex(c, s)
    y[..., ia], y[..., ib] = z.real, z.imag
    return y


def _exact_cached(x, cache):
    """What a cache gives back of x."""
    if cache == "bf16":
        return x
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0))
    e = torch.where(torch.exp2(e) * 448.0 < top, e + 1, torch.where(torch.exp2(e - 1) * 448.0 >= top, e - 1, e))
    e = torch.where(top > 0, e, 0.0).clamp_min(-126)
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _exact_rope(s):
    c = s["case"]
    p, f = s["positions"].double(), s["freqs"].double()
    p = p[None] if p.dim() == 2 else p
    angle = torch.einsum("bal,ai->bli", p, f)[:, None]
    cs, sn = torch.cos(angle), torch.sin(angle)
    outs, grads, wgrads = [], [], []
    for n in ("q", "k"):
        x, w = s[n].double(), s[n + "_weight"]
        wide = None if w is None else (w.double().view(1, -1) if w.dim() == 1 else w.double()).expand(x.shape[1], c["d"])[:, None, :]
        ss = (x * x).sum(-1, keepdim=True)
        r = torch.ones_like(ss) if c["norm"] == "none" else 1.0 / torch.maximum(torch.sqrt(ss), torch.full_like(ss, 1e-12)) if c["norm"] == "l2" \
            else 1.0 / torch.sqrt(ss / c["d"] + 1e-6)
        u = x * r
        outs.append(_exact_rotate(u if wide is None else u * wide, cs, sn, c["interleaved"]))
        if c["how"] == "train":
            gu = _exact_rotate(s["g" + n].double(), cs, -sn, c["interleaved"])
            gn = gu if wide is None else gu * wide
            dot = (gn * u).sum(-1, keepdim=True)
            grads.append(r * (gn - u * (dot if c["norm"] == "l2" else dot / c["d"] if c["norm"] == "rms" else 0.0)))
            if w is not None:
                dw = (gu * u).sum((0, 2))
                wgrads.append(dw.sum(0) if w.dim() == 1 else dw.sum(-1, keepdim=True) if w.shape[1] == 1 else dw)
    if c["how"] == "append":
        return outs[0], _exact_cached(outs[1], c["cache"]), _exact_cached(s["v"].double(), c["cache"])
    return tuple(outs + grads + wgrads)


def _exact_values(s, name):
    x = s[name + "_pages"].double()
    return x if s[name + "_exp"] is None else x * torch.exp2(s[name + "_exp"].double() - 127.0)[..., None]


def _exact_fork(s):
    """Entry by entry, with lists."""
    c, page = s["case"], s["case"]["page"]
    S, n = c["S"], c["n"]
    table, refs, lengths = s["table"].tolist(), s["refs"].tolist(), _fork_lengths(c)
    free = [p for p, r in enumerate(refs) if r == 0]
    copies = []
    for i in range(S * n):
        b, to = i // n, S + i
        whole, rest = lengths[b] // page, lengths[b] % page
        for e in range(whole):
            table[to][e] = table[b][e]
            refs[table[b][e]] += 1
        if rest:
            table[to][whole] = free.pop(0)
            refs[table[to][whole]] = 1
            copies.append((table[b][whole], table[to][whole], rest, i))
    for i in range(S * n):
        first = -(-lengths[i // n] // page)
        for e in range(first, first + c["grow"]):
            table[S + i][e] = free.pop(0)
            refs[table[S + i][e]] = 1
    outs = []
    for name in ("k", "v"):
        x = _exact_values(s, name)
        y = x if c["cache"] == "bf16" else torch.zeros((S * n, c["Hkv"], page, c["d"]), dtype=torch.float64, device="cuda")
        for frm, to, rest, i in copies:
            y[to if c["cache"] == "bf16" else i, :, :rest] = x[frm, :, :rest]
        outs.append(y)
    return (_i32(table), _i32(refs)) + tuple(outs)


def _exact_compact(s):
    c, page = s["case"], s["case"]["page"]
    outs = []
    for name in ("k", "v"):
        x = _exact_values(s, name)
        packed = torch.zeros((c["B"], c["Hkv"], c["keep"], c["d"]), dtype=torch.float64, device="cuda")
        for b, n in enumerate(_kept(c)):
            line = x[s["table"][b].long()].transpose(0, 1).flatten(1, 2)        # [Hkv, tokens, d]
            for h in range(c["Hkv"]):
                packed[b, h, :n] = line[h].index_select(0, s["keep"][b, h, :n])
        if c["cache"] == "bf16":
            for b, n in enumerate(_kept(c)):
                for e in range(-(-n // page)):
                    rows = packed[b, :, e * page:min(n, (e + 1) * page)]
                    x[int(s["out_table"][b, e]), :, :rows.shape[1]] = rows
            packed = x
        outs.append(packed)
    return tuple(outs)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "rope": _exact_rope, "fork": _exact_fork, "compact": _exact_compact}[case["kind"]](s)
