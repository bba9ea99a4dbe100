"""The operators around a growing key/value cache, as cases that can be timed: norms of queries and keys per head with the
position rotation in the same pass (and their gradients), writing new keys and values into a paged cache and reading them
back, and the attention of the newest tokens over such a cache.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, with ``own``
set, through the entry points of ``lvar_amd.kv_cache_ops``.  Sizes are those of the Infinity-2B schedule (2 x 16 heads of
128, 13 scales up to 64 x 64, 10521 tokens in all) and of VAR-d16 (heads of 64, 680 tokens) where a name says so, and
generic serving sizes (32 query heads over 8 key/value heads) elsewhere; drawn cases spread over the same ranges.

Lengths of ragged batches follow a fixed formula of the case, so that ``work`` can count them; everything else comes from
the seed.
"""
import math

import torch

own = False

LOG2E = 1.4426950408889634
E4M3_MAX = 448.0


def listed():
    return [
        # scale 4 of an image: 16 new tokens, normalised and rotated straight from the fused projection; launch and latency
        dict(name="norm_rope_scale_4", kind="norm_rope", train=False, B=2, H=16, Hkv=16, L=16, d=128, rot=128, norm="l2", weight="head", interleaved=True),
        # the last scale of an image
        dict(name="norm_rope_scale_64", kind="norm_rope", train=False, B=2, H=16, Hkv=16, L=4096, d=128, rot=128, norm="l2", weight="head", interleaved=True),
        # a training step over the whole schedule of an image: outputs, and gradients of q, k and the per-head factors
        dict(name="norm_rope_train_10521", kind="norm_rope", train=True, B=4, H=16, Hkv=16, L=10521, d=128, rot=128, norm="l2", weight="head", interleaved=True),
        # grouped heads with learned columns, half of them rotated, odd length
        dict(name="norm_rope_train_grouped", kind="norm_rope", train=True, B=2, H=32, Hkv=8, L=2047, d=128, rot=64, norm="rms", weight="dim", interleaved=False),
        # one token of each of 64 sequences being served
        dict(name="append_decode", kind="append", fused=True, B=64, H=32, Hkv=8, L=1, d=128, rot=128, norm="rms", weight="dim", interleaved=False, start=1000, page=16, cache="bf16"),
        # the last scale of an image into an 8-bit cache
        dict(name="append_scale_64_e4m3", kind="append", fused=True, B=2, H=16, Hkv=16, L=4096, d=128, rot=128, norm="l2", weight="head", interleaved=True, start=6425, page=64, cache="e4m3"),
        # keys and values that are ready, an odd number of them at odd places, heads of 64
        dict(name="append_ready_e4m3", kind="append", fused=False, B=8, H=16, Hkv=16, L=999, d=64, start=680, page=32, cache="e4m3"),
        # the whole cache of an image, for the operators that take packed keys and values
        dict(name="read_10521_e4m3", kind="read", B=2, Hkv=16, Lmax=10521, d=128, page=64, cache="e4m3", ragged=False),
        # scale 4 of an image over its 21 tokens: the smallest attention
        dict(name="attn_scale_4", kind="attn", B=2, H=16, Hkv=16, Lq=16, Lmax=21, d=128, page=64, cache="bf16", causal=False, ragged=False),
        # one new token of each of 32 sequences of very different lengths
        dict(name="attn_decode_ragged", kind="attn", B=32, H=32, Hkv=8, Lq=1, Lmax=32768, d=128, page=16, cache="bf16", causal=True, ragged=True),
        # one new token of one long sequence, 8-bit cache
        dict(name="attn_decode_long_e4m3", kind="attn", B=1, H=32, Hkv=8, Lq=1, Lmax=131071, d=128, page=64, cache="e4m3", causal=True, ragged=False),
        # several new tokens at once (a small scale, or drafted tokens), padded batch
        dict(name="attn_chunk_ragged", kind="attn", B=8, H=32, Hkv=8, Lq=61, Lmax=4001, d=128, page=64, cache="bf16", causal=True, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most=40):
    Hkv = rng.choice((1, 2, 3, 4, 5, 8, 12, 16))
    return Hkv * rng.choice([g for g in (1, 1, 2, 3, 4, 7, 8) if g * Hkv <= most]), Hkv


def draw(rng):
    kind = rng.choice(("norm_rope", "norm_rope", "append", "append", "read", "attn", "attn", "attn"))
    most = work(listed()[9])["bytes"] if kind == "attn" else work(listed()[2])["bytes"] / 2
    while True:
        H, Hkv = _heads(rng)
        c = dict(kind=kind, B=_log_int(rng, 1, 64), Hkv=Hkv, d=rng.choice((64, 128, 128, 256)))
        if kind in ("norm_rope", "append"):
            c.update(H=H, norm=rng.choice(("l2", "rms")), weight=rng.choice(("none", "head", "dim", "full")), interleaved=rng.random() < 0.5)
            c["rot"] = c["d"] // rng.choice((1, 1, 2))
            c["L"] = _log_int(rng, 1, 10521)
        if kind == "norm_rope":
            c.update(train=rng.random() < 0.5, d=rng.choice((c["d"], 32, 16)))
            c["rot"] = min(c["rot"], c["d"])
        else:
            c.update(page=rng.choice((16, 32, 64, 128, 256)), cache=rng.choice(("bf16", "e4m3")))
        if kind == "append":
            c.update(fused=rng.random() < 0.6, start=_log_int(rng, 1, 8000))
        if kind == "read":
            c.update(Lmax=_log_int(rng, 1, 32768), ragged=rng.random() < 0.5)
        if kind == "attn":
            c.update(H=H, Lq=rng.choice((1, 1, 1, 4, _log_int(rng, 2, 256))), causal=rng.random() < 0.5, ragged=rng.random() < 0.5)
            c["Lmax"] = max(c["Lq"], _log_int(rng, 1, 131072))
        w = work(c)
        slots = c["B"] * Hkv * c["d"] * (c.get("Lmax", 0) + c.get("L", 0) + c.get("start", 0))
        if w["bytes"] <= most and w["flops"] <= 5e11 and slots <= 1.2e9:
            return c


# ---- what a case is made of ----

def _lengths(c):
    """Tokens of every sequence with the new ones, and how many of them are new (fixed by the case)."""
    B, Lmax, Lq = c["B"], c["Lmax"], c.get("Lq", 1)
    if not c["ragged"]:
        return [Lmax] * B, [Lq] * B
    new = [max(1, Lq - int(Lq * ((b * 0.381966) % 1.0))) for b in range(B)]
    return [max(n, int(Lmax * (1.0 - (b * 0.618034) % 1.0))) for b, n in enumerate(new)], new


def _starts(c):
    return [c["start"] + (7 * b) % 50 for b in range(c["B"])]


def _pages(c, tokens, gen, dev):
    """A pool with the pages of every sequence in random places, and the table that finds them."""
    per = -(-tokens // c["page"])
    P = c["B"] * per + 3
    table = torch.randperm(P, generator=gen, device=dev)[: c["B"] * per].to(torch.int32).view(c["B"], per)
    shape = (P, c["Hkv"], c["page"], c["d"])
    s = dict(table=table)
    for n in ("k", "v"):
        if c["cache"] == "bf16":
            s[n + "_pages"] = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16).mul_(0.5)
            s[n + "_exp"] = None
        else:
            s[n + "_pages"] = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16).mul_(64).to(torch.float8_e4m3fn)
            s[n + "_exp"] = torch.randint(118, 122, shape[:3], generator=gen, device=dev, dtype=torch.uint8)
    return s


def _weight(c, heads, gen, dev):
    if c["weight"] == "none":
        return None
    shape = {"head": (heads, 1), "dim": (c["d"],), "full": (heads, c["d"])}[c["weight"]]
    w = torch.randn(shape, generator=gen, device=dev)
    return torch.exp(1.4 + 0.3 * w) if c["norm"] == "l2" else 1.0 + 0.2 * w


def _projection(c, gen, dev, rows):
    """q, k and v as the views on one fused projection that a model has."""
    H, Hkv, L, d = c.get("H", c["Hkv"]), c["Hkv"], rows, c["d"]
    x = torch.randn((c["B"], L, H + 2 * Hkv, d), generator=gen, device=dev, dtype=torch.bfloat16).mul_(0.5).transpose(1, 2)
    return x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]


def prepare(case, seed):
    c, dev = case, "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = dict(case=c)
    if c["kind"] in ("norm_rope", "append"):
        s["q"], s["k"], s["v"] = _projection(c, gen, dev, c["L"])
        if c["kind"] == "norm_rope" or c["fused"]:
            rows = c["L"] + (max(_starts(c)) if c["kind"] == "append" else 0)
            freq = 10000.0 ** (-torch.arange(c["rot"] // 2, device=dev, dtype=torch.float64) * 2 / c["rot"])
            angle = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
            s["q_weight"], s["k_weight"] = _weight(c, c["H"], gen, dev), _weight(c, c["Hkv"], gen, dev)
    if c["kind"] == "norm_rope" and c["train"]:
        s["gq"] = torch.randn((c["B"], c["H"], c["L"], c["d"]), generator=gen, device=dev, dtype=torch.bfloat16)
        s["gk"] = torch.randn((c["B"], c["Hkv"], c["L"], c["d"]), generator=gen, device=dev, dtype=torch.bfloat16)
    if c["kind"] == "append":
        s.update(_pages(c, max(_starts(c)) + c["L"], gen, dev))
        s["start"], s["lengths"] = i32(_starts(c)), i32([x + c["L"] for x in _starts(c)])
    if c["kind"] in ("read", "attn"):
        s.update(_pages(c, c["Lmax"], gen, dev))
        lengths, new = _lengths(c)
        s["lengths"], s["new"] = i32(lengths), i32(new) if c["ragged"] else None
    if c["kind"] == "attn":
        q = torch.randn((c["B"], c["Lq"], c["H"], c["d"]), generator=gen, device=dev, dtype=torch.bfloat16)
        s["q"] = q.transpose(1, 2)
    return s


# ---- plain forms: 32 bits, rounded once ----

def _plain_norm_rope(x, w, cos, sin, norm, interleaved):
    """x [B,H,L,d] -> fp32, cos and sin [..., L, rot/2]"""
    x = x.float()
    if norm == "l2":
        x = x / x.square().sum(-1, keepdim=True).sqrt().clamp_min(1e-12)
    else:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    if w is not None:
        x = x * (w if w.dim() == 1 else w[:, None, :])
    half = cos.shape[-1]
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, rest), -1)


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


def _plain_place(s, positions):
    """Page and slot of positions [B, n]."""
    page = s["case"]["page"]
    return torch.gather(s["table"].long(), 1, positions // page), positions % page


def _plain_write(s, name, x, positions):
    """x [B,Hkv,n,d] into the pages"""
    at, slot = _plain_place(s, positions)
    x, pages, exps = x.float().transpose(1, 2), s[name + "_pages"], s[name + "_exp"]
    if exps is None:
        pages[at, :, slot] = x.to(torch.bfloat16)
    else:
        codes, e = _plain_codes(x)
        pages.view(torch.uint8)[at, :, slot] = codes
        exps[at, :, slot] = e


def _plain_read(s, name, positions):
    """[B,Hkv,n,d] fp32"""
    at, slot = _plain_place(s, positions)
    pages, exps = s[name + "_pages"], s[name + "_exp"]
    if exps is None:
        return pages[at, :, slot].transpose(1, 2).float()
    x = pages.view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn).float()
    return (x * _two_to(exps[at, :, slot].int() - 127)[..., None]).transpose(1, 2)


def _plain_whole(s, name):
    """Everything that the table names, [B,Hkv,n,d] fp32: whole pages at once."""
    pages, exps, table = s[name + "_pages"], s[name + "_exp"], s["table"].long()
    if exps is None:
        x = pages[table].float()
    else:
        x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * _two_to(exps[table].int() - 127)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attn(s):
    c, q = s["case"], s["q"].float()
    B, H, Lq, d = q.shape
    k, v = _plain_whole(s, "k"), _plain_whole(s, "v")
    G, n = H // c["Hkv"], k.shape[2]
    rows = q.reshape(B, c["Hkv"], G * Lq, d)
    x = torch.matmul(rows, k.transpose(-1, -2)).mul_(LOG2E / math.sqrt(d)).view(B, c["Hkv"], G, Lq, n)
    lengths = s["lengths"].long()
    new = torch.full_like(lengths, Lq) if s["new"] is None else s["new"].long()
    i, j = torch.arange(Lq, device=q.device), torch.arange(n, device=q.device)
    limit = lengths[:, None] - new[:, None] + i + 1 if c["causal"] else lengths[:, None].expand(B, Lq)
    limit = torch.where(i < new[:, None], limit, 0)
    x.masked_fill_((j >= limit[..., None])[:, None, None], -math.inf)
    M = x.amax(-1, keepdim=True)
    x.sub_(torch.where(M == -math.inf, 0.0, M)).exp2_()
    L = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, c["Hkv"], G * Lq, n), v).view(B, c["Hkv"], G, Lq, d) / torch.where(L == 0, 1.0, L)
    L = torch.where(L == 0, 1.0, L)
    return o.view(B, H, Lq, d).to(torch.bfloat16), M.view(B, H, Lq, 1), L.view(B, H, Lq, 1)


def _gradients(outs, leaves, grads):
    some = [x for x in leaves if x is not None]
    return torch.autograd.grad(outs, some, grads)


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if own:
        from lvar_amd import kv_cache_ops as kv
    if kind == "norm_rope":
        q, k, wq, wk = s["q"], s["k"], s["q_weight"], s["k_weight"]
        if c["train"]:
            q, k, wq, wk = (None if x is None else x.detach().requires_grad_() for x in (q, k, wq, wk))
        if own:
            oq, ok = kv.qk_norm_rope(q, k, s["cos"], s["sin"], q_weight=wq, k_weight=wk, norm=c["norm"], interleaved=c["interleaved"])
        else:
            oq = _plain_norm_rope(q, wq, s["cos"], s["sin"], c["norm"], c["interleaved"]).to(torch.bfloat16)
            ok = _plain_norm_rope(k, wk, s["cos"], s["sin"], c["norm"], c["interleaved"]).to(torch.bfloat16)
        if not c["train"]:
            return oq, ok
        return (oq.detach(), ok.detach()) + _gradients((oq, ok), (q, k, wq, wk), (s["gq"], s["gk"]))
    if kind == "append":
        if own:
            cache = kv.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
            if c["fused"]:
                q = kv.qk_norm_rope_append(cache, s["q"], s["k"], s["v"], s["table"], s["start"], s["cos"], s["sin"], q_weight=s["q_weight"],
                                           k_weight=s["k_weight"], norm=c["norm"], interleaved=c["interleaved"])
            else:
                q = None
                kv.kv_cache_append(cache, s["k"], s["v"], s["table"], s["start"])
            return (q,) + kv.kv_cache_read(cache, s["table"], s["lengths"], max_len=c["L"], start=s["start"])
        positions = s["start"].long()[:, None] + torch.arange(c["L"], device=s["k"].device)
        q, k = None, s["k"]
        if c["fused"]:
            cos, sin = s["cos"][positions][:, None], s["sin"][positions][:, None]
            q = _plain_norm_rope(s["q"], s["q_weight"], cos, sin, c["norm"], c["interleaved"]).to(torch.bfloat16)
            k = _plain_norm_rope(k, s["k_weight"], cos, sin, c["norm"], c["interleaved"])
        _plain_write(s, "k", k, positions)
        _plain_write(s, "v", s["v"], positions)
        return q, _plain_read(s, "k", positions).to(torch.bfloat16), _plain_read(s, "v", positions).to(torch.bfloat16)
    if kind == "read":
        if own:
            return kv.kv_cache_read(kv.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"]), s["table"], s["lengths"], max_len=c["Lmax"])
        behind = (torch.arange(c["Lmax"], device=s["table"].device) >= s["lengths"][:, None])[:, None, :, None]
        return tuple(_plain_whole(s, n)[:, :, : c["Lmax"]].masked_fill(behind, 0.0).to(torch.bfloat16) for n in ("k", "v"))
    if own:
        cache = kv.PagedKVCache(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"])
        o, (M, L) = kv.paged_attn(s["q"], cache, s["table"], s["lengths"], causal=c["causal"], counts=s["new"])
        return o, M, L
    return _plain_attn(s)


def work(case):
    """Every input read once, every output written once."""
    c = case
    B, Hkv, d, kind = c["B"], c["Hkv"], c["d"], c["kind"]
    row = 2 * d if c.get("cache", "bf16") == "bf16" else d + 1                 # bytes of a cached key or value
    if kind == "norm_rope":
        n, table = B * (c["H"] + Hkv) * c["L"] * d, 4 * c["L"] * c["rot"]
        # forward x -> y; with gradients also x, dL/dy -> dL/dx
        return {"bytes": (10 if c["train"] else 4) * n + table * (2 if c["train"] else 1), "flops": (30 if c["train"] else 10) * n}
    if kind == "append":
        n, rows = B * Hkv * c["L"] * d, B * Hkv * c["L"]
        q = B * c["H"] * c["L"] * d if c["fused"] else 0
        table = 4 * c["L"] * c["rot"] if c["fused"] else 0
        # q, k, v in, q out, k and v into the cache, out of it, and out packed
        return {"bytes": 4 * q + 2 * (2 * n + 2 * row * rows + 2 * n) + table, "flops": 10 * (q + 2 * n)}
    lengths, new = _lengths(c)
    if kind == "read":
        return {"bytes": 2 * Hkv * (row * sum(lengths) + 2 * d * B * c["Lmax"]), "flops": 2 * Hkv * d * sum(lengths)}
    pairs = sum(n * x - (n * (n - 1) // 2 if c["causal"] else 0) for x, n in zip(lengths, new))
    out = B * c["H"] * c["Lq"] * (4 * d + 8)
    return {"bytes": 2 * Hkv * row * sum(lengths) + out, "flops": 4 * c["H"] * d * pairs}


# ---- the definitions in 64 bits, apart from the above ----

def _exact_rotate(u, c, s, interleaved, back=False):
    """Rotation of the first columns of u by angles with cosines c and sines s; the other way round with ``back``."""
    half = c.shape[-1]
    y = u.clone()
    ia = torch.arange(half, device=u.device) * 2 if interleaved else torch.arange(half, device=u.device)
    ib = ia + 1 if interleaved else ia + half
    z = torch.complex(u[..., ia], u[..., ib]) * torch.complex(c, -s if back else s)
    y[..., ia], y[..., ib] = z.real, z.imag
    return y


def _exact_factor(x, norm):
    ss = (x * x).sum(-1, keepdim=True)
    return 1.0 / torch.maximum(torch.sqrt(ss), torch.full_like(ss, 1e-12)) if norm == "l2" else 1.0 / torch.sqrt(ss / x.shape[-1] + 1e-6)


def _exact_wide(w, heads, d):
    if w is None:
        return None
    w = w.double()
    return (w.view(1, -1) if w.dim() == 1 else w).expand(heads, d)[:, None, :]


def _exact_norm_rope(x, w, c, s, norm, interleaved):
    x = x.double()
    u = x * _exact_factor(x, norm)
    wide = _exact_wide(w, x.shape[1], x.shape[3])
    return _exact_rotate(u if wide is None else u * wide, c, s, interleaved)


def _exact_gradients(x, w, c, s, norm, interleaved, g):
    x = x.double()
    r = _exact_factor(x, norm)
    n, wide = x * r, _exact_wide(w, x.shape[1], x.shape[3])
    gu = _exact_rotate(g.double(), c, s, interleaved, back=True)
    gn = gu if wide is None else gu * wide
    dot = (gn * n).sum(-1, keepdim=True)
    dx = r * (gn - n * (dot if norm == "l2" else dot / x.shape[-1]))
    if w is None:
        return dx, None
    dw = (gu * n).sum((0, 2))
    return dx, dw.sum(0) if w.dim() == 1 else dw.sum(-1, keepdim=True) if w.shape[1] == 1 else dw


def _exact_cached(x, cache):
    """What a cache gives back of x."""
    if cache == "bf16":
        return x
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / E4M3_MAX))
    e = torch.where(torch.exp2(e) * E4M3_MAX < top, e + 1, torch.where(torch.exp2(e - 1) * E4M3_MAX >= top, e - 1, e))
    e = torch.where(top > 0, e, 0.0).clamp_min(-126)
    y = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _exact_sequence(s, name, b, n):
    """The first n keys or values of sequence b, [Hkv, n, d]."""
    c = s["case"]
    at = s["table"][b, : -(-n // c["page"])].long()
    x = s[name + "_pages"][at].double()
    if s[name + "_exp"] is not None:
        x = x * torch.exp2(s[name + "_exp"][at].double() - 127.0)[..., None]
    return x.permute(1, 0, 2, 3).reshape(c["Hkv"], -1, c["d"])[:, :n]


def exact(case, seed):
    s, c = prepare(case, seed), case
    kind, dev = c["kind"], "cuda"
    if kind == "norm_rope":
        cs, sn, how = s["cos"].double(), s["sin"].double(), (c["norm"], c["interleaved"])
        outs = [_exact_norm_rope(s[n], s[n + "_weight"], cs, sn, *how) for n in ("q", "k")]
        if not c["train"]:
            return tuple(outs)
        (dq, dwq), (dk, dwk) = (_exact_gradients(s[n], s[n + "_weight"], cs, sn, *how, s["g" + n]) for n in ("q", "k"))
        return tuple(outs) + tuple(x for x in (dq, dk, dwq, dwk) if x is not None)
    if kind == "append":
        q, k = None, s["k"].double()
        if c["fused"]:
            at = torch.stack([torch.arange(x, x + c["L"], device=dev) for x in _starts(c)])
            cs, sn = s["cos"].double()[at][:, None], s["sin"].double()[at][:, None]
            q = _exact_norm_rope(s["q"], s["q_weight"], cs, sn, c["norm"], c["interleaved"])
            k = _exact_norm_rope(s["k"], s["k_weight"], cs, sn, c["norm"], c["interleaved"])
        return q, _exact_cached(k, c["cache"]), _exact_cached(s["v"].double(), c["cache"])
    lengths, new = _lengths(c)
    if kind == "read":
        outs = []
        for name in ("k", "v"):
            y = torch.zeros((c["B"], c["Hkv"], c["Lmax"], c["d"]), dtype=torch.float64, device=dev)
            for b, n in enumerate(lengths):
                y[b, :, :n] = _exact_sequence(s, name, b, n)
            outs.append(y)
        return tuple(outs)
    B, H, Lq, d = s["q"].shape
    o = torch.zeros((B, H, Lq, d), dtype=torch.float64, device=dev)
    M = torch.full((B, H, Lq, 1), -math.inf, dtype=torch.float64, device=dev)
    L = torch.ones_like(M)
    for b, (n, m) in enumerate(zip(lengths, new)):
        k, v = _exact_sequence(s, "k", b, n), _exact_sequence(s, "v", b, n)
        last = torch.arange(n - m, n, device=dev) if c["causal"] else torch.full((m,), n - 1, device=dev)
        hidden = torch.arange(n, device=dev)[None, :] > last[:, None]
        for h in range(c["Hkv"]):
            heads = range(h * (H // c["Hkv"]), (h + 1) * (H // c["Hkv"]))
            for at in heads:
                x = (s["q"][b, at, :m].double() @ k[h].T) * (LOG2E / math.sqrt(d))
                x = x.masked_fill(hidden, -math.inf)
                M[b, at, :m] = x.amax(-1, keepdim=True)
                p = torch.exp2(x - M[b, at, :m])
                L[b, at, :m] = p.sum(-1, keepdim=True)
                o[b, at, :m] = (p @ v[h]) / L[b, at, :m]
    return o, M, L
