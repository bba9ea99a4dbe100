"""Plain CPU implementations in 64 bits of the operators around the paged key/value cache: norm and rotation with their
gradients, the 8-bit row format, writing and reading pages, attention over them.  Loops over what the definitions loop over."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def rotate(u, cos, sin, interleaved: bool, back: bool = False):
    """u [...,d] with the first columns rotated by the angles of cos, sin [..., rot/2] (the other way round with ``back``)."""
    half = cos.shape[-1]
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    s = -sin if back else sin
    out = u.clone()
    out[..., a] = u[..., a] * cos - u[..., b] * s
    out[..., b] = u[..., a] * s + u[..., b] * cos
    return out


def table_rows(B: int, L: int, rows: int, positions=None, start=None):
    """Row of the tables of every token, int64 [B,L]."""
    at = torch.arange(L).expand(B, L) + (0 if start is None else start.long()[:, None])
    if positions is not None:
        at = positions.long().expand(B, L)
    return at.clamp(0, rows - 1)


def factor(x, norm, eps: float):
    ss = x.square().sum(-1, keepdim=True)
    if norm == "l2":
        return 1.0 / ss.sqrt().clamp_min(eps)
    if norm == "rms":
        return 1.0 / (ss / x.shape[-1] + eps).sqrt()
    return torch.ones_like(ss)


def wide(w, heads: int, d: int):
    """A weight as [heads,1,d]."""
    if w is None:
        return torch.ones(heads, 1, d, dtype=torch.float64)
    w = w.detach().double().cpu()
    return (w[None] if w.dim() == 1 else w).expand(heads, d)[:, None]


def norm_rope(x, w, cos, sin, at, norm, eps: float, interleaved: bool):
    """x [B,H,L,d] -> fp64; ``at`` [B,L] from :func:`table_rows`, cos None: no rotation."""
    x = x.double().cpu()
    u = x * factor(x, norm, eps) * wide(w, x.shape[1], x.shape[3])
    if cos is None:
        return u
    return rotate(u, cos.double().cpu()[at][:, None], sin.double().cpu()[at][:, None], interleaved)


def norm_rope_grads(x, w, cos, sin, at, norm, eps: float, interleaved: bool, g):
    """(dx, dw of w's shape) of sum(g * norm_rope(x)), by the formulas."""
    x, g = x.double().cpu(), g.double().cpu()
    gu = g if cos is None else rotate(g, cos.double().cpu()[at][:, None], sin.double().cpu()[at][:, None], interleaved, back=True)
    r = factor(x, norm, eps)
    n = x * r
    gn = gu * wide(w, x.shape[1], x.shape[3])
    dot = (gn * n).sum(-1, keepdim=True)
    if norm == "l2":
        flat = x.square().sum(-1, keepdim=True).sqrt() <= eps
        dx = r * torch.where(flat, gn, gn - n * dot)
    elif norm == "rms":
        dx = r * (gn - n * dot / x.shape[-1])
    else:
        dx = gn
    if w is None:
        return dx, None
    dw = (gu * n).sum((0, 2))                      # [H,d]
    if w.dim() == 1:
        return dx, dw.sum(0)
    for axis in (0, 1):
        if w.shape[axis] == 1:
            dw = dw.sum(axis, keepdim=True)
    return dx, dw


def e4m3_values():
    """The finite values of e4m3, by code 0 .. 126 (the sign bit apart)."""
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append(m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


def quantise(x):
    """Rows x [...,d] as (codes uint8 [...,d], bytes uint8 [...]): by search among the 127 values, ties to the even code."""
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), 0.0).amax(-1)
    byte = torch.full(top.shape, 1, dtype=torch.int64)
    for b in range(1, 255):
        byte = torch.where(top > E4M3_MAX * 2.0 ** (b - 127), b + 1, byte)
    y = torch.where(finite, x.abs(), 0.0) / torch.exp2(byte.double() - 127)[..., None]
    values = e4m3_values()
    hi = torch.searchsorted(values, y.contiguous()).clamp(0, 126)
    lo = (hi - 1).clamp_min(0)
    dl, dh = y - values[lo], values[hi] - y
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = torch.where(finite, code, 127) | (torch.signbit(x).long() << 7)
    return code.to(torch.uint8), byte.to(torch.uint8)


def dequantise(codes, byte):
    values = torch.cat([e4m3_values(), torch.tensor([math.nan], dtype=torch.float64)])
    c = codes.long()
    return values[c & 127] * torch.where(c >= 128, -1.0, 1.0) * torch.exp2(byte.double() - 127)[..., None]


def place(table, page_size: int, num_pages: int, b: int, pos: int):
    """(page, slot) of token ``pos`` of sequence b, or None."""
    if pos < 0 or pos // page_size >= table.shape[1]:
        return None
    page = int(table[b, pos // page_size])
    return (page, pos % page_size) if 0 <= page < num_pages else None


def append(pages, exps, table, x, start, counts=None):
    """Writes x [B,Hkv,L,d] (what is to be cached) into clones of the CPU tensors pages, exps; returns them."""
    pages, exps = pages.clone(), None if exps is None else exps.clone()
    B, _, L, _ = x.shape
    codes, byte = (None, None) if exps is None else quantise(x)
    for b in range(B):
        for i in range(L if counts is None else max(0, min(L, int(counts[b])))):
            at = place(table, pages.shape[2], pages.shape[0], b, int(start[b]) + i)
            if at is None:
                continue
            if exps is None:
                pages[at[0], :, at[1]] = x[b, :, i].to(torch.bfloat16)
            else:
                pages.view(torch.uint8)[at[0], :, at[1]] = codes[b, :, i]
                exps[at[0], :, at[1]] = byte[b, :, i]
    return pages, exps


def read(pages, exps, table, lengths, max_len: int, start=None):
    """([B,Hkv,max_len,d] fp64, bool [B,max_len]: the token is there)."""
    B, (P, Hkv, page, d) = table.shape[0], pages.shape
    out, there = torch.zeros(B, Hkv, max_len, d, dtype=torch.float64), torch.zeros(B, max_len, dtype=torch.bool)
    for b in range(B):
        for i in range(max_len):
            pos = i + (0 if start is None else int(start[b]))
            at = place(table, page, P, b, pos) if pos < int(lengths[b]) else None
            if at is None:
                continue
            there[b, i] = True
            x = pages[at[0], :, at[1]]
            out[b, :, i] = x.double() if exps is None else dequantise(x.view(torch.uint8), exps[at[0], :, at[1]])
    return out, there


def paged_attn(q, k, v, there, lengths, scale: float, causal: bool = False, counts=None):
    """(o, M, L, spread) fp64 over keys and values [B,Hkv,n,d] of which ``there`` [B,n] exist; spread = sum p |v| / sum p."""
    q = q.double().cpu()
    B, H, Lq, d = q.shape
    group, n = H // k.shape[1], k.shape[2]
    o, spread = torch.zeros(B, H, Lq, d, dtype=torch.float64), torch.zeros(B, H, Lq, d, dtype=torch.float64)
    M, L = torch.full((B, H, Lq, 1), -math.inf, dtype=torch.float64), torch.ones(B, H, Lq, 1, dtype=torch.float64)
    for b in range(B):
        new = Lq if counts is None else max(0, min(Lq, int(counts[b])))
        length = max(0, min(int(lengths[b]), n))
        for i in range(new):
            seen = there[b] & (torch.arange(n) < (length - new + i + 1 if causal else length))
            if not bool(seen.any()):
                continue
            for h in range(H):
                s = (k[b, h // group][seen] @ q[b, h, i]) * (scale * math.log2(math.e))
                M[b, h, i] = s.max()
                p = torch.exp2(s - s.max())
                L[b, h, i] = p.sum()
                o[b, h, i] = p @ v[b, h // group][seen] / p.sum()
                spread[b, h, i] = p @ v[b, h // group][seen].abs() / p.sum()
    return o, M, L, spread
