"""Plain CPU implementation in 64 bits of the attention over packed sequences and its gradients, with how far a kernel may be off that rounds
what the operator says it rounds: probabilities, their gradients, and results once each to bf16, sums in 32 bits."""
from __future__ import annotations

import math

import torch

BF16 = 2.0 ** -8          # half a step, relative
F32 = 2.0 ** -24


def visible(n: int, m: int, causal: bool):
    """bool [n,m]: which keys a row sees."""
    i, j = torch.arange(n)[:, None], torch.arange(m)[None]
    return (j < m - n + i + 1) if causal else torch.ones(n, m, dtype=torch.bool)


def sequence(q, k, v, scale: float, causal: bool, go=None):
    """One head of one sequence: q [n,d], k and v [m,d] fp64 -> dict of o, M, L (and dq, dk, dv) and of their tolerances (``t_...``)."""
    n, m, d = q.shape[0], k.shape[0], q.shape[1]
    see = visible(n, m, causal)
    some = see.any(-1, keepdim=True)
    c = scale * math.log2(math.e)
    x = (q @ k.T * c).masked_fill(~see, -math.inf)
    M = x.amax(-1, keepdim=True) if m else torch.full((n, 1), -math.inf, dtype=torch.float64)
    p = torch.exp2(x - torch.where(some, M, 0.0)).masked_fill(~see, 0.0)
    L = torch.where(some, p.sum(-1, keepdim=True), 1.0)
    p = p / L
    o = p @ v
    # scores: d products in 32 bits; the same again where the backward pass forms them, and 32-bit sums over the keys
    ex = (q.abs() @ k.abs().T * c).masked_fill(~see, 0.0).amax(-1, keepdim=True) * (d + 8) * F32 if m else torch.zeros(n, 1, dtype=torch.float64)
    rel = 2 * ex + (m + 16) * F32                         # of p, L and what is summed with them (ln 2 < 1)
    spread = p @ v.abs()
    r = dict(o=o, M=M, L=L, t_o=BF16 * o.abs() + (BF16 + rel) * spread + 1e-38, t_M=ex + F32 * torch.where(some, M.abs(), 0.0), t_L=rel * L)
    if go is None:
        return r
    delta = (go * o).sum(-1, keepdim=True)
    dp = go @ v.T
    ds = (p * (dp - delta)).masked_fill(~see, 0.0)
    # delta comes from o as it was rounded, dp from d products in 32 bits
    t_delta = (go.abs() * r["t_o"]).sum(-1, keepdim=True) + (d + 8) * F32 * (go.abs() * o.abs()).sum(-1, keepdim=True)
    t_ds = (BF16 + 3 * rel) * ds.abs() + p * (t_delta + (d + 8) * F32 * (go.abs() @ v.abs().T))
    t_p = (BF16 + 3 * rel) * p
    r.update(dq=scale * ds @ k, dk=scale * ds.T @ q, dv=p.T @ go)
    r["t_dq"] = BF16 * r["dq"].abs() + scale * t_ds @ k.abs() * (1 + (m + 8) * F32) + 1e-38
    r["t_dk"] = BF16 * r["dk"].abs() + scale * t_ds.T @ q.abs() + 1e-38       # (summed over query heads by the caller)
    r["t_dv"] = BF16 * r["dv"].abs() + t_p.T @ go.abs() + 1e-38
    sums = (n + 8) * F32
    r["t_dk"] += sums * scale * ds.abs().T @ q.abs()
    r["t_dv"] += sums * p.T @ go.abs()
    return r


def packed_attn(q, k, v, offsets, k_offsets=None, scale=None, causal: bool = True, go=None):
    """q [1,H,T,d], k and v [1,Hkv,Tk,d] -> dict of fp64 tensors as :func:`sequence`, whole."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    go = None if go is None else go.double().cpu()
    _, H, T, d = q.shape
    Hkv, Tk = k.shape[1:3]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    off = [int(x) for x in offsets]
    koff = off if k_offsets is None else [int(x) for x in k_offsets]
    z = lambda h, t, w=d: torch.zeros(1, h, t, w, dtype=torch.float64)  # noqa: E731
    out = dict(o=z(H, T), M=z(H, T, 1) - math.inf, L=z(H, T, 1) + 1, t_o=z(H, T), t_M=z(H, T, 1), t_L=z(H, T, 1))
    if go is not None:
        out.update(dq=z(H, T), t_dq=z(H, T), dk=z(Hkv, Tk), t_dk=z(Hkv, Tk), dv=z(Hkv, Tk), t_dv=z(Hkv, Tk))
    for b in range(len(off) - 1):
        rows, cols = slice(off[b], off[b + 1]), slice(koff[b], koff[b + 1])
        for h in range(H):
            g = h // (H // Hkv)
            r = sequence(q[0, h, rows], k[0, g, cols], v[0, g, cols], scale, causal, None if go is None else go[0, h, rows])
            for name, x in r.items():
                if name.endswith(("dk", "dv")):
                    out[name][0, g, cols] += x
                else:
                    out[name][0, h, rows] = x
    return out
