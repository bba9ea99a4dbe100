"""Attention over packed sequences where finite or infinite elements leave rows without any weight, and keys without any: the row counts as one that sees
no key (o = 0, M = -inf, L = 1) and adds nothing to the gradients, and neither does padding of a tile beside such elements."""
import math

import pytest
import torch

from oracle import packed_oracle as ref
from test_gpu_packed import i32, inputs, near, rand

pytestmark = pytest.mark.gpu

LEAST = -1e30          # scores below this (in units of a factor of two of the probability) have no weight at all

CASES = [
    # lengths, key lengths, H, Hkv, d, causal; rows in whole tiles of the kernels and not
    ([150, 40], None, 2, 1, 64, True),
    ([100, 70], [130, 30], 2, 2, 128, True),
    ([90], None, 2, 1, 256, True),
    ([64], [70], 2, 1, 64, False),
    ([65], [70], 2, 1, 64, False),
    ([64], [128], 2, 1, 128, False),
    ([60, 66], [70, 90], 1, 1, 128, False),
    ([32], [33], 1, 1, 256, False),
    ([33], [64], 1, 1, 256, False),
    # several workgroups share the query rows of a key tile, or the keys of a query tile
    ([600], [70], 1, 1, 64, True),
    ([1500], [70], 1, 1, 64, False),
    ([70, 3], [3300, 3000], 1, 1, 64, True),
    ([33, 8], [900, 2900], 1, 1, 128, False),
]


def by_rows(q, k, v, go, off, koff, causal):
    """Results and tolerances, row by row from the keys that have a weight; what has none adds 0 times its element."""
    q, k, v, go = (t.double() for t in (q, k, v, go))
    H, T, d = q.shape[1:]
    G, scale = H // k.shape[1], 1 / math.sqrt(d)
    out = {n: torch.zeros_like(q) for n in ("o", "dq", "t_o", "t_dq")}
    out.update({n: torch.zeros_like(k) for n in ("dk", "dv", "t_dk", "t_dv")})
    out.update(M=torch.full((1, H, T, 1), -math.inf, dtype=torch.float64), L=torch.ones(1, H, T, 1, dtype=torch.float64))
    out.update(t_M=torch.zeros(1, H, T, 1, dtype=torch.float64), t_L=torch.zeros(1, H, T, 1, dtype=torch.float64))
    for b in range(len(off) - 1):
        n, m = off[b + 1] - off[b], koff[b + 1] - koff[b]
        for h in range(H):
            for i in range(n):
                seen = max(0, min(m, m - n + i + 1)) if causal else m
                if seen == 0:
                    continue
                at, keys = (0, h, slice(off[b] + i, off[b] + i + 1)), (0, h // G, slice(koff[b], koff[b] + seen))
                some = (k[keys] @ q[at][0]) * scale * math.log2(math.e) > LEAST
                out["dq"][at] += (0 * k[keys][~some]).sum(0)
                out["dk"][keys] += torch.where(some[:, None], 0.0, 0 * q[at])
                if not bool(some.any()):
                    continue
                r = ref.sequence(q[at], k[keys][some], v[keys][some], scale, False, go[at])
                for name in ("o", "M", "L", "dq"):
                    out[name][at] = r[name] + (out[name][at] if name == "dq" else 0)
                    out["t_" + name][at] = r["t_" + name]
                where = some[:, None].expand(seen, d)
                for name in ("dk", "dv"):
                    x = torch.zeros(seen, d, dtype=torch.float64).masked_scatter(where, r[name])
                    out[name][keys] += x
                    out["t_" + name][keys] += torch.zeros(seen, d, dtype=torch.float64).masked_scatter(where, r["t_" + name]) + (n * G + 8) * ref.F32 * x.abs()
    return out


def check(q, k, v, off, koff, causal):
    from lvar_amd.packed_ops import packed_attn
    go = rand(*q.shape, seed=6)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    o, (M, L) = packed_attn(*leaves, i32(off), i32(koff), causal=causal)
    grads = torch.autograd.grad(o, leaves, go.cuda())
    r = by_rows(q, k, v, go, off, off if koff is None else koff, causal)
    for name, x in (("o", o), ("M", M), ("L", L), ("dq", grads[0]), ("dk", grads[1]), ("dv", grads[2])):
        fine = torch.isfinite(r[name])
        got = x.detach().cpu().double()
        if name == "M":
            assert bool((got[~fine] == -math.inf).all()), "M of a row without weight"
        else:
            assert bool((~torch.isfinite(got))[~fine].all()), name + " hides a value that is not finite"
        near(got.masked_fill(~fine, 0), r[name].masked_fill(~fine, 0), r["t_" + name].masked_fill(~fine, 0), name)
    return r


def made(case):
    lens, klens, H, Hkv, d, causal = case
    q, k, v, off, koff = (x if not torch.is_tensor(x) else x.contiguous() for x in inputs(lens, klens, H, Hkv, d, seed=d))
    return q, k, v, off, koff, causal


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("power", [60, 100])
def test_rows_of_finite_elements(case, power):
    """Every fifth row meets every key at -2^120 (a number) or -2^200 (which 32 bits do not hold)."""
    q, k, v, off, koff, causal = made(case)
    k[..., 0] = 2.0 ** power
    q[..., 0] = 0
    q[:, :, ::5, 0] = -2.0 ** power
    r = check(q, k, v, off, koff, causal)
    assert bool((r["M"][:, :, ::5] == -math.inf).all()) and bool(torch.isfinite(r["M"]).any())
    assert all(bool(torch.isfinite(r[n]).all()) for n in ("o", "dq", "dk", "dv"))


@pytest.mark.parametrize("case", CASES, ids=str)
def test_keys_with_an_infinite_element(case):
    """The first key of a sequence, and one behind it, at -infinity for all rows (causal: all that the first row sees)."""
    q, k, v, off, koff, causal = made(case)
    q[..., 0] = 1
    for first, end in zip((koff or off)[:-1], (koff or off)[1:]):
        k[:, :, first, 0] = -math.inf
        k[:, :, (first + end) // 2, 0] = -math.inf
    r = check(q, k, v, off, koff, causal)
    assert all(bool(torch.isfinite(r[n]).all()) for n in ("o", "dk", "dv")) and bool(torch.isfinite(r["dq"][..., 1:]).all())


@pytest.mark.parametrize("case", CASES, ids=str)
def test_rows_with_an_infinite_element(case):
    """Every seventh row at -infinity for all keys."""
    q, k, v, off, koff, causal = made(case)
    k[..., 0] = 1
    q[:, :, ::7, 0] = -math.inf
    r = check(q, k, v, off, koff, causal)
    assert all(bool(torch.isfinite(r[n]).all()) for n in ("o", "dq", "dv")) and bool(torch.isfinite(r["dk"][..., 1:]).all())
