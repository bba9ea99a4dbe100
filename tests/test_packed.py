"""Attention over packed sequences without a GPU: the oracle against independent statements, refusals of the operator and of the C entry points."""
import ctypes as C
import math

import pytest
import torch

from oracle import packed_oracle as ref


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_against_softmax(causal):
    off, koff = [1, 5, 5, 12], [0, 6, 9, 13]
    q, k, v = normal(1, 4, 14, 16, seed=1), normal(1, 2, 15, 16, seed=2), normal(1, 2, 15, 16, seed=3)
    r = ref.packed_attn(q, k, v, off, koff, causal=causal)
    for b in range(3):
        n, m = off[b + 1] - off[b], koff[b + 1] - koff[b]
        for h in range(4):
            x = q[0, h, off[b]:off[b + 1]] @ k[0, h // 2, koff[b]:koff[b + 1]].T / 4
            for i in range(n):
                seen = max(0, min(m, m - n + i + 1)) if causal else m
                at = off[b] + i
                if seen == 0:
                    assert float(r["L"][0, h, at]) == 1 and float(r["M"][0, h, at]) == -math.inf and not bool(r["o"][0, h, at].any())
                    continue
                w = torch.softmax(x[i, :seen], 0)
                assert torch.allclose(w @ v[0, h // 2, koff[b]:koff[b] + seen], r["o"][0, h, at], atol=1e-12)
                lse = (r["M"][0, h, at] + torch.log2(r["L"][0, h, at])) * math.log(2)
                assert torch.allclose(torch.logsumexp(x[i, :seen], 0), lse, atol=1e-12)
    for at in (0, 12, 13):
        assert not bool(r["o"][0, :, at].any()) and bool((r["L"][0, :, at] == 1).all())


@pytest.mark.parametrize("causal", [True, False])
def test_gradient_formulas_against_differences(causal):
    off, koff = [0, 4, 4, 9], [0, 5, 7, 11]
    x = [normal(1, 4, 10, 8, seed=4), normal(1, 2, 11, 8, seed=5), normal(1, 2, 11, 8, seed=6)]
    go = normal(1, 4, 10, 8, seed=7)
    f = lambda *x: float((go * ref.packed_attn(*x, off, koff, scale=0.7, causal=causal)["o"]).sum())  # noqa: E731
    r = ref.packed_attn(*x, off, koff, scale=0.7, causal=causal, go=go)
    step = 1e-6                                # central differences in 64 bits: off by about step^2 and 2^-52 / step
    for i, name in enumerate(("dq", "dk", "dv")):
        for trial in range(3):
            t = normal(*x[i].shape, seed=20 + trial)
            up, down = list(x), list(x)
            up[i], down[i] = x[i] + step * t, x[i] - step * t
            assert abs((f(*up) - f(*down)) / (2 * step) - float((r[name] * t).sum())) < 1e-6 * max(1.0, float(r[name].norm()))


# ---- refusals ----

def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_operator_refuses_cpu_tensors_and_other_types():
    from lvar_amd.packed_ops import packed_attn
    off = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        packed_attn(bf(1, 2, 4, 64), bf(1, 2, 4, 64), bf(1, 2, 4, 64), off)
    with pytest.raises(TypeError, match="bfloat16"):
        packed_attn(bf(1, 2, 4, 64).float(), bf(1, 2, 4, 64), bf(1, 2, 4, 64), off)
    with pytest.raises(AssertionError):
        packed_attn(bf(2, 4, 64), bf(1, 2, 4, 64), bf(1, 2, 4, 64), off)


@pytest.fixture(scope="module")
def lib():
    import os
    from lvar_amd import _lib
    from lvar_amd.build import LIB_PATH, build_library
    if not os.path.exists(LIB_PATH):
        build_library()
    return _lib.load()


GOOD = dict(batch=2, tokens=8, k_tokens=8, H=4, kv_heads=2, head_dim=128, causal=1, scale=0.1)
BAD = [
    (dict(batch=0), -1), (dict(tokens=-1), -1), (dict(k_tokens=-1), -1), (dict(H=3), -1), (dict(kv_heads=0), -1), (dict(H=16386), -1),
    (dict(head_dim=96), -2), (dict(head_dim=32), -2), (dict(scale=0.0), -1), (dict(scale=math.nan), -1), (dict(scale=math.inf), -1), (dict(scale=-1.0), -1),
    (dict(scale=1e-40), -1), (dict(scale=2.9e38), -1),
    (dict(q=8), -1), (dict(k=0), -1), (dict(v=4), -1), (dict(o=2), -1), (dict(offsets=2), -1), (dict(k_offsets=0), -1), (dict(M=0), -1), (dict(L=2), -1),
    (dict(row=130), -1), (dict(head=4), -1), (dict(row=-128), -1), (dict(row=1 << 29), -1), (dict(tokens=1 << 23, row=1024), -1),
]


def call(lib, name, **change):
    """A call with made-up addresses: everything here is refused before anything is launched."""
    from lvar_amd._lib import LvarTensor
    a = dict(GOOD, q=4096, k=4096, v=4096, o=4096, go=4096, dq=4096, dk=4096, dv=4096, offsets=4096, k_offsets=4096, M=4096, L=4096, row=128, head=1024,
             workspace=4096, workspace_bytes=1 << 40)
    a.update(change)
    view = lambda n: LvarTensor(a[n] or None, 0, a["head"], a["row"])  # noqa: E731
    sizes = [a[n] for n in ("batch", "tokens", "k_tokens", "H", "kv_heads", "head_dim", "causal")]
    stats = [C.c_void_p(a[n] or None) for n in ("offsets", "k_offsets", "M", "L")]
    if name == "fwd":
        return lib.lvar_packed_attn_fwd(*map(view, ("q", "k", "v", "o")), *stats, C.c_void_p(a["workspace"] or None), a["workspace_bytes"], *sizes, a["scale"], None)
    return lib.lvar_packed_attn_bwd(*map(view, ("q", "k", "v", "o", "go")), *stats, *map(view, ("dq", "dk", "dv")), C.c_void_p(a["workspace"] or None),
                                    a["workspace_bytes"], *sizes, a["scale"], None)


@pytest.mark.parametrize("change,status", BAD)
@pytest.mark.parametrize("name", ["fwd", "bwd"])
def test_entry_points_refuse(lib, name, change, status):
    assert call(lib, name, **change) == status


@pytest.mark.parametrize("change", [dict(go=8), dict(dq=8), dict(dk=2), dict(dv=1), dict(workspace=0), dict(workspace=8), dict(workspace_bytes=255)])
def test_backward_entry_point_refuses(lib, change):
    assert call(lib, "bwd", **change) == -1


def test_workspace(lib):
    size = lambda batch=2, tokens=8, k_tokens=8, H=4, kv_heads=2, head_dim=128, causal=1: lib.lvar_packed_attn_bwd_workspace_bytes(  # noqa: E731
        batch, tokens, k_tokens, H, kv_heads, head_dim, causal)
    assert size() == 256                        # two statistics per row and head
    assert size(tokens=1 << 30, k_tokens=0, H=16384) == 8 << 44
    for bad in (dict(batch=0), dict(tokens=-1), dict(k_tokens=-1), dict(H=3), dict(kv_heads=0)):
        assert size(**bad) == -1
    assert size(head_dim=80) == -2
    fwd = lib.lvar_packed_attn_fwd_workspace_bytes
    assert fwd(2, 8, 8, 4, 2, 128, 1) == 0 and fwd(0, 8, 8, 4, 2, 128, 1) == -1 and fwd(2, 8, 8, 4, 2, 96, 1) == -2
