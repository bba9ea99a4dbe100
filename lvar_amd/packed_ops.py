"""Attention over packed sequences of different lengths (:func:`packed_attn`), causal or not, with grouped heads, differentiable: whole
prompts in one launch, a training step over packed texts, image tokens that attend to texts of different lengths.

Tensor contract as in :mod:`lvar_amd.sparse_attn_ops`, with a batch of one whose tokens are those of all sequences, one sequence behind the
other: bf16 on a HIP device, ``[1,H,T,d]`` with unit stride on d, outputs freshly allocated, work enqueued on the current torch stream of the
tensors' device; wrong shapes raise :class:`ShapeError`, wrong dtypes ``TypeError``, CPU tensors ``RuntimeError``.  There is no PyTorch or CPU
fallback.
"""
from __future__ import annotations

from typing import Tuple

import torch

from . import _lib
from .kv_cache_ops import _no_tangent, _rows, _rows_like
from .sparse_attn_ops import ShapeError, _native, _on_device, _pad_head_dim, _plain_scale, _ptr, _require, _scale_for, _stream

__all__ = ["packed_attn", "ShapeError"]

def _addressable(t) -> bool:
    """The rows of a head span less than 2^31 bytes, and two of them are at most 2^20 elements apart (a tile may end behind the last one)."""
    return t.shape[2] <= 1 or (t.stride(2) <= 1 << 20 and (t.shape[2] - 1) * t.stride(2) * 2 + t.shape[3] * 2 < 2 ** 31 - 1)


def _tokens(t, name: str):
    """``t`` as the kernels read it."""
    t = _rows(t, name)
    if not _addressable(t):
        t = t.clone(memory_format=torch.contiguous_format)
        _require(_addressable(t), lambda: f"{name} has {t.shape[2]} tokens: a head's rows must span less than 2^31 bytes")
    return t


def _like(t):
    """Memory for a result in t's own order of axes, or by heads where only that can be addressed."""
    r = _rows_like(t)
    return r if _addressable(r) else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _view(t) -> _lib.LvarTensor:
    """(axes of one element may have any stride)"""
    if t is None:
        return _lib.LvarTensor(None, 0, 0, 0)
    return _lib.LvarTensor(t.data_ptr(), 0, t.stride(1) if t.shape[1] > 1 else 0, t.stride(2) if t.shape[2] > 1 else t.shape[3])


def _offsets(t, name: str, device):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    _require(t.dim() == 1 and t.shape[0] > 1, lambda: f"{name} must be [sequences + 1], got {tuple(t.shape)}")
    _require(t.device == device, lambda: f"{name} must be on the device of the tensors")
    return t.contiguous()


def _launch(q, k, v, offsets, k_offsets, causal, scale):
    _, H, T, d = q.shape
    o = _like(q)
    M, L = torch.empty((2, 1, H, T, 1), dtype=torch.float32, device=q.device).unbind(0)
    if o.numel():
        lib, sizes = _lib.load(), (offsets.shape[0] - 1, T, k.shape[2], H, k.shape[1], d, 1 if causal else 0)
        with _on_device(q):
            nbytes = max(0, int(lib.lvar_packed_attn_fwd_workspace_bytes(*sizes)))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
            st = lib.lvar_packed_attn_fwd(_view(q), _view(k), _view(v), _view(o), offsets.data_ptr(), k_offsets.data_ptr(), M.data_ptr(), L.data_ptr(),
                                          _ptr(ws), nbytes, *sizes, scale, _stream(q))
        _lib.check(st, "lvar_packed_attn_fwd")
    return o, M, L


class _PackedAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, k_offsets, causal, scale):
        o, M, L = _launch(q, k, v, offsets, k_offsets, causal, scale)
        ctx.how = (causal, scale)
        ctx.save_for_backward(q, k, v, o, M, L, offsets, k_offsets)
        ctx.mark_non_differentiable(M, L)
        ctx.set_materialize_grads(False)
        return o, M, L

    @staticmethod
    def backward(ctx, go, *_):
        if torch.is_grad_enabled():
            raise RuntimeError("packed_attn can be differentiated once: its gradients have no graph (create_graph)")
        if go is None:
            return (None,) * 7
        _no_tangent("the gradient of packed_attn", go)
        q, k, v, o, M, L, offsets, k_offsets = ctx.saved_tensors
        causal, scale = ctx.how
        # (hooks on saved tensors may return copies of another layout, or on another device)
        q, k, v, o, go = _tokens(q, "q"), _tokens(k, "k"), _tokens(v, "v"), _tokens(o, "o"), _tokens(go, "gradient")
        M, L = M.contiguous(), L.contiguous()
        offsets, k_offsets = _offsets(offsets, "offsets", q.device), _offsets(k_offsets, "k_offsets", q.device)
        for t in (k, v, o, go, M, L):
            _require(t.device == q.device, "saved tensors and gradient must be on the device of q")
        _, H, T, d = q.shape
        Hkv, Tk = k.shape[1:3]
        dq, dk, dv = (_like(t) if need else None for t, need in zip((q, k, v), ctx.needs_input_grad))
        lib = _lib.load()
        with _on_device(q):
            nbytes = int(lib.lvar_packed_attn_bwd_workspace_bytes(offsets.shape[0] - 1, T, Tk, H, Hkv, d, 1 if causal else 0))
            ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
            st = lib.lvar_packed_attn_bwd(_view(q), _view(k), _view(v), _view(o), _view(go), offsets.data_ptr(), k_offsets.data_ptr(), M.data_ptr(), L.data_ptr(),
                                          _view(dq), _view(dk), _view(dv), _ptr(ws), nbytes, offsets.shape[0] - 1, T, Tk, H, Hkv, d,
                                          1 if causal else 0, scale, _stream(q))
        _lib.check(st, "lvar_packed_attn_bwd")
        return dq, dk, dv, None, None, None, None


def packed_attn(q, k, v, offsets, k_offsets=None, scale=None, causal: bool = True) -> Tuple[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention inside each of B sequences that lie one behind the other: ``(o, (M, L))`` as
    :func:`lvar_amd.sparse_attn_ops.dense_attn`, differentiable in q, k and v (``M`` and ``L`` take no gradient).

    ``q`` ``[1,H,T,d]``, ``k`` and ``v`` ``[1,Hkv,Tk,d]`` with H a multiple of Hkv (query head h reads key/value head ``h // (H // Hkv)``), of
    any strides: the views of a fused projection are read in place.  ``offsets`` int32 ``[B+1]``, on the device, ascending: sequence b has the
    queries ``offsets[b] .. offsets[b+1]-1``; and the keys ``k_offsets[b] .. k_offsets[b+1]-1``, the same by default.  ``causal``: row i of n queries
    sees keys ``j < m - n + i + 1`` of m, its own position and those ahead of it where n = m; otherwise all.  Sequences may be empty.  Rows that see
    no key (or only scores below -10^30, -infinity among them), and rows ahead of the first sequence or behind the last, get ``o = 0, M = -inf, L = 1``; rows of no sequence get zero gradients.
    The lengths are read by the kernels: a captured call is replayed with others.

    ``head_dim`` 16, 32, 64, 128 or 256.  Scores, statistics and sums are fp32 (a score x is off by up to 2^-24 of
    ``|x|``, its probability by a factor of 2 to that: scores belong below 2^20); probabilities (and in the backward pass their gradients) are rounded to
    bf16 where they enter a product.  The order of all sums is fixed: the same call gives the same bits.  A value that is not finite reaches the
    rows that see it, and through them the gradients, and nothing else.  ``o`` and the gradients have the order of axes of their inputs.  Once
    differentiable, in reverse mode."""
    fast = _native()
    if fast is not None:
        r = fast.fast_packed_attn(q, k, v, offsets, k_offsets, _plain_scale(scale), causal)
        if r is not None:
            return r[0], (r[1], r[2])
    _no_tangent("packed_attn", q, k, v)
    d = q.shape[-1] if q.dim() else 0
    q, k, v, small = _pad_head_dim(q, k, v)
    q, k, v = _tokens(q, "q"), _tokens(k, "k"), _tokens(v, "v")
    qs, ks = q.shape, k.shape
    _require(ks == v.shape, lambda: f"k/v shape mismatch: {tuple(k.shape)} vs {tuple(v.shape)}")
    _require(qs[0] == 1 and ks[0] == 1, lambda: f"packed sequences are a batch of one, got {tuple(q.shape)} and {tuple(k.shape)}")
    _require(qs[3] == ks[3] and ks[1] > 0 and qs[1] > 0 and qs[1] % ks[1] == 0,
             lambda: f"q and k must be [1,H,T,d] and [1,Hkv,Tk,d] with H a positive multiple of Hkv, got {tuple(qs)}, {tuple(ks)}")
    _require(qs[3] in (64, 128, 256), lambda: f"head_dim must be 16, 32, 64, 128 or 256, got {d}")
    _require(q.device == k.device == v.device, "q, k, v must be on the same device")
    offsets = _offsets(offsets, "offsets", q.device)
    if k_offsets is None:
        _require(qs[2] == ks[2], lambda: f"q has {qs[2]} tokens and k {ks[2]}: give k_offsets")
        k_offsets = offsets
    else:
        k_offsets = _offsets(k_offsets, "k_offsets", q.device)
        _require(k_offsets.shape == offsets.shape, lambda: f"offsets and k_offsets must be of the same sequences, got {offsets.shape[0]} and {k_offsets.shape[0]}")
    args = (q, k, v, offsets, k_offsets, bool(causal), _scale_for(d, scale))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        o, M, L = _PackedAttn.apply(*args)
    else:
        o, M, L = _launch(*args)
    return (o if small is None else o[..., :small].contiguous()), (M, L)
