"""Operators around a growing key/value cache: norms of queries and keys per head with the position rotation in the same pass
(:func:`qk_norm_rope`, differentiable), a paged cache of bf16 or 8-bit keys and values (:class:`PagedKVCache`,
:func:`kv_cache_append`, :func:`qk_norm_rope_append`, :func:`kv_cache_read`) and the attention of the newest tokens over it
(:func:`paged_attn`).

They stand between a model's fused projection and the attention operators of :mod:`lvar_amd.sparse_attn_ops`: the reference
normalises, rotates and concatenates in eager PyTorch around every attention call (models/sparvar/basic_sparvar.py:326-350).

Tensor contract as there: bf16 on a HIP device, ``[B,H,L,d]`` with unit stride on d, outputs freshly allocated, work enqueued on
the current torch stream of the tensors' device; wrong shapes raise :class:`ShapeError`, wrong dtypes ``TypeError``, CPU tensors
``RuntimeError``.  There is no PyTorch or CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .sparse_attn_ops import ShapeError, _native, _on_device, _plain_scale, _prep, _ptr, _require, _scale, _stream, _view

__all__ = ["PagedKVCache", "qk_norm_rope", "qk_norm_rope_append", "kv_cache_append", "kv_cache_read", "paged_attn", "ShapeError"]

_NORMS = {None: 0, "l2": 1, "rms": 2}
_EPS = {None: 0.0, "l2": 1e-12, "rms": 1e-6}
_LEAST, _MOST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


class PagedKVCache(NamedTuple):
    """Keys and values in pages: ``k`` and ``v`` ``[num_pages, kv_heads, page_size, head_dim]``, either bf16 or
    ``float8_e4m3fn`` codes with one power of two per row: ``k_exp`` and ``v_exp`` uint8 ``[num_pages, kv_heads, page_size]``,
    value = code * 2^(byte - 127) with bytes from 1 to 254.  ``page_size`` is a power of two from 16 to 1024, ``head_dim`` 64, 128 or 256; ``k`` and ``v``
    have the same strides, unit stride on the last axis, and rows that are 16-byte aligned.  The tuple only names
    the tensors: it holds no state.

    Which page holds which tokens is the caller's business: a ``page_table`` int32 ``[B, max_pages]`` names the pages of each
    sequence in order.  Entries outside ``[0, num_pages)`` name no page: tokens there are not written, read as zeros, and take
    no part in an attention.  Sequences may share pages that are only read."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: Optional[torch.Tensor] = None
    v_exp: Optional[torch.Tensor] = None

    @classmethod
    def alloc(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype=torch.bfloat16, device="cuda") -> "PagedKVCache":
        """A cache of zeros."""
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise TypeError(f"a cache holds bfloat16 or float8_e4m3fn, got {dtype}")
        shape = (num_pages, kv_heads, page_size, head_dim)
        if dtype is torch.bfloat16:
            return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
        pages = [torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
        exps = [torch.full(shape[:3], 127, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*pages, *exps)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def _rows(t, name: str):
    """``t`` as the kernels read it.  (A tensor whose base is misaligned, or with odd strides on axes of one element, may count as contiguous: it is copied.)"""
    t = _prep(t, name)
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:-1]) else t


def _same_strides(a, b) -> bool:
    return all(n <= 1 or x == y for n, x, y in zip(a.shape, a.stride(), b.stride()))


def _cache_arg(cache, page_table, B: int, device) -> _lib.LvarPagedCache:
    k, v, ke, ve = cache.k, cache.v, cache.k_exp, cache.v_exp
    _require(k.dim() == 4 and k.shape == v.shape, lambda: f"cache.k and cache.v must be [pages,kv_heads,page_size,d] alike, got {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype not in (torch.bfloat16, torch.float8_e4m3fn) or v.dtype != k.dtype:
        raise TypeError(f"a cache holds bfloat16 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
    if not k.is_cuda:
        raise RuntimeError("the cache must live on a HIP device; lvar_amd has no CPU path")
    P, Hkv, page, d = k.shape
    _require(d in (64, 128, 256), lambda: f"head_dim of a cache must be 64, 128 or 256, got {d}")
    _require(16 <= page <= 1024 and page & (page - 1) == 0, lambda: f"page_size must be a power of two from 16 to 1024, got {page}")
    _require(P > 0 and Hkv > 0, "a cache needs pages and heads")
    size = k.element_size()
    _require(k.stride(3) == 1 and _same_strides(k, v) and v.stride(3) == 1, "cache.k and cache.v must have the same strides, 1 on the last axis")
    rows_ok = all(t.data_ptr() % 16 == 0 for t in (k, v)) and k.stride(2) * size % 16 == 0 and k.stride(2) >= d \
        and (Hkv == 1 or k.stride(1) * size % 16 == 0) and (P == 1 or k.stride(0) * size % 16 == 0)
    _require(rows_ok, "rows of the cache must be 16-byte aligned and apart from each other")
    es = (0, 0)
    if k.dtype == torch.bfloat16:
        _require(ke is None and ve is None, "a bfloat16 cache has no exponents")
    else:
        _require(ke is not None and ve is not None and tuple(ke.shape) == (P, Hkv, page) == tuple(ve.shape),
                 "a float8_e4m3fn cache needs k_exp and v_exp [pages,kv_heads,page_size]")
        if ke.dtype != torch.uint8 or ve.dtype != torch.uint8:
            raise TypeError("k_exp and v_exp must be uint8")
        es = (0 if P == 1 else ke.stride(0), 0 if Hkv == 1 else ke.stride(1))
        _require(ke.stride(2) == 1 and ve.stride(2) == 1 and _same_strides(ke, ve) and es[0] % 4 == 0 and es[1] % 4 == 0
                 and ke.data_ptr() % 4 == 0 and ve.data_ptr() % 4 == 0,
                 "k_exp and v_exp must have the same strides, 1 on the last axis and multiples of 4 on the others, and be 4-byte aligned")
    _require(page_table.dim() == 2 and page_table.shape[0] == B and page_table.shape[1] > 0,
             lambda: f"page_table must be [B = {B}, max_pages > 0], got {tuple(page_table.shape)}")
    if page_table.dtype != torch.int32:
        raise TypeError("page_table must be int32")
    for t in (k, v, ke, ve, page_table):
        _require(t is None or t.device == device, "the cache and its page table must be on the device of the tensors")
    _require(page_table.stride(1) == 1 or page_table.shape[1] == 1, "page_table must have unit stride along the pages")
    return _lib.LvarPagedCache(k.data_ptr(), v.data_ptr(), _ptr(ke), _ptr(ve), 0 if P == 1 else k.stride(0), 0 if Hkv == 1 else k.stride(1), k.stride(2),
                               es[0], es[1], page_table.data_ptr(), 0 if B == 1 else page_table.stride(0), P, Hkv, page, d, page_table.shape[1])


def _per_sequence(t, name: str, B: int, device):
    if t is None:
        return None
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    _require(t.dim() == 1 and t.shape[0] == B, lambda: f"{name} must be [B = {B}], got {tuple(t.shape)}")
    _require(t.device == device, lambda: f"{name} must be on the device of the tensors")
    return t.contiguous()


def _weight_arg(w, heads: int, d: int, name: str, device):
    """The weight as the kernels read it, and its descriptor."""
    if w is None:
        return None, _lib.LvarWeight(None, 0, 0, 0)
    if w.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{name} must be float32 or bfloat16, got {w.dtype}")
    ok = tuple(w.shape) == (d,) or (w.dim() == 2 and w.shape[0] in (1, heads) and w.shape[1] in (1, d))
    _require(ok, lambda: f"{name} must be [d], [H,1], [1,d] or [H,d] for H = {heads}, d = {d}, got {tuple(w.shape)}")
    _require(w.device == device, lambda: f"{name} must be on the device of q")
    w2 = w if w.dim() == 2 else w.unsqueeze(0)
    rows, cols = w2.shape
    if rows > 1 and w2.stride(0) == 0:
        w2 = w2.contiguous()       # a stride of 0 would say that the heads share one factor, and one gradient
    if cols > 1 and (w2.stride(1) != 1 or w2.data_ptr() % 16 or (rows > 1 and w2.stride(0) % 8)):
        w2 = w2.clone(memory_format=torch.contiguous_format)
    return w2, _lib.LvarWeight(w2.data_ptr(), w2.stride(0) if rows > 1 else 0, 1 if cols > 1 else 0, 1 if w2.dtype == torch.bfloat16 else 0)


def _table_arg(cos, sin, d: int, device):
    if cos is None and sin is None:
        return None, None
    _require(cos is not None and sin is not None, "cos and sin come together")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("cos and sin must be float32")
    _require(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[0] > 0, lambda: f"cos and sin must be [rows, rot/2] alike, got {tuple(cos.shape)}, {tuple(sin.shape)}")
    rot = 2 * cos.shape[1]
    _require(0 < rot <= d and rot % 16 == 0, lambda: f"the rotated columns (2 * {cos.shape[1]}) must be a multiple of 16 up to head_dim = {d}")
    _require(cos.device == device and sin.device == device, "cos and sin must be on the device of q")
    if cos.requires_grad or sin.requires_grad:
        raise RuntimeError("cos and sin take no gradient: detach them")
    if cos.stride(1) != 1 or sin.stride(1) != 1 or cos.stride(0) != sin.stride(0) or cos.stride(0) % 4 or cos.data_ptr() % 16 or sin.data_ptr() % 16:
        cos, sin = (t.clone(memory_format=torch.contiguous_format) for t in (cos, sin))
    return cos, sin


def _how(cos, sin, positions, wq: "_lib.LvarWeight", wk: "_lib.LvarWeight", norm, eps: float, interleaved: bool, B: int, L: int, device):
    h = _lib.LvarNormRope()
    h.norm, h.eps, h.q_weight, h.k_weight = _NORMS[norm], eps, wq, wk
    if cos is not None:
        h.cos, h.sin, h.table_stride, h.table_rows = cos.data_ptr(), sin.data_ptr(), cos.stride(0), cos.shape[0]
        h.rot_dim, h.interleaved = 2 * cos.shape[1], 1 if interleaved else 0
        if positions is not None:
            h.positions, h.positions64 = positions.data_ptr(), 1 if positions.dtype == torch.int64 else 0
            h.pos_stride_b = positions.stride(0) if positions.dim() == 2 and B > 1 else 0
            h.pos_stride_row = positions.stride(-1)
    return h


def _norm_args(q, k, cos, sin, positions, norm, eps):
    """Checks that the plain and the appending form share."""
    qs, ks = q.shape, k.shape
    _require(qs[0] == ks[0] and qs[2] == ks[2] and qs[3] == ks[3] and ks[1] > 0 and qs[1] > 0 and qs[1] % ks[1] == 0,
             lambda: f"q and k must be [B,H,L,d] and [B,Hkv,L,d] with H a positive multiple of Hkv, got {tuple(qs)}, {tuple(ks)}")
    _require(q.device == k.device, "q and k must be on the same device")
    _require(norm in _NORMS, lambda: f"norm must be 'l2', 'rms' or None, got {norm!r}")
    eps = _EPS[norm] if eps is None else float(eps)
    # (the reciprocal of a smaller one is no fp32 number, and rows of zeros would come out as NaN)
    _require(eps == 0.0 or _LEAST <= eps <= _MOST, "eps must be 0 or a normal fp32 number, and not negative")
    cos, sin = _table_arg(cos, sin, qs[3], q.device)
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be int32 or int64")
        _require(tuple(positions.shape) in ((qs[2],), (qs[0], qs[2])), lambda: f"positions must be [L] or [B,L], got {tuple(positions.shape)}")
        _require(positions.device == q.device, "positions must be on the device of q")
    return cos, sin, eps


def _no_tangent(name: str, *tensors) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative: call it on tensors without a tangent")


def _no_gradient(name: str, *tensors) -> None:
    _no_tangent(name, *tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")


def _norm_rope_launch(q, k, wq, wk, cos, sin, positions, norm, eps, interleaved):
    B, H, L, d = q.shape
    Hkv = k.shape[1]
    oq = torch.empty((B, H, L, d), dtype=q.dtype, device=q.device)
    ok = torch.empty((B, Hkv, L, d), dtype=q.dtype, device=q.device)
    if oq.numel() == 0:
        return oq, ok
    (wq, dq), (wk, dk) = _weight_arg(wq, H, d, "q_weight", q.device), _weight_arg(wk, Hkv, d, "k_weight", q.device)
    with _on_device(q):
        st = _lib.load().lvar_qk_norm_rope_fwd(_view(q), _view(k), _how(cos, sin, positions, dq, dk, norm, eps, interleaved, B, L, q.device),
                                              oq.data_ptr(), ok.data_ptr(), B, H, Hkv, L, d, _stream(q))
    _lib.check(st, "lvar_qk_norm_rope_fwd")
    return oq, ok


def _rows_like(t):
    """Memory for a gradient of t in t's own order of axes, if the kernels can write it."""
    g = torch.empty_like(t)
    ok = g.stride(-1) == 1 and all(s % 8 == 0 for s in g.stride()[:-1])
    return g if ok else torch.empty(t.shape, dtype=t.dtype, device=t.device)


class _NormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, norm, eps, interleaved):
        ctx.how = (norm, eps, interleaved)
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions)
        return _norm_rope_launch(q, k, wq, wk, cos, sin, positions, norm, eps, interleaved)

    @staticmethod
    def backward(ctx, gq, gk):
        if torch.is_grad_enabled():
            raise RuntimeError("qk_norm_rope can be differentiated once: its gradients have no graph (create_graph)")
        _no_tangent("the gradient of qk_norm_rope", gq, gk)
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        norm, eps, interleaved = ctx.how
        B, H, L, d = q.shape
        Hkv = k.shape[1]
        # (hooks on saved tensors may return copies of another layout, or on another device)
        q, k = _rows(q, "q"), _rows(k, "k")
        cos, sin = _table_arg(cos, sin, d, q.device)
        _require(positions is None or positions.device == q.device, "positions must be on the device of q")
        dq, dk = _rows_like(q), _rows_like(k)
        dwq = torch.empty_like(wq, memory_format=torch.contiguous_format) if wq is not None and ctx.needs_input_grad[2] else None
        dwk = torch.empty_like(wk, memory_format=torch.contiguous_format) if wk is not None and ctx.needs_input_grad[3] else None
        if q.numel() == 0:
            for t in (dwq, dwk):
                if t is not None:
                    t.zero_()
            return dq, dk, dwq, dwk, None, None, None, None, None, None
        gq, gk = _rows(gq.contiguous(), "gradient"), _rows(gk.contiguous(), "gradient")
        (wq, aq), (wk, ak) = _weight_arg(wq, H, d, "q_weight", q.device), _weight_arg(wk, Hkv, d, "k_weight", q.device)
        lib = _lib.load()
        with _on_device(q):
            nbytes = int(lib.lvar_qk_norm_rope_bwd_scratch_bytes(B, H, Hkv, L, d)) if dwq is not None or dwk is not None else 0
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes > 0 else None
            st = lib.lvar_qk_norm_rope_bwd(_view(q), _view(k), _how(cos, sin, positions, aq, ak, norm, eps, interleaved, B, L, q.device),
                                           gq.data_ptr(), gk.data_ptr(), _view(dq), _view(dk), _ptr(dwq), _ptr(dwk), _ptr(scratch), nbytes,
                                           B, H, Hkv, L, d, _stream(q))
        _lib.check(st, "lvar_qk_norm_rope_bwd")
        return dq, dk, dwq, dwk, None, None, None, None, None, None


def qk_norm_rope(q, k, cos=None, sin=None, positions=None, q_weight=None, k_weight=None, norm: Optional[str] = "l2",
                 eps: Optional[float] = None, interleaved: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries ``[B,H,L,d]`` and keys ``[B,Hkv,L,d]`` normalised per head, scaled and rotated, in one pass: ``(q, k)`` contiguous bf16.

    ``norm``: ``"l2"`` is ``x / max(|x|, eps)`` (eps 1e-12), ``"rms"`` ``x / sqrt(mean(x^2) + eps)`` (eps 1e-6), ``None`` leaves x; an
    eps of its own is 0 or a normal fp32 number.
    ``q_weight`` / ``k_weight`` (fp32 or bf16; ``[d]``, ``[H,1]``, ``[1,d]`` or ``[H,d]``) multiply the result.  ``cos`` / ``sin``
    fp32 ``[rows, rot/2]`` rotate the first ``rot`` columns (a multiple of 16) in pairs ``(2i, 2i+1)``, or ``(i, i + rot/2)``
    with ``interleaved=False``; token i takes row i, or row ``positions[i]`` / ``positions[b,i]`` (clamped to the table).
    ``head_dim`` 16, 32, 64, 128 or 256.  All in fp32, rounded once.  Differentiable in q, k and the weights (once, in
    reverse mode: inputs with a forward-mode tangent are refused); a backward pass that is captured in a graph wants leaves without a live eager
    graph, as always with autograd.  The
    reference's counterpart is models/sparvar/basic_sparvar.py:326-342, eager."""
    fast = _native()
    if fast is not None:
        r = fast.fast_qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, norm, eps, interleaved)
        if r is not None:
            return r
    _no_tangent("qk_norm_rope", q, k, cos, sin, q_weight, k_weight)
    q, k = _rows(q, "q"), _rows(k, "k")
    cos, sin, eps = _norm_args(q, k, cos, sin, positions, norm, eps)
    _require(q.shape[3] in (16, 32, 64, 128, 256), lambda: f"head_dim must be 16, 32, 64, 128 or 256, got {q.shape[3]}")
    _require(cos is None or positions is not None or cos.shape[0] >= q.shape[2],
             lambda: f"cos and sin have {cos.shape[0]} rows for {q.shape[2]} tokens: give positions, or a longer table")
    for w, heads, name in ((q_weight, q.shape[1], "q_weight"), (k_weight, k.shape[1], "k_weight")):
        _weight_arg(w, heads, q.shape[3], name, q.device)
    args = (q, k, q_weight, k_weight, cos, sin, positions, norm, eps, bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _NormRope.apply(*args)
    return _norm_rope_launch(*args)


def _append(cache, q, k, v, page_table, start, counts, how, oq):
    B, Hkv, L, d = k.shape
    with _on_device(k):
        st = _lib.load().lvar_kv_cache_append(_view(q), _view(k), _view(v), None if how is None else C.byref(how), _ptr(oq),
                                             _cache_arg(cache, page_table, B, k.device), start.data_ptr(), _ptr(counts),
                                             B, Hkv if q is None else q.shape[1], L, _stream(k))
    _lib.check(st, "lvar_kv_cache_append")
    # (autograd finds out where it has saved them; tensors of inference mode have no version)
    torch.autograd.graph.increment_version([t for t in cache if t is not None and not t.is_inference()])


def _append_args(cache, k, v, page_table, start, counts):
    _require(k.shape == v.shape, lambda: f"k/v shape mismatch: {tuple(k.shape)} vs {tuple(v.shape)}")
    _require(k.device == v.device, "k and v must be on the same device")
    B = k.shape[0]
    _cache_arg(cache, page_table, B, k.device)
    _require(cache.k.shape[1] == k.shape[1] and cache.k.shape[3] == k.shape[3],
             lambda: f"the cache holds {cache.k.shape[1]} heads of {cache.k.shape[3]}, k is {tuple(k.shape)}")
    _require(start is not None, "start must be given")
    return _per_sequence(start, "start", B, k.device), _per_sequence(counts, "counts", B, k.device)


def kv_cache_append(cache: PagedKVCache, k, v, page_table, start, counts=None) -> None:
    """Writes the L tokens of ``k`` and ``v`` ``[B,Hkv,L,d]`` to positions ``start[b] ..`` of their sequences, in place;
    ``counts`` int32 ``[B]`` limits a padded batch to the first ``counts[b]`` tokens.  An 8-bit cache gets, per token and
    head, the smallest power of two with ``max|x| <= 448 * 2^e`` and codes rounded to nearest even; infinities become NaN there.
    Positions outside the page table are dropped.  Two tokens of one call that go to the same row leave it undefined."""
    fast = _native()
    if fast is not None and fast.fast_kv_append(cache, page_table, start, counts, None, k, v):
        return
    _no_gradient("kv_cache_append", k, v, cache.k, cache.v)
    k, v = _rows(k, "k"), _rows(v, "v")
    start, counts = _append_args(cache, k, v, page_table, start, counts)
    if k.numel():
        _append(cache, None, k, v, page_table, start, counts, None, None)


def qk_norm_rope_append(cache: PagedKVCache, q, k, v, page_table, start, cos=None, sin=None, counts=None, positions=None, q_weight=None,
                        k_weight=None, norm: Optional[str] = "l2", eps: Optional[float] = None, interleaved: bool = True) -> torch.Tensor:
    """:func:`qk_norm_rope` on q and k and :func:`kv_cache_append` of the keys and of ``v``, in one launch; returns the queries.
    Without ``positions`` token i of sequence b takes row ``start[b] + i`` of the tables (clamped to them).  The keys are rounded once, from fp32 to
    the cache's type."""
    fast = _native()
    if fast is not None:
        r = fast.fast_kv_append(cache, page_table, start, counts, q, k, v, cos, sin, positions, q_weight, k_weight,
                                norm, eps, interleaved)
        if r is not None:
            return r
    _no_gradient("qk_norm_rope_append", q, k, v, q_weight, k_weight, cache.k, cache.v)
    _no_tangent("qk_norm_rope_append", cos, sin)
    q, k, v = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    cos, sin, eps = _norm_args(q, k, cos, sin, positions, norm, eps)
    start, counts = _append_args(cache, k, v, page_table, start, counts)
    B, H, L, d = q.shape
    oq = torch.empty((B, H, L, d), dtype=q.dtype, device=q.device)
    (wq, aq), (wk, ak) = _weight_arg(q_weight, H, d, "q_weight", q.device), _weight_arg(k_weight, k.shape[1], d, "k_weight", q.device)
    if oq.numel():
        _append(cache, q, k, v, page_table, start, counts, _how(cos, sin, positions, aq, ak, norm, eps, bool(interleaved), B, L, q.device), oq)
    return oq


def kv_cache_read(cache: PagedKVCache, page_table, lengths, max_len: Optional[int] = None, start=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens ``start[b] ..`` (default 0) of every sequence as contiguous bf16 ``(k, v)`` ``[B,Hkv,max_len,d]``, the form that the
    dense and sparse attention operators take; zeros from position ``lengths[b]`` on.  ``max_len`` defaults to all that the page
    table can name.  Every value that an append has written is a bf16 value and comes back exactly, but at the ends of the range: rounded below
    2^-130, and infinite from 2^128 on, to which an 8-bit cache rounds elements of 1.9375 * 2^127 and more."""
    fast = _native()
    if fast is not None:
        r = fast.fast_kv_read(cache, page_table, lengths, max_len, start)
        if r is not None:
            return r
    _no_gradient("kv_cache_read", cache.k, cache.v)
    device = cache.k.device
    B = page_table.shape[0]
    arg = _cache_arg(cache, page_table, B, device)
    _require(lengths is not None, "lengths must be given")
    lengths, start = _per_sequence(lengths, "lengths", B, device), _per_sequence(start, "start", B, device)
    max_len = page_table.shape[1] * cache.page_size if max_len is None else int(max_len)
    _require(max_len >= 0, "max_len must not be negative")
    Hkv, d = cache.k.shape[1], cache.k.shape[3]
    k, v = (torch.empty((B, Hkv, max_len, d), dtype=torch.bfloat16, device=device) for _ in range(2))
    if k.numel():
        with _on_device(k):
            st = _lib.load().lvar_kv_cache_read(arg, _ptr(start), lengths.data_ptr(), k.data_ptr(), v.data_ptr(), B, max_len, _stream(k))
        _lib.check(st, "lvar_kv_cache_read")
    return k, v


def paged_attn(q, cache: PagedKVCache, page_table, lengths, scale=None, causal: bool = False, counts=None, max_len: Optional[int] = None):
    """Attention of the newest tokens ``q`` ``[B,H,Lq,d]`` over the first ``lengths[b]`` tokens of a cache that holds them already:
    ``(o, (M, L))`` as :func:`lvar_amd.sparse_attn_ops.dense_attn`.  One token, a small scale, or a chunk; query head h reads key/value
    head ``h // (H // Hkv)``.  ``causal``: row i of sequence b sees tokens ``j < lengths[b] - n + i + 1`` with ``n = counts[b]``
    (default Lq) new tokens; otherwise all ``lengths[b]``.  Rows ``i >= counts[b]`` of a padded batch and rows that see no token
    get ``o = 0, M = -inf, L = 1``.  What the cache holds behind ``lengths`` does not matter; a value that is not finite reaches the rows that
    see it and no others.  Scores, statistics and sums are fp32; the probabilities enter the second product as two bf16 terms (2^-16) up to 32 rows
    (query heads per key/value head times Lq; up to 16 for 8-bit caches of head_dim 256), as one (2^-8) beyond, and for bf16 caches of head_dim 256.  ``max_len`` bounds the lengths (longer ones are clamped to it; default: all that the page table
    can name): a small bound lets the launch do without the pass that joins the parts of long sequences."""
    fast = _native()
    if fast is not None:
        r = fast.fast_paged_attn(q, cache, page_table, lengths, counts, _plain_scale(scale), causal, max_len)
        if r is not None:
            return r[0], (r[1], r[2])
    _no_gradient("paged_attn", q, cache.k, cache.v)
    q = _rows(q, "q")
    B, H, Lq, d = q.shape
    arg = _cache_arg(cache, page_table, B, q.device)
    Hkv = cache.k.shape[1]
    _require(cache.k.shape[3] == d and H > 0 and H % Hkv == 0, lambda: f"the cache holds {Hkv} heads of {cache.k.shape[3]}, q is {tuple(q.shape)}")
    _require(lengths is not None, "lengths must be given")
    lengths, counts = _per_sequence(lengths, "lengths", B, q.device), _per_sequence(counts, "counts", B, q.device)
    reach = page_table.shape[1] * cache.page_size
    max_len = reach if max_len is None else min(int(max_len), reach)
    _require(max_len >= 0, "max_len must not be negative")
    o = torch.empty((B, H, Lq, d), dtype=q.dtype, device=q.device)
    M, L = torch.empty((2, B, H, Lq, 1), dtype=torch.float32, device=q.device).unbind(0)
    if o.numel():
        lib = _lib.load()
        with _on_device(q):
            nbytes = int(lib.lvar_paged_attn_workspace_bytes(B, H, Hkv, Lq, max_len, d))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes > 0 else None
            st = lib.lvar_paged_attn_fwd(_view(q), arg, lengths.data_ptr(), _ptr(counts), o.data_ptr(), M.data_ptr(), L.data_ptr(), _ptr(ws), max(0, nbytes),
                                         B, H, Lq, max_len, 1 if causal else 0, _scale(q, scale), _stream(q))
        _lib.check(st, "lvar_paged_attn_fwd")
    return o, (M, L)
