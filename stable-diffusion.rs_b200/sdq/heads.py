"""Queries, keys and values made ready for attention (include/sdq.h, ``sdq_qk_norm_rope``)."""
from __future__ import annotations

import ctypes

import torch

from ._abi import SDQ_ERR_INVALID, SDQ_ERR_UNSUPPORTED, SdqError, SdqHeads, check, lib
from .fp8 import _SOURCE, _current_device, _elsewhere, _raw_stream

_byref = ctypes.byref
_PAIRS = {"interleaved": 1, "halves": 0}


def _heads(t: torch.Tensor, tokens_axis: int) -> SdqHeads:
    st = t.stride()
    return SdqHeads(t.data_ptr(), t.shape[3 - tokens_axis], st[0], st[tokens_axis], st[3 - tokens_axis])


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 eps: float = 1e-6, positions: torch.Tensor | None = None, pairs: str = "interleaved", out=None, stream=None):
    """RMS norm of each query and key head, rotation by position, and the transposition that attention
    wants, in one pass: q [b, n, heads, d], k and v [b, n, kv_heads, d] -> (q, k, v) as [b, heads, n, d].

    The inputs are bf16 or f32 views of any strides whose last axis is contiguous, such as slices of a
    fused projection.  ``q_weight`` / ``k_weight`` [d] scale the normed vectors (None: no norm).  ``cos``
    and ``sin`` are f32 tables [positions, rope / 2] (None: no rotation), read at the token's index or at
    ``positions`` [b, n] (int32 or int64); a position outside the tables makes its token's queries and
    keys NaN.  ``pairs`` says which values turn together: ``"interleaved"`` (2i, 2i + 1) or ``"halves"``
    (i, i + rope / 2); values from rope on stay.  ``out`` gives the three results' places, views
    [b, heads, n, d] of any strides with a contiguous last axis, for instance parts of a joint sequence.
    An output may be its input's own memory (with the same strides), and must not overlap otherwise."""
    dev = q.device
    if dev.type != "cuda":
        raise SdqError(SDQ_ERR_INVALID, "libsdq takes device tensors (no CPU fallback)")
    if stream is not None or dev.index != _current_device():
        return _elsewhere(qk_norm_rope, dev, stream, q, k, v, q_weight, k_weight, cos, sin, eps, positions, pairs, out)
    if pairs not in _PAIRS:
        raise SdqError(SDQ_ERR_INVALID, f"pairs must be 'interleaved' or 'halves', not {pairs!r}")
    dtype = q.dtype
    if dtype not in _SOURCE:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"q must be bf16 or f32, not {dtype}")
    if q.dim() != 4:
        raise SdqError(SDQ_ERR_INVALID, f"q must be [batch, tokens, heads, head_dim], got shape {list(q.shape)}")
    b, n, _, d = q.shape
    srcs = (q, k) if v is None else (q, k, v)
    if out is None:
        outs = [torch.empty((b, t.shape[2], n, d), dtype=dtype, device=dev) if t.dim() == 4 else t for t in srcs]
    else:
        outs = [t for t in out if t is not None]
        if len(outs) != len(srcs):
            raise SdqError(SDQ_ERR_INVALID, f"out must hold {len(srcs)} tensors, got {len(outs)}")
    for name, t, o in zip("qkv", srcs, outs):
        if t.dim() != 4 or t.shape[0] != b or t.shape[1] != n or t.shape[3] != d:
            raise SdqError(SDQ_ERR_INVALID, f"{name} must be [{b}, {n}, heads, {d}], got shape {list(t.shape)}")
        if tuple(o.shape) != (b, t.shape[2], n, d):
            raise SdqError(SDQ_ERR_INVALID, f"{name}'s output must be {[b, t.shape[2], n, d]}, got shape {list(o.shape)}")
        for x in (t, o):
            if x.dtype is not dtype or x.device != dev:
                raise SdqError(SDQ_ERR_INVALID, f"{name} and its output must be {dtype} on {dev}, not {x.dtype} on {x.device}")
            if x.stride(3) != 1 and d > 1 and x.numel() > 0:
                raise SdqError(SDQ_ERR_INVALID, f"{name} and its output must have a contiguous last axis")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.dtype is not dtype or w.device != dev or w.numel() != d or not w.is_contiguous()):
            raise SdqError(SDQ_ERR_INVALID, f"{name} must hold {d} contiguous values of {dtype} on {dev}")
    rows = rope = wide = stride = 0
    if (cos is None) != (sin is None):
        raise SdqError(SDQ_ERR_INVALID, "cos and sin come together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dim() != 2 or t.shape != cos.shape or t.dtype is not torch.float32 or t.device != dev or not t.is_contiguous():
                raise SdqError(SDQ_ERR_INVALID, f"{name} must be a contiguous f32 [positions, rope / 2] on {dev}")
        rows, rope = cos.shape[0], 2 * cos.shape[1]
    if positions is not None:
        if cos is None:
            raise SdqError(SDQ_ERR_INVALID, "positions without cos and sin")
        if tuple(positions.shape) != (b, n) or positions.device != dev or positions.dtype not in (torch.int32, torch.int64) \
                or (n > 1 and positions.stride(1) != 1):
            raise SdqError(SDQ_ERR_INVALID, f"positions must be int32 or int64 [{b}, {n}] on {dev}, contiguous along the tokens")
        wide, stride = int(positions.dtype is torch.int64), positions.stride(0)
    i = [_heads(t, 1) for t in srcs]
    o = [_heads(t, 2) for t in outs]
    check(lib().sdq_qk_norm_rope(
        _byref(i[0]), _byref(i[1]), _byref(i[2]) if v is not None else None, _byref(o[0]), _byref(o[1]),
        _byref(o[2]) if v is not None else None, _SOURCE[dtype], b, n, d,
        None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
        None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(), rows, rope, _PAIRS[pairs],
        None if positions is None else positions.data_ptr(), wide, stride, _raw_stream(dev)))
    return (outs[0], outs[1], outs[2] if v is not None else None)
