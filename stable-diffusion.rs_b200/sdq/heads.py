"""Queries, keys and values made ready for attention (include/sdq.h, ``sdq_qk_norm_rope``)."""
from __future__ import annotations

import ctypes

import torch

from ._abi import SDQ_ERR_INVALID, SDQ_ERR_UNSUPPORTED, SdqError, SdqHeads, check, lib, native
from .fp8 import _SOURCE, _current_device, _elsewhere, _raw_stream

_PAIRS = {"interleaved": 1, "halves": 0}
_heads = native("qk_norm_rope")


def _like(t, dev: int, dtype, count: int) -> bool:
    return t.dtype is dtype and t.numel() == count and t.get_device() == dev and t.is_contiguous()


def _struct(t: torch.Tensor, tokens_axis: int):
    st = t.stride()
    return ctypes.byref(SdqHeads(t.data_ptr(), t.shape[3 - tokens_axis], st[0], st[tokens_axis], st[3 - tokens_axis]))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 eps: float = 1e-6, positions: torch.Tensor | None = None, pairs: str = "interleaved", out=None, stream=None):
    """RMS norm of each query and key head, rotation by position, and the transposition that attention
    wants, in one pass: q [b, n, heads, d], k and v [b, n, kv_heads, d] -> (q, k, v) as [b, heads, n, d].

    The inputs are bf16 or f32 views of any strides whose last axis is contiguous, such as slices of a
    fused projection.  ``q_weight`` / ``k_weight`` [d] scale the normed vectors (None: no norm).  ``cos``
    and ``sin`` are f32 tables [positions, rope / 2] (None: no rotation), read at the token's index or at
    ``positions`` [b, n] (int32 or int64); a position outside the tables makes the rotated values of its
    token's queries and keys NaN.  ``pairs`` says which values turn together: ``"interleaved"`` (2i, 2i + 1) or ``"halves"``
    (i, i + rope / 2); values from rope on stay.  ``out`` gives the three results' places, views
    [b, heads, n, d] of any strides with a contiguous last axis, for instance parts of a joint sequence.
    An output may be its input's own memory (with the same strides), and must not overlap otherwise."""
    if stream is None:
        done = _heads(q, k, v, q_weight, k_weight, cos, sin, eps, positions, pairs, out)
        if done is not None:
            return done
    dev = q.get_device()
    if stream is not None or dev < 0 or dev != _current_device():
        return _elsewhere(qk_norm_rope, q.device, stream, q, k, v, q_weight, k_weight, cos, sin, eps, positions, pairs, out)
    if pairs not in _PAIRS:
        raise SdqError(SDQ_ERR_INVALID, f"pairs must be 'interleaved' or 'halves', not {pairs!r}")
    dtype = q.dtype
    if dtype not in _SOURCE:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"q must be bf16 or f32, not {dtype}")
    if q.dim() != 4:
        raise SdqError(SDQ_ERR_INVALID, f"q must be [batch, tokens, heads, head_dim], got shape {list(q.shape)}")
    b, n, _, d = q.shape
    srcs = (q, k) if v is None else (q, k, v)
    if out is not None:
        outs = tuple(t for t in out if t is not None)
        if len(outs) != len(srcs):
            raise SdqError(SDQ_ERR_INVALID, f"out must hold {len(srcs)} tensors, got {len(outs)}")
    else:
        outs = tuple(t.new_empty((b, t.shape[2], n, d)) if t.dim() == 4 else t for t in srcs)
    for name, t, o in zip("qkv", srcs, outs):
        if t.dim() != 4 or t.shape[0] != b or t.shape[1] != n or t.shape[3] != d:
            raise SdqError(SDQ_ERR_INVALID, f"{name} must be [{b}, {n}, heads, {d}], got shape {list(t.shape)}")
        if tuple(o.shape) != (b, t.shape[2], n, d):
            raise SdqError(SDQ_ERR_INVALID, f"{name}'s output must be {[b, t.shape[2], n, d]}, got shape {list(o.shape)}")
        for x in (t, o):
            if x.dtype is not dtype or x.get_device() != dev:
                raise SdqError(SDQ_ERR_INVALID, f"{name} and its output must be {dtype} on cuda:{dev}, not {x.dtype} on {x.device}")
            if x.stride(3) != 1:
                raise SdqError(SDQ_ERR_INVALID, f"{name} and its output must have a contiguous last axis")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and not _like(w, dev, dtype, d):
            raise SdqError(SDQ_ERR_INVALID, f"{name} must hold {d} contiguous values of {dtype} on cuda:{dev}")
    if (cos is None) != (sin is None):
        raise SdqError(SDQ_ERR_INVALID, "cos and sin come together")
    rows = rope = wide = stride = 0
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dim() != 2 or t.shape != cos.shape or not _like(t, dev, torch.float32, cos.numel()):
                raise SdqError(SDQ_ERR_INVALID, f"{name} must be a contiguous f32 [positions, rope / 2] on cuda:{dev}")
        rows, rope = cos.shape[0], 2 * cos.shape[1]
    if positions is not None:
        if cos is None:
            raise SdqError(SDQ_ERR_INVALID, "positions without cos and sin")
        if tuple(positions.shape) != (b, n) or positions.get_device() != dev or positions.dtype not in (torch.int32, torch.int64) \
                or (n > 1 and positions.stride(1) != 1):
            raise SdqError(SDQ_ERR_INVALID, f"positions must be int32 or int64 [{b}, {n}] on cuda:{dev}, contiguous along the tokens")
        wide, stride = int(positions.dtype is torch.int64), positions.stride(0)
    i = [_struct(t, 1) for t in srcs] + [None]
    o = [_struct(t, 2) for t in outs] + [None]
    check(lib().sdq_qk_norm_rope(
        i[0], i[1], i[2], o[0], o[1], o[2], _SOURCE[dtype], b, n, d, None if q_weight is None else q_weight.data_ptr(),
        None if k_weight is None else k_weight.data_ptr(), eps, None if cos is None else cos.data_ptr(),
        None if sin is None else sin.data_ptr(), rows, rope, _PAIRS[pairs],
        None if positions is None else positions.data_ptr(), wide, stride, _raw_stream(dev)))
    return (*outs, None) if v is None else outs
