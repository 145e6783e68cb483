"""Queries, keys and values made ready for attention (include/sdq.h, ``sdq_qk_norm_rope``)."""
from __future__ import annotations

import ctypes
from array import array

import torch

from ._abi import SDQ_ERR_INVALID, SDQ_ERR_UNSUPPORTED, SdqError, SdqHeads, check, lib
from .fp8 import _SOURCE, _current_device, _elsewhere, _empty_strided, _like, _raw_stream

_PAIRS = {"interleaved": 1, "halves": 0}
_WIDE = {torch.int32: 0, torch.int64: 1}
_HEADS = ctypes.sizeof(SdqHeads)               # five 64-bit fields


def _refuse(dev: int, dtype, b: int, n: int, d: int, tensors, weights, cos, sin, positions) -> None:
    """Raise for the first argument that is not what the call needs (the caller has seen that one is)."""
    for name, t, o in tensors:
        if t.dim() != 4 or t.shape[0] != b or t.shape[1] != n or t.shape[3] != d:
            raise SdqError(SDQ_ERR_INVALID, f"{name} must be [{b}, {n}, heads, {d}], got shape {list(t.shape)}")
        if o is not None and tuple(o.shape) != (b, t.shape[2], n, d):
            raise SdqError(SDQ_ERR_INVALID, f"{name}'s output must be {[b, t.shape[2], n, d]}, got shape {list(o.shape)}")
        for x in (t, t if o is None else o):
            if x.dtype is not dtype or x.get_device() != dev:
                raise SdqError(SDQ_ERR_INVALID, f"{name} and its output must be {dtype} on cuda:{dev}, not {x.dtype} on {x.device}")
            if x.stride(3) != 1:
                raise SdqError(SDQ_ERR_INVALID, f"{name} and its output must have a contiguous last axis")
    for name, w in weights:
        if w is not None and not _like(w, dev, dtype, d):
            raise SdqError(SDQ_ERR_INVALID, f"{name} must hold {d} contiguous values of {dtype} on cuda:{dev}")
    if (cos is None) != (sin is None):
        raise SdqError(SDQ_ERR_INVALID, "cos and sin come together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dim() != 2 or t.shape != cos.shape or not _like(t, dev, torch.float32, cos.numel()):
                raise SdqError(SDQ_ERR_INVALID, f"{name} must be a contiguous f32 [positions, rope / 2] on cuda:{dev}")
    if positions is not None:
        if cos is None:
            raise SdqError(SDQ_ERR_INVALID, "positions without cos and sin")
        raise SdqError(SDQ_ERR_INVALID, f"positions must be int32 or int64 [{b}, {n}] on cuda:{dev}, contiguous along the tokens")
    raise SdqError(SDQ_ERR_INVALID, "invalid arguments")


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
    dev = q.get_device()
    if stream is not None or dev < 0 or dev != _current_device():
        return _elsewhere(qk_norm_rope, q.device, stream, q, k, v, q_weight, k_weight, cos, sin, eps, positions, pairs, out)
    turn = _PAIRS.get(pairs)
    if turn is None:
        raise SdqError(SDQ_ERR_INVALID, f"pairs must be 'interleaved' or 'halves', not {pairs!r}")
    dtype = q.dtype
    dt = _SOURCE.get(dtype)
    if dt is None:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"q must be bf16 or f32, not {dtype}")
    if q.dim() != 4:
        raise SdqError(SDQ_ERR_INVALID, f"q must be [batch, tokens, heads, head_dim], got shape {list(q.shape)}")
    b, n, _, d = q.shape
    srcs = (q, k) if v is None else (q, k, v)
    good, table, outs = True, array("q"), out
    if out is not None:
        outs = [t for t in out if t is not None]
        if len(outs) != len(srcs):
            raise SdqError(SDQ_ERR_INVALID, f"out must hold {len(srcs)} tensors, got {len(outs)}")
    else:
        outs = []
    for i, t in enumerate(srcs):
        if t.dim() != 4:
            good = False
            break
        tb, tn, h, td = t.shape
        if not (tb == b and tn == n and td == d and t.dtype is dtype and t.get_device() == dev):
            good = False
            break
        s0, s1, s2, s3 = t.stride()
        if out is None:
            o, o0, o1, o2 = _empty_strided((b, h, n, d), (h * n * d, n * d, d, 1), dtype), h * n * d, n * d, d
            outs.append(o)
        else:
            o = outs[i]
            if not (o.shape == (b, h, n, d) and o.dtype is dtype and o.get_device() == dev):
                good = False
                break
            o0, o1, o2, o3 = o.stride()
            good = good and o3 == 1
        good = good and s3 == 1
        table.extend((t.data_ptr(), h, s0, s1, s2, o.data_ptr(), h, o0, o2, o1))
    rows = rope = wide = stride = cp = sp = pp = 0
    if good and cos is not None and sin is not None and cos.dim() == 2 and sin.shape == cos.shape:
        rows, rope = cos.shape
        good = _like(cos, dev, torch.float32, rows * rope) and _like(sin, dev, torch.float32, rows * rope)
        rope, cp, sp = 2 * rope, cos.data_ptr(), sin.data_ptr()
    elif cos is not None or sin is not None:
        good = False
    if positions is not None:
        wide = _WIDE.get(positions.dtype)
        good = good and cos is not None and wide is not None and positions.shape == (b, n) and positions.get_device() == dev
        if good:
            stride, step = positions.stride()
            good = step == 1 or n == 1
            pp = positions.data_ptr()
    if not (good and (q_weight is None or _like(q_weight, dev, dtype, d)) and (k_weight is None or _like(k_weight, dev, dtype, d))):
        _refuse(dev, dtype, b, n, d, [(*x, outs[i] if out is not None else None) for i, x in enumerate(zip("qkv", srcs))], (("q_weight", q_weight), ("k_weight", k_weight)), cos, sin,
                positions)
    at = table.buffer_info()[0]                    # sdq_heads: input and output of q, of k, of v
    check(lib().sdq_qk_norm_rope(
        at, at + 2 * _HEADS, None if v is None else at + 4 * _HEADS, at + _HEADS, at + 3 * _HEADS,
        None if v is None else at + 5 * _HEADS, dt, b, n, d, None if q_weight is None else q_weight.data_ptr(),
        None if k_weight is None else k_weight.data_ptr(), eps, cp, sp, rows, rope, turn, pp, wide, stride, _raw_stream(dev)))
    return (*outs, None) if v is None else tuple(outs)
