"""Weights and activations in block-scaled 8-bit floating point (include/sdq.h, "Block-scaled").

A value is one e4m3 number; every 128 values along the inner axis share a power-of-two scale, one
e8m0 byte: ``xs[k // 128, row]`` for activations, ``ws[row // 128, k // 128]`` (128 x 128 blocks)
for weights.  The tensors carry torch's own types, ``float8_e4m3fn`` and ``float8_e8m0fnu``, so
``q.float()`` and ``s.float()`` are the numbers.  Beside the affine form (:class:`sdq.QuantizedArray`)
this one needs no unpacking before the product and its activations are 8 bits too, which runs the
tensor cores at twice their bf16 rate; it keeps 4 significant bits of every value.

Like the rest of the package: device tensors only, contiguous, no CPU fallback, asynchronous on
``stream`` (default: the current stream of the tensors' device).  With an explicit ``stream`` the
results are allocated on it.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _ACTS
from ._abi import SDQ_BF16, SDQ_ERR_INVALID, SDQ_ERR_UNSUPPORTED, SDQ_F32, SdqError, as_result, check, lib, native, on

#: Values that share a scale, along a row (activations) or both ways (weights).
BLOCK = 128

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_SOURCE = {torch.bfloat16: SDQ_BF16, torch.float32: SDQ_F32}
_NAMES = {torch.bfloat16: "bf16", torch.float32: "f32"}
_current_device = torch.cuda.current_device


_raw_stream = torch._C._cuda_getCurrentRawStream
_quantize, _quantize_weight, _matmul = native("fp8_quantize"), native("fp8_quantize_weight"), native("fp8_matmul")


def _elsewhere(fn, device, stream, *args, **kw):
    """``fn`` again with ``stream`` current (allocations included), or on another device."""
    if device.type != "cuda":
        raise SdqError(SDQ_ERR_INVALID, "libsdq takes device tensors (no CPU fallback)")
    with on(stream, device):
        return fn(*args, **kw)


def _demand(name: str, first: torch.Tensor, expected) -> None:
    """Raise for the first of ``expected`` -- (name, tensor, dtypes, shape or count) -- that is not a
    contiguous tensor like that on ``first``'s device."""
    if not first.is_cuda:
        raise SdqError(SDQ_ERR_INVALID, "libsdq takes device tensors (no CPU fallback)")
    for n, t, dtypes, shape in expected:
        if t is None:
            continue
        if t.device != first.device:
            raise SdqError(SDQ_ERR_INVALID, f"{n} is on {t.device}, {name} on {first.device}")
        if not t.is_contiguous():
            raise SdqError(SDQ_ERR_INVALID, f"libsdq takes contiguous row-major tensors; {n} is not")
        if isinstance(shape, int) and (t.numel() != shape or t.dtype not in dtypes):
            raise SdqError(SDQ_ERR_INVALID, f"{n} must hold {shape} values of {dtypes[0]}, not {t.numel()} of {t.dtype}")
        if t.dtype not in dtypes:
            raise SdqError(SDQ_ERR_UNSUPPORTED, f"{n} must be {' or '.join(_NAMES.get(d, str(d)) for d in dtypes)}, not {t.dtype}")
        if isinstance(shape, tuple) and tuple(t.shape) != shape:
            raise SdqError(SDQ_ERR_INVALID, f"{n} must have shape {list(shape)}, not {list(t.shape)}")


def _rows(x: torch.Tensor, name: str):
    """(rows, width) of a tensor whose last axis is the inner one."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise SdqError(SDQ_ERR_INVALID, f"{name} needs an inner axis of at least one value, got shape {list(x.shape)}")
    k = x.shape[-1]
    return x.numel() // k, k


def fp8_quantize(x: torch.Tensor, stream=None):
    """Activations x [..., k] (bf16 or f32) -> (xq [..., k] e4m3, xs [ceil(k / 128), rows] e8m0),
    rows the product of the leading axes (``sdq_fp8_quantize``).  k is a multiple of 16."""
    if stream is None:
        done = _quantize(x)
        if done is not None:
            return done
    dev = x.get_device()
    if stream is not None or dev < 0 or dev != _current_device():
        return _elsewhere(fp8_quantize, x.device, stream, x)
    _demand("x", x, [("x", x, tuple(_SOURCE), None)])
    m, k = _rows(x, "x")
    xq = torch.empty_like(x, dtype=E4M3)
    xs = x.new_empty((-(-k // BLOCK), m), dtype=E8M0)
    check(lib().sdq_fp8_quantize(x.data_ptr(), _SOURCE[x.dtype], m, k, xq.data_ptr(), xs.data_ptr(), _raw_stream(dev)))
    return xq, xs


def fp8_quantize_weight(w: torch.Tensor, stream=None):
    """A weight w [n, k] (bf16 or f32) -> (wq [n, k] e4m3, ws [ceil(n / 128), ceil(k / 128)] e8m0)
    (``sdq_fp8_quantize_weight``).  k is a multiple of 16."""
    if stream is None:
        done = _quantize_weight(w)
        if done is not None:
            return done
    dev = w.get_device()
    if stream is not None or dev < 0 or dev != _current_device():
        return _elsewhere(fp8_quantize_weight, w.device, stream, w)
    _demand("w", w, [("w", w, tuple(_SOURCE), None)])
    if w.dim() != 2:
        raise SdqError(SDQ_ERR_INVALID, f"fp8_quantize_weight wants a 2-D weight, got shape {list(w.shape)}")
    n, k = w.shape
    wq = torch.empty_like(w, dtype=E4M3)
    ws = w.new_empty((-(-n // BLOCK), -(-k // BLOCK)), dtype=E8M0)
    check(lib().sdq_fp8_quantize_weight(w.data_ptr(), _SOURCE[w.dtype], n, k, wq.data_ptr(), ws.data_ptr(), _raw_stream(dev)))
    return wq, ws


def fp8_dequantize(q: torch.Tensor, scales: torch.Tensor, weight: bool, out_dtype=torch.bfloat16, stream=None):
    """The values that e4m3 codes and their scales stand for, rounded once (``sdq_fp8_dequantize``).
    ``weight`` says which scales they are: a weight's 128 x 128 blocks or an activation's groups."""
    dev = q.get_device()
    if stream is not None or dev < 0 or dev != _current_device():
        return _elsewhere(fp8_dequantize, q.device, stream, q, scales, weight, out_dtype)
    rows, k = _rows(q, "q")
    kb = -(-k // BLOCK)
    _demand("q", q, [("q", q, (E4M3,), None), ("scales", scales, (E8M0,), (-(-rows // BLOCK), kb) if weight else (kb, rows))])
    if out_dtype not in _SOURCE:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"out must be bf16 or f32, not {out_dtype}")
    out = torch.empty_like(q, dtype=out_dtype)
    check(lib().sdq_fp8_dequantize(q.data_ptr(), scales.data_ptr(), rows, k, int(bool(weight)), out.data_ptr(),
                                   _SOURCE[out_dtype], _raw_stream(dev)))
    return out


def fp8_matmul(xq: torch.Tensor, xs: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, bias=None, act=None,
               gate=None, residual=None, out=None, out_dtype=None, stream=None) -> torch.Tensor:
    """``residual + gate * act(x . w^T + bias)`` of block-scaled operands, [..., k] x [n, k] -> [..., n]
    (``sdq_fp8_matmul``): f32 sums, rounded once to bf16 (or f32, which takes a bias only).

    ``act`` is None, ``"gelu_approx"`` or ``"silu"``; ``bias`` and ``gate`` hold n values, ``residual``
    has the result's shape and may be ``out`` itself."""
    if stream is None:
        done = _matmul(xq, xs, wq, ws, bias, act, gate, residual, out, out_dtype)
        if done is not None:
            return done
    dev = xq.get_device()
    if stream is not None or dev < 0 or dev != _current_device():
        return _elsewhere(fp8_matmul, xq.device, stream, xq, xs, wq, ws, bias, act, gate, residual, out, out_dtype)
    if act not in _ACTS:
        raise SdqError(SDQ_ERR_INVALID, f"unknown activation {act!r}")
    m, k = _rows(xq, "xq")
    if wq.dim() != 2:
        raise SdqError(SDQ_ERR_INVALID, f"wq must be 2-D, got shape {list(wq.shape)}")
    n, kb = wq.shape[0], -(-k // BLOCK)
    shape = (*xq.shape[:-1], n)
    dtype = out_dtype if out_dtype is not None else torch.bfloat16 if out is None else out.dtype
    if dtype not in _SOURCE:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"out must be bf16 or f32, not {dtype}")
    _demand("xq", xq, [
        ("xq", xq, (E4M3,), None), ("xs", xs, (E8M0,), (kb, m)), ("wq", wq, (E4M3,), (n, k)), ("ws", ws, (E8M0,), (-(-n // BLOCK), kb)),
        ("out", out, (dtype,), shape), ("bias", bias, (dtype,), n), ("gate", gate, (dtype,), n), ("residual", residual, (dtype,), m * n)])
    if out is None:
        out = xq.new_empty(shape, dtype=dtype)
    check(lib().sdq_fp8_matmul(xq.data_ptr(), xs.data_ptr(), m, k, wq.data_ptr(), ws.data_ptr(), n,
                               None if bias is None else bias.data_ptr(), _ACTS[act],
                               None if gate is None else gate.data_ptr(),
                               None if residual is None else residual.data_ptr(), out.data_ptr(), _SOURCE[dtype], _raw_stream(dev)))
    return out


def debug_fp8_plan(m: int, k: int, n: int, fused: bool = False, aligned: bool = True) -> dict:
    """How :func:`fp8_matmul` would run on the current device (``sdq_debug_fp8_plan``), for tests."""
    plan = (ctypes.c_int32 * 6)()
    check(lib().sdq_debug_fp8_plan(m, k, n, int(bool(fused)), int(bool(aligned)), plan))
    return dict(zip(("pair", "split", "features", "tiles", "at_once", "group"), plan))


@dataclass
class Fp8Array:
    """A weight held as e4m3 with a scale for each 128 x 128 block: what :class:`sdq.QuantizedArray`
    is for the affine form, with the same methods.  ``matmul`` quantises its activations."""
    weight: torch.Tensor
    scales: torch.Tensor

    @classmethod
    def quantize(cls, w: torch.Tensor, stream=None) -> "Fp8Array":
        return cls(*fp8_quantize_weight(w, stream))

    def dequantize(self, out_dtype=torch.bfloat16, stream=None) -> torch.Tensor:
        return fp8_dequantize(self.weight, self.scales, True, out_dtype, stream)

    def matmul(self, x: torch.Tensor, bias=None, stream=None, out=None) -> torch.Tensor:
        """``x @ weight.T`` (+ bias) in x's type or ``out``'s, x [..., k] bf16 or f32.  A bias of another
        float type is converted for the call."""
        xq, xs = fp8_quantize(x, stream)
        bias = as_result(bias, x.dtype if out is None else out.dtype, stream)
        return fp8_matmul(xq, xs, self.weight, self.scales, bias=bias, out=out, out_dtype=x.dtype if out is None else None,
                          stream=stream)

    def matmul_fused(self, x: torch.Tensor, bias=None, act=None, gate=None, residual=None, out=None,
                     stream=None) -> torch.Tensor:
        """``residual + gate * act(x @ weight.T + bias)``, rounded to bf16 once.  A bias or gate of another
        float type is converted for the call."""
        xq, xs = fp8_quantize(x, stream)
        bias, gate = (as_result(t, torch.bfloat16 if out is None else out.dtype, stream) for t in (bias, gate))
        return fp8_matmul(xq, xs, self.weight, self.scales, bias=bias, act=act, gate=gate, residual=residual, out=out,
                          stream=stream)

    def resident_bytes(self) -> int:
        return self.weight.numel() + self.scales.numel()

    @property
    def shape(self):
        return tuple(self.weight.shape)
