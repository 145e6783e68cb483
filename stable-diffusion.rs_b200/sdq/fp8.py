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

from dataclasses import dataclass

import torch

from ._abi import SDQ_BF16, SDQ_ERR_INVALID, SDQ_ERR_UNSUPPORTED, SDQ_F32, SdqError, check, lib

#: Values that share a scale, along a row (activations) or both ways (weights).
BLOCK = 128

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
_SOURCE = {torch.bfloat16: SDQ_BF16, torch.float32: SDQ_F32}
_current_device = torch.cuda.current_device


def _raw_stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _elsewhere(fn, device, stream, *args, **kw):
    """``fn`` again with ``stream`` current (allocations included), or on another device."""
    if stream is not None:
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=device)
        if stream.device != device:
            raise SdqError(SDQ_ERR_INVALID, f"a stream of {stream.device} cannot run work on {device}")
        with torch.cuda.device(device), torch.cuda.stream(stream):
            return fn(*args, **kw)
    with torch.cuda.device(device):
        return fn(*args, **kw)


def _device_of(name: str, first: torch.Tensor, **others) -> torch.device:
    """The device that every tensor given lies on; they must be contiguous device tensors."""
    device = first.device
    if device.type != "cuda":
        raise SdqError(SDQ_ERR_INVALID, "libsdq takes device tensors (no CPU fallback)")
    if not first.is_contiguous():
        raise SdqError(SDQ_ERR_INVALID, f"libsdq takes contiguous row-major tensors; {name} is not")
    for n, t in others.items():
        if t is None:
            continue
        if t.device != device:
            raise SdqError(SDQ_ERR_INVALID, f"{n} is on {t.device}, {name} on {device}")
        if not t.is_contiguous():
            raise SdqError(SDQ_ERR_INVALID, f"libsdq takes contiguous row-major tensors; {n} is not")
    return device


def _want(name: str, t: torch.Tensor, dtype, shape) -> None:
    if t.dtype is not dtype:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"{name} must be {dtype}, not {t.dtype}")
    if tuple(t.shape) != shape:
        raise SdqError(SDQ_ERR_INVALID, f"{name} must have shape {list(shape)}, not {list(t.shape)}")


def _rows(x: torch.Tensor, name: str):
    """(rows, width) of a tensor whose last axis is the inner one."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise SdqError(SDQ_ERR_INVALID, f"{name} needs an inner axis of at least one value, got shape {list(x.shape)}")
    k = x.shape[-1]
    return x.numel() // k, k


def _source(t: torch.Tensor, name: str) -> int:
    code = _SOURCE.get(t.dtype)
    if code is None:
        raise SdqError(SDQ_ERR_UNSUPPORTED, f"{name} must be bf16 or f32, not {t.dtype}")
    return code


def fp8_quantize(x: torch.Tensor, stream=None):
    """Activations x [..., k] (bf16 or f32) -> (xq [..., k] e4m3, xs [ceil(k / 128), rows] e8m0),
    rows the product of the leading axes (``sdq_fp8_quantize``).  k is a multiple of 16."""
    dev = _device_of("x", x)
    if stream is not None or dev.index != _current_device():
        return _elsewhere(fp8_quantize, dev, stream, x)
    dt = _source(x, "x")
    m, k = _rows(x, "x")
    xq = torch.empty_like(x, dtype=E4M3)
    xs = torch.empty((-(-k // BLOCK), m), dtype=E8M0, device=dev)
    check(lib().sdq_fp8_quantize(x.data_ptr(), dt, m, k, xq.data_ptr(), xs.data_ptr(), _raw_stream(dev)))
    return xq, xs


def fp8_quantize_weight(w: torch.Tensor, stream=None):
    """A weight w [n, k] (bf16 or f32) -> (wq [n, k] e4m3, ws [ceil(n / 128), ceil(k / 128)] e8m0)
    (``sdq_fp8_quantize_weight``).  k is a multiple of 16."""
    dev = _device_of("w", w)
    if stream is not None or dev.index != _current_device():
        return _elsewhere(fp8_quantize_weight, dev, stream, w)
    dt = _source(w, "w")
    if w.dim() != 2:
        raise SdqError(SDQ_ERR_INVALID, f"fp8_quantize_weight wants a 2-D weight, got shape {list(w.shape)}")
    n, k = w.shape
    wq = torch.empty((n, k), dtype=E4M3, device=dev)
    ws = torch.empty((-(-n // BLOCK), -(-k // BLOCK)), dtype=E8M0, device=dev)
    check(lib().sdq_fp8_quantize_weight(w.data_ptr(), dt, n, k, wq.data_ptr(), ws.data_ptr(), _raw_stream(dev)))
    return wq, ws


def fp8_dequantize(q: torch.Tensor, scales: torch.Tensor, weight: bool, out_dtype=torch.bfloat16, stream=None):
    """The values that e4m3 codes and their scales stand for, rounded once (``sdq_fp8_dequantize``).
    ``weight`` says which scales they are: a weight's 128 x 128 blocks or an activation's groups."""
    dev = _device_of("q", q, scales=scales)
    if stream is not None or dev.index != _current_device():
        return _elsewhere(fp8_dequantize, dev, stream, q, scales, weight, out_dtype)
    rows, k = _rows(q, "q")
    kb = -(-k // BLOCK)
    _want("q", q, E4M3, tuple(q.shape))
    _want("scales", scales, E8M0, (-(-rows // BLOCK), kb) if weight else (kb, rows))
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
    dev = _device_of("xq", xq, xs=xs, wq=wq, ws=ws, bias=bias, gate=gate, residual=residual, out=out)
    if stream is not None or dev.index != _current_device():
        return _elsewhere(fp8_matmul, dev, stream, xq, xs, wq, ws, bias, act, gate, residual, out, out_dtype)
    from . import _ACTS

    if act not in _ACTS:
        raise SdqError(SDQ_ERR_INVALID, f"unknown activation {act!r}")
    m, k = _rows(xq, "xq")
    if wq.dim() != 2:
        raise SdqError(SDQ_ERR_INVALID, f"wq must be 2-D, got shape {list(wq.shape)}")
    n, kb = wq.shape[0], -(-k // BLOCK)
    shape = (*xq.shape[:-1], n)
    _want("xq", xq, E4M3, tuple(xq.shape))
    _want("xs", xs, E8M0, (kb, m))
    _want("wq", wq, E4M3, (n, k))
    _want("ws", ws, E8M0, (-(-n // BLOCK), kb))
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16 if out_dtype is None else out_dtype, device=dev)
    dt = _source(out, "out")
    _want("out", out, out.dtype if out_dtype is None else out_dtype, shape)
    for name, t, count in (("bias", bias, n), ("gate", gate, n), ("residual", residual, m * n)):
        if t is not None and (t.numel() != count or t.dtype is not out.dtype):
            raise SdqError(SDQ_ERR_INVALID, f"{name} must hold {count} values of {out.dtype}, not {t.numel()} of {t.dtype}")
    check(lib().sdq_fp8_matmul(xq.data_ptr(), xs.data_ptr(), m, k, wq.data_ptr(), ws.data_ptr(), n,
                               None if bias is None else bias.data_ptr(), _ACTS[act],
                               None if gate is None else gate.data_ptr(),
                               None if residual is None else residual.data_ptr(), out.data_ptr(), dt, _raw_stream(dev)))
    return out


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
        """``x @ weight.T`` (+ bias) in x's type, x [..., k] bf16 or f32."""
        xq, xs = fp8_quantize(x, stream)
        return fp8_matmul(xq, xs, self.weight, self.scales, bias=bias, out=out, out_dtype=x.dtype, stream=stream)

    def matmul_fused(self, x: torch.Tensor, bias=None, act=None, gate=None, residual=None, out=None,
                     stream=None) -> torch.Tensor:
        """``residual + gate * act(x @ weight.T + bias)``, rounded to bf16 once."""
        xq, xs = fp8_quantize(x, stream)
        return fp8_matmul(xq, xs, self.weight, self.scales, bias=bias, act=act, gate=gate, residual=residual, out=out,
                          stream=stream)

    def resident_bytes(self) -> int:
        return self.weight.numel() + self.scales.numel()

    @property
    def shape(self):
        return tuple(self.weight.shape)
