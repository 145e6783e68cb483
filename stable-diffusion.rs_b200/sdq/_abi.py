"""ctypes binding of libsdq.so (the C ABI declared in include/sdq.h).

The library is loaded from the package directory's parent
(``stable-diffusion.rs_b200/libsdq.so``), where ``build.py`` writes it.  There
is no fallback: if the library is missing or the device is not an sm_100 part,
every call raises :class:`SdqError`.
"""
from __future__ import annotations

import contextlib
import ctypes
import os

import torch  # (the shortcut below links against its libraries)

try:
    from . import _native
except ImportError:
    _native = None

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("SDQ_LIB", os.path.join(os.path.dirname(HERE), "libsdq.so"))

SDQ_OK = 0
SDQ_ERR_INVALID = 1
SDQ_ERR_UNSUPPORTED = 2
SDQ_ERR_CUDA = 3
SDQ_ERR_TIMEOUT = 4
SDQ_ERR_NCCL = 5

SDQ_F32 = 0
SDQ_BF16 = 1
SDQ_F16 = 2


class SdqHeads(ctypes.Structure):
    """``sdq_heads``: head vectors [batch, tokens, heads, head_dim], strides in elements."""
    _fields_ = [("data", ctypes.c_void_p), ("heads", ctypes.c_int64), ("batch_stride", ctypes.c_int64),
                ("token_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


#: Every symbol include/sdq.h declares, with (restype, argtypes).
_p, _i64, _i32, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
SIGNATURES = {
    "sdq_last_error": (ctypes.c_char_p, []),
    "sdq_abi_version": (_i32, []),
    "sdq_quantize": (_i32, [_p, _i32, _i64, _i64, _i32, _i32, ctypes.c_char_p, _p, _p, _p, _i32, _p]),
    "sdq_dequantize": (_i32, [_p, _p, _p, _i32, _i64, _i64, _i32, _i32, ctypes.c_char_p, _p, _i32, _p]),
    "sdq_quantized_matmul": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p, _i32, _i64, _i32, _i32, _i32,
                                    ctypes.c_char_p, _p, _p, _i32, _p]),
    "sdq_quantized_matmul_host": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p, _i32, _i64, _i32, _i32, _p, _p,
                                         _i32, _p, _p, _i64, _p]),
    "sdq_quantized_matmul_epilogue": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p, _i32, _i64, _i32, _i32,
                                             _p, _i32, _p, _p, _p, _i32, _p]),
    "sdq_fp8_quantize": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p]),
    "sdq_fp8_quantize_weight": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p]),
    "sdq_fp8_dequantize": (_i32, [_p, _p, _i64, _i64, _i32, _p, _i32, _p]),
    "sdq_fp8_matmul": (_i32, [_p, _p, _i64, _i64, _p, _p, _i64, _p, _i32, _p, _p, _p, _i32, _p]),
    "sdq_qk_norm_rope": (_i32, [_p, _p, _p, _p, _p, _p, _i32, _i64, _i64, _i32, _p, _p, ctypes.c_float, _p, _p,
                                _i64, _i32, _i32, _p, _i32, _i64, _p]),
    "sdq_resident_bytes": (_sz, [_i64, _i64, _i32, _i32, _i32]),
    "sdq_gguf_bytes": (_sz, [_i32, _i64]),
    "sdq_seeded_normals": (_i32, [ctypes.c_uint64, _i64, _p, _p]),
    "sdq_gguf_quantize": (_i32, [_p, _i32, _i64, _i64, _i32, _i32, _p, _p, _p, _i32, _p]),
    "sdq_gguf_dequantize": (_i32, [_p, _i32, _i64, _p, _i32, _p]),
    "sdq_device_status": (_i32, [_p]),
    "sdq_debug_wait_hook": (_i32, [ctypes.c_uint64, _i32, _p]),
    "sdq_debug_fp8_plan": (_i32, [_i64, _i64, _i64, _i32, _i32, _p]),
    "sdq_comm_unique_id": (_i32, [_p]),
    "sdq_comm_init": (_i32, [_p, _i32, _i32, ctypes.POINTER(ctypes.c_void_p)]),
    "sdq_comm_destroy": (_i32, [_p]),
    "sdq_comm_output": (_i32, [_p, _i64, _i64, ctypes.POINTER(ctypes.c_void_p)]),
    "sdq_quantized_matmul_sharded": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p, _i32, _i64, _i32, _i32,
                                            _p, _p, _p, _i32, _p, _p]),
    "sdq_quantized_matmul_sharded_static": (_i32, [_p, _i32, _i64, _i64, _p, _p, _p, _i32, _i64, _i32,
                                                   _i32, _p, _p, _i32, _p, _p]),
}


class SdqError(RuntimeError):
    """A nonzero status from libsdq, with the library's per-thread message."""

    def __init__(self, code: int, message: str):
        super().__init__(f"libsdq error {code}: {message}")
        self.code = code
        self.message = message


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise SdqError(SDQ_ERR_CUDA, f"{LIB_PATH} is missing; build it with "
                                         "`python stable-diffusion.rs_b200/build.py`")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _lib = L
        if _native is not None:
            _native.bind(*(ctypes.cast(getattr(L, f), ctypes.c_void_p).value for f in (
                "sdq_fp8_quantize", "sdq_fp8_quantize_weight", "sdq_fp8_matmul", "sdq_qk_norm_rope")))
    return _lib


def native(name: str):
    """The C++ shortcut of an entry point (binding/sdq_native.cpp): it returns None, having done
    nothing, unless the call is an ordinary one.  Where it was not built, ctypes makes every call."""
    return getattr(_native, name) if _native is not None else lambda *args: None


def last_error() -> str:
    return lib().sdq_last_error().decode("utf-8", "replace")


def check(rc: int) -> None:
    if rc != SDQ_OK:
        raise SdqError(rc, last_error())


@contextlib.contextmanager
def on(stream, device: torch.device):
    """``device`` current and, where it is not None, ``stream`` (a torch stream or a raw handle).  What is
    copied, allocated and dropped between kernels then belongs to the stream that these run on: the
    allocator hands a dropped block on at once, in the order of that stream."""
    if device.type != "cuda":
        yield
        return
    with torch.cuda.device(device):
        if stream is None:
            yield
            return
        if not isinstance(stream, torch.cuda.Stream):
            handle = stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)
            # (torch takes a handle of 0, the default stream's, for none and hands out a stream of its own.)
            stream = torch.cuda.ExternalStream(handle) if handle else torch.cuda.default_stream()
        if stream.device_index != torch.cuda.current_device():
            raise SdqError(SDQ_ERR_INVALID, f"a stream of {stream.device} cannot run work on {device}")
        with torch.cuda.stream(stream):
            yield


def as_result(t, dtype: torch.dtype, stream=None):
    """A bias or gate (or None) in the result's type, which is what the kernels read."""
    if t is None or t.dtype == dtype or not t.is_floating_point():
        return t
    with on(stream, t.device):
        return t.to(dtype)
