"""Block-scaled e4m3 without a GPU: the oracle's codes against torch's own conversion, and the
refusals of the fp8 entry points, through the C ABI and through the package."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import oracle as O
import sdq
from conftest import gpu_available
from sdq import _abi


def test_oracle_codes_equal_torchs_conversion():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    got = O.e4m3_decode(codes)
    assert np.array_equal(got, want, equal_nan=True)
    # every finite code, every midpoint between neighbours, and a step either side of each
    v = O.e4m3_values()
    mid = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9)]).astype(np.float32)
    x = np.concatenate([x, -x, np.float32([0.0, -0.0])])
    got = O.e4m3_encode(x.astype(np.float64))
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(got, want)


def test_oracle_scales_are_the_least_power_of_two():
    for a, e in ((448.0, 0), (448.0000001, 1), (224.0, -1), (225.0, 0), (1.75, -8), (1.7500001, -7), (0.0, -126), (1e-40, -126)):
        q, byte = O.fp8_quantize(np.array([[a] + [0.0] * 15]))
        assert int(byte[0, 0]) - 127 == e
    q, byte = O.fp8_quantize(np.array([[1.0, np.inf] + [0.0] * 14]))
    assert byte[0, 0] == 255 and (q == 0x7F).all()


def _p(v):
    return ctypes.c_void_p(v) if v else None


def _mm(xq=0x1000, xs=0x2000, m=4, k=128, wq=0x3000, ws=0x4000, n=64, bias=0, act=0, gate=0, res=0, y=0x5000, ydt=1):
    return _abi.lib().sdq_fp8_matmul(_p(xq), _p(xs), m, k, _p(wq), _p(ws), n, _p(bias), act, _p(gate), _p(res), _p(y), ydt, None)


@pytest.mark.parametrize("kwargs,code,needle", [
    (dict(m=-1), _abi.SDQ_ERR_INVALID, "m (rows of x)"),
    (dict(m=1 << 31), _abi.SDQ_ERR_INVALID, "m (rows of x)"),
    (dict(n=0), _abi.SDQ_ERR_INVALID, "n (rows"),
    (dict(k=0), _abi.SDQ_ERR_INVALID, "k must be"),
    (dict(k=120), _abi.SDQ_ERR_INVALID, "multiple of 16"),
    (dict(act=7), _abi.SDQ_ERR_INVALID, "act must be"),
    (dict(ydt=2), _abi.SDQ_ERR_UNSUPPORTED, "y must be"),
    (dict(ydt=0, act=2), _abi.SDQ_ERR_UNSUPPORTED, "bias only"),
    (dict(ydt=0, res=0x9000), _abi.SDQ_ERR_UNSUPPORTED, "bias only"),
    (dict(xq=0), _abi.SDQ_ERR_INVALID, "non-null"),
    (dict(ws=0), _abi.SDQ_ERR_INVALID, "non-null"),
    (dict(xq=0x1008), _abi.SDQ_ERR_INVALID, "misaligned"),
    (dict(wq=0x3001), _abi.SDQ_ERR_INVALID, "misaligned"),
    (dict(y=0x5001), _abi.SDQ_ERR_INVALID, "misaligned"),
    (dict(ydt=0, y=0x5000, bias=0x6002), _abi.SDQ_ERR_INVALID, "misaligned"),
    (dict(res=0x5010), _abi.SDQ_ERR_INVALID, "overlaps"),
])
def test_matmul_refusals(kwargs, code, needle):
    assert _mm(**kwargs) == code
    assert needle in _abi.last_error()


def test_quantize_refusals():
    L = _abi.lib()
    for f, what in ((L.sdq_fp8_quantize, "m (rows)"), (L.sdq_fp8_quantize_weight, "n (rows")):
        call = lambda x=0x1000, dt=1, r=4, k=128, q=0x2000, s=0x3000: f(_p(x), dt, r, k, _p(q), _p(s), None)  # noqa: E731
        for kw, code, needle in ((dict(r=-1), _abi.SDQ_ERR_INVALID, what), (dict(k=8), _abi.SDQ_ERR_INVALID, "multiple of 16"),
                                 (dict(k=-16), _abi.SDQ_ERR_INVALID, "k must be"), (dict(dt=2), _abi.SDQ_ERR_UNSUPPORTED, "bf16 or f32"),
                                 (dict(x=0), _abi.SDQ_ERR_INVALID, "non-null"), (dict(s=0), _abi.SDQ_ERR_INVALID, "non-null"),
                                 (dict(x=0x1008), _abi.SDQ_ERR_INVALID, "misaligned"), (dict(q=0x2004), _abi.SDQ_ERR_INVALID, "misaligned")):
            assert call(**kw) == code and needle in _abi.last_error(), kw
    call = lambda q=0x1000, s=0x2000, r=4, k=128, w=0, o=0x3000, dt=1: L.sdq_fp8_dequantize(_p(q), _p(s), r, k, w, _p(o), dt, None)  # noqa: E731
    for kw, code in ((dict(r=-1), _abi.SDQ_ERR_INVALID), (dict(k=24), _abi.SDQ_ERR_INVALID), (dict(dt=2), _abi.SDQ_ERR_UNSUPPORTED),
                     (dict(o=0), _abi.SDQ_ERR_INVALID), (dict(o=0x3008), _abi.SDQ_ERR_INVALID)):
        assert call(**kw) == code, kw


def test_nothing_to_do_is_done_without_a_device():
    L = _abi.lib()
    assert _mm(m=0, xq=0, xs=0, y=0) == _abi.SDQ_OK
    assert L.sdq_fp8_quantize(None, 1, 0, 128, None, None, None) == _abi.SDQ_OK
    assert L.sdq_fp8_dequantize(None, None, 0, 128, 0, None, 1, None) == _abi.SDQ_OK


@pytest.mark.skipif(gpu_available(), reason="checks the no-device path")
def test_no_cpu_fallback():
    assert _mm() == _abi.SDQ_ERR_CUDA and _abi.last_error()
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    for call in (lambda: sdq.fp8_quantize(x), lambda: sdq.fp8_quantize_weight(x), lambda: sdq.Fp8Array.quantize(x)):
        with pytest.raises(sdq.SdqError, match="no CPU fallback"):
            call()


def test_plan_refusals():
    for args, needle in (((0, 128, 64), "m (rows of x)"), ((4, 0, 64), "k must be"), ((4, 120, 64), "multiple of 16"), ((4, 128, 0), "n (rows"),
                         ((4, 128, 60), "not aligned")):
        with pytest.raises(sdq.SdqError) as e:
            sdq.debug_fp8_plan(*args)
        assert e.value.code == _abi.SDQ_ERR_INVALID and needle in str(e.value)
