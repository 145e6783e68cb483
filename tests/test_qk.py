"""The refusals of the query / key preparation without a GPU, through the C ABI."""
from __future__ import annotations

import ctypes

import pytest
import torch

import sdq
from conftest import gpu_available
from sdq import _abi


def _call(dtype=1, b=2, n=3, d=64, qh=4, kh=2, vh=2, ohq=None, q=0x1000, qo=0x2000, st=None, rope=64, rows=3, cos=0x7000,
          pos=0, pos64=0, w=0x8000, eps=1e-6, no_v=False, no_vout=False, zero=None):
    def h(ptr, heads, token_stride=None):
        return _abi.SdqHeads(ptr, heads, n * heads * d, heads * d if token_stride is None else token_stride, d)

    qi, ki, vi = h(q, qh, st), h(0x3000, kh), h(0x4000, vh)
    qo, ko, vo = h(qo, qh if ohq is None else ohq), h(0x5000, kh), h(0x6000, vh)
    r = ctypes.byref
    if zero:
        setattr(qo, zero, 0)
    return _abi.lib().sdq_qk_norm_rope(r(qi), r(ki), None if no_v else r(vi), r(qo), r(ko), None if no_vout else r(vo), dtype,
                                       b, n, d, w, w, eps, cos, cos, rows, rope, 1, pos or None, pos64, n, None)


@pytest.mark.parametrize("kwargs,code,needle", [
    (dict(dtype=2), _abi.SDQ_ERR_UNSUPPORTED, "bf16 or f32"),
    (dict(d=60), _abi.SDQ_ERR_UNSUPPORTED, "head_dim"),
    (dict(d=264), _abi.SDQ_ERR_UNSUPPORTED, "head_dim"),
    (dict(rope=72), _abi.SDQ_ERR_UNSUPPORTED, "rope_dim"),
    (dict(rope=8), _abi.SDQ_ERR_UNSUPPORTED, "rope_dim"),
    (dict(rope=80), _abi.SDQ_ERR_UNSUPPORTED, "rope_dim"),
    (dict(b=-1), _abi.SDQ_ERR_INVALID, "batch and tokens"),
    (dict(b=1 << 16, n=1 << 16), _abi.SDQ_ERR_INVALID, "batch and tokens"),
    (dict(eps=-1.0), _abi.SDQ_ERR_INVALID, "eps"),
    (dict(eps=float("nan")), _abi.SDQ_ERR_INVALID, "eps"),
    (dict(ohq=5), _abi.SDQ_ERR_INVALID, "heads"),
    (dict(qh=-1), _abi.SDQ_ERR_INVALID, "heads"),
    (dict(no_vout=True), _abi.SDQ_ERR_INVALID, "v_out"),
    (dict(q=0), _abi.SDQ_ERR_INVALID, "have data"),
    (dict(q=0x1008), _abi.SDQ_ERR_INVALID, "aligned"),
    (dict(st=4 * 64 + 4), _abi.SDQ_ERR_INVALID, "aligned"),
    (dict(zero="batch_stride"), _abi.SDQ_ERR_INVALID, "q's output has a stride of 0"),
    (dict(zero="token_stride"), _abi.SDQ_ERR_INVALID, "q's output has a stride of 0"),
    (dict(zero="head_stride"), _abi.SDQ_ERR_INVALID, "q's output has a stride of 0"),
    (dict(w=0x8008), _abi.SDQ_ERR_INVALID, "norm weight"),
    (dict(cos=0), _abi.SDQ_ERR_INVALID, "cos and sin"),
    (dict(cos=0x7004), _abi.SDQ_ERR_INVALID, "cos or sin"),
    (dict(rows=2), _abi.SDQ_ERR_INVALID, "2 rows for 3 tokens"),
    (dict(pos=0x9004, pos64=1), _abi.SDQ_ERR_INVALID, "positions"),
])
def test_refusals(kwargs, code, needle):
    assert _call(**kwargs) == code
    assert needle in _abi.last_error()


@pytest.mark.parametrize("kwargs", [dict(b=0), dict(n=0), dict(qh=0, kh=0, no_v=True)])
def test_nothing_to_do_is_done_without_a_device(kwargs):
    assert _call(**kwargs) == _abi.SDQ_OK


@pytest.mark.skipif(gpu_available(), reason="checks the no-device path")
def test_no_cpu_fallback():
    assert _call() == _abi.SDQ_ERR_CUDA
    x = torch.zeros(1, 2, 4, 64)
    with pytest.raises(sdq.SdqError, match="no CPU fallback"):
        sdq.qk_norm_rope(x, x, x)


@pytest.mark.parametrize("kwargs", [dict(n=0, cos=0, rows=0), dict(b=0, cos=0, rows=0), dict(qh=0, kh=0, no_v=True, cos=0, rows=0)])
def test_nothing_to_do_needs_no_tables(kwargs):
    assert _call(**kwargs) == _abi.SDQ_OK


@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")
def test_no_tokens_with_an_empty_part_of_the_tables():
    """As a joint sequence's stream that holds nothing gives them: cos[0:0] has no address."""
    q = torch.zeros(1, 0, 2, 64, device="cuda", dtype=torch.bfloat16)
    w, table = torch.ones(64, device="cuda", dtype=torch.bfloat16), torch.zeros(5, 32, device="cuda")
    joint = torch.full((3, 1, 2, 5, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    got = sdq.qk_norm_rope(q, q, q, w, w, table[0:0], table[0:0], out=tuple(joint[:, :, :, 0:0]))
    assert all(t.shape == (1, 2, 0, 64) for t in got) and (joint == 7).all()
