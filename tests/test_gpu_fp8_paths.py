"""GPU: every form in which the block-scaled product runs -- one CTA a tile, a pair, a cluster that
shares k; one tile each or several in turn; rows on 32 bytes and not; a last group of token tiles that
is smaller than the others -- each against 64 bits on every row, with the plan asked for, so that another
tile choice cannot leave a form without a test.  Tolerances as derived in test_gpu_fp8.py."""
from __future__ import annotations

import time

import pytest
import torch

import sdq
from conftest import gpu_available
from test_gpu_fp8 import check, normals, operands, product, sums_tol

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")]

PAIRS, SINGLE, SHARED = "pairs", "single CTAs", "clusters that share k"


def expect(shape, wanted, several, ragged, fused=False, aligned=None):
    m, k, n = shape
    plan = sdq.debug_fp8_plan(m, k, n, fused, n % 16 == 0 if aligned is None else aligned)
    assert wanted == (PAIRS if plan["pair"] == 2 else SINGLE if plan["split"] == 1 else SHARED), plan
    assert (plan["tiles"] > plan["at_once"]) == several, plan
    token_tiles = -(-m // (128 * plan["pair"]))
    assert (token_tiles % plan["group"] != 0) == ragged, plan


# (m, k, n), what the plan is, whether CTAs take several tiles, whether the last group is smaller
PLAIN = [
    ((300, 4096, 4096), PAIRS, False, False), ((257, 2640, 4096), PAIRS, False, False), ((300, 2640, 4099), PAIRS, False, False),
    ((129, 8192, 4099), PAIRS, False, False), ((513, 4096, 2056), PAIRS, False, False), ((700, 1024, 2048), PAIRS, False, False),
    ((1037, 2640, 4099), PAIRS, True, False), ((3000, 2576, 2048), PAIRS, True, False), ((3000, 2576, 2051), PAIRS, True, False),
    ((4796, 8192, 1008), PAIRS, True, True), ((4796, 8192, 1000), PAIRS, True, True), ((9000, 4112, 1024), PAIRS, True, True),
    ((9000, 4112, 1030), PAIRS, True, True),
    ((2100, 272, 3008), SINGLE, True, False), ((2100, 272, 3001), SINGLE, True, False), ((20000, 48, 400), SINGLE, True, False),
    ((20000, 48, 403), SINGLE, True, False), ((130000, 272, 130), SINGLE, True, True), ((130000, 272, 144), SINGLE, True, True),
    ((7, 9728, 2560), SHARED, False, False), ((100, 4112, 99), SHARED, False, False),
]


@pytest.mark.parametrize("shape,wanted,several,ragged", PLAIN)
def test_each_plan_in_bf16_and_f32(shape, wanted, several, ragged):
    m, k, n = shape
    expect(shape, wanted, several, ragged)
    ops = operands(m + k + n, m, k, n)
    want, s = product(*ops)
    bias = normals(1, n) * want.abs().mean()
    for dt, step in ((torch.bfloat16, 2.0 ** -8), (torch.float32, 2.0 ** -24)):
        b = bias.to(dt)
        room = torch.full((m * n + 64,), -7.0, device="cuda", dtype=dt)
        y = sdq.fp8_matmul(*ops, bias=b, out=room[: m * n].view(m, n))
        z = want + b.double()
        check(y, z, sums_tol(s, k) + z.abs() * (step + 2.0 ** -23))
        assert (room[m * n:] == -7).all()
    sdq.device_status()


FUSED = [((300, 4096, 4096), PAIRS, False, False), ((300, 2640, 4099), PAIRS, False, False), ((1037, 2640, 4099), PAIRS, True, False),
         ((3000, 2576, 2048), PAIRS, True, False), ((9000, 4112, 1030), PAIRS, True, True), ((2100, 272, 3008), SINGLE, True, False),
         ((2100, 272, 3001), SINGLE, True, False)]


@pytest.mark.parametrize("oy,orr", [(0, 0), (1, 1), (3, 8), (8, 0)])
@pytest.mark.parametrize("shape,wanted,several,ragged", FUSED)
def test_gate_and_residual_of_each_plan(shape, wanted, several, ragged, oy, orr):
    """y and the residual ``oy`` and ``orr`` values past 512 bytes, apart and in place; sentinels stay."""
    m, k, n = shape
    expect(shape, wanted, several, ragged, True, n % 16 == 0 and oy % 16 == 0 and orr % 16 == 0)
    ops = operands(m + n, m, k, n)
    want, s = product(*ops)
    bias, gate = (normals(6, n) * want.abs().mean()).to(torch.bfloat16), normals(7, n).to(torch.bfloat16)
    place = lambda o: torch.full((m * n + 128,), -7.0, device="cuda", dtype=torch.bfloat16)[o: o + m * n + 64]  # noqa: E731
    ry, rr = place(oy), place(orr)
    res, y = rr[: m * n].view(m, n), ry[: m * n].view(m, n)
    res.copy_(normals(8, m, n) * want.abs().mean())
    v = want + bias.double()
    z = res.double() + gate.double() * v
    tol = gate.double().abs() * (sums_tol(s, k) + v.abs() * 2.0 ** -22) + (z.abs() + (gate.double() * v).abs() * 2.0 ** -14) * 2.0 ** -8
    sdq.fp8_matmul(*ops, bias=bias, gate=gate, residual=res, out=y)
    check(y, z, tol)
    sdq.fp8_matmul(*ops, bias=bias, gate=gate, residual=res, out=res)
    check(res, z, tol)
    sdq.device_status()
    for room, t in ((ry, y), (rr, res)):
        assert (room[m * n:] == -7).all() and (t._base[: t.storage_offset()] == -7).all()


@pytest.mark.parametrize("shape,wanted,several,ragged", FUSED + [((7, 9728, 2560), SHARED, False, False),
                                                                        ((100, 4112, 99), SHARED, False, False)])
@pytest.mark.parametrize("act", ["silu", "gelu_approx"])
def test_activations_of_each_plan(shape, wanted, several, ragged, act):
    """The tolerance of an activation as in test_gpu_fp8.py."""
    m, k, n = shape
    expect(shape, wanted, several, ragged, True)
    ops = operands(m + n, m, k, n)
    want, s = product(*ops)
    bias = (normals(9, n) * want.abs().mean()).to(torch.bfloat16)
    v = want + bias.double()
    a = v * torch.sigmoid(v if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    y = sdq.fp8_matmul(*ops, bias=bias, act=act)
    check(y, a, 1.13 * (sums_tol(s, k) + v.abs() * 2.0 ** -23) + 2.0 ** -10 * (1 + v.abs()) + a.abs() * 2.0 ** -8)
    sdq.device_status()


@pytest.mark.parametrize("withhold", [1, 2, 3])
@pytest.mark.parametrize("shape,wanted,several,ragged", [
    ((300, 4096, 4096), PAIRS, False, False), ((300, 2640, 4099), PAIRS, False, False), ((9000, 4112, 1024), PAIRS, True, True),
    ((2100, 272, 3008), SINGLE, True, False), ((7, 9728, 2560), SHARED, False, False)])
def test_waits_that_run_out_in_each_plan(shape, wanted, several, ragged, withhold):
    """As test_gpu_abort.py, without a fault: each CTA withholds its first copy, or one CTA of a pair all of
    its copies; the waits give up, what was started lands, and the next call is right."""
    m, k, n = shape
    expect(shape, wanted, several, ragged)
    ops = operands(m, m, k, n)
    want = sdq.fp8_matmul(*ops)
    sdq.device_status()
    for _ in range(2):
        sdq.debug_wait_hook(20_000_000, withhold)
        try:
            t0 = time.monotonic()
            sdq.fp8_matmul(*ops)
            torch.cuda.synchronize()
            elapsed = time.monotonic() - t0
            with pytest.raises(sdq.SdqError, match="gave up"):
                sdq.device_status()
        finally:
            sdq.debug_wait_hook(0, False)
        assert elapsed < 1.0, elapsed                      # one 20 ms limit; the copies land at once
        assert torch.equal(sdq.fp8_matmul(*ops), want)
        sdq.device_status()


@pytest.mark.parametrize("act", ["silu", "gelu_approx"])
@pytest.mark.parametrize("shape,wanted", [((1, 16, 65280), SINGLE), ((3, 16, 65279), SINGLE), ((300, 4096, 65280), PAIRS), ((300, 4096, 65277), PAIRS),
                                          ((16, 8192, 1020), SHARED), ((16, 8192, 1008), SHARED)])
def test_activations_of_every_bf16_number(shape, wanted, act):
    """A product of zeros, so that the bias is the activation's exact argument: every finite bf16 number (of
    shared tiles, every 64th).  The exponential's argument, at most 64 where it matters, is rounded four times and
    its constants once each, 5 x 2^-24 of it, which gives 64 x 5 x 2^-24 ln 2 < 2^-16 of the value; exponential,
    reciprocal and products some 2^-21.  Rounding to bf16 is off by 2^-8 of a result at most, and by 2^-134 of one
    below 2^-126, where its numbers are 2^-133 apart.  Arguments below -43 and -7.6 have the value there,
    43 e^-43 < 2^-56 and 7.6 e^-43 < 2^-59."""
    m, k, n = shape
    expect(shape, wanted, wanted == PAIRS or n > 60000 and sdq.debug_fp8_plan(m, k, n, True, n % 16 == 0)["tiles"] > 148, False, True)
    every = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    every = every[every.isfinite()]
    bias = every[:n] if n > 60000 else every[5::64][:n].contiguous()
    ops = (*sdq.fp8_quantize(torch.zeros(m, k, device="cuda")), *sdq.fp8_quantize_weight(normals(1, n, k)))
    v = bias.double()
    a = v * torch.sigmoid(v if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    low, most = (-43, 2.0 ** -56) if act == "silu" else (-7.6, 2.0 ** -59)
    tol = a.abs() * (2.0 ** -8 + 2.0 ** -14) + 2.0 ** -134 + torch.where(v < low, most, 0.0)
    y = sdq.fp8_matmul(*ops, bias=bias, act=act)
    check(y, a.expand(m, n), tol.expand(m, n))
    sdq.device_status()
