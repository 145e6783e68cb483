"""GPU: block-scaled e4m3 against the oracle and 64-bit sums.

Codes and scales are compared for equality: dividing by a power of two is exact, so each value has
one right code.  A product's tolerance counts its roundings.  Products of two 4-bit significands and
of two powers of two are exact in f32; the sum of K of them is taken 32 at a time and each addition
into the f32 accumulator, rounded or truncated, is off by at most 2^-23 of the partial sum, the sum
inside one step by at most as much for each of its 32 terms' alignment.  With S = sum |x w| bounding
every partial sum:  |error| <= (K/32 + 32) 2^-23 S, and 2^-8 of the value for the bf16 rounding.
"""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import oracle as O
import sdq
from conftest import gpu_available

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")]

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def u8(t):
    return t.view(torch.uint8).cpu().numpy()


def normals(seed, *shape):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g)


def spread(seed, m, k):
    """Normals whose rows and columns differ by powers of two over a wide range."""
    g = torch.Generator("cuda").manual_seed(seed + 1000)
    x = normals(seed, m, k)
    x *= torch.exp2(torch.randint(-20, 20, (m, 1), device="cuda", generator=g).float())
    return x * torch.exp2(torch.randint(-3, 3, (1, k), device="cuda", generator=g).float())


SHAPES = [(1, 16), (1, 128), (3, 144), (4, 256), (5, 112), (33, 272), (129, 128), (130, 400), (257, 2576)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k", SHAPES)
def test_quantize_matches_the_oracle(m, k, dtype):
    x = spread(m + k, m, k).to(DT[dtype])
    q, s = sdq.fp8_quantize(x)
    assert q.shape == (m, k) and s.shape == (-(-k // 128), m)
    wq, ws = O.fp8_quantize(x.double().cpu().numpy())
    assert np.array_equal(u8(s), ws)
    assert np.array_equal(u8(q), wq)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,k", SHAPES)
def test_quantize_weight_matches_the_oracle(n, k, dtype):
    w = spread(n + k, n, k).to(DT[dtype])
    q, s = sdq.fp8_quantize_weight(w)
    wq, ws = O.fp8_quantize_weight(w.double().cpu().numpy())
    assert np.array_equal(u8(s), ws)
    assert np.array_equal(u8(q), wq)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_edges(dtype):
    """Groups of zeros, of the smallest and the largest numbers, at the border of two scales, with
    exact ties, and with an infinity or a NaN (which make their own group NaN and no other)."""
    fi = torch.finfo(DT[dtype])
    x = torch.zeros(12, 256)
    x[1] = fi.smallest_normal
    x[2, 5] = fi.max
    x[3, :8] = torch.tensor([448.0, 432.0, 17.0, 19.0, -21.0, 2.0 ** -10, 3 * 2.0 ** -10, -(2.0 ** -10)])
    x[4, 0], x[4, 1] = 450.0, 1.0
    x[5, 128] = float("inf")
    x[6, 3] = float("nan")
    x[7, :] = -float("inf")
    x[8, 0], x[8, 200] = -0.0, 2.0 ** -130
    x[9] = torch.linspace(-448, 448, 256)
    x[10] = fi.tiny * 0.5 if dtype == "f32" else 2.0 ** -133
    x = x.to(DT[dtype]).cuda()
    q, s = sdq.fp8_quantize(x)
    wq, ws = O.fp8_quantize(x.double().cpu().numpy())
    assert np.array_equal(u8(s), ws) and np.array_equal(u8(q) & 0x7F, wq & 0x7F)
    live = wq != 0x7F
    assert np.array_equal(u8(q)[live], wq[live])
    q, s = sdq.fp8_quantize_weight(x)
    wq, ws = O.fp8_quantize_weight(x.double().cpu().numpy())
    assert np.array_equal(u8(s), ws) and (u8(q) & 0x7F == wq & 0x7F).all()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("weight", [False, True])
def test_dequantize_matches_the_oracle(weight, out):
    m, k = 131, 272
    q = torch.randint(0, 256, (m, k), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    kb, nb = 3, 2
    # every byte of e8m0 that keeps the value in range, 0 (2^-127), and 255 (NaN)
    s = torch.randint(0, 240, (nb, kb) if weight else (kb, m), device="cuda", dtype=torch.uint8)
    s.view(-1)[:3] = torch.tensor([0, 255, 1], dtype=torch.uint8)
    got = sdq.fp8_dequantize(q, s.view(torch.float8_e8m0fnu), weight, out)
    want = torch.from_numpy(O.fp8_dequantize(u8(q), u8(s), weight)).to(out)
    assert torch.equal(got.cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))


def product(xq, xs, wq, ws):
    """(sum of x w, sum of |x w|) in f64 on the device."""
    x = xq.double() * xs.double().t().repeat_interleave(128, 1)[:, : xq.shape[1]]
    w = wq.double() * ws.double().repeat_interleave(128, 0).repeat_interleave(128, 1)[: wq.shape[0], : wq.shape[1]]
    return x @ w.t(), x.abs() @ w.abs().t()


def operands(seed, m, k, n):
    return (*sdq.fp8_quantize(spread(seed, m, k)), *sdq.fp8_quantize_weight(spread(seed + 7, n, k)))


def sums_tol(s, k):
    return (k / 32 + 32) * 2.0 ** -23 * s


def check(got, want, tol):
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])


# m: one row, a tile's edges, pairs' edges; n and k ragged and whole.
MM = [(1, 16, 1), (1, 128, 128), (2, 256, 130), (3, 144, 8), (5, 2576, 333), (8, 512, 640), (9, 400, 257), (16, 1024, 256),
      (17, 128, 100), (33, 272, 515), (64, 640, 128), (65, 1040, 384), (128, 512, 129), (129, 4096, 256), (224, 256, 512),
      (225, 768, 1000), (333, 2576, 499), (512, 1024, 2048), (1000, 208, 3001),
      # few tiles and a long K, shared by 2, 4 or 8 CTAs; steps that do not divide evenly, a ragged last one
      (1, 9728, 1024), (3, 2064, 24), (16, 8192, 40), (100, 4112, 99), (128, 4096, 512), (200, 8080, 130), (7, 9728, 2560),
      (300, 6000, 64), (1, 16384, 8)]


@pytest.mark.parametrize("m,k,n", MM)
def test_matmul_matches_64_bits(m, k, n):
    ops = operands(m + k + n, m, k, n)
    want, s = product(*ops)
    y = sdq.fp8_matmul(*ops)
    sdq.device_status()
    check(y, want, want.abs() * 2.0 ** -8 + sums_tol(s, k))
    y = sdq.fp8_matmul(*ops, out_dtype=torch.float32)
    sdq.device_status()
    check(y, want, want.abs() * 2.0 ** -24 + sums_tol(s, k))


@pytest.mark.parametrize("m,k,n", [(1, 512, 256), (7, 400, 130), (40, 272, 300), (300, 640, 1024), (226, 144, 77), (5, 8192, 96),
                                   (130, 4096, 51)])
@pytest.mark.parametrize("act", [None, "silu", "gelu_approx"])
def test_output_stage(m, k, n, act):
    """bias, activation, gate and residual, all of them and in place, against the chain in f64.  The
    activations' slopes are at most 1.13, their own error at most 2^-10 (1 + |v|) (hardware tanh 2^-11
    relative, __expf and the fast division 2^-20), times the gate."""
    ops = operands(m * n + k, m, k, n)
    want, s = product(*ops)
    scale = want.abs().mean()
    ops = (ops[0], ops[1], ops[2], ops[3])
    bias = (normals(1, n) * scale).to(torch.bfloat16)
    gate, res = (normals(2, n) / scale).to(torch.bfloat16), normals(3, m, n).to(torch.bfloat16)
    v = want + bias.double()
    tol_v = sums_tol(s, k) + v.abs() * 2.0 ** -23
    if act == "silu":
        a = v * torch.sigmoid(v)
    elif act:
        a = v * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    else:
        a = v
    tol_a = 1.13 * tol_v + (2.0 ** -10 * (1 + v.abs()) if act else 0)
    y = sdq.fp8_matmul(*ops, bias=bias, act=act)
    check(y, a, tol_a + a.abs() * 2.0 ** -8)
    z = res.double() + gate.double() * a
    tol = tol_a * gate.double().abs() + (z.abs() + (gate.double() * a).abs() * 2.0 ** -14) * 2.0 ** -8
    check(sdq.fp8_matmul(*ops, bias=bias, act=act, gate=gate, residual=res), z, tol)
    r = res.clone()
    assert sdq.fp8_matmul(*ops, bias=bias, act=act, gate=gate, residual=r, out=r) is r
    check(r, z, tol)
    sdq.device_status()


@pytest.mark.parametrize("m", [1, 6, 40, 300])
def test_f32_result_with_an_f32_bias(m):
    k, n = 272, 130
    ops = operands(m, m, k, n)
    bias = normals(4, n)
    want, s = product(*ops)
    y = sdq.fp8_matmul(*ops, bias=bias, out_dtype=torch.float32)
    check(y, want + bias.double(), sums_tol(s, k) + (want + bias.double()).abs() * 2.0 ** -23)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_scales_far_apart_and_codes_of_any_value(m):
    """Scales from 2^-40 to 2^40 in no order, every finite code, operands that no quantiser made."""
    k, n = 400, 200
    g = torch.Generator("cuda").manual_seed(m)
    code = lambda r: (lambda c: torch.where((c & 0x7F) == 0x7F, c - 1, c))(torch.randint(0, 256, (r, k), device="cuda", generator=g)).to(torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    byte = lambda *s: torch.randint(87, 168, s, device="cuda", generator=g).to(torch.uint8).view(torch.float8_e8m0fnu)  # noqa: E731
    ops = (code(m), byte(4, m), code(n), byte(2, 4))
    want, s = product(*ops)
    check(sdq.fp8_matmul(*ops, out_dtype=torch.float32), want, want.abs() * 2.0 ** -24 + sums_tol(s, k))
    check(sdq.fp8_matmul(*ops), want, want.abs() * 2.0 ** -8 + sums_tol(s, k))


@pytest.mark.parametrize("m", [2, 20, 300])
def test_nan_stays_in_its_row_and_its_features(m):
    """A NaN group of an activation makes that token's row NaN and nothing else; a NaN block of a
    weight its 128 features."""
    k, n = 512, 300
    x, w = normals(5, m, k), normals(6, n, k)
    x[1, 130] = float("inf")
    xq, xs = sdq.fp8_quantize(x)
    wq, ws = sdq.fp8_quantize_weight(w)
    y = sdq.fp8_matmul(xq, xs, wq, ws)
    nan = torch.isnan(y)
    assert nan[1].all() and nan.sum() == n
    w[140, 3] = float("nan")
    x[1, 130] = 0
    y = sdq.fp8_matmul(*sdq.fp8_quantize(x), *sdq.fp8_quantize_weight(w))
    nan = torch.isnan(y)
    assert nan[:, 128:256].all() and nan.sum() == m * 128


@pytest.mark.parametrize("act", [None, "silu", "gelu_approx"])
@pytest.mark.parametrize("m,k,n", [(40, 144, 320), (40, 144, 77), (8, 8192, 64), (8, 8192, 51)])
def test_one_feature_out_of_range(m, k, n, act):
    """A NaN, an infinity and numbers near f32's end in the bias: each in its own feature.  SiLU of
    numbers far below 0 is 0 (to 2^-50), of numbers far above themselves."""
    ops = operands(m + k, m, k, n)
    bias = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    free = sdq.fp8_matmul(*ops, bias=bias, act=act)
    odd = {3: float("nan"), 6: float("inf"), 9: -3e38, 12: 3e38, 16: -100.0, 21: float("nan")}
    big = float(product(*ops)[0].abs().max())
    for f, v in odd.items():
        bias[f] = v if v != -100.0 else -100.0 - 2 * big
    y = sdq.fp8_matmul(*ops, bias=bias, act=act)
    rest = [f for f in range(n) if f not in odd]
    assert torch.equal(y[:, rest], free[:, rest])
    assert y[:, [3, 21]].isnan().all() and (y[:, 6] == float("inf")).all() and (y[:, 12] > 2.9e38).all()
    if act:
        assert (y[:, [9, 16]].abs() <= 2.0 ** -50).all()
    sdq.device_status()


@pytest.mark.parametrize("m", [1, 5, 20, 300])
def test_nothing_beside_the_result_is_written(m):
    """Sentinels around y, odd n (an unaligned pitch) and a y that starts off 16 bytes."""
    k, n = 144, 131
    ops = operands(m, m, k, n)
    room = torch.full((m * n + 64,), -7.0, device="cuda", dtype=torch.bfloat16)
    y = room[33: 33 + m * n].view(m, n)
    sdq.fp8_matmul(*ops, out=y)
    torch.cuda.synchronize()
    assert (room[:33] == -7).all() and (room[33 + m * n:] == -7).all()
    want, s = product(*ops)
    check(y, want, want.abs() * 2.0 ** -8 + sums_tol(s, k))


@pytest.mark.parametrize("oy,orr", [(0, 0), (1, 1), (3, 8), (6, 1), (8, 0), (16, 16)])
@pytest.mark.parametrize("m,n", [(1, 5), (34, 1), (70, 8), (97, 13), (33, 24), (300, 77), (130, 256), (40, 233), (2300, 500)])
def test_result_and_residual_at_any_offset(m, n, oy, orr):
    """y and the residual ``oy`` and ``orr`` values past 512 bytes, at the same place within 16 bytes and
    not, rows of every length: the tensors' ends, chunks that a tile cuts, in place; and y in f32.
    Sentinels around y stay."""
    k = 272
    ops = operands(m + n, m, k, n)
    want, s = product(*ops)
    gate = normals(7, n).to(torch.bfloat16)
    place = lambda o, dt: torch.full((m * n + 128,), -7.0, device="cuda", dtype=dt)[o: o + m * n + 64]  # noqa: E731
    ry, rr, rf = place(oy, torch.bfloat16), place(orr, torch.bfloat16), place(oy, torch.float32)
    res, y, yf = (t[: m * n].view(m, n) for t in (rr, ry, rf))
    res.copy_(normals(8, m, n) * want.abs().mean())
    z = res.double() + gate.double() * want
    tol = gate.double().abs() * (sums_tol(s, k) + want.abs() * 2.0 ** -23) + (z.abs() + (gate.double() * want).abs() * 2.0 ** -14) * 2.0 ** -8
    sdq.fp8_matmul(*ops, gate=gate, residual=res, out=y)
    check(y, z, tol)
    sdq.fp8_matmul(*ops, gate=gate, residual=res, out=res)
    check(res, z, tol)
    sdq.fp8_matmul(*ops, out=yf)
    check(yf, want, want.abs() * 2.0 ** -24 + sums_tol(s, k))
    for room in (ry, rr, rf):
        assert (room[m * n:] == -7).all()
    for t in (y, yf, res):
        before = t._base[: t.storage_offset()]
        assert (before == -7).all()


@pytest.mark.parametrize("m,k,n", [(1, 1040, 700), (40, 1040, 700), (300, 1040, 700), (9, 9728, 512), (70, 8192, 72)])
def test_same_call_same_bits(m, k, n):
    ops = operands(9, m, k, n)
    a = sdq.fp8_matmul(*ops)
    for _ in range(5):
        assert torch.equal(sdq.fp8_matmul(*ops), a)


def test_offsets_past_32_bits():
    """More than 2^31 values in x and in y: the last rows of each."""
    m, k = 131136, 16400
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    x[-3:] = spread(1, 3, k).to(torch.bfloat16)
    q, s = sdq.fp8_quantize(x)
    wq, ws = O.fp8_quantize(x[-3:].double().cpu().numpy())
    assert np.array_equal(u8(q[-3:]), wq) and np.array_equal(u8(s[:, -3:].contiguous()), ws)
    assert not q[:1000].view(torch.uint8).any()
    del x, q, s
    m, k, n = 65600, 16, 32784
    ops = operands(2, m, k, n)
    y = sdq.fp8_matmul(*ops)
    assert y.numel() > 2 ** 31
    for rows in (slice(0, 2), slice(m - 3, m)):
        want, tot = product(ops[0][rows], ops[1][:, rows], *ops[2:])
        check(y[rows], want, want.abs() * 2.0 ** -8 + sums_tol(tot, k))
    sdq.device_status()


def test_two_streams_at_once():
    """Products of different shapes, quantisers and heads in flight together; each has its own result."""
    shapes = [(7, 512, 3000), (300, 1024, 2000), (1000, 512, 999)]
    ops = [operands(30 + i, *s) for i, s in enumerate(shapes)]
    want = [sdq.fp8_matmul(*o) for o in ops]
    streams = [torch.cuda.Stream() for _ in shapes]
    torch.cuda.synchronize()
    got = [[] for _ in shapes]
    for _ in range(10):
        for g, o, st in zip(got, ops, streams):
            g.append(sdq.fp8_matmul(*o, stream=st))
    torch.cuda.synchronize()
    sdq.device_status()
    for g, w in zip(got, want):
        assert all(torch.equal(y, w) for y in g)


def test_beside_the_affine_kernels_on_another_stream():
    """Both take an SM's tensor memory: whichever comes second waits for it."""
    w, x = normals(40, 2048, 1024), normals(41, 700, 1024).to(torch.bfloat16)
    affine, fp8 = sdq.QuantizedArray.quantize(w), sdq.Fp8Array.quantize(w)
    want = affine.matmul(x), fp8.matmul(x), affine.matmul(x[:4]), fp8.matmul(x[:4])
    streams = [torch.cuda.Stream() for _ in want]
    torch.cuda.synchronize()
    got = [[] for _ in want]
    for _ in range(10):
        for g, a, v, st in zip(got, (affine, fp8) * 2, (x, x, x[:4], x[:4]), streams):
            g.append(a.matmul(v, stream=st))
    torch.cuda.synchronize()
    sdq.device_status()
    for g, y in zip(got, want):
        assert all(torch.equal(v, y) for v in g)


def test_empty_batch():
    wq, ws = sdq.fp8_quantize_weight(normals(1, 64, 128))
    x = torch.empty(0, 128, device="cuda", dtype=torch.bfloat16)
    xq, xs = sdq.fp8_quantize(x)
    assert xq.shape == (0, 128) and xs.shape == (1, 0)
    assert sdq.fp8_matmul(xq, xs, wq, ws).shape == (0, 64)
    assert sdq.fp8_dequantize(xq, xs, False).shape == (0, 128)


def test_leading_axes_and_the_array_class():
    x = normals(2, 2, 7, 256).to(torch.bfloat16)
    w = normals(3, 300, 256) / 16
    a = sdq.Fp8Array.quantize(w)
    assert a.shape == (300, 256) and a.resident_bytes() == 300 * 256 + 3 * 2
    y = a.matmul(x)
    assert y.shape == (2, 7, 300) and y.dtype is torch.bfloat16
    xq, xs = sdq.fp8_quantize(x)
    want, s = product(xq.view(14, 256), xs, a.weight, a.scales)
    check(y.view(14, 300), want, want.abs() * 2.0 ** -8 + sums_tol(s, 256))
    f = a.matmul(x.float())
    assert f.dtype is torch.float32
    half = torch.empty(*x.shape[:-1], 300, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(a.matmul(x.float(), out=half), f.to(torch.bfloat16))
    check(f.view(14, 300), want, want.abs() * 2.0 ** -24 + sums_tol(s, 256))
    # each value is within half an e4m3 step (2^-4 of it; 2^-10 of the scale below the normals)
    d = a.dequantize(torch.float32).double()
    step = w.double().abs() * 2.0 ** -4 + 2.0 ** -10 * a.scales.double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:300]
    assert ((d - w.double()).abs() <= step).all()


def test_another_stream_and_a_captured_graph():
    ops = operands(11, 50, 512, 384)
    want = sdq.fp8_matmul(*ops)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y = sdq.fp8_matmul(*ops, stream=s)
    s.synchronize()
    assert torch.equal(y, want)
    x, w = normals(12, 50, 512), normals(13, 384, 512)
    a = sdq.Fp8Array.quantize(w)
    out = torch.empty(50, 384, device="cuda")
    a.matmul(x, out=out)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                       # two graphs of the same call, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            a.matmul(x, out=out)
        graphs.append(g)
    for i in range(4):
        x.copy_(normals(20 + i, 50, 512))
        want = a.matmul(x)
        graphs[i % 2].replay()
        assert torch.equal(out, want)
    sdq.device_status()


def test_the_first_calls_of_a_process_may_be_captured():
    """Kernels' attributes and the tile choice's device queries are made by the first call: in a capture."""
    code = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import sdq
x, w = torch.randn(2, 8192, device="cuda"), torch.randn(128, 8192, device="cuda")
qkv = torch.randn(1, 4, 6, 64, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    xq, xs = sdq.fp8_quantize(x)
    wq, ws = sdq.fp8_quantize_weight(w)
    y = sdq.fp8_matmul(xq, xs, wq, ws, out_dtype=torch.float32)
    z = sdq.qk_norm_rope(*qkv.split(2, 2))[0]
g.replay()
assert torch.equal(y, sdq.fp8_matmul(xq, xs, wq, ws, out_dtype=torch.float32)) and y.abs().min() > 0
assert torch.equal(z, sdq.qk_norm_rope(*qkv.split(2, 2))[0])
sdq.device_status()
"""
    done = subprocess.run([sys.executable, "-c", code, os.path.dirname(os.path.dirname(sdq.__file__))], capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("m", [3, 200])
def test_the_shortcut_and_ctypes_make_the_same_calls(m, monkeypatch):
    """An ordinary call goes through the C++ shortcut, any other through ctypes: the same results."""
    from sdq import _abi, fp8

    assert _abi._native is not None, "binding/sdq_native.cpp was not built"
    x, w = spread(1, m, 272), spread(2, 130, 272)
    bias, gate, res = (normals(3 + i, *shape).to(torch.bfloat16) for i, shape in enumerate(((130,), (130,), (m, 130))))

    def run():
        a, b = sdq.fp8_quantize(x), sdq.fp8_quantize_weight(w)
        return [*a, *b, sdq.fp8_matmul(*a, *b, bias=bias, act="silu", gate=gate, residual=res), sdq.fp8_matmul(*a, *b, out_dtype=torch.float32),
                sdq.fp8_quantize(x.view(1, m, 272))[0]]

    quick = run()
    for name in ("_quantize", "_quantize_weight", "_matmul"):
        monkeypatch.setattr(fp8, name, lambda *args: None)
    for a, b in zip(quick, run()):
        assert a.dtype is b.dtype and a.shape == b.shape and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals_of_the_package():
    xq, xs, wq, ws = operands(3, 4, 256, 130)
    bad = [
        (lambda: sdq.fp8_matmul(xq, xs.t().contiguous(), wq, ws), "xs must have shape"),
        (lambda: sdq.fp8_matmul(xq, xs, wq[:, :128].contiguous(), ws), "wq must have shape"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws[:1].contiguous()), "ws must have shape"),
        (lambda: sdq.fp8_matmul(xq.view(torch.uint8), xs, wq, ws), "xq must be"),
        (lambda: sdq.fp8_matmul(xq, xs.view(torch.uint8), wq, ws), "xs must be"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, bias=torch.zeros(129, device="cuda", dtype=torch.bfloat16)), "bias must hold 130"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, bias=torch.zeros(130, device="cuda")), "bias must hold 130"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, bias=torch.zeros(130)), "bias is on cpu"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, act="relu"), "unknown activation"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, out=torch.empty(4, 131, device="cuda")), "out must have shape"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, out=torch.empty(4, 130, device="cuda", dtype=torch.float16)), "out must be bf16 or f32"),
        (lambda: sdq.fp8_matmul(xq, xs, wq, ws, act="silu", out_dtype=torch.float32), "bias only"),
        (lambda: sdq.fp8_matmul(xq[:, ::2], xs, wq, ws), "contiguous"),
        (lambda: sdq.fp8_quantize(torch.zeros(4, 120, device="cuda")), "multiple of 16"),
        (lambda: sdq.fp8_quantize(torch.zeros(4, 128, device="cuda", dtype=torch.float16)), "bf16 or f32"),
        (lambda: sdq.fp8_quantize(torch.zeros(4, 129, device="cuda")[:, :128]), "contiguous"),
        (lambda: sdq.fp8_quantize(torch.zeros(4 * 128 + 1, device="cuda")[1:].view(4, 128)), "misaligned"),
        (lambda: sdq.fp8_quantize_weight(torch.zeros(2, 4, 128, device="cuda")), "2-D"),
        (lambda: sdq.fp8_dequantize(xq, xs, True), "scales must have shape"),
        (lambda: sdq.fp8_dequantize(xq, xs, False, torch.float16), "bf16 or f32"),
    ]
    for call, needle in bad:
        with pytest.raises(sdq.SdqError, match=needle):
            call()


@pytest.mark.parametrize("m,k,n", [(100, 1024, 4096), (300, 1024, 4096), (20, 8192, 128)])
def test_withheld_copy_times_out_then_the_next_call_is_correct(m, k, n):
    """The bounded waits (see test_gpu_abort.py) of the fp8 kernel: single CTAs, pairs, shared tiles."""
    ops = operands(5, m, k, n)
    want = sdq.fp8_matmul(*ops)
    sdq.device_status()
    sdq.debug_wait_hook(20_000_000, True)
    try:
        sdq.fp8_matmul(*ops)
        torch.cuda.synchronize()
        with pytest.raises(sdq.SdqError, match="gave up"):
            sdq.device_status()
    finally:
        sdq.debug_wait_hook(0, False)
    sdq.device_status()
    assert torch.equal(sdq.fp8_matmul(*ops), want)
