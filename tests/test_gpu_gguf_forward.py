"""GPU: a checkpoint read from GGUF, whose biases and norm scales are f32, through a forward in bf16."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import sdq
from conftest import gpu_available
from sdq import flux
from sdq import gguf as G
from sdq import quantized as Q

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")]

CFG = flux.FluxShape(hidden=256, heads=2, depth=1, depth_single=1, txt_tokens=32, img_tokens=64, context_dim=128, vec_dim=64)


def checkpoint(path):
    """Linears N(0, 1/K), biases N(0, 0.02) that no bf16 holds, norm scales around 1 that one does."""
    rng, tensors = np.random.default_rng(1), []
    for name, n, k, _ in flux.linear_table(CFG):
        tensors.append((name, (n, k), G.F32, (rng.standard_normal((n, k)) / k ** 0.5).astype(np.float32)))
    for name, shape in flux.dense_tensor_table(CFG):
        v = rng.standard_normal(shape).astype(np.float32)
        tensors.append((name, shape, G.F32, 0.02 * v if name.endswith("bias") else 1 + np.round(16 * v) / 128))
    G.write(path, [(n, s, kind, np.ascontiguousarray(v, np.float32).reshape(-1).view(np.uint8)) for n, s, kind, v in tensors])


@pytest.mark.parametrize("bits", [Q.FP8, 4])
def test_forward_in_bf16(tmp_path, bits):
    path = str(tmp_path / "flux.gguf")
    checkpoint(path)
    held = Q.from_gguf(path, bits)
    forms = {type(q) for q in held.quantized.values()}
    assert forms == ({sdq.Fp8Array, sdq.QuantizedArray} if bits == Q.FP8 else {sdq.QuantizedArray})
    assert all(t.dtype is torch.float32 for t in held.dense.values())
    # the same weights with the dense tensors rounded beforehand: the same forward, bit for bit
    narrow = Q.QuantizedWeights(held.quantized, {n: t.to(torch.bfloat16) for n, t in held.dense.items()})
    dense = Q.DenseWeights({**narrow.dense, **{n: q.dequantize(torch.bfloat16) for n, q in held.quantized.items()}})
    rope, args = flux.rope_tables(CFG), flux.inputs(CFG, seed=4)
    for fused in (False, True):
        got = flux.forward(held, *args, CFG, rope, fused_heads=fused)
        assert got.dtype is torch.bfloat16 and torch.equal(got, flux.forward(narrow, *args, CFG, rope, fused_heads=fused))
        # and the forward on dense weights, whose activations are not quantised (the bars of the fp8 stack)
        want = flux.forward(dense, *args, CFG, rope).double().flatten()
        g = got.double().flatten()
        assert float(g @ want / (g.norm() * want.norm())) >= 0.98 and float((g - want).norm() / want.norm()) <= 0.2
    sdq.device_status()


@pytest.mark.parametrize("form", ["fp8", "affine"])
def test_a_bias_of_another_float_type(form):
    m, k, n = 37, 256, 130
    g = torch.Generator("cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    w = (sdq.Fp8Array if form == "fp8" else sdq.QuantizedArray).quantize(rand(n, k) / 16)
    x, bias, gate, res = rand(m, k).to(torch.bfloat16), rand(n), rand(n), rand(m, n).to(torch.bfloat16)
    b, gt = bias.to(torch.bfloat16), gate.to(torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for stream in (None, s, s.cuda_stream):
        y, z = w.matmul(x, bias=bias, stream=stream), w.matmul_fused(x, bias=bias, act="silu", gate=gate, residual=res, stream=stream)
        wide = w.matmul(x.float(), bias=b, stream=stream)
        s.synchronize()
        assert torch.equal(y, w.matmul(x, bias=b)) and y.dtype is torch.bfloat16
        assert torch.equal(z, w.matmul_fused(x, bias=b, act="silu", gate=gt, residual=res))
        assert torch.equal(wide, w.matmul(x.float(), bias=b.float())) and wide.dtype is torch.float32
    with pytest.raises(sdq.SdqError):
        w.matmul(x, bias=torch.zeros(n, device="cuda", dtype=torch.int32))
    sdq.device_status()
