"""GPU: the fp8 linears and the head preparation together, as a model runs them -- a small
Flux-shaped stack held as block-scaled e4m3, against dense weights and against the op-by-op path.

The stack's products quantise their activations to 4 significant bits (each value off by at most
2^-4 of itself, as if at random), which a dense source does not; the bars on cosine and norm are for
that, the codes themselves are pinned by test_gpu_fp8.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle as O
import sdq
from conftest import gpu_available
from sdq import flux
from sdq import gguf as G
from sdq import quantized as Q
from test_gguf import random_raw

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")]

CFG = flux.FluxShape(hidden=256, heads=2, depth=2, depth_single=2, txt_tokens=32, img_tokens=64, context_dim=128, vec_dim=64)


class Rounded(Q.DenseWeights):
    """Dense weights whose linears see their activations as the fp8 ones do: quantised and back."""

    def linear(self, x, name, bias=None):
        xq, xs = sdq.fp8_quantize(x.contiguous())
        return super().linear(sdq.fp8_dequantize(xq, xs, False, torch.float32), name, None if bias is None else bias.float()).to(x.dtype)


def close(got, want, cos_bar, rel_bar):
    g, w = got.double().flatten(), want.double().flatten()
    cos, rel = float(g @ w / (g.norm() * w.norm())), float((g - w).norm() / w.norm())
    assert cos >= cos_bar and rel <= rel_bar, (cos, rel)


@pytest.mark.parametrize("fused", [False, True])
def test_fp8_stack_matches_dense_weights_on_rounded_activations(fused):
    """Every linear, its bias and output stage, and the heads: the same forward on dequantised
    weights with torch's products."""
    qw, dense = flux.random_weights(CFG, seed=3, bits=lambda name: Q.FP8, keep_dense=True)
    assert all(isinstance(q, sdq.Fp8Array) for q in qw.quantized.values())
    rope, args = flux.rope_tables(CFG), flux.inputs(CFG, seed=4)
    got = flux.forward(qw, *args, CFG, rope, fused_heads=fused)
    want = flux.forward(Rounded(dense), *args, CFG, rope)
    sdq.device_status()
    assert got.shape == (1, CFG.img_tokens, CFG.in_channels)
    close(got, want, 0.995, 0.1)
    # and not far from full-precision activations
    close(got, flux.forward(Q.DenseWeights(dense), *args, CFG, rope), 0.98, 0.2)


def test_fused_heads_match_the_op_by_op_heads():
    """One rounding instead of two, in every block: the affine stack both ways."""
    qw = flux.random_weights(CFG, seed=5)
    rope, args = flux.rope_tables(CFG), flux.inputs(CFG, seed=6)
    close(flux.forward(qw, *args, CFG, rope, fused_heads=True), flux.forward(qw, *args, CFG, rope), 0.999, 0.05)


def test_one_block_of_the_run_in_64_bits():
    """quantise -> qkv product -> norm, rotation, transposition, on the values each step hands on.
    Tolerances as in test_gpu_fp8.py and test_gpu_qk.py, one step at a time."""
    b, n, h, d, k = 2, 37, 3, 64, 320
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(b, n, k, device="cuda", generator=g).to(torch.bfloat16)
    w = sdq.Fp8Array.quantize(torch.randn(3 * h * d, k, device="cuda", generator=g) / k ** 0.5)
    norm = torch.ones(d, device="cuda", dtype=torch.bfloat16)
    angle = torch.arange(n, device="cuda")[:, None] * 1e2 ** (-torch.arange(d // 2, device="cuda") / d)
    qkv = w.matmul(x)
    xq, xs = O.fp8_quantize(x.view(b * n, k).double().cpu().numpy())
    xv = torch.from_numpy(O.fp8_dequantize(xq, xs, False)).cuda()
    wv = torch.from_numpy(O.fp8_dequantize(w.weight.view(torch.uint8).cpu().numpy(), w.scales.view(torch.uint8).cpu().numpy(), True)).cuda()
    want, s = xv @ wv.t(), xv.abs() @ wv.abs().t()
    assert ((qkv.view(b * n, -1).double() - want).abs() <= want.abs() * 2.0 ** -8 + (k / 32 + 32) * 2.0 ** -23 * s).all()
    q, key, v = qkv.unflatten(-1, (3, h, d)).unbind(2)
    qo, ko, vo = sdq.qk_norm_rope(q, key, v, norm, norm, angle.cos(), angle.sin())
    for got, src in ((qo, q), (ko, key)):
        y = src.double()
        y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        z = torch.complex(y[..., 0::2], y[..., 1::2]) * torch.complex(angle.cos(), angle.sin())[None, :, None]
        ref = torch.view_as_real(z).flatten(-2).transpose(1, 2)
        size = (z.real.abs() + z.imag.abs()).repeat_interleave(2, -1).transpose(1, 2) * 2
        assert ((got.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + size * (d / 8 + 20) * 2.0 ** -24).all()
    assert torch.equal(vo, v.transpose(1, 2))
    sdq.device_status()


def test_the_run_in_a_captured_graph_on_new_inputs():
    qw = flux.random_weights(CFG, seed=8, bits=Q.mixed(Q.FP8))
    rope, args = flux.rope_tables(CFG), flux.inputs(CFG, seed=9)
    flux.forward(qw, *args, CFG, rope, fused_heads=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = flux.forward(qw, *args, CFG, rope, fused_heads=True)
    for seed in (10, 11):
        for a, new in zip(args, flux.inputs(CFG, seed=seed)):
            a.copy_(new)
        g.replay()
        assert torch.equal(out, flux.forward(qw, *args, CFG, rope, fused_heads=True))
    sdq.device_status()


def test_from_dense_and_from_gguf(tmp_path):
    n, k = 96, 256
    raw = random_raw(G.Q8_0, n * k, seed=2)
    bias = np.arange(n, dtype=np.float32)
    path = str(tmp_path / "w.gguf")
    G.write(path, [("blk.0.attn.weight", (n, k), G.Q8_0, raw), ("blk.0.attn.bias", (n,), G.F32, bias.view(np.uint8))])
    held = Q.from_gguf(path, Q.FP8)
    a = held.quantized["blk.0.attn.weight"]
    assert isinstance(a, sdq.Fp8Array) and held.resident_bytes() == n * k + 2 + 4 * n
    dense = O.gguf_dequantize(raw, O.GGML_Q8_0, n * k).reshape(n, k)
    wq, ws = O.fp8_quantize_weight(dense.astype(np.float64))
    assert np.array_equal(a.weight.view(torch.uint8).cpu().numpy(), wq) and np.array_equal(a.scales.view(torch.uint8).cpu().numpy(), ws)
    same = Q.from_dense({"blk.0.attn.weight": torch.from_numpy(dense).cuda()}, Q.FP8).quantized["blk.0.attn.weight"]
    assert torch.equal(same.weight.view(torch.uint8), a.weight.view(torch.uint8))
    x = torch.randn(5, k, device="cuda")
    y = held.linear(x, "blk.0.attn.weight", held.optional("blk.0.attn.bias"))
    assert torch.equal(y, a.matmul(x, bias=torch.from_numpy(bias).cuda())) and y.dtype is torch.float32
    with pytest.raises(sdq.SdqError, match="is quantised"):
        held.dense_tensor("blk.0.attn.weight")
