"""GPU: the fp8 and head-preparation kernels beside one another.  They start while the kernel before them
in their stream still runs, and wait for it; on other streams others of them run meanwhile.  Every result
is compared, bit for bit, with the one that the call gives alone."""
from __future__ import annotations

import pytest
import torch

import sdq
from conftest import gpu_available
from test_gpu_fp8 import normals, operands, u8

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")]


def same(got, want):
    return all(a is None and b is None or (u8(a) == u8(b)).all() for a, b in zip(got, want))


def heads_case(dtype, b, n, hq, hkv, d, pairs):
    qkv = normals(b + n, b, n, hq + 2 * hkv, d).to(dtype)
    q, k, v = qkv.split([hq, hkv, hkv], 2)
    w = normals(3, d).to(dtype)
    angle = torch.arange(n, device="cuda")[:, None] * 1e3 ** (-torch.arange(d // 2, device="cuda") / d)
    positions = torch.randint(0, n, (b, n), device="cuda")
    return lambda stream=None, out=None: sdq.qk_norm_rope(q, k, v, w, w, angle.cos(), angle.sin(), positions=positions, pairs=pairs,
                                                           out=out, stream=stream)


def test_every_kernel_on_a_stream_of_its_own_at_once():
    x, w = normals(1, 2000, 3008).to(torch.bfloat16), normals(2, 2049, 1040)
    one, pairs, shared = operands(3, 70, 528, 3001), operands(4, 300, 4096, 4096), operands(5, 7, 9728, 2560)
    xq, xs = sdq.fp8_quantize(x)
    calls = [lambda s: sdq.fp8_quantize(x, stream=s), lambda s: sdq.fp8_quantize_weight(w, stream=s),
             lambda s: (sdq.fp8_dequantize(xq, xs, False, stream=s),)]
    calls += [lambda s, o=o: (sdq.fp8_matmul(*o, stream=s),) for o in (one, pairs, shared)]
    for case in ((torch.bfloat16, 1, 1500, 24, 24, 128, "interleaved"), (torch.float32, 3, 301, 8, 2, 80, "halves")):
        calls.append(heads_case(*case))
    want = [c(None) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    got = [[] for _ in calls]
    for _ in range(10):
        for g, c, s in zip(got, calls, streams):
            g.append(c(s))
    torch.cuda.synchronize()
    sdq.device_status()
    for g, y in zip(got, want):
        assert all(same(r, y) for r in g)


def test_chains_that_reuse_their_buffers():
    """copy -> quantise -> qkv product -> heads -> quantise -> product with residual, in place, again and again in
    the same memory, two chains of different sizes on two streams."""

    class Chain:
        def __init__(self, m, k, h, d, seed):
            self.inputs = [normals(seed + i, m, k).to(torch.bfloat16) for i in range(6)]
            self.qkv_w = sdq.Fp8Array.quantize(normals(seed + 10, 3 * h * d, k) / k ** 0.5)
            self.out_w = sdq.Fp8Array.quantize(normals(seed + 11, k, h * d) / (h * d) ** 0.5)
            self.norm = normals(seed + 12, d).to(torch.bfloat16)
            angle = torch.arange(m, device="cuda")[:, None] * 1e3 ** (-torch.arange(d // 2, device="cuda") / d)
            self.cos, self.sin, self.shape = angle.cos(), angle.sin(), (1, m, 3, h, d)
            empty = lambda *s: torch.empty(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
            self.x, self.qkv, self.heads = empty(m, k), empty(m, 3 * h * d), [empty(1, m, h, d) for _ in range(3)]

        def run(self):
            results = []
            for given in self.inputs:
                self.x.copy_(given)
                self.qkv_w.matmul(self.x, out=self.qkv)
                q, k, v = self.qkv.view(self.shape).unbind(2)
                sdq.qk_norm_rope(q, k, v, self.norm, self.norm, self.cos, self.sin, out=tuple(t.transpose(1, 2) for t in self.heads))
                self.out_w.matmul_fused(self.heads[0].view(self.shape[1], -1), residual=self.x, out=self.x)
                results.append((self.x.clone(), self.qkv.clone(), *(t.clone() for t in self.heads)))
            return results

    chains = [Chain(300, 1024, 8, 128, 100), Chain(37, 528, 4, 64, 200)]
    want = [c.run() for c in chains]
    for c in chains:                                              # step by step, nothing overlapping
        for i, given in enumerate(c.inputs):
            c.inputs, keep = [given], c.inputs
            torch.cuda.synchronize()
            alone = c.run()[0]
            torch.cuda.synchronize()
            c.inputs = keep
            assert same(alone, want[chains.index(c)][i])
    streams = [torch.cuda.Stream() for _ in chains]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(chains, streams):
        with torch.cuda.stream(s):
            got.append([c.run() for _ in range(3)])
    torch.cuda.synchronize()
    sdq.device_status()
    for g, w in zip(got, want):
        assert all(same(a, b) for again in g for a, b in zip(again, w))


def test_calls_of_several_threads_at_once():
    """The library's calls run without the interpreter's lock; each thread has a stream of its own."""
    from concurrent.futures import ThreadPoolExecutor

    x = normals(21, 130, 528).to(torch.bfloat16)
    ws = [sdq.Fp8Array.quantize(normals(22 + i, 3 * 4 * 64 + 16 * i, 528)) for i in range(4)]
    heads = heads_case(torch.bfloat16, 1, 130, 4, 4, 64, "halves")
    run = lambda w: (w.matmul(x), w.matmul_fused(x, act="silu"), *heads(), *sdq.fp8_quantize(x))  # noqa: E731
    want = [run(w) for w in ws]
    torch.cuda.synchronize()

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = [run(ws[i]) for _ in range(25)]
        s.synchronize()
        return all(same(g, want[i]) for g in got)

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))
    sdq.device_status()
