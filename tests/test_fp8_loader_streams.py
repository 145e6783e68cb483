"""Where the loaders' temporaries live: a tensor that a kernel on an explicit stream reads must not go
back to another stream's allocator while that kernel is still to run."""
from __future__ import annotations

import contextlib

import numpy as np
import pytest
import torch

import oracle as O
import sdq
from conftest import gpu_available
from sdq import gguf as G
from sdq import quantized as Q
from test_gguf import random_raw


class Device:
    """Stands in for a device: whose stream is current while each step runs."""

    def __init__(self, monkeypatch):
        self.current, self.steps = "own", []

        @contextlib.contextmanager
        def on(stream, device):
            was, self.current = self.current, stream if stream is not None else self.current
            yield
            self.current = was

        monkeypatch.setattr(Q, "_on", on, raising=False)
        step = lambda name, value: (lambda *a, **k: (self.steps.append((name, k.get("stream") or self.current)), value)[1])  # noqa: E731
        monkeypatch.setattr(Q.Fp8Array, "quantize", step("fp8", "fp8"))
        monkeypatch.setattr(Q.QuantizedArray, "quantize", step("affine", "affine"))
        monkeypatch.setattr(sdq, "gguf_quantize", step("gguf affine", (None, None, None)))
        monkeypatch.setattr(sdq, "gguf_dequantize", lambda raw, kind, shape, dtype, stream=None: step("gguf dense", torch.zeros(shape))())
        plain = torch.Tensor.contiguous
        monkeypatch.setattr(torch.Tensor, "contiguous", lambda t, *a, **k: (t.is_contiguous() or step("copy", None)(), plain(t, *a, **k))[1])
        to = torch.Tensor.to
        monkeypatch.setattr(torch.Tensor, "to", lambda t, d, *a, **k: (step("upload", None)(), t if isinstance(d, torch.device) else to(t, d, *a, **k))[1])


def test_every_step_of_a_loader_is_on_the_given_stream(monkeypatch, tmp_path):
    dev = Device(monkeypatch)
    held = Q.from_dense_with({"a.weight": torch.zeros(128, 64).t(), "b.weight": torch.zeros(64, 64).t(), "c.weight": torch.zeros(6, 20).t()},
                             lambda name: {"a": Q.FP8, "b": 4, "c": Q.FP8}[name[0]], stream="given")
    assert held.quantized == {"a.weight": "fp8", "b.weight": "affine"} and list(held.dense) == ["c.weight"]
    assert dev.steps == [("copy", "given"), ("fp8", "given"), ("copy", "given"), ("affine", "given"), ("copy", "given")]
    dev.steps.clear()
    path = str(tmp_path / "w.gguf")
    G.write(path, [("blk.0.weight", (8, 64), G.Q8_0, random_raw(G.Q8_0, 512, 1)), ("x_embedder.weight", (8, 64), G.F32, random_raw(G.F32, 512, 2)),
                   ("blk.0.bias", (8,), G.F32, random_raw(G.F32, 8, 3))])
    monkeypatch.setattr(Q, "sensitive", lambda name: name.startswith("x_"))
    held = Q.from_gguf(path, Q.FP8, device="cuda:0", stream="given")
    assert held.quantized["blk.0.weight"] == "fp8" and list(held.dense) == ["blk.0.bias"]
    assert {s for _, s in dev.steps} == {"given"} and [n for n, _ in dev.steps] == [
        "upload", "gguf dense", "fp8", "upload", "gguf affine", "upload", "gguf dense"]


def busy(stream):
    """Some 100 ms of work ahead on ``stream``: what the host queues next runs well after it was queued."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(200_000_000)


@pytest.mark.parametrize("raw_handle", [False, True])
@pytest.mark.parametrize("bits", [Q.FP8, 4])
@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")
def test_a_checkpoint_loaded_on_a_busy_stream(tmp_path, bits, raw_handle):
    """Tensors of one size, so that a block given back too early would be the next one's."""
    n, k, count = 512, 1024, 6
    raws = [random_raw(G.Q8_0, n * k, seed=s) for s in range(count)]
    path = str(tmp_path / "w.gguf")
    G.write(path, [(f"blk.{i}.weight", (n, k), G.Q8_0, r) for i, r in enumerate(raws)])
    want = Q.from_gguf(path, bits)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    busy(s)
    held = Q.from_gguf(path, bits, stream=s.cuda_stream if raw_handle else s)
    other = [torch.full((n, k), float("nan"), device="cuda") for _ in range(count)]      # the current stream goes on
    s.synchronize()
    for name, w in want.quantized.items():
        assert torch.equal(held.quantized[name].weight.view(torch.uint8), w.weight.view(torch.uint8))
        assert torch.equal(held.quantized[name].scales.view(torch.uint8), w.scales.view(torch.uint8))
    if bits == Q.FP8:
        wq, ws = O.fp8_quantize_weight(O.gguf_dequantize(raws[3], O.GGML_Q8_0, n * k).reshape(n, k).astype(np.float64))
        a = held.quantized["blk.3.weight"]
        assert np.array_equal(a.weight.view(torch.uint8).cpu().numpy(), wq) and np.array_equal(a.scales.view(torch.uint8).cpu().numpy(), ws)
    assert len(other) == count


@pytest.mark.parametrize("bits", [Q.FP8, 8])
@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")
def test_transposed_weights_quantised_on_a_busy_stream(bits):
    """A weight that is not contiguous is copied first; the copy is the loader's own."""
    w = {f"blk.{i}.weight": torch.randn(1024, 512, device="cuda").t() for i in range(6)}
    want = Q.from_dense_with(w, lambda name: bits)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    busy(s)
    held = Q.from_dense_with(w, lambda name: bits, stream=s)
    other = [torch.full((512, 1024), float("nan"), device="cuda") for _ in w]
    s.synchronize()
    for name, q in want.quantized.items():
        assert torch.equal(held.quantized[name].weight.view(torch.uint8), q.weight.view(torch.uint8))
        assert torch.equal(held.quantized[name].scales.view(torch.uint8), q.scales.view(torch.uint8))
    assert len(other) == len(w)


def test_which_stream_a_raw_handle_is(monkeypatch):
    """0 is the default stream's handle, which torch's ExternalStream does not take for it."""
    from sdq import _abi

    here, used = contextlib.nullcontext(), []
    monkeypatch.setattr(torch.cuda, "device", lambda d: here)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)

    class Some:
        device_index, device = 0, "cuda:0"

        def __init__(self, name):
            self.name = name

    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle: Some(handle))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda: Some("default"))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: (used.append(s.name), here)[1])

    class Foreign:
        cuda_stream = 78

    for given in (0, 77, Foreign()):
        with _abi.on(given, torch.device("cuda", 0)):
            pass
    assert used == ["default", 77, 78]


@pytest.mark.gpu
@pytest.mark.skipif(not gpu_available(), reason="needs an sm_100 device")
def test_work_on_the_default_streams_handle_is_in_its_order():
    x, w = torch.randn(300, 512, device="cuda"), sdq.Fp8Array.quantize(torch.randn(130, 512, device="cuda"))
    q = torch.randn(2, 30, 4, 64, device="cuda")
    new_x, new_q = torch.randn_like(x), torch.randn_like(q)
    want = w.matmul(new_x), sdq.qk_norm_rope(new_q, new_q, eps=1e-6)[0]
    assert torch.cuda.current_stream().cuda_stream == 0
    busy(torch.cuda.current_stream())
    x.copy_(new_x)
    q.copy_(new_q)
    got = w.matmul(x, stream=0), sdq.qk_norm_rope(q, q, eps=1e-6, stream=0)[0]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_stream_of_another_device_is_refused(monkeypatch):
    from sdq import _abi

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle: handle)

    class Handle:
        cuda_stream = type("S", (), {"device_index": 1, "device": "cuda:1"})()

    with pytest.raises(sdq.SdqError, match="cannot run work"):
        with _abi.on(Handle(), torch.device("cuda", 0)):
            pass
