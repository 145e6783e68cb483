"""Host logic of holding weights as block-scaled e4m3 (no device)."""
from __future__ import annotations

import pytest

import sdq
from sdq import quantized as Q


def test_mixed_gives_fp8_to_the_ordinary_layers_only():
    f = Q.mixed(Q.FP8)
    assert f("double_blocks.0.img_attn.qkv.weight") == Q.FP8
    assert f("img_in.weight") == 8 and f("final_layer.linear.weight") == 8
    assert f("model.embed_tokens.weight") == 0


@pytest.mark.parametrize("shape,fits", [((5, 16), True), ((1, 48), True), ((4, 8), False), ((4, 100), False), ((64,), False),
                                        ((2, 4, 16), False), ((0, 16), False), ((4, 0), False)])
def test_shapes_that_fp8_takes(shape, fits):
    assert Q.fp8_quantizable(shape) is fits


def test_another_name_is_refused():
    import torch
    with pytest.raises(sdq.SdqError, match="'int8'"):
        Q.mixed("int8")
    with pytest.raises(sdq.SdqError, match="'FP8'"):
        Q.from_dense_with({"a.weight": torch.zeros(2, 64)}, lambda name: "FP8")


def test_a_policy_keeps_unfit_tensors_dense():
    import torch
    w = {"a.bias": torch.zeros(7), "b.weight": torch.zeros(3, 20), "c.weight": torch.zeros(3, 24)}
    held = Q.from_dense_with(w, lambda name: Q.FP8 if name != "c.weight" else 0)
    assert not held.quantized and sorted(held.dense) == sorted(w)
