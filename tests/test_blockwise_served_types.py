"""A served blockwise linear keeps its bytes when a model's type changes: no GPU needed to see that."""
import copy

import pytest
import torch
import torch.nn as nn

import float8_experimental_amd as f8


def served(device="cpu", bias=True):
    layer = f8.Float8BlockwiseInferenceLinear(200, 130, torch.randn(130) if bias else None, device=device)
    if device == "cpu":
        for t in (layer.weight_data.view(torch.uint8), layer.weight_scales):
            t.copy_(torch.randint(0, 120, t.shape, dtype=torch.uint8))
    return layer


@pytest.mark.parametrize("change", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.float(), lambda m: m.double(), lambda m: m.to("cpu", torch.bfloat16),
                                    lambda m: m.bfloat16().float(), lambda m: m.type(torch.float16)])
def test_the_weight_keeps_its_type_and_bytes(change):
    layer = served()
    model = nn.Sequential(nn.LayerNorm(200), copy.deepcopy(layer))
    values = layer.dequantized_weight()
    change(model)
    got = model[1]
    assert got.weight_data.dtype is torch.float8_e4m3fn and got.weight_scales.dtype is torch.uint8 and got.bias.dtype is model[0].weight.dtype
    assert torch.equal(got.weight_data.view(torch.uint8), layer.weight_data.view(torch.uint8)) and torch.equal(got.weight_scales, layer.weight_scales)
    assert torch.equal(got.dequantized_weight(), values)
    assert set(got.state_dict()) == {"weight_data", "weight_scales", "bias"}
    served().to(torch.bfloat16).load_state_dict(got.state_dict())


def test_the_weight_moves_between_devices():
    layer = served(bias=False).to("meta")
    assert layer.weight_data.device.type == "meta" and layer.weight_data.dtype is torch.float8_e4m3fn
    layer = layer.to_empty(device="cpu")
    assert layer.weight_data.device.type == "cpu" and layer.weight_data.dtype is torch.float8_e4m3fn and layer.weight_data.shape == served().weight_data.shape
