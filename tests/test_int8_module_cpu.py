"""The module of products in 8 bits when a model is cast, moved and loaded (no GPU: its buffers alone)."""
import copy

import pytest
import torch

from fgms_b200 import nn


def quantized(x):
    """``nn.quantize_rows`` on the host: codes whose rows are a multiple of 16 bytes apart."""
    scale = x.float().abs().amax(1) / 127
    room = torch.zeros((x.size(0), (x.size(1) + 15) // 16 * 16), dtype=torch.int8)
    room[:, :x.size(1)] = (x.float() / scale[:, None]).round()
    return room[:, :x.size(1)], scale


@pytest.fixture
def layer(monkeypatch):
    monkeypatch.setattr(nn, "quantize_rows", quantized)
    return nn.Int8GroupedLinear(torch.randn((3, 50, 20), generator=torch.Generator().manual_seed(1)).bfloat16())


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16)])
def test_scales_stay_in_32_bits(layer, cast):
    kernel, scale = layer.kernel.clone(), layer.kernel_scale.clone()
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), layer)
    cast(model)
    assert model[0].weight.dtype != torch.float32 and layer.kernel_scale.dtype == torch.float32 and layer.dtype == torch.bfloat16
    assert torch.equal(layer.kernel_scale, scale) and torch.equal(layer.kernel, kernel)
    assert set(layer.state_dict()) == {"kernel", "kernel_scale"}
