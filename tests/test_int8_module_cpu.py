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


def stays(layer, kernel):
    assert torch.equal(layer.kernel, kernel) and layer.kernel.shape == (3, 20, 50) and layer.kernel.stride() == (20 * 64, 64, 1) and layer.kernel.data_ptr() % 16 == 0


def test_codes_stay_16_bytes_apart(layer):
    """Through everything that copies a module's buffers, or puts others in their place."""
    kernel = layer.kernel.clone()
    stays(layer, kernel)
    stays(copy.deepcopy(layer), kernel)
    layer._apply(lambda t: t.clone())  # what a move to another device does
    stays(layer, kernel)
    for assign in (False, True):
        other = copy.deepcopy(layer)
        other.kernel.zero_()
        other.load_state_dict({k: v.clone(memory_format=torch.contiguous_format) for k, v in layer.state_dict().items()}, assign=assign)
        stays(other, kernel)
    empty = copy.deepcopy(layer).to("meta").to_empty(device="cpu")
    empty.load_state_dict(layer.state_dict())
    stays(empty, kernel)


def test_a_saved_module(layer, tmp_path):
    kernel = layer.kernel.clone()
    torch.save(layer, tmp_path / "layer.pt")
    stays(torch.load(tmp_path / "layer.pt", weights_only=False), kernel)
    layer._buffers["kernel"] = kernel  # as an earlier release may have saved it
    torch.save(layer, tmp_path / "layer.pt")
    stays(torch.load(tmp_path / "layer.pt", weights_only=False), kernel)
