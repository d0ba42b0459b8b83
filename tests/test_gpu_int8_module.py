"""The module of products in 8 bits after a model was cast and moved."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def made(c_in, c_out=40, groups=2):
    from fgms_b200 import nn
    gen = torch.Generator(device="cuda").manual_seed(c_in)
    x = torch.randn((30, c_in), generator=gen, device="cuda").bfloat16()
    layer = nn.Int8GroupedLinear((torch.randn((groups, c_in, c_out), generator=gen, device="cuda") * c_in ** -0.5).bfloat16())
    return layer, x, torch.tensor([0, 11, 30], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.float(), lambda m: m.to("cuda", torch.float16)])
def test_a_cast_changes_nothing(cast):
    layer, x, kpos = made(50)
    want = layer(x, kpos)
    assert torch.equal(cast(layer)(x, kpos), want)


@pytest.mark.parametrize("c_in", [50, 64])
def test_a_module_that_was_moved_copies_no_weights(c_in):
    from fgms_b200 import _lib, nn
    layer, x, kpos = made(c_in)
    want = layer(x, kpos)
    for moved in (copy.deepcopy(layer), layer.cpu().cuda()):
        codes, scale = nn.quantize_rows(x)
        assert _lib.lib.fgms_b200_grouped_i8_workspace_bytes(codes.data_ptr(), codes.stride(0), moved.kernel.data_ptr(), moved.kernel.stride(1), 30, c_in, 40, 2) == 0
        assert torch.equal(moved((codes, scale), kpos), want)
