"""The choice of experts on both ways through ``nn.expert_layer``: the kernel for a few rows, the grouped products for more of them or with gradients."""
import pytest
import torch

from tests.layers_ref import near
from tests.test_gpu_experts import Layer

pytestmark = pytest.mark.gpu


def ways(layer, top_k=None):
    """(few rows, many rows, with gradients) of one layer's rows."""
    from fgms_b200 import backend, nn
    args = (layer.router, layer.w_in, layer.w_out, top_k or layer.top_k)
    before = backend.launch_count()
    few = nn.expert_layer(layer.x, *args)
    assert backend.launch_count() - before == 2
    many = nn.expert_layer(layer.x.repeat(3, 1), *args)[:layer.x.size(0)]
    x = layer.x.clone().requires_grad_()
    return few, many, nn.expert_layer(x, *args).detach()


def definition(layer):
    """The layer in 64 bits and what either way may be off by.  Through the grouped products u, h and the experts' outputs are each rounded to the rows' type as well: h is off
    by 3.2 half steps of its size then (u in both factors, the activation's slope, itself), the output by that of the sum of the magnitudes of what it is added up from, and by
    one more half step of each expert's part."""
    out, allowed, chosen, gates = layer.exact()
    share = torch.zeros((layer.x.size(0), layer.router.size(0)), dtype=torch.float64, device="cuda").scatter_(1, chosen.long(), gates)
    u, hidden = torch.einsum("tc,ech->teh", layer.x.double(), layer.w_in.double()), layer.w_out.size(1)
    size = torch.einsum("teh,eho,te->to", 1.1 * u[..., :hidden].abs() * u[..., hidden:].abs(), layer.w_out.double().abs(), share)
    return out, allowed + 4.5 * torch.finfo(layer.type).eps / 2 * size


def test_a_router_row_that_is_not_a_number_is_the_last_choice():
    """One row of the router is NaN: its expert is chosen by nobody while others are left, and has no weight where all are chosen; tokens whose logits are
    all NaN have outputs of NaN."""
    layer = Layer("bf16", 30, 8, 3, 64, 96, seed=21)
    layer.router[2] = float("nan")
    layer.x[11, 5] = float("nan")
    fine = [t for t in range(30) if t != 11]
    without = [e for e in range(8) if e != 2]
    sane = Layer("bf16", 30, 8, 3, 64, 96, seed=21)
    sane.router, sane.w_in, sane.w_out = (getattr(sane, n)[without].contiguous() for n in ("router", "w_in", "w_out"))
    for top_k, others in ((3, 3), (8, 7)):
        sane.top_k = others
        want, allowed = definition(sane)
        for got in ways(layer, top_k):
            assert torch.isnan(got[11]).all()
            near(got[fine], want[fine], allowed[fine])


@pytest.fixture(params=["as it is", "tf32 allowed", "tf32 by name", "autocast"])
def process(request):
    """What a process allows products of float32 matrices."""
    matmul = torch.backends.cuda.matmul
    if request.param == "tf32 allowed":
        was, matmul.allow_tf32 = matmul.allow_tf32, True
        yield
        matmul.allow_tf32 = was
    elif request.param == "tf32 by name":
        was, matmul.fp32_precision = matmul.fp32_precision, "tf32"
        yield
        matmul.fp32_precision = was
    elif request.param == "autocast":
        with torch.autocast("cuda", dtype=torch.bfloat16):
            yield
    else:
        yield


def test_a_choice_that_32_bits_tell_and_fewer_do_not(process):
    """Experts 1 and 6 have rows of the router in the ratio 1 : 1 + 2^-14, which TF32 and bf16 round to the same; all logits are positive multiples of what 32 bits add up without
    an error of that size (256 values of one sign: 257 2^-24 = 2^-16 at most)."""
    layer = Layer("bf16", 20, 8, 1, 256, 64, seed=22, router_type=torch.float32)
    layer.x.abs_()
    layer.router.abs_()
    layer.router[1] = layer.router[1].bfloat16().float() * 4
    layer.router[6] = layer.router[1] * (1 + 2.0 ** -14)
    with torch.autocast("cuda", enabled=False):
        want, allowed = definition(layer)
        assert (layer.exact()[2] == 6).all()
    for got in ways(layer):
        near(got, want, allowed)
    x, router = layer.x.repeat(4, 1).requires_grad_(), layer.router.clone().requires_grad_()
    from fgms_b200 import nn
    grads = torch.autograd.grad(nn.expert_layer(x, router, layer.w_in, layer.w_out, 3).float().square().sum(), (x, router))
    assert all(torch.isfinite(g).all() for g in grads) and grads[1].abs().amax(1)[[1, 6]].min() > 0
    assert nn.expert_layer(x[:0], router, layer.w_in, layer.w_out, 3).shape == (0, 256)
