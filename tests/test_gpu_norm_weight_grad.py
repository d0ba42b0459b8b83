"""The gradient of a weight in 16 bits is as exact as its type: it does not see how the sum was rounded where that was stored."""
import pytest
import torch

from tests.layers_ref import Norm, near
from tests.test_gpu_norm import SEED, Case, mask_of

pytestmark = pytest.mark.gpu

SHAPES = [(1, 8), (3, 5), (130, 64), (700, 512), (33, 257), (301, 1001), (400, 2056), (400, 5000), (160, 8200), (150, 16390), (2, 32768)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("weight", ["same", "fp32"])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_the_sum_is_not_rounded(dtype, weight, rows, width):
    from fgms_b200 import nn
    c = Case(dtype, rows, width, weight, seed=7 * rows + width)
    for residual, p in ((c.res, 0.0), (c.res, 0.25), (None, 0.25)):
        x, w = c.x.clone().requires_grad_(), c.w.clone().requires_grad_()
        res = None if residual is None else residual.clone().requires_grad_()
        got = nn.rms_norm(x, w, 1e-5, residual=res, dropout=p, rng=nn.rng_state(SEED) if p else None)
        ref = Norm(c.x, c.w, 1e-5, residual, mask_of(c, p) if p else None)
        ref.stored = 0.0
        leaves, out, flows = ((x, w), (got,), (c.dy,)) if residual is None else ((x, w, res), got, (c.dy, c.dsum))
        grads = torch.autograd.grad(out, leaves, flows)
        dx, dres, dw = ref.backward(c.dy, c.dsum if residual is not None else None, c.w.dtype)
        near(grads[0], *dx)
        near(grads[1], *dw)
        if residual is not None:
            near(grads[2], *dres)


def test_either_of_the_two_is_given():
    from fgms_b200 import backend
    c = Case("bf16", 50, 136)
    out, total, rstd = torch.empty_like(c.x), torch.empty_like(c.x), torch.empty(50, device="cuda")
    backend.fgms_rms_norm_cuda(c.x, c.w, out, 1e-5, residual=c.res, residual_out=total, rstd=rstd)
    ref = Norm(c.x, c.w, 1e-5, c.res)
    for stored, h in ((ref.unit, dict(h=total)), (0.0, dict(h=None, x=c.x, residual=c.res))):
        ref.stored = stored
        grads = torch.empty_like(c.x), torch.empty_like(c.x), torch.empty_like(c.w)
        backend.fgms_rms_norm_bwd_cuda(c.dy, weight=c.w, rstd=rstd, x_grad=grads[0], residual_grad=grads[1], weight_grad=grads[2], h_grad=c.dsum, **h)
        for got, want in zip(grads, ref.backward(c.dy, c.dsum, torch.bfloat16)):
            near(got, *want)
    f = Case("fp32", 50, 136)
    with pytest.raises(ValueError, match="x is read for rows in 16 bits"):
        backend.fgms_rms_norm_bwd_cuda(f.dy, None, f.w, rstd, x_grad=torch.empty_like(f.x), x=f.x)
