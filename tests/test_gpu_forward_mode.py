"""Forward-mode differentiation is refused by what has none, instead of losing a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    from fgms_b200 import nn
    normal = lambda *s: torch.randn(s, device="cuda").bfloat16()
    x, res, w, rng = normal(20, 64), normal(20, 64), normal(64), nn.rng_state(1)
    router, w_in, w_out = normal(4, 64), normal(4, 64, 64), normal(4, 32, 64)
    codes, scale = nn.quantize_rows(x)
    kernel, kernel_scale = nn.quantize_rows(normal(32, 64))
    many = x.repeat(5, 1)
    calls = [
        (lambda d: nn.rms_norm(d(x), w)), (lambda d: nn.rms_norm(x, d(w))), (lambda d: nn.rms_norm(x, w, residual=d(res))), (lambda d: nn.rms_norm(d(x).requires_grad_(), w)),
        (lambda d: nn.rms_norm_int8(d(x), w)), (lambda d: nn.rms_norm_int8(x, d(w))), (lambda d: nn.rms_norm_int8(x, w, residual=d(res))), (lambda d: nn.quantize_rows(d(x))),
        (lambda d: nn.dropout(d(x), 0.5, rng)), (lambda d: nn.dropout(x, 0.5, rng, residual=d(res))),
        (lambda d: nn.int8_linear(codes, d(scale), kernel, kernel_scale)), (lambda d: nn.int8_linear(codes, scale, kernel, d(kernel_scale))),
        (lambda d: nn.expert_layer(d(x), router, w_in, w_out, 2)), (lambda d: nn.expert_layer(x, d(router), w_in, w_out, 2)),
        (lambda d: nn.expert_layer(x, router, d(w_in), w_out, 2)), (lambda d: nn.expert_layer(x, router, w_in, d(w_out), 2)),
        (lambda d: nn.expert_layer(d(many), router, w_in, w_out, 2)), (lambda d: nn.expert_layer(many, router, w_in, d(w_out), 2)),
    ]
    for call in calls:
        call(lambda t: t.clone())
    rng.copy_(nn.rng_state(1))
    with forward_ad.dual_level():
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                call(lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t)))
    assert rng.tolist() == [1, 0, 0]
