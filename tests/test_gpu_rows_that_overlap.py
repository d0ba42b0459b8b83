"""Rows that share memory (expanded ones) are inputs like any others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expanded_rows(dtype):
    from fgms_b200 import nn
    x, w, res = torch.randn(72, device="cuda").to(dtype), torch.rand(72, device="cuda").to(dtype), torch.randn((10, 72), device="cuda").to(dtype)
    windows = torch.randn(200, device="cuda").to(dtype).as_strided((10, 72), (3, 1))
    for rows in (x.expand(10, 72), windows, x[:1].expand(10, 1)):
        weight, other = w[:rows.size(1)], res[:, :rows.size(1)]
        dense = rows.contiguous()
        for call in (lambda t: nn.quantize_rows(t), lambda t: nn.rms_norm_int8(t, weight, residual=other), lambda t: nn.rms_norm(t, weight, residual=other),
                     lambda t: nn.rms_norm(other, weight, residual=t), lambda t: (nn.dropout(t, 0.5, nn.rng_state(1), residual=t),)):
            assert all(torch.equal(a, b) for a, b in zip(call(rows), call(dense)))
