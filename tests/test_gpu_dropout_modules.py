"""Modules that drop values, several of them in one network."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_modules_at_their_defaults_drop_different_values():
    """Four modules over 20000 values each, p = 0.5.  Two masks that are independent agree in half of the values; 6 standard deviations of that are 6 sqrt(20000 / 4) = 425."""
    from fgms_b200 import nn
    x, w = torch.ones((100, 200), device="cuda"), torch.ones(200, device="cuda")
    drops = [nn.Dropout(0.5), nn.Dropout(0.5)]
    norms = [nn.RMSNorm(200, dropout=0.5), nn.RMSNorm(200, dropout=0.5)]
    masks = []
    for _ in range(2):  # two steps
        masks += [d(x) != 0 for d in drops] + [n(x, torch.zeros_like(x))[1].detach() != 0 for n in norms]
    for i in range(8):
        for j in range(i):
            assert abs((masks[i] == masks[j]).sum().item() - 10000) < 425, (i, j)
    torch.manual_seed(7)
    a = nn.Dropout(0.5)
    torch.manual_seed(7)
    b = nn.Dropout(0.5)
    assert torch.equal(a(x), b(x))
