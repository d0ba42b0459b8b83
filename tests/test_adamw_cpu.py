"""What the AdamW step refuses, before it touches a device."""
import ctypes

import pytest
import torch

from fgms_b200 import _lib, optim

P = 1 << 20  # never dereferenced: validation fails first


def call(n=2, options=(), **tensor):
    o = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=64 * P, state_bits=8)
    o.update(options)
    list_ = (_lib.AdamwTensor * 2)()
    for i, t in enumerate(list_):
        fields = dict(param=(10 * i + 1) * P, grad=(10 * i + 2) * P, exp_avg=(10 * i + 3) * P, exp_avg_sq=(10 * i + 4) * P,
                      exp_avg_scale=(10 * i + 5) * P, exp_avg_sq_scale=(10 * i + 6) * P, count=100, param_dtype=0, grad_dtype=0)
        if i == 1:
            fields.update(tensor)
        for k, v in fields.items():
            setattr(t, k, v)
    return _lib.lib.fgms_b200_adamw(list_, n, ctypes.byref(_lib.AdamwOptions(**o)), None)


@pytest.mark.parametrize("options,tensor,text", [
    (dict(lr=-1.0), {}, "lr"), (dict(lr=float("inf")), {}, "lr"), (dict(lr=float("nan")), {}, "lr"),
    (dict(beta1=1.0), {}, "betas"), (dict(beta2=float("nan")), {}, "betas"), (dict(eps=0.0), {}, "eps"), (dict(eps=1e-50), {}, "eps"),
    (dict(weight_decay=-0.1), {}, "weight_decay"), (dict(state_bits=16), {}, "state_bits"), (dict(step=None), {}, "null"),
    (dict(step=64 * P + 2), {}, "aligned"), (dict(grad_scale=P // 2 + 1), {}, "aligned"),
    ({}, dict(param=None), "tensor 1: null"), ({}, dict(grad=None), "tensor 1: null"), ({}, dict(exp_avg_scale=None), "tensor 1: null"),
    ({}, dict(count=-1), "count"), ({}, dict(count=1 << 41), "count"), ({}, dict(param_dtype=3), "dtype"), ({}, dict(grad_dtype=-1), "dtype"),
    ({}, dict(param=11 * P + 2), "boundary"), ({}, dict(param=11 * P + 1, param_dtype=1), "boundary"),
    ({}, dict(param=P), "overlaps"), ({}, dict(param=P + 396), "overlaps"), ({}, dict(grad=P + 4), "overlaps"), ({}, dict(exp_avg=14 * P + 99), "overlaps"),
    ({}, dict(exp_avg_scale=64 * P), "overlaps"), (dict(grad_scale=11 * P + 8), {}, "overlaps"),
])
def test_refusals(options, tensor, text):
    assert call(options=options, **tensor) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), _lib.last_error()


def test_null_lists():
    o = _lib.AdamwOptions(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=P, state_bits=32)
    assert _lib.lib.fgms_b200_adamw(None, 1, ctypes.byref(o), None) == _lib.ERR_INVALID_ARG
    assert _lib.lib.fgms_b200_adamw(None, 0, None, None) == _lib.ERR_INVALID_ARG
    assert _lib.lib.fgms_b200_adamw(None, -1, ctypes.byref(o), None) == _lib.ERR_INVALID_ARG


def test_parameters_on_the_host_are_refused():
    w = torch.nn.Parameter(torch.zeros(4))
    w.grad = torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([w]).step()
    with pytest.raises(ValueError):
        optim.AdamW([w], state_bits=4)
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])
