"""Norm, dropout and rows in 8 bits: the generator's definition, and what is refused before a device is touched."""
import ctypes

import numpy as np
import pytest
import torch

from fgms_b200 import _lib, backend, nn
from tests.layers_ref import kept, philox

P = 1 << 20  # never dereferenced: validation fails first
L = _lib.lib


def test_the_generator_is_philox():
    """Known answers of Philox 4x32-10."""
    full = 0xFFFFFFFF
    assert philox(np.zeros((1, 4), np.uint64), (0, 0)).tolist() == [[0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]]
    assert philox(np.full((1, 4), full, np.uint64), (full, full)).tolist() == [[0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]]
    pi = [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344]
    assert philox(np.array([pi], np.uint64), (0xA4093822, 0x299F31D0)).tolist() == [[0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]]


def test_the_mean_is_kept():
    """Of 200000 values with p = 0.3 the kept ones are within six standard deviations of what they should be."""
    m = kept(400, 500, 0.3, 12345, 2)
    p = round(0.3 * 65536) / 65536
    n = m.size
    assert abs((m > 0).sum() - n * (1 - p)) < 6 * (n * p * (1 - p)) ** 0.5
    assert not np.array_equal(m, kept(400, 500, 0.3, 12345, 3)) and not np.array_equal(m, kept(400, 500, 0.3, 12346, 2))


def norm(**change):
    a = _lib.RmsNormArgs(x=P, weight=2 * P, out=3 * P, x_pitch=64, residual_pitch=64, out_pitch=64, sum_pitch=64, rows=4, width=64, eps=1e-6, p=0.0,
                         dtype=_lib.DTYPE_BF16, weight_dtype=_lib.DTYPE_BF16)
    for k, v in change.items():
        setattr(a, k, v)
    return L.fgms_b200_rms_norm(ctypes.byref(a), None)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "x: null"), (dict(out=None), "out: null"), (dict(weight=None), "weight: null"),
    (dict(rows=-1), "rows -1"), (dict(rows=2 ** 31), "rows"), (dict(width=0), "width 0"), (dict(width=32769), "width 32769"),
    (dict(dtype=5), "unknown dtype"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(p=-0.1), "probability"), (dict(p=1.5), "probability"), (dict(p=float("nan")), "probability"),
    (dict(p=0.5), "rng: null"), (dict(p=0.5, rng=4 * P + 4), "rng is not on a boundary"), (dict(x_pitch=63), "apart"), (dict(x=P + 1), "boundary"),
    (dict(scale=4 * P + 2), "scale is not on a boundary"), (dict(weight=2 * P + 1), "boundary"),
    (dict(out=P + 2), "overlaps"), (dict(out=2 * P - 4), "overlaps"), (dict(residual=5 * P, sum=5 * P + 32), "overlaps"), (dict(sum=3 * P), "two outputs"),
    (dict(rstd=2 * P + 16), "overlaps"), (dict(scale=3 * P + 16), "two outputs"), (dict(p=0.5, rng=3 * P + 8), "two outputs"),
    (dict(p=0.5, rng=4 * P, rng_used=4 * P + 8), "two outputs"), (dict(out=P, x_pitch=128), "overlaps"), (dict(scale=4 * P, out=P), "overlaps"),
])
def test_the_norm_refuses(change, text):
    assert norm(**change) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), _lib.last_error()


def test_the_norm_refuses_what_it_is_not_built_for():
    assert norm(weight_dtype=_lib.DTYPE_F16) == _lib.ERR_UNSUPPORTED
    assert norm(scale=4 * P, p=0.5, rng=5 * P) == _lib.ERR_UNSUPPORTED and "8 bits" in _lib.last_error()
    assert L.fgms_b200_rms_norm(None, None) == _lib.ERR_INVALID_ARG


def test_no_rows_are_no_error():
    assert norm(rows=0, x=None, out=None) == _lib.OK
    assert drop(rows=0, x=None, out=None) == _lib.OK
    assert L.fgms_b200_quantize_rows(None, 64, None, 64, None, 0, 64, _lib.DTYPE_F32, None) == _lib.OK


def test_the_gradient_refuses():
    def bwd(**change):
        a = _lib.RmsNormBwdArgs(out_grad=P, sum=2 * P, weight=3 * P, rstd=4 * P, x_grad=5 * P, rows=4, width=64, p=0.0, dtype=_lib.DTYPE_F16,
                                weight_dtype=_lib.DTYPE_F32, **{n: 64 for n in ("out_grad_pitch", "sum_pitch", "sum_grad_pitch", "x_grad_pitch",
                                                                               "residual_grad_pitch")})
        for k, v in change.items():
            setattr(a, k, v)
        return L.fgms_b200_rms_norm_bwd(ctypes.byref(a), None)

    for change, text in ((dict(out_grad=None), "out_grad: null"), (dict(sum=None), "sum: null"), (dict(rstd=None), "rstd: null"), (dict(weight=None), "weight: null"),
                         (dict(width=32769), "width"), (dict(rows=-3), "rows"), (dict(p=2.0), "probability"), (dict(p=0.5), "rng_used: null"),
                         (dict(dtype=9), "dtype"), (dict(x_grad_pitch=3), "apart"), (dict(residual_grad=6 * P + 1), "boundary")):
        assert bwd(**change) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), _lib.last_error()
    assert bwd(weight_dtype=_lib.DTYPE_BF16) == _lib.ERR_UNSUPPORTED
    assert bwd(x=8 * P, weight_dtype=_lib.DTYPE_F16) == _lib.ERR_UNSUPPORTED and "x is read" in _lib.last_error()
    assert bwd(x=8 * P + 1, x_pitch=64) == _lib.ERR_INVALID_ARG and "x is not" in _lib.last_error()
    assert L.fgms_b200_rms_norm_bwd(None, None) == _lib.ERR_INVALID_ARG
    assert L.fgms_b200_rms_norm_bwd_workspace_bytes(0, 64) == 0 and L.fgms_b200_rms_norm_bwd_workspace_bytes(4, 40000) == 0


def drop(backward=False, **change):
    a = _lib.DropoutArgs(x=P, out=2 * P, x_pitch=64, residual_pitch=64, out_pitch=64, rows=4, width=64, rng=3 * P, p=0.5, dtype=_lib.DTYPE_F32)
    for k, v in change.items():
        setattr(a, k, v)
    return (L.fgms_b200_dropout_bwd if backward else L.fgms_b200_dropout)(ctypes.byref(a), None)


@pytest.mark.parametrize("change,text", [
    (dict(x=None), "x: null"), (dict(out=None), "out: null"), (dict(rng=None), "rng: null"), (dict(rng=3 * P + 4), "rng is not"), (dict(rows=-1), "rows"),
    (dict(width=0), "width"), (dict(width=2 ** 31), "width"), (dict(p=-0.5), "probability"), (dict(p=1.01), "probability"), (dict(dtype=-1), "dtype"),
    (dict(out=P + 4), "overlaps"), (dict(residual=2 * P + 128), "overlaps"), (dict(rng=2 * P + 8), "state"), (dict(rng_used=P), "state"),
    (dict(rng_used=3 * P + 16), "rng_used overlaps"), (dict(x_pitch=60), "apart"), (dict(backward=True), "rng_used: null"),
])
def test_dropout_refuses(change, text):
    assert drop(**change) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), _lib.last_error()


def test_rows_in_8_bits_refuse():
    q = lambda x=P, codes=2 * P, scale=3 * P, rows=4, width=64, dtype=0, pitch=64: L.fgms_b200_quantize_rows(x, pitch, codes, 64, scale, rows, width, dtype, None)
    for kw, text in ((dict(x=None), "x: null"), (dict(codes=None), "out: null"), (dict(scale=None), "scale: null"), (dict(codes=P + 5), "overlaps"),
                     (dict(codes=P), "overlaps"), (dict(scale=2 * P + 4), "overlap"), (dict(dtype=3), "dtype"), (dict(width=0), "width"), (dict(pitch=63), "apart")):
        assert q(**kw) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), (kw, _lib.last_error())


def test_tensors_on_the_host_are_refused():
    x, w, rng = torch.zeros(4, 8), torch.ones(8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: nn.rms_norm(x, w), lambda: nn.rms_norm_int8(x, w), lambda: nn.quantize_rows(x), lambda: nn.dropout(x, 0.5, rng),
                 lambda: backend.fgms_rms_norm_cuda(x, w, x.clone()), lambda: backend.fgms_dropout_cuda(x, x.clone(), 0.5, rng)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: nn.rms_norm(None, w), lambda: nn.dropout(x, 0.5, None), lambda: nn.rms_norm(x, "weight")):
        with pytest.raises(TypeError, match="torch.Tensor"):
            call()


def test_modules_refuse():
    for make in (lambda: nn.Dropout(1.5, device="cpu"), lambda: nn.RMSNorm(8, dropout=-0.1, device="cpu"), lambda: nn.rng_state(-1, "cpu")):
        with pytest.raises(ValueError):
            make()
    assert nn.RMSNorm(8, device="cpu").rng is None and nn.rng_state(5, "cpu").tolist() == [5, 0, 0]


def product(codes=P, codes_pitch=64, scale=2 * P, kernel=3 * P, kernel_pitch=64, kernel_scale=4 * P, out=5 * P, kpos=6 * P, rows=4, c_in=64, c_out=32, groups=3,
            dtype=_lib.DTYPE_BF16, ws=None, ws_bytes=0):
    return L.fgms_b200_grouped_i8_fwd(codes, codes_pitch, scale, kernel, kernel_pitch, kernel_scale, out, kpos, rows, c_in, c_out, groups, dtype, 0, ws, ws_bytes, None)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "negative"), (dict(c_in=0), "channel counts"), (dict(c_out=-1), "channel counts"), (dict(c_in=131072), "131071"), (dict(groups=0), "groups 0"),
    (dict(groups=1025), "groups 1025"), (dict(groups=1024, c_out=1 << 21), "int32 range"), (dict(dtype=7), "dtype"), (dict(kpos=None), "kpos"),
    (dict(rows=2 ** 31 - 1024), "rows or channels"), (dict(rows=2 ** 31 - 1026, c_out=2 ** 20), "tiles"), (dict(codes=None), "codes: null"),
    (dict(kernel=None), "kernel: null"), (dict(out=None), "out: null"), (dict(scale=None), "code_scale: null"), (dict(kernel_scale=None), "kernel_scale: null"),
    (dict(out=5 * P + 1), "boundary"), (dict(scale=2 * P + 2), "boundary"), (dict(kpos=6 * P + 1), "boundary"), (dict(codes_pitch=63), "apart"),
    (dict(out=P + 128), "overlaps"), (dict(out=3 * P), "overlaps"), (dict(out=4 * P + 4), "overlaps"), (dict(out=6 * P), "overlaps"),
])
def test_products_in_8_bits_refuse(change, text):
    assert product(**change) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), _lib.last_error()


def test_products_in_8_bits_say_what_they_copy():
    size = L.fgms_b200_grouped_i8_workspace_bytes
    assert size(P, 64, 3 * P, 64, 4, 64, 32, 3) == 0 and size(P, 64, 3 * P, 64, 4, 50, 32, 3) == 0
    assert size(P + 1, 64, 3 * P, 64, 4, 64, 32, 3) == 256 and size(P, 50, 3 * P, 64, 4, 50, 32, 3) == 256
    assert size(P, 64, 3 * P, 65, 4, 64, 32, 3) == 3 * 32 * 64 and size(P + 1, 65, 3 * P, 65, 4, 64, 32, 3) == 256 + 3 * 32 * 64
    assert product(codes=P + 1) == _lib.ERR_WORKSPACE and product(codes=P + 1, ws=7 * P, ws_bytes=255) == _lib.ERR_WORKSPACE
    assert product(codes=P + 1, ws=7 * P + 16, ws_bytes=512) == _lib.ERR_WORKSPACE and product(codes=P + 1, ws=5 * P, ws_bytes=512) == _lib.ERR_WORKSPACE
    assert product(rows=0, codes=None, out=None, scale=None) == _lib.OK


def experts(**change):
    a = _lib.ExpertLayerArgs(x=P, router=2 * P, w_in=3 * P, w_out=4 * P, out=5 * P, chosen=6 * P, gates=7 * P, x_pitch=64, out_pitch=64, tokens=4, experts=8, top_k=2,
                             width=64, hidden=32, out_width=64, gated=1, activation=1, dtype=_lib.DTYPE_BF16, router_dtype=_lib.DTYPE_BF16)
    for k, v in change.items():
        setattr(a, k, v)
    return L.fgms_b200_expert_layer(ctypes.byref(a), None)


@pytest.mark.parametrize("change,text", [
    (dict(tokens=-1), "tokens -1"), (dict(tokens=65), "tokens 65"), (dict(experts=0), "experts 0"), (dict(experts=513), "experts 513"), (dict(top_k=0), "top_k 0"),
    (dict(top_k=9), "top_k 9"), (dict(top_k=17, experts=64), "top_k 17"), (dict(width=60), "multiples of 8"), (dict(hidden=0), "multiples of 8"),
    (dict(out_width=2 ** 20 + 8), "multiples of 8"), (dict(width=2 ** 20, hidden=2 ** 20, experts=512, x_pitch=2 ** 20), "too large"), (dict(activation=2), "activation"),
    (dict(x=None), "x: null"), (dict(router=None), "router: null"), (dict(w_in=None), "w_in: null"), (dict(w_out=None), "w_out: null"), (dict(out=None), "out: null"),
    (dict(chosen=None), "chosen: null"), (dict(gates=None), "gates: null"), (dict(x=P + 2), "16-byte"), (dict(x_pitch=68), "16-byte"), (dict(w_in=3 * P + 8), "16-byte"),
    (dict(out=5 * P + 1), "boundary"), (dict(chosen=6 * P + 2), "boundary"), (dict(x_pitch=56), "apart"), (dict(out=P + 64), "overlaps"), (dict(out=2 * P), "overlaps"),
    (dict(out=4 * P + 2), "overlaps"), (dict(chosen=P), "overlaps"), (dict(gates=6 * P + 16), "two outputs"), (dict(chosen=5 * P + 4), "two outputs"),
])
def test_a_layer_of_experts_refuses(change, text):
    assert experts(**change) == _lib.ERR_INVALID_ARG and text in _lib.last_error(), _lib.last_error()


def test_a_layer_of_experts_refuses_what_it_is_not_built_for():
    assert experts(dtype=_lib.DTYPE_F32, router_dtype=_lib.DTYPE_F32) == _lib.ERR_UNSUPPORTED
    assert experts(router_dtype=_lib.DTYPE_F16) == _lib.ERR_UNSUPPORTED and "router" in _lib.last_error()
    assert L.fgms_b200_expert_layer(None, None) == _lib.ERR_INVALID_ARG
    assert experts(tokens=0, x=None, out=None, chosen=None, gates=None) == _lib.OK
    size = L.fgms_b200_expert_layer_workspace_bytes
    assert size(0, 8, 2, 32, 64) == 0 and size(65, 8, 2, 32, 64) == 0 and size(4, 513, 2, 32, 64) == 0 and size(4, 8, 17, 32, 64) == 0
    with pytest.raises(ValueError, match="top_k"):
        nn.ExpertLayer(8, 8, 4, 5, device="cpu")
