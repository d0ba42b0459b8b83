"""What the grouped products refuse, before they touch a device."""
import os
import shutil
import subprocess

import pytest
import torch

from fgms_b200 import _lib, backend, nn

P = 1 << 20  # never dereferenced: validation fails first


def fwd(x=P, w=2 * P, out=3 * P, kpos=4 * P, rows=10, c_in=8, c_out=8, groups=4, dtype=_lib.DTYPE_BF16):
    return _lib.lib.fgms_b200_grouped_fwd(x, w, out, kpos, rows, c_in, c_out, groups, dtype, 0, None, 0, None)


@pytest.mark.parametrize("args,text", [
    (dict(rows=-1), "negative row count"),
    (dict(c_in=0), "channel counts"),
    (dict(c_out=-3), "channel counts"),
    (dict(groups=0), "groups 0 outside"),
    (dict(groups=1025), "groups 1025 outside"),
    (dict(groups=1024, c_in=1 << 21), "int32 range"),
    (dict(groups=1024, c_out=1 << 21), "int32 range"),
    (dict(dtype=3), "unknown dtype"),
    (dict(dtype=-1), "unknown dtype"),
    (dict(kpos=None), "null pointer"),
    (dict(x=None), "null pointer"),
    (dict(w=None), "null pointer"),
    (dict(out=None), "null pointer"),
    (dict(out=P + 16), "overlaps"),
    (dict(out=2 * P + 8), "overlaps"),
    (dict(out=4 * P - 2), "overlaps"),
])
def test_forward_refuses(args, text):
    assert fwd(**args) == _lib.ERR_INVALID_ARG and text in _lib.last_error()


def test_gradients_refuse():
    L = _lib.lib
    assert L.fgms_b200_grouped_dgrad(P, 2 * P, 2 * P, 4 * P, 10, 8, 8, 4, 1, 0, None, 0, None) == _lib.ERR_INVALID_ARG and "overlaps" in _lib.last_error()
    assert L.fgms_b200_grouped_dgrad(P, 2 * P, 3 * P, None, 10, 8, 8, 4, 1, 0, None, 0, None) == _lib.ERR_INVALID_ARG
    assert L.fgms_b200_grouped_wgrad(P, 2 * P, None, 4 * P, 10, 8, 8, 4, 1, None, 0, None) == _lib.ERR_INVALID_ARG
    assert L.fgms_b200_grouped_wgrad(P, 2 * P, 2 * P, 4 * P, 10, 8, 8, 4, 1, None, 0, None) == _lib.ERR_INVALID_ARG and "overlaps" in _lib.last_error()
    assert L.fgms_b200_grouped_wgrad(None, None, 3 * P, 4 * P, 10, 8, 8, 4, 1, None, 0, None) == _lib.ERR_INVALID_ARG


def test_nothing_to_write_is_no_error():
    assert fwd(x=None, out=None, rows=0) == _lib.OK
    assert _lib.lib.fgms_b200_grouped_dgrad(None, P, None, 2 * P, 0, 8, 8, 4, 0, 0, None, 0, None) == _lib.OK


def test_the_operator_of_a_map_still_refuses_bf16():
    assert _lib.lib.fgms_b200_fusion_fwd(None, None, None, None, None, None, None, 0, 4, 4, 8, 8, 8, 27, 0, _lib.DTYPE_BF16, 0, 0, None) == _lib.ERR_INVALID_ARG


def test_tensors_on_the_host_are_refused():
    x, w, out, kpos = torch.zeros(4, 8), torch.zeros(2, 8, 16), torch.zeros(4, 16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        backend.fgms_grouped_fwd_cuda(x, w, out, kpos)
    with pytest.raises(ValueError, match="CUDA"):
        backend.fgms_grouped_dgrad_cuda(out, w, x, kpos)
    with pytest.raises(ValueError, match="CUDA"):
        backend.fgms_grouped_wgrad_cuda(x, out, w, kpos)
    with pytest.raises(ValueError, match="CUDA"):
        nn.grouped_linear(x, w, kpos)
    with pytest.raises(TypeError):
        backend.fgms_grouped_fwd_cuda(None, w, out, kpos)
    with pytest.raises(ValueError, match="int32"):
        nn.grouped_linear(x, w, None)


def test_workspace_for_rows_off_a_boundary():
    """None where none is needed (whole rows of 16 bytes, fp32), where the call is too small for copies to pay, or where nothing is right."""
    q = _lib.lib.fgms_b200_grouped_workspace_bytes
    F16, BF16, F32 = _lib.DTYPE_F16, _lib.DTYPE_BF16, _lib.DTYPE_F32
    assert q(0, P, P, P, 5000, 1024, 1024, 8, F16) == 0
    assert q(0, P, P, P, 5000, 1001, 1003, 8, F32) == 0
    assert q(0, P, P, P, 5, 1001, 1003, 8, F16) == 0
    up = lambda rows, width: (rows * width * 2 + 255) // 256 * 256
    assert q(0, P, P, P, 5000, 1001, 1003, 8, BF16) == up(5000, 1008) + up(8 * 1001, 1008) + up(5000, 1008)
    assert q(1, P, P, P, 5000, 1024, 1003, 8, F16) == up(5000, 1008) + up(8 * 1024, 1008)   # in_grad has whole rows
    assert q(2, P, P, P, 5000, 1003, 1024, 8, F16) == up(5000, 1008)
    assert q(0, P + 2, P, P, 5000, 1024, 1024, 8, F16) == up(5000, 1024)                    # a view
    assert q(0, P, P, P + 8, 5000, 1024, 1024, 8, F16) == up(5000, 1024)
    assert q(3, P, P, P, 5000, 1001, 1003, 8, F16) == 0 and q(0, P, P, P, 0, 1001, 1003, 8, F16) == 0 and q(0, P, P, P, 5, 0, 3, 8, F16) == 0


MOST = 0x7fffffff - 1024


@pytest.mark.parametrize("size", ["rows", "c_in", "c_out"])
def test_rows_and_channels_whose_steps_an_int_does_not_hold_are_refused(size):
    """The kernels go from the first to behind the last in steps of up to 256."""
    for n in (MOST + 1, 0x7fffffff):
        sizes = {"rows": 10, "c_in": 8, "c_out": 8, "groups": 1, **{size: n}}
        assert fwd(**sizes) == _lib.ERR_INVALID_ARG and "more than" in _lib.last_error()
        dims = (sizes["rows"], sizes["c_in"], sizes["c_out"], 1, _lib.DTYPE_BF16)
        assert _lib.lib.fgms_b200_grouped_dgrad(P, 2 * P, 3 * P, 4 * P, *dims, 0, None, 0, None) == _lib.ERR_INVALID_ARG and "more than" in _lib.last_error()
        assert _lib.lib.fgms_b200_grouped_wgrad(P, 2 * P, 3 * P, 4 * P, *dims, None, 0, None) == _lib.ERR_INVALID_ARG and "more than" in _lib.last_error()
        assert _lib.lib.fgms_b200_grouped_workspace_bytes(0, P + 2, 2 * P, 3 * P, *dims) == 0
    assert fwd(**{"groups": 1, size: MOST}) == _lib.ERR_INVALID_ARG and "overlaps" in _lib.last_error()  # taken, were it not for these addresses


def program(name, tmp_path):
    """The program ``tests/plans/<name>.cu``: a function that runs it and returns what it prints."""
    nvcc = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
    if not (os.path.exists(nvcc) or shutil.which(nvcc)):
        pytest.skip("nvcc not available")
    exe = str(tmp_path / name)
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "plans", name + ".cu")
    build = subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-o", exe, src], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout + build.stderr

    def run(*args):
        done = subprocess.run([exe, *map(str, args)], capture_output=True, text=True, timeout=60)
        assert done.returncode == 0, done.stdout + done.stderr
        return done.stdout
    return run


def test_shares_of_a_group(tmp_path):
    """How a group's rows are shared out over its tiles, up to the most rows there may be."""
    program("grouped_share", tmp_path)()


def test_the_cut_does_not_depend_on_the_calls_before(tmp_path):
    """Clusters of eight for one row 4096 -> 1024: in a fresh process, behind a call with fewer parts, and once a question that failed is answered."""
    run = program("grouped_limit", tmp_path)
    alone = run(0, 0)
    assert "clusters of 8" in alone
    assert run(1, 0) == alone
    assert run(2, 3) == alone


@pytest.mark.parametrize("dtype,off", [(_lib.DTYPE_BF16, 1), (_lib.DTYPE_F16, 3), (_lib.DTYPE_F32, 2)])
def test_pointers_off_a_boundary_of_their_type_are_refused(dtype, off):
    for name, at in (("x", P), ("w", 2 * P), ("out", 3 * P)):
        assert fwd(**{name: at + off}, dtype=dtype) == _lib.ERR_INVALID_ARG and "boundary" in _lib.last_error()
    assert fwd(kpos=4 * P + 2, dtype=dtype) == _lib.ERR_INVALID_ARG and "boundary" in _lib.last_error()
    for call, tail in ((_lib.lib.fgms_b200_grouped_dgrad, (0, None, 0, None)), (_lib.lib.fgms_b200_grouped_wgrad, (None, 0, None))):
        assert call(P + off, 2 * P, 3 * P, 4 * P, 10, 8, 8, 4, dtype, *tail) == _lib.ERR_INVALID_ARG and "boundary" in _lib.last_error()


@pytest.mark.parametrize("source", ["grouped.cuh", "grouped_umma.cuh", "grouped_ffma.cuh", "grouped_pitch.cuh", "adamw.cuh"])
def test_nothing_behind_is_let_go_early_with_sms_kept_free(source):
    """``fgms_b200_set_reserved_sms``: what is enqueued behind a launch starts when it has ended, so no kernel lets it go before."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "fgms_b200", "csrc", source)) as f:
        for line in f:
            if "griddep_launch_dependents()" in line:
                assert "if (!p.alone)" in line or "if (!alone)" in line, line
