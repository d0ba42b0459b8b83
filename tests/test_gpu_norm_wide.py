"""Wide rows, more of them than there are SMs: with dropout a thread has two chunks of a row, and the gradient's blocks go from row to row."""
import pytest

from tests import test_gpu_norm as norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,weight", [("fp32", "same"), ("fp16", "same"), ("bf16", "fp32"), ("bf16", "same"), ("fp16", "fp32")])
@pytest.mark.parametrize("rows,width", [(400, 5000), (700, 8192), (301, 4104), (149, 8191)])
def test_forward_and_gradients(dtype, weight, rows, width):
    norm.test_forward_and_gradients(dtype, weight, rows, width)


@pytest.mark.parametrize("dtype", norm.TYPES)
@pytest.mark.parametrize("rows,width", [(400, 5000), (700, 8192), (149, 8191)])
def test_an_output_in_8_bits(dtype, rows, width):
    norm.test_an_output_in_8_bits(dtype, rows, width)
