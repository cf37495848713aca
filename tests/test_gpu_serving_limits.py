"""The serving operators on the GPU at the ends of their ranges: the longest K of
every type, scores and sums that float32 holds only just, infinities, and calls
that are captured, overlap or want gradients.  Values of the operators in float64
and the meaning of U are those of test_gpu_serving."""
import pytest

from test_gpu_serving import _types, _w4_case, _w4_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,pad", [(1, 0), (1, 1), (3, 0), (3, 1)])
def test_linear_w4_longest_k(cuda, dtype, group, M, pad):
    """K = 131072 in every type and group, rows of wq on and off 16-byte
    boundaries."""
    t = _types()[dtype]
    _w4_check(*_w4_case(cuda, M, 33, 131072, group, t, t, True, True, pad=pad), group)
