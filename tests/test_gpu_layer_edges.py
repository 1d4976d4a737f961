"""The layer operators at the edges of their range: the bounds are those of
test_gpu_layer.py unless a test derives its own."""
import pytest

from test_gpu_layer import forward_case, grad_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,xl", [(17, 4999, 4096, "plain"), (20, 2501, 4096, "plain"),
                                      (68, 5001, 4096, "plain"), (122, 5001, 8192, "plain"),
                                      (43, 4999, 4096, "transposed")])
def test_few_rows_into_an_odd_width(dtype, m, n, k, xl):
    """Wide split tiles whose rows leave through slabs: the most shared memory."""
    forward_case(dtype, m, n, k, "relu", None, False, True, False, m, xl)


def test_gradient_of_few_rows_and_an_odd_width():
    grad_case("bf16", 20, 4096, 2501, "none", None, 1)
