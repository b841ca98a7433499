"""sg_rmsnorm_fp8_rows on rows whose products or scales lie near fp32's smallest values, against the formula in 64 bits."""
import pytest
import torch
from test_gpu_norm import check, expected, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sg():
    import rocm_dev_amd
    return rocm_dev_amd


@pytest.mark.parametrize("cols", [64, 1040, 8192, 65552])
@pytest.mark.parametrize("v", [-62, -60, -55, -48])
def test_means_below_the_normal_range(sg, cols, v):
    """eps = 0: two values in a row of zeros, whose squares fp32 holds to all bits, and a row of zeros and one full of such values."""
    X = torch.zeros((4, cols), device="cuda")
    X[0, 7], X[0, cols - 1] = 2.0 ** v, -1.25 * 2.0 ** v
    X[1] = 1.5 * 2.0 ** v
    X[3, 3] = 1.75 * 2.0 ** v
    X = X.bfloat16()
    _, y = expected(X, None, None, 0.0)
    rows = [0, 1, 3]                                # (a row of zeros is 0 / 0)
    Q, s, _, Y = run(sg, X, eps=0.0)
    check(Q[rows], s[rows], Y[rows], y[rows])
