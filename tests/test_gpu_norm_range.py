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


# 448 / max|v * w| is beyond fp32's largest value below 2^-119.2, wherever rstd leaves the scale itself
@pytest.mark.parametrize("cols", [64, 1040, 8192, 65552])
@pytest.mark.parametrize("v,w,eps", [(-120, 0, 1e-6), (-120, None, 1e-8), (-119, 0, 1e-5), (-126, 0, 1e-12), (-60, -60, 0.0), (-50, -73, 0.0), (-62, -48, 0.0)])
def test_small_products_with_a_scale_in_range(sg, cols, v, w, eps):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(cols)
    X = ((torch.rand((5, cols), generator=gen, device="cuda") * 2 - 1) * 2.0 ** v).bfloat16()
    X[:, ::5] = 0
    X[2] = 0
    X[2, 7], X[2, 8] = 2.0 ** v, -2.0 ** v
    weight = None if w is None else torch.full((cols,), 2.0 ** w, device="cuda").bfloat16()
    _, y = expected(X, weight, None, eps)
    Q, s, _, Y = run(sg, X, weight, eps=eps)
    check(Q, s, Y, y)
    assert not Q[:, ::5].view(torch.float8_e4m3fn).float().any()
    assert Q[2, 7] == 0x7e and Q[2, 8] == 0xfe


@pytest.mark.parametrize("cols", [64, 1040, 65552])
@pytest.mark.parametrize("w", range(-80, -64))
def test_scales_at_the_end_of_the_range(sg, cols, w):
    """eps = 1 makes the root 1 to fp32's last bit: y is v * w, at most 2^(w - 70).  The scale is a multiple of 2^-149, or, where
    448ths of the largest are nearer to zero, 1; codes are of y over that scale, cut off at 448."""
    X = torch.tensor([0, 1, -1, 0.5, -0.75, 0.125, 2.0 ** -6, 0], device="cuda").mul(2.0 ** -70).bfloat16().repeat(3, cols // 8)
    weight = torch.full((cols,), 2.0 ** w, device="cuda").bfloat16()
    Q, s, _, _ = run(sg, X, weight, eps=1.0)
    y = X.double() * 2.0 ** w
    want = 2.0 ** (w - 70) / 448
    steps = round(want * 2.0 ** 149)                # (no 448th of a power of two lies between two multiples)
    assert (s.double() == (steps * 2.0 ** -149 if steps else 1.0)).all()
    codes = (y / s.double()[:, None]).clamp(-448, 448).float().to(torch.float8_e4m3fn)
    assert torch.equal(Q.view(torch.float8_e4m3fn).float(), codes.float())
