"""sg_int4_gemm on activations at the ends of bf16's range, against the formula in 64 bits."""
import pytest
import torch
from test_gpu_int4 import Weights, activations, check, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sg():
    import rocm_dev_amd
    return rocm_dev_amd


def weights(sg, n, k, group, zeros, f16, scale):
    w = Weights(sg, n, k, group, zeros, f16, seed=group)
    w.S[:] = scale * (1 + torch.arange(w.S.numel(), device="cuda").remainder(7).view_as(w.S) / 8)
    if zeros:
        w.Z[:] = torch.arange(w.Z.numel(), device="cuda").remainder(256).view_as(w.Z).byte()       # up to 255, as they are
    sg.int4_pack(w.B, w.S, w.P, w.Z, check=True)
    return w


# every build by its rows: activations to themselves, shared by waves; whole K and parts of it
@pytest.mark.parametrize("n,k", [(48, 256), (512, 16384)])
@pytest.mark.parametrize("m", [1, 5, 13, 30, 64])
@pytest.mark.parametrize("group,zeros,f16", [(32, True, False), (64, False, True), (128, False, False), (128, True, True)])
@pytest.mark.parametrize("signs", [False, True])
def test_no_sum_inside_overflows(sg, m, n, k, group, zeros, f16, signs):
    """Every activation within a factor of four of bf16's largest value, of one sign or of both: a group's 128 * 2^128 is beyond fp32 long before
    the scales bring the result back."""
    w = weights(sg, n, k, group, zeros, f16, 2.0 ** -24)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m)
    A = ((1 + 0.99 * torch.rand((m, k), generator=gen, device="cuda", dtype=torch.float64)) * 2.0 ** torch.randint(126, 128, (m, k), generator=gen, device="cuda")).bfloat16()
    assert A.isfinite().all()
    if signs:
        A = torch.where(torch.rand((m, k), generator=gen, device="cuda") < 0.5, -A, A)
    D = run(sg, A, w)
    ref, tol = w.expected(A)
    assert ref.abs().max() < 2.0 ** 127
    assert D.isfinite().all() and ((D.double() - ref).abs() <= tol).all()


def test_of_one_group_at_2_to_121(sg):
    w = weights(sg, 33, 128, 128, False, False, 2.0 ** -10)
    A = torch.full((3, 128), 2.0 ** 121, device="cuda").bfloat16()
    D = run(sg, A, w)
    ref, tol = w.expected(A)
    assert D.isfinite().all() and ((D.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("m", [1, 5, 13, 30, 64])
@pytest.mark.parametrize("group", [32, 128])
def test_small_activations(sg, m, group):
    """Activations around 2^-90: nothing inside is rounded but to fp32's 24 bits."""
    w = weights(sg, 100, 512, group, True, False, 1.0)
    check(sg, (activations(m, 512, seed=3).float() * 2.0 ** -90).bfloat16(), w)
