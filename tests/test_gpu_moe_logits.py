"""sg_moe_route's logits: sums in 64 bits, rounded to fp32 once.  Inputs are multiples of powers of two so that every sum is exact in 64
bits, in whatever order; the choice has to be the order of those sums rounded to fp32, with no room for another."""
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sg():
    import rocm_dev_amd
    return rocm_dev_amd


def routed(sg, X, R, top_k, layer=False):
    ids = torch.full((X.shape[0], top_k), -7, dtype=torch.int32, device="cuda")
    weights = torch.full((X.shape[0], top_k), -7.0, device="cuda")
    if layer:
        hidden, experts = X.shape[1], R.shape[0]
        W1 = torch.zeros((experts, 32, hidden), dtype=torch.uint8, device="cuda")
        W2 = torch.zeros((experts, hidden, 16), dtype=torch.uint8, device="cuda")
        assert sg.moe_layer(X, R, W1, W2, torch.empty_like(X), ids, weights) == 0
    else:
        assert sg.moe_route(X, R, ids, weights) == 0
    torch.cuda.synchronize()
    return ids, weights


def check(ids, weights, X, R, top_k):
    logits = (X.double().cpu() @ R.double().cpu().t()).float()
    order = logits.sort(dim=1, descending=True, stable=True)
    assert torch.equal(ids.cpu().long(), order.indices[:, :top_k])
    want = torch.softmax(order.values[:, :top_k].double(), 1)
    # differences of fp32 logits, rounded by half a unit of at most 128, the exponential's rounding, a sum of at most 16 terms, a quotient
    assert ((weights.double().cpu() - want).abs() <= want * 2.0 ** -16 + 2.0 ** -126).all()


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("m", [1, 8, 12])
@pytest.mark.parametrize("hidden", [16, 64, 528, 4112])
def test_terms_that_cancel(sg, m, hidden, layer):
    """2^24 + 1 - 2^24 is 1, within eight columns and apart from each other, and beats 1/2."""
    experts = 12
    R = torch.zeros((experts, hidden), device="cuda")
    X = torch.ones((m, hidden), device="cuda")
    X[:, 0] = X[:, 2] = X[:, hidden - 1] = 4096
    X[:, 9] = 0.5
    R[:, 9] = 1                                              # 0.5 for all ...
    for e, (one, minus) in {3: (1, 2), 7: (1, hidden - 1), 10: (5, 2)}.items():
        R[e, 9] = 0
        R[e, 0], R[e, one], R[e, minus] = 4096, 1 + e / 16, -4096
    X, R = X.bfloat16(), R.bfloat16()
    ids, weights = routed(sg, X, R, 5, layer)
    assert ids.tolist() == [[10, 7, 3, 0, 1]] * m
    check(ids, weights, X, R, 5)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("m,experts,top_k,hidden", [(1, 256, 8, 4096), (7, 64, 6, 2048), (13, 512, 16, 4096), (64, 130, 8, 1040)])
def test_logits_a_unit_apart(sg, m, experts, top_k, hidden, layer):
    """Pairs of experts whose logits differ by about fp32's last bit, on activations with rare large entries."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(experts)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    X = (normal(m, hidden) * 64).round() / 64                # bf16 of a multiple of 2^-6 is one
    X = torch.where(torch.rand((m, hidden), generator=gen, device="cuda") < 0.01, (20 * X).round(), X).bfloat16()
    R = ((normal(experts, hidden) * 256).round() / 2048).bfloat16()
    # the second of a pair: the first, but for a few columns by the step of their values
    odd = R[1::2]
    odd.copy_(R[0::2][:odd.shape[0]])
    at = torch.randint(0, hidden, (odd.shape[0], 3), generator=gen, device="cuda")
    odd.scatter_(1, at, (odd.gather(1, at).float() + 2.0 ** -11 * torch.randint(-1, 2, at.shape, generator=gen, device="cuda")).bfloat16())
    # products are multiples of 2^-17 and sums below 2^20: 37 bits
    assert (X.double().abs() @ R.double().abs().t()).max() < 2 ** 20
    assert (X.float() * 64 == (X.float() * 64).round()).all() and (R.float() * 2048 == (R.float() * 2048).round()).all()
    ids, weights = routed(sg, X, R, top_k, layer)
    check(ids, weights, X, R, top_k)


def test_products_beyond_fp32(sg):
    """Products that overflow fp32 and cancel, and products below its smallest value that add up: in 64 bits both are held.  The order is that of
    the sums as fractions; 2^200 and -2^200 stand beside each other and in front of what they would swallow, so that 64 bits hold every sum."""
    R = torch.zeros((6, 32), device="cuda")
    X = torch.zeros((2, 32), device="cuda")
    X[0, 0] = X[0, 1] = 2.0 ** 100
    X[0, 2] = 1
    R[1, 0], R[1, 1], R[1, 2] = 2.0 ** 100, -2.0 ** 100, 3
    R[4, 0], R[4, 1], R[4, 2] = 2.0 ** 100, -2.0 ** 100, 5
    X[1] = 2.0 ** -100
    R[2] = 2.0 ** -50                                        # 2^-145 in token 1; in fp32 every product is a few steps
    R[5] = 2.0 ** -48 + 2.0 ** -55
    X, R = X.bfloat16(), R.bfloat16()
    ids, _ = routed(sg, X, R, 3)
    logits = [[sum(Fraction(x) * Fraction(r) for x, r in zip(row, expert)) for expert in R.double().tolist()] for row in X.double().tolist()]
    want = [sorted(range(6), key=lambda e: (-row[e], e))[:3] for row in logits]
    assert want == [[5, 2, 4], [4, 1, 5]] and ids.tolist() == want
