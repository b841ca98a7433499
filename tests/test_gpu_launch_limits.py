"""Rows beyond what one launch has threads for: the first and the last ones, and those where launches meet, against the same rows by themselves."""
import pytest
import torch
from test_gpu_norm import operands

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sg():
    import rocm_dev_amd
    yield rocm_dev_amd
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols", [16, 144, 528])
def test_norm(sg, cols):
    rows, part = 2 ** 22 + 99, 200
    X, weight, residual = operands(part, cols, seed=cols)
    small = [torch.empty((part, cols), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(part, device="cuda"), torch.empty_like(X), torch.empty_like(X)]
    assert sg.rmsnorm_fp8_rows(X, small[0], small[1], weight, residual, small[2], small[3], 1e-5) == 0
    times = -(-rows // part)
    big = [torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(rows, device="cuda"),
           torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")]
    assert sg.rmsnorm_fp8_rows(X.repeat(times, 1)[:rows], big[0], big[1], weight, residual.repeat(times, 1)[:rows], big[2], big[3], 1e-5) == 0
    for b, s in zip(big, small):
        b, s = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (b, s))
        for first in (0, 2 ** 21 - 300, 2 ** 22 - 300, rows - 300):
            at = torch.arange(first, min(first + 600, rows), device="cuda")
            # (64 threads a row and fewer add the squares up in one order whatever the rows)
            assert torch.equal(b[at], s[at % part])


def test_products_of_many_rows(sg):
    m, n, k, group = 2 ** 29 + 77, 16, 32, 32
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    B = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    S = (torch.rand((n, 1), generator=gen, device="cuda") + 0.1).bfloat16()
    P = torch.empty(sg.int4_packed_bytes(n, k, group), dtype=torch.uint8, device="cuda")
    sg.int4_pack(B, S, P, check=True)
    A = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    part = torch.randn((640, k), generator=gen, device="cuda").bfloat16()
    places = [0, 2 ** 27 - 320, 2 ** 28 - 320, m - 640]        # (launches meet at 2^28 + 64)
    for at in places:
        A[at:at + 640] = part
    D = torch.full((m, n), -7.0, dtype=torch.bfloat16, device="cuda")
    assert sg.int4_gemm(A, P, D, group=group) == 0
    q = torch.stack((B & 15, B >> 4), 2).reshape(n, k).double() - 8
    want = part.double() @ (q * S.double()).t()
    for at in places:
        # half a bf16 step, and 2^-23 for each of 2 * 32 + 8 steps of terms up to 16 |s| (3 + 8 / 8) |a|
        tol = 2.0 ** -8 * want.abs() + 2.0 ** -23 * 72 * (part.double().abs().sum(1, keepdim=True) * 64 * S.double().t())
        assert ((D[at:at + 640].double() - want).abs() <= tol).all()
        assert torch.equal(D[at:at + 640], D[:640])
    assert not D[640:100000].any() and not D[2 ** 28 + 320:2 ** 28 + 10 ** 6].any()


def test_pack_of_many_rows(sg):
    n, k = 2 ** 30 + 53, 128
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    B = torch.zeros((n, k // 2), dtype=torch.uint8, device="cuda")
    S = torch.zeros((n, 1), dtype=torch.bfloat16, device="cuda")
    part = 533
    codes = torch.randint(0, 256, (part, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (torch.rand((part, 1), generator=gen, device="cuda") + 0.1).bfloat16()
    for at in (0, n - part):                                 # (the last ones across the 2^30 - 64, where launches meet)
        B[at:at + part], S[at:at + part] = codes, scales
    P = torch.full((sg.int4_packed_bytes(n, k, 128),), 0x5a, dtype=torch.uint8, device="cuda")
    sg.int4_pack(B, S, P, check=True)
    A = torch.randn((2, k), generator=gen, device="cuda").bfloat16()
    D = torch.full((2, n), -7.0, dtype=torch.bfloat16, device="cuda")
    assert sg.int4_gemm(A, P, D) == 0
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(part, k).double() - 8
    want = A.double() @ (q * scales.double()).t()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -23 * 2 * 136 * (A.double().abs().sum(1, keepdim=True) * 64 * scales.double().t())
    for at in (0, n - part):
        assert ((D[:, at:at + part].double() - want).abs() <= tol).all()
    assert not D[:, part:10 ** 6].any() and not D[:, n - 10 ** 6:n - part].any()
