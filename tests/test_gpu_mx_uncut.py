"""E4M3 x MXFP4 products whose operands no matrix instruction cuts off (mx_uncut.py): as exact as MXFP4 x MXFP4 ones, and to the bit
where every partial sum fits fp32.  Other operands, against the same sums of products that are cut off as the instruction does."""
import numpy as np
import pytest
import torch

import mx_reference as ref
import mx_uncut
import rocm_dev_amd as sg
from rocm_dev_amd._lib import lib

pytestmark = pytest.mark.gpu

BUILDS = [1101, 1104, 1108, 1201, 1204, 1208, 1301, 1304, 1308, 1404, 1604, 1702, 1704, 2001, 2005, 2010, 2011, 2012, 2013, 2015,
          3001, 3002, 3003, 3004, 3006, 3007]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def bits(t):
    return t.cpu().view(torch.int16).numpy().view(np.uint16)


def operands(rng, m, n, k, whole):
    A = mx_uncut.e4m3_codes(rng, m, k)
    B, SB = mx_uncut.whole_sums(rng, n, k) if whole else (rng.integers(0, 256, (n, k // 2), dtype=np.uint8),
                                                          rng.integers(121, 134, (n, k // 32), dtype=np.uint8))
    P = torch.empty((sg.mxfp4_packed_bytes(n, k),), dtype=torch.uint8, device="cuda")
    sg.mxfp4_pack(dev(B), dev(SB), P, check=True)
    return dev(A), P, ref.e4m3(A), ref.values(B, SB)


@pytest.mark.parametrize("m,n,k,splits", [(1, 1, 32, (1,)), (3, 33, 512, (1,)), (16, 40, 4096, (1, 2, 5, 8)), (33, 70, 1120, (1, 3)),
                                          (130, 130, 2080, (1, 2, 5)), (300, 515, 2400, (1, 2)), (129, 257, 3584, (1, 7))])
def test_whole_sums_to_the_bit_on_every_build(m, n, k, splits):
    A, P, a, b = operands(np.random.default_rng(m + k), m, n, k, True)
    want = mx_uncut.bf16_bits(a @ b.T + 0.0)
    for build in BUILDS:
        for s in splits:
            D = torch.full((m + 1, n), -7.0, dtype=torch.bfloat16, device="cuda")
            assert lib.sg_debug_mxfp4_gemm(A.data_ptr(), 0, P.data_ptr(), D.data_ptr(), 0, 0, m, n, k, build + (10000 * s if s > 1 else 0),
                                           torch.cuda.current_stream().cuda_stream) == 0
            assert np.array_equal(bits(D[:m] + 0.0), want), (build, s)          # (+ 0.0: a zero of either sign)
            assert (D[m] == -7).all(), (build, s)


@pytest.mark.parametrize("n,k", [(1, 32), (31, 512), (33, 544), (129, 608), (257, 2080), (100, 4096), (18, 5440), (2373, 5440), (515, 10944)])
@pytest.mark.parametrize("m", [1, 2, 8, 16, 17, 33, 64, 100, 129, 257])
def test_sums_of_fp32(m, n, k):
    rng = np.random.default_rng(m * 7 + n + k)
    A, P, a, b = operands(rng, m, n, k, False)
    D = torch.full((m + 1, n), -7.0, dtype=torch.bfloat16, device="cuda")
    scale, row = torch.tensor([0.37], device="cuda"), rng.uniform(0.5, 1.5, m).astype(np.float32)
    sg.mxfp4_gemm_fp8act(A, P, D[:m], scale, dev(row), check=True)
    factor = np.float64(np.float32(0.37)) * row.astype(np.float64)[:, None]
    want, slack = mx_uncut.gemm(a, b)
    ref.check(bits(D[:m]), want * factor, slack * factor)
    assert (D[m] == -7).all()


@pytest.mark.parametrize("m,n,k", [(1, 33, 512), (8, 40, 4096), (33, 70, 1120), (130, 65, 2080), (260, 40, 1376)])
def test_sums_of_cut_products(m, n, k):
    """Operands of all sizes: the products are cut off as the model says, and nothing else is lost."""
    rng = np.random.default_rng(m + n + k)
    A = rng.integers(0, 256, (m, k), dtype=np.uint8)
    A = np.where((A & 127) == 127, 0x38, A).astype(np.uint8)
    B, SB = rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(121, 134, (n, k // 32), dtype=np.uint8)
    P = torch.empty((sg.mxfp4_packed_bytes(n, k),), dtype=torch.uint8, device="cuda")
    sg.mxfp4_pack(dev(B), dev(SB), P, check=True)
    want, (_, slack) = mx_uncut.cut_sums(A, B, SB), mx_uncut.gemm(ref.e4m3(A), ref.values(B, SB))
    a = dev(A)
    for build in BUILDS:
        D = torch.full((m, n), -7.0, dtype=torch.bfloat16, device="cuda")
        assert lib.sg_debug_mxfp4_gemm(a.data_ptr(), 0, P.data_ptr(), D.data_ptr(), 0, 0, m, n, k, build,
                                       torch.cuda.current_stream().cuda_stream) == 0
        ref.check(bits(D), want, slack)
