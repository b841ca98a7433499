"""A product of MXFP4 activations whose copied scales are too large for a workspace: it runs without, and is right."""
import numpy as np
import pytest
import torch

import mx_reference as ref
import rocm_dev_amd as sg
from rocm_dev_amd._lib import lib

pytestmark = pytest.mark.gpu


def test_scales_too_large_for_a_workspace_are_read_where_they_lie():
    m, n, k = 140000, 512, 131104
    assert lib.sg_debug_mxfp4_choice(1, m, n, k, 1) % 10000 >= 3000       # a wide build, on copied scales: 575 MB of them
    rng = np.random.default_rng(0)
    b, sb = rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(121, 134, (n, k // 32), dtype=np.uint8)
    P = torch.empty((sg.mxfp4_packed_bytes(n, k),), dtype=torch.uint8, device="cuda")
    sg.mxfp4_pack(torch.from_numpy(b).cuda(), torch.from_numpy(sb).cuda(), P, check=True)
    # rows of their own at both ends and in the middle, zeros elsewhere
    rows = np.r_[0:3, m // 2:m // 2 + 2, m - 5:m]
    a, sa = rng.integers(0, 256, (rows.size, k // 2), dtype=np.uint8), rng.integers(121, 134, (rows.size, k // 32), dtype=np.uint8)
    at = torch.from_numpy(rows).cuda()
    A = torch.zeros((m, k // 2), dtype=torch.uint8, device="cuda")
    SA = torch.full((m, k // 32), 127, dtype=torch.uint8, device="cuda")
    A[at], SA[at] = torch.from_numpy(a).cuda(), torch.from_numpy(sa).cuda()
    D = torch.full((m, n), -7.0, dtype=torch.bfloat16, device="cuda")
    sg.release_workspaces()
    sg.mxfp4_gemm(A, SA, P, D, check=True)
    torch.cuda.synchronize()
    assert sg.workspace_bytes() == 0
    want, slack = ref.gemm(ref.values(a, sa), ref.values(b, sb), False)
    ref.check(D[at].cpu().view(torch.int16).numpy().view(np.uint16), want, slack)
    D[at] = 0
    assert not D.any()
