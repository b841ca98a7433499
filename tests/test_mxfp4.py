"""MXFP4 without a GPU: the numpy definitions themselves, sizes, and what the entry points refuse."""
import numpy as np
import pytest
import torch

import mx_reference as ref
import rocm_dev_amd as sg
import rocm_dev_amd.torch_ops  # noqa: F401
from rocm_dev_amd._lib import host, lib


def bf16(x):
    return torch.tensor(x, dtype=torch.float32).bfloat16().view(torch.int16).numpy().view(np.uint16)


def test_reference_rounds_ties_to_even_codes_and_saturates():
    x = np.zeros((1, 32), np.float32)
    x[0, :16] = [4, 0.25, 0.26, 0.75, 1.25, 1.26, 1.75, 2.5, 2.52, 3.5, 5, 5.03, 7.9, -0.25, -5, -0.0]
    codes, scales = ref.encode(bf16(x))
    assert scales[0, 0] == 127                   # floor(log2(7.9)) = 2
    want = [4, 0, 0.5, 1, 1, 1.5, 2, 2, 3, 4, 4, 6, 6, 0, -4, 0]
    assert np.array_equal(ref.values(codes, scales)[0, :16], want)
    nibbles = np.stack((codes & 15, codes >> 4), 2).reshape(-1)
    assert nibbles[13] == 8 and nibbles[15] == 8 and nibbles[16] == 0       # zeros keep their sign


def test_reference_scales_at_the_ends():
    x = np.zeros((7, 32), np.uint16)
    x[1, 3] = 0x0001       # 2^-133
    x[2, 3] = 0x7f7f       # the largest
    x[3, 3] = 0xff80       # -inf
    x[4, 3] = 0x7fc0       # NaN
    x[5, 3] = 0x0100       # 2^-125
    x[6, 3] = 0x0180       # 2^-124
    codes, scales = ref.encode(x)
    assert scales[:, 0].tolist() == [127, 0, 252, 255, 255, 0, 1]
    assert not codes[3].any() and not codes[4].any()


def test_reference_pack_is_a_permutation():
    rng = np.random.default_rng(0)
    n, k = 19, 160
    codes, scales = rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(0, 255, (n, k // 32), dtype=np.uint8)
    p = ref.pack(codes, scales)
    assert p.size == sg.mxfp4_packed_bytes(n, k) == 2 * 2 * 1024 + 2 * 256
    assert np.array_equal(p[:16], codes[0, :16]) and np.array_equal(p[16:32], codes[1, :16])   # lanes 0 and 1: rows 0 and 1
    assert np.array_equal(p[16 * 16:17 * 16], codes[0, 16:32])                                  # lane 16: the next block
    at = 2 * 2 * 1024
    assert p[at] == scales[0, 0] and p[at + 1] == scales[0, 4] and p[at + 2] == 127             # lane 0: blocks 0, 4, none, none
    assert p[at + 4 * 16] == scales[0, 1]


def test_reference_e4m3_is_torchs():
    c = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(c).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.e4m3(c), want, equal_nan=True)


@pytest.mark.parametrize("n,k,want", [(1, 32, 2048 + 256), (16, 256, 2048 + 256), (17, 128, 2 * (2048 + 256)), (16, 640, 6 * 1024 + 512),
                                      (4096, 4096, 4096 * 4096 // 32 * 17), (1 << 20, 32768, (1 << 30) * 17)])
def test_packed_bytes(n, k, want):
    assert sg.mxfp4_packed_bytes(n, k) == want


@pytest.mark.parametrize("n,k", [(0, 32), (-1, 32), (16, 0), (16, 16), (16, 48), (16, -32)])
def test_packed_bytes_refuses(n, k):
    assert lib.sg_mxfp4_packed_bytes(n, k) == 0
    with pytest.raises(ValueError):
        sg.mxfp4_packed_bytes(n, k)


P = 0x1000       # no call below reaches a device: what it is told is refused first


@pytest.mark.parametrize("call,code", [
    (("encode_rows", 0, P, P, 4, 64), 9), (("encode_rows", P, 0, P, 4, 64), 9), (("encode_rows", P, P, 0, 4, 64), 9),
    (("encode_rows", P, P, P, 0, 64), 9), (("encode_rows", P, P, P, 4, 0), 9), (("encode_rows", P, P, P, 4, 48), 9),
    (("encode_rows", P, P, P, -4, 64), 9), (("encode_rows", P + 8, P, P, 4, 64), 8), (("encode_rows", P, P + 4, P, 4, 64), 8),
    (("decode_rows", 0, P, P, 4, 64), 9), (("decode_rows", P, 0, P, 4, 64), 9), (("decode_rows", P, P, 0, 4, 64), 9),
    (("decode_rows", P, P, P, 4, 16), 9), (("decode_rows", P + 1, P, P, 4, 64), 8), (("decode_rows", P, P, P + 2, 4, 64), 8),
    (("pack", 0, P, P, 16, 64, 32), 9), (("pack", P, 0, P, 16, 64, 32), 9), (("pack", P, P, 0, 16, 64, 32), 9),
    (("pack", P, P, P, 16, 64, 16), 9), (("pack", P, P, P, 0, 64, 32), 9), (("pack", P, P, P, 16, 80, 48), 3),
    (("pack", P, P, P, 16, 64, 40), 8), (("pack", P + 8, P, P, 16, 64, 32), 8), (("pack", P, P, P + 8, 16, 64, 32), 8),
    (("gemm", 0, P, P, P, 0, 4, 16, 64), 9), (("gemm", P, 0, P, P, 0, 4, 16, 64), 9), (("gemm", P, P, 0, P, 0, 4, 16, 64), 9),
    (("gemm", P, P, P, 0, 0, 4, 16, 64), 9), (("gemm", P, P, P, P, 0, 0, 16, 64), 9), (("gemm", P, P, P, P, 0, 4, 0, 64), 9),
    (("gemm", P, P, P, P, 0, 4, 16, 0), 9), (("gemm", P, P, P, P, 0, 4, 16, 48), 3), (("gemm", P + 8, P, P, P, 0, 4, 16, 64), 8),
    (("gemm", P, P, P + 8, P, 0, 4, 16, 64), 8), (("gemm", P, P, P, P + 4, 0, 4, 16, 64), 8),
    (("gemm_fp8act", 0, P, P, 0, 0, 4, 16, 64), 9), (("gemm_fp8act", P, P, P, 0, 0, 4, 16, 80), 3),
    (("gemm_fp8act", P + 4, P, P, 0, 0, 4, 16, 64), 8), (("gemm_fp8act", P, P, P + 2, 0, 0, 4, 16, 64), 8),
])
def test_c_abi_refuses(call, code):
    assert getattr(lib, "sg_mxfp4_" + call[0])(*call[1:], None) == code


def _u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


@pytest.mark.parametrize("call", [
    lambda: sg.mxfp4_encode_rows(torch.zeros(4, 48, dtype=torch.bfloat16), _u8(4, 24), _u8(4, 1)),
    lambda: sg.mxfp4_encode_rows(torch.zeros(4, 64, dtype=torch.bfloat16), _u8(4, 64), _u8(4, 2)),
    lambda: sg.mxfp4_encode_rows(torch.zeros(4, 64, dtype=torch.bfloat16), _u8(4, 32), _u8(4, 64)),
    lambda: sg.mxfp4_encode_rows(torch.zeros(64, 4, dtype=torch.bfloat16).t(), _u8(4, 32), _u8(4, 2)),
    lambda: sg.mxfp4_encode_rows(torch.zeros(4, 64, dtype=torch.bfloat16), _u8(4, 32), _u8(4, 2)),           # not on a GPU
    lambda: sg.mxfp4_decode_rows(_u8(4, 32), _u8(2, 4).t(), torch.zeros(4, 64, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_pack(_u8(16, 40), _u8(16, 2), _u8(2304)),
    lambda: sg.mxfp4_pack(_u8(16, 32), _u8(16, 3), _u8(2304)),
    lambda: sg.mxfp4_pack(_u8(16, 32), _u8(16, 2), _u8(2303)),
    lambda: sg.mxfp4_pack(_u8(16, 32), _u8(16, 2), _u8(4608)[::2]),
    lambda: sg.mxfp4_pack(_u8(32, 16).t(), _u8(16, 2), _u8(2304)),
    lambda: sg.mxfp4_gemm(_u8(4, 32), _u8(4, 2), _u8(2304), torch.zeros(5, 16, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_gemm(_u8(4, 32), _u8(4, 2), _u8(2304), torch.zeros(4, 17, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_gemm(_u8(4, 32), _u8(4, 1), _u8(2304), torch.zeros(4, 16, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_gemm(_u8(4, 24), _u8(4, 1), _u8(2304), torch.zeros(4, 16, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_gemm_fp8act(_u8(4, 48), _u8(2304), torch.zeros(4, 16, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_gemm_fp8act(_u8(64, 4).t(), _u8(2304), torch.zeros(4, 16, dtype=torch.bfloat16)),
    lambda: sg.mxfp4_gemm_fp8act(_u8(4, 64), _u8(2304), torch.zeros(16, 4, dtype=torch.bfloat16).t()),
    lambda: sg.mxfp4_gemm_fp8act(_u8(4, 64), _u8(2304), torch.zeros(4, 16, dtype=torch.bfloat16)),           # not on a GPU
])
def test_python_refuses(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("name,count", [("mxfp4_encode_rows", 3), ("mxfp4_decode_rows", 3), ("mxfp4_gemm", 5), ("mxfp4_gemm_fp8act", 5)])
def test_extension_leaves_host_tensors_and_non_tensors_to_python(name, count):
    fn = getattr(host, name)
    assert fn(*[_u8(16, 16)] * count) is None
    assert fn(*[3] * count) is None
    assert fn(*[None] * count) is None
    with pytest.raises(TypeError):
        fn(*[None] * (count - 1))


def test_registered_operators_infer_their_shapes():
    def meta(*shape, dtype=torch.uint8):
        return torch.empty(shape, dtype=dtype, device="meta")

    Q, S = torch.ops.sgemm.mxfp4_encode_rows(meta(5, 96, dtype=torch.bfloat16))
    assert Q.shape == (5, 48) and S.shape == (5, 3) and Q.dtype == S.dtype == torch.uint8
    assert torch.ops.sgemm.mxfp4_decode_rows(Q, S).shape == (5, 96)
    for n, k in ((33, 96), (16, 640), (100, 2048)):
        Pk = torch.ops.sgemm.mxfp4_pack(meta(n, k // 2), meta(n, k // 32))
        assert Pk.shape == (sg.mxfp4_packed_bytes(n, k),)
    D = torch.ops.sgemm.mxfp4_gemm(Q, S, meta(100), 33)
    assert D.shape == (5, 33) and D.dtype == torch.bfloat16
    assert torch.ops.sgemm.mxfp4_gemm_fp8act(meta(5, 96), meta(100), 33).shape == (5, 33)


SPLIT, WIDE = 10000, 3000


@pytest.mark.parametrize("fp4", [0, 1])
def test_choice_without_a_workspace_needs_none(fp4):
    """Under capture: no K split, and no build that would have to copy scales."""
    rng = np.random.default_rng(0)
    for _ in range(300):
        m, n, k = int(np.exp(rng.uniform(0, 8))), int(np.exp(rng.uniform(0, 11))), 32 * int(np.exp(rng.uniform(0, 7)))
        build = lib.sg_debug_mxfp4_choice(fp4, m, n, k, 0)
        assert 1100 < build < SPLIT
        if fp4 and k % 512:
            assert build < WIDE
        splits, build = divmod(lib.sg_debug_mxfp4_choice(fp4, m, n, k, 1), SPLIT)
        assert 1100 < build < 3100 and splits <= max(1, -(-k // 512))


def test_choice_refuses_what_the_products_refuse():
    for shape in ((0, 16, 64), (4, 0, 64), (4, 16, 0), (4, 16, 48)):
        assert lib.sg_debug_mxfp4_choice(1, *shape, 1) == 0


def test_choice_splits_few_tiles_with_a_long_k_only():
    assert lib.sg_debug_mxfp4_choice(0, 8, 256, 16384, 1) >= SPLIT
    assert lib.sg_debug_mxfp4_choice(0, 8, 28672, 4096, 1) < SPLIT
    assert WIDE < lib.sg_debug_mxfp4_choice(1, 1024, 57344, 8192, 1) < SPLIT
