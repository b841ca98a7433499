"""E4M3 operands of an MXFP4 product that no matrix instruction cuts off, so that its sums are those of fp32.

Inside a run of 8 products the instruction cuts off what is 13 binades below the largest exponent sum of the two operands.  E4M3 magnitudes
in [2^e, 2^(e + 3)) are multiples of 2^(e - 3), E2M1 magnitudes are multiples of 1/2 below 8: exponent sums are at most e + 4,
products multiples of 2^(e - 4), and the cut is at 2^(e - 9) or lower."""
import numpy as np


def e4m3_codes(rng, rows, k):
    """Exponents of three neighbouring binades, the same for the whole matrix; one value in sixteen is a zero."""
    e = int(rng.integers(2, 12))
    c = (rng.integers(0, 2, (rows, k)) << 7) | (rng.integers(e, e + 3, (rows, k)) << 3) | rng.integers(0, 8, (rows, k))
    return np.where(rng.random((rows, k)) < 1 / 16, 0, c).astype(np.uint8)


def whole_sums(rng, n, k):
    """(codes, scales) with one scale a weight row, in [2^-6, 2^6]: with e4m3_codes every partial sum of up to 4096 products is a whole
    multiple of 2^(e - 4) times that scale, less than 4096 * 2^(e + 3) * 6 - 24 bits - so that fp32 sums are exact in any order."""
    assert k <= 4096
    return rng.integers(0, 256, (n, k // 2), dtype=np.uint8), np.broadcast_to(rng.integers(121, 134, (n, 1), dtype=np.uint8), (n, k // 32)).copy()


def bf16_bits(x):
    """64-bit values that fp32 holds exactly -> bf16 bit patterns, to nearest even (no NaNs)."""
    u = np.asarray(x, np.float64).astype(np.float32)
    assert np.array_equal(u.astype(np.float64), x)
    u = u.view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def gemm(a, b):
    """(a @ b.T, how far fp32 sums of it may be off): an instruction adds 16 runs of 8 and the running sum, rounding or cutting at fp32
    precision at most 17 times for every 128 products; waves' and splits' sums are added at most 16 times more."""
    total = np.abs(a) @ np.abs(b).T
    return a @ b.T, (17 * -(-a.shape[1] // 128) + 16) * 2.0 ** -23 * total
