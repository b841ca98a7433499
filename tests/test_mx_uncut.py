"""The operands of mx_uncut.py do what they say, and a check on them sees a single lost column."""
import numpy as np
import pytest

import mx_reference as ref
import mx_uncut


def test_no_product_is_cut_and_sums_are_whole():
    rng = np.random.default_rng(0)
    for _ in range(20):
        a = ref.e4m3(mx_uncut.e4m3_codes(rng, 3, 4096))
        b = ref.values(*mx_uncut.whole_sums(rng, 5, 4096))
        low = np.abs(a[a != 0]).min()
        low = 2.0 ** np.floor(np.log2(low))                      # 2^e
        assert np.abs(a).max() < 8 * low
        for row in b:
            scale = np.abs(row[row != 0]).min() * 2              # the row's 2^(S - 127)
            unit = low * scale / 16                              # 2^(e - 4)
            p = a * row
            assert np.array_equal(np.rint(p / unit), p / unit)
            runs = np.abs(p.reshape(3, -1, 8)).max(2)
            cut = 2.0 ** (np.floor(np.log2(low)) + 4 - 13) * scale
            assert cut < unit and runs.max() < 2.0 ** 5.6 * low * scale
            assert np.abs(p).sum(1).max() < 2.0 ** 24 * unit


def test_rounding_is_to_nearest_even():
    x = np.array([1, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 1 + 2.0 ** -8 + 2.0 ** -20, -1 - 2.0 ** -8, 0, -3.5, 2.0 ** -130])
    assert np.array_equal(ref.bf16_to_f64(mx_uncut.bf16_bits(x)), [1, 1, 1 + 2.0 ** -6, 1 + 2.0 ** -7, -1, 0, -3.5, 2.0 ** -130])


@pytest.mark.parametrize("k", [96, 1120, 4096])
def test_a_lost_column_is_seen(k):
    """Planted in the reference: sums without one column, or with one column twice, do not round to the sums' bits."""
    rng = np.random.default_rng(k)
    a = ref.e4m3(mx_uncut.e4m3_codes(rng, 16, k))
    b = ref.values(*mx_uncut.whole_sums(rng, 33, k))
    whole = mx_uncut.bf16_bits(a @ b.T)
    for c in rng.choice(k, 40, replace=False):
        column = np.outer(a[:, c], b[:, c])
        for wrong in (a @ b.T - column, a @ b.T + column):
            seen = (mx_uncut.bf16_bits(wrong) != whole).mean()
            assert seen > 0.3, (c, seen)


def test_a_lost_column_is_seen_under_scales_of_all_sizes():
    rng = np.random.default_rng(1)
    k = 2080
    a = ref.e4m3(mx_uncut.e4m3_codes(rng, 16, k))
    b = ref.values(rng.integers(0, 256, (33, k // 2), dtype=np.uint8), rng.integers(121, 134, (33, k // 32), dtype=np.uint8))
    want, slack = mx_uncut.gemm(a, b)
    ref.check(mx_uncut.bf16_bits(want.astype(np.float32).astype(np.float64)), want, slack)
    most = slack + np.abs(want) * 2.0 ** -8
    columns = np.abs(a.T[:, :, None] * b.T[:, None, :])          # [k, 16, 33]
    lost = (columns > 2 * most).any((1, 2))
    assert lost.all()                                            # every column shows in some output
