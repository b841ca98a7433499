"""sg_rmsnorm_fp8_rows against its formula in 64 bits."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

# fp32 in the kernel: a thread adds at most 64 squares and the workgroup's 22 partial sums behind it, each addition off by 2^-24 of the sum;
# the root halves that, and four more roundings (mean, root, reciprocal, product) come on top: below 2^-17 of y.  Rows beyond 65536 columns:
# 8 values a thread for every 8192 columns more.
FP32 = 2.0 ** -17


@pytest.fixture(scope="module")
def sg():
    import rocm_dev_amd
    return rocm_dev_amd


def operands(rows, cols, seed, residual=True):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")
    X = normal(rows, cols) * torch.exp2(4 * normal(rows, 1))
    return X.bfloat16(), (1 + 0.5 * normal(cols)).bfloat16(), (3 * normal(rows, cols)).bfloat16() if residual else None


def run(sg, X, weight=None, residual=None, total=True, y=True, eps=1e-5, **more):
    rows, cols = X.shape
    # a guard row behind every output
    Q = torch.full((rows + 1, cols), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((rows + 1,), -7.0, device="cuda")
    S, Y = (torch.full((rows + 1, cols), -7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert sg.rmsnorm_fp8_rows(X, Q[:rows], s[:rows], weight, residual, S[:rows] if total else None, Y[:rows] if y else None, eps, **more) == 0
    torch.cuda.synchronize()
    assert (Q[rows] == 0x55).all() and s[rows] == -7 and (S[rows] == -7).all() and (Y[rows] == -7).all()
    assert total or (S == -7).all()
    assert y or (Y == -7).all()
    return Q[:rows], s[:rows], S[:rows], Y[:rows]


def expected(X, weight, residual, eps):
    v = X if residual is None else (X.float() + residual.float()).bfloat16()
    y = v.double() / (v.double().square().mean(1, keepdim=True) + eps).sqrt()
    return v, y if weight is None else y * weight.double()


def check(Q, s, Y, y):
    top = y.abs().amax(1)
    want = torch.where(top == 0, 1.0, top / 448)
    assert ((s.double() - want).abs() <= 2 * FP32 * want).all()
    # a code is the nearest one: half a step, 2^-4 of the value or 2^-10 of the scale
    got = Q.view(torch.float8_e4m3fn).double() * s.double()[:, None]
    assert ((got - y).abs() <= y.abs() * (2.0 ** -4 + 4 * FP32) + want[:, None] * 2.0 ** -10 * (1 + 4 * FP32)).all()
    if Y is not None:
        assert ((Y.double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * FP32)).all()


# around every change of build: lanes of a wave, one to sixteen waves, two to eight chunks, the two passes
@pytest.mark.parametrize("cols", [16, 32, 48, 128, 144, 512, 528, 1024, 1040, 2048, 2064, 4096, 4112, 8192, 8208, 10944, 16384, 16400, 32768,
                                  32784, 65536, 65552, 131088])
@pytest.mark.parametrize("rows", [1, 3, 67])
def test_rows(sg, rows, cols):
    X, w, res = operands(rows, cols, seed=rows * 7 + cols)
    v, y = expected(X, w, res, 1e-5)
    Q, s, S, Y = run(sg, X, w, res)
    assert torch.equal(S, v)
    check(Q, s, Y, y)
    # each optional operand left out
    Q2, s2, _, _ = run(sg, X, w, res, total=False, y=False)
    assert torch.equal(Q2, Q) and torch.equal(s2, s)
    Q3, s3, _, Y3 = run(sg, v, w)
    assert torch.equal(Q3, Q) and torch.equal(s3, s) and torch.equal(Y3, Y)
    Q4, s4, _, Y4 = run(sg, X, None, None, eps=0.25)
    check(Q4, s4, Y4, expected(X, None, None, 0.25)[1])


@pytest.mark.parametrize("cols", [64, 4096, 70000 // 16 * 16])
def test_many_rows(sg, cols):
    rows = 20011 if cols < 8192 else 300
    X, w, res = operands(rows, cols, seed=cols)
    v, y = expected(X, w, res, 1e-5)
    Q, s, S, Y = run(sg, X, w, res)
    assert torch.equal(S, v)
    check(Q, s, Y, y)


@pytest.mark.parametrize("cols", [48, 4096, 65552])
@pytest.mark.parametrize("place", ["X", "residual"])
def test_sum_in_place(sg, cols, place):
    X, w, res = operands(5, cols, seed=cols)
    Q, s, S, Y = run(sg, X, w, res)
    X2, res2 = X.clone(), res.clone()
    Q2, s2, Y2 = torch.empty_like(Q), torch.empty_like(s), torch.empty_like(Y)
    assert sg.rmsnorm_fp8_rows(X2, Q2, s2, w, res2, X2 if place == "X" else res2, Y2, 1e-5) == 0
    torch.cuda.synchronize()
    assert torch.equal(Q2, Q) and torch.equal(s2, s) and torch.equal(Y2, Y)
    assert torch.equal(X2 if place == "X" else res2, S) and torch.equal(res2 if place == "X" else X2, res if place == "X" else X)


@pytest.mark.parametrize("cols", [64, 1040, 65552])
def test_rows_out_of_range(sg, cols):
    """Zeros, NaNs, infinities, squares that overflow, rows and weights at the ends of the range; no row touches another."""
    X, w, _ = operands(9, cols, seed=1, residual=False)
    clean = run(sg, X, w)
    X[0] = 0
    X[2, 5] = float("nan")
    X[4, 7] = float("inf")
    X[6] = 1e30
    X[8] = 2.0 ** -133          # subnormal
    Q, s, S, Y = run(sg, X, w)
    assert torch.equal(S.view(torch.int16), X.view(torch.int16))
    for r in (1, 3, 5, 7):
        assert all(torch.equal(a[r], b[r]) for a, b in zip((Q, s, S, Y), clean))
    assert s[0] == 1 and not Q[0].view(torch.float8_e4m3fn).float().any() and not Y[0].any()
    assert s[2] == 1 and (Q[2] == 0x7f).all() and Y[2].isnan().all()
    assert s[4] == 1 and Q[4, 7] == 0x7f and Y[4, 7].isnan()
    rest = [c for c in range(cols) if c != 7]
    assert not Q[4].view(torch.float8_e4m3fn).float()[rest].any() and not Y[4][rest].any()
    assert s[6] == 1 and not Q[6].view(torch.float8_e4m3fn).float().any()
    # a norm whose scale has no fp32 reciprocal
    tiny = torch.full_like(w, 2.0 ** -126)
    Q, s, _, _ = run(sg, X[1:2], tiny, eps=1.0)
    y = expected(X[1:2], tiny, None, 1.0)[1]
    want = y.abs().amax(1) / 448
    # here y and the scale are subnormal: steps of 2^-149, of which y's and the scale's roundings are half of one each
    assert ((s.double() - want).abs() <= want * FP32 + 2.0 ** -149).all()
    got = Q.view(torch.float8_e4m3fn).double()
    assert (got - y / s.double()).abs().le((y / s.double()).abs() * (2.0 ** -4 + 2 * FP32) + 2.0 ** -10 + 2.0 ** -149 / s.double()).all()


def test_stream_and_graph(sg):
    X, w, res = operands(33, 4096, seed=3)
    want = [t.clone() for t in run(sg, X, w, res)]
    out = [torch.empty_like(t) for t in want]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        sg.rmsnorm_fp8_rows(X, out[0], out[1], w, res, out[2], out[3], 1e-5, check=True)
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        sg.rmsnorm_fp8_rows(X, torch.empty_like(out[0]), torch.empty_like(out[1]), w, check=True)


def test_registered_operator(sg):
    import rocm_dev_amd.torch_ops  # noqa: F401
    X, w, res = operands(7, 1040, seed=5)
    want = run(sg, X, w, res, eps=1e-6)
    got = torch.ops.sgemm.rmsnorm_fp8_rows(X.t().contiguous().t(), w, res, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    Q, s, total, _ = torch.ops.sgemm.rmsnorm_fp8_rows(X)
    assert torch.equal(total, X) and torch.equal(Q, run(sg, X, eps=1e-6)[0])
    torch.library.opcheck(torch.ops.sgemm.rmsnorm_fp8_rows.default, (X, w, res), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("seed", range(16))
def test_drawn_sizes(sg, seed):
    rng = random.Random(seed)
    rows, cols = rng.randint(1, rng.choice((8, 700))), 16 * rng.randint(1, rng.choice((64, 1100)))
    X, weight, residual = operands(rows, cols, seed, residual=rng.random() < 0.6)
    weight = weight if rng.random() < 0.8 else None
    Q, s, S, Y = run(sg, X, weight, residual)
    v, y = expected(X, weight, residual, 1e-5)
    assert torch.equal(S, v)
    check(Q, s, Y, y)


@pytest.mark.parametrize("cols", [512, 8192, 98304])
def test_matrices_beyond_4_gigabytes(sg, cols):
    rows = 2 ** 32 // cols + 5
    X = torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")
    part, weight, _ = operands(64, cols, seed=5)
    X[:64] = part
    X[64:] = 1
    X[-64:] = part
    Q, s = torch.empty((rows, cols), dtype=torch.uint8, device="cuda"), torch.empty(rows, device="cuda")
    total = torch.empty_like(X)
    assert sg.rmsnorm_fp8_rows(X, Q, s, weight, None, total, None, 1e-5) == 0
    # (64 rows by themselves may add their squares up in another order than as many of these)
    _, y = expected(part, weight, None, 1e-5)
    for rows_at in (slice(0, 64), slice(rows - 64, rows)):
        check(Q[rows_at], s[rows_at], None, y)
        assert torch.equal(Q[rows_at], Q[:64]) and torch.equal(s[rows_at], s[:64]) and torch.equal(total[rows_at], part)
    assert torch.equal(Q[64:80], Q[-80:-64]) and (s[64:-64] == s[64]).all()
