"""The norm, the products with 4-bit integer weights and the mixture-of-experts layer: what is refused before any device is touched, sizes,
schemas and shape inference.  All on the CPU."""
import math

import pytest
import torch

P0 = 0x10000      # a pointer that no launch sees


@pytest.fixture(scope="module")
def lib():
    from rocm_dev_amd._lib import lib
    return lib


@pytest.fixture(scope="module")
def sg():
    import rocm_dev_amd
    return rocm_dev_amd


def test_norm_refusals(lib):
    def call(X=P0, res=None, w=None, total=None, Y=None, Q=P0, s=P0, eps=1e-6, rows=4, cols=32):
        return lib.sg_rmsnorm_fp8_rows(X, res, w, total, Y, Q, s, eps, rows, cols, None)
    assert call(cols=24) == 9 and call(cols=0) == 9 and call(rows=0) == 9 and call(rows=-1) == 9
    assert call(X=0) == 9 and call(Q=0) == 9 and call(s=0) == 9
    assert call(eps=-1e-9) == 9 and call(eps=math.nan) == 9 and call(eps=math.inf) == 9
    for name in ("X", "res", "w", "total", "Y", "Q"):
        assert call(**{name: P0 + 8}) == 8, name
    assert call(s=P0 + 2) == 8
    assert call() == 11 or torch.cuda.is_available()          # as far as the device


def test_int4_refusals(lib):
    def pack(B=P0, s=P0, z=None, P=P0, n=32, k=256, group=128, flags=0, stride=128):
        return lib.sg_int4_pack(B, s, z, P, n, k, group, flags, stride, None)

    def gemm(A=P0, P=P0, D=P0, m=1, n=32, k=256, group=128, flags=0):
        return lib.sg_int4_gemm(A, P, D, m, n, k, group, flags, None)
    for call in (pack, gemm):
        assert call(n=0) == 9 and call(k=0) == 9 and call(group=16) == 9 and call(group=256) == 9 and call(flags=4) == 9 and call(flags=-1) == 9
        assert call(k=192) == 9 and call(k=192, group=64) in (9, 11) and call(P=0) == 9 and call(P=P0 + 8) == 8
    assert pack(stride=112) == 9 and pack(stride=136) == 8 and pack(B=P0 + 4) == 8 and pack(s=P0 + 1) == 8 and pack(B=0) == 9 and pack(s=0) == 9
    assert pack(flags=1) == 9 and pack(z=P0) == 9               # zeros and the flag go together
    assert gemm(m=0) == 9 and gemm(A=0) == 9 and gemm(D=0) == 9 and gemm(A=P0 + 8) == 8 and gemm(D=P0 + 4) == 8
    assert lib.sg_int4_packed_bytes(32, 192, 128, 0) == 0 and lib.sg_int4_packed_bytes(0, 128, 128, 0) == 0


@pytest.mark.parametrize("n,k,group,zeros", [(1, 32, 32, False), (16, 128, 128, False), (17, 160, 32, True), (2373, 5440, 64, True)])
def test_int4_packed_bytes(sg, n, k, group, zeros):
    tiles, steps = -(-n // 16), -(-k // 128)
    assert sg.int4_packed_bytes(n, k, group, zeros) == tiles * steps * (1024 + 128 // group * 16 * (3 if zeros else 2))


def test_moe_refusals(lib):
    sizes = dict(m=4, hidden=64, inner=32, experts=8, top_k=2)

    def need(**kw):
        s = {**sizes, **kw}
        return lib.sg_moe_workspace_bytes(s["m"], s["hidden"], s["inner"], s["experts"], s["top_k"])

    def layer(X=P0, R=P0, W1=P0, S1=None, W2=P0, S2=None, D=P0, ids=P0, w=P0, ws=P0, room=None, **kw):
        s = {**sizes, **kw}
        return lib.sg_moe_layer(X, R, W1, S1, W2, S2, D, ids, w, s["m"], s["hidden"], s["inner"], s["experts"], s["top_k"], 1, ws,
                                need(**kw) if room is None else room, None)

    def experts(X=P0, W1=P0, S1=None, W2=P0, S2=None, D=P0, ids=P0, w=P0, ws=P0, room=None, **kw):
        s = {**sizes, **kw}
        return lib.sg_moe_experts(X, ids, w, W1, S1, W2, S2, D, s["m"], s["hidden"], s["inner"], s["experts"], s["top_k"], ws,
                                  need(**kw) if room is None else room, None)
    for bad in (dict(m=0), dict(m=65), dict(hidden=72), dict(hidden=0), dict(inner=24), dict(inner=0), dict(experts=0), dict(experts=513),
                dict(top_k=0), dict(top_k=9), dict(top_k=17, experts=64), dict(m=-1)):
        assert need(**bad) == 0 and layer(room=1 << 20, **bad) == 9 and experts(room=1 << 20, **bad) == 9, bad
    for call in (layer, experts):
        for name in ("X", "W1", "W2", "D", "ids", "w"):
            assert call(**{name: 0}) == 9, name
        for name in ("X", "W1", "W2", "D"):
            assert call(**{name: P0 + 8}) == 8, name
        for name in ("S1", "S2", "ids", "w"):
            assert call(**{name: P0 + 2}) == 8, name
        assert call(ws=0) == 10 and call(room=need() - 1) == 10 and call(ws=P0 + 128) == 8
    assert layer(R=0) == 9 and layer(R=P0 + 8) == 8
    route = [P0, P0, P0, P0, 4, 64, 8, 2, 1, P0, 4 * 8 * 4, None]
    for at, value, code in ((1, 0, 9), (5, 72, 9), (4, 65, 9), (7, 9, 9), (9, 0, 10), (10, 4 * 8 * 4 - 1, 10), (2, P0 + 2, 8)):
        assert lib.sg_moe_route(*[value if i == at else v for i, v in enumerate(route)]) == code, at


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def test_python_layer_refuses_other_layouts(sg):
    f32, i32 = torch.float32, torch.int32
    m, cols = 4, 64
    norm = dict(X=bf16(m, cols), Q=u8(m, cols), scales=torch.ones(m))
    W1, W2 = u8(8, 64, 64), u8(8, 64, 32)
    moe = dict(X=bf16(m, 64), router=bf16(8, 64), W_gate_up=W1, W_down=W2, D=bf16(m, 64), ids=torch.zeros((m, 2), dtype=i32), weights=torch.zeros((m, 2)))
    P = u8(sg.int4_packed_bytes(32, 256))
    gemm = dict(A=bf16(m, 256), P=P, D=bf16(m, 32))
    pack = dict(B=u8(32, 128), scales=bf16(32, 2), P=P)
    cases = {
        "norm, strided rows": (sg.rmsnorm_fp8_rows, norm, dict(X=bf16(m, 2 * cols)[:, :cols])),
        "norm, codes of another shape": (sg.rmsnorm_fp8_rows, norm, dict(Q=u8(m, cols + 16))),
        "norm, odd columns": (sg.rmsnorm_fp8_rows, norm, dict(X=bf16(m, 40), Q=u8(m, 40))),
        "norm, scales": (sg.rmsnorm_fp8_rows, norm, dict(scales=torch.ones(m + 1))),
        "norm, weight": (sg.rmsnorm_fp8_rows, norm, dict(weight=bf16(cols - 1))),
        "norm, strided weight": (sg.rmsnorm_fp8_rows, norm, dict(weight=bf16(2 * cols)[::2])),
        "norm, residual": (sg.rmsnorm_fp8_rows, norm, dict(residual=bf16(m + 1, cols))),
        "norm, transposed sum": (sg.rmsnorm_fp8_rows, norm, dict(sum_out=bf16(cols, m).t())),
        "norm, Y": (sg.rmsnorm_fp8_rows, norm, dict(Y=bf16(m, cols - 16))),
        "int4, columns": (sg.int4_gemm, gemm, dict(A=bf16(m, 384))),
        "int4, strided activations": (sg.int4_gemm, gemm, dict(A=bf16(m, 512)[:, :256])),
        "int4, rows": (sg.int4_gemm, gemm, dict(D=bf16(m + 1, 32))),
        "int4, group": (sg.int4_gemm, gemm, dict(group=64)),
        "int4, a group that there is not": (sg.int4_gemm, gemm, dict(group=256)),
        "int4, zeros": (sg.int4_gemm, gemm, dict(zeros=True)),
        "int4, scales' type": (sg.int4_gemm, gemm, dict(scale_dtype=f32)),
        "pack, scales' type": (sg.int4_pack, pack, dict(scales=torch.ones(32, 2))),
        "pack, scales' rows": (sg.int4_pack, pack, dict(scales=bf16(31, 2))),
        "pack, no scales": (sg.int4_pack, pack, dict(scales=bf16(32, 0))),
        "pack, zeros": (sg.int4_pack, pack, dict(zeros=u8(32, 4))),
        "pack, zeros that P has no place for": (sg.int4_pack, pack, dict(zeros=u8(32, 2))),
        "pack, transposed": (sg.int4_pack, pack, dict(B=u8(128, 32).t())),
        "moe, strided tokens": (sg.moe_layer, moe, dict(X=bf16(m, 128)[:, :64])),
        "moe, router": (sg.moe_layer, moe, dict(router=bf16(7, 64))),
        "moe, gate and up": (sg.moe_layer, moe, dict(W_gate_up=u8(8, 63, 64))),
        "moe, transposed weights": (sg.moe_layer, moe, dict(W_down=u8(8, 32, 64).transpose(1, 2))),
        "moe, down": (sg.moe_layer, moe, dict(W_down=u8(8, 64, 64))),
        "moe, ids": (sg.moe_layer, moe, dict(ids=torch.zeros((m + 1, 2), dtype=i32))),
        "moe, weights": (sg.moe_layer, moe, dict(weights=torch.zeros((m, 3)))),
        "moe, scales": (sg.moe_layer, moe, dict(gate_up_scales=torch.ones(8, 32))),
        "moe, more choices than experts": (sg.moe_layer, moe, dict(ids=torch.zeros((m, 9), dtype=i32), weights=torch.zeros((m, 9)))),
        "moe, too many tokens": (sg.moe_layer, moe, dict(X=bf16(65, 64), D=bf16(65, 64), ids=torch.zeros((65, 2), dtype=i32), weights=torch.zeros((65, 2)))),
    }
    for what, (call, good, bad) in cases.items():
        with pytest.raises(ValueError) as e:
            call(**{**good, **bad})
            pytest.fail(what + " was accepted")
        assert "CUDA" not in str(e.value), what
    experts = {k: v for k, v in moe.items() if k != "router"}
    route = {k: moe[k] for k in ("X", "router", "ids", "weights")}
    for call, good in ((sg.rmsnorm_fp8_rows, norm), (sg.int4_gemm, gemm), (sg.int4_pack, pack), (sg.moe_layer, moe), (sg.moe_experts, experts), (sg.moe_route, route)):
        with pytest.raises(ValueError, match="CUDA"):           # well-formed operands get as far as the device check
            call(**good)


def test_shape_inference_on_meta_tensors(sg):
    import rocm_dev_amd.torch_ops  # noqa: F401
    ops = torch.ops.sgemm

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")
    q, s, total, y = ops.rmsnorm_fp8_rows(meta(8, 512), meta(512), meta(8, 512), 1e-5)
    assert q.shape == (8, 512) and q.dtype == torch.uint8 and s.shape == (8,) and s.dtype == torch.float32
    assert total.shape == y.shape == (8, 512) and total.dtype == y.dtype == torch.bfloat16
    for n, k, group, zeros in ((17, 160, 32, False), (32, 256, 128, True)):
        P = ops.int4_pack(meta(n, k // 2, dtype=torch.uint8), meta(n, k // group), meta(n, k // group, dtype=torch.uint8) if zeros else None)
        assert P.shape == (sg.int4_packed_bytes(n, k, group, zeros),)
        assert ops.int4_gemm(meta(3, k), P, n, group, zeros).shape == (3, n)
    ids, w = ops.moe_route(meta(8, 64), meta(16, 64), 4)
    assert ids.shape == w.shape == (8, 4) and ids.dtype == torch.int32 and w.dtype == torch.float32
    D = ops.moe_experts(meta(8, 64), ids, w, meta(16, 64, 64, dtype=torch.uint8), meta(16, 64, 32, dtype=torch.uint8))
    assert D.shape == (8, 64) and D.dtype == torch.bfloat16
