"""What the MXFP4 products launch, without a GPU: on the stand-in for the HIP runtime (launch_recorder.py)."""
import pytest

import launch_recorder

LAYER_8B = [(6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336)]
LAYER_70B = [(10240, 8192), (8192, 8192), (57344, 8192), (8192, 28672)]


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("fake"))


def product(r, kind, m, n, k):
    if kind == "mx":
        return r.of("sg_mxfp4_gemm", r.A, r.R, r.B, r.D, 0, m, n, k, 0)
    return r.of("sg_mxfp4_gemm_fp8act", r.A, r.B, r.D, 0, 0, m, n, k, 0)


# ---- the shapes whose builds a thread keeps ----

def searches(r, shapes):
    """[searches of the first pass over the shapes, of the second, of the third]"""
    out = []
    for _ in range(3):
        before = r.lib.sg_debug_mxfp4_searches()
        for shape in shapes:
            assert product(r, *shape)[0] == 0
        out.append(r.lib.sg_debug_mxfp4_searches() - before)
    return out


@pytest.mark.parametrize("layer", [LAYER_8B, LAYER_70B])
@pytest.mark.parametrize("kind", ["mx", "fp8act"])
@pytest.mark.parametrize("m", [1, 8, 128])
def test_a_layers_projections_are_searched_once(fake, layer, kind, m):
    shapes = [(kind, m, n, k) for n, k in layer]
    assert launch_recorder.scenario(fake, "test_mx_launches", "searches", shapes) == [4, 0, 0]


@pytest.mark.parametrize("shapes", [
    [(kind, m, n, k) for kind in ("mx", "fp8act") for m in (1, 7) for n, k in LAYER_8B],       # 16: a draft and a verify step, both formats
    [("mx", m, 4096, 4096) for m in range(1, 17)],
    [("fp8act", 16, 256 * n, 512) for n in range(1, 17)],
    [("fp8act", 16, 256, 512 * k) for k in range(1, 17)]])
def test_the_last_sixteen_shapes_are_kept(fake, shapes):
    assert launch_recorder.scenario(fake, "test_mx_launches", "searches", shapes) == [16, 0, 0]


def builds_again(r, shapes):
    """launches of every shape, first in a fresh thread's order, then with every answer kept or pushed out by others"""
    first = [product(r, *s) for s in shapes]
    return [[product(r, *s) for s in order] == [first[shapes.index(s)] for s in order]
            for order in (shapes, shapes[::-1], shapes[:20] + shapes[:20])]


def test_a_kept_answer_is_the_shapes_own(fake):
    shapes = [(kind, m, n, k) for kind in ("mx", "fp8act") for m in (1, 33, 600) for n, k in LAYER_8B + LAYER_70B]
    assert launch_recorder.scenario(fake, "test_mx_launches", "builds_again", shapes) == [True, True, True]
