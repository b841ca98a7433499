"""What the MXFP4 products launch, without a GPU: on the stand-in for the HIP runtime (launch_recorder.py)."""
import re

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


# ---- calls that get no workspace ----

def kernels(launches):
    return [re.search(r"sg::(mx_\w+)", name).group(1) for name, *_ in launches]


def without_memory(r, shapes):
    """[(shape, rc and launches with a workspace, with none to be had, under capture, allocations of the last two)]"""
    out = []
    for s in shapes:
        with_memory = product(r, *s)
        r.call("sg_release_workspaces")
        before = r.fake.rec_allocations()
        r.fake.rec_largest_allocation(1 << 16)
        refused = product(r, *s)
        r.fake.rec_largest_allocation(-1)
        r.fake.rec_capturing(1)
        recorded = product(r, *s)
        r.fake.rec_capturing(0)
        out.append([s, with_memory, refused, recorded, r.fake.rec_allocations() - before])
    return out


def test_a_call_without_device_memory_launches_what_a_recorded_one_does(fake):
    split = [("fp8act", 8, 256, 16384), ("mx", 8, 256, 16384), ("mx", 128, 8192, 28672), ("mx", 200, 512, 8192 + 32)]
    copied = [("mx", 1024, 4096, 5440), ("mx", 2048, 8192, 10944)]
    for s, (rc, launches), refused, recorded, allocations in launch_recorder.scenario(fake, "test_mx_launches", "without_memory", split + copied):
        names = kernels(launches)
        assert rc == 0 and (names[-1] == "mx_sum_kernel" if tuple(s) in split else names[0] == "mx_scale_rows_kernel"), s
        for code, alone in (refused, recorded):
            assert code == 0 and len(alone) == 1 and kernels(alone)[0] in ("mx_gemm_kernel", "mx_tile_kernel"), s
        assert refused == recorded and allocations == 0, s


def over_the_limit(r, shapes):
    out = []
    for s in shapes:
        before = r.fake.rec_allocations()
        rc, launches = product(r, *s)
        out.append([r.lib.sg_debug_mxfp4_choice(1, *s[1:], 1), rc, launches, r.fake.rec_allocations() - before,
                    r.lib.sg_debug_mxfp4_choice(1, *s[1:], 0)])
    return out


def test_scales_too_large_for_a_workspace_are_not_copied(fake):
    """More than 512 MB of copied scales: the build without a workspace, by size alone."""
    for wanted, rc, launches, allocations, alone in launch_recorder.scenario(
            fake, "test_mx_launches", "over_the_limit", [("mx", 1 << 20, 4096, 16416), ("mx", 140000, 512, 131104)]):
        assert 3000 <= wanted % 10000 and alone < 3000
        assert rc == 0 and allocations == 0 and kernels(launches) == ["mx_tile_kernel"]
