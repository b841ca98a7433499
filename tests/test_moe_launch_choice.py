"""How many workgroups share a tile of the experts' down projections: the best for the build that is launched - its waves, and how many of its
workgroups the LDS has room for - by the times that the rule in sg_moe.hip states (no GPU: launches on a stand-in for the runtime)."""
import random

import launch_recorder
import pytest

CUS, LDS = 256, 160 * 1024
# parts of 32 columns have no build of eight waves, those of 16 off their lines have none above some number of tokens
SHAPES = [(45, 480, 4976, 8, 2), (63, 864, 1104, 32, 7), (57, 560, 1456, 16, 4), (58, 688, 1216, 16, 2), (60, 656, 3584, 8, 2), (56, 128, 4448, 8, 1),
          (57, 912, 656, 32, 6), (64, 2048, 1408, 8, 4), (64, 1024, 4096, 8, 4), (61, 2064, 1376, 40, 6), (1, 2048, 1408, 64, 6), (8, 4096, 14336, 8, 2)]


def drawn():
    rng = random.Random(5)
    out = list(SHAPES)
    for _ in range(400):
        experts = rng.choice((4, 8, 16, 32, 64, 128, 256))
        out.append((rng.randint(1, 64), 16 * rng.randint(8, 512), 16 * rng.randint(4, 900), experts, rng.randint(1, min(8, experts))))
    return out


def launches(rec, shapes):
    out = []
    for m, hidden, inner, experts, top_k in shapes:
        rc, calls = rec.of("sg_moe_experts", rec.A, rec.COL, rec.S, rec.B, None, rec.B, None, rec.D, m, hidden, inner, experts, top_k, rec.WS, 1 << 30, None)
        assert rc == 0
        out.append([c for c in calls if "moe_down" in c[0] or "moe_sum" in c[0]])
    return out


def microseconds(shape, splits, slots):
    m, hidden, inner, experts, top_k = shape
    tiles = hidden // 16 * splits
    used = tiles / (-(-tiles // slots) * slots)
    read = experts * (1 - (1 - top_k / experts) ** m) * hidden * inner / (6e6 * min(1.0, 1.4 * used))
    return read + (4 + splits * m * hidden * 8 / 4e6 if splits > 1 else 0)


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("fake"))


def test_the_split_is_the_best_of_the_build_that_runs(fake):
    shapes = drawn()
    one_a_cu = split = 0
    for shape, calls in zip(shapes, launch_recorder.scenario(fake, "test_moe_launch_choice", "launches", shapes)):
        m, hidden, inner, experts, top_k = shape
        _, grid, threads, lds = calls[0]
        splits, waves = grid // (hidden // 16), threads // 64
        assert grid == splits * (hidden // 16) and len(calls) == (2 if splits > 1 else 1) and lds <= LDS
        room = 128 // -(-lds // 1280)
        slots = CUS * (2 if waves == 4 and room > 1 else 1)
        most = 8 if 8 * hidden <= 16384 else max(1, 16384 // hidden)
        steps = -(-inner // 128) * top_k
        allowed = [s for s in range(1, most + 1) if s == 1 or steps >= 2 * s * waves]
        assert splits in allowed, shape
        # a split is taken where it saves 3 %
        assert microseconds(shape, splits, slots) <= 1.001 / 0.97 * min(microseconds(shape, s, slots) for s in allowed), (shape, splits, slots)
        one_a_cu += waves == 4 and room == 1
        split += splits > 1
    assert one_a_cu > 20 and split > 20
