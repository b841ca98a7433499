"""Every build of the norm's, the 4-bit integer products' and the experts' kernels in the library is one that some size, alignment and state
of its stream reaches (no GPU: launches on a stand-in for the runtime)."""
import ctypes as C
import math
import random
import re
import subprocess

import launch_recorder
import pytest


def between(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high))))


def reached(rec):
    rng = random.Random(3)
    names = set()

    def call(*args):
        rc, launches = rec.of(*args)
        assert rc == 0, args
        names.update(x[0].replace("void ", "", 1).split("(")[0] for x in launches)
    X, R, D, S, IDS, W, WS = rec.A, rec.R, rec.D, rec.S, rec.COL, rec.B, rec.WS
    for capturing in (0, 1):
        rec.fake.rec_capturing(capturing)
        for _ in range(20000):
            group = rng.choice((32, 64, 128))
            call("sg_int4_gemm", X, W, D, between(rng, 1, 140), between(rng, 1, 80000), group * between(rng, 1, 65536 // group), group, rng.randint(0, 3), None)
    rec.fake.rec_capturing(0)
    sizes = [(50, 2048, 1408, 512, 16)]                      # many choices: a plan that leaves fewer stages room
    for _ in range(9000):
        experts = between(rng, 1, 513)
        hidden, inner = (unit * between(rng, 1, 20000 // unit) for unit in (rng.choice((16, 128)), rng.choice((16, 128))))
        sizes.append((rng.randint(1, rng.choice((4, 9, 20, 64))), hidden, inner, experts, rng.randint(1, min(16, experts))))
    for i, (m, hidden, inner, experts, top_k) in enumerate(sizes):
        w = W + 16 * (i % 2)
        call("sg_moe_experts", X, IDS, S, w, None, w, None, D, m, hidden, inner, experts, top_k, WS, 1 << 30, None)
        call("sg_moe_layer", X, R, w, None, w, None, D, IDS, S, m, hidden, inner, experts, top_k, 1, WS, 1 << 30, None)
    for _ in range(5000):
        call("sg_rmsnorm_fp8_rows", X, None, None, None, None, D, S, C.c_float(1e-5), between(rng, 1, 40000), 16 * between(rng, 1, 8000), None)
    return sorted(names)


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("fake"))


def test_no_build_that_nothing_reaches(fake):
    symbols = subprocess.run(["nm", "-C", launch_recorder.LIBRARY], check=True, capture_output=True, text=True).stdout
    built = {"sg::" + x for x in re.findall(r"sg::__device_stub__((?:int4_gemm|int4_sum|moe_|rmsnorm)\w*(?:<[^(]*>)?)\(", symbols)}
    assert len(built) > 200
    missed = sorted(built - set(launch_recorder.scenario(fake, "test_reached_builds", "reached")))
    assert not missed, missed
