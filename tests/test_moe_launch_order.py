"""Host threads that call the experts' entry points on one stream with one workspace: a call's launches hand each other logits, the
plan, h and partial sums through it, so they stay together (no GPU: the calls run on a stand-in for the runtime, on which every
launch takes long enough for another thread to get in between)."""
import threading

import launch_recorder
import pytest

THREADS, CALLS = 3, 5
# entry: what a call launches, in order; m, hidden, inner, experts, top_k (the second layer chooses in a launch of its own, and its down
# projections' tiles are shared, so that their sums are added up by another one)
CALLS_OF = {
    "route": (["moe_logits", "moe_choose"], (12, 512, 16, 64, 4)),
    "experts": (["moe_gate_up", "moe_down", "moe_sum"], (61, 2064, 1376, 40, 6)),
    "layer": (["moe_logits", "moe_gate_up", "moe_down"], (4, 4096, 14336, 8, 2)),
    "larger layer": (["moe_logits", "moe_choose", "moe_gate_up", "moe_down", "moe_sum"], (61, 2064, 1376, 40, 6)),
}


def threads_on_one_stream(rec, kinds):
    """kinds[i % len(kinds)] on thread i; [[kernel, thread]] in the order of the launches"""
    rec.fake.rec_pause(300)
    start = threading.Barrier(THREADS)
    codes = []
    X, R, D, S, IDS, W, WS = rec.A, rec.R, rec.D, rec.S, rec.COL, rec.B, rec.WS

    def work(kind):
        m, hidden, inner, experts, top_k = CALLS_OF[kind][1]
        start.wait()
        for _ in range(CALLS):
            if kind == "route":
                codes.append(rec.call("sg_moe_route", X, R, IDS, S, m, hidden, experts, top_k, 1, WS, 1 << 30, None))
            elif kind == "experts":
                codes.append(rec.call("sg_moe_experts", X, IDS, S, W, None, W, None, D, m, hidden, inner, experts, top_k, WS, 1 << 30, None))
            else:
                codes.append(rec.call("sg_moe_layer", X, R, W, None, W, None, D, IDS, S, m, hidden, inner, experts, top_k, 1, WS, 1 << 30, None))

    threads = [threading.Thread(target=work, args=(kinds[i % len(kinds)],)) for i in range(THREADS)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert codes == [0] * (THREADS * CALLS), codes
    return [[x[0], x[4]] for x in rec.launches()]


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return launch_recorder.build(tmp_path_factory.mktemp("fake"))


@pytest.mark.parametrize("kinds", [["route"], ["experts"], ["layer"], ["larger layer"], ["route", "layer", "larger layer"]])
def test_the_launches_of_a_call_stay_together(fake, kinds):
    launches = launch_recorder.scenario(fake, "test_moe_launch_order", "threads_on_one_stream", kinds)
    threads = {t for _, t in launches}
    assert len(threads) == THREADS
    names = [next(n for n in ("moe_logits", "moe_choose", "moe_gate_up", "moe_down", "moe_sum") if n in kernel) for kernel, _ in launches]
    orders = [CALLS_OF[kind][0] for kind in kinds]
    at = calls = 0
    while at < len(launches):
        # one whole call: the launches of one thread, as one of the entry points makes them (the longest that fits)
        fits = [o for o in orders if names[at:at + len(o)] == o and len({t for _, t in launches[at:at + len(o)]}) == 1]
        assert fits, (names[at:at + 5], [t for _, t in launches[at:at + 5]])
        at += max(len(o) for o in fits)
        calls += 1
    assert calls == THREADS * CALLS
