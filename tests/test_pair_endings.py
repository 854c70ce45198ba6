"""Pairs of CTAs in the loss's products: the first CTA's issuing thread commits to barriers of both, and an arrival in the second CTA's shared memory
takes as long as it likes.  The second CTA must not end before the last of them, or it lands in the memory of the next CTA on that SM.  On the CPU:
what the source says of a CTA's end, and the two CTAs played with arrivals of any delay, with and without an abort."""
import random
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parents[1] / "lookahead_keys_attention_b200" / "csrc" / "linear_ce.cu"


@pytest.fixture(scope="module")
def kernel():
    text = re.sub(r"//[^\n]*", "", SOURCE.read_text())
    start = text.index(") castle_ce_kernel(")
    return text[start:text.index("castle_ce_sum_kernel", start)]


def waits(kernel):
    """Whether the second CTA waits for its stages, and for the issuer's last commit behind the cluster's last barrier."""
    loader = kernel[kernel.index("if (warp == 0) {"):kernel.index("} else if (warp == 1) {")]
    stages = re.search(r"if \(rank == 1\)\s+for \(int j = 0; j < ring\.stages && !\*abortp; \+\+j, ring\.next\(\)\) mbar_wait_ok<true>\(&bar_free\[ring\.s\], ring\.phase \^ 1u, abortp\);",
                       loader[loader.rindex("load("):])
    last = re.search(r"if \(rank == 1 && tid == 0\) mbar_drain\(&bar_end, 0\);", kernel[kernel.rindex("cluster_sync();"):])
    return bool(stages), bool(last)


def test_what_the_source_says(kernel):
    assert waits(kernel) == (True, True)
    issuer = kernel[kernel.index("} else if (warp == 1) {"):kernel.index("} else {", kernel.index("mbar_drain(&bar_end, 0);"))]
    assert set(re.findall(r"commit\(&(\w+)", issuer)) == {"bar_free", "bar_done", "bar_end"}
    end = issuer[issuer.rindex("commit("):]
    assert end.startswith("commit(&bar_end)") and "mbar_drain(&bar_end, 0)" in end   # the last, and on every path
    indents = re.findall(r"\n( *)(?:for \(int i = 0; work|commit\(&bar_end\))", issuer)
    assert len(indents) == 2 and indents[0] == indents[1]


def play(steps, stages, flush, seed, abort, in_order, tail, last):
    """True: no arrival came after the second CTA's end.  in_order: arrivals at one CTA keep the commits' order."""
    rng = random.Random(seed)
    flying = []                       # [due, barrier] of the second CTA, in the order of the commits
    come = {"end": 0}                 # arrivals at the second CTA's barriers
    clock, issued, first_done = 0, 0, False
    stop = rng.randrange(steps) if abort else steps
    loaded = done = 0
    ended = None

    def commit(bar):
        due = clock + rng.choice([0, 1, 5, 60])
        if in_order and flying:
            due = max(due, flying[-1][0])
        flying.append([due, bar])

    while ended is None or flying:
        for f in [f for f in flying if f[0] <= clock]:
            if ended is not None:
                return False
            flying.remove(f)
            come[f[1]] = come.get(f[1], 0) + 1
        aborted = abort and issued >= stop
        if not first_done and rng.random() < 0.7:       # the first CTA's issuing thread; its own arrivals are there at once
            if issued < stop:
                commit(("free", issued % stages))
                issued += 1
                if issued % flush == 0 or issued == steps:
                    commit(("done", (issued + flush - 1) // flush - 1))
            else:
                commit("end")
                first_done = True
        if ended is None:
            if loaded < steps and not aborted and (loaded < stages or come.get(("free", loaded % stages), 0) > loaded // stages - 1):
                loaded += 1
            if done * flush < steps and not aborted and come.get(("done", done), 0):
                done += 1
            whole = loaded == steps and done * flush >= steps
            if tail and whole:
                whole = all(come.get(("free", s), 0) == len(range(s, steps, stages)) for s in range(min(stages, steps)))
            if (whole or aborted) and first_done and (not last or come["end"]):   # (both CTAs are at the cluster's barrier)
                ended = clock
        clock += 1
        if clock > 100000:
            return False
    return True


@pytest.mark.parametrize("steps,stages,flush", [(1, 6, 8), (5, 6, 8), (17, 6, 8), (40, 3, 1), (40, 6, 1 << 30)])
def test_no_arrival_after_the_end(kernel, steps, stages, flush):
    tail, last = waits(kernel)
    flush = min(flush, steps)
    for seed in range(200):
        assert play(steps, stages, flush, seed, False, False, tail, last)
        assert play(steps, stages, flush, seed, False, True, tail, last)
        assert play(steps, stages, flush, seed, True, True, tail, last)
    # the model does show the fault
    assert not all(play(steps, stages, flush, seed, False, True, False, False) for seed in range(200))
    assert not all(play(steps, stages, flush, seed, True, True, False, False) for seed in range(200))
