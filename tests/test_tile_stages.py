"""CPU: the roles of the tile kernel of the products with 4-bit weights (csrc/linear_4bit_tile.cu) around its stages, with barriers whose waits see a phase's parity
alone, as the hardware's do, in any order: no role passes a wait early, nothing waits for good.  The numbers are the source's."""
import random
import re

import pytest

from lookahead_keys_attention_b200 import _lib

SOURCE = (_lib.CSRC / "linear_4bit_tile.cu").read_text()
GROUPS = int(re.search(r"kTileGroups = (\d+)", SOURCE).group(1))
STAGES = [int(v) for v in re.search(r"p\.stages = p\.bn <= 128 \? (\d+) : (\d+)", SOURCE).groups()]


class Barrier:
    def __init__(self, count):
        self.count, self.arrived, self.phase = count, 0, 0

    def arrive(self):
        self.arrived += 1
        if self.arrived == self.count:
            self.arrived, self.phase = 0, self.phase + 1

    def over(self, parity):      # whether the phase before the running one has that parity
        return (self.phase - 1) % 2 == parity


def _roles(groups, stages, chunks, rng):
    full, free = [Barrier(5) for _ in range(stages)], [Barrier(1) for _ in range(stages)]
    issued, ended = [], [-1]

    def fill(first, step):       # a loading or an unpacking warp
        s, turn = first % stages, first // stages
        for c in range(first, chunks, step):
            if turn > 0:
                while not free[s].over((turn - 1) & 1):
                    yield
                assert ended[0] >= c - stages, "a stage is filled while its products are still to come"
            yield
            full[s].arrive()
            yield
            s += step
            while s >= stages:
                s, turn = s - stages, turn + 1

    def issue():
        s = turn = 0
        for c in range(chunks):
            while not full[s].over(turn & 1):
                yield
            issued.append((c, s))
            yield
            s += 1
            if s == stages:
                s, turn = 0, turn + 1

    def products():
        while ended[0] < chunks - 1:
            if issued and rng.random() < 0.3:
                ended[0], s = issued.pop(0)
                free[s].arrive()
            yield

    return [fill(0, 1), issue(), products()] + [fill(g, groups) for g in range(groups) for _ in range(4)]


def _run(groups, stages, seed):
    rng = random.Random(seed)
    roles, steps = _roles(groups, stages, rng.randint(1, 40), rng), 0
    while roles:
        role, steps = rng.choice(roles), steps + 1
        assert steps < 200000, "a wait without an end"
        for _ in range(rng.randint(1, 8)):
            try:
                next(role)
            except StopIteration:
                roles.remove(role)
                break


@pytest.mark.parametrize("stages", STAGES)
def test_no_wait_is_passed_early(stages):
    assert stages % GROUPS == 0
    for seed in range(150):
        _run(GROUPS, stages, seed)


def test_a_group_that_comes_to_a_stage_now_and_then_would_pass_one():
    failed = 0
    for seed in range(40):
        try:
            _run(4, 3, seed)
        except AssertionError:
            failed += 1
    assert failed > 10
