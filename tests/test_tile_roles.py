"""CPU: the roles of the tile kernel of the products with 4-bit weights (csrc/linear_4bit_tile.cu) where waits run out, in any order, with copies and products that take any
time: a barrier takes as many arrivals a phase as it was made for and no more, nobody waits for good, and neither copies nor products are on their way when the CTA leaves."""
import random
import re

import pytest
from test_paged_roles import Barrier

from lookahead_keys_attention_b200 import _lib

SOURCE = (_lib.CSRC / "linear_4bit_tile.cu").read_text()
GROUPS = int(re.search(r"kTileGroups = (\d+)", SOURCE).group(1))
STAGES = [int(v) for v in re.search(r"p\.stages = p\.bn <= 128 \? (\d+) : (\d+)", SOURCE).groups()]
DRAIN = 3000   # polls of the loading thread's last waits here, for 2^16: longer than any copy takes


class Cta:
    """`patience`: polls after which the issuing thread's and the unpacking warps' waits run out; `former`: unpacking warps go on arriving after that, and the loading thread waits
    for its copies only if it has seen it."""

    def __init__(self, rng, stages, patience, former=False):
        self.rng, self.stages, self.patience, self.former, self.abort = rng, stages, patience, former, False
        self.full, self.free, self.done = [Barrier(5) for _ in range(stages)], [Barrier(1) for _ in range(stages)], Barrier(1)
        self.chunks, self.flight, self.issued, self.ran, self.left = rng.randint(1, 30), [], [], 0, False

    def wait(self, bar, parity, patience=10 ** 9):
        polls = 0
        while polls < patience:
            if bar.over(parity):
                return True
            if self.abort:
                return False
            polls += 1
            yield
        self.abort = True
        return False

    def loads(self):
        c = s = turn = 0
        while c < self.chunks:
            if turn > 0:
                yield from self.wait(self.free[s], (turn - 1) & 1)
            if self.abort:
                break
            self.full[s].arrive(1)
            self.flight.append(self.full[s])
            yield
            c, s = c + 1, s + 1
            if s == self.stages:
                s, turn = 0, turn + 1
        if self.abort or not self.former:
            last = [(i, p) for i in range(self.stages) for p in (0, 1)] if self.former else [(i % self.stages, i // self.stages & 1) for i in range(max(0, c - self.stages), c)]
            for i, parity in last:
                for _ in range(DRAIN):
                    if self.full[i].over(parity):
                        break
                    yield

    def issues(self):
        s = turn = 0
        for _ in range(self.chunks):
            yield from self.wait(self.full[s], turn & 1, self.patience)
            if self.abort:
                break
            self.issued.append(self.free[s])
            yield
            s += 1
            if s == self.stages:
                s, turn = 0, turn + 1
        self.issued.append(self.done)

    def unpacks(self, group):
        s, turn = group, 0
        for _ in range(group, self.chunks, GROUPS):
            if turn > 0 and not (yield from self.wait(self.free[s], (turn - 1) & 1, self.patience)) and not self.former:
                break
            yield
            self.full[s].arrive()
            yield
            s += GROUPS
            if s >= self.stages:
                s, turn = s - self.stages, turn + 1
        yield from self.wait(self.done, 0)
        while not self.done.over(0):     # (an abort: the products have ended before tensor memory is given back)
            yield

    def run(self):
        roles, steps = [self.loads(), self.issues()] + [self.unpacks(g) for g in range(GROUPS) for _ in range(4)], 0
        slow = self.rng.choice([0.5, 0.05, 0.02])
        while roles:
            steps += 1
            assert steps < 200000, "a wait without an end"
            if self.flight and self.rng.random() < slow:
                self.flight.pop(self.rng.randrange(len(self.flight))).landed()
            if self.issued and self.rng.random() < slow:
                self.issued.pop(0).arrive()
            role = self.rng.choice(roles)
            for _ in range(self.rng.randint(1, 6)):
                try:
                    next(role)
                except StopIteration:
                    roles.remove(role)
                    break
        assert not self.flight, "the CTA has left while its copies are on their way"
        assert not self.issued, "the CTA has left while its products are on their way"


def _patience(rng):
    return rng.choice([0, 1, 3, 10, 30, 100])


@pytest.mark.parametrize("stages", STAGES)
def test_without_one_that_runs_out(stages):
    for seed in range(40):
        cta = Cta(random.Random(seed), stages, 10 ** 9)
        cta.run()
        assert not cta.abort


@pytest.mark.parametrize("stages", STAGES)
def test_where_waits_run_out(stages):
    aborted = 0
    for seed in range(250):
        rng = random.Random(seed)
        cta = Cta(rng, stages, _patience(rng))
        cta.run()
        aborted += cta.abort
    assert aborted > 100


@pytest.mark.parametrize("stages", STAGES)
def test_arrivals_after_it_would_be_more_than_a_phase_takes(stages):
    found = set()
    for seed in range(250):
        rng = random.Random(seed)
        try:
            Cta(rng, stages, _patience(rng), former=True).run()
        except AssertionError as e:
            found.add(str(e).splitlines()[0])
    assert "an arrival that the phase has no place for" in found


def test_the_source_plays_these_roles():
    body = SOURCE[SOURCE.index("if (warp == kTileWarps) {"):SOURCE.index("// ---- the results")]
    loads, rest = body.split("} else if (warp == kTileWarps + 1) {")
    assert loads.count("if (*abortp) break;") == 1 and loads.count("abortp") == 2 and loads.count("mbar_drain(") == 1   # (the drain under no condition)
    unpacks = rest[rest.index("a weight row for each thread"):]
    assert unpacks.count("mbar_wait") == 1 and re.search(r"if \(turn > 0 && mbar_wait_failed\(&free_\[s\], .*abortp\)\) break;", unpacks)
