"""CPU: the roles of the paged step's CTA (csrc/paged.cu) around its barriers where waits run out: the warp that copies and the four that work, in any order, with
copies that take any time.  A barrier takes as many arrivals a phase as it was made for and no more, what is read has arrived and is not written meanwhile, nobody waits for
good, and none of the CTA's copies is on its way when its last warp has left."""
import random
import re

import pytest

from lookahead_keys_attention_b200 import _lib

SOURCE = (_lib.CSRC / "paged.cu").read_text()
STAGES = int(re.search(r"kPagedStages = (\d+)", SOURCE).group(1))
WARPS = int(re.search(r"kPagedThreads = (\d+)", SOURCE).group(1)) // 32


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.bytes, self.phase = count, count, 0, 0

    def arrive(self, expect=0):
        assert self.pending > 0, "an arrival that the phase has no place for"
        self.bytes += expect
        self.pending -= 1
        self._end()

    def landed(self):
        self.bytes -= 1
        self._end()

    def _end(self):
        if self.pending == 0 and self.bytes == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def over(self, parity):
        return (self.phase - 1) % 2 == parity


class Cta:
    """`patience`: polls after which a wait of the working warps runs out; `former`: the copying warp goes on arriving after that, and waits for its copies only if
    it has seen it; `forgets`: a working warp waits again after one of its waits ran out."""

    def __init__(self, rng, patience, former=False, forgets=False):
        self.rng, self.patience, self.former, self.forgets, self.abort, self.flight = rng, patience, former, forgets, False, []
        self.full, self.empty = [Barrier(1) for _ in range(STAGES)], [Barrier(WARPS) for _ in range(STAGES)]
        self.new_full, self.new_place, self.new_empty = [Barrier(1) for _ in range(2)], [Barrier(1) for _ in range(2)], [Barrier(WARPS) for _ in range(2)]
        self.segments = [(rng.randint(0, 5), rng.random() < 0.5) for _ in range(rng.randint(1, 6))]   # tiles with rows; whether the pair ends with it
        self.content, self.reading = [None] * STAGES, [0] * STAGES
        self.seen = [[] for _ in range(WARPS)]

    def copy(self, bar, stage=None, what=None):
        self.flight.append((bar, stage, what))

    def wait(self, bar, parity, patience):
        """What the wait's caller is told: whether the phase ended."""
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

    def copies(self):
        segments = count = 0
        over = False
        for tiles, _ in self.segments:
            slot = segments & 1
            if segments >= 2:
                yield from self.wait(self.new_empty[slot], ((segments >> 1) - 1) & 1, 10 ** 9)
            over = self.abort
            if over and not self.former:
                break
            self.new_full[slot].arrive(0 if over else 1)
            if not over:
                self.copy(self.new_full[slot])
            if not self.former:
                segments += 1
            yield
            for tile in range(tiles):
                st = count % STAGES
                if count >= STAGES:
                    yield from self.wait(self.empty[st], (count // STAGES - 1) & 1, 10 ** 9)
                over = self.abort
                if over and not self.former:
                    break
                yield
                if not over:
                    assert self.reading[st] == 0, "a stage is written while it is read"
                    self.content[st] = None
                self.full[st].arrive(0 if over else 1)
                if not over:
                    self.copy(self.full[st], st, count)
                count += 1
                yield
            if over and not self.former:
                break
            self.new_place[slot].arrive()
            if self.former:
                segments += 1
            yield
        if self.abort or not self.former:
            for bars, n, end in ((self.full, STAGES, count), (self.new_full, 2, segments)):
                for i in range(max(0, end - n), end):
                    while not bars[i % n].over((i // n) & 1):
                        yield

    def works(self, warp):
        segments = count = 0
        there = True
        for tiles, ends in self.segments:
            slot, turn = segments & 1, (segments >> 1) & 1
            segments += 1
            there = (there or self.forgets) and (yield from self.wait(self.new_full[slot], turn, self.patience))
            whole = there
            for _ in range(tiles):
                st = count % STAGES
                arrived = there and (yield from self.wait(self.full[st], (count // STAGES) & 1, self.patience))
                there = arrived or (there and self.forgets)
                whole = whole and arrived
                if arrived:
                    assert self.content[st] == count, "what is read has not arrived"
                    self.reading[st] += 1
                    yield
                    self.reading[st] -= 1
                self.empty[st].arrive()
                count += 1
                yield
            if ends and warp == 0 and there:
                there = whole = whole and (yield from self.wait(self.new_place[slot], turn, self.patience))
            self.new_empty[slot].arrive()
            self.seen[warp].append((whole, there))
            yield

    def run(self):
        roles, steps = [self.copies()] + [self.works(w) for w in range(WARPS)], 0
        slow = self.rng.choice([0.5, 0.05, 0.01])
        while roles:
            steps += 1
            assert steps < 100000, "a wait without an end"
            if self.flight and self.rng.random() < slow:
                bar, stage, what = self.flight.pop(self.rng.randrange(len(self.flight)))
                if stage is not None:
                    self.content[stage] = what
                bar.landed()
            role = self.rng.choice(roles)
            for _ in range(self.rng.randint(1, 6)):
                try:
                    next(role)
                except StopIteration:
                    roles.remove(role)
                    break
        assert not self.flight, "the CTA has left while its copies are on their way"


def test_without_one_that_runs_out():
    for seed in range(300):
        cta = Cta(random.Random(seed), 10 ** 9)
        cta.run()
        assert not cta.abort and all(all(whole for whole, _ in seen) for seen in cta.seen)


def test_where_waits_run_out():
    aborted = 0
    for seed in range(1500):
        rng = random.Random(seed)
        cta = Cta(rng, rng.choice([0, 1, 3, 10, 30, 100]))
        cta.run()
        aborted += cta.abort
        # a warp that has not got all of a segment's rows knows it at the segment's end
        assert all(whole or not there for seen in cta.seen for whole, there in seen)
    assert aborted > 500


def test_arrivals_after_it_would_be_more_than_a_phase_takes_and_copies_outlive_the_cta():
    found = set()
    for seed in range(1500):
        rng = random.Random(seed)
        try:
            Cta(rng, rng.choice([0, 1, 3, 10, 30, 100]), former=True).run()
        except AssertionError as e:
            found.add(str(e).splitlines()[0])
    assert found >= {"an arrival that the phase has no place for", "the CTA has left while its copies are on their way"}


def test_a_warp_that_forgets_would_read_what_has_not_arrived():
    found = set()
    for seed in range(1500):
        rng = random.Random(seed)
        try:
            Cta(rng, rng.choice([0, 1, 3, 10, 30, 100]), forgets=True).run()
        except AssertionError as e:
            found.add(str(e).splitlines()[0])
    assert found == {"what is read has not arrived"}


def test_the_source_plays_these_roles():
    """The copying warp looks at the flag behind each wait and leaves its loops, and its last waits are made in any case."""
    start = SOURCE.index("castle_paged_step_kernel(const")
    body = SOURCE[start:SOURCE.index("const int sub = lane % LPR", start)]
    look = "if ((over = __any_sync(0xffffffffu, *abortp != 0))) break;"
    waits = [m.end() for m in re.finditer(r"mbar_wait\(.*?abortp\);\s*", body)]
    assert len(waits) == 2 and all(body[at:].startswith(look) for at in waits) and "at < end && !over;" in body
    assert re.search(r"if \(over\) break;[^}]*mbar_arrive\(&new_place", body)
    end = body[body.index("paged_outside<T, D>(p, lengths);"):]
    assert end.count("mbar_drain(") == 2 and "abortp" not in end
    works = SOURCE[SOURCE.index("const int sub = lane % LPR", start):]
    waits = re.findall(r"(.*)mbar_wait_failed\(", works)
    assert len(waits) == 3 and all(w.strip() == "there = there && !" for w in waits)
