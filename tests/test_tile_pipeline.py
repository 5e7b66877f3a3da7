"""The barriers of the attention kernel for many query rows (csrc/kv_tiles.cu),
stepped on the CPU under schedules that hold a role back as long as anything
else can move.  Every run has to end, and every role has to find in a ring's
place what belongs to its tile.

A wait on an mbarrier names a phase by its parity alone: it returns when the
phase with that parity is the last one completed.  So a role that waits for a
phase must be one without which the phase after it cannot complete.
"""
import random

import pytest


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def done(self, parity):
        return self.phase & 1 != parity


class Meeting:
    """A named barrier of the two warps that share rows."""

    def __init__(self):
        self.here, self.round = 0, 0


class Kernel:
    """One CTA's roles as generators: they yield a condition to wait for, or
    None where another role may go on before them.  `gate`: the scores of a
    tile wait for its blocks' scales."""

    WARPS = 2  # of each kind that arrives with several warps

    def __init__(self, count, used, apart, gate, rng):
        self.count, self.used, self.apart, self.gate, self.rng = count, used, apart, gate, rng
        n = self.WARPS
        self.k_full, self.v_full = ([Barrier(n) for _ in range(2)] for _ in range(2))
        self.k_free, self.v_free = ([Barrier(used) for _ in range(2)] for _ in range(2))
        self.q_full, self.s_read, self.p_full, self.turn = ([Barrier(2 * n) for _ in range(2)] for _ in range(4))
        self.s_full, self.o_done = ([Barrier(1) for _ in range(2)] for _ in range(2))
        self.info_full = [Barrier(1) for _ in range(4)]
        self.k, self.v, self.info = [[None] * n for _ in range(2)], [[None] * n for _ in range(2)], [None] * 4
        self.scores, self.weights, self.sums = [None, None], [[None] * 2 * n for _ in range(2)], [-1, -1]
        self.pipe = []  # products in flight: (work, barriers), in order
        self.meet = [[Meeting() for _ in range(n)] for _ in range(2)]
        self.roles = {"info": self.bring_info()}
        for w in range(n):
            self.roles[f"convert{w}"] = self.convert(w)
        for t in range(used):
            self.roles[f"mma{t}"] = self.products(t)
            for half in range(2):
                for w in range(n):
                    self.roles[f"softmax{t}.{half}.{w}"] = self.softmax(t, half, w)

    def bring_info(self):
        for i in range(self.count):
            yield None  # the table's and the scales' latency
            if i >= 2:
                yield lambda: self.k_free[i & 1].done(((i >> 1) & 1) ^ 1)
            self.info[i & 3] = i
            self.info_full[i & 3].arrive()

    def convert(self, w):
        for i in range(self.count):
            for full, free, place in ((self.k_full, self.k_free, self.k), (self.v_full, self.v_free, self.v)):
                if i >= 2:
                    yield lambda: free[i & 1].done(((i >> 1) & 1) ^ 1)
                place[i & 1][w] = i
                yield None
                full[i & 1].arrive()

    def products(self, t):
        def scores(i):
            def work():
                assert self.k[i & 1] == [i] * self.WARPS, "keys of another tile"
                self.scores[t] = i
            self.pipe.append((work, [self.s_full[t], self.k_free[i & 1]]))

        def output(i):
            def work():
                assert self.v[i & 1] == [i] * self.WARPS, "values of another tile"
                assert self.weights[t] == [i] * 2 * self.WARPS, "weights of another tile"
                self.sums[t] = i
            self.pipe.append((work, [self.o_done[t], self.v_free[i & 1]]))

        def next_scores(i, before):
            yield lambda: self.k_full[i & 1].done((i >> 1) & 1)
            if self.gate:
                yield lambda: self.info_full[i & 3].done((i >> 2) & 1)
            if before is not None:
                yield lambda: before.done((i - 1) & 1)
            scores(i)

        yield lambda: self.q_full[t].done(0)
        yield from next_scores(0, None)
        for i in range(self.count):
            if self.apart and i + 1 < self.count:
                yield from next_scores(i + 1, self.s_read[t])
            yield lambda: self.v_full[i & 1].done((i >> 1) & 1)
            yield lambda: self.p_full[t].done(i & 1)
            output(i)
            if not self.apart and i + 1 < self.count:
                yield from next_scores(i + 1, self.o_done[t])

    def together(self, t, w):
        m = self.meet[t][w]
        mine = m.round
        m.here += 1
        if m.here == 2:
            m.here, m.round = 0, m.round + 1
        yield lambda: m.round != mine

    def softmax(self, t, half, w):
        self.q_full[t].arrive()
        for i in range(self.count):
            yield lambda: self.info_full[i & 3].done((i >> 2) & 1)
            yield lambda: self.s_full[t].done(i & 1)
            if self.used == 2 and i + t > 0:
                yield lambda: self.turn[t].done((i + t - 1) & 1)
            raised = i == 0 or self.rng.random() < 0.2
            for again in range(2 if raised and i > 0 else 1):
                assert self.scores[t] == i and self.info[i & 3] == i, "scores or scales of another tile"
                yield None
                if again == 0 and self.used == 2:
                    self.turn[t ^ 1].arrive()
                if again == 1 and self.apart:
                    yield lambda: self.o_done[t].done((i - 1) & 1)
                if again == 1:
                    assert self.sums[t] == i - 1, "sums raised before they are complete"
            yield from self.together(t, w)
            if self.apart:
                self.s_read[t].arrive()
                if i > 0:
                    yield lambda: self.o_done[t].done((i - 1) & 1)
            elif i > 0:
                assert self.sums[t] == i - 1
            self.weights[t][half * self.WARPS + w] = i
            yield None
            assert self.info[i & 3] == i, "scales of another tile"
            self.p_full[t].arrive()
        if self.count:
            yield lambda: self.o_done[t].done((self.count - 1) & 1)
            assert self.sums[t] == self.count - 1

    def run(self, held):
        """True if every role ends.  `held` takes a step only when nothing else can."""
        waits = {name: next(role, "end") for name, role in self.roles.items()}
        while any(w != "end" for w in waits.values()):
            ready = [n for n, w in waits.items() if w is None or w != "end" and w()]
            if self.pipe:
                ready.append("pipe")
            first = [n for n in ready if n != held] or ready
            if not first:
                return False
            name = self.rng.choice(first)
            if name == "pipe":
                work, barriers = self.pipe.pop(0)
                work()
                for b in barriers:
                    b.arrive()
            else:
                waits[name] = next(self.roles[name], "end")
        return True


def _held(used, n=Kernel.WARPS):
    names = [None, "info", "pipe", *(f"convert{w}" for w in range(n))]
    for t in range(used):
        names += [f"mma{t}", *(f"softmax{t}.{half}.{w}" for half in range(2) for w in range(n))]
    return names


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("used", [1, 2])
def test_every_schedule_ends(apart, used):
    for held in _held(used):
        for seed in range(12):
            for count in (1, 2, 3, 5, 17):
                rng = random.Random(f"{seed} {held} {count}")
                assert Kernel(count, used, apart, True, rng).run(held), (held, seed, count)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("used", [1, 2])
def test_scales_that_nothing_waits_for_can_be_overtaken(apart, used):
    """The planted mistake: without the gate the scores of a tile complete while
    its scales are on their way, and the warp that brings them waits for a
    parity that the barrier has passed twice."""
    ended = [Kernel(17, used, apart, False, random.Random(seed)).run("info") for seed in range(20)]
    assert not all(ended)
