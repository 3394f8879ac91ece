"""The hand-overs of linear attention's scan, on the CPU: its roles as they wait and arrive, run in random orders.  A wait sees only the parity of a
barrier's phase, so a barrier that completes twice before one of its waiters has looked leaves that waiter behind for good.

The model follows avelang_b200/csrc/linear_scan.cuh role by role; it also notes reads and writes of the buffers that are handed over, and that each is
written only when it has been read."""
import random

import pytest

GROUPS = 2  # of four warps each, for the state and P'; one for the outputs and one for the images
STAGES = {"STATE": 4, "OUT2": 4, "OUT3": 4, "GRAD": 3}


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def seen(self, parity):  # phase - 1 is the last that completed
        return (self.phase & 1) != parity


class Scan:
    def __init__(self, mode, n, halves, ragged):
        self.mode, self.n, self.fh, self.ragged = mode, n, halves if mode == "GRAD" else 1, ragged
        halves = self.fh
        self.state, self.grad, self.shared = mode == "STATE", mode == "GRAD", mode != "OUT2"  # shared: outputs go where the scores were
        S = self.S = STAGES[mode]
        B = Barrier
        self.full, self.gates, self.empty = [B(1) for _ in range(S)], [B(1) for _ in range(S)], [B(4 * GROUPS + (1 if self.state else 4)) for _ in range(S)]
        self.p_full, self.pp_ready = B(1), B(6)
        self.img_ready, self.img_read = [B(4), B(4)], [B(1), B(1)]
        self.ds_full, self.ds_empty = [B(1), B(1)], [B(4 * GROUPS // halves), B(4 * GROUPS // halves)]
        self.h_ready, self.h_read, self.o_full, self.o_empty, self.cleared = B(4 * GROUPS), B(1), B(1), B(4), B(4)
        self.done = {}   # what has happened, as (what, chunk) -> times
        self.log = []

    def mark(self, what, c):
        self.done[what, c] = self.done.get((what, c), 0) + 1

    def need(self, what, c, times=1):
        assert c < 0 or self.done.get((what, c), 0) >= times, (self.mode, what, c)

    # a role yields lists of (barrier, parity) to wait for
    def loader(self):
        s, ph = 0, 1
        for c in range(self.n):
            if c >= self.S:
                yield [(self.empty[s], ph)]
            if not self.state:
                self.need("stored", c - self.S, 4)
            self.need("decayed", c - self.S, 4 * GROUPS)
            self.mark("loaded", c)
            self.full[s].arrive()
            s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)

    def gate(self):
        s, ph = 0, 1
        for c in range(self.n):
            if c >= self.S:
                yield [(self.empty[s], ph)]
            self.mark("gates", c)
            self.gates[s].arrive()
            s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)

    def images(self, w, group=0):
        s, ph = group, 0
        for c in range(group, self.n, 2 if self.state else 1):
            cp = c & 1
            yield [(self.full[s], ph), (self.gates[s], ph)]
            self.need("loaded", c); self.need("gates", c)
            if self.state:  # two groups, chunks and places in turn
                yield [(self.img_read[cp], (c >> 1 & 1) ^ 1)]
                self.need("increment", c - 2)
                self.mark("image0", c); self.mark("image1", c)
                self.img_ready[cp].arrive()
                s, ph = (s + 2 - self.S, ph ^ 1) if s + 2 >= self.S else (s + 2, ph)
                continue
            if c == self.ragged:
                self.cleared.arrive()
            for q in range(2):
                yield [(self.img_read[q], cp ^ 1)]
                self.need("increment", c - 1, self.fh)
                self.mark(f"image{q}", c)
                self.img_ready[q].arrive()
            s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)

    def issue_state(self):
        s = 0
        for c in range(self.n):
            cp = c & 1

            def part(f, q):
                self.need(f"image{q}", c, 4)
                self.need("drained%d" % (f if not (self.grad and self.fh == 2) else 1 - f), c - 1 if f == 0 or not self.grad else c, 4 * GROUPS // self.fh)
            if self.state:
                yield [(self.ds_empty[cp], (c >> 1 & 1) ^ 1), (self.img_ready[cp], c >> 1 & 1)]
                self.need("image1", c, 4); self.need("drained0", c - 2, 4 * GROUPS)
                self.mark("increment", c)
                for b in (self.ds_full[cp], self.img_read[cp], self.empty[s]):
                    b.arrive()
                s = 0 if s + 1 == self.S else s + 1
                continue
            if self.grad and self.fh == 2:
                yield [(self.ds_empty[1], cp ^ 1), (self.img_ready[0], cp), (self.img_ready[1], cp)]
                part(0, 0); part(0, 1)
                self.mark("increment", c)
                self.ds_full[0].arrive()
                yield [(self.ds_empty[0], cp)]
                part(1, 0); part(1, 1)
                self.mark("increment", c)
                for b in (self.img_read[0], self.img_read[1], self.ds_full[1]):
                    b.arrive()
            else:
                yield [(self.ds_empty[0], cp ^ 1), (self.img_ready[0], cp)]
                part(0, 0)
                self.mark("increment", c)
                self.img_read[0].arrive()
                yield [(self.img_ready[1], cp)]
                part(0, 1)
                self.ds_full[0].arrive()
                self.img_read[1].arrive()
            yield [(self.h_ready, cp), (self.o_empty, cp ^ 1)]
            self.need("published", c, 4 * GROUPS)
            self.need("taken", c - 1, 4)
            self.mark("inter", c)
            self.h_read.arrive()
            s = 0 if s + 1 == self.S else s + 1

    def issue_scores(self):
        def scores(c):
            self.need("loaded", c)
            self.need("weighed", c - 1, 6)
            if self.shared:
                self.need("taken", c - 1, 4)
            self.mark("scores", c)
            self.p_full.arrive()
        yield [(self.full[0], 0)]
        scores(0)
        s, ph = 0, 0
        for c in range(self.n):
            cp = c & 1
            s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)
            yield [(self.pp_ready, cp)] + self.outputs_gone(cp)
            if c == self.ragged:
                yield [(self.cleared, 0)]
            self.need("weighed", c, 6)
            self.need("taken", c - 1, 4)
            self.mark("intra", c)
            self.o_full.arrive()
            if c + 1 < self.n:
                yield [(self.full[s], ph)] + ([(self.o_empty, cp)] if self.shared else [])
                scores(c + 1)

    def outputs_gone(self, cp):
        return [] if self.shared else [(self.o_empty, cp ^ 1)]

    def states(self, w):
        half = w // 4 // (GROUPS // 2) if self.fh == 2 else 0
        part = w % 4 != 2
        s, ph = 0, 0
        for c in range(self.n):
            cp = c & 1
            def weigh():
                if part:
                    yield [(self.p_full, cp), (self.gates[s], ph), (self.o_full, cp ^ 1)]
                    self.need("scores", c); self.need("intra", c - 1); self.need("gates", c)
                    self.mark("weighed", c)
                    self.pp_ready.arrive()
            if not self.state:
                self.need("inter", c - 1)
                self.mark("published", c)
                self.h_ready.arrive()
                if not self.grad:
                    yield from weigh()
            at = cp if self.state else half
            yield [(self.ds_full[at], c >> 1 & 1 if self.state else cp)]
            self.need("increment", c, half + 1)
            self.mark(f"drained{half}", c)
            self.mark("decayed", c)
            self.ds_empty[at].arrive()
            self.empty[s].arrive()
            if self.grad:
                yield from weigh()
            s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)
            if not self.state and c + 1 < self.n:
                yield [(self.h_read, cp)]

    def outputs(self, w):
        s, before = 0, -1
        for c in range(self.n):
            cp = c & 1
            yield [(self.o_full, cp), (self.h_read, cp)]
            self.need("intra", c); self.need("inter", c)
            self.mark("taken", c)
            self.o_empty.arrive()
            if before >= 0:
                self.mark("stored", c - 1)
                self.empty[before].arrive()
            before, s = s, 0 if s + 1 == self.S else s + 1

    def run(self, rng):
        roles = [self.loader(), self.gate(), self.issue_state()] + [self.images(w) for w in range(4)] + [self.states(w) for w in range(4 * GROUPS)]
        if self.state:
            roles += [self.images(w, 1) for w in range(4)]
        else:
            roles += [self.issue_scores()] + [self.outputs(w) for w in range(4)]
        speed = [rng.choice([1, 1, 4, 30]) for _ in roles]  # some roles are slow for a while
        waiting = [None] * len(roles)
        live, stuck = set(range(len(roles))), 0
        while live:
            i = rng.choice(sorted(live))
            if rng.randrange(speed[i]):
                continue
            if rng.random() < 0.01:
                speed[i] = rng.choice([1, 1, 4, 30])
            if waiting[i] is not None and not all(b.seen(p) for b, p in waiting[i]):
                stuck += 1
                assert stuck < 20000, (self.mode, "roles that wait for good", sorted(live))
                continue
            stuck = 0
            try:
                waiting[i] = next(roles[i])
            except StopIteration:
                live.discard(i)


@pytest.mark.parametrize("mode", list(STAGES))
@pytest.mark.parametrize("halves", [1, 2])
def test_no_role_is_left_behind(mode, halves):
    rng = random.Random(5)
    for n in (1, 2, 3, 5, 9, 24):
        for trial in range(4):
            Scan(mode, n, halves, rng.choice([-1, n - 1, 0])).run(rng)


def test_the_model_sees_outputs_that_are_not_waited_for():
    class Early(Scan):
        def outputs_gone(self, cp):
            return []

    rng = random.Random(6)
    with pytest.raises(AssertionError):
        for trial in range(40):
            Early("OUT2", 24, 2, -1).run(rng)
