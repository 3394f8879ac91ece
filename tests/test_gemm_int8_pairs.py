"""The hand-overs of the 8-bit product's pairs of CTAs, on the CPU: the roles as they wait and arrive, run in random orders, copies and products that complete late, waits that may give up.

The model follows gemm_int8_pair_kernel in avelang_b200/csrc/gemm_int8.cu role by role.  Undisturbed, every tile is finished, no stage is filled before its products are done, no accumulator is
overwritten before all warps have read it, and nothing is on its way when the CTAs end; a wait that gives up ends every role, again with nothing on its way into a CTA that has ended."""
import random

import pytest

WARPS = 8  # that finish results, a CTA


class Barrier:  # an mbarrier: arrivals and bytes; a wait sees the parity of the last phase that completed
    def __init__(self, count):
        self.count, self.left, self.tx, self.phase = count, count, 0, 0

    def settle(self):
        assert self.left >= 0, "an arrival too many in one phase"
        if self.left == 0 and self.tx == 0:
            self.left, self.phase = self.count, self.phase + 1

    def arrive(self, expect=0):
        self.left -= 1
        self.tx += expect
        self.settle()

    def complete(self, n):
        self.tx -= n
        self.settle()

    def passed(self, parity):
        return (self.phase & 1) != parity


class Pair:
    def __init__(self, rng, tiles, blocks, stages, narrow, give_up):
        self.rng, self.tiles, self.kb, self.S, self.narrow, self.give_up = rng, tiles, blocks, stages, narrow, give_up
        B = Barrier
        self.full = [B(1) for _ in range(stages)]
        self.empty = [[B(1) for _ in range(stages)] for _ in range(2)]
        self.acc_full = [[B(1), B(1)] for _ in range(2)]
        self.acc_empty = [B(2 * WARPS), B(2 * WARPS)]
        self.drained = [B(1), B(1)]
        self.abort = [False, False]
        self.issued = [0, 0]
        self.copies, self.tensor = [], []           # on their way: copies in any order, products and commits in theirs
        self.slot = [[None] * stages for _ in range(2)]  # what a stage holds: (block index, landed)
        self.reading = [[None] * stages for _ in range(2)]
        self.accumulator = [None, None]             # the tile whose sums it holds
        self.read = {}                              # (tile, rank) -> warps that have them
        self.met, self.finished = [], []

    def wait(self, rank, bar, parity):              # yields until it has passed or given up
        polls = 0
        while not bar.passed(parity):
            polls += 1
            if self.abort[rank] or (self.give_up and polls > self.give_up):
                self.abort[rank] = True
                return False
            if not self.give_up:
                assert polls < 200000, "a role waits for good"
            yield
        return True

    def producer(self, rank):
        s, ph, turns, ok = 0, 0, 0, True
        for _ in range(self.tiles):
            for _ in range(self.kb):
                ok = yield from self.wait(rank, self.empty[rank][s], ph ^ 1)
                if not ok:
                    break
                assert self.reading[rank][s] is None, "a stage is filled under its products"
                if rank == 0:
                    self.full[s].arrive(expect=2)
                self.slot[rank][s] = (turns, False)
                self.copies.append((rank, s, turns))
                yield
                turns += 1
                s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)
            if not ok:
                break
        if ok:
            for _ in range(min(self.S, turns)):
                if not (yield from self.wait(rank, self.empty[rank][s], ph ^ 1)):
                    break
                s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)
        self.issued[rank] = turns

    def issuer(self):
        s, ph, block, ok = 0, 0, 0, True
        for tile in range(self.tiles):
            buf = tile & 1
            ok = yield from self.wait(0, self.acc_empty[buf], ((tile >> 1) & 1) ^ 1)
            if not ok:
                break
            before = self.accumulator[buf]
            assert before is None or all(self.read.get((before, r), 0) == WARPS for r in (0, 1)), "sums overwritten before they are read"
            for _ in range(self.kb):
                ok = yield from self.wait(0, self.full[s], ph)
                if not ok:
                    break
                for r in (0, 1):
                    assert self.slot[r][s] == (block, True), "products of a stage that has not landed"
                    self.reading[r][s] = block
                self.tensor.append(("free", s))
                yield
                block += 1
                s, ph = (0, ph ^ 1) if s + 1 == self.S else (s + 1, ph)
            if not ok:
                break
            self.tensor.append(("tile", buf, tile))
            yield

    def finisher(self, rank, warp):
        for tile in range(self.tiles):
            buf = tile & 1
            if not (yield from self.wait(rank, self.acc_full[rank][buf], (tile >> 1) & 1)):
                return
            assert self.accumulator[buf] == tile
            if not (self.narrow and warp >= WARPS // 2):  # (a narrow last tile has no chunk for the second half of the warps)
                yield
            self.read[tile, rank] = self.read.get((tile, rank), 0) + 1
            self.acc_empty[buf].arrive()
            yield
        self.finished.append((rank, warp))

    def land(self):  # something that is on its way arrives
        if self.copies and (not self.tensor or self.rng.random() < 0.5):
            rank, s, i = self.copies.pop(self.rng.randrange(len(self.copies)))
            assert self.slot[rank][s] == (i, False)
            self.slot[rank][s] = (i, True)
            self.full[s].complete(1)
        elif self.tensor:
            what = self.tensor.pop(0)
            if what[0] == "free":
                for r in (0, 1):
                    self.reading[r][what[1]] = None
                    self.empty[r][what[1]].arrive()
            elif what[0] == "tile":
                self.accumulator[what[1]] = what[2]
                for r in (0, 1):
                    self.acc_full[r][what[1]].arrive()
            else:
                for r in (0, 1):
                    self.drained[r].arrive()

    def settle(self):  # the leader, behind the first meeting of both CTAs, where a wait has given up
        own, other = self.issued
        total = max(own, other)
        for i in range(own, other):
            self.full[i % self.S].arrive(expect=1)
        for i in range(other, own):
            self.full[i % self.S].complete(1)
        for i in range(max(0, total - self.S), total):
            while not self.full[i % self.S].passed((i // self.S) & 1):
                yield
        self.tensor.append(("drained",))
        while not self.drained[0].passed(0):
            yield

    def run(self, slow):
        roles = {("producer", r): self.producer(r) for r in (0, 1)}
        roles["issuer", 0] = self.issuer()
        roles.update({("finisher", r, w): self.finisher(r, w) for r in (0, 1) for w in range(WARPS)})
        speed = {k: self.rng.choice([1, 1, 4, 30]) for k in roles}
        steps = 0
        while roles:
            steps += 1
            assert steps < 3000000
            if self.rng.random() < slow:
                self.land()
            k = self.rng.choice(list(roles))
            if self.rng.random() * speed[k] > 1:
                continue
            try:
                next(roles[k])
            except StopIteration:
                del roles[k]
        if any(self.abort):
            for _ in self.settle():
                steps += 1
                assert steps < 3000000, "the leader waits for what nobody has asked for"
                self.land()
        assert not self.copies and not self.tensor, "copies or products on their way in CTAs that have ended"


@pytest.mark.parametrize("tiles,blocks,stages,narrow", [(1, 1, 5, False), (1, 7, 2, True), (3, 4, 5, False), (5, 3, 3, True), (4, 9, 9, False), (6, 1, 2, False)])
def test_every_order_ends(tiles, blocks, stages, narrow):
    for seed in range(40):
        pair = Pair(random.Random(seed), tiles, blocks, stages, narrow, None)
        pair.run(0.6)
        assert len(pair.finished) == 2 * WARPS and all(pair.read[t, r] == WARPS for t in range(tiles) for r in (0, 1))
        assert pair.issued == [tiles * blocks] * 2 and not any(pair.abort)


@pytest.mark.parametrize("tiles,blocks,stages", [(2, 4, 3), (3, 5, 5), (4, 2, 2)])
def test_a_wait_that_gives_up_ends_everything(tiles, blocks, stages):
    ended = whole = 0
    for seed in range(150):
        rng = random.Random(seed)
        pair = Pair(rng, tiles, blocks, stages, False, rng.choice([3, 10, 40, 200]))
        pair.run(rng.choice([0.02, 0.1, 0.4]))
        ended += any(pair.abort)
        whole += not any(pair.abort)
    assert ended > 20 and whole > 5
