"""The hand-offs of the paired products (csrc/tkv_vloss_tc.cu) as a simulation: two CTAs' copies, the even CTA's products, sixteen warps of
the epilogue, mbarriers with arrivals and byte counts, copies that land and products that finish at any later time.

Checked at every event: a copy never lands in a stage that a product has yet to read; a product reads what both CTAs fetched for its step;
a sum starts in an accumulator only when every warp has read the last one there; a warp reads whole sums; everything ends."""
import random

import pytest

STAGES, WARPS = 6, 8


class Bar:
    """An mbarrier: phase completes when its arrivals and bytes are there."""

    def __init__(self, count):
        self.count = self.pending = count
        self.tx = self.phase = 0

    def _check(self):
        if self.pending == 0 and self.tx == 0:
            self.phase ^= 1
            self.pending = self.count

    def arrive(self):
        assert self.pending > 0, "more arrivals than the barrier counts"
        self.pending -= 1
        self._check()

    def expect(self, n):
        self.tx += n
        self.arrive()

    def land(self, n):
        self.tx -= n
        self._check()

    def passed(self, parity):
        return self.phase != parity


class Pair:
    def __init__(self, tiles, sum_steps, rng, fault=None):
        self.tiles, self.sum_steps, self.rng, self.fault = tiles, sum_steps, rng, fault
        self.full = [Bar(1) for _ in range(STAGES)]                             # of the even CTA
        self.empty = [[Bar(1) for _ in range(STAGES)] for _ in range(2)]
        self.acc_full = [[Bar(1) for _ in range(2)] for _ in range(2)]
        self.acc_empty = [Bar(2 * WARPS) for _ in range(2)]                     # of the even CTA
        self.stage = [[None] * STAGES for _ in range(2)]                        # step that a CTA's part of a stage holds
        self.unread = [0] * STAGES                                              # products issued that have yet to read a stage
        self.sums = [[] for _ in range(2)]                                      # steps that an accumulator holds
        self.readers = [0, 0]                                                   # warps that have yet to read it
        self.copies, self.products = [], []                                     # in flight; products finish in order

    def producer(self, rank):
        it = 0
        for tile, steps in enumerate(self.tiles):
            for k in range(steps):
                s = it % STAGES
                if self.fault != "no empty wait":
                    yield lambda s=s, it=it: self.empty[rank][s].passed(((it // STAGES) & 1) ^ 1)
                if rank == 0:
                    self.full[s].expect(2)
                self.copies.append((rank, s, (tile, k)))
                it += 1
                yield None
        for i in range(max(0, it - STAGES), it):
            yield lambda i=i: self.empty[rank][i % STAGES].passed((i // STAGES) & 1)

    def land(self, i):
        rank, s, step = self.copies.pop(i)
        assert self.unread[s] == 0, "a copy landed where a product had yet to read"
        self.stage[rank][s] = step
        self.full[s].land(1)

    def issuer(self):
        it = acc = 0
        for tile, steps in enumerate(self.tiles):
            in_sum = 0
            for k in range(max(steps, 1)):
                buf = acc & 1
                if in_sum == 0 and self.fault != "no accumulator wait":
                    yield lambda: self.acc_empty[buf].passed(((acc >> 1) & 1) ^ 1)
                s = it % STAGES
                if steps:
                    yield lambda: self.full[s].passed((it // STAGES) & 1)
                last = in_sum == self.sum_steps - 1 or k >= steps - 1
                if steps:
                    self.unread[s] += 1
                    self.products.append(("product", s, buf, (tile, k), in_sum == 0))
                    self.products.append(("empty", s))
                    it += 1
                if last:
                    self.products.append(("full", buf))
                in_sum += 1
                if last:
                    in_sum, acc = 0, acc + 1
                yield None

    def finish(self):
        kind, *what = self.products.pop(0)
        if kind == "product":
            s, buf, step, first = what
            assert self.stage[0][s] == self.stage[1][s] == step, "a product read another step"
            if first:
                assert self.readers[buf] == 0, "a sum started over one that was yet to be read"
                self.sums[buf] = []
            self.sums[buf].append(step)
            self.unread[s] -= 1
        elif kind == "empty":
            for rank in range(2):
                self.empty[rank][what[0]].arrive()
        else:
            self.readers[what[0]] = 2 * WARPS
            for rank in range(2):
                self.acc_full[rank][what[0]].arrive()

    def reader(self, rank):
        acc = 0
        for tile, steps in enumerate(self.tiles):
            got = []
            for k in range(0, max(steps, 1), self.sum_steps):
                buf = acc & 1
                yield lambda: self.acc_full[rank][buf].passed((acc >> 1) & 1)
                if steps:
                    want = [(tile, j) for j in range(k, min(k + self.sum_steps, steps))]
                    assert self.sums[buf] == want, "a warp read part of a sum"
                    got += want
                yield None
                self.readers[buf] -= 1
                self.acc_empty[buf].arrive()
                acc += 1
            assert len(got) == steps

    def run(self):
        actors = [self.producer(0), self.producer(1), self.issuer()] + [self.reader(r) for r in range(2) for _ in range(WARPS)]
        waiting = {i: None for i in range(len(actors))}
        while waiting or self.copies or self.products:
            ready = [i for i, c in waiting.items() if c is None or c()]
            events = [("actor", i) for i in ready] + [("copy", i) for i in range(len(self.copies))] + ([("product", 0)] if self.products else [])
            assert events, "nothing can go on"
            kind, i = self.rng.choice(events)
            if kind == "actor":
                try:
                    waiting[i] = next(actors[i])
                except StopIteration:
                    del waiting[i]
            elif kind == "copy":
                self.land(i)
            else:
                self.finish()


TILES = [[1], [0, 0, 0], [5, 0, 7, 1], [16, 16, 16], [13, 2, 2, 2, 2, 30], [6, 12, 18], [1] * 9]


@pytest.mark.parametrize("tiles", TILES)
@pytest.mark.parametrize("sum_steps", [1, 2, 16, 2 ** 31 - 1])
def test_every_order_of_events_is_safe_and_ends(tiles, sum_steps):
    for seed in range(12):
        Pair(tiles, sum_steps, random.Random(seed)).run()


@pytest.mark.parametrize("fault", ["no empty wait", "no accumulator wait"])
def test_the_simulation_finds_a_missing_wait(fault):
    found = 0
    for seed in range(20):
        try:
            Pair([16, 16, 16], 2, random.Random(seed), fault).run()
        except AssertionError:
            found += 1
    assert found > 10


PAIRS = 74


def _deal(dx, dw, extra):
    """The tiles of every pair as VtTiles deals them out: dx tiles 0 .., dw tiles dx .."""
    more = dx % PAIRS
    fewer = PAIRS - more
    extra = min(extra, dw // fewer) if more else 0
    out = []
    for pair in range(PAIRS):
        mine, tile, turn = [], pair - PAIRS, 0
        while True:
            if tile + PAIRS < dx:
                tile += PAIRS
                mine.append(tile)
                continue
            tile = dx
            own, j = 0 if pair < more else extra, turn
            turn += 1
            i = pair - more + fewer * j if j < own else extra * fewer + (pair + PAIRS - more) % PAIRS + PAIRS * (j - own)
            if i >= dw:
                break
            mine.append(dx + i)
        out.append(mine)
    return out


def test_every_tile_of_the_gradients_is_dealt_once_and_the_busiest_pair_is_known():
    """And the work of the busiest pair is what vloss_rows_grad_kernel chooses the number of shares by."""
    rng = random.Random(0)
    for _ in range(1500):
        dx = rng.choice([0, 1, 73, 74, 75, 128, rng.randrange(600)])
        dw = rng.choice([0, 1, rng.randrange(50), rng.randrange(3000)])
        cd, cw = rng.randrange(1, 500), rng.randrange(1, 200)
        more = dx % PAIRS
        fewer = PAIRS - more
        x = min(cd // cw, dw // fewer) if more else 0
        for extra in (x, x + rng.randrange(5)):                               # a last piece has fewer tiles than the choice was made for
            assert sorted(t for mine in _deal(dx, dw, extra) for t in mine) == list(range(dx + dw))
        worst = max(sum(cd if t < dx else cw for t in mine) for mine in _deal(dx, dw, x))
        rest = dw - x * fewer
        last = rest % PAIRS
        busy = (dx // PAIRS + 1) * cd + (rest // PAIRS + (last > fewer)) * cw if more else 0
        idle = dx // PAIRS * cd + (x + rest // PAIRS + (last > 0)) * cw
        assert worst == max(busy, idle)
