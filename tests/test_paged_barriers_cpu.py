"""The barriers of the many-row attention kernel (csrc/paged_attention_tc.cu) as a model: every warp
role is a coroutine that arrives at and waits for the same barriers in the same order, a scheduler
runs them in any order with some of them slowed down. A wait tells a barrier's phase from the one
before it only, as mbarrier parities do. Found this way: a product warp whose tile has no rows in a
piece could fall two phases of a barrier behind, unless a piece's end waits for it too."""
import random

import pytest

SOFTMAX, LOADERS, BATCH, BATCHES, PIECES = 8, 4, 8, 2, 4


class Fault(Exception):
    pass


class Bar:
    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0  # completed phases

    def arrive(self):
        self.left -= 1
        if not self.left:
            self.left, self.phase = self.count, self.phase + 1


class Model:
    def __init__(self, rng, stages, takes, end_waits_for_products, query_bars):
        self.rng, self.stages, self.takes = rng, stages, takes  # takes: blocks after which f32 sums move out (0: never)
        self.joined, self.query_bars = end_waits_for_products, query_bars
        few = rng.random() < 0.7  # mostly pieces of one or two key blocks
        idle = rng.choice([0, 0.3, 0.8])
        self.pieces = [(rng.choice([1, 1, 2, 3]) if few else rng.randint(1, 20), rng.random() < idle)
                       for _ in range(rng.randint(1, 14))] + [(-1, False)]  # key blocks, rows in tile 1
        counts = dict(Q=SOFTMAX, K=LOADERS, V=LOADERS, KF=2, VF=2, S=1, P=SOFTMAX // 2, PV=1, PIECE=1,
                      DONE=SOFTMAX + self.joined, PLAN=1, PF=2, ROUND=SOFTMAX)
        self.bars = {(name, i): Bar(c) for name, c in counts.items() for i in range(4)}
        self.places = [None] * PIECES

    def arrive(self, name, i=0):
        self.bars[name, i].arrive()

    def piece(self, k):
        at, p = self.places[k % PIECES]
        if at != k:
            raise Fault(f"piece {at} taken for {k}")
        return p

    def walker(self):
        for k, p in enumerate(self.pieces):
            if k >= PIECES:
                yield "DONE", k % PIECES, k // PIECES - 1
            self.places[k % PIECES] = k, p
            self.arrive("PIECE", k % PIECES)
            yield None

    def taken(self, k):
        return "PIECE", k % PIECES, k // PIECES

    def lookup(self):
        batch = k = 0
        while True:
            yield self.taken(k)
            n, _ = self.piece(k)
            if n < 0:
                return
            for _ in range(0, n, BATCH):
                if batch >= BATCHES:
                    yield "PF", batch % BATCHES, batch // BATCHES - 1
                yield None
                self.arrive("PLAN", batch % BATCHES)
                batch += 1
            k += 1

    def products(self, x):
        done = batch = mine = k = 0
        while True:
            yield self.taken(k)
            n, _ = self.piece(k)
            yield None
            active = x == 0 or self.piece(k)[1]
            if n < 0:
                return
            yield "Q", k % self.query_bars, k // self.query_bars
            for i in range(-2, n):
                now, ahead, t = done + i, done + i + 2, mine + i
                if i + 2 < n:
                    yield "K", ahead % self.stages, ahead // self.stages
                elif i >= 0:
                    yield "V", now % self.stages, now // self.stages
                if i >= 0:
                    if active:
                        yield "P", 2 * x + t % 2, t // 2
                        self.arrive("PV", 2 * x + t % 2)
                    self.arrive("VF", now % self.stages)
                    if i % BATCH == BATCH - 1 or i == n - 1:
                        self.arrive("PF", batch % BATCHES)
                        batch += 1
                if i + 2 < n:
                    if active:
                        self.arrive("S", 2 * x + t % 2)
                    self.arrive("KF", ahead % self.stages)
                yield None
            done += n
            mine += n if active else 0
            if x == 1 and self.joined:
                self.arrive("DONE", k % PIECES)
            k += 1

    def loader(self):
        done = batch = k = 0
        while True:
            yield self.taken(k)
            n, _ = self.piece(k)
            if n < 0:
                return
            for i in range(-1, n):
                if i + 1 < n and (i + 1) % BATCH == 0:
                    t = batch + (i + 1) // BATCH
                    yield "PLAN", t % BATCHES, t // BATCHES
                at = done + i
                for full, free in (("K", "KF"), ("V", "VF")) if i >= 0 else ():
                    if at >= self.stages:
                        yield free, at % self.stages, at // self.stages - 1
                    self.arrive(full, at % self.stages)
                    yield None
            done, batch, k = done + n, batch + -(-n // BATCH), k + 1

    def softmax(self, x):
        batch = mine = k = 0
        while True:
            yield self.taken(k)
            n, rows = self.piece(k)
            if n < 0:
                return
            active = x == 0 or rows
            self.arrive("Q", k % self.query_bars)
            yield None
            for i in range(n if active else 0):
                t, b = mine + i, batch + i // BATCH
                if i % BATCH == 0:
                    yield "PLAN", b % BATCHES, b // BATCHES
                yield "S", 2 * x + t % 2, t // 2
                if i and (self.takes and i % self.takes == 0 or self.rng.random() < 0.3):
                    yield "PV", 2 * x + (t - 1) % 2, (t - 1) // 2
                self.arrive("P", 2 * x + t % 2)
                yield None
            if active:
                mine += n
                yield "PV", 2 * x + (mine - 1) % 2, (mine - 1) // 2
            self.arrive("ROUND")
            yield "ROUND", 0, k
            self.piece(k)
            batch += -(-n // BATCH)
            self.arrive("DONE", k % PIECES)
            yield None
            k += 1

    def run(self):
        """None, or what went wrong."""
        roles = {"walker": self.walker(), "lookup": self.lookup(), "products 0": self.products(0), "products 1": self.products(1)}
        roles.update({f"loader {i}": self.loader() for i in range(LOADERS)})
        roles.update({f"softmax {i}": self.softmax(i // 4) for i in range(SOFTMAX)})
        speed = {r: self.rng.choice([1, 1, 1, 0.1, 0.003]) for r in roles}
        speed["products 1"] = self.rng.choice([1, 0.1, 0.003, 0.0005])
        at = dict.fromkeys(roles)
        while roles:
            ready = [r for r in roles if at[r] is None or self.bars[at[r][:2]].phase % 2 != at[r][2] % 2]
            if not ready:
                return f"everyone waits: {at}"
            r = self.rng.choices(ready, [speed[r] for r in ready])[0]
            if at[r] and self.bars[at[r][:2]].phase <= at[r][2]:
                return f"{r} passed {at[r]} early"
            try:
                at[r] = next(roles[r])
            except StopIteration:
                del roles[r], at[r]
            except Fault as e:
                return f"{r}: {e}"
        return None


def outcomes(runs, **kw):
    found = []
    for seed in range(runs):
        model = Model(random.Random(seed), stages=(2, 4)[seed % 2], takes=(0, 4)[seed // 2 % 2], **kw)
        found.append(model.run())
    return found


def test_no_schedule_confuses_phases():
    assert outcomes(1500, end_waits_for_products=True, query_bars=PIECES) == [None] * 1500


@pytest.mark.parametrize("query_bars", [2, PIECES])
def test_the_model_shows_what_the_arrival_of_the_products_is_for(query_bars):
    assert any(outcomes(200, end_waits_for_products=False, query_bars=query_bars))


def test_more_places_than_query_barriers_are_shown():
    assert any(outcomes(600, end_waits_for_products=True, query_bars=2))
