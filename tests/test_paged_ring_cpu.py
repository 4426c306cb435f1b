"""CPU test of the ring of K and V tiles of the paged attention for few rows (16-bit caches): a model of its roles and of an
mbarrier's phases, run in random order with copies that land in any order.  A wait has to pass only when what it names has
happened, and no barrier may get an arrival that its phase does not expect."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-v100_b200", "csrc",
                      "paged_few_kernel.cuh")


class Broken(Exception):
    pass


class Barrier:
    def __init__(self, count=1):
        self.count, self.pending, self.phase, self.landing = count, count, 0, 0

    def arrive(self, landing=0):
        if self.pending == 0:
            raise Broken("an arrival that the phase does not expect")
        self.pending -= 1
        self.landing += landing
        self.check()

    def landed(self):
        self.landing -= 1
        self.check()

    def check(self):
        if self.pending == 0 and self.landing == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def passed(self, parity):
        return self.phase & 1 != parity


class Ring:
    """``per_tile``: a full barrier belongs to a tile's K or V, not to a slot."""

    def __init__(self, stages, tiles, per_tile, rng):
        self.stages, self.tiles, self.per_tile, self.rng = stages, tiles, per_tile, rng
        self.k_full = [Barrier() for _ in range(stages)]
        self.v_full = [Barrier() for _ in range(stages)] if per_tile else self.k_full
        self.empty = [Barrier() for _ in range(stages)]
        self.s_full, self.s_free = [Barrier(), Barrier()], [Barrier(4), Barrier(4)]
        self.p_full, self.p_free = [Barrier(4), Barrier(4)], [Barrier(), Barrier()]
        self.holds = [None] * stages  # what has landed in a slot
        self.flying, self.done = [], set()

    def full(self, n, kind):
        """Barrier and parity of K (0) or V (1) of tile n."""
        at = 2 * n + kind
        i, turn = (n % self.stages, n // self.stages) if self.per_tile else (at % self.stages, at // self.stages)
        return (self.v_full if kind else self.k_full)[i], turn & 1

    def producer(self):
        for n in range(self.tiles):
            for kind in (0, 1):
                at = 2 * n + kind
                yield self.empty[at % self.stages], at // self.stages & 1 ^ 1
            for kind in (0, 1):
                bar, _ = self.full(n, kind)
                bar.arrive(landing=1)
                self.flying.append((bar, (2 * n + kind) % self.stages, (n, kind)))

    def need(self, n, kind):
        slot = (2 * n + kind) % self.stages
        if self.holds[slot] != (n, kind):
            raise Broken(f"{'KV'[kind]}({n}) is read where the slot has {self.holds[slot]}")

    def scores(self):  # S(n) = Q K(n)
        for n in range(self.tiles):
            yield self.full(n, 0)
            if n >= 2:
                yield self.s_free[n & 1], (n >> 1) - 1 & 1
            self.need(n, 0)
            self.s_full[n & 1].arrive()
            self.empty[2 * n % self.stages].arrive()

    def softmax(self):
        for n in range(self.tiles):
            yield self.s_full[n & 1], n >> 1 & 1
            if n >= 2:
                yield self.p_free[n & 1], (n >> 1) - 1 & 1
            self.s_free[n & 1].arrive()
            self.p_full[n & 1].arrive()
            self.done.add(n)

    def outputs(self):  # O += P(n) V(n)
        for n in range(self.tiles):
            yield self.full(n, 1)
            yield self.p_full[n & 1], n >> 1 & 1
            self.need(n, 1)
            self.empty[(2 * n + 1) % self.stages].arrive()
            self.p_free[n & 1].arrive()

    def run(self):
        roles = [[r, None] for r in (self.producer(), self.scores(), self.outputs(), *(self.softmax() for _ in range(4)))]
        late = self.rng.choice((0.02, 0.2, 0.7))  # how soon copies land, one by one
        while roles:
            ready = [r for r in roles if r[1] is None or r[1][0].passed(r[1][1])]
            if self.flying and (not ready or self.rng.random() < late):
                bar, slot, what = self.flying.pop(self.rng.randrange(len(self.flying)))
                self.holds[slot] = what
                bar.landed()
                continue
            if not ready:
                raise Broken("nobody can go on")
            r = self.rng.choice(ready)
            try:
                r[1] = next(r[0])
            except StopIteration:
                roles.remove(r)


def _broken(stages, per_tile, seeds):
    out = []
    for seed in range(seeds):
        try:
            Ring(stages, 40, per_tile, random.Random(seed)).run()
        except Broken as e:
            out.append(str(e))
    return out


@pytest.mark.parametrize("stages", [4, 5, 6, 9, 12])
def test_waits_name_what_they_wait_for(stages):
    assert _broken(stages, True, 300) == []


def test_the_model_sees_a_parity_of_the_phase_before():
    """Full barriers of slots: with five of them K and V share a slot by turns, and the issuer of S passes its wait for K
    while the V before it in the slot is on its way.  With six they never do."""
    assert _broken(5, False, 300) != []
    assert _broken(6, False, 300) == []


def test_the_kernel_waits_by_tile():
    with open(SOURCE) as f:
        text = f.read()
    waits = re.findall(r"rolled_wait(?:_warp)?\(smem_u32\(&(bar_[kv]_full)\[([^\]]+)\]\)", text)
    assert len(waits) == 4 and {i for _, i in waits} == {"tile", "n % kStages", "slot"}
    # (the one by slot is of 8-bit caches, whose ring has V alone: the slot of V(n) is n modulo kStages)
    assert text.count("const uint32_t slot = n % kStages;") == 1
    assert "bar_kv_full" not in text
