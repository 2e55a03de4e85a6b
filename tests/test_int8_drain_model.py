"""The bookkeeping by which the int8 kernels wait for copies in flight after a wait ran
out (drain_copies in qx_int8_tc.cuh), on a model of the barriers: whatever each copy
thread had issued, the drain's waits end once exactly those copies have landed, and not
before. The former rule (wait for phase 0 of every stage, in the weight thread, if that
thread's own wait ran out) does not hold up: the last test shows where."""

import random

import pytest


class Barrier:
    """An mbarrier with one expected arrival: a phase ends when it has come and the
    announced bytes are all in."""

    def __init__(self):
        self.phase, self.arrived, self.tx = 0, False, 0

    def _step(self):
        if self.arrived and self.tx == 0:
            self.phase, self.arrived = self.phase + 1, False

    def arrive_expect(self, n):
        assert not self.arrived
        self.arrived, self.tx = True, self.tx + n
        self._step()

    def complete(self, n):
        self.tx -= n
        self._step()

    def done(self, parity):
        return (self.phase - 1) % 2 == parity if self.phase else parity == 1


class Ring:
    def __init__(self, ns, sizes):
        self.ns, self.sizes, self.full = ns, sizes, [Barrier() for _ in range(ns)]
        self.flight, self.issued = [], [0] * len(sizes)

    def issue(self, i):
        f = self.issued[i]
        if i == 0:
            self.full[f % self.ns].arrive_expect(sum(self.sizes))
        self.flight.append((f, i))
        self.issued[i] += 1

    def land(self, j):
        f, i = self.flight.pop(j)
        self.full[f % self.ns].complete(self.sizes[i])

    def drain(self):
        """The barriers and parities that the drain waits for, after its bookkeeping."""
        last, waits = max(self.issued), []
        for f in range(max(0, last - self.ns), last):
            bar = self.full[f % self.ns]
            come = sum(n for n, k in zip(self.sizes, self.issued) if f < k)
            missing = sum(self.sizes) - come
            if f >= self.issued[0]:
                bar.arrive_expect(come)
            elif missing:
                bar.complete(missing)
            waits.append((bar, f // self.ns % 2))
        return waits


def give_up(rng, ns, sizes, fills):
    """A run of the ring that stops at a random point: the consumer has taken `taken` fills,
    every copy thread is up to one round ahead of it."""
    ring, taken, stop = Ring(ns, sizes), 0, rng.randint(0, fills)
    while taken < stop:
        for i in range(len(sizes)):
            while ring.issued[i] < min(taken + ns, fills) and rng.random() < 0.7:
                ring.issue(i)
        while ring.flight and rng.random() < 0.8:
            ring.land(rng.randrange(len(ring.flight)))
        if ring.full[taken % ns].done(taken // ns % 2):
            taken += 1
    for i in range(len(sizes)):
        while ring.issued[i] < min(taken + ns, fills) and rng.random() < 0.6:
            ring.issue(i)
    return ring


@pytest.mark.parametrize("sizes", [(128, 16), (96, 64, 96, 64)])
def test_drain_waits_for_every_copy(sizes):
    rng = random.Random(5)
    for _ in range(3000):
        ns = rng.randint(1, 12)
        ring = give_up(rng, ns, sizes, rng.randint(1, 4 * ns))
        waits = ring.drain()
        assert len({id(b) for b, _ in waits}) == len(waits)
        while ring.flight:
            assert not all(b.done(p) for b, p in waits)
            ring.land(rng.randrange(len(ring.flight)))
        assert all(b.done(p) for b, p in waits)


def test_waiting_for_phase_zero_is_not_enough():
    ring = Ring(2, (128, 16))
    for _ in range(2):
        for i in (0, 1):
            ring.issue(i)
    while ring.flight:
        ring.land(0)
    for i in (0, 1):
        ring.issue(i)                                   # the second round's first fill, under way
    assert ring.full[0].done(0) and ring.flight
    assert not all(b.done(p) for b, p in ring.drain())
