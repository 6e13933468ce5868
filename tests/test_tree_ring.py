"""The barriers of tree_attention's tcgen05 kernel, walked on the CPU.

A model of its twelve warps: two producers, two MMA warps, eight softmax warps, the ring of key and
value tiles, and mbarriers as the hardware has them: a wait names a phase's parity, so one that is two
phases late or early would pass.  Delays are random.  Checked: no wait passes before its phase is
over or finds it gone, no tile is overwritten before its products, everything ends.
"""
from __future__ import annotations

import heapq
import random

import pytest


class Bar:
    def __init__(self, count, name):
        self.count = self.left = count
        self.tx = self.phase = 0
        self.name = name

    def _look(self):
        if self.left == 0 and self.tx == 0:
            self.phase += 1
            self.left = self.count

    def arrive(self):
        assert self.left > 0, f"{self.name}: more arrivals than counted"
        self.left -= 1
        self._look()

    def expect(self):
        self.tx += 1
        self.arrive()

    def land(self):
        self.tx -= 1
        self._look()

    def passes(self, parity):
        return (self.phase & 1) != parity


class Clock:
    def __init__(self, seed, live):
        self.events, self.now, self.n, self.live = [], 0.0, 0, live
        self.rng = random.Random(seed)

    def after(self, dt, f):
        self.n += 1
        heapq.heappush(self.events, (self.now + dt, self.n, f))

    def step(self, warp):
        try:
            want = next(warp)
        except StopIteration:
            self.live -= 1
            return
        if isinstance(want, tuple):
            self.poll(warp, *want, 0)
        else:
            self.after(want, lambda: self.step(warp))

    def poll(self, warp, bar, phase, tries):
        if bar.passes(phase & 1):
            assert bar.phase == phase + 1, f"{bar.name}: wait for phase {phase} passed in {bar.phase}"
            self.after(1, lambda: self.step(warp))
        else:
            assert bar.phase <= phase, f"{bar.name}: phase {phase} missed, now {bar.phase}"
            assert tries < 20000, f"{bar.name}: phase {phase} never ends"
            self.after(50, lambda: self.poll(warp, bar, phase, tries + 1))

    def run(self):
        while self.events:
            self.now, _, f = heapq.heappop(self.events)
            f()
        assert self.live == 0, f"{self.live} warps never end"


def lead(two):
    return 1 if two else 2


def place(is_v, i, n, two):
    """Where the i-th of n key or value tiles of a piece stands in the ring, from the piece's first."""
    k = lead(two)
    if is_v:
        return 2 * i + k + 1 if i + k < n else n + i
    return i if i < k else 2 * i - k


def walk(seed, pieces, stages, skip=False):
    """``pieces``: (two tiles of rows, steps, last values end inside a tile).  ``skip``: MMA warps wait
    for their own tiles alone."""
    readers, items_ahead = 11, 4
    clock = Clock(seed, 12)
    r = clock.rng
    rnd = r.uniform

    def bars(n, count, name):
        return [Bar(count, f"{name}{i}") for i in range(n)]

    full, empty = bars(stages, 1, "full"), bars(stages, 2, "empty")
    q_full, q_empty = bars(2, 1, "q_full"), bars(2, 2, "q_empty")
    s_full, p_ready, pv_done = ([bars(2, c, f"{n}{t}.") for t in (0, 1)]
                                for c, n in ((1, "s_full"), (4, "p_ready"), (1, "pv_done")))
    it_full, it_empty = bars(items_ahead, 1, "it_full"), bars(items_ahead, readers, "it_empty")
    done, read, tail = bars(8, 1, "done"), bars(8, 1, "read"), Bar(1, "tail")
    items, held, pipe = {}, [None] * stages, [0.0]
    slow = [rnd(1, 4) for _ in range(8)]

    def product(time, commits):
        end = max(clock.now, pipe[0]) + time
        pipe[0] = end
        for b in commits:
            clock.after(end - clock.now + rnd(5, 60), b.arrive)

    def fetch(n):
        yield it_full[n % items_ahead], n // items_ahead
        it_empty[n % items_ahead].arrive()
        return items[n]

    def producer(is_v):
        base, n, n_tail, ones, uses = 0, 0, 0, 0, [0, 0]

        def publish(n):
            nonlocal ones
            if n >= items_ahead:
                yield it_empty[n % items_ahead], n // items_ahead - 1
            if n < len(pieces):
                two, steps, tails = pieces[n]
                items[n] = (two, steps, ones & 1, tails)
                ones += not two
            else:
                items[n] = (0, 0, 0, 0)
            it_full[n % items_ahead].arrive()

        def prepare(n):
            if is_v:
                return (yield from fetch(n))
            yield from publish(n)
            return items[n]

        after = yield from prepare(0)
        while after[1]:
            two, steps, slot, tails = after
            n += 1
            yield rnd(100, 1500)
            for t in () if is_v else (0, 1) if two else (slot,):
                if uses[t]:
                    yield q_empty[t], uses[t] - 1
                uses[t] += 1
                q_full[t].expect()
                clock.after(rnd(500, 4000), q_full[t].land)
            for i in range(steps):
                x = base + place(is_v, i, steps, two)
                s = x % stages
                if x >= stages:
                    yield empty[s], x // stages - 1
                held[s] = x
                tailed = is_v and tails and i + 1 == steps
                bar = tail if tailed else full[s]
                bar.expect()
                clock.after(rnd(500, 12000 if r.random() < .05 else 2500), bar.land)
                yield rnd(20, 500)
                if i == (min(2, steps - 1) if is_v else 0):
                    after = yield from prepare(n)
                if tailed:
                    yield tail, n_tail
                    n_tail += 1
                    yield rnd(50, 300)
                    full[s].arrive()
            base += 2 * steps

    def issuer(t):
        base, n, n_qk, n_pv, uses = 0, 0, 0, 0, [0, 0]
        while True:
            two, steps, slot, _ = yield from fetch(n)
            n += 1
            if steps == 0:
                return
            q = t if two else slot
            use = uses[q]
            for u in (0, 1) if two else (slot,):
                uses[u] += 1
            left = steps if two else (steps + 1 - t) >> 1
            yield q_full[q], use
            if left == 0:
                q_empty[q].arrive()
            j_k = j_v = 0
            for i in range(2 * steps):
                is_k = j_k < steps and (i <= lead(two) or (i - lead(two)) % 2 == 0)
                j = j_k if is_k else j_v
                j_k, j_v = j_k + is_k, j_v + (not is_k)
                assert i == place(not is_k, j, steps, two)
                x = base + i
                s = x % stages
                mine = two or j & 1 == t
                if mine or not skip:
                    yield full[s], x // stages
                if not mine:
                    if not skip:
                        empty[s].arrive()
                    continue
                free = [empty[s]] * (2 if skip and not two else 1)
                if is_k:
                    if n_qk >= 2:
                        yield pv_done[t][n_qk & 1], (n_qk - 2) >> 1
                    left -= 1
                    yield rnd(50, 300)
                    assert held[s] == x
                    last = [q_empty[q]] * (2 if two else 1) if left == 0 else []
                    product(512, [s_full[t][n_qk & 1], *last, *free])
                    n_qk += 1
                else:
                    yield p_ready[t][n_pv & 1], n_pv >> 1
                    yield rnd(50, 300)
                    assert held[s] == x
                    product(256, [pv_done[t][n_pv & 1], *free])
                    n_pv += 1
            base += 2 * steps

    def softmax(w):
        t, n, n_s, n_pair = w >> 2, 0, 0, 0
        while True:
            two, steps, _, _ = yield from fetch(n)
            n += 1
            if steps == 0:
                return
            mine = steps if two else (steps + 1 - t) >> 1
            for i in range(mine):
                yield s_full[t][n_s & 1], n_s >> 1
                yield rnd(300, 1500) * slow[w]
                if i > 0 and r.random() < .2:  # the result is rescaled
                    yield pv_done[t][(n_s - 1) & 1], (n_s - 1) >> 1
                p_ready[t][n_s & 1].arrive()
                n_s += 1
            if mine > 1:
                yield pv_done[t][n_s & 1], (n_s - 2) >> 1
            if mine > 0:
                yield pv_done[t][(n_s - 1) & 1], (n_s - 1) >> 1
            if not two:
                done[w].arrive()
                yield done[w ^ 4], n_pair
            yield rnd(500, 4000)
            if not two:
                read[w].arrive()
                yield read[w ^ 4], n_pair
                n_pair += 1

    for warp in [producer(False), producer(True), issuer(0), issuer(1)] + [softmax(w) for w in range(8)]:
        clock.after(0, lambda warp=warp: clock.step(warp))
    clock.run()


def _pieces(seed):
    r = random.Random(seed)
    share = r.choice([0, 0, .3, 1])
    return [(r.random() < share, r.choice([1, 1, 2, 3, 4, 5, r.randint(1, 30)]), r.random() < .7)
            for _ in range(r.randint(1, 7))]


@pytest.mark.parametrize("stages", [8, 16])
def test_every_wait_is_for_its_phase(stages):
    for seed in range(60):
        walk(seed, _pieces(seed), stages)


def test_places_fill_the_ring_once():
    for two in (False, True):
        for n in range(1, 12):
            at = [place(v, i, n, two) for v in (False, True) for i in range(n)]
            assert sorted(at) == list(range(2 * n))


def test_a_warp_that_skips_tiles_is_caught():
    """The model sees the mistake it is there for."""
    caught = 0
    for seed in range(60):
        try:
            walk(seed, [(False, 33, True)] * 4, 8, skip=True)
        except AssertionError:
            caught += 1
    assert caught > 0
