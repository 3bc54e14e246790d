"""The barriers of the chunk attention kernel (paged_tc.cu), modelled on the CPU: the warps that bring k and v, issue the two
products and do the softmax, run in random order against mbarriers that a waiter sees by parity alone. Every schedule has to end,
with each product on the tiles, score buffers and output that belong to it: a phase that completes twice between two looks of
its waiter, or a buffer that is written before it is read, shows as a schedule that stops or as a wrong owner."""
import random

import pytest


class Barrier:
    """An mbarrier: `count` arrivals complete a phase; a wait names the parity of the phase it wants to be complete."""

    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def done(self, parity):
        return (self.phase & 1) != parity  # the phase in progress has the other parity


class Model:
    def __init__(self, items, nk, nv, apart, rng):
        self.items, self.nk, self.nv, self.apart, self.rng = items, nk, nv, apart, rng
        b = lambda n, c=1: [Barrier(c) for _ in range(n)]  # noqa: E731
        self.kv_full, self.kv_empty = b(nk + nv), b(nk + nv)
        self.q_full, self.p_full, self.pv_done = b(2), b(2), b(2, 2)
        self.s_full, self.s_free, self.o_free = [b(2, 2), b(2, 2)], b(3), Barrier(1)
        self.slot = [None] * (nk + nv)  # what a k or v slot holds
        self.score = [None] * 3         # what a score buffer holds: ("s" or "p", item, unit, tile)
        self.out = None                 # the output buffer
        self.q = [None, None]
        self.queue = []                 # products in flight
        self.loads = []                 # loads in flight, which land in any order
        self.summed = []

    # each warp is a generator that yields a condition to wait for, or None to let others run
    def loader(self, kinds):
        """The warp that fills the slots of k, that of v, or (32-bit pools) the warps that fill both in turn."""
        n = {"k": 0, "v": 0}
        for it, (n_m, n_it) in enumerate(self.items):
            for i in range(n_it):
                for kind in kinds:
                    slots = self.nv if kind == "v" else self.nk
                    s, use = n[kind] % slots + (self.nk if kind == "v" else 0), n[kind] // slots
                    if use:
                        yield lambda: self.kv_empty[s].done((use - 1) & 1)
                    assert self.slot[s] is None
                    self.slot[s] = "on its way"
                    self.loads.append((s, (kind, it, i)))
                    n[kind] += 1
                    yield None

    def scores(self):
        n = buf = 0
        n_q, n_s = [0, 0], [0, 0]
        for it, (n_m, n_it) in enumerate(self.items):
            for m in range(n_m):
                yield lambda: self.q_full[m].done(n_q[m] & 1)
                n_q[m] += 1
            for i in range(n_it):
                for m in range(n_m):
                    b, use = buf % 3, buf // 3
                    if use:
                        yield lambda: self.s_free[b].done((use - 1) & 1)
                    if n_m == 1 and buf >= 2:
                        yield lambda: self.s_free[(buf - 2) % 3].done(((buf - 2) // 3) & 1)
                    buf += 1
                    full = self.s_full[m][n_s[m] & 1]
                    n_s[m] += 1
                    s = n % self.nk
                    if m == 0:
                        yield lambda: self.kv_full[s].done((n // self.nk) & 1)
                    self.queue.append(("s", s, b, m, it, i, m == n_m - 1, full))
                    full.arrive()
                    yield None
                n += 1

    def values(self):
        n = buf = 0
        n_p = [0, 0]
        for it, (n_m, n_it) in enumerate(self.items):
            for i in range(n_it):
                s = self.nk + n % self.nv
                yield lambda: self.kv_full[s].done((n // self.nv) & 1)
                for m in range(n_m):
                    if buf:
                        yield lambda: self.o_free.done((buf - 1) & 1)
                    yield lambda: self.p_full[m].done(n_p[m] & 1)
                    n_p[m] += 1
                    self.queue.append(("o", s, buf % 3, m, it, i, m == n_m - 1, None))
                    buf += 1
                    self.pv_done[m].arrive()
                    yield None
                n += 1

    def softmax(self, m):
        buf = n_pv = n_s = 0
        for it, (n_m, n_it) in enumerate(self.items):
            if m >= n_m:
                buf += n_it
                continue
            self.q[m] = it
            self.q_full[m].arrive()
            buf += m
            for i in range(n_it + 1):
                if i:
                    yield lambda: self.pv_done[m].done(n_pv & 1)
                    n_pv += 1
                    assert self.out == (it, i - 1, m)
                    self.summed.append(self.out)
                    yield None
                    self.out = None
                    self.o_free.arrive()
                if i == n_it:
                    break
                yield lambda: self.s_full[m][n_s & 1].done((n_s >> 1) & 1)
                n_s += 1
                b = buf % 3
                assert self.score[b] == ("s", it, i, m)
                yield None
                self.score[b] = ("p", it, i, m)
                self.p_full[m].arrive()
                buf += n_m
            buf -= m

    def finish_load(self):
        s, what = self.loads.pop(self.rng.randrange(len(self.loads)))
        self.slot[s] = what
        self.kv_full[s].arrive()

    def finish_product(self):
        # products of one warp end in its order; those of the two warps in any
        kinds = sorted({x[0] for x in self.queue})
        kind = self.rng.choice(kinds)
        at = next(k for k, x in enumerate(self.queue) if x[0] == kind)
        kind, s, b, m, it, i, last, full = self.queue.pop(at)
        if kind == "s":
            assert self.slot[s] == ("k", it, i) and self.q[m] == it and self.score[b] is None
            self.score[b] = ("s", it, i, m)
            full.arrive()
        else:
            assert self.slot[s] == ("v", it, i) and self.score[b] == ("p", it, i, m) and self.out is None
            self.out, self.score[b] = (it, i, m), None
            self.pv_done[m].arrive()
            self.s_free[b].arrive()
        if last:
            self.slot[s] = None
            self.kv_empty[s].arrive()

    def run(self, lazy):
        """lazy: the actor that is chosen least often."""
        actors = {"qk": self.scores(), "pv": self.values(), "s0": self.softmax(0), "s1": self.softmax(1)}
        if self.apart:
            actors["k"], actors["v"] = self.loader("k"), self.loader("v")
        else:
            actors["k"] = self.loader("kv")
        waiting = {a: None for a in actors}
        while actors or self.loads or self.queue:
            ready = [a for a in actors if waiting[a] is None or waiting[a]()]
            ready += ["land"] * bool(self.loads) + ["product"] * bool(self.queue)
            assert ready, "no warp can go on: %s" % sorted(actors)
            some = [a for a in ready if a != lazy]
            a = self.rng.choice(some if some and self.rng.random() < 0.98 else ready)
            if a == "land":
                self.finish_load()
            elif a == "product":
                self.finish_product()
            else:
                try:
                    waiting[a] = next(actors[a])
                except StopIteration:
                    del actors[a]
        want = [(it, i, m) for it, (n_m, n_it) in enumerate(self.items) for i in range(n_it) for m in range(n_m)]
        assert self.summed == want


@pytest.mark.parametrize("nk,nv,two", [(2, 1, True), (4, 4, True), (1, 1, False)])  # 16-bit heads of 128 and 64, 32-bit
@pytest.mark.parametrize("lazy", [None, "k", "v", "qk", "pv", "s0", "s1", "land", "product"])
def test_every_schedule_ends(nk, nv, two, lazy):
    rng = random.Random(7)
    for _ in range(60):
        items = [(rng.choice([1, 2]) if two else 1, rng.randint(1, 7)) for _ in range(rng.randint(1, 6))]
        Model(items, nk, nv, two, rng).run(lazy)
