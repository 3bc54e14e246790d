"""The bytes of a row tile's q in the chunk attention kernel (paged_tc.cu), modelled on the CPU: its four softmax warps write q, the
product reads it, and each warp's output passes through the same bytes on its way out while the others may already write the next
q. The warps wait for the product alone, never for each other, so every order of theirs has to leave each its own bytes. The
two layouts are taken from the kernel's source."""
import os
import random
import re

import pytest

import eahmmf_b200 as eb

SOURCE = os.path.join(os.path.dirname(eb.__file__), "csrc", "paged_tc.cu")
BLK = 128 * 128  # bytes of a column block


def layout(name):
    """The expression that a function of the kernel returns, as a function of (row, chunk)."""
    m = re.search(r"constexpr int %s\(int row, int (\w+)\) \{[^\n]*\n\s*return ([^;]+);" % name, open(SOURCE).read())
    code = compile(m.group(2), name, "eval")
    return lambda row, c: eval(code, {"row": row, m.group(1): c})


def linear(hd):
    """Every warp's output rows as one run, which is no layout for bytes shared with q."""
    return lambda row, c: row * hd * 4 + c * 16


class Tile:
    def __init__(self, hd, items, stage, rng):
        self.hd, self.items, self.stage, self.rng = hd, items, stage, rng
        self.q = layout("q_at")
        self.bytes = {}          # 16 bytes at an offset: who wrote them last
        self.arrived = 0         # warps that have written the q of the item in progress
        self.done = -1           # last item whose products are done

    def warp(self, w):
        rows = range(32 * w, 32 * w + 32)
        q = [(part * (self.hd // 64) * BLK + self.q(r, ch), r, part, ch) for part in (0, 1) for r in rows for ch in range(self.hd // 8)]
        out = [(self.stage(r, c), r, c) for r in rows for c in range(self.hd // 4)]
        for it in range(self.items):
            for i in range(0, len(q), 64):
                for at, *what in q[i:i + 64]:
                    self.bytes[at] = ("q", it, *what)
                yield None
            self.arrived += 1
            yield lambda: self.done >= it
            for i in range(0, len(out), 64):
                for at, *what in out[i:i + 64]:
                    self.bytes[at] = ("out", it, *what)
                yield None
            for i in range(0, len(out), 64):
                for at, *what in out[i:i + 64]:
                    assert self.bytes[at] == ("out", it, *what)
                yield None

    def product(self):
        for it in range(self.items):
            yield lambda: self.arrived == 4
            for part in (0, 1):
                for r in range(128):
                    for ch in range(self.hd // 8):
                        assert self.bytes[part * (self.hd // 64) * BLK + self.q(r, ch)] == ("q", it, r, part, ch)
            self.arrived, self.done = 0, it
            yield None

    def run(self, lazy):
        actors = {w: self.warp(w) for w in range(4)} | {"product": self.product()}
        waiting = {a: None for a in actors}
        while actors:
            ready = [a for a in actors if waiting[a] is None or waiting[a]()]
            some = [a for a in ready if a != lazy]
            a = self.rng.choice(some if some and self.rng.random() < 0.95 else ready)
            try:
                waiting[a] = next(actors[a])
            except StopIteration:
                del actors[a]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lazy", [None, 0, 1, 2, 3])
def test_no_warp_touches_the_bytes_of_another(hd, lazy):
    rng = random.Random(3)
    for _ in range(3):
        Tile(hd, 3, layout("stage_at"), rng).run(lazy)


@pytest.mark.parametrize("hd", [64, 128])
def test_layouts_fill_the_same_bytes_once(hd):
    for w in range(4):
        rows = range(32 * w, 32 * w + 32)
        q = [part * (hd // 64) * BLK + layout("q_at")(r, ch) for part in (0, 1) for r in rows for ch in range(hd // 8)]
        out = [layout("stage_at")(r, c) for r in rows for c in range(hd // 4)]
        assert len(set(q)) == len(q) and sorted(q) == sorted(out)


@pytest.mark.parametrize("hd", [64, 128])
def test_the_model_sees_warps_in_each_others_bytes(hd):
    rng = random.Random(3)
    with pytest.raises(AssertionError):
        for lazy in (0, 1, 2, 3) * 5:
            Tile(hd, 3, linear(hd), rng).run(lazy)
