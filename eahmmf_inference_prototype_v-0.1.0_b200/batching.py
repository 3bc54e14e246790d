"""A minimal continuous-batching scheduler over the engine's sequence slots (eahmmf_engine_set_slots /
prefill_slot / step_slots).

The reference serves one sequence at a time (its Engine holds one KV cache, qwen3moe.cpp:791, :910-913,
and its generate loop feeds one token per forward call, :1294-1310). Here requests queue up; whenever a
slot is free the next request's prompt is prefilled into it, and every step runs one token of every
active sequence as a single forward pass. A sequence leaves when it has its tokens, and its slot takes
the next request at once. Greedy selection; per-sequence tokens equal that sequence decoded alone.

With `pages` the slots share a paged cache (eahmmf_engine_set_paged): a request is admitted when the pages
for its prompt and all of its tokens are free beside those that the running ones will still take, and its
pages go back when it leaves. Keys and values are then held in 16 bits unless dtype is "f32" (contiguous slots
hold 32), and attention sums over a batch's pages in an order that depends on the batch: tokens equal those of
the sequence alone in the same kind of cache up to the rounding of a logit.
"""
from __future__ import annotations

import dataclasses
from collections import deque


@dataclasses.dataclass
class Request:
    prompt: list
    n_gen: int
    tokens: list = dataclasses.field(default_factory=list)  # generated so far (the first from the prompt)
    slot: int = -1
    pos: int = 0  # position of the next input token


class ContinuousBatcher:
    """Run requests through an engine with `n_slots` sequence slots, at most `max_rows` (<= 64) per step."""

    def __init__(self, engine, n_slots: int, max_rows: int = 64, n_batch: int = 64, pages: int = 0, page: int = 64,
                 dtype: str = "f16"):
        if pages:
            if engine.set_paged(n_slots, pages, page, dtype):
                raise RuntimeError("eahmmf_engine_set_paged failed")
        elif engine.set_slots(n_slots):
            raise RuntimeError("eahmmf_engine_set_slots failed")
        self.pages, self.page = pages, page
        self.e, self.n_slots, self.max_rows, self.n_batch = engine, n_slots, min(max_rows, 64), n_batch
        self.queue: deque = deque()
        self.active: dict = {}  # slot -> Request
        self.steps = 0
        self.rows = 0  # sequence-tokens decoded by steps (throughput accounting)

    def _need(self, r: Request) -> int:
        """Pages of a request's positions: its prompt, which is always prefilled, and every token but the last, which is
        not fed."""
        return -(-(len(r.prompt) + max(r.n_gen, 1) - 1) // self.page)

    def submit(self, prompt, n_gen: int) -> Request:
        r = Request(list(map(int, prompt)), int(n_gen))
        if self.pages and self._need(r) > self.pages:
            raise ValueError(f"the request needs {self._need(r)} pages, the cache has {self.pages}")
        self.queue.append(r)
        return r

    def _admit(self):
        free = [s for s in range(self.n_slots) if s not in self.active]
        while free and self.queue and len(self.active) < self.max_rows:
            if self.pages and sum(map(self._need, self.active.values())) + self._need(self.queue[0]) > self.pages:
                break
            r = self.queue[0]
            rc, first = self.e.prefill_slot(free[0], r.prompt, self.n_batch)
            if rc:  # the request stays at the head of the queue
                raise RuntimeError(f"eahmmf_engine_prefill_slot returned {rc}")
            self.queue.popleft()
            r.slot = free.pop(0)
            r.tokens.append(first)
            r.pos = len(r.prompt)
            if len(r.tokens) < r.n_gen:
                self.active[r.slot] = r
            elif self.pages:
                self.e.free_slot(r.slot)

    def step(self) -> bool:
        """Admit what fits, then one token of every active sequence. False when nothing is left."""
        self._admit()
        if not self.active:
            return False
        rs = list(self.active.values())
        rc, nxt = self.e.step_slots([r.slot for r in rs], [r.pos for r in rs], [r.tokens[-1] for r in rs])
        if rc:
            raise RuntimeError(f"eahmmf_engine_step_slots returned {rc}")
        self.steps += 1
        self.rows += len(rs)
        for r, t in zip(rs, nxt):
            r.tokens.append(int(t))
            r.pos += 1
            if len(r.tokens) >= r.n_gen:
                del self.active[r.slot]
                if self.pages:
                    self.e.free_slot(r.slot)
        return True

    def run(self):
        while self.step():
            pass
