"""The engine's slots over a paged cache (eahmmf_engine_set_paged): against every sequence decoded alone by the single-sequence
engine path, with requests that come and go, sequences that share a prompt and part, and a cache that runs out of pages.

With 32-bit pages the attention differs from the contiguous path's in the order of its sums alone (about 1e-6 of a logit), far
inside the gaps between the largest logits of these models, so greedy tokens are equal; with 16-bit pages a sequence is compared
with the same sequence in the same kind of cache."""
import os

import numpy as np
import pytest

import batching
import eahmmf_b200 as eb
import synth

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TINY = os.path.join(ROOT, "tests", "golden", "ref_tiny.gguf")


@pytest.fixture(scope="module")
def kquant_path(tmp_path_factory):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required")
    return synth.write_gguf(str(tmp_path_factory.mktemp("kp") / "ks.gguf"), synth.config_kquant_small())


def generate(e, slot, first, n):
    toks = [first]
    while len(toks) < n:
        rc, nxt = e.step_slots([slot], [e.slot_len(slot)], [toks[-1]])
        assert rc == 0
        toks.append(int(nxt[0]))
    return toks


@pytest.mark.parametrize("model,page", [("kquant", 16), ("kquant", 48), ("tiny", 16)])
def test_paged_requests_match_single_sequence_decode(kquant_path, model, page):
    path = kquant_path if model == "kquant" else TINY
    rng = np.random.default_rng(3)
    vocab = 1000 if model == "kquant" else 250
    reqs = [(rng.integers(0, vocab, int(rng.integers(1, 80))).astype(np.int32), int(rng.integers(2, 18))) for _ in range(10)]
    e = eb.Engine(path, 128)
    try:
        want = []
        for prompt, n in reqs:
            rc, out, _ = e.greedy(prompt, n, 64)
            assert rc == 0
            want.append(out)
        b = batching.ContinuousBatcher(e, n_slots=5, pages=320 // page, page=page, dtype="f32")
        rs = [b.submit(p, n) for p, n in reqs]
        b.run()
        for r, w in zip(rs, want):
            np.testing.assert_array_equal(r.tokens, w)
        assert e.free_pages() == 320 // page
        # the single-sequence calls keep their own cache
        rc, out, _ = e.greedy(reqs[0][0], reqs[0][1], 64)
        assert rc == 0
        np.testing.assert_array_equal(out, want[0])
    finally:
        e.close()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_forked_sequences_share_and_part(kquant_path, dtype):
    rng = np.random.default_rng(5)
    start = rng.integers(0, 1000, 41).astype(np.int32)
    tails = [rng.integers(0, 1000, n).astype(np.int32) for n in (1, 9, 30)]
    e = eb.Engine(kquant_path, 256)
    try:
        assert e.set_paged(6, 40, 16, dtype) == 0
        want = []
        for t in tails:
            rc, first = e.prefill_slot(0, np.concatenate([start, t]), 7)
            assert rc == 0
            want.append(generate(e, 0, first, 12))
        assert e.free_slot(0) == 0 and e.free_pages() == 40
        rc, _ = e.prefill_slot(5, start, 64)
        assert rc == 0 and e.free_pages() == 37
        got, firsts = {}, []
        for i, t in enumerate(tails):
            assert e.fork_slot(5, i, 41) == 0
            assert e.free_pages() == 37 - sum(-(-(41 + len(x)) // 16) - 2 for x in tails[:i])
            rc, first = e.extend_slot(i, t, 64)
            assert rc == 0
            firsts.append(first)
            got[i] = [first]
        for _ in range(11):  # the forks together, one token of each
            rc, nxt = e.step_slots([0, 1, 2], [e.slot_len(i) for i in range(3)], [got[i][-1] for i in range(3)])
            assert rc == 0
            for i in range(3):
                got[i].append(int(nxt[i]))
        assert [got[i] for i in range(3)] == want
        # a fork of a part of the start, whose cut lies inside a shared page
        assert e.free_slot(0) == 0 and e.fork_slot(5, 0, 20) == 0
        rc, first = e.extend_slot(0, np.concatenate([start[20:], tails[1]]), 64)
        assert rc == 0 and generate(e, 0, first, 12) == want[1]
        for s in range(6):
            assert e.free_slot(s) == 0
        assert e.free_pages() == 40
    finally:
        e.close()


def test_paged_calls_refuse_and_keep_the_slot(kquant_path):
    e = eb.Engine(kquant_path, 100)
    try:
        assert e.fork_slot(0, 1, 0) == eb.ST_BAD_ARG and e.free_slot(0) == eb.ST_BAD_ARG and e.free_pages() == -1
        assert e.extend_slot(0, [1])[0] == eb.ST_BAD_ARG
        for bad in ((0, 4, 16), (2, 0, 16), (2, 4, 8), (2, 4, 24), (2, 4, 2048)):
            assert e.set_paged(*bad, "f16") == eb.ST_BAD_ARG
        assert e.set_paged(3, 3, 16, "f16") == 0
        assert e.set_paged(4, 1 << 30, 1024, "f32") == eb.ST_CAPACITY  # more memory than there is: the cache stays
        rc, a = e.prefill_slot(0, np.arange(31))
        assert rc == 0 and e.slot_len(0) == 31 and e.free_pages() == 1
        rc, b = e.prefill_slot(1, np.arange(16))
        assert rc == 0 and e.free_pages() == 0
        assert e.prefill_slot(2, [1])[0] == eb.ST_CAPACITY and e.slot_len(2) == 0
        # row 0 fits its page, row 1 needs one that is not there: neither is taken
        assert e.step_slots([0, 1], [31, 16], [a, b])[0] == eb.ST_CAPACITY
        assert e.slot_len(0) == 31 and e.slot_len(1) == 16
        assert e.step_slots([0], [30], [a])[0] == eb.ST_BAD_ARG  # not its next position
        assert e.step_slots([0], [31], [a])[0] == 0
        assert e.extend_slot(1, [1, 2, 3])[0] == eb.ST_CAPACITY and e.slot_len(1) == 16
        assert e.fork_slot(0, 1, 5) == eb.ST_BAD_ARG  # not empty
        assert e.fork_slot(0, 2, 33) == eb.ST_BAD_ARG and e.fork_slot(0, 2, 32) == 0
        assert e.extend_slot(2, [5000])[0] == eb.ST_BAD_ARG  # no such token
        assert e.set_slots(2) == 0 and e.free_pages() == -1
        rc, c = e.prefill_slot(1, np.arange(31))
        assert rc == 0
    finally:
        e.close()
