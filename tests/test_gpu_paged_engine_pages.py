"""The pages of the engine's paged slots when a step is refused or fails: no row is taken, no page is lost, and what the slots give
back can be taken again."""
import os

import dataclasses

import numpy as np
import pytest

import eahmmf_b200 as eb
import synth

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kquant_path(tmp_path_factory):
    import torch
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required")
    return synth.write_gguf(str(tmp_path_factory.mktemp("kp") / "ks.gguf"), synth.config_kquant_small())


def test_a_refused_step_with_a_shared_page_loses_nothing(kquant_path):
    e = eb.Engine(kquant_path, 100)
    try:
        assert e.set_paged(4, 4, 16, "f16") == 0
        rc, a = e.prefill_slot(0, np.arange(20))
        assert rc == 0 and e.fork_slot(0, 1, 20) == 0
        rc, c = e.prefill_slot(2, np.arange(16))
        assert rc == 0 and e.free_pages() == 1
        for _ in range(2):  # slot 1 would copy the shared page, slot 2 needs another one: there is one
            assert e.step_slots([1, 2], [20, 16], [a, c])[0] == eb.ST_CAPACITY
            assert e.step_slots([2, 1], [16, 20], [c, a])[0] == eb.ST_CAPACITY
            assert [e.slot_len(s) for s in range(3)] == [20, 20, 16] and e.free_pages() == 1
        # the page is there for whoever steps alone
        assert e.step_slots([2], [16], [c])[0] == 0 and e.free_pages() == 0
        assert e.step_slots([0], [20], [a])[0] == eb.ST_CAPACITY
        assert e.free_slot(2) == 0 and e.free_pages() == 2
        # both holders of the shared page in one step: the first takes a copy, the second keeps it
        rc, two = e.step_slots([0, 1], [20, 20], [a, a])
        assert rc == 0 and e.free_pages() == 1 and two[0] == two[1]
        for s in range(4):
            assert e.free_slot(s) == 0
        assert e.free_pages() == 4
        rc, again = e.prefill_slot(3, np.arange(20))
        assert rc == 0 and again == a
    finally:
        e.close()


def test_slots_emptied_after_a_refused_step_give_every_page_back(kquant_path):
    e = eb.Engine(kquant_path, 100)
    try:
        assert e.set_paged(3, 4, 16, "f16") == 0
        rc, a = e.prefill_slot(0, np.arange(20))
        assert rc == 0 and e.fork_slot(0, 1, 20) == 0
        rc, c = e.prefill_slot(2, np.arange(16))
        assert e.step_slots([1, 2], [20, 16], [a, c])[0] == eb.ST_CAPACITY
        for s in range(3):
            assert e.free_slot(s) == 0
        assert e.free_pages() == 4
        rc, b = e.prefill_slot(0, np.arange(60))
        assert rc == 0 and e.free_pages() == 0
    finally:
        e.close()


BAD_TOKEN = 777


@pytest.fixture(scope="module")
def nan_path(tmp_path_factory):
    """The same model with NaN in one token's embedding: its routing is no expert's, which raises EAHMMF_ST_BAD_INDEX."""
    cfg = synth.config_kquant_small()
    path = synth.write_gguf(str(tmp_path_factory.mktemp("kn") / "kn.gguf"), cfg)
    header, specs, offsets, _ = synth._layout(cfg)
    assert specs[0].name == "token_embd.weight" and cfg.embd_type == synth.Q4_K
    row = synth.row_bytes(cfg.embd_type, cfg.D)
    with open(path, "r+b") as f:
        for block in range(cfg.D // 256):
            f.seek(len(header) + offsets[0] + BAD_TOKEN * row + 144 * block)
            f.write(np.float16("nan").tobytes())  # the scale of a block
    return path


@pytest.mark.parametrize("n_batch", [2, 64])
def test_a_failed_call_takes_no_position(nan_path, n_batch):
    e = eb.Engine(nan_path, 100)
    try:
        assert e.set_paged(4, 12, 16, "f16") == 0
        rc, a = e.prefill_slot(0, np.arange(20))
        assert rc == 0 and e.fork_slot(0, 1, 20) == 0
        rc, b = e.prefill_slot(2, np.arange(7))
        assert rc == 0 and e.free_pages() == 9
        assert e.extend_slot(0, [5, 6, BAD_TOKEN, 7], n_batch)[0] == eb.ST_BAD_INDEX
        assert e.slot_len(0) == 20
        assert e.step_slots([2, 1], [7, 20], [b, BAD_TOKEN])[0] == eb.ST_BAD_INDEX
        assert [e.slot_len(s) for s in range(3)] == [20, 20, 7]
        assert e.prefill_slot(3, [1, BAD_TOKEN], n_batch)[0] == eb.ST_BAD_INDEX and e.slot_len(3) == 0
        # each goes on as if nothing had been: the NaN lie behind its positions
        rc, nxt = e.step_slots([0, 1, 2], [20, 20, 7], [a, a, b])
        assert rc == 0 and nxt[0] == nxt[1]
        rc, same = e.prefill_slot(3, np.arange(7))
        assert rc == 0 and same == b
        rc, step = e.step_slots([3], [7], [b])
        assert rc == 0 and step[0] == nxt[2]
        for s in range(4):
            assert e.free_slot(s) == 0
        assert e.free_pages() == 12
    finally:
        e.close()


def test_a_paged_cache_without_room_leaves_the_slots(tmp_path_factory):
    """Memory for the pages, but not for the one contiguous slot that takes the place of two: nothing changes."""
    import torch
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required")
    cfg = dataclasses.replace(synth.config_kquant_small(), ctx_train=1 << 16)
    path = synth.write_gguf(str(tmp_path_factory.mktemp("kc") / "kc.gguf"), cfg)
    e = eb.Engine(path, 1 << 16)  # a slot: 100 MB of k and as much of v
    hog = None
    try:
        assert e.set_slots(2) == 0
        nxt = [e.prefill_slot(s, np.arange(10 + s)) for s in range(2)]
        assert [rc for rc, _ in nxt] == [0, 0]
        rc, want = e.step_slots([0, 1], [10, 11], [t for _, t in nxt])
        assert rc == 0
        torch.cuda.empty_cache()
        hog = torch.empty(torch.cuda.mem_get_info()[0] - (150 << 20), dtype=torch.uint8, device="cuda")
        assert e.set_paged(2, 64, 16, "f16") == eb.ST_CAPACITY
        hog = None
        torch.cuda.empty_cache()
        assert e.free_pages() == -1 and e.slot_len(0) == -1
        rc, again = e.step_slots([0, 1], [10, 11], [t for _, t in nxt])
        assert rc == 0 and list(again) == list(want)
        assert e.set_paged(2, 64, 16, "f16") == 0 and e.free_pages() == 64
    finally:
        hog = None
        torch.cuda.empty_cache()
        e.close()
