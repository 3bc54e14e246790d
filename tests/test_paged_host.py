"""The paged cache on the host: refusals of the C entry points before anything is launched, the frequency tables of rotary
positions against their formulas, and the page bookkeeping against a plain model of it."""
import ctypes as C
import math
import random

import numpy as np
import pytest

import eahmmf_b200 as eb

BAD, TYPE, CAP, IDX = eb.ST_BAD_ARG, eb.ST_BAD_TYPE, eb.ST_CAPACITY, eb.ST_BAD_INDEX
FAKE = 0x10000  # an aligned address that is never read: every call below is refused on the host


def kv(**o):
    d = dict(d_k=FAKE, d_v=FAKE, type=1, n_layer=2, n_pages=8, n_kv=2, page=16, hd=64, layer_stride=8 * 2 * 16 * 64,
             page_stride=2 * 16 * 64)
    d.update(o)
    return eb.EahmmfPagedKv(*[d[f[0]] for f in eb.EahmmfPagedKv._fields_])


def seqs(**o):
    d = dict(n_seq=2, n_tok=5, max_q=4, max_kv=40, d_cu_q=FAKE, d_kv_len=FAKE, d_table=FAKE, table_ld=3)
    d.update(o)
    return eb.EahmmfPagedSeqs(*[d[f[0]] for f in eb.EahmmfPagedSeqs._fields_])


def rope(**o):
    d = dict(style=0, n_rot=64, mscale=1.0, d_inv_freq=FAKE)
    d.update(o)
    return eb.EahmmfRope(*[d[f[0]] for f in eb.EahmmfRope._fields_])


BAD_KV = [(dict(type=8), TYPE), (dict(d_k=None), BAD), (dict(d_v=FAKE + 8), BAD), (dict(n_layer=0), BAD),
          (dict(n_pages=0), BAD), (dict(n_kv=0), BAD), (dict(page=8), BAD), (dict(page=24), BAD), (dict(page=2048), BAD),
          (dict(hd=96), BAD), (dict(page_stride=2 * 16 * 64 - 8), BAD), (dict(page_stride=2 * 16 * 64 + 4), BAD),
          (dict(layer_stride=7 * 2 * 16 * 64), BAD)]
BAD_SEQS = [dict(n_seq=-1), dict(n_tok=-1), dict(max_q=-1), dict(max_kv=-1), dict(d_cu_q=None), dict(d_kv_len=None),
            dict(d_table=None), dict(table_ld=0)]


def attention(k=None, s=None, layer=0, n_head=4, q=FAKE, ldq=256, scale=0.1, window=0, sinks=0, out=FAKE, ldo=256, ws=FAKE,
              ws_bytes=1 << 40):
    k, s = k or kv(), s or seqs()
    return eb.lib().eahmmf_cuda_paged_attention(C.addressof(k), layer, C.addressof(s), n_head, q, ldq, scale, window, sinks,
                                                out, ldo, ws, ws_bytes, None, None)


def append(k=None, s=None, r=None, layer=0, n_head=4, x=FAKE, ld=512, qn=None, kn=None, eps=1e-6, q=FAKE, ldq=256):
    k, s, r = k or kv(), s or seqs(), r or rope()
    return eb.lib().eahmmf_cuda_rope_append(C.addressof(k), layer, C.addressof(s), C.addressof(r), n_head, x, ld, qn, kn,
                                            eps, q, ldq, None, None)


@pytest.mark.parametrize("o,want", BAD_KV)
def test_pools_are_checked(o, want):
    k = kv(**o)
    assert attention(k=k) == want
    assert append(k=k) == want
    pairs = np.array([[0, 1]], np.int32)
    assert eb.lib().eahmmf_cuda_pages_copy(C.addressof(k), pairs.ctypes.data, 1, None) == want
    assert eb.lib().eahmmf_cuda_paged_attention_workspace_bytes(C.addressof(k), C.byref(seqs()), 4) == 0


def test_a_page_may_hold_its_layers_side_by_side():
    own = 2 * 16 * 64
    k = kv(layer_stride=own, page_stride=2 * own)
    assert attention(k=k, ws_bytes=0) == CAP  # past every check of the pools
    assert attention(k=kv(layer_stride=own, page_stride=2 * own - 8), ws_bytes=0) == BAD  # layers of two pages overlap


@pytest.mark.parametrize("o", BAD_SEQS)
def test_sequences_are_checked(o):
    assert attention(s=seqs(**o)) == BAD
    assert append(s=seqs(**o)) == BAD


@pytest.mark.parametrize("o", [dict(layer=-1), dict(layer=2), dict(n_head=3), dict(n_head=0), dict(n_head=130), dict(q=None),
                               dict(q=FAKE + 4), dict(ldq=255), dict(ldq=258), dict(scale=math.inf), dict(scale=math.nan),
                               dict(window=-1), dict(sinks=-1), dict(out=None), dict(ldo=252), dict(ws=None),
                               dict(ws=FAKE + 128)])
def test_attention_arguments_are_checked(o):
    assert attention(**o) == BAD


def test_attention_workspace_is_checked():
    need = eb.lib().eahmmf_cuda_paged_attention_workspace_bytes(C.byref(kv()), C.byref(seqs()), 4)
    assert need > 0
    assert attention(ws_bytes=need - 1) == CAP


@pytest.mark.parametrize("o", [dict(layer=2), dict(n_head=5), dict(x=None), dict(x=FAKE + 8), dict(ld=511), dict(ld=514),
                               dict(q=FAKE + 4), dict(ldq=252), dict(eps=-1.0), dict(eps=math.nan), dict(qn=FAKE + 4),
                               dict(kn=FAKE + 8), dict(r=rope(style=2)), dict(r=rope(n_rot=0)), dict(r=rope(n_rot=66)),
                               dict(r=rope(n_rot=7)), dict(r=rope(d_inv_freq=None))])
def test_append_arguments_are_checked(o):
    assert append(**o) == BAD


def test_calls_without_rows_launch_nothing():
    assert attention(s=seqs(n_seq=0, d_cu_q=None, d_kv_len=None, d_table=None)) == 0
    assert append(s=seqs(n_tok=0)) == 0
    assert eb.lib().eahmmf_cuda_pages_copy(C.byref(kv()), None, 0, None) == 0


@pytest.mark.parametrize("pairs,want", [([[0, 8]], IDX), ([[-1, 2]], IDX), ([[0, 3], [1, 3]], BAD), ([[0, 1], [1, 2]], BAD),
                                        ([[4, 4]], BAD), ([[5, 6], [2, 3], [6, 1]], BAD)])
def test_page_copies_are_checked(pairs, want):
    p = np.array(pairs, np.int32)
    assert eb.lib().eahmmf_cuda_pages_copy(C.byref(kv()), p.ctypes.data, len(p), None) == want


# ---- frequency tables ------------------------------------------------------------------------------
@pytest.mark.parametrize("n_rot", [2, 8, 64, 128])
def test_plain_and_linear_frequencies(n_rot):
    i = np.arange(n_rot // 2)
    f = 1e6 ** (-2.0 * i / n_rot)
    got, m = eb.rope_inv_freq(n_rot, 1e6)
    # pow is off by a few units of 64 bits, so only the one rounding to 32 bits (half a step) shows
    np.testing.assert_allclose(got, f, rtol=1.01 * 2.0 ** -24)
    assert m == 1.0
    got, m = eb.rope_inv_freq(n_rot, 1e6, "linear", 4.0)
    np.testing.assert_allclose(got, f / 4, rtol=1.01 * 2.0 ** -24)
    assert m == 1.0


def test_ntk_frequencies():
    got, m = eb.rope_inv_freq(64, 1e4, "ntk", 8.0)
    f = (1e4 * 8.0 ** (64 / 62)) ** (-2.0 * np.arange(32) / 64)
    np.testing.assert_allclose(got, f, rtol=1.01 * 2.0 ** -24)
    assert m == 1.0


@pytest.mark.parametrize("n_rot,base,factor,ctx", [(128, 1e6, 4.0, 32768), (64, 1e4, 16.0, 4096), (64, 1e4, 1.0, 4096)])
def test_yarn_frequencies(n_rot, base, factor, ctx):
    got, m = eb.rope_inv_freq(n_rot, base, "yarn", factor, ctx)
    lo = max(0, math.floor(n_rot * math.log(ctx / (32 * 2 * math.pi)) / (2 * math.log(base))))
    hi = min(n_rot - 1, math.ceil(n_rot * math.log(ctx / (1 * 2 * math.pi)) / (2 * math.log(base))))
    for i in range(n_rot // 2):
        f = base ** (-2.0 * i / n_rot)
        r = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        assert got[i] == pytest.approx(f * (1 - r) + f / factor * r, rel=1.01 * 2.0 ** -24)
    assert m == pytest.approx(0.1 * math.log(factor) + 1, rel=2.0 ** -23)
    # the fastest pairs keep their angle, the slowest are stretched by the factor
    assert got[0] == 1.0
    assert got[-1] == pytest.approx(base ** (-2.0 * (n_rot // 2 - 1) / n_rot) / factor, rel=1e-6) or hi > n_rot // 2 - 1


@pytest.mark.parametrize("args", [(0, 3, 1e6, 1.0, 0), (0, 0, 1e6, 1.0, 0), (0, 64, 1.0, 1.0, 0), (0, 64, math.inf, 1.0, 0),
                                  (1, 64, 1e6, 0.5, 0), (2, 2, 1e6, 2.0, 0), (3, 64, 1e6, 2.0, 0), (4, 64, 1e6, 2.0, 9),
                                  (1, 64, 1e6, math.nan, 0)])
def test_frequency_arguments_are_checked(args):
    out = np.zeros(64, np.float32)
    assert eb.lib().eahmmf_rope_inv_freq(*args, 32.0, 1.0, out.ctypes.data, None) == BAD


# ---- pages -----------------------------------------------------------------------------------------
def test_pages_create_checks():
    for a in [(0, 16, 1, 1), (4, 8, 1, 1), (4, 24, 1, 1), (4, 16, 0, 1), (4, 16, 1, 0), (4, 1024, 1, 1 << 22)]:
        with pytest.raises(RuntimeError):
            eb.Pages(*a)


def test_extend_takes_the_lowest_pages_and_refuses_without_a_trace():
    p = eb.Pages(5, 16, 2, 4)
    p.extend(0, 1)
    p.extend(1, 33)
    t, n = p.table()
    assert t.tolist() == [[0, -1, -1, -1], [1, 2, 3, -1]] and n.tolist() == [1, 33] and p.free == 1
    with pytest.raises(RuntimeError, match=str(CAP)):
        p.extend(0, 49)  # three more pages, one is free
    with pytest.raises(RuntimeError, match=str(CAP)):
        p.extend(1, 65)  # more than max_pages
    with pytest.raises(RuntimeError, match=str(BAD)):
        p.extend(1, 32)
    assert p.table()[0].tolist() == t.tolist() and p.free == 1
    p.truncate(1, 16)
    assert p.free == 3 and p.table()[0][1].tolist() == [1, -1, -1, -1]
    p.truncate(0)
    p.extend(1, 48)
    assert p.table()[0][1].tolist() == [1, 0, 2, -1]


def test_fork_shares_and_copies_the_part_filled_page():
    p = eb.Pages(8, 16, 3, 4)
    p.extend(0, 40)
    p.fork(0, 1)
    p.fork(1, 2)
    assert p.free == 5 and [p.refs(i) for i in range(3)] == [3, 3, 3]
    with pytest.raises(RuntimeError, match=str(BAD)):
        p.fork(0, 1)  # not empty
    p.extend(1, 41)
    p.extend(2, 48)
    p.extend(0, 41)  # the last holder writes in place
    assert p.take_copies().tolist() == [[2, 3], [2, 4]]
    assert p.table()[0].tolist() == [[0, 1, 2, -1], [0, 1, 3, -1], [0, 1, 4, -1]]
    p.extend(0, 48)
    assert len(p.take_copies()) == 0
    p.truncate(0)
    p.truncate(1)
    p.truncate(2)
    assert p.free == 8


def test_a_copy_of_a_page_not_yet_filled_reads_what_fills_it():
    p = eb.Pages(8, 16, 4, 2)
    p.extend(0, 5)
    p.fork(0, 1)
    p.extend(1, 6)      # records 0 -> 1
    p.fork(1, 2)
    p.extend(2, 7)      # page 1 is not filled yet: 0 -> 2
    p.truncate(0)       # page 0 is still read by the recorded copies: not handed out
    p.extend(3, 1)
    assert p.table()[0][3].tolist() == [3, -1]
    pairs = p.take_copies()
    assert pairs.tolist() == [[0, 1], [0, 2]]
    p.extend(3, 17)
    assert p.table()[0][3].tolist() == [3, 0]


def test_slide_gives_back_what_the_window_left():
    p = eb.Pages(8, 16, 1, 8)
    p.extend(0, 100)
    p.slide(0, 70, 4)  # keeps page 0 (sinks) and pages 4 ..
    assert p.table()[0][0].tolist() == [0, -1, -1, -1, 4, 5, 6, -1] and p.free == 4
    p.slide(0, 70, 4)
    assert p.free == 4
    with pytest.raises(RuntimeError, match=str(BAD)):
        p.truncate(0, 40)  # inside a page that is gone
    p.truncate(0, 64)
    assert p.table()[0][0].tolist() == [0, -1, -1, -1, -1, -1, -1, -1]
    p.extend(0, 65)
    assert p.table()[0][0].tolist() == [0, -1, -1, -1, 1, -1, -1, -1]
    p.slide(0, 1 << 30, 0)
    assert p.free == 7  # the part-filled page stays
    p.truncate(0)
    assert p.free == 8


def test_compact_moves_pages_to_the_front():
    p = eb.Pages(10, 16, 3, 4)
    p.extend(0, 64)
    p.extend(1, 40)
    p.fork(1, 2)
    p.truncate(0)
    p.compact()
    pairs = p.take_copies()
    assert pairs.tolist() == [[4, 0], [5, 1], [6, 2]]
    assert p.table()[0].tolist() == [[-1] * 4, [0, 1, 2, -1], [0, 1, 2, -1]] and p.free == 7
    p.extend(1, 41)
    with pytest.raises(RuntimeError, match=str(BAD)):
        p.compact()  # a recorded copy waits
    p.take_copies()
    p.compact()
    assert len(p.take_copies()) == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_calls_keep_every_sequence_its_positions(seed):
    """A model with real bytes: page contents are lists, copies run when they are taken, and every position of every sequence
    keeps what its own history wrote there."""
    rng = random.Random(seed)
    n_pages, page, n_seq, most = 24, 16, 5, 6
    p = eb.Pages(n_pages, page, n_seq, most)
    pool = [[None] * page for _ in range(n_pages)]
    want = [[] for _ in range(n_seq)]  # the value at every position; None where slide gave it back
    serial = 0
    for _ in range(400):
        s = rng.randrange(n_seq)
        todo = rng.random()
        if todo < 0.5:
            grow = len(want[s]) + rng.randint(0, 20)
            before, free = p.table(), p.free
            try:
                p.extend(s, grow)
            except RuntimeError:
                assert [x.tolist() for x in p.table()] == [x.tolist() for x in before] and p.free == free
                continue
            pairs = p.take_copies() if rng.random() < 0.8 or grow > len(want[s]) else []
            for a, b in pairs:
                assert a not in [y for _, y in pairs]
                pool[b] = list(pool[a])
            row = p.table()[0][s]
            for i in range(len(want[s]), grow):
                serial += 1
                assert p.refs(int(row[i // page])) == 1  # nobody else sees what is written
                pool[row[i // page]][i % page] = serial
                want[s].append(serial)
        elif todo < 0.65:
            d = rng.randrange(n_seq)
            if d != s and not want[d]:
                p.fork(s, d)
                want[d] = list(want[s])
        elif todo < 0.8:
            n = rng.randint(0, len(want[s]))
            if n % page == 0 or want[s][n // page * page] is not None:
                p.truncate(s, n)
                want[s] = want[s][:n]
        elif todo < 0.9:
            f, k = rng.randint(0, len(want[s])), rng.choice([0, 3, 20])
            p.slide(s, f, k)
            for i in range(-(-k // page) * page, f // page * page):
                want[s][i] = None
        else:
            p.compact()
            for a, b in p.take_copies():
                pool[b] = list(pool[a])
        table, n = p.table()
        held = {}
        for i in range(n_seq):
            assert n[i] == len(want[i])
            for j, x in enumerate(want[i]):
                if x is not None:
                    assert pool[table[i][j // page]][j % page] == x
            for x in table[i]:
                if x >= 0:
                    held[int(x)] = held.get(int(x), 0) + 1
        assert all(p.refs(x) == held.get(x, 0) for x in range(n_pages))
        assert p.free == n_pages - len(held)


# ---- the scheduler over a paged cache ----------------------------------------------------------------
class PagedEngine:
    """Counts pages as the engine does: a sequence of n positions holds ceil(n / page) of them."""

    def set_paged(self, n_slots, n_pages, page, dtype):
        self.n_slots, self.n_pages, self.page, self.len = n_slots, n_pages, page, {}
        return 0

    def used(self):
        return sum(-(-n // self.page) for n in self.len.values())

    def prefill_slot(self, slot, prompt, n_batch):
        assert slot not in self.len
        self.len[slot] = len(prompt)
        assert self.used() <= self.n_pages
        return 0, 1

    def step_slots(self, slots, pos, toks):
        for s, p in zip(slots, pos):
            assert self.len[s] == p
            self.len[s] += 1
        assert self.used() <= self.n_pages  # an admitted request never runs out of pages
        return 0, [1] * len(slots)

    def free_slot(self, slot):
        del self.len[slot]
        return 0


def test_scheduler_admits_what_the_pages_hold():
    import batching
    rng = random.Random(1)
    e = PagedEngine()
    b = batching.ContinuousBatcher(e, n_slots=6, pages=10, page=16)
    reqs = [b.submit([1] * rng.randint(1, 90), rng.randint(1, 60)) for _ in range(40)]
    b.run()
    assert all(len(r.tokens) == r.n_gen for r in reqs)
    assert not e.len
    with pytest.raises(ValueError):
        b.submit([1] * 150, 12)  # 161 positions fed: 11 pages
    b.submit([1] * 150, 11)
    b.run()
