"""The paged cache on the GPU (paged.cu) against its definitions in 64 bits.

Tolerances are worst-case bounds of the arithmetic, per element, formed from the inputs:
  u = 2^-23 a multiply-add in 32 bits (the matrix instructions may cut instead of rounding)
  scores     q and p carry 22 bits in two parts (2^-22 relative, 2^-21 with 32-bit keys whose low parts' product is left
             out), hd sums:  |ds| <= A (2^-21 + hd u), A = scale sum |q||k|
  weights    a relative error of 2 |ds| against their sum, exp of an argument of size x: (2 + x) u
  output     n sums of p v: (2 max|ds| + (4 + max x) u + 2^-21 + n u) sum p |v| / sum p
  append     hd squares, two roundings each of the scale, the weight and the turn: (hd / 2 + 8) u (|a| + |b|), and half a
             step of the pool's type (2^-11 relative, 2^-25 below the normal range of 16 bits)
"""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import eahmmf_b200 as eb

pytestmark = pytest.mark.gpu
U = 2.0 ** -23


@pytest.fixture(scope="module")
def torch():
    import torch
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required")
    return torch


class Call:
    """Pools with noise everywhere (NaN where nothing is cached), sequences with scattered pages, and the 64-bit answers."""

    def __init__(self, torch, type="f16", hd=128, n_kv=2, grp=8, page=16, q=(1,), kv=(20,), n_layer=1, layer=0, pad=0,
                 pool_of=None, seed=0, q_scale=3.0):
        self.torch, self.hd, self.n_kv, self.grp, self.page = torch, hd, n_kv, grp, page
        self.q_len, self.kv_len, self.n_head, self.layer = list(q), list(kv), n_kv * grp, layer
        rng = np.random.default_rng(seed)
        dt = torch.float16 if type == "f16" else torch.float32
        need = [max(0, -(-n // page)) for n in kv]
        n_pages = sum(need) + 2
        ids = rng.permutation(n_pages)
        ld = max([1] + need) + 1
        table = np.full((len(kv), ld), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = ids[at:at + n]
            at += n
        shape = (n_layer, n_pages, n_kv, page, hd)
        k, v = (rng.standard_normal(shape).astype(np.float16 if type == "f16" else np.float32) for _ in range(2))
        used = np.zeros((n_pages, page), bool)
        for s, n in enumerate(kv):
            for j in range(n):
                used[table[s, j // page], j % page] = True
        hide = np.broadcast_to(~used[None, :, None, :, None], shape)
        k[hide] = np.nan
        v[hide] = np.nan
        self.k64, self.v64, self.table_h = k.astype(np.float64), v.astype(np.float64), table
        make = pool_of or (lambda shape, dt: torch.empty(shape, dtype=dt, device="cuda"))
        self.k, self.v = make(shape, dt), make(shape, dt)
        self.k.copy_(torch.from_numpy(k))
        self.v.copy_(torch.from_numpy(v))
        n = sum(q)
        self.n_tok = n + pad
        self.q_h = (q_scale * rng.standard_normal((self.n_tok, self.n_head * hd))).astype(np.float32)
        self.q = torch.from_numpy(self.q_h).cuda()
        self.out = torch.full((self.n_tok, self.n_head * hd), 7.5, device="cuda")
        self.table = torch.from_numpy(table).cuda()
        self.cu = torch.tensor([0] + list(np.cumsum(q)), dtype=torch.int32, device="cuda")
        self.len = torch.tensor(kv, dtype=torch.int32, device="cuda")
        self.cache = eb.PagedCache(self.k, self.v)
        self.batch = eb.PagedBatch(self.table, self.cu, self.len, self.n_tok, max(list(q) + [0]), max(list(kv) + [0]))
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def attention(self, **o):
        self.cache.attention(self.layer, self.batch, self.q, self.n_head, self.out, d_status=self.status, **o)
        self.torch.cuda.synchronize()
        return self.out.cpu().numpy().astype(np.float64)

    def seq_kv(self, s, n):
        j = np.arange(n)
        pg = self.table_h[s, j // self.page]
        return self.k64[self.layer][pg, :, j % self.page], self.v64[self.layer][pg, :, j % self.page]  # [n][n_kv][hd]

    def want(self, scale=None, window=0, n_sink=0, q=None):
        """(output, bound) of every row; rows behind the last sequence keep what was there."""
        scale = self.hd ** -0.5 if scale is None else scale
        qh = (self.q_h if q is None else q).astype(np.float64).reshape(self.n_tok, self.n_head, self.hd)
        out = np.full((self.n_tok, self.n_head, self.hd), 7.5)
        tol = np.zeros_like(out)
        row = 0
        for s, (n, m) in enumerate(zip(self.q_len, self.kv_len)):
            ks, vs = self.seq_kv(s, m)
            for i in range(n):
                p = m - n + i
                j = np.arange(m)
                see = j <= p
                if window:
                    see &= (j > p - window) | (j < n_sink)
                for h in range(self.n_head):
                    g = h // self.grp
                    if not see.any():
                        out[row, h] = 0
                        continue
                    kk, vv, x = ks[see, g], vs[see, g], qh[row, h]
                    sc = scale * (kk @ x)
                    ds = abs(scale) * (np.abs(kk) @ np.abs(x)).max() * (2.0 ** -21 + self.hd * U)
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    out[row, h] = w @ vv
                    rel = 2 * ds + (4 + 1.5 * (sc.max() - sc.min())) * U + 2.0 ** -21 + len(w) * U
                    tol[row, h] = rel * (w @ np.abs(vv))
                row += 1
        shape = (self.n_tok, self.n_head * self.hd)
        return out.reshape(shape), tol.reshape(shape)

    def check(self, **o):
        got = self.attention(**o)
        o.pop("ws", None)
        want, tol = self.want(**o)
        assert np.isfinite(got).all()
        bad = np.abs(got - want) > tol
        assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want).max(), tol.max())
        assert int(self.status.item()) == 0
        return got


SHAPES = [  # head size, kv heads, q heads to each, page
    (128, 4, 8, 16), (128, 1, 1, 64), (64, 8, 2, 16), (64, 2, 7, 48), (128, 2, 16, 32), (64, 1, 20, 128), (128, 2, 4, 1024)]
STEPS = [((1,), (1,)), ((1,), (201,)), ((1, 1, 1), (17, 64, 1)), ((0, 1, 1, 0, 1), (5, 16, 300, 0, 63)), ((1, 1), (0, 33)),
         ((1,) * 9, (1, 2, 15, 16, 31, 130, 257, 64, 65))]
CHUNKS = [((2,), (2,)), ((3, 1), (130, 47)), ((17, 0, 33), (17, 9, 290)), ((64,), (200,)), ((5, 20), (3, 61)),
          ((150,), (150,))]


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", STEPS)
def test_single_tokens(torch, type, shape, lens):
    hd, n_kv, grp, page = shape
    Call(torch, type, hd, n_kv, grp, page, *lens, pad=2).check()


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", CHUNKS)
def test_chunks(torch, type, shape, lens):
    hd, n_kv, grp, page = shape
    Call(torch, type, hd, n_kv, grp, page, *lens, pad=1).check()


@pytest.mark.parametrize("type,hd,grp,page", [("f16", 128, 8, 16), ("f32", 64, 2, 32), ("f16", 64, 16, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (64, 0), (100, 70), (40, 1000), (10000, 3), (0, 9)])
@pytest.mark.parametrize("lens", [((1, 1, 1), (1, 90, 400)), ((40, 3), (300, 64))])
def test_windows_and_sinks(torch, type, hd, grp, page, window, sinks, lens):
    c = Call(torch, type, hd, 2, grp, page, *lens, seed=3)
    if window:  # pages that no row sees are gone from the table
        for s, (n, m) in enumerate(zip(*lens)):
            low = max(0, m - n - window + 1)
            c.table_h = c.table_h.copy()
            for i in range(-(-sinks // page), low // page):
                c.table[s, i] = -1
    c.check(window=window, n_sink=sinks)


@pytest.mark.parametrize("type,hd,grp", [("f16", 128, 8), ("f32", 64, 2), ("f16", 64, 1)])
@pytest.mark.parametrize("window", [1, 7, (1 << 31) - 9, (1 << 31) - 1])
@pytest.mark.parametrize("lens", [((12, 5, 1), (3, 1, 0)), ((40, 3, 150), (20, 1, 140)), ((300,), (270,))])
def test_more_rows_than_positions_in_a_window(torch, type, hd, grp, window, lens):
    Call(torch, type, hd, 2, grp, 16, *lens, seed=19).check(window=window, n_sink=2)


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_long_sequences_are_split_and_joined(torch, type):
    c = Call(torch, type, 128, 2, 8, 64, (1, 1), (9001, 37), seed=5)
    c.check()
    c.check(window=5000, n_sink=130)


def test_scores_of_every_size(torch):
    for q_scale in (0.0, 1e-30, 1e-6, 40.0, 1e5):
        c = Call(torch, "f16", 128, 1, 8, 16, (1, 2), (50, 30), seed=6, q_scale=q_scale)
        c.check()
        c.check(scale=-0.3 if q_scale < 1e4 else 1e-6)
        c.check(scale=0.0)


def test_one_position_far_above_the_rest(torch):
    """The rest's weights, each 2e-9 of the largest, add up to a visible part of the sum."""
    c = Call(torch, "f16", 128, 1, 8, 64, (1,), (30000,), seed=7, q_scale=0.0)
    c.q.zero_()
    c.q_h[:] = 0
    c.q_h[:, ::128] = 1.0
    c.q[:, ::128] = 1.0
    k = c.k64
    k[..., 0][~np.isnan(k[..., 0])] = 0.0
    pg = c.table_h[0, 777 // 64]
    k[0, pg, 0, 777 % 64, 0] = 20.0
    c.k.copy_(torch.from_numpy(k.astype(np.float16)))
    c.v.abs_()
    c.v64 = np.abs(c.v64)
    c.check(scale=1.0)


@pytest.mark.parametrize("page_major", [False, True])
@pytest.mark.parametrize("lens", [((1, 1), (40, 100)), ((20, 3), (50, 77))])
def test_layers_strides_and_row_strides(torch, page_major, lens):
    def pool(shape, dt):
        n_layer, n_pages, n_kv, page, hd = shape
        if page_major:
            return torch.empty(n_pages, n_layer, n_kv, page, hd, dtype=dt, device="cuda").transpose(0, 1)
        return torch.empty(n_layer, n_pages, n_kv + 1, page, hd, dtype=dt, device="cuda")[:, :, :n_kv]
    c = Call(torch, "f16", 64, 2, 4, 16, *lens, n_layer=3, layer=1, pool_of=pool, seed=8)
    c.q = torch.cat([c.q, c.q + 1], 1)[:, : c.q.shape[1]]
    wide = torch.full((c.n_tok, c.out.shape[1] + 12), 7.5, device="cuda")
    c.out = wide[:, 4:-8]
    c.check()
    assert (wide[:, :4] == 7.5).all() and (wide[:, -8:] == 7.5).all()


@pytest.mark.parametrize("type", ["f16", "f32"])
def test_offsets_past_32_bits(torch, type):
    far = (1 << 31) + (1 << 20)  # elements from page to page
    base = {}

    def pool(shape, dt):
        n = far * (shape[1] - 1) + int(np.prod(shape[2:]))
        if "t" not in base:
            base["t"] = torch.empty(n + int(np.prod(shape[2:])), dtype=dt, device="cuda")
        off = int(np.prod(shape[2:])) if "k" in base else 0
        base["k"] = 1
        return torch.as_strided(base["t"], shape, (far * shape[1], far, shape[3] * shape[4], shape[4], 1), off)
    c = Call(torch, type, 128, 1, 8, 16, (1, 2), (16, 30), pool_of=pool, seed=9)
    assert c.k.shape[1] == 5
    c.check()
    rope_case(torch, c, "half", 128, True)


def test_bad_pages_and_lengths_are_skipped_and_flagged(torch):
    for q in ((1,), (20,)):
        c = Call(torch, "f16", 128, 2, 8, 16, q, (100,), seed=10)
        for bad in (-1, c.k.shape[1], 1 << 30, -(1 << 31)):
            c.table.copy_(torch.from_numpy(c.table_h))
            c.table[0, 2] = bad
            got = c.attention()
            assert np.isfinite(got).all() and int(c.status.item()) == eb.ST_BAD_INDEX
            c.status.zero_()
        c.table.copy_(torch.from_numpy(c.table_h))
        c.len.fill_(1 << 30)  # more than the table names: cut to its capacity, whose last page is no page (the call then
        c.attention()         # sees positions 100 .. 111, which hold NaN here)
        assert int(c.status.item()) == eb.ST_BAD_INDEX
        c.status.zero_()
        c.len.fill_(-5)
        assert (c.attention() == 0).all() and int(c.status.item()) == eb.ST_BAD_INDEX
        c.status.zero_()
        c.len.fill_(100)
        c.cu[1] = c.n_tok + 1000
        c.attention()
        assert int(c.status.item()) == eb.ST_BAD_INDEX
        c.status.zero_()
        c.cu[0], c.cu[1] = 5, 1
        c.out.fill_(7.5)
        assert (c.attention() == 7.5).all() and int(c.status.item()) == eb.ST_BAD_INDEX


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("lens", [((1, 1), (40, 700)), ((5, 1, 40), (40, 700, 90))])
@pytest.mark.parametrize("max_q,max_kv", [(0, 0), (1, 1 << 30), (1 << 30, 0), (1 << 30, 1 << 30)])
def test_bounds_of_the_lengths_do_not_matter(torch, type, lens, max_q, max_kv):
    c = Call(torch, type, 128, 2, 8, 16, *lens, seed=14)
    c.batch = eb.PagedBatch(c.table, c.cu, c.len, c.n_tok, max_q, max_kv)
    c.check()
    c.check(window=(1 << 31) - 1, n_sink=(1 << 31) - 1)


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("q", [(1,), (0, 1, 3, 20, 1, 0)])
def test_many_sequences(torch, type, q):
    n = 900
    qs = tuple(q[i % len(q)] for i in range(n))
    Call(torch, type, 64, 1, 2, 16, qs, tuple(m + (7 * i) % 61 for i, m in enumerate(qs)), seed=15).check()


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("n_kv,grp,longest", [(1, 2, 1500), (1, 16, 1100), (3, 5, 300), (2, 8, 700)])
def test_many_sequences_with_a_few_long_ones(torch, type, n_kv, grp, longest):  # tiles cut, or whole with several a block
    lens = tuple(longest - i % 13 if i % 61 == 60 else 1 + (11 * i) % 47 for i in range(300))
    qs = tuple((0 if i % 7 == 3 else 1) for i in range(300))
    Call(torch, type, 64, n_kv, grp, 16, qs, lens, seed=18).check()


def test_the_first_call_of_a_process_may_be_captured(torch):
    code = """
import sys; sys.path[:0] = [%r, %r]
import torch, test_gpu_paged as t
for q in ((1,), (40,)):
    for type in ("f16", "f32"):
        c = t.Call(torch, type, 128, 2, 8, 16, q, (900,), seed=16)
        ws = c.cache.attention_workspace(c.batch, c.n_head)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.cache.attention(0, c.batch, c.q, c.n_head, c.out, ws=ws, d_status=c.status)
        g.replay(); torch.cuda.synchronize()
        want, tol = c.want()
        assert (abs(c.out.cpu().numpy() - want) <= tol).all()
""" % (os.path.dirname(eb.__file__), os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=200)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_check_status_workspace_and_table(torch):
    c = Call(torch, "f16", 64, 2, 2, 16, (2,), (20,), seed=17)
    x, rope = torch.randn(2, 8 * 64, device="cuda"), eb.Rope(torch.ones(32, device="cuda"))
    for status in (torch.zeros(1, dtype=torch.int32), c.status.long(), c.status[:0]):
        with pytest.raises(ValueError):
            c.cache.attention(0, c.batch, c.q, c.n_head, c.out, d_status=status)
        with pytest.raises(ValueError):
            c.cache.append(0, c.batch, x, c.n_head, rope, c.out, d_status=status)
    ws = c.cache.attention_workspace(c.batch, c.n_head)
    for bad in (ws.cpu(), torch.cat([ws, ws])[::2]):
        with pytest.raises(ValueError):
            c.cache.attention(0, c.batch, c.q, c.n_head, c.out, ws=bad)
    with pytest.raises(RuntimeError):
        c.cache.attention(0, c.batch, c.q, c.n_head, c.out, ws=ws[:-256])
    rope.index += 1  # as of a table on another device
    with pytest.raises(ValueError):
        c.cache.append(0, c.batch, x, c.n_head, rope, c.out)
    for pairs in ([0, 1], [[[0, 1]]], [[0], [1]]):
        with pytest.raises(ValueError):
            c.cache.copy_pages(pairs)
    c.cache.copy_pages([])


def test_calls_check_their_tensors(torch):
    c = Call(torch, "f16", 64, 2, 2, 16, (2,), (20,), seed=17)
    for bad in (c.q.double(), c.q[:1], c.q[:, :-4], c.q.cpu(), c.q.t()):
        with pytest.raises(ValueError):
            c.cache.attention(0, c.batch, bad, c.n_head, c.out)
    with pytest.raises(ValueError):
        c.cache.attention(0, c.batch, c.q, c.n_head, c.out, stream=torch.cuda.Stream())  # no workspace of its own
    with pytest.raises(RuntimeError):
        c.cache.attention(1, c.batch, c.q, c.n_head, c.out)
    for bad in ([[0, 1 << 32]], [[0, -1]], [[0.0, 1.0]], [[0, 1, 2]]):
        with pytest.raises(ValueError):
            c.cache.copy_pages(bad)
    with pytest.raises(RuntimeError):
        c.cache.copy_pages([[0, 0]])
    with pytest.raises(ValueError):
        eb.PagedCache(c.k, c.v.float())
    with pytest.raises(ValueError):
        eb.PagedCache(c.k[..., ::2], c.v[..., ::2])
    with pytest.raises(ValueError):
        eb.PagedBatch(c.table.long(), c.cu, c.len, 2, 1, 1)
    with pytest.raises(ValueError):
        eb.PagedBatch(c.table, c.cu[:-1], c.len, 2, 1, 1)


@pytest.mark.parametrize("lens", [((1, 1, 1), (30, 700, 64)), ((30, 1), (30, 700))])
def test_captured_calls_follow_the_lengths_on_the_device(torch, lens):
    c = Call(torch, "f16", 128, 2, 8, 16, *lens, seed=11)
    ws = c.cache.attention_workspace(c.batch, c.n_head)
    first = c.check(ws=ws)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.cache.attention(0, c.batch, c.q, c.n_head, c.out, ws=ws, d_status=c.status)
    c.out.fill_(7.5)
    g.replay()
    torch.cuda.synchronize()
    assert (c.out.cpu().numpy() == first).all()
    c.kv_len = [m - 10 for m in c.kv_len]
    c.len.copy_(torch.tensor(c.kv_len, dtype=torch.int32))
    ws.fill_(255)
    c.out.fill_(7.5)
    g.replay()
    torch.cuda.synchronize()
    want, tol = c.want()
    assert (np.abs(c.out.cpu().numpy() - want) <= tol).all()


def test_two_calls_at_once_with_a_workspace_each(torch):
    cs = [Call(torch, "f16", 128, 2, 8, 16, q, kv, seed=12 + i)
          for i, (q, kv) in enumerate([((1,), (5000,)), ((1, 1), (4000, 90)), ((40,), (900,))])]
    alone = [c.attention() for c in cs]
    ws = [c.cache.attention_workspace(c.batch, c.n_head) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    for c in cs:
        c.out.fill_(0)
    torch.cuda.synchronize()
    for _ in range(20):
        for c, w, s in zip(cs, ws, streams):
            with torch.cuda.stream(s):
                c.cache.attention(0, c.batch, c.q, c.n_head, c.out, ws=w)
    torch.cuda.synchronize()
    for c, a in zip(cs, alone):
        assert (c.out.cpu().numpy() == a).all()


# ---- rotary positions + append ----------------------------------------------------------------------
def rope_case(torch, c, style, n_rot, norm, mscale=1.0, base=1e4):
    rng = np.random.default_rng(99)
    hd, n_all = c.hd, c.n_head + 2 * c.n_kv
    x = rng.standard_normal((c.n_tok, n_all * hd)).astype(np.float32)
    wq, wk = ((1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    f, _ = eb.rope_inv_freq(n_rot, base)
    rope = eb.Rope(torch.from_numpy(f).cuda(), style, mscale)
    dq, dk = (torch.from_numpy(wq).cuda(), torch.from_numpy(wk).cuda()) if norm else (None, None)
    q_out = torch.full((c.n_tok, c.n_head * hd), 7.5, device="cuda")
    before = [t.clone() for t in (c.k, c.v)]
    c.cache.append(c.layer, c.batch, torch.from_numpy(x).cuda(), c.n_head, rope, q_out, dq, dk, 1e-6, d_status=c.status)
    torch.cuda.synchronize()
    x = x.astype(np.float64).reshape(c.n_tok, n_all, hd)
    want_q = np.full((c.n_tok, c.n_head, hd), 7.5)
    tol_q = np.zeros_like(want_q)
    wants = [b.double().cpu().numpy() for b in before]
    tols = [np.zeros_like(w) for w in wants]
    es = 2.0 ** -11 if c.k.dtype == torch.float16 else 0.0
    row = 0
    for s, (n, m) in enumerate(zip(c.q_len, c.kv_len)):
        for i in range(n):
            p = m - n + i
            y = x[row].copy()
            if norm:
                y[: c.n_head + c.n_kv] /= np.sqrt((y[: c.n_head + c.n_kv] ** 2).mean(-1, keepdims=True) + 1e-6)
                y[: c.n_head] *= wq
                y[c.n_head: c.n_head + c.n_kv] *= wk
            mag = np.abs(y)
            h = n_rot // 2
            a, b = (np.arange(h), np.arange(h) + h) if style == "half" else (2 * np.arange(h), 2 * np.arange(h) + 1)
            ang = p * f.astype(np.float64)
            rot = y[: c.n_head + c.n_kv].copy()
            ya, yb = rot[:, a].copy(), rot[:, b].copy()
            rot[:, a] = (ya * np.cos(ang) - yb * np.sin(ang)) * mscale
            rot[:, b] = (ya * np.sin(ang) + yb * np.cos(ang)) * mscale
            both = mag[: c.n_head + c.n_kv].copy()
            both[:, a] = both[:, b] = (np.abs(ya) + np.abs(yb)) * mscale
            bound = (hd / 2 + 8) * U * both
            if p < 0:
                want_q[row] = 0
            else:
                want_q[row], tol_q[row] = rot[: c.n_head], bound[: c.n_head]
                pg, o = c.table_h[s, p // c.page], p % c.page
                wants[0][c.layer, pg, :, o] = rot[c.n_head:]
                tols[0][c.layer, pg, :, o] = bound[c.n_head:] + es * np.abs(rot[c.n_head:]) + 2.0 ** -25
                wants[1][c.layer, pg, :, o] = y[c.n_head + c.n_kv:]
                tols[1][c.layer, pg, :, o] = es * np.abs(y[c.n_head + c.n_kv:]) + 2.0 ** -25 * (es > 0)
            row += 1
    got = q_out.cpu().numpy().reshape(want_q.shape)
    assert (np.abs(got - want_q) <= tol_q).all(), np.abs(got - want_q).max()
    for t, w, tol in zip((c.k, c.v), wants, tols):
        g = t.double().cpu().numpy()
        assert ((np.isnan(g) & np.isnan(w)) | (np.abs(g - w) <= tol)).all()
    assert int(c.status.item()) == 0


@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("type,hd,n_kv,grp,page,n_rot", [
    ("f16", 128, 4, 8, 16, 128), ("f32", 128, 2, 16, 64, 64), ("f16", 64, 1, 7, 48, 64), ("f32", 64, 3, 2, 32, 20),
    ("f16", 64, 2, 1, 16, 2), ("f32", 128, 1, 3, 16, 126), ("f16", 128, 8, 8, 128, 36)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(torch, style, type, hd, n_kv, grp, page, n_rot, norm):
    c = Call(torch, type, hd, n_kv, grp, page, (1, 0, 20, 3, 1), (1, 7, 33, 2, 150), pad=2, seed=20, n_layer=2, layer=1)
    rope_case(torch, c, style, n_rot, norm, mscale=1.25 if norm else 1.0)


def test_append_far_positions(torch):
    """At position 1e5 a 32-bit angle would be off by 4e-3."""
    c = Call(torch, "f16", 64, 1, 2, 1024, (2,), (131001,), seed=21)
    rope_case(torch, c, "half", 64, False)


def test_append_one_norm_and_many_sequences(torch):
    c = Call(torch, "f32", 64, 1, 1, 16, (1,) * 700, tuple(1 + i % 40 for i in range(700)), seed=22)
    rope_case(torch, c, "interleaved", 64, True)


def test_append_skips_bad_pages(torch):
    c = Call(torch, "f16", 128, 2, 8, 16, (1, 1), (20, 40), seed=23)
    rope = eb.Rope(torch.ones(64, device="cuda"))
    x = torch.randn(2, 20 * 128, device="cuda")
    k0 = c.k.clone()
    for bad in (-1, c.k.shape[1], 1 << 30):
        c.table[0, 1] = bad
        c.table[1, 2] = bad
        c.cache.append(0, c.batch, x, 16, rope, c.out, d_status=c.status)
        torch.cuda.synchronize()
        assert int(c.status.item()) == eb.ST_BAD_INDEX
        assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))
        c.status.zero_()


# ---- pages ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,n_layer,n_kv,page,hd,n", [("float16", 3, 2, 16, 64, 5), ("float32", 1, 4, 48, 128, 1),
                                                         ("float16", 2, 1, 16, 64, 1100), ("float32", 48, 3, 16, 64, 7)])
def test_page_copies(torch, dtype, n_layer, n_kv, page, hd, n):
    shape = (n_layer, 2 * n + 3, n_kv, page, hd)
    k, v = (torch.randn(shape, device="cuda").to(getattr(torch, dtype)) for _ in range(2))
    ids = np.random.default_rng(n).permutation(2 * n + 3)[: 2 * n].astype(np.int32)
    pairs = ids.reshape(n, 2)
    want = []
    for t in (k, v):
        w = t.clone()
        w[:, torch.from_numpy(pairs[:, 1]).long().cuda()] = t[:, torch.from_numpy(pairs[:, 0]).long().cuda()]
        want.append(w)
    eb.PagedCache(k, v).copy_pages(pairs)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_page_copies_of_page_major_pools(torch):
    base = [torch.randn(6, 3, 2, 16, 64, device="cuda") for _ in range(2)]
    want = [b.clone() for b in base]
    for w in want:
        w[4] = w[1]
    eb.PagedCache(base[0].transpose(0, 1), base[1].transpose(0, 1)).copy_pages([[1, 4]])
    torch.cuda.synchronize()
    assert all(torch.equal(b, w) for b, w in zip(base, want))


# ---- together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("type", ["f16", "f32"])
def test_sequences_grow_fork_slide_and_compact(torch, type):
    """Prompts, single tokens, a fork that diverges, a window that gives pages back and a compaction: every output equals the
    attention over the sequence's own history kept in a plain list."""
    hd, n_kv, grp, page, n_pages, window, sinks = 64, 2, 4, 16, 40, 50, 3
    n_head, rng = n_kv * grp, np.random.default_rng(31)
    dt = torch.float16 if type == "f16" else torch.float32
    k, v = (torch.full((2, n_pages, n_kv, page, hd), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    cache, pages = eb.PagedCache(k, v), eb.Pages(n_pages, page, 4, 12)
    f, _ = eb.rope_inv_freq(hd, 1e4)
    rope = eb.Rope(torch.from_numpy(f).cuda())
    hist = [[] for _ in range(4)]  # per sequence: (rotated k, v) as the pool holds them, read back after each append
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(grow):
        for s, n in grow:
            pages.extend(s, int(pages.table()[1][s]) + n)
        cache.copy_pages(pages.take_copies())
        table, length = pages.table()
        q_len = [dict(grow).get(s, 0) for s in range(4)]
        n = sum(q_len)
        x = torch.from_numpy(rng.standard_normal((n, (n_head + 2 * n_kv) * hd)).astype(np.float32)).cuda()
        cu = torch.tensor([0] + list(np.cumsum(q_len)), dtype=torch.int32, device="cuda")
        batch = eb.PagedBatch(torch.from_numpy(table).cuda(), cu, torch.from_numpy(length).cuda(), n, max(q_len),
                              int(length.max()))
        q, out = torch.empty(n, n_head * hd, device="cuda"), torch.empty(n, n_head * hd, device="cuda")
        cache.append(1, batch, x, n_head, rope, q, d_status=status)
        cache.attention(1, batch, q, n_head, out, window=window, n_sink=sinks, d_status=status)
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        row = 0
        for s, m in enumerate(q_len):
            for i in range(m):
                p = int(length[s]) - m + i
                hist[s].append((k[1, table[s, p // page], :, p % page].double(), v[1, table[s, p // page], :, p % page].double()))
            for i in range(m):
                p = int(length[s]) - m + i
                j = [a for a in range(p + 1) if a > p - window or a < sinks]
                ks, vs = (torch.stack([hist[s][a][z] for a in j]) for z in (0, 1))
                qq = q[row].double().view(n_kv, grp, hd)
                sc = torch.einsum("ngd,jnd->ngj", qq, ks) / math.sqrt(hd)
                o = torch.einsum("ngj,jnd->ngd", torch.softmax(sc, -1), vs)
                # |q.k| / 8 stays below 8 here, so the bound above is under 2 * 8 * 9e-6 + 1e-5 of |v| < 6
                assert (out[row].double().view(n_kv, grp, hd) - o).abs().max() < 1e-3
                row += 1

    step([(0, 37), (1, 5)])
    step([(0, 1), (1, 1)])
    pages.fork(0, 2)
    hist[2] = list(hist[0])
    step([(0, 1), (2, 1), (1, 1)])
    pages.fork(2, 3)
    hist[3] = list(hist[2])
    for _ in range(4):
        step([(0, 20), (1, 1), (2, 1), (3, 9)])
        for s in range(4):
            n = int(pages.table()[1][s])
            pages.slide(s, max(0, n - window + 1), sinks)
    pages.truncate(1)
    pages.compact()
    cache.copy_pages(pages.take_copies())
    used = n_pages - pages.free
    t = pages.table()[0]
    assert t.max() < used
    k[:, used:] = float("nan")  # what lies behind the used pages belongs to nobody
    hist[1] = []
    step([(0, 1), (1, 30), (2, 2), (3, 1)])
