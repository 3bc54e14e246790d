"""Chunks of new tokens over the paged cache (paged_tc.cu) where a block has several row tiles one after another.

The answers are torch's in 64 bits, with the bounds that test_gpu_paged.py derives, formed on the device: per row
(2 max|ds| + (4 + 1.5 range of the scores) u + 2^-21 + n u) sum p |v|,  |ds| <= scale sum |q||k| (2^-21 + hd u),  u = 2^-23."""
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


class Chunks:
    """Sequences of q new tokens each behind kv cached positions (with them), every activation and element given by `make`."""

    def __init__(self, torch, type, hd, n_kv, grp, page, q, kv, seed=0, make=None):
        self.torch, self.hd, self.n_kv, self.grp, self.page, self.q_len, self.kv_len = torch, hd, n_kv, grp, page, q, kv
        g = torch.Generator("cuda")
        g.manual_seed(seed)
        make = make or (lambda what, shape: torch.randn(shape, generator=g, device="cuda"))
        self.n_head, rows, dt = n_kv * grp, sum(q), torch.float16 if type == "f16" else torch.float32
        need = [-(-n // page) for n in kv]
        ids = torch.randperm(sum(need) + 1, generator=g, device="cuda").to(torch.int32)
        table = np.full((len(kv), max(need)), -1, np.int64)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = np.arange(at, at + n)
            at += n
        t = torch.from_numpy(table).cuda()
        self.table = torch.where(t >= 0, ids[t.clamp(min=0)], -1).to(torch.int32).contiguous()
        shape = (1, sum(need) + 1, n_kv, page, hd)
        self.k, self.v = (torch.full(shape, float("nan"), dtype=dt, device="cuda") for _ in "kv")
        self.hist = []  # of each sequence: k and v [kv][n_kv][hd] as the pools hold them
        for s, n in enumerate(kv):
            both = []
            for what, pool in (("k", self.k), ("v", self.v)):
                x = make(what, (n, n_kv, hd)).to(dt)
                pos = torch.arange(n, device="cuda")
                pool[0, self.table[s].long()[pos // page], :, pos % page] = x
                both.append(x.double())
            self.hist.append(both)
        self.q = make("q", (rows, self.n_head * hd)).float()
        self.out = torch.full((rows, self.n_head * hd), 7.5, device="cuda")
        cu = torch.tensor([0] + list(np.cumsum(q)), dtype=torch.int32, device="cuda")
        self.cache = eb.PagedCache(self.k, self.v)
        self.batch = eb.PagedBatch(self.table, cu, torch.tensor(kv, dtype=torch.int32, device="cuda"), rows, max(q), max(kv))
        self.ws = self.cache.attention_workspace(self.batch, self.n_head)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def attention(self, **o):
        self.cache.attention(0, self.batch, self.q, self.n_head, self.out, ws=self.ws, d_status=self.status, **o)
        return self.out

    def want(self, scale=None, window=0, n_sink=0):
        torch, hd = self.torch, self.hd
        scale = hd ** -0.5 if scale is None else scale
        out, tol, row = torch.zeros_like(self.out, dtype=torch.float64), torch.zeros_like(self.out, dtype=torch.float64), 0
        for (k, v), n, m in zip(self.hist, self.q_len, self.kv_len):
            x = self.q[row:row + n].double().view(n, self.n_kv, self.grp, hd)
            j, p = torch.arange(m, device="cuda"), torch.arange(m - n, m, device="cuda")[:, None]
            see = j <= p
            if window:
                see &= (j > p - window) | (j < n_sink)
            for g in range(self.n_kv):
                hide = ~see[:, None].expand(n, self.grp, m)
                sc = (torch.einsum("rgd,jd->rgj", x[:, g], k[:, g]) * scale)
                ds = (torch.einsum("rgd,jd->rgj", x[:, g].abs(), k[:, g].abs()) * abs(scale)).masked_fill(hide, 0.0).amax(-1)
                ds = ds * (2.0 ** -21 + hd * U)
                span = sc.masked_fill(hide, -np.inf).amax(-1) - sc.masked_fill(hide, np.inf).amin(-1)
                w = torch.softmax(sc.masked_fill(hide, -np.inf), -1)
                rel = 2 * ds + (4 + 1.5 * span) * U + 2.0 ** -21 + m * U
                o = torch.einsum("rgj,jd->rgd", w, v[:, g])
                b = torch.einsum("rgj,jd->rgd", w, v[:, g].abs()) * rel[..., None]
                at = slice(g * self.grp * hd, (g + 1) * self.grp * hd)
                out[row:row + n, at], tol[row:row + n, at] = o.reshape(n, -1), b.reshape(n, -1)
            row += n
        return out, tol

    def check(self, **o):
        got = self.attention(**o).double()
        want, tol = self.want(**o)
        far = (got - want).abs() - tol
        assert bool((far <= 0).all()), (int((far > 0).sum()), float(far.max()))
        assert int(self.status.item()) == 0
        return got


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("hd,n_kv,grp,q,kv", [(128, 4, 16, [1500], [1500]), (64, 8, 8, [1300, 700], [1301, 2100]),
                                              (128, 8, 7, [500, 401, 300], [900, 402, 340])])
def test_several_row_tiles_a_block_are_the_same_every_time(torch, type, hd, n_kv, grp, q, kv):
    """A tile's output leaves through the bytes that the next tile's q takes; a warp that runs ahead or stays behind would show as
    an output that differs from call to call, or from the formula's."""
    c = Chunks(torch, type, hd, n_kv, grp, 64, q, kv, seed=1)
    first = c.check().float()
    load = torch.randn(4096, 4096, device="cuda")
    for i in range(30):
        c.out.fill_(7.5)
        if i % 3 == 1:
            load @ load  # another state of the clocks and the caches
        assert torch.equal(c.attention(), first), i
    c.check(window=200, n_sink=3)


LENS = [([40, 3, 17], [300, 50, 17]), ([130], [1000])]


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("hd,grp", [(128, 8), (64, 8), (128, 5)])
@pytest.mark.parametrize("lens", LENS)
def test_rows_of_very_different_size_do_not_disturb_each_other(torch, type, hd, grp, lens):
    """A third of the tokens and one head have a q 2^45 as large: the others' outputs are as without them."""
    c = Chunks(torch, type, hd, 2, grp, 16, *lens, seed=2)
    large = torch.zeros(c.q.shape, dtype=torch.bool, device="cuda")
    large[1::3] = True
    large[:, 3 * hd:4 * hd] = True
    for o in (dict(), dict(scale=-0.05, window=100, n_sink=2)):
        want, tol = c.want(**o)
        c.q[large] *= 2.0 ** 45
        got = c.attention(**o).double()
        c.q[large] *= 2.0 ** -45
        far = ((got - want).abs() - tol)[~large]
        assert bool((far <= 0).all()), (int((far > 0).sum()), float(far.max()))


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e-6, 40.0, 1e5])
@pytest.mark.parametrize("lens", LENS)
def test_chunk_scores_of_every_size(torch, type, q_scale, lens):
    g = torch.Generator("cuda")
    g.manual_seed(4)
    c = Chunks(torch, type, 128, 2, 8, 16, *lens, seed=4,
               make=lambda what, shape: torch.randn(shape, generator=g, device="cuda") * (q_scale if what == "q" else 1.0))
    for scale in (None, -0.3 if q_scale < 1e4 else -1e-6, 0.0, 1e-36):
        c.check(scale=scale)


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("lens", LENS)
def test_a_row_that_is_not_finite_is_alone(torch, type, lens):
    c = Chunks(torch, type, 128, 2, 8, 16, *lens, seed=5)
    want, tol = c.want()
    rows = {1: float("nan"), 7: float("inf"), 30: float("-inf")}
    for r, x in rows.items():
        c.q[r, 5 * 128 + 17] = x  # head 5 of the row
    got = c.attention().double()
    for r in rows:
        assert not bool(torch.isfinite(got[r, 5 * 128:6 * 128]).any())
        got[r, 5 * 128:6 * 128] = want[r, 5 * 128:6 * 128]
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("lens", LENS + [([1, 1], [300, 40]), ([2], [500])])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("x", [float("nan"), float("inf"), float("-inf")])
def test_a_cached_element_that_is_not_finite_reaches_the_rows_that_see_it(torch, type, lens, what, x):
    c = Chunks(torch, type, 128, 2, 8, 16, *lens, seed=6)
    want, tol = c.want()
    n, m = c.q_len[0], c.kv_len[0]
    at = m - (n + 1) // 2  # a position in the middle of the first sequence's new ones
    (c.k if what == "k" else c.v)[0, c.table[0, at // 16], 1, at % 16, 9] = x
    got = c.attention().double()
    first, half = n - (m - at), 8 * 128  # the rows from `first` on see it, in the heads of kv head 1
    seen = got[first:n, half:]
    if what == "v":
        assert not bool(torch.isfinite(seen.view(-1, 8, 128)[..., 9]).any())
    elif x != x:
        assert not bool(torch.isfinite(seen).any())
    ok = (got - want).abs() <= tol
    ok[first:n, half:] = True
    if what == "v":
        ok[:first, half:] = True  # an earlier row of the sequence: a weight of zero does not hide it
    assert bool(ok.all())


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("hd", [64, 128])
def test_wide_ranges_over_32_bit_pages(torch, hd, lens):
    """k and v of 2^-30 to 2^10 beside each other: an element is held to 2^-22 of itself or 2^-39 of the largest of its unit, so a
    score is off by 2^-39 max|k| sum|q| and an output by 2^-39 max|v| more."""
    g = torch.Generator("cuda")
    g.manual_seed(7)

    def make(what, shape):
        x = torch.randn(shape, generator=g, device="cuda")
        return x * 2.0 ** -8 if what == "q" else x * 2.0 ** torch.randint(-30, 11, shape, generator=g, device="cuda").float()
    c = Chunks(torch, "f32", hd, 2, 8, 16, *lens, seed=7, make=make)
    got = c.attention().double()
    want, tol = c.want()
    row = 0
    for (k, v), n, m in zip(c.hist, c.q_len, c.kv_len):
        s = slice(row, row + n)
        extra = c.q[s].double().abs().view(n, -1, hd).sum(-1) * hd ** -0.5 * float(k.abs().max()) * 2.0 ** -39
        tol[s] += (2 * extra[..., None] * float(v.abs().max()) + float(v.abs().max()) * 2.0 ** -39).expand(n, -1, hd).reshape(n, -1)
        row += n
    assert bool(((got - want).abs() <= tol).all())
    assert int(c.status.item()) == 0


def far_scores(torch, type, hd, grp, lens, e):
    """Small whole numbers in q and k, q times 2^e: the scores are exact, and a row's largest ones outweigh the rest by 2^256 at
    least, so that it has the mean of their v. The weights of the largest are equal; their sum and the products with v round n
    times in 32 bits and once to 22."""
    g = torch.Generator("cuda")
    g.manual_seed(8)

    def make(what, shape):
        x = torch.randint(-3, 4, shape, generator=g, device="cuda").float()
        return torch.randn(shape, generator=g, device="cuda") if what == "v" else x * 2.0 ** e if what == "q" else x
    c = Chunks(torch, type, hd, 2, grp, 16, *lens, seed=8, make=make)
    for scale in (1.0, -1.0):
        want, _ = c.want(scale=scale)
        got = c.attention(scale=scale).double()
        assert bool(torch.isfinite(got).all())
        vmax = max(float(v.abs().max()) for _, v in c.hist)
        assert float((got - want).abs().max()) <= vmax * (2.0 ** -21 + max(c.kv_len) * U)


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("hd,grp", [(128, 8), (64, 6)])
@pytest.mark.parametrize("lens", LENS + [([24], [24])])
@pytest.mark.parametrize("e", [8, 14, 15, 16, 17, 18, 20, 23, 26, 40, 80])
def test_chunk_scores_past_24_bits(torch, type, hd, grp, lens, e):
    far_scores(torch, type, hd, grp, lens, e)


@pytest.mark.parametrize("type", ["f16", "f32"])
@pytest.mark.parametrize("hd,grp", [(128, 8), (64, 5), (128, 16)])  # tiles of 8 and of 16 rows
@pytest.mark.parametrize("lens", [([1, 1], [300, 40]), ([1], [3000]), ([1] * 40, [41] * 40)])
@pytest.mark.parametrize("e", [8, 14, 15, 16, 17, 18, 20, 23, 26, 40, 80])
def test_step_scores_past_24_bits(torch, type, hd, grp, lens, e):
    far_scores(torch, type, hd, grp, lens, e)


def test_calls_refuse_numbers_past_32_bits(torch):
    c = Chunks(torch, "f16", 64, 1, 2, 16, [20], [30], seed=9)
    first = c.check(window=7)
    far = 1 << 32
    for o in (dict(window=far), dict(window=far + 7), dict(window=7, n_sink=far)):
        with pytest.raises(ValueError):
            c.attention(**o)
    with pytest.raises(ValueError):
        c.cache.attention(far, c.batch, c.q, c.n_head, c.out, ws=c.ws)
    rope = eb.Rope(torch.ones(32, device="cuda"))
    with pytest.raises(ValueError):
        c.cache.append(far, c.batch, torch.zeros(20, 4 * 64, device="cuda"), c.n_head, rope, c.out)
    for o in ((far + 20, 20, 30), (20, far + 20, 30), (20, 20, far)):
        with pytest.raises(ValueError):
            eb.PagedBatch(c.table, c.batch._keep[1], c.batch._keep[2], *o)
    assert torch.equal(c.attention(window=7).double(), first)


def test_rows_too_far_apart_are_refused(torch):
    c = Chunks(torch, "f16", 64, 1, 2, 16, [2], [30], seed=9)
    w = c.q.shape[1]
    far = torch.empty((1 << 32) + 2 * w, device="cuda").as_strided((2, w), ((1 << 32) + w, 1))  # w apart, modulo 2^32
    for q, out in ((far, c.out), (c.q, far)):
        with pytest.raises(ValueError):
            c.cache.attention(0, c.batch, q, c.n_head, out, ws=c.ws)
