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
