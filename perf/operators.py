"""The paged key/value cache: its operators in plain torch and as the framework's own calls.

Three operators share one cache. A cache is a pair of pools k, v [layer][page][kv head][position in page][hd]; a
sequence is a row of a block table that names its pages in order, and a call takes new tokens of several
sequences at once: sequence s owns the rows cu_q[s] .. cu_q[s + 1] of the activations, and they are the last
positions of its kv_len[s].

  append     rows of a q|k|v projection: RMSNorm of every q and k head (optional), rotary positions (half or
             interleaved pairs, the first n_rot elements of a head), q to an output, k and v into the pages
  attention  softmax(scale q k^T) v of every row over its sequence's pages: causal, optionally with a sliding
             window and a few first positions that stay visible
  pages      copies of whole pages in every layer of the pools (what forking and compacting sequences cost)

Activations are 32-bit; the pools hold 32 or 16 bits.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16}
EPS = 1e-6
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eahmmf_inference_prototype_v-0.1.0_b200")


# ---- cases ---------------------------------------------------------------------------------------------------
def _attention(name, heads, kv, hd, page, type, n_seq, q, length, window=0, sinks=0, lens=1):
    return dict(name=name, op="attention", n_head=heads, n_kv=kv, hd=hd, page=page, type=type, n_seq=n_seq,
                q_lo=q[0], q_hi=q[1], kv_lo=length[0], kv_hi=length[1], window=window, sinks=sinks, lens=lens)


def _append(name, heads, kv, hd, page, type, n_seq, q, length, style, n_rot, norm, lens=1):
    return dict(name=name, op="append", n_head=heads, n_kv=kv, hd=hd, page=page, type=type, n_seq=n_seq,
                q_lo=q[0], q_hi=q[1], kv_lo=length[0], kv_hi=length[1], style=style, n_rot=n_rot, norm=norm, lens=lens)


def _pages(name, layers, kv, hd, page, type, copies):
    return dict(name=name, op="pages", n_layer=layers, n_kv=kv, hd=hd, page=page, type=type, copies=copies)


def listed():
    return [
        # one sequence's next token early in an answer: launch and load latency
        _attention("step_one", 32, 4, 128, 16, "f16", 1, (1, 1), (201, 201)),
        # a batch of 32 sequences, each at its own length: one decode step of the batch
        _attention("step_batch", 32, 4, 128, 64, "f16", 32, (1, 1), (300, 4500), lens=2),
        # two long documents: the length split over the whole GPU
        _attention("step_long", 32, 4, 128, 64, "f16", 2, (1, 1), (127000, 131003), lens=3),
        # the same step over the cache kept in 32 bits
        _attention("step_batch_f32", 32, 4, 128, 32, "f32", 32, (1, 1), (200, 2050), lens=4),
        # small heads, a window over long sequences, four first positions kept
        _attention("step_window", 16, 8, 64, 16, "f16", 64, (1, 1), (900, 9000), window=1024, sinks=4, lens=5),
        # the engine's largest prompt pass (64 tokens) over a 32-bit cache
        _attention("pass_f32", 32, 4, 128, 64, "f32", 1, (64, 64), (2111, 2111)),
        # chunks of prompts beside single tokens, 16 heads to a kv head
        _attention("mixed", 64, 4, 128, 64, "f16", 8, (1, 513), (100, 6000), lens=7),
        # a long prompt's chunk over what is cached of it
        _attention("prompt", 32, 4, 128, 64, "f16", 1, (4096, 4096), (12289, 12289)),
        # one decode step's rows into the pages
        _append("append_step", 32, 4, 128, 64, "f16", 32, (1, 1), (300, 4500), "half", 128, True, lens=2),
        # a prompt chunk's rows, interleaved pairs over half of each head
        _append("append_prompt", 32, 4, 128, 64, "f32", 3, (1200, 1500), (1500, 40000), "interleaved", 64, False, lens=9),
        # forks of a few sequences: their last, part-filled pages in all 48 layers
        _pages("fork", 48, 4, 128, 16, "f16", 7),
        # compacting a pool
        _pages("compact", 8, 4, 128, 64, "f16", 501),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv = rng.choice([2, 4, 8])
    group = rng.choice([1, 2, 4, 7, 8, 16])
    hd = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    type = rng.choice(["f16", "f16", "f32"])
    kind = rng.choice(["step", "step", "chunk", "chunk", "append", "pages"])
    if kind == "pages":
        copies, layers = _log(rng, 1, 600), rng.randint(1, 48)
        copies = max(1, min(copies, int(4e8 / (layers * kv * hd * page * 4))))
        return dict(_pages("", layers, kv, hd, page, type, copies), **{}) | {"lens": rng.randrange(1 << 20)}
    if kind == "append":
        n_seq = _log(rng, 1, 64)
        q_hi = 1 if rng.random() < 0.3 else _log(rng, 2, max(2, 6000 // n_seq))
        most = int(1e8 / (n_seq * kv * hd))
        kv_lo = _log(rng, 1, most // 2)
        c = _append("", kv * group, kv, hd, page, type, n_seq, (1, q_hi), (kv_lo, kv_lo + _log(rng, 1, most // 2)),
                    rng.choice(["half", "interleaved"]), 2 * rng.randint(4, hd // 2), rng.random() < 0.5)
    else:
        if kind == "step":
            n_seq, q_hi = _log(rng, 1, 128), 1
            most = int(2.6e5 * 4 * 128 / (n_seq * kv * hd))
        else:
            n_seq = _log(rng, 1, 8)
            q_hi = _log(rng, 2, (256 if type == "f32" else 2048) // n_seq)
            most = int(min(20000, 1.2e9 / (n_seq * q_hi * kv * group)))
        kv_hi = _log(rng, 20, max(21, most))
        w = rng.random() < 0.3
        c = _attention("", kv * group, kv, hd, page, type, n_seq, (1, q_hi), (max(1, kv_hi // _log(rng, 1, 16)), kv_hi),
                       window=_log(rng, 1, 4000) if w else 0, sinks=rng.choice([0, 1, 4, 70]) if w else 0)
    c["lens"] = rng.randrange(1 << 20)
    return c


def _lengths(case):
    """(new tokens, cached positions with them) of each sequence: a function of the case alone."""
    r = random.Random(case["lens"])
    q, kv = [], []
    for s in range(case["n_seq"]):
        n = case["q_hi"] if s == 0 else r.randint(case["q_lo"], case["q_hi"])
        q.append(n)
        kv.append(max(n, case["kv_hi"] if s == 0 else _log(r, case["kv_lo"], case["kv_hi"])))
    return q, kv


def _positions(case):
    """Positions of every row, as a flat list."""
    q, kv = _lengths(case)
    return [k - n + i for n, k in zip(q, kv) for i in range(n)]


# ---- inputs --------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(DEV)
    g.manual_seed(seed)
    dt, hd, n_kv, page = TYPES[case["type"]], case["hd"], case["n_kv"], case["page"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    st = {"case": case}
    if case["op"] == "pages":
        n, order = case["copies"], np.random.default_rng(seed)
        n_pages = 2 * n + 5
        st["k"], st["v"] = (randn(case["n_layer"], n_pages, n_kv, page, hd, dtype=dt) for _ in range(2))
        ids = order.permutation(n_pages)[: 2 * n]
        st["pairs"] = np.ascontiguousarray(np.stack([ids[:n], ids[n:]], 1).astype(np.int32))  # (from, to), on the host
        if own:
            st["cache"] = _framework().PagedCache(st["k"], st["v"])
        return st
    q_len, kv_len = _lengths(case)
    n_seq, n_head = case["n_seq"], case["n_head"]
    need = [-(-k // page) for k in kv_len]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)  # pages of a pool in use lie anywhere
    table = np.full((n_seq, max(need)), -1, np.int64)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = np.arange(at, at + n)
        at += n
    idx = torch.from_numpy(table).to(DEV)
    st["table"] = torch.where(idx >= 0, ids[idx.clamp(min=0)], torch.full_like(idx, -1, dtype=torch.int32)).contiguous()
    st["cu_q"] = torch.tensor([0] + list(np.cumsum(q_len)), dtype=torch.int32, device=DEV)
    st["kv_len"] = torch.tensor(kv_len, dtype=torch.int32, device=DEV)
    rows = sum(q_len)
    st["k"], st["v"] = (randn(1, n_pages, n_kv, page, hd, dtype=dt) for _ in range(2))
    st["out"] = torch.zeros(rows, n_head * hd, device=DEV)
    if case["op"] == "append":
        st["qkv"] = randn(rows, (n_head + 2 * n_kv) * hd)
        n_rot = case["n_rot"]
        st["inv_freq"] = torch.tensor([1e6 ** (-2.0 * i / n_rot) for i in range(n_rot // 2)], dtype=torch.float64).float().to(DEV)
        st["q_norm"], st["k_norm"] = (1 + 0.2 * randn(hd), 1 + 0.2 * randn(hd)) if case["norm"] else (None, None)
    else:
        st["q"] = randn(rows, n_head * hd) * 3.0  # scores of a spread that lets some positions stand out
    if own:
        eb = _framework()
        st["cache"] = eb.PagedCache(st["k"], st["v"])
        st["batch"] = eb.PagedBatch(st["table"], st["cu_q"], st["kv_len"], rows, max(q_len), max(kv_len))
        if case["op"] == "attention":
            st["ws"] = st["cache"].attention_workspace(st["batch"], n_head)
        else:
            st["rope"] = eb.Rope(st["inv_freq"], case["style"])
    return st


def _framework():
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import eahmmf_b200
    return eahmmf_b200


# ---- one pass ------------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        if op == "pages":
            st["cache"].copy_pages(st["pairs"])
            return st["k"], st["v"]
        if op == "append":
            st["cache"].append(0, st["batch"], st["qkv"], st["case"]["n_head"], st["rope"], st["out"], st["q_norm"],
                               st["k_norm"], EPS)
            return st["out"], st["k"], st["v"]
        st["cache"].attention(0, st["batch"], st["q"], st["case"]["n_head"], st["out"], window=st["case"]["window"],
                              n_sink=st["case"]["sinks"], ws=st["ws"])
        return st["out"]
    return {"pages": _plain_pages, "append": _plain_append, "attention": _plain_attention}[op](st)


def _plain_pages(st):
    p = torch.from_numpy(st["pairs"]).to(DEV).long()
    st["k"][:, p[:, 1]] = st["k"][:, p[:, 0]]
    st["v"][:, p[:, 1]] = st["v"][:, p[:, 0]]
    return st["k"], st["v"]


def _rows(st):
    """Sequence and position of every row."""
    cu, n = st["cu_q"].long(), st["out"].shape[0]
    r = torch.arange(n, device=DEV)
    seq = torch.searchsorted(cu, r, right=True) - 1
    return seq, st["kv_len"].long()[seq] - cu[seq + 1] + r


def _plain_append(st):
    c = st["case"]
    hd, n_head, n_kv, n_rot = c["hd"], c["n_head"], c["n_kv"], c["n_rot"]
    seq, pos = _rows(st)
    x = st["qkv"].view(-1, n_head + 2 * n_kv, hd)
    qk, v = x[:, : n_head + n_kv], x[:, n_head + n_kv:]
    if c["norm"]:
        w = torch.cat([st["q_norm"].expand(n_head, hd), st["k_norm"].expand(n_kv, hd)])
        qk = qk * (1.0 / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS)) * w
    ang = pos.double()[:, None] * st["inv_freq"].double()
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    h = n_rot // 2
    a, b = (qk[..., :h], qk[..., h:n_rot]) if c["style"] == "half" else (qk[..., 0:n_rot:2], qk[..., 1:n_rot:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    r = torch.cat([ra, rb], -1) if c["style"] == "half" else torch.stack([ra, rb], -1).flatten(-2)
    qk = torch.cat([r, qk[..., n_rot:]], -1)
    st["out"].copy_(qk[:, :n_head].reshape(st["out"].shape))
    page = st["table"][seq, pos // c["page"]].long()
    at = pos % c["page"]
    st["k"][0][page, :, at] = qk[:, n_head:].to(st["k"].dtype)
    st["v"][0][page, :, at] = v.to(st["v"].dtype)
    return st["out"], st["k"], st["v"]


def _plain_attention(st):
    c = st["case"]
    hd, n_head, n_kv, page, n_seq = c["hd"], c["n_head"], c["n_kv"], c["page"], c["n_seq"]
    q_most = c["q_hi"]
    seq, pos = _rows(st)
    at = torch.arange(st["out"].shape[0], device=DEV) - st["cu_q"].long()[seq]  # the row's place in its sequence
    n_pages = st["table"].shape[1]
    ids = st["table"].long().clamp(min=0)

    def gather(pool):  # [sequence][kv head][position][hd], sequences side by side up to the longest
        return pool[0][ids].float().permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, n_pages * page, hd)

    q = torch.zeros(n_seq, q_most, n_head, hd, device=DEV)
    q[seq, at] = st["q"].view(-1, n_head, hd)
    q = q.view(n_seq, q_most, n_kv, n_head // n_kv, hd).permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, -1, hd)
    s = torch.matmul(q, gather(st["k"]).transpose(-1, -2)) * (1.0 / math.sqrt(hd))
    p = torch.full((n_seq, q_most), -1, device=DEV, dtype=torch.int64)
    p[seq, at] = pos
    j = torch.arange(n_pages * page, device=DEV)
    see = j <= p[..., None]
    if c["window"]:
        see &= (j > p[..., None] - c["window"]) | (j < c["sinks"])
    s = s.view(n_seq, n_kv, q_most, n_head // n_kv, -1)
    s.masked_fill_(~see[:, None, :, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp(min=-1e30)
    s.exp_()
    s /= s.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(s.view(n_seq, n_kv, -1, n_pages * page), gather(st["v"]))
    o = o.view(n_seq, n_kv, q_most, n_head // n_kv, hd).permute(0, 2, 1, 3, 4)
    st["out"].copy_(o[seq, at].reshape(st["out"].shape))
    return st["out"]


# ---- from the definitions, in 64 bits, sequence by sequence -----------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    st = prepare(case, seed)
    own = was
    if case["op"] == "pages":
        k, v = st["k"].double(), st["v"].double()
        for a, b in st["pairs"].tolist():
            k[:, b], v[:, b] = st["k"][:, a].double(), st["v"][:, a].double()
        return k, v
    hd, n_head, n_kv, page = case["hd"], case["n_head"], case["n_kv"], case["page"]
    q_len, kv_len = _lengths(case)
    table = st["table"].tolist()
    out = torch.zeros(sum(q_len), n_head, hd, dtype=torch.float64, device=DEV)
    if case["op"] == "append":
        k, v = st["k"].double(), st["v"].double()
        n_rot = case["n_rot"]
        pos = torch.tensor(_positions(case), dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.ones_like(pos)[:, None], pos[:, None] * st["inv_freq"].double()[None])[:, None]
        x = st["qkv"].double().view(-1, n_head + 2 * n_kv, hd)
        q_all, k_all, v_all = x[:, :n_head], x[:, n_head:n_head + n_kv], x[:, n_head + n_kv:]
        got = []
        for y, w in ((q_all, st["q_norm"]), (k_all, st["k_norm"])):
            if w is not None:
                y = y * w.double() / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / hd + EPS)
            y = y.clone()
            first, second = (slice(0, n_rot // 2), slice(n_rot // 2, n_rot)) if case["style"] == "half" else (slice(0, n_rot, 2), slice(1, n_rot, 2))
            z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
            y[..., first], y[..., second] = z.real, z.imag
            got.append(y)
        out.copy_(got[0])
        where = [(table[s][p // page], p % page) for s, (n, m) in enumerate(zip(q_len, kv_len)) for p in range(m - n, m)]
        pg, at = (torch.tensor(w, device=DEV) for w in zip(*where))
        k[0][pg, :, at], v[0][pg, :, at] = got[1], v_all
        return out.view(st["out"].shape), k, v
    row = 0
    for s, (n, m) in enumerate(zip(q_len, kv_len)):
        pages = torch.tensor(table[s][: -(-m // page)], device=DEV)
        ks, vs = (st[x][0][pages].double().transpose(1, 2).reshape(-1, n_kv, hd)[:m] for x in "kv")
        j = torch.arange(m, device=DEV)
        for r0 in range(0, n, 256):
            r1 = min(n, r0 + 256)
            p = torch.arange(m - n + r0, m - n + r1, device=DEV)[:, None]
            hidden = j > p
            if case["window"]:
                hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
            for h in range(n_head):
                qh = st["q"].view(-1, n_head, hd)[row + r0:row + r1, h].double()
                sc = (qh @ ks[:, h * n_kv // n_head].T) / math.sqrt(hd)
                sc[hidden] = -math.inf
                out[row + r0:row + r1, h] = torch.softmax(sc, -1) @ vs[:, h * n_kv // n_head]
        row += n
    return out.view(st["out"].shape)


# ---- what a pass cannot do without ----------------------------------------------------------------------------
def work(case):
    es, hd, n_kv = (2 if case["type"] == "f16" else 4), case["hd"], case["n_kv"]
    if case["op"] == "pages":
        return {"bytes": 4.0 * case["copies"] * case["n_layer"] * n_kv * case["page"] * hd * es, "flops": 0.0}
    q_len, kv_len = _lengths(case)
    rows, n_head = sum(q_len), case["n_head"]
    if case["op"] == "append":
        return {"bytes": rows * hd * (4.0 * (2 * n_head + 2 * n_kv) + 2.0 * n_kv * es), "flops": 10.0 * rows * hd * (n_head + n_kv)}
    read = seen = 0
    w, sinks = case["window"], case["sinks"]
    for n, m in zip(q_len, kv_len):
        p = np.arange(m - n, m)
        if w:
            low = np.maximum(0, p - w + 1)
            seen += int((p + 1 - low + np.minimum(low, sinks)).sum())
            read += int(m - low[0] + min(low[0], sinks))
        else:
            seen += int((p + 1).sum())
            read += m
    return {"bytes": 2.0 * read * n_kv * hd * es + 8.0 * rows * n_head * hd, "flops": 4.0 * seen * n_head * hd}
