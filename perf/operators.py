"""The operators of batched serving, measured: appending to a paged KV cache,
attention over it (with and without a shared prefix) and sampling.

A case is a dict of plain values; ``kind`` picks the operator:

  append     q and k of a batch normalised per head and rotated, k and v stored
             into the pages of their sequences (DenseOps.kv_append)
  attention  every row of a batch against its own sequence's pages, up to its
             own position (DenseOps.paged_attention); ``prefix`` > 0: the first
             positions of all sequences lie in the same pages
  sample     one token per row of logits from given random numbers: temperature,
             top-k, top-p, min-p (DenseOps.sample)

A batch is ``seqs`` sequences of ``rows_lo`` to ``rows_hi`` new rows each behind
``past_lo`` to ``past_hi`` earlier positions, spread unevenly; ``pad`` more rows
stand behind the last sequence and are left as they were.  Pages are handed out
in a random order.  Values are what the path meets: projections of normed rows
N(0, 1), norm weights near 1, logits N(0, 2.5).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-5

# attention of the two model widths of the repository's own configurations
OLMOE = dict(heads=16, kv_heads=16, head_dim=128, theta=10000.0, norm=True)
MIXTRAL = dict(heads=32, kv_heads=8, head_dim=128, theta=1e6, norm=False)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- the cases ------------------------------------------------------------------------


def _append(name, model, seqs, rows, past, x, cache, page=16, rotary=None, pairs="half",
            stretch=1.0, pad=0):
    return dict(name=name, kind="append", **model, seqs=seqs, rows_lo=rows[0], rows_hi=rows[1],
                past_lo=past[0], past_hi=past[1], pad=pad, x=x, cache=cache, page=page,
                rotary=model["head_dim"] if rotary is None else rotary, pairs=pairs,
                stretch=stretch)


def _attention(name, model, seqs, rows, past, x, cache, page=16, prefix=0, pad=0):
    return dict(name=name, kind="attention", heads=model["heads"], kv_heads=model["kv_heads"],
                head_dim=model["head_dim"], seqs=seqs, rows_lo=rows[0], rows_hi=rows[1],
                past_lo=past[0], past_hi=past[1], pad=pad, x=x, cache=cache, page=page,
                prefix=prefix)


def listed():
    return [
        # one conversation's next token, f32 throughout as the decoder keeps it
        _append("append_one", OLMOE, 1, (1, 1), (200, 200), "f32", "f32"),
        # a step of 64 conversations, bf16 cache, positions stretched fourfold
        _append("append_step_64", MIXTRAL, 64, (1, 1), (100, 8000), "f32", "bf16", stretch=4.0),
        # the prompts of five conversations at once, ragged, half of each head rotated
        _append("append_prompts", MIXTRAL, 5, (37, 1900), (0, 3000), "bf16", "bf16", page=64,
                rotary=64, pairs="interleaved", pad=11),
        # one conversation's next token early on, f32 cache, multi-head
        _attention("attention_one", OLMOE, 1, (1, 1), (200, 200), "f32", "f32"),
        # a step of 32 conversations of very different lengths, grouped heads
        _attention("attention_step_32", MIXTRAL, 32, (1, 1), (60, 8100), "f32", "bf16"),
        # a step of 48 conversations, multi-head, all in bf16
        _attention("attention_step_48", OLMOE, 48, (1, 1), (100, 4000), "bf16", "bf16", page=64),
        # a long prompt from its start
        _attention("attention_prompt", MIXTRAL, 1, (2500, 2500), (0, 0), "bf16", "bf16", page=64),
        # turns of several chats, new rows behind a long past, f32 activations
        _attention("attention_turns", MIXTRAL, 6, (9, 400), (0, 4000), "f32", "bf16", pad=5),
        # a step of 64 conversations that share a long system prompt
        _attention("prefix_step_64", MIXTRAL, 64, (1, 1), (20, 600), "f32", "bf16", prefix=4096),
        # a few conversations behind a short one, multi-head, f32 cache, ragged turns
        _attention("prefix_turns_8", OLMOE, 8, (1, 30), (5, 300), "f32", "f32", page=32,
                   prefix=500),
        # one conversation's next token at the chat's defaults
        dict(name="sample_one", kind="sample", rows=1, vocab=50304, sigma=2.5, mix=False, ties=False),
        # a step of 64 conversations, each with settings of its own, many equal logits
        dict(name="sample_step_64", kind="sample", rows=64, vocab=50304, sigma=2.5, mix=True,
             ties=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _model(rng):
    heads, kv = rng.choice([(16, 16), (32, 8), (32, 8), (8, 1), (24, 8), (12, 4), (7, 7), (40, 8)])
    hd = rng.choice([64, 128, 128, 256])
    if heads * hd > 8192:
        hd = 128
    return dict(heads=heads, kv_heads=kv, head_dim=hd, theta=rng.choice([10000.0, 1e6]),
                norm=rng.random() < 0.5)


def _types(rng):
    return rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])


def draw(rng):
    kind = rng.choice(["append", "append", "step", "step", "turns", "prefix", "prefix", "sample",
                       "sample"])
    if kind == "sample":
        rows = _log_int(rng, 1, 64)
        return dict(kind=kind, rows=rows, vocab=_log_int(rng, 1000, min(150000, 3200000 // rows)),
                    sigma=rng.choice([1.0, 2.5, 6.0]), mix=rng.random() < 0.7,
                    ties=rng.random() < 0.4)
    m, (x, cache) = _model(rng), _types(rng)
    page = rng.choice([8, 16, 16, 32, 64, 256])
    # (a position's bytes over those of the widest listed case bound the lengths)
    wide = max(1.0, m["kv_heads"] * m["head_dim"] * (4 if cache == "f32" else 2) / 2048.0)
    if kind == "append":
        seqs = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, max(1, 3000 // seqs))
        past = _log_int(rng, 1, 6000)
        c = _append("", m, seqs, (rng.randint(1, hi), hi), (rng.randint(0, past), past), x, cache,
                    page, rng.choice([m["head_dim"], m["head_dim"], m["head_dim"] // 2, 32]),
                    rng.choice(["half", "interleaved"]), rng.choice([1.0, 1.0, 4.0, 8.0]),
                    rng.choice([0, 0, 3]))
    elif kind == "step":
        seqs = _log_int(rng, 1, 40)
        past = _log_int(rng, 16, max(64, int(min(8000, 160000 / seqs / wide))))
        c = _attention("", m, seqs, (1, 1), (rng.randint(0, past), past), x, cache, page)
    elif kind == "turns":
        seqs = _log_int(rng, 1, 6)
        hi = _log_int(rng, 2, 1000 // seqs)
        past = _log_int(rng, 1, int(3000 / wide))
        c = _attention("", m, seqs, (rng.randint(1, hi), hi), (0, past), x, cache, page,
                       pad=rng.choice([0, 7]))
    else:
        seqs = _log_int(rng, 2, 48)
        hi = _log_int(rng, 1, max(1, 64 // seqs))
        past = _log_int(rng, 4, int(500 / wide) + 4)
        c = _attention("", m, seqs, (1, hi), (rng.randint(0, past), past), x, cache, page,
                       prefix=_log_int(rng, 32, int(3500 / wide)))
    del c["name"]
    return c


# ---- the batch ------------------------------------------------------------------------


def _spread(n, lo, hi, turn):
    """n whole numbers in [lo, hi], unevenly spread, both ends among them (n > 1)."""
    f = [(0.5 + 0.6180339887 * (i + turn)) % 1.0 for i in range(n)]
    v = [lo + int(round((hi - lo) * t * t)) for t in f]
    v[turn % n] = hi
    if n > 1:
        v[(turn + 1) % n] = lo
    return v


def _batch(c):
    """(new rows, positions after them) of each sequence."""
    rows = _spread(c["seqs"], c["rows_lo"], c["rows_hi"], 0)
    past = _spread(c["seqs"], c["past_lo"], c["past_hi"], 3)
    return rows, [r + p + c.get("prefix", 0) for r, p in zip(rows, past)]


def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + stream)
    return g


def _normal(shape, seed, stream, sigma=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=_gen(seed, stream), device=DEV) * sigma).to(dtype)


def _plan(c, seed):
    """row_start, kv_len, the sequences' pages (the prefix' pages first) and the
    number of pages there are."""
    rows, length = _batch(c)
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    ps, prefix = c["page"], c.get("prefix", 0)
    need = [-(-n // ps) for n in length]
    full = prefix // ps    # pages wholly of the prefix are shared, one in part is each one's own
    total = full + sum(n - full for n in need) + 3
    # (the one page that the prefix ends in: a copy of it for the prefix itself)
    total += 1
    order = torch.randperm(total, generator=_gen(seed, 50), device=DEV).cpu().numpy()
    table = np.zeros((c["seqs"], max(need)), np.int32)
    at = full
    for s, n in enumerate(need):
        table[s, :full] = order[:full]
        table[s, full:n] = order[at:at + n - full]
        at += n - full
    # the prefix' own table: its last, partial page is the first sequence's
    own_table = table[0, :-(-prefix // ps)].copy() if prefix else np.zeros(1, np.int32)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)
    return dev(start), dev(length), dev(table), dev(own_table), total, int(start[-1])


def _cache(c, seed, pages, table):
    shape = (pages, c["page"], c["kv_heads"], c["head_dim"])
    k = _normal(shape, seed, 2, 1.0, DTYPES[c["cache"]])
    v = _normal(shape, seed, 3, 1.0, DTYPES[c["cache"]])
    ps, prefix = c["page"], c.get("prefix", 0)
    if prefix % ps:   # every sequence's copy of the page that the prefix ends in holds the same there
        at, n = table[:, prefix // ps].long(), prefix % ps
        for t in (k, v):
            t[at, :n] = t[at[:1], :n].clone()
    return k, v


def _frequencies(c):
    """theta^(-2 i / rotary) with the slow pairs' angles divided by ``stretch``:
    wavelengths over a quarter of 2048 positions stretched, those under a
    thirty-second kept, blended between; and the amplitude that goes with it."""
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64)
    f = c["theta"] ** (-2.0 * i / c["rotary"])
    if c["stretch"] == 1.0:
        return f.float().to(DEV), 1.0
    turns = 2048.0 * f / (2.0 * math.pi)
    keep = ((turns - 4.0) / 28.0).clamp(0.0, 1.0)
    return (f * keep + f / c["stretch"] * (1.0 - keep)).float().to(DEV), \
        0.1 * math.log(c["stretch"]) + 1.0


def _sample_inputs(c, seed):
    rows, V = c["rows"], c["vocab"]
    stride = (V + 3) // 4 * 4
    logits = _normal((rows, stride), seed, 1, c["sigma"])
    if c["ties"]:   # as logits that went through bf16
        logits = logits.to(torch.bfloat16).float()
    u = torch.rand((rows,), generator=_gen(seed, 2), device=DEV)
    full = torch.full((rows,), 1.0, device=DEV)
    if not c["mix"]:
        return logits, u, 0.7 * full, (0 * full).int(), 0.9 * full, 0 * full
    g = _gen(seed, 3)
    pick = torch.rand((5, rows), generator=g, device=DEV)
    temp = 0.2 + 1.3 * pick[0]
    temp[pick[1] < 0.15] = 0.0
    k = torch.exp(pick[2] * math.log(min(V, 2000))).int()
    k[pick[1] > 0.6] = 0
    p = torch.where(pick[3] < 0.3, full, 0.3 + 0.69 * pick[3])
    m = torch.where(pick[4] < 0.5, 0 * full, 0.2 * (pick[4] - 0.5))
    return logits, u, temp, k, p, m


def prepare(case, seed):
    c = case
    if c["kind"] == "sample":
        logits, u, temp, k, p, m = _sample_inputs(c, seed)
        rows = c["rows"]
        return dict(case=c, logits=logits, u=u, temp=temp, k=k, p=p, m=m,
                    tokens=torch.zeros((rows,), dtype=torch.int32, device=DEV),
                    probs=torch.zeros((rows,), device=DEV))
    start, length, table, prefix_table, pages, rows = _plan(c, seed)
    kc, vc = _cache(c, seed, pages, table)
    n, hd = rows + c["pad"], c["head_dim"]
    qd, kvd = c["heads"] * hd, c["kv_heads"] * hd
    st = dict(case=c, start=start, length=length, table=table, kc=kc, vc=vc, rows=rows,
              prefix_table=prefix_table)
    if c["kind"] == "append":   # the projections' rows, q, k and v side by side
        st["qkv"] = _normal((n, qd + 2 * kvd), seed, 1, 1.0, DTYPES[c["x"]])
        st["qw"] = (1 + _normal((hd,), seed, 4, 0.1)).to(torch.bfloat16)
        st["kw"] = (1 + _normal((hd,), seed, 5, 0.1)).to(torch.bfloat16)
        st["freq"], st["amp"] = _frequencies(c)
        st["out"] = torch.zeros((n, qd), dtype=DTYPES[c["x"]], device=DEV)
    else:
        st["q"] = _normal((n, qd), seed, 1, 1.0, DTYPES[c["x"]])
        st["out"] = torch.zeros((n, qd), dtype=DTYPES[c["x"]], device=DEV)
    return st


# ---- one pass: the plain forms ---------------------------------------------------------


def _places(st):
    """Sequence and position of every row of the batch (not of the padding)."""
    start, length = st["start"].long(), st["length"].long()
    row = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(start, row, right=True) - 1
    return seq, length[seq] - (start[seq + 1] - row)


def _rotate(x, cos, sin, pairs):
    """x [rows, heads, head_dim]: the first 2 * cos.shape[1] dims of each head."""
    h = cos.shape[1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if pairs == "half":
        a, b, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
    a, b, rest = x[..., 0:2 * h:2], x[..., 1:2 * h:2], x[..., 2 * h:]
    both = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((both, rest), -1)


def _plain_append(st):
    c = st["case"]
    hd, hq, hk = c["head_dim"], c["heads"], c["kv_heads"]
    seq, pos = _places(st)
    x = st["qkv"][:st["rows"]].float()
    q = x[:, :hq * hd].reshape(-1, hq, hd)
    k = x[:, hq * hd:(hq + hk) * hd].reshape(-1, hk, hd)
    v = x[:, (hq + hk) * hd:].reshape(-1, hk, hd)
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * st["qw"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * st["kw"].float()
    angle = pos.double()[:, None] * st["freq"].double()[None, :]
    cos, sin = (angle.cos() * st["amp"]).float(), (angle.sin() * st["amp"]).float()
    q, k = _rotate(q, cos, sin, c["pairs"]), _rotate(k, cos, sin, c["pairs"])
    page, slot = st["table"].long()[seq, pos // c["page"]], pos % c["page"]
    st["kc"][page, slot] = k.to(st["kc"].dtype)
    st["vc"][page, slot] = v.to(st["vc"].dtype)
    st["out"][:st["rows"]] = q.reshape(-1, hq * hd).to(st["out"].dtype)
    return st["out"], st["kc"], st["vc"]


def _plain_attention(st):
    c = st["case"]
    hd, hk = c["head_dim"], c["kv_heads"]
    share, B = c["heads"] // hk, c["seqs"]
    rows, length = _batch(c)
    R, L = max(rows), max(length)
    start, kv = st["start"].long(), st["length"].long()
    n = start[1:] - start[:-1]
    # every sequence's positions, padded to the longest (its own last one again)
    at = torch.minimum(torch.arange(L, device=DEV)[None, :], kv[:, None] - 1)
    page = st["table"].long().gather(1, at // c["page"])
    k = st["kc"][page, at % c["page"]].float().permute(0, 2, 3, 1).contiguous()
    v = st["vc"][page, at % c["page"]].float().permute(0, 2, 1, 3).contiguous()
    # and its rows
    i = torch.minimum(torch.arange(R, device=DEV)[None, :], n[:, None] - 1)
    q = st["q"][start[:-1, None] + i].float().reshape(B, R, hk, share, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(B, hk, R * share, hd)
    s = torch.matmul(q, k) * (1.0 / math.sqrt(hd))
    pos = (kv[:, None] - n[:, None] + i).repeat_interleave(share, 1)
    hide = torch.arange(L, device=DEV)[None, None, :] > pos[:, :, None]
    s.masked_fill_(hide[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.reshape(B, hk, R, share, hd).permute(0, 2, 1, 3, 4).reshape(B, R, -1)
    real = torch.arange(R, device=DEV)[None, :] < n[:, None]
    st["out"][:st["rows"]] = o[real].to(st["out"].dtype)
    return st["out"]


def _plain_sample(st):
    c = st["case"]
    x = st["logits"][:, :c["vocab"]].double()
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    rank = torch.arange(c["vocab"], device=DEV)[None, :]
    first = rank == 0
    t = st["temp"].double()[:, None]
    w = ((x - x[:, :1]) / torch.where(t > 0, t, 1.0)).exp()
    w = torch.where(t > 0, w, first.double())
    k = st["k"].long()[:, None]
    w = w * ((rank < k) | (k <= 0))
    cum = w.cumsum(1)
    p = st["p"].double()[:, None]
    keep = first | ((((cum - w) < p * cum[:, -1:]) | (p >= 1)) & (w >= st["m"].double()[:, None]) & (w > 0))
    w = w * keep
    total = w.sum(1, keepdim=True)
    n = (w.cumsum(1) < st["u"].double()[:, None] * total).sum(1, keepdim=True)
    n = torch.minimum(n, keep.sum(1, keepdim=True) - 1)
    return order.gather(1, n)[:, 0].int(), (w.gather(1, n) / total)[:, 0].float()


# ---- one pass: the framework's operators -----------------------------------------------

_ops = None


def _dense_ops():
    """The program's one context (the operators need its stream and workspace)."""
    global _ops
    if _ops is None:
        from m1moe_amd import DenseOps, HIPContext, make_shape
        _ops = DenseOps(HIPContext(make_shape(64, 1, 1, 64)))
    return _ops


def _handles(st):
    """What a program keeps of a batch: the descriptions of its cache and rows."""
    if "handles" not in st:
        from m1moe_amd import KVAppend, PagedBatch, PagedKV, SampleParams
        c = st["case"]
        if c["kind"] == "sample":
            st["handles"] = SampleParams.make(st["u"].data_ptr(), st["temp"].data_ptr(),
                                              st["k"].data_ptr(), st["p"].data_ptr(),
                                              st["m"].data_ptr())
            return st["handles"]
        prefix = c.get("prefix", 0)
        kv = PagedKV.make(st["kc"].data_ptr(), st["vc"].data_ptr(), c["cache"], st["kc"].shape[0],
                          c["page"], c["kv_heads"], c["head_dim"])
        batch = PagedBatch.make(c["seqs"], st["out"].shape[0], st["start"].data_ptr(),
                                st["length"].data_ptr(), st["table"].data_ptr(),
                                st["table"].shape[1], prefix,
                                st["prefix_table"].data_ptr() if prefix else None)
        st["handles"] = (kv, batch)
        if c["kind"] == "append":
            size, hd = st["qkv"].element_size(), c["head_dim"]
            at, n = st["qkv"].data_ptr(), st["qkv"].shape[1]
            qd, kvd = c["heads"] * hd, c["kv_heads"] * hd
            st["handles"] += (KVAppend.make(
                c["x"], c["heads"], at, at + qd * size, at + (qd + kvd) * size, n, n, n,
                st["out"].data_ptr(), qd,
                st["qw"].data_ptr() if c["norm"] else None,
                st["kw"].data_ptr() if c["norm"] else None, EPS, c["rotary"],
                c["pairs"] == "interleaved", st["freq"].data_ptr(), st["amp"]),)
    return st["handles"]


def run(state):
    st, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention,
                "sample": _plain_sample}[c["kind"]](st)
    ops, h = _dense_ops(), st.get("handles") or _handles(st)
    if c["kind"] == "append":
        ops.kv_append(*h)
        return st["out"], st["kc"], st["vc"]
    if c["kind"] == "attention":
        qd = st["q"].shape[1]
        ops.paged_attention(h[0], h[1], st["q"].data_ptr(), qd, st["out"].data_ptr(), qd, c["x"],
                            c["heads"])
        return st["out"]
    ops.sample(st["logits"].data_ptr(), c["rows"], c["vocab"], st["logits"].shape[1], h,
               st["tokens"].data_ptr(), st["probs"].data_ptr())
    return st["tokens"], st["probs"]


# ---- what a pass cannot do without -----------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "sample":
        return {"bytes": 4.0 * c["rows"] * c["vocab"] + 28.0 * c["rows"],
                "flops": 4.0 * c["rows"] * c["vocab"]}
    rows, length = _batch(c)
    qd, kvd = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    xb, cb = (4 if c["x"] == "f32" else 2), (4 if c["cache"] == "f32" else 2)
    n = float(sum(rows))
    if c["kind"] == "append":
        return {"bytes": n * (2 * qd * xb + 2 * kvd * (xb + cb)), "flops": n * 8.0 * (qd + kvd)}
    prefix = c["prefix"]
    pairs = sum(r * (k - r) + r * (r + 1) / 2.0 for r, k in zip(rows, length))
    seen = prefix + sum(k - prefix for k in length)
    return {"bytes": 2.0 * seen * kvd * cb + 2.0 * n * qd * xb, "flops": 4.0 * pairs * qd}


# ---- the same in 64 bits ---------------------------------------------------------------


def _exact_append(c, seed):
    start, length, table, _, pages, rows = _plan(c, seed)
    kc, vc = _cache(c, seed, pages, table)
    st = prepare(c, seed)
    out, kc, vc = st["out"].double(), kc.double(), vc.double()
    x, hd, hq, hk = st["qkv"].double(), c["head_dim"], c["heads"], c["kv_heads"]
    half, ps = c["rotary"] // 2, c["page"]
    # pair i of a head: dims (i, i + half) or (2 i, 2 i + 1)
    first = torch.arange(half, device=DEV) * (1 if c["pairs"] == "half" else 2)
    second = first + (half if c["pairs"] == "half" else 1)
    start, length, tab = start.tolist(), length.tolist(), table.long()

    def turn(y, w, at):
        if c["norm"]:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = y.clone()
        a = torch.polar(torch.full_like(at, st["amp"]), at)[:, None, :]
        r = torch.complex(y[..., first], y[..., second]) * a
        z[..., first], z[..., second] = r.real, r.imag
        return z
    for s in range(c["seqs"]):
        lo, hi = start[s], start[s + 1]
        p = torch.arange(length[s] - (hi - lo), length[s], device=DEV)
        at = p.double()[:, None] * st["freq"].double()
        blk = x[lo:hi].reshape(hi - lo, hq + 2 * hk, hd)
        out[lo:hi] = turn(blk[:, :hq], st["qw"], at).reshape(hi - lo, -1)
        where = tab[s][torch.div(p, ps, rounding_mode="floor")]
        kc[where, p % ps] = turn(blk[:, hq:hq + hk], st["kw"], at)
        vc[where, p % ps] = blk[:, hq + hk:]
    return out, kc, vc


def _exact_attention(c, seed):
    st = prepare(c, seed)
    hd, share, ps = c["head_dim"], c["heads"] // c["kv_heads"], c["page"]
    out = st["out"].double()
    start, length, tab = st["start"].tolist(), st["length"].tolist(), st["table"].long()
    for s in range(c["seqs"]):
        lo, hi, n = start[s], start[s + 1], length[s]
        p = torch.arange(n, device=DEV)
        k = st["kc"][tab[s][torch.div(p, ps, rounding_mode="floor")], p % ps].double()
        v = st["vc"][tab[s][torch.div(p, ps, rounding_mode="floor")], p % ps].double()
        mine = torch.arange(n - (hi - lo), n, device=DEV)
        for g in range(c["kv_heads"]):
            kt, vg = k[:, g].t().contiguous(), v[:, g].contiguous()
            for h in range(g * share, (g + 1) * share):
                e = (st["q"][lo:hi, h * hd:(h + 1) * hd].double() @ kt) / math.sqrt(hd)
                e = torch.where(p[None, :] <= mine[:, None], e, -math.inf)
                out[lo:hi, h * hd:(h + 1) * hd] = torch.softmax(e, 1) @ vg
    return out


def _exact_sample(c, seed):
    logits, u, temp, top_k, top_p, min_p = (a.cpu().numpy() for a in _sample_inputs(c, seed))
    tokens, probs = [], []
    for r in range(c["rows"]):
        x = logits[r, :c["vocab"]].astype(np.float64)
        order = np.argsort(-x, kind="stable")
        if not temp[r] > 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        if top_k[r] > 0:
            order = order[:top_k[r]]
        w = np.exp((x[order] - x[order[0]]) / np.float64(temp[r]))
        run_sum = np.cumsum(w)
        n = len(w)
        if top_p[r] < 1:
            n = min(n, int(np.searchsorted(run_sum, np.float64(top_p[r]) * run_sum[-1])) + 1)
        n = max(1, min(n, int(np.count_nonzero(w >= np.float64(min_p[r])))))
        i = min(int(np.searchsorted(run_sum[:n], np.float64(u[r]) * run_sum[n - 1])), n - 1)
        tokens.append(int(order[i]))
        probs.append(float(w[i] / run_sum[n - 1]))
    return (torch.tensor(tokens, dtype=torch.int32, device=DEV),
            torch.tensor(probs, dtype=torch.float64, device=DEV))


def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention,
            "sample": _exact_sample}[case["kind"]](case, seed)
