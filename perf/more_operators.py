"""The operators of steps over drafted tokens, measured: the plan of a batch of
token trees, appending a tree's rows to a paged KV cache, attention in which a
drafted token sees the conversation and its own ancestors, taking over the tokens
that the model agrees with, and products with 4-bit weights.

A case is a dict of plain values; ``kind`` picks the operator:

  plan       parents of the drafted tokens -> who sees whom, and depths
             (DenseOps.tree_plan)
  append     q and k normalised and rotated by the position of their depth, k and
             v stored row by row behind the conversation (DenseOps.tree_append)
  attention  every drafted token against its conversation's positions, its
             ancestors and itself (DenseOps.tree_attention); ``prefix`` > 0: the
             first positions of all sequences lie in the same pages
  accept     the path of drafts that equal the tokens drawn at their parents, and
             its rows of all layers' caches moved together (DenseOps.tree_accept)
  q4         y = x W^T (+ residual), W in 4 bits with a scale and a bias per group
             of columns (DenseOps.matmul_q4)

A batch is ``seqs`` trees of ``nodes_lo`` to ``nodes_hi`` tokens behind ``past_lo``
to ``past_hi`` positions, spread unevenly; row 0 of a tree is the last token that
is certain, every other row hangs on an earlier one.  ``pad`` more rows stand
behind the last tree.  Pages are handed out in a random order.  Values are what
the path meets: projections of normed rows N(0, 1), norm weights near 1; weights in
4 bits as a quantizer makes them of normal ones.
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


def _trees(name, kind, seqs, nodes, past=(0, 0), pad=0, **more):
    return dict(name=name, kind=kind, seqs=seqs, nodes_lo=nodes[0], nodes_hi=nodes[1],
                past_lo=past[0], past_hi=past[1], pad=pad, **more)


def _append(name, model, seqs, nodes, past, x, cache, page=16, rotary=None, pairs="half", pad=0):
    return _trees(name, "append", seqs, nodes, past, pad, **model, x=x, cache=cache, page=page,
                  rotary=model["head_dim"] if rotary is None else rotary, pairs=pairs)


def _attention(name, model, seqs, nodes, past, x, cache, page=16, prefix=0, pad=0):
    return _trees(name, "attention", seqs, nodes, past, pad, heads=model["heads"],
                  kv_heads=model["kv_heads"], head_dim=model["head_dim"], x=x, cache=cache,
                  page=page, prefix=prefix)


def _accept(name, model, seqs, nodes, past, cache, layers, page=16, pad=0):
    return _trees(name, "accept", seqs, nodes, past, pad, kv_heads=model["kv_heads"],
                  head_dim=model["head_dim"], cache=cache, page=page, layers=layers)


def _q4(name, tokens, rows, cols, x, y, group=64, residual=False, pad=0):
    return dict(name=name, kind="q4", tokens=tokens, rows=rows, cols=cols, group=group, x=x, y=y,
                residual=residual, pad=pad)


def listed():
    return [
        # one conversation's tree of drafts
        _trees("plan_one", "plan", 1, (26, 26)),
        # a step of 64 conversations with trees of any size
        _trees("plan_64", "plan", 64, (1, 64), pad=5),
        # one conversation's tree behind a short past, f32 throughout
        _append("append_tree_one", OLMOE, 1, (26, 26), (200, 200), "f32", "f32"),
        # a step of 32 conversations, bf16 throughout, half of each head rotated
        _append("append_tree_32", MIXTRAL, 32, (8, 64), (60, 8000), "bf16", "bf16", page=64,
                rotary=64, pairs="interleaved", pad=3),
        # one conversation's tree, multi-head, f32 cache
        _attention("tree_one", OLMOE, 1, (26, 26), (700, 700), "f32", "f32"),
        # a step of 32 conversations of very different lengths, grouped heads
        _attention("tree_step_32", MIXTRAL, 32, (8, 64), (60, 8100), "f32", "bf16"),
        # large trees behind a long system prompt that all share, multi-head, all in bf16
        _attention("tree_prefix_24", OLMOE, 24, (1, 100), (20, 600), "bf16", "bf16", page=64,
                   prefix=4096, pad=3),
        # what one conversation keeps of its drafts, 16 layers
        _accept("accept_one", OLMOE, 1, (26, 26), (200, 200), "f32", 16),
        # what 32 conversations keep, 32 layers
        _accept("accept_32", MIXTRAL, 32, (8, 64), (20, 200), "bf16", 32),
        # one token through an output projection, onto the residual
        _q4("q4_one", 1, 2048, 2048, "f32", "f32", residual=True),
        # a tree's logits over the whole vocabulary
        _q4("q4_head", 26, 50304, 2048, "bf16", "f32"),
        # the rows of many trees through the projections of q, k and v
        _q4("q4_batch", 800, 6144, 4096, "f32", "f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _model(rng):
    heads, kv = rng.choice([(16, 16), (32, 8), (32, 8), (8, 1), (20, 4), (12, 4), (7, 7), (40, 8)])
    hd = rng.choice([64, 128, 128, 256])
    if heads * hd > 8192:
        hd = 128
    return dict(heads=heads, kv_heads=kv, head_dim=hd, theta=rng.choice([10000.0, 1e6]),
                norm=rng.random() < 0.5)


def _types(rng):
    return rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])


def draw(rng):
    kind = rng.choice(["plan", "append", "attention", "attention", "attention", "accept", "q4",
                       "q4", "q4"])
    if kind == "q4":
        group = rng.choice([32, 64, 64, 128])
        cols = group * _log_int(rng, max(1, 256 // group), 8192 // group)
        rows = _log_int(rng, 40, min(50000, 100000000 // cols))
        tokens = _log_int(rng, 1, max(1, min(700, 16000000000 // (rows * cols))))
        x, y = rng.choice([("f32", "f32"), ("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
        c = _q4("", tokens, rows, cols, x, y, group, rng.random() < 0.4, rng.choice([0, 0, 64]))
        del c["name"]
        return c
    seqs = _log_int(rng, 1, 48)
    hi = _log_int(rng, 1, 250 if seqs <= 4 else 64)
    nodes, pad = (rng.randint(1, hi), hi), rng.choice([0, 0, 3])
    if kind == "plan":
        c = _trees("", "plan", seqs, nodes, pad=pad)
        del c["name"]
        return c
    m, (x, cache) = _model(rng), _types(rng)
    page = rng.choice([8, 16, 16, 32, 64, 256])
    # (a position's bytes over those of the widest listed case bound the lengths)
    wide = max(1.0, m["kv_heads"] * m["head_dim"] * (4 if cache == "f32" else 2) / 2048.0)
    if kind == "append":
        past = _log_int(rng, 1, 6000)
        c = _append("", m, seqs, nodes, (rng.randint(0, past), past), x, cache, page,
                    rng.choice([m["head_dim"], m["head_dim"], m["head_dim"] // 2, 32]),
                    rng.choice(["half", "interleaved"]), pad)
    elif kind == "accept":
        past = _log_int(rng, 1, 200)
        c = _accept("", m, seqs, nodes, (rng.randint(0, past), past), cache,
                    _log_int(rng, 1, max(1, int(32 / wide))), min(page, 64), pad)
    else:
        seqs = min(seqs, 32)
        nodes = (min(nodes[0], 2000 // seqs), min(nodes[1], 2000 // seqs))
        prefix = _log_int(rng, 32, int(3500 / wide)) if rng.random() < 0.35 else 0
        past = _log_int(rng, 4, int(500 / wide) + 4) if prefix else \
            _log_int(rng, 16, max(64, int(min(8000, 100000 / seqs / wide))))
        c = _attention("", m, seqs, nodes, (rng.randint(0, past), past), x, cache, page, prefix, pad)
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
    """(rows, positions after them) of each sequence."""
    rows = _spread(c["seqs"], c["nodes_lo"], c["nodes_hi"], 0)
    past = _spread(c["seqs"], c["past_lo"], c["past_hi"], 3)
    return rows, [r + p + c.get("prefix", 0) for r, p in zip(rows, past)]


def _words(c):
    """64-bit words of a row's mask."""
    return (c["nodes_hi"] + 63) // 64


def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + stream)
    return g


def _normal(shape, seed, stream, sigma=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=_gen(seed, stream), device=DEV) * sigma).to(dtype)


def _dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(DEV)


def _tree(c, seed):
    """Row starts, every row's number in its tree and its parent's (-1: none), on the host."""
    rows = _batch(c)[0]
    start = np.concatenate([[0], np.cumsum(rows)])
    i = np.arange(start[-1]) - np.repeat(start[:-1], rows)
    r = np.random.default_rng(seed * 7 + 5)
    chain, pick = r.random(len(i)), r.random(len(i))
    parent = np.where(chain < 0.4, i - 1, np.floor(pick * i)).astype(np.int64)
    return start, i, np.where(i == 0, -1, parent)


def _plan_of(c, seed):
    """(64-bit words of who sees whom, depths) by walking up from every row."""
    start, i, parent = _tree(c, seed)
    W, n = _words(c), len(i)
    mask = np.zeros((n + c["pad"], W), np.uint64)
    depth = np.zeros(n + c["pad"], np.int64)
    for r in range(n):
        if parent[r] >= 0:
            up = r - i[r] + parent[r]
            mask[r], depth[r] = mask[up], depth[up] + 1
        mask[r, i[r] // 64] |= np.uint64(1) << np.uint64(i[r] % 64)
    return mask.view(np.int64), depth


def _pages(c, seed):
    """The sequences' pages (the prefix' pages first), the prefix' own, how many there are."""
    length = _batch(c)[1]
    ps, prefix = c["page"], c.get("prefix", 0)
    need = [-(-n // ps) for n in length]
    full = prefix // ps    # pages wholly of the prefix are shared, one in part is each one's own
    total = full + sum(n - full for n in need) + 4
    order = torch.randperm(total, generator=_gen(seed, 50), device=DEV).cpu().numpy()
    table = np.zeros((c["seqs"], max(need)), np.int32)
    at = full
    for s, n in enumerate(need):
        table[s, :full] = order[:full]
        table[s, full:n] = order[at:at + n - full]
        at += n - full
    own_table = table[0, :-(-prefix // ps)].copy() if prefix else np.zeros(1, np.int32)
    return _dev(table), _dev(own_table), total


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


def _layers(c, seed, pages):
    """Every layer's k and v in one allocation."""
    return _normal((c["layers"], 2, pages, c["page"], c["kv_heads"], c["head_dim"]), seed, 2, 1.0,
                   DTYPES[c["cache"]])


def _tokens(c, seed):
    """Drafted tokens, and those drawn at every row: seven times in ten one of the row's own
    drafts (some trees hold the same draft twice)."""
    start, i, parent = _tree(c, seed)
    r = np.random.default_rng(seed * 7 + 6)
    n = len(i)
    draft, drawn = r.integers(0, 50304, n), r.integers(0, 50304, n)
    twin = r.random(n) < 0.1
    draft[1:] = np.where(twin[1:], draft[:-1], draft[1:])
    up = np.arange(n) - i + parent
    order = np.flatnonzero((parent >= 0) & (r.random(n) < 0.7))
    r.shuffle(order)
    drawn[up[order]] = draft[order]
    return draft, drawn


def _frequencies(c):
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64)
    return (c["theta"] ** (-2.0 * i / c["rotary"])).float().to(DEV)


def _weights(c, seed):
    """Packed nibbles (column 8 w + j in bits 4 j of word w), scales and biases: a group's 16
    steps over about what normal weights of 0.02 span."""
    N, K, G = c["rows"], c["cols"], c["group"]
    w = torch.randint(-(1 << 31), 1 << 31, (N, K // 8), generator=_gen(seed, 4), device=DEV,
                      dtype=torch.int64).to(torch.int32)
    lo = -0.05 * (1 + 0.15 * _normal((N, K // G), seed, 5))
    hi = 0.05 * (1 + 0.15 * _normal((N, K // G), seed, 6))
    return w, ((hi - lo) / 15).to(torch.bfloat16), lo.to(torch.bfloat16)


def prepare(case, seed):
    c = case
    if c["kind"] == "q4":
        T, N, K = c["tokens"], c["rows"], c["cols"]
        w, s, b = _weights(c, seed)
        st = dict(case=c, w=w, s=s, b=b, x=_normal((T, K + c["pad"]), seed, 1, 1.0, DTYPES[c["x"]]),
                  y=torch.zeros((T, (N + 7) // 8 * 8), dtype=DTYPES[c["y"]], device=DEV))
        if c["residual"]:
            st["r"] = _normal(st["y"].shape, seed, 7, 1.0, DTYPES[c["y"]])
        return st
    start, _, parent = _tree(c, seed)
    mask, depth = _plan_of(c, seed)
    n = int(start[-1]) + c["pad"]
    st = dict(case=c, start=_dev(start), parent=_dev(np.concatenate([parent, np.full(c["pad"], -1)])),
              nodes=int(start[-1]))
    if c["kind"] == "plan":
        st["mask"] = torch.zeros((n, _words(c)), dtype=torch.int64, device=DEV)
        st["depth"] = torch.zeros((n,), dtype=torch.int32, device=DEV)
        return st
    st["mask"], st["depth"] = _dev(mask, np.int64), _dev(depth)
    st["length"] = _dev(_batch(c)[1])
    st["table"], st["prefix_table"], pages = _pages(c, seed)
    st["pages"] = pages
    hd = c["head_dim"]
    if c["kind"] == "accept":
        st["kv"] = _layers(c, seed, pages)
        draft, drawn = _tokens(c, seed)
        pad = np.zeros(c["pad"], np.int64)
        st["draft"], st["drawn"] = (_dev(np.concatenate([t, pad])) for t in (draft, drawn))
        st["path"] = torch.zeros((n,), dtype=torch.int32, device=DEV)
        st["some"] = torch.zeros((3, c["seqs"]), dtype=torch.int32, device=DEV)
        return st
    st["kc"], st["vc"] = _cache(c, seed, pages, st["table"])
    qd, kvd = c["heads"] * hd, c["kv_heads"] * hd
    st["out"] = torch.zeros((n, qd), dtype=DTYPES[c["x"]], device=DEV)
    if c["kind"] == "append":   # the projections' rows, q, k and v side by side
        st["qkv"] = _normal((n, qd + 2 * kvd), seed, 1, 1.0, DTYPES[c["x"]])
        st["qw"] = (1 + _normal((hd,), seed, 4, 0.1)).to(torch.bfloat16)
        st["kw"] = (1 + _normal((hd,), seed, 5, 0.1)).to(torch.bfloat16)
        st["freq"] = _frequencies(c)
    else:
        st["q"] = _normal((n, qd), seed, 1, 1.0, DTYPES[c["x"]])
    return st


# ---- one pass: the plain forms ---------------------------------------------------------


def _places(st):
    """Sequence, number in its tree and base position of every row (not of the padding)."""
    start, length = st["start"].long(), st["length"].long()
    row = torch.arange(st["nodes"], device=DEV)
    seq = torch.searchsorted(start, row, right=True) - 1
    return seq, row - start[seq], length[seq] - (start[seq + 1] - start[seq])


def _padded(st):
    """[seqs][largest tree]: the rows (the last one again past a tree's end), which are real."""
    start, R = st["start"].long(), max(_batch(st["case"])[0])
    n = start[1:] - start[:-1]
    i = torch.arange(R, device=DEV)[None, :]
    return start[:-1, None] + torch.minimum(i, n[:, None] - 1), i < n[:, None], n


def _plain_plan(st):
    c, R = st["case"], max(_batch(st["case"])[0])
    row, real, n = _padded(st)
    i = torch.arange(R, device=DEV)
    parent = st["parent"].long()[row]
    # one step up or none, R - 1 times: the ancestors and itself
    step = ((parent[:, :, None] == i) | (i[:, None] == i)).double()
    sees = torch.linalg.matrix_power(step, max(R - 1, 1)) > 0
    W = _words(c)
    bits = torch.zeros((c["seqs"], R, 64 * W), dtype=torch.int64, device=DEV)
    bits[:, :, :R] = sees
    bits = bits.reshape(c["seqs"], R, W, 64) << torch.arange(64, device=DEV)
    st["mask"][:st["nodes"]] = bits.sum(-1)[real]
    st["depth"][:st["nodes"]] = (sees.sum(-1) - 1)[real].int()
    return st["mask"], st["depth"]


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
    c, T = st["case"], st["nodes"]
    hd, hq, hk = c["head_dim"], c["heads"], c["kv_heads"]
    seq, i, base = _places(st)
    x = st["qkv"][:T].float()
    q = x[:, :hq * hd].reshape(-1, hq, hd)
    k = x[:, hq * hd:(hq + hk) * hd].reshape(-1, hk, hd)
    v = x[:, (hq + hk) * hd:].reshape(-1, hk, hd)
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * st["qw"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * st["kw"].float()
    angle = (base + st["depth"][:T]).double()[:, None] * st["freq"].double()[None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    q, k = _rotate(q, cos, sin, c["pairs"]), _rotate(k, cos, sin, c["pairs"])
    at = base + i
    page, slot = st["table"].long()[seq, at // c["page"]], at % c["page"]
    st["kc"][page, slot] = k.to(st["kc"].dtype)
    st["vc"][page, slot] = v.to(st["vc"].dtype)
    st["out"][:T] = q.reshape(-1, hq * hd).to(st["out"].dtype)
    return st["out"], st["kc"], st["vc"]


def _plain_attention(st):
    c = st["case"]
    hd, hk = c["head_dim"], c["kv_heads"]
    share, B, L = c["heads"] // hk, c["seqs"], max(_batch(c)[1])
    row, real, n = _padded(st)
    R, kv = row.shape[1], st["length"].long()
    # every sequence's positions, padded to the longest (its own last one again)
    l = torch.arange(L, device=DEV)[None, :]
    at = torch.minimum(l, kv[:, None] - 1)
    page = st["table"].long().gather(1, at // c["page"])
    k = st["kc"][page, at % c["page"]].float().permute(0, 2, 3, 1).contiguous()
    v = st["vc"][page, at % c["page"]].float().permute(0, 2, 1, 3).contiguous()
    q = st["q"][row].float().reshape(B, R, hk, share, hd)
    q = q.permute(0, 2, 1, 3, 4).reshape(B, hk, R * share, hd)
    s = torch.matmul(q, k) * (1.0 / math.sqrt(hd))
    # hidden: past the tree, or in it and no ancestor
    rel = l - (kv - n)[:, None]
    word = (rel >> 6).clamp(0, _words(c) - 1)[:, None, :].expand(B, R, L)
    sees = (st["mask"][row].gather(2, word) >> (rel & 63)[:, None, :]) & 1
    hide = ((rel >= 0)[:, None, :] & (sees == 0)) | (rel >= n[:, None])[:, None, :]
    s.masked_fill_(hide.repeat_interleave(share, 1)[:, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.reshape(B, hk, R, share, hd).permute(0, 2, 1, 3, 4).reshape(B, R, -1)
    st["out"][:st["nodes"]] = o[real].to(st["out"].dtype)
    return st["out"]


def _plain_accept(st):
    c = st["case"]
    row, real, n = _padded(st)
    B, R = row.shape
    i = torch.arange(R, device=DEV)[None, :]
    parent = st["parent"].long()[row]
    draft, drawn = st["draft"].long()[row], st["drawn"].long()[row]
    up = parent.clamp(min=0)
    good = real & ((parent < 0) & (i == 0) | (parent >= 0) & (draft == drawn.gather(1, up)))
    # of the good ones with one parent the first
    twin = (parent[:, :, None] == parent[:, None, :]) & good[:, None, :] & (i[..., None] > i[:, None, :])
    good = good & ~twin.any(2)
    # taken: with all their ancestors good
    word = (i >> 6).expand(B, R)[:, None, :].expand(B, R, R)
    sees = ((st["mask"][row].gather(2, word) >> (i & 63)[:, None, :]) & 1).bool()
    taken = real & ~(sees & ~good[:, None, :]).any(2)
    count = taken.sum(1)
    order = torch.where(taken, i, R).sort(1).values
    last = order.gather(1, count[:, None] - 1)
    path = torch.where(i < count[:, None], order, -1)
    base = st["length"].long() - n
    # every row of a tree from the place that its new content has now
    src = torch.where(path >= 0, path, torch.minimum(i, n[:, None] - 1))[real]
    seq = torch.arange(B, device=DEV)[:, None].expand(B, R)[real]
    at, to, table = base[seq] + src, (base[:, None] + i)[real], st["table"].long()
    moved = st["kv"][:, :, table[seq, at // c["page"]], at % c["page"]]
    st["kv"][:, :, table[seq, to // c["page"]], to % c["page"]] = moved
    st["path"][:st["nodes"]] = path[real].int()
    st["some"][0], st["some"][1] = count, drawn.gather(1, last)[:, 0]
    st["some"][2] = base + count
    return st["path"], st["some"], st["kv"]


def _plain_q4(st):
    c = st["case"]
    N, K, G = c["rows"], c["cols"], c["group"]
    n = (st["w"][:, :, None] >> (4 * torch.arange(8, device=DEV, dtype=torch.int32))) & 15
    w = n.reshape(N, K // G, G).float() * st["s"].float()[:, :, None] + st["b"].float()[:, :, None]
    y = st["x"][:, :K].float() @ w.reshape(N, K).t()
    if c["residual"]:
        y = y + st["r"][:, :N].float()
    st["y"][:, :N] = y.to(st["y"].dtype)
    return st["y"]


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
    """What a program keeps of a batch: the descriptions of its caches, rows and weights."""
    from m1moe_amd import KVAppend, PagedBatch, PagedKV, Q4Weights
    c = st["case"]
    if c["kind"] == "plan":
        st["handles"] = True
        return True
    if c["kind"] == "q4":
        st["handles"] = Q4Weights.make(st["w"].data_ptr(), st["s"].data_ptr(), st["b"].data_ptr(),
                                       c["rows"], c["cols"], c["group"])
        return st["handles"]

    def cache(k, v):
        return PagedKV.make(k.data_ptr(), v.data_ptr(), c["cache"], st["pages"], c["page"],
                            c["kv_heads"], c["head_dim"])
    prefix = c.get("prefix", 0)
    batch = PagedBatch.make(c["seqs"], st["nodes"] + c["pad"], st["start"].data_ptr(),
                            st["length"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1],
                            prefix, st["prefix_table"].data_ptr() if prefix else None)
    if c["kind"] == "accept":
        st["handles"] = (PagedKV.array([cache(l[0], l[1]) for l in st["kv"]]), batch)
    elif c["kind"] == "attention":
        st["handles"] = (cache(st["kc"], st["vc"]), batch)
    else:
        size, hd = st["qkv"].element_size(), c["head_dim"]
        at, n = st["qkv"].data_ptr(), st["qkv"].shape[1]
        qd, kvd = c["heads"] * hd, c["kv_heads"] * hd
        st["handles"] = (cache(st["kc"], st["vc"]), batch, KVAppend.make(
            c["x"], c["heads"], at, at + qd * size, at + (qd + kvd) * size, n, n, n,
            st["out"].data_ptr(), qd, st["qw"].data_ptr() if c["norm"] else None,
            st["kw"].data_ptr() if c["norm"] else None, EPS, c["rotary"],
            c["pairs"] == "interleaved", st["freq"].data_ptr(), 1.0))
    return st["handles"]


def run(state):
    st, c = state, state["case"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention,
                "accept": _plain_accept, "q4": _plain_q4}[c["kind"]](st)
    ops, h = _dense_ops(), st.get("handles") or _handles(st)
    if c["kind"] == "plan":
        ops.tree_plan(c["seqs"], st["nodes"] + c["pad"], st["start"].data_ptr(),
                      st["parent"].data_ptr(), _words(c), st["mask"].data_ptr(),
                      st["depth"].data_ptr())
        return st["mask"], st["depth"]
    if c["kind"] == "append":
        ops.tree_append(h[0], h[1], h[2], st["depth"].data_ptr())
        return st["out"], st["kc"], st["vc"]
    if c["kind"] == "attention":
        qd = st["q"].shape[1]
        ops.tree_attention(h[0], h[1], st["mask"].data_ptr(), _words(c), st["q"].data_ptr(), qd,
                           st["out"].data_ptr(), qd, c["x"], c["heads"])
        return st["out"]
    if c["kind"] == "accept":
        ops.tree_accept(h[0], h[1], st["parent"].data_ptr(), st["draft"].data_ptr(),
                        st["drawn"].data_ptr(), st["path"].data_ptr(), st["some"][0].data_ptr(),
                        st["some"][1].data_ptr(), st["some"][2].data_ptr())
        return st["path"], st["some"], st["kv"]
    ops.matmul_q4(h, st["x"].data_ptr(), c["x"], st["x"].shape[1], c["tokens"], st["y"].data_ptr(),
                  c["y"], st["y"].shape[1], st["r"].data_ptr() if c["residual"] else None)
    return st["y"]


# ---- what a pass cannot do without -----------------------------------------------------


def _size(t):
    return 4.0 if t == "f32" else 2.0


def work(case):
    c = case
    if c["kind"] == "q4":
        T, N, K = float(c["tokens"]), c["rows"], c["cols"]
        return {"bytes": N * K / 2.0 + 4.0 * N * K / c["group"] + T * K * _size(c["x"]) +
                T * N * _size(c["y"]) * (2 if c["residual"] else 1), "flops": 2.0 * T * N * K}
    rows, length = _batch(c)
    n = float(sum(rows))
    if c["kind"] == "plan":
        return {"bytes": n * (8.0 + 8.0 * _words(c)) + 4.0 * c["seqs"], "flops": n}
    kvd = c["kv_heads"] * c["head_dim"]
    if c["kind"] == "accept":   # (a path of about one row per level; nearly all of them move)
        kept = sum(min(r, 1 + math.log(r)) for r in rows)
        return {"bytes": 16.0 * n + 4.0 * kvd * _size(c["cache"]) * c["layers"] * kept, "flops": n}
    qd = c["heads"] * c["head_dim"]
    if c["kind"] == "append":
        return {"bytes": n * (2 * qd * _size(c["x"]) + 2 * kvd * (_size(c["x"]) + _size(c["cache"]))),
                "flops": n * 8.0 * (qd + kvd)}
    prefix = c["prefix"]
    # (in its tree a row sees about one row per level)
    pairs = sum(r * (k - r) + r * min(r, 1 + math.log(r)) for r, k in zip(rows, length))
    seen = prefix + sum(k - prefix for k in length)
    return {"bytes": 2.0 * seen * kvd * _size(c["cache"]) + n * (2.0 * qd * _size(c["x"]) + 8 * _words(c)),
            "flops": 4.0 * pairs * qd}


# ---- the same in 64 bits ---------------------------------------------------------------


def _ancestors(parent):
    """Of every row of one tree the rows it sees, from the root down."""
    sees = []
    for r, p in enumerate(parent):
        sees.append((sees[p] if p >= 0 else []) + [r])
    return sees


def _exact_append(c, seed):
    st = prepare(c, seed)
    out, kc, vc = st["out"].double(), st["kc"].double(), st["vc"].double()
    x, hd, hq, hk = st["qkv"].double(), c["head_dim"], c["heads"], c["kv_heads"]
    half, ps = c["rotary"] // 2, c["page"]
    start, _, parent = _tree(c, seed)
    length, tab = _batch(c)[1], st["table"].long()
    # pair i of a head: dims (i, i + half) or (2 i, 2 i + 1)
    first = torch.arange(half, device=DEV) * (1 if c["pairs"] == "half" else 2)
    second = first + (half if c["pairs"] == "half" else 1)

    def turn(y, w, at):
        if c["norm"]:
            y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / hd + EPS) * w.double()
        z = y.clone()
        r = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.ones_like(at), at)[:, None, :]
        z[..., first], z[..., second] = r.real, r.imag
        return z
    for s in range(c["seqs"]):
        lo, hi = int(start[s]), int(start[s + 1])
        base = length[s] - (hi - lo)
        level = torch.tensor([len(a) - 1 for a in _ancestors(parent[lo:hi])], device=DEV)
        at = (base + level).double()[:, None] * st["freq"].double()
        blk = x[lo:hi].reshape(hi - lo, hq + 2 * hk, hd)
        out[lo:hi] = turn(blk[:, :hq], st["qw"], at).reshape(hi - lo, -1)
        p = torch.arange(base, length[s], device=DEV)
        where = tab[s][torch.div(p, ps, rounding_mode="floor")]
        kc[where, p % ps] = turn(blk[:, hq:hq + hk], st["kw"], at)
        vc[where, p % ps] = blk[:, hq + hk:]
    return out, kc, vc


def _exact_attention(c, seed):
    st = prepare(c, seed)
    hd, share, ps = c["head_dim"], c["heads"] // c["kv_heads"], c["page"]
    out = st["out"].double()
    start, _, parent = _tree(c, seed)
    length, tab = _batch(c)[1], st["table"].long()
    for s in range(c["seqs"]):
        lo, hi, n = int(start[s]), int(start[s + 1]), length[s]
        base = n - (hi - lo)
        seen = torch.zeros((hi - lo, n), dtype=torch.bool)
        seen[:, :base] = True
        for r, a in enumerate(_ancestors(parent[lo:hi])):
            seen[r, base + torch.tensor(a)] = True
        seen = seen.to(DEV)
        p = torch.arange(n, device=DEV)
        k = st["kc"][tab[s][torch.div(p, ps, rounding_mode="floor")], p % ps].double()
        v = st["vc"][tab[s][torch.div(p, ps, rounding_mode="floor")], p % ps].double()
        for g in range(c["kv_heads"]):
            kt, vg = k[:, g].t().contiguous(), v[:, g].contiguous()
            for h in range(g * share, (g + 1) * share):
                e = (st["q"][lo:hi, h * hd:(h + 1) * hd].double() @ kt) / math.sqrt(hd)
                out[lo:hi, h * hd:(h + 1) * hd] = torch.softmax(torch.where(seen, e, -math.inf), 1) @ vg
    return out


def _exact_plan(c, seed):
    start, _, parent = _tree(c, seed)
    mask = np.zeros((int(start[-1]) + c["pad"], _words(c)), np.uint64)
    depth = np.zeros(len(mask), np.int32)
    for s in range(c["seqs"]):
        for r, a in enumerate(_ancestors(parent[int(start[s]):int(start[s + 1])])):
            word = sum(1 << int(j) for j in a)
            mask[start[s] + r] = [(word >> 64 * w) & (2 ** 64 - 1) for w in range(_words(c))]
            depth[start[s] + r] = len(a) - 1
    return _dev(mask.view(np.int64), np.int64), _dev(depth)


def _exact_accept(c, seed):
    st = prepare(c, seed)
    start, _, parent = _tree(c, seed)
    draft, drawn = _tokens(c, seed)
    length, tab, kv, ps = _batch(c)[1], st["table"].long(), st["kv"].double(), c["page"]
    path, some = np.zeros(int(start[-1]) + c["pad"], np.int32), np.zeros((3, c["seqs"]), np.int32)
    path[:start[-1]] = -1
    for s in range(c["seqs"]):
        lo, hi = int(start[s]), int(start[s + 1])
        base, way = length[s] - (hi - lo), [0]
        while True:
            on = [r for r in range(hi - lo) if parent[lo + r] == way[-1] and draft[lo + r] == drawn[lo + way[-1]]]
            if not on:
                break
            way.append(on[0])
        path[lo:lo + len(way)] = way
        some[:, s] = len(way), drawn[lo + way[-1]], base + len(way)
        at = base + torch.tensor(way, device=DEV)
        to = base + torch.arange(len(way), device=DEV)
        rows = kv[:, :, tab[s][at // ps], at % ps].clone()
        kv[:, :, tab[s][to // ps], to % ps] = rows
    return _dev(path), _dev(some), kv


def _exact_q4(c, seed):
    st = prepare(c, seed)
    N, K, G = c["rows"], c["cols"], c["group"]
    y, w = st["y"].double(), torch.empty((N, K), dtype=torch.float64, device=DEV)
    s, b = (t.double().repeat_interleave(G, 1) for t in (st["s"], st["b"]))
    for j in range(8):   # column 8 i + j is bits 4 j .. 4 j + 3 of word i
        nib = torch.div(st["w"].long() & 0xFFFFFFFF, 1 << 4 * j, rounding_mode="floor") % 16
        w[:, j::8] = nib.double() * s[:, j::8] + b[:, j::8]
    y[:, :N] = st["x"][:, :K].double() @ w.t()
    if c["residual"]:
        y[:, :N] += st["r"][:, :N].double()
    return y


def exact(case, seed):
    return {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention,
            "accept": _exact_accept, "q4": _exact_q4}[case["kind"]](case, seed)
