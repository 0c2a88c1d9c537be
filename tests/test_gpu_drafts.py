"""GPU parity of the drafted tokens' operators (tree plan, append, attention, accept) and of the
products with 4-bit weights against f64 references (draft_cases.py), through the C ABI.  Bounds
are elementwise and derived there or in serving_cases.py; whole numbers are equal."""
import numpy as np
import pytest

import m1moe_amd as m
from m1moe_amd import KVAppend, M1MoEError, PagedKV, Q4Weights, SampleParams, _lib
from m1moe_amd.decoder import DenseOps, rope_frequencies
from m1moe_amd.quant import quantize_4bit

from cases import rel_l2, say
from draft_cases import (accept_ref, plan_ref, q4_bound, q4_dense, q4_weights, tree_attention_ref, tree_parents)
from serving_cases import Batch, append_ref, as_dtype, attention_bound, bf16, f64
from test_gpu_serving import Held, cache_of

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")]


@pytest.fixture(scope="module")
def dev():
    say("drafts context")
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    yield ctx, DenseOps(ctx)
    ctx.close()


def words_of(b):
    return max(1, -(-max(b.rows) // 64))


def trees(rng, b, chain=0.4):
    """(parents of all rows, masks, depths), the padding's masks full."""
    W = words_of(b)
    par = [tree_parents(rng, n, chain) if n else [] for n in b.rows]
    mask = np.full((b.num_rows, W), np.uint64(2 ** 64 - 1))
    depth = np.zeros(b.num_rows, np.int32)
    for s, p in enumerate(par):
        r0 = int(b.row_start[s])
        mask[r0:r0 + len(p)], depth[r0:r0 + len(p)] = plan_ref(p, W)
    flat = np.array([x for p in par for x in p] + [-1] * b.pad, np.int32)
    return flat, mask, depth


# ---- plan ----------------------------------------------------------------------------------

def run_plan(dev, rows, parents, words, pad=2, starts=None):
    ctx, ops = dev
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32) if starts is None else starts
    n = int(sum(rows)) + pad
    par = np.full(n, 99, np.int32)
    par[:len(parents)] = parents
    held = [ctx.to_device(start), ctx.to_device(par), ctx.to_device(np.full((n, words), 7, np.uint64)),
            ctx.to_device(np.full(n, 7, np.int32))]
    ops.tree_plan(len(rows), n, held[0], held[1], words, held[2], held[3])
    try:
        ctx.sync()
        err = None
    except M1MoEError as e:
        err = e
    mask, depth = held[2].download(np.uint64).reshape(n, words), held[3].download(np.int32)
    for h in held:
        h.free()
    return mask, depth, err


@pytest.mark.parametrize("words", [1, 2, 3, 4])
@pytest.mark.parametrize("chain", [0.0, 0.4, 1.0])
def test_plan(dev, words, chain):
    rng = np.random.default_rng(words)
    N = 64 * words
    rows = [1, 0, 2, N, 33, 0, N - 1, 64, 5]
    par = [tree_parents(rng, n, chain) if n else [] for n in rows]
    for p in par:       # forests too: some rows without a parent
        if len(p) > 30:
            p[7] = p[20] = -1
    par[-1] = [-1, 0, 0, 0, 0]
    say(f"plan words {words} chain {chain}")
    mask, depth, err = run_plan(dev, rows, [x for p in par for x in p], words)
    assert err is None
    at = 0
    for p in par:
        want, deep = plan_ref(p, words)
        assert np.array_equal(mask[at:at + len(p)], want) and np.array_equal(depth[at:at + len(p)], deep)
        at += len(p)
    assert np.all(mask[at:] == 7) and np.all(depth[at:] == 7)


def test_plan_many_sequences(dev):
    rng = np.random.default_rng(5)
    rows = rng.integers(0, 9, 1024).tolist()
    par = [tree_parents(rng, n) if n else [] for n in rows]
    mask, depth, err = run_plan(dev, rows, [x for p in par for x in p], 1)
    want = [plan_ref(p, 1) for p in par]
    assert err is None
    assert np.array_equal(mask[:-2], np.concatenate([w[0] for w in want]))
    assert np.array_equal(depth[:-2], np.concatenate([w[1] for w in want]))


def test_plan_reports_bad_trees(dev):
    """A parent that is not lower than its row counts as none; a tree of more rows than the masks
    have bits, or with wrong starts, is left out; the others are right."""
    say("plan bad trees")
    par = [-1, 0, 2, 1, -5, 3, -1, 0]
    mask, depth, err = run_plan(dev, [6, 2], par, 1)
    assert err is not None and err.code == _lib.M1MOE_ERR_DEVICE and "tree" in str(err)
    want, deep = plan_ref([-1, 0, -1, 1, -1, 3], 1)
    assert np.array_equal(mask[:6], want) and np.array_equal(depth[:6], deep)
    assert np.array_equal(mask[6:8], plan_ref([-1, 0], 1)[0])
    mask, depth, err = run_plan(dev, [65, 2], [-1] + list(range(64)) + [-1, 0], 1)
    assert err is not None and "tree" in str(err)
    assert np.all(mask[:65] == 7) and np.array_equal(mask[65:67], plan_ref([-1, 0], 1)[0])
    mask, depth, err = run_plan(dev, [2, 2], [-1, 0, -1, 0], 1, starts=np.array([0, 2, 900], np.int32))
    assert err is not None and "paged batch" in str(err)
    assert np.array_equal(mask[:2], plan_ref([-1, 0], 1)[0]) and np.all(mask[2:] == 7)
    dev[0].sync()


# ---- append --------------------------------------------------------------------------------

class At:
    """A batch whose rows stand at given positions (append_ref asks for no more)."""

    def __init__(self, b, pos):
        self.T, self.pos = b.T, pos

    def places(self):
        return [(0, int(p)) for p in self.pos]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("hd,rotary,inter,norm", [(64, 64, 0, True), (128, 64, 1, False), (256, 256, 0, True),
                                                  (128, 0, 0, True)])
def test_append(dev, types, hd, rotary, inter, norm):
    ctx, ops = dev
    rng = np.random.default_rng(hd + rotary)
    x, cache = types
    heads, kv_heads = 6, 2
    b = Batch(rng, [9, 1, 0, 70, 2], [3, 100, 5, 40, 8000], 16, pad=2)
    _, _, depth = trees(rng, b)
    n = (heads + 2 * kv_heads) * hd
    qkv = as_dtype(rng.normal(0, 1, (b.num_rows, n)), x)
    w = [bf16(1 + 0.1 * rng.normal(0, 1, hd)) for _ in range(2)]
    freq, amp = rope_frequencies(1e4, rotary or 16)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    es = 2 if x == "bf16" else 4
    buf, out = d.up(qkv), d.up(as_dtype(np.full((b.num_rows, heads * hd), 5.0), x))
    args = KVAppend.make(x, heads, buf, buf.addr + heads * hd * es, buf.addr + (heads + kv_heads) * hd * es, n, n, n,
                         out, heads * hd, d.up(w[0]) if norm else None, d.up(w[1]) if norm else None, 1e-5, rotary,
                         bool(inter), d.up(freq), amp)
    say(f"tree append {types} {hd} rotary {rotary}")
    ops.tree_append(d.kv, d.batch, args, d.up(depth))
    ctx.sync()
    ut = np.uint16 if x == "bf16" else np.float32
    uc = np.uint16 if cache == "bf16" else np.float32
    got = f64(out.download(ut)).reshape(b.num_rows, heads, hd)
    gk, gv = d.k.download(uc).reshape(kc.shape), d.v.download(uc).reshape(vc.shape)
    d.free()
    base = np.array([int(b.kv_len[s]) - b.rows[s] for s, _ in b.places()])
    at = At(b, base + depth[:b.T])
    q_, k_, v_ = qkv[:, :heads * hd], qkv[:, heads * hd:(heads + kv_heads) * hd], qkv[:, (heads + kv_heads) * hd:]
    # (f32: the norm's sum of hd squares, its root and the products, the angle's cos and sin)
    eps = (hd / 8 + 16) * 2.0 ** -24
    for name, src, h, wt, g, dt in (("q", q_, heads, w[0], got[:b.T], x), ("k", k_, kv_heads, w[1], None, cache)):
        ref, size = append_ref(at, np.ascontiguousarray(src), h, hd, wt if norm else None, 1e-5, rotary, inter, freq, amp)
        if g is None:
            pg, sl = np.array([[c[0] for c in b.cell(s, np.array([p]))] for s, p in b.places()]).T
            g = f64(gk[pg, sl])
            assert np.array_equal(f64(gv[pg, sl]).reshape(b.T, -1), f64(as_dtype(f64(v_[:b.T]), cache)))
        bound = eps * size + (2.0 ** -8 * np.abs(ref) if dt == "bf16" else 0) + 1e-30
        assert np.all(np.abs(g - ref) <= bound), name
    assert np.all(got[b.T:] == 5.0)
    mine = np.zeros(kc.shape[:2], bool)
    mine[pg, sl] = True
    assert np.array_equal(gk[~mine], kc[~mine]) and np.array_equal(gv[~mine], vc[~mine])


def test_append_of_a_chain_is_the_plain_append(dev):
    """Depths 0, 1, 2, ..: the same bits."""
    ctx, ops = dev
    rng = np.random.default_rng(3)
    b = Batch(rng, [5, 12], [30, 4], 8)
    heads, kv_heads, hd = 4, 2, 128
    n = (heads + 2 * kv_heads) * hd
    qkv = rng.normal(0, 1, (b.T, n)).astype(np.float32)
    freq, _ = rope_frequencies(1e4, hd)
    kc, vc = cache_of(rng, b, kv_heads, hd, "f32")
    got = []
    for tree in (False, True):
        d = Held(ctx, b, kc, vc, "f32", kv_heads, hd)
        buf, out = d.up(qkv), d.up(np.zeros((b.T, heads * hd), np.float32))
        args = KVAppend.make("f32", heads, buf, buf.addr + 4 * heads * hd, buf.addr + 4 * (heads + kv_heads) * hd, n, n,
                             n, out, heads * hd, rotary_dim=hd, inv_freq=d.up(freq))
        if tree:
            ops.tree_append(d.kv, d.batch, args, d.up(np.concatenate([np.arange(5), np.arange(12)]).astype(np.int32)))
        else:
            ops.kv_append(d.kv, d.batch, args)
        ctx.sync()
        got.append([out.download(np.float32), d.k.download(np.float32), d.v.download(np.float32)])
        d.free()
    assert all(np.array_equal(x, y) for x, y in zip(*got))


# ---- attention -----------------------------------------------------------------------------

def attend(dev, b, mask, heads, kv_heads, hd, types, seed, fill=np.nan, edit=None):
    """(output rows, the padding's rows, f64 reference, bound) of one call."""
    ctx, ops = dev
    rng = np.random.default_rng(seed)
    x, cache = types
    q = as_dtype(rng.normal(0, 1, (b.num_rows, heads * hd)), x)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache, fill)
    if edit:
        edit(kc, vc, cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    out = d.up(as_dtype(np.full((b.num_rows, heads * hd), 7.0), x))
    ops.tree_attention(d.kv, d.batch, d.up(mask), mask.shape[1], d.up(q), heads * hd, out, heads * hd, x, heads)
    ctx.sync()
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
    d.free()
    ref, mag, top = tree_attention_ref(b, mask, q, kc, vc, heads, kv_heads, hd)
    return got[:b.T], got[b.T:], ref, attention_bound(ref, mag, top, hd, x)


def check_close(got, ref, bound, dtype):
    assert np.all(np.isfinite(got))
    worst = np.max(np.abs(got - ref) / bound) if ref.size else 0.0
    assert worst <= 1.0, worst
    # (in the 2-norm the roundings of a row's f32 sums are independent: 128 of them of 2^-24,
    # scores up to a few units; bf16: two roundings of at most 2^-8)
    assert rel_l2(got, ref) < (1e-5 if dtype == "f32" else 2.0 ** -7)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 4, 128, 16), (8, 2, 128, 64), (7, 1, 64, 8), (5, 1, 256, 32),
                                                    (40, 1, 128, 16), (16, 2, 64, 256)])
def test_attention(dev, types, heads, kv_heads, hd, page):
    """Trees of any size behind any past, empty sequences and rows behind the last one."""
    rng = np.random.default_rng(heads)
    b = Batch(rng, [1, 26, 0, 64, 2, 33, 17, 0, 63], [0, 5, 9, 31, 400, 32, 63, 2, 1001], page, pad=3)
    _, mask, _ = trees(rng, b)
    say(f"tree attention {types} {heads}/{kv_heads}x{hd} page {page}")
    got, rest, ref, bound = attend(dev, b, mask, heads, kv_heads, hd, types, 2)
    check_close(got, ref, bound, types[0])
    assert np.all(rest == 7.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [[65, 1], [128, 3], [129, 64], [200, 192], [256, 255]])
def test_attention_large_trees(dev, types, rows):
    """Masks of two to four words."""
    rng = np.random.default_rng(sum(rows))
    b = Batch(rng, rows, [77, 40], 16, pad=1)
    _, mask, _ = trees(rng, b, 0.8)
    say(f"tree attention rows {rows} {types}")
    got, rest, ref, bound = attend(dev, b, mask, 6, 2, 128, types, 3)
    check_close(got, ref, bound, types[0])
    assert np.all(rest == 7.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("prefix", [1, 31, 32, 100, 777])
def test_attention_prefix(dev, types, prefix):
    rng = np.random.default_rng(prefix)
    b = Batch(rng, [1, 20, 3, 0, 64, 40, 1], [prefix + p for p in (0, 0, 64, 2, 31, 10, 300)], 16, prefix=prefix, pad=2)
    _, mask, _ = trees(rng, b)
    say(f"tree attention prefix {prefix} {types}")
    got, rest, ref, bound = attend(dev, b, mask, 8, 2, 128, types, prefix + 1)
    check_close(got, ref, bound, types[0])
    assert np.all(rest == 7.0)


@pytest.mark.parametrize("types", TYPES)
def test_attention_any_mask(dev, types):
    """Masks that are no trees: random bits, rows that do not see themselves, bits of later rows
    (no effect), and without a past rows that see nothing: zeros."""
    rng = np.random.default_rng(7)
    b = Batch(rng, [40, 64, 9, 1], [0, 50, 0, 0], 16)
    mask = rng.integers(0, 1 << 64, (b.T, 1), dtype=np.uint64) & rng.integers(0, 1 << 64, (b.T, 1), dtype=np.uint64)
    mask[[0, 5, 104, 107, 113]] = 0
    mask[108] = np.uint64(2 ** 64 - 1) << np.uint64(5)       # only later rows: nothing
    say(f"tree attention any mask {types}")
    got, _, ref, bound = attend(dev, b, mask, 8, 2, 64, types, 8)
    check_close(got, ref, bound, types[0])
    for r in (0, 5, 104, 107, 108, 113):
        assert np.all(got[r] == 0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_attention_values_that_are_not_seen(dev, types, what):
    """What a row's siblings hold does not reach it, whatever it is: row 1's branch is not finite,
    row 2's sees it nowhere."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [30, 20], [40, 3], 16)
    par = [-1, 0, 0] + [1 + i % 2 for i in range(27)]        # odd rows under row 1, even ones under row 2
    mask = np.concatenate([plan_ref(par, 1)[0], plan_ref(tree_parents(rng, 20), 1)[0]])

    def edit(kc, vc, cache):
        for i in range(1, 30, 2):
            pg, sl = b.cell(0, np.array([40 + i]))
            kc[pg, sl] = as_dtype(np.full(kc.shape[2:], what), cache)
            vc[pg, sl] = as_dtype(np.full(vc.shape[2:], what), cache)
    say(f"tree attention unseen {what} {types}")
    got, _, ref, bound = attend(dev, b, mask, 4, 2, 128, types, 10, edit=edit)
    clean = [0] + list(range(2, 30, 2)) + list(range(30, 50))
    check_close(got[clean], ref[clean], bound[clean], types[0])
    assert not np.isfinite(got[1:30:2]).any()


@pytest.mark.parametrize("types", TYPES)
def test_attention_of_a_chain_is_the_plain_one(dev, types):
    """Every row sees all earlier ones: paged attention's bits."""
    ctx, ops = dev
    rng = np.random.default_rng(11)
    x, cache = types
    heads, kv_heads, hd = 8, 2, 128
    b = Batch(rng, [33, 64, 1], [900, 0, 31], 16)
    mask = np.array([[(1 << i + 1) - 1] for n in b.rows for i in range(n)], np.uint64)
    q = as_dtype(rng.normal(0, 1, (b.T, heads * hd)), x)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    ut = np.uint16 if x == "bf16" else np.float32
    dq, outs = d.up(q), [d.up(np.zeros((b.T, heads * hd), ut)) for _ in range(2)]
    ops.paged_attention(d.kv, d.batch, dq, heads * hd, outs[0], heads * hd, x, heads)
    ops.tree_attention(d.kv, d.batch, d.up(mask), 1, dq, heads * hd, outs[1], heads * hd, x, heads)
    ctx.sync()
    a, c = (o.download(ut) for o in outs)
    d.free()
    assert np.array_equal(a, c)


def test_attention_skips_trees_past_the_masks(dev):
    ctx, ops = dev
    rng = np.random.default_rng(12)
    heads, kv_heads, hd = 4, 2, 64
    for prefix in (0, 40):
        b = Batch(rng, [10, 65, 3], [prefix + p for p in (20, 30, 100)], 16, prefix=prefix)
        mask = np.full((b.T, 1), np.uint64(2 ** 64 - 1))
        q = rng.normal(0, 1, (b.T, heads * hd)).astype(np.float32)
        kc, vc = cache_of(rng, b, kv_heads, hd, "f32")
        ref, mag, top = tree_attention_ref(b, np.concatenate([mask, mask], 1), q, kc, vc, heads, kv_heads, hd)
        bound = attention_bound(ref, mag, top, hd, "f32")
        d = Held(ctx, b, kc, vc, "f32", kv_heads, hd)
        out = d.up(np.full((b.T, heads * hd), 3.0, np.float32))
        say(f"tree attention past the masks, prefix {prefix}")
        ops.tree_attention(d.kv, d.batch, d.up(mask), 1, d.up(q), heads * hd, out, heads * hd, "f32", heads)
        with pytest.raises(M1MoEError) as e:
            ctx.sync()
        assert e.value.code == _lib.M1MOE_ERR_DEVICE and "tree" in str(e.value)
        got = out.download(np.float32).reshape(b.T, heads, hd).astype(np.float64)
        d.free()
        keep = list(range(10)) + list(range(75, 78))
        assert np.all(np.abs(got[keep] - ref[keep]) <= bound[keep]) and np.all(got[10:75] == 3.0)


# ---- accept --------------------------------------------------------------------------------

class Taken:
    """One accept over `layers` caches of random values; what it leaves."""

    def __init__(self, dev, b, parents, drafts, drawn, kv_heads, hd, cache, layers, seed):
        ctx, ops = dev
        rng = np.random.default_rng(seed)
        shape = (b.num_pages, b.page, kv_heads, hd)
        self.before = [as_dtype(rng.normal(0, 1, shape), cache) for _ in range(2 * layers)]
        planes = [ctx.to_device(p) for p in self.before]
        up = [ctx.to_device(np.ascontiguousarray(a)) for a in (b.row_start, b.kv_len, b.table, parents, drafts, drawn)]
        outs = [ctx.to_device(np.full(max(n, 1), 55, np.int32)) for n in (b.num_rows, b.B, b.B, b.B)]
        caches = PagedKV.array([PagedKV.make(planes[2 * i], planes[2 * i + 1], cache, b.num_pages, b.page, kv_heads, hd)
                                for i in range(layers)])
        batch = m.PagedBatch.make(b.B, b.num_rows, up[0], up[1], up[2], b.stride)
        ops.tree_accept(caches, batch, up[3], up[4], up[5], *outs)
        try:
            ctx.sync()
            self.err = None
        except M1MoEError as e:
            self.err = e
        ut = np.uint16 if cache == "bf16" else np.float32
        self.after = [p.download(ut).reshape(shape) for p in planes]
        self.path, self.accepted, self.next, self.past = (o.download(np.int32) for o in outs)
        for x in planes + up + outs:
            x.free()


def check_taken(t, b, parents, drafts, drawn, skip=()):
    want = [p.copy() for p in t.before]
    for s, n in enumerate(b.rows):
        if n == 0:
            assert (t.accepted[s], t.next[s], t.past[s]) == (0, -1, b.kv_len[s])
            continue
        r0, base = int(b.row_start[s]), int(b.kv_len[s]) - n
        way = accept_ref(parents[r0:r0 + n], drafts[r0:r0 + n], drawn[r0:r0 + n])
        assert t.path[r0:r0 + n].tolist() == way + [-1] * (n - len(way))
        assert (t.accepted[s], t.next[s], t.past[s]) == (len(way), drawn[r0 + way[-1]], base + len(way))
        pg, sl = b.cell(s, base + np.array(way))
        to_pg, to_sl = b.cell(s, base + np.arange(len(way)))
        for w, p in zip(want, t.before):
            for i in range(len(way)):
                if (s, way[i]) not in skip and (s, i) not in skip:
                    w[to_pg[i], to_sl[i]] = p[pg[i], sl[i]]
    assert all(np.array_equal(a, w) for a, w in zip(t.after, want))
    assert np.all(t.path[b.T:] == 55)


def drafted(rng, b, parents, often=0.8):
    """Tokens, drawn ones mostly those of one of the row's drafts, some drafts twice."""
    drafts, drawn = rng.integers(0, 50, b.num_rows), rng.integers(0, 50, b.num_rows)
    for s, n in enumerate(b.rows):
        r0 = int(b.row_start[s])
        for i in rng.permutation(np.arange(1, n)) if n > 1 else []:
            if rng.random() < often and parents[r0 + i] >= 0:
                drawn[r0 + parents[r0 + i]] = drafts[r0 + i]
    return drafts.astype(np.int32), drawn.astype(np.int32)


@pytest.mark.parametrize("cache", ["f32", "bf16"])
@pytest.mark.parametrize("kv_heads,hd,page,layers", [(1, 64, 8, 1), (2, 128, 16, 3), (24, 64, 64, 2), (16, 256, 8, 1)])
def test_accept(dev, cache, kv_heads, hd, page, layers):
    rng = np.random.default_rng(kv_heads)
    b = Batch(rng, [1, 26, 0, 64, 7, 256, 2, 100], [0, 5, 9, 31, 70, 0, 64, 17], page, pad=3)
    for chain in (0.3, 0.95):
        parents, _, _ = trees(rng, b, chain)
        drafts, drawn = drafted(rng, b, parents, 0.95)
        say(f"accept {cache} {kv_heads}x{hd} page {page} chain {chain}")
        t = Taken(dev, b, parents, drafts, drawn, kv_heads, hd, cache, layers, 4)
        assert t.err is None
        check_taken(t, b, parents, drafts, drawn)


def test_accept_most_caches_and_long_paths(dev):
    """64 caches; a path of all 256 rows, one of every second row (each move's source is free for
    a later one's target), and drafts that stand twice under one parent."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [256, 255, 6], [3, 8, 1], 16)
    par = [list(range(-1, 255)), [-1] + [max(0, i - 2) if i % 2 == 0 else i - 1 for i in range(1, 255)],
           [-1, 0, 0, 2, 1, 1]]
    parents = np.array(sum(par, []), np.int32)
    drafts = np.full(b.T, 7, np.int32)
    drafts[256:511] = np.arange(255)
    drawn = np.full(b.T, 7, np.int32)
    drawn[256:511] = np.arange(255) + 2
    say("accept 64 caches")
    t = Taken(dev, b, parents, drafts, drawn, 1, 64, "bf16", 64, 5)
    assert t.err is None
    check_taken(t, b, parents, drafts, drawn)
    assert t.accepted.tolist() == [256, 128, 3] and t.path[511:517].tolist() == [0, 1, 4, -1, -1, -1]


def test_accept_reports_what_is_wrong(dev):
    rng = np.random.default_rng(8)

    def case(rows, past):
        b = Batch(rng, rows, past, 8)
        parents = np.array([i - 1 for n in rows for i in range(n)], np.int32)
        return b, parents, np.zeros(b.T, np.int32), np.zeros(b.T, np.int32)
    say("accept wrong batches")
    # a parent that is not lower than its row counts as none
    b, parents, drafts, drawn = case([5, 5], [9, 2])
    parents[3], parents[5] = 3, 1
    t = Taken(dev, b, parents, drafts, drawn, 1, 64, "f32", 2, 9)
    assert t.err is not None and "tree" in str(t.err)
    fixed = parents.copy()
    fixed[[3, 5]] = -1
    check_taken(t, b, fixed, drafts, drawn)
    # rows past 256, a length out of range
    b, parents, drafts, drawn = case([257, 4, 3], [0, 6, 1])
    b.kv_len[2] = b.stride * 8 + 1
    t = Taken(dev, b, parents, drafts, drawn, 1, 64, "f32", 1, 9)
    assert t.err is not None
    assert t.accepted.tolist() == [0, 4, 0] and t.next.tolist() == [-1, 0, -1]
    assert t.past.tolist() == [257, 10, b.stride * 8 + 1] and np.all(t.path[:257] == 55)
    assert all(np.array_equal(x, y) for x, y in zip(t.after, t.before))     # (chains: nothing moves)
    # pages outside the cache: those moves are left out
    b, _, drafts, drawn = case([20, 20], [0, 8])
    parents = np.array(2 * [-1] + [0] * 18 + 2 * [-1] + [0] * 18, np.int32)
    parents[[12, 32]], parents[[19, 39]] = 2, 12
    b.table[0, 1] = b.num_pages      # rows 8 .. 15 of the first tree
    t = Taken(dev, b, parents, drafts, drawn, 1, 64, "f32", 1, 9)
    assert t.err is not None and "page" in str(t.err)
    skip = {(0, i) for i in range(8, 16)}
    b.table[0, 1] = 0
    check_taken(t, b, parents, drafts, drawn, skip)
    dev[0].sync()


# ---- products with 4-bit weights -----------------------------------------------------------

def product(dev, x, w, s, b, group, x_dtype="f32", y_dtype="f32", residual=None, pad=0, inplace=False):
    """y of one call; x and y as columns of wider rows with `pad`."""
    ctx, ops = dev
    T, K, N = x.shape[0], x.shape[1], w.shape[0]
    xs, ys = K + pad, (N + 7) // 8 * 8 + pad
    xb = as_dtype(np.full((T, xs), np.nan), x_dtype)
    xb[:, :K] = x
    yb = as_dtype(np.full((T, ys), 3.0), y_dtype)
    rb = None
    if residual is not None:
        rb = as_dtype(np.full((T, ys), np.nan), y_dtype)
        rb[:, :N] = residual
        if inplace:
            yb[:, :N] = residual
    held = [ctx.to_device(a) for a in (xb, w, s, b, yb)]
    dr = None if rb is None else held[4] if inplace else ctx.to_device(rb)
    ops.matmul_q4(Q4Weights.make(held[1], held[2], held[3], N, K, group), held[0], x_dtype, xs, T, held[4], y_dtype, ys,
                  dr)
    ctx.sync()
    y = f64(held[4].download(np.uint16 if y_dtype == "bf16" else np.float32)).reshape(T, ys)
    for h in held + ([dr] if dr is not None and not inplace else []):
        h.free()
    assert np.all(y[:, N:] == 3.0)
    return y[:, :N]


def check_product(y, x, w, s, b, group, y_dtype, residual=None):
    dense, size = q4_dense(w, s, b, group)
    ref = f64(x) @ dense.T
    if residual is not None:
        ref = ref + f64(residual)
    bound = q4_bound(f64(x), size, ref, group, y_dtype)
    assert np.all(np.isfinite(y))
    worst = np.max(np.abs(y - ref) / bound)
    assert worst <= 1.0, worst
    return ref


KINDS = [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")]


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("group,rows,cols", [(64, 40, 256), (64, 129, 2048), (32, 100, 352), (128, 16, 128),
                                             (32, 1, 32), (64, 7, 64), (128, 300, 1152), (32, 48, 4096),
                                             (64, 513, 192)])
def test_q4(dev, kinds, group, rows, cols):
    rng = np.random.default_rng(rows)
    w, s, b = q4_weights(rng, rows, cols, group)
    dense, _ = q4_dense(w, s, b, group)
    for T in (1, 2, 3, 5, 8, 9, 16, 17, 33, 64, 65, 130):
        x = as_dtype(rng.normal(0, 1, (T, cols)), kinds[0])
        r = as_dtype(rng.normal(0, 1, (T, rows)), kinds[1]) if T % 2 else None
        say(f"q4 {kinds} group {group} {rows} x {cols}, {T} tokens")
        y = product(dev, x, w, s, b, group, *kinds, residual=r, pad=8 * (T % 3), inplace=T % 4 == 1)
        ref = check_product(y, x, w, s, b, group, kinds[1], r)
        if kinds[1] == "f32":
            # (roundings are independent: about 16 of 2^-24 in a group's sum of x n, which is twice the
            # size of its x w, as many of the groups' sum; 2^-23 of an f32 x.  Against the size
            # that sums of independent x w have, as a single result may cancel)
            size = np.sqrt(f64(x) ** 2 @ (dense ** 2).T + (0 if r is None else f64(r) ** 2))
            assert np.linalg.norm(y - ref) < 2e-6 * np.linalg.norm(size)


@pytest.mark.parametrize("tokens", [1, 4, 20, 70, 300])
@pytest.mark.parametrize("kinds", KINDS)
def test_q4_wide_and_tall(dev, kinds, tokens):
    """Many rows of few columns, few rows of many."""
    rng = np.random.default_rng(tokens)
    for rows, cols, group in ((9000, 256, 64), (24, 14336, 128), (70, 65536, 32)):
        if rows * cols * tokens > 4e8:
            continue
        w, s, b = q4_weights(rng, rows, cols, group)
        x = as_dtype(rng.normal(0, 1, (tokens, cols)), kinds[0])
        say(f"q4 {kinds} {rows} x {cols}, {tokens} tokens")
        y = product(dev, x, w, s, b, group, *kinds)
        check_product(y, x, w, s, b, group, kinds[1])


@pytest.mark.parametrize("tokens", [1, 9, 40])
def test_q4_of_a_quantizer(dev, tokens):
    """What m1moe_quantize_4bit makes of normal weights, and how near the product is to theirs."""
    rng = np.random.default_rng(21)
    for group in (32, 64, 128):
        dense = rng.normal(0, 0.02, (200, 1024)).astype(np.float32)
        w, s, b = quantize_4bit(dense, group)
        x = rng.normal(0, 1, (tokens, 1024)).astype(np.float32)
        y = product(dev, x, w.reshape(200, -1), s.reshape(200, -1), b.reshape(200, -1), group)
        check_product(y, x, w.reshape(200, -1), s.reshape(200, -1), b.reshape(200, -1), group, "f32")
        # (a step is about 1 / 15 of the range, at most 8 deviations: 0.16 deviations rms)
        assert rel_l2(y, x.astype(np.float64) @ dense.T.astype(np.float64)) < 0.2


@pytest.mark.parametrize("tokens", [1, 6, 12, 50])
@pytest.mark.parametrize("x_dtype", ["f32", "bf16"])
def test_q4_sizes_of_values(dev, tokens, x_dtype):
    """Rows of very small and very large values, of zeros, and of values that differ by 2^30."""
    rng = np.random.default_rng(tokens)
    w, s, b = q4_weights(rng, 70, 640, 64)
    x = rng.normal(0, 1, (tokens, 640))
    scale = 2.0 ** np.array([0, -100, 90, -30, 60, -120])[np.arange(tokens) % 6]
    x = x * scale[:, None]
    x[0] *= 2.0 ** rng.integers(-30, 1, 640)
    if tokens > 3:
        x[3] = 0
    x = as_dtype(x, x_dtype)
    say(f"q4 sizes {x_dtype}, {tokens} tokens")
    y = product(dev, x, w, s, b, 64, x_dtype)
    check_product(y, x, w, s, b, 64, "f32")
    if tokens > 3:
        assert np.all(y[3] == 0)


@pytest.mark.parametrize("tokens", [3, 40])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_q4_what_is_not_finite_stays_in_its_row(dev, tokens, what):
    rng = np.random.default_rng(tokens)
    w, s, b = q4_weights(rng, 50, 512, 64)
    s[7, 3], b[9, 0] = bf16(np.full(1, what))[0], bf16(np.full(1, what))[0]
    x = rng.normal(0, 1, (tokens, 512)).astype(np.float32)
    x[1, 77] = what
    y = product(dev, x, w, s, b, 64)
    fine_t, fine_n = [t for t in range(tokens) if t != 1], [n for n in range(50) if n not in (7, 9)]
    assert not np.isfinite(y[1]).any() and not np.isfinite(y[:, [7, 9]]).any()
    check_product(y[np.ix_(fine_t, fine_n)], x[fine_t], w[fine_n], s[fine_n], b[fine_n], 64, "f32")


@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("tokens,rows,cols,group", [(500, 9000, 1216, 64), (33, 5000, 1024, 128), (290, 9300, 544, 32),
                                                    (12, 700, 4736, 64), (32, 260, 8192, 128)])
def test_q4_shared_columns(dev, tokens, rows, cols, group, kinds):
    """Tiles behind the last whole round, and tiles too few for the card, whose columns workgroups
    share: in one order whoever is last."""
    rng = np.random.default_rng(tokens)
    w, s, b = q4_weights(rng, rows, cols, group)
    x = as_dtype(rng.normal(0, 1, (tokens, cols)), kinds[0])
    say(f"q4 shared {kinds} {tokens} x {rows} x {cols}")
    y = product(dev, x, w, s, b, group, *kinds)
    check_product(y, x, w, s, b, group, kinds[1])
    for _ in range(3):
        assert np.array_equal(product(dev, x, w, s, b, group, *kinds), y)


@pytest.mark.parametrize("tokens,kinds", [(1, KINDS[0]), (4, KINDS[2]), (6, KINDS[0]), (20, KINDS[1]), (32, KINDS[0])])
@pytest.mark.parametrize("rows", [32790, 49150, 66001])
def test_q4_rows_for_every_wave(dev, rows, tokens, kinds):
    """Workgroups of 9 to 16 waves."""
    rng = np.random.default_rng(rows + tokens)
    w, s, b = q4_weights(rng, rows, 192, 64)
    x = as_dtype(rng.normal(0, 1, (tokens, 192)), kinds[0])
    say(f"q4 {kinds} {rows} rows, {tokens} tokens")
    check_product(product(dev, x, w, s, b, 64, *kinds), x, w, s, b, 64, kinds[1])


@pytest.mark.parametrize("tokens", [2, 7, 14, 30, 45])
def test_q4_sums_past_the_largest_float(dev, tokens):
    """Groups whose x add up to more than an f32 holds, with results that one does."""
    rng = np.random.default_rng(tokens)
    w, s, b = q4_weights(rng, 70, 640, 64, sigma=0.002)
    x = np.full((tokens, 640), 3e38, np.float32) * (1 - 0.1 * rng.random((tokens, 640))).astype(np.float32)
    ref = f64(x) @ q4_dense(w, s, b, 64)[0].T
    assert np.abs(ref).max() < 3.3e38 and f64(x)[:, :64].sum() > 1e40
    say(f"q4 large sums, {tokens} tokens")
    check_product(product(dev, x, w, s, b, 64), x, w, s, b, 64, "f32")


@pytest.mark.parametrize("rows,cols,group", [(3, 128, 64), (5, 64, 64), (1, 128, 128)])
def test_q4_of_most_tokens(dev, rows, cols, group):
    """Less than a unit's groups, and a little more."""
    rng = np.random.default_rng(rows)
    w, s, b = q4_weights(rng, rows, cols, group)
    x = rng.normal(0, 1, (65536, cols)).astype(np.float32)
    say(f"q4 65536 tokens {rows} x {cols}")
    check_product(product(dev, x, w, s, b, group), x, w, s, b, group, "f32")


def test_q4_of_many_tiles(dev):
    """More workgroups than one dimension of a grid takes here (17262), the last of them shared."""
    rng = np.random.default_rng(9)
    T, N, K = 2001, 70001, 64
    w, s, b = q4_weights(rng, N, K, 32)
    x = as_dtype(rng.normal(0, 1, (T, K)), "bf16")
    say(f"q4 {T} x {N} x {K}")
    y = product(dev, x, w, s, b, 32, "bf16", "bf16")
    t = np.r_[0:40, 1000:1040, 1960:2001]
    n = np.r_[0:300, 35000:35300, 69700:70001]
    check_product(y[np.ix_(t, n)], x[t], w[n], s[n], b[n], 32, "bf16")
    sums = np.abs(y).sum(1), np.abs(y).sum(0)
    assert sums[0].min() > 0 and sums[1].min() > 0


class Product:
    """A call whose operands stay on the device."""

    def __init__(self, dev, tokens, rows, cols, group=64):
        self.ctx, self.ops = dev
        rng = np.random.default_rng(tokens)
        self.w, self.s, self.b = q4_weights(rng, rows, cols, group)
        self.x = rng.normal(0, 1, (tokens, cols)).astype(np.float32)
        self.shape, self.group = (tokens, rows), group
        self.held = [self.ctx.to_device(a) for a in (self.w, self.s, self.b, self.x, np.zeros((tokens, rows), np.float32))]
        self.weights = Q4Weights.make(*self.held[:3], rows, cols, group)

    def __call__(self):
        (t, n), k = self.shape, self.x.shape[1]
        self.ops.matmul_q4(self.weights, self.held[3], "f32", k, t, self.held[4], "f32", n)

    def result(self):
        """y, and zeros in its place."""
        self.ctx.sync()
        y = self.held[4].download(np.float32).reshape(self.shape)
        self.held[4].upload(np.zeros(self.shape, np.float32))
        return y

    def free(self):
        for h in self.held:
            h.free()


def test_q4_graphs_share_a_workspace():
    """Two graphs and eager calls on one context's workspace, in turns; a call that needs more of it
    is refused in a capture, and behind it the graphs of the smaller one are."""
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    dev = ctx, DenseOps(ctx)
    big, small, few, huge, alone = (Product(dev, *a) for a in ((100, 512, 1024), (40, 96, 2048), (10, 48, 4096),
                                                               (400, 512, 1024), (1, 48, 256)))
    say("q4 capture without a workspace")
    ctx.graph_begin()
    with pytest.raises(M1MoEError) as e:
        big()
    assert e.value.code == _lib.M1MOE_ERR_INVALID and "capture" in str(e.value)
    alone()                             # (needs none)
    one = ctx.graph_end()
    one.launch()
    want = []
    check_product(alone.result(), alone.x, alone.w, alone.s, alone.b, 64, "f32")
    for p in (big, small, few):
        p()
        want.append(p.result())
        check_product(want[-1], p.x, p.w, p.s, p.b, p.group, "f32")
    say("q4 two graphs")
    ctx.graph_begin()
    big(), few()
    one = ctx.graph_end()
    ctx.graph_begin()
    few(), small(), few()
    two = ctx.graph_end()
    for i in range(3):
        one.launch(), two.launch()
        assert np.array_equal(big.result(), want[0]) and np.array_equal(small.result(), want[1]), i
        assert np.array_equal(few.result(), want[2]), i
        two.launch(), small(), one.launch()
        assert np.array_equal(small.result(), want[1]) and np.array_equal(few.result(), want[2]), i
        assert np.array_equal(big.result(), want[0]), i
    huge()
    check_product(huge.result(), huge.x, huge.w, huge.s, huge.b, 64, "f32")
    with pytest.raises(M1MoEError) as e:
        one.launch()
    assert "capture it again" in str(e.value)
    big()
    assert np.array_equal(big.result(), want[0])
    del one, two
    for p in (big, small, few, huge, alone):
        p.free()
    ctx.close()


def test_q4_rows_past_32_bits(dev):
    """x and y whose last rows lie past 2^32 bytes."""
    ctx, ops = dev
    rng = np.random.default_rng(30)
    w, s, b = q4_weights(rng, 40, 128, 64)
    T, stride = 3, 1 << 29      # f32: 2 GiB a row
    dx, dy = ctx.alloc(4 * (2 * stride + 128)), ctx.alloc(4 * (2 * stride + 128))
    held = [ctx.to_device(a) for a in (w, s, b)]
    x = rng.normal(0, 1, (T, 128)).astype(np.float32)
    lib = ctx.lib
    for t in range(T):
        row = np.ascontiguousarray(x[t])
        _lib.check(lib.m1moe_copy_h2d(ctx.handle, dx.addr + 4 * t * stride, row.ctypes.data, row.nbytes), "copy")
    say("q4 far rows")
    ops.matmul_q4(Q4Weights.make(*held, 40, 128, 64), dx, "f32", stride, T, dy, "f32", stride)
    ctx.sync()
    y = np.zeros((T, 40), np.float32)
    for t in range(T):
        row = np.zeros(40, np.float32)
        _lib.check(lib.m1moe_copy_d2h(ctx.handle, row.ctypes.data, dy.addr + 4 * t * stride, row.nbytes), "copy")
        y[t] = row
    for h in held + [dx, dy]:
        h.free()
    check_product(y.astype(np.float64), x, w, s, b, 64, "f32")


# ---- together --------------------------------------------------------------------------------

class Step:
    """A verification step of one layer: plan, products for q, k and v, append, attention, output
    product onto the residual, logits, drawn tokens, acceptance."""

    def __init__(self, dev, seed, rows=(12, 1, 30), past=(20, 7, 64), cache="bf16"):
        self.ctx, self.ops = dev
        rng = self.rng = np.random.default_rng(seed)
        ctx = self.ctx
        self.heads, self.kv_heads, self.hd, self.hidden, self.vocab = 4, 2, 64, 128, 96
        h, g, hd, H, V = self.heads, self.kv_heads, self.hd, self.hidden, self.vocab
        self.b = b = Batch(rng, rows, past, 8, pad=1)
        self.parents, self.mask, self.depth = trees(rng, b)
        self.kc, self.vc = cache_of(rng, b, g, hd, cache)
        self.d = d = Held(ctx, b, self.kc, self.vc, cache, g, hd)
        up, T, n = d.up, b.num_rows, (h + 2 * g) * hd
        self.x = rng.normal(0, 1, (T, H)).astype(np.float32)
        self.weights = [q4_weights(rng, r, c, 64, 0.05) for r, c in ((n, H), (H, h * hd), (V, H))]
        self.q4 = [Q4Weights.make(up(w), up(s), up(bb), w.shape[0], 8 * w.shape[1], 64) for w, s, bb in self.weights]
        self.drafts = rng.integers(0, V, T).astype(np.int32)
        z = lambda *shape, dt=np.float32: up(np.zeros(shape, dt))  # noqa: E731
        self.dx, self.qkv, self.q, self.o, self.y, self.logits = (up(self.x), z(T, n), z(T, h * hd), z(T, h * hd),
                                                                  z(T, H), z(T, V))
        self.dmask, self.ddepth = z(T, words_of(b), dt=np.uint64), z(T, dt=np.int32)
        self.dpar, self.ddraft, self.tok = up(self.parents), up(self.drafts), z(T, dt=np.int32)
        self.u, self.temp = up(rng.random(T).astype(np.float32)), up(np.full(T, 0.5, np.float32))
        self.topk = up(np.full(T, 4, np.int32))
        self.outs = [z(T, dt=np.int32)] + [z(b.B, dt=np.int32) for _ in range(3)]
        self.freq = up(rope_frequencies(1e4, hd)[0])
        self.caches = PagedKV.array([d.kv])

    def __call__(self):
        o, d, b, n = self.ops, self.d, self.b, (self.heads + 2 * self.kv_heads) * self.hd
        h, g, hd, H, V, T = self.heads, self.kv_heads, self.hd, self.hidden, self.vocab, b.num_rows
        W = words_of(b)
        o.tree_plan(b.B, T, d.start, self.dpar, W, self.dmask, self.ddepth)
        o.matmul_q4(self.q4[0], self.dx, "f32", H, T, self.qkv, "f32", n)
        o.tree_append(d.kv, d.batch, KVAppend.make(
            "f32", h, self.qkv, self.qkv.addr + 4 * h * hd, self.qkv.addr + 4 * (h + g) * hd, n, n, n, self.q, h * hd,
            rotary_dim=hd, inv_freq=self.freq), self.ddepth)
        o.tree_attention(d.kv, d.batch, self.dmask, W, self.q, h * hd, self.o, h * hd, "f32", h)
        o.matmul_q4(self.q4[1], self.o, "f32", h * hd, T, self.y, "f32", H, residual=self.dx)
        o.matmul_q4(self.q4[2], self.y, "f32", H, T, self.logits, "f32", V)
        o.sample(self.logits, T, V, V, SampleParams.make(self.u, self.temp, self.topk), self.tok)
        o.tree_accept(self.caches, d.batch, self.dpar, self.ddraft, self.tok, *self.outs)

    def results(self):
        self.ctx.sync()
        f, i = np.float32, np.int32
        return ([t.download(f) for t in (self.qkv, self.q, self.o, self.y, self.logits)] +
                [t.download(i) for t in [self.tok] + self.outs] +
                [self.d.k.download(np.uint8), self.d.v.download(np.uint8)])

    def restore(self):
        self.d.k.upload(self.kc)
        self.d.v.upload(self.vc)

    def draft_well(self):
        """Drafts that are mostly drawn: the tokens that a first pass draws do not depend on them."""
        self()
        tok, b = self.results()[5], self.b
        for r in range(b.T):
            s = int(np.searchsorted(b.row_start, r, side="right")) - 1
            if self.parents[r] >= 0 and self.rng.random() < 0.7:
                self.drafts[r] = tok[int(b.row_start[s]) + self.parents[r]]
        self.ddraft.upload(self.drafts)
        self.restore()


def test_a_step_together(dev):
    """The accepted rows' cache is what the plain append of the path's tokens stores, the layer's
    results at them are those of plain paged attention over it, and the path is the drawn tokens'."""
    say("a step over drafted tokens")
    st = Step(dev, 40, cache="f32")
    b, h, g, hd = st.b, st.heads, st.kv_heads, st.hd
    st.draft_well()
    st()
    qkv, q, o, y, logits, tok, path, accepted, nxt, past = st.results()[:10]
    kc, vc = (t.download(np.float32).reshape(st.kc.shape) for t in (st.d.k, st.d.v))
    n = (h + 2 * g) * hd
    qkv, o = qkv.reshape(-1, n), o.reshape(-1, h, hd)
    assert accepted.max() > 1
    # the same tokens as plain turns
    rows = [int(a) for a in accepted]
    p = Batch(st.rng, rows, [int(x) - int(a) for x, a in zip(past, accepted)], 8, pages=b.num_pages)
    p.table, p.stride = b.table, b.stride
    at = [int(b.row_start[s]) + int(path[int(b.row_start[s]) + i]) for s in range(b.B) for i in range(rows[s])]
    for s in range(b.B):
        r0 = int(b.row_start[s])
        way = accept_ref(st.parents[r0:r0 + b.rows[s]], st.drafts[r0:r0 + b.rows[s]], tok[r0:r0 + b.rows[s]])
        assert path[r0:r0 + b.rows[s]].tolist() == way + [-1] * (b.rows[s] - len(way))
        assert nxt[s] == tok[r0 + way[-1]]
    d = Held(st.ctx, p, st.kc, st.vc, "f32", g, hd)
    turn = d.up(qkv[at])
    qq, oo = d.up(np.zeros((p.T, h * hd), np.float32)), d.up(np.zeros((p.T, h * hd), np.float32))
    st.ops.kv_append(d.kv, d.batch, KVAppend.make("f32", h, turn, turn.addr + 4 * h * hd, turn.addr + 4 * (h + g) * hd, n,
                                                  n, n, qq, h * hd, rotary_dim=hd, inv_freq=d.up(rope_frequencies(1e4, hd)[0])))
    st.ops.paged_attention(d.kv, d.batch, qq, h * hd, oo, h * hd, "f32", h)
    st.ctx.sync()
    k2, v2 = (t.download(np.float32).reshape(st.kc.shape) for t in (d.k, d.v))
    o2 = oo.download(np.float32).reshape(-1, h, hd)
    for s in range(p.B):
        pg, sl = p.cell(s, np.arange(int(p.kv_len[s])))
        assert np.array_equal(kc[pg, sl], k2[pg, sl]) and np.array_equal(vc[pg, sl], v2[pg, sl])
    d.free()
    st.d.free()
    # (two results within the bound of f32 sums of one value)
    assert rel_l2(o[at], o2) < 2e-6


@pytest.mark.parametrize("seed", [41, 42])
def test_a_step_captured_and_replayed(dev, seed):
    """A graph of the whole step, replayed between other calls, gives the eager step's bits."""
    ctx, ops = dev
    st, other = Step(dev, seed), Step(dev, seed + 10, rows=(40, 3), past=(5, 200))
    st.draft_well()
    st()
    want = st.results()
    other()
    ctx.sync()
    st.restore()
    say("captured step")
    ctx.graph_begin()
    st()
    graph = ctx.graph_end()
    for i in range(3):
        st.restore()
        graph.launch()
        got = st.results()
        assert all(np.array_equal(a, c) for a, c in zip(got, want)), i
        other.restore()
        other()
        ctx.sync()
    del graph
    st.d.free()
    other.d.free()
