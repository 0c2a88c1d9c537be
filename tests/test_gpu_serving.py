"""GPU parity of the paged KV cache, attention over it and the sampler against
f64 references (serving_cases.py), through the C ABI.  Bounds are elementwise
and derived there (attention_bound) or beside the test; sampled tokens are equal."""
import ctypes
import gc
import math

import numpy as np
import pytest

import m1moe_amd as m
from m1moe_amd import KVAppend, M1MoEError, PagedBatch, PagedKV, SampleParams, _lib, synth
from m1moe_amd.decoder import DenseOps

from cases import rel_l2, say
from serving_cases import (Batch, append_ref, as_dtype, attention_bound, attention_ref, bf16, f64,
                           sample_ref)

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")]


@pytest.fixture(scope="module")
def dev():
    say("serving context")
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    yield ctx, DenseOps(ctx)
    ctx.close()


class Held:
    """Device copies of a batch and a cache, freed together."""

    def __init__(self, ctx, b: Batch, kc, vc, cache, kv_heads, hd):
        self.ctx, self.b = ctx, b
        up = ctx.to_device
        self.start, self.len, self.table = up(b.row_start), up(b.kv_len), up(b.table)
        self.pre = up(b.prefix_table) if b.prefix else None
        self.k, self.v = up(kc), up(vc)
        self.kv = PagedKV.make(self.k, self.v, cache, kc.shape[0], b.page, kv_heads, hd)
        self.batch = PagedBatch.make(b.B, b.num_rows, self.start, self.len, self.table, b.stride,
                                     b.prefix, self.pre)
        self.more = []

    def up(self, a):
        self.more.append(self.ctx.to_device(a))
        return self.more[-1]

    def free(self):
        for x in [self.start, self.len, self.table, self.k, self.v, self.pre] + self.more:
            if x is not None:
                x.free()


def cache_of(rng, b, kv_heads, hd, cache, fill=None):
    """Random where some sequence has a position, `fill` (or random) elsewhere."""
    shape = (b.num_pages, b.page, kv_heads, hd)
    kc, vc = (as_dtype(rng.normal(0, 1, shape), cache) for _ in range(2))
    if fill is not None:
        used = np.zeros(shape[:2], bool)
        for s in range(b.B):
            pg, sl = b.cell(s, np.arange(int(b.kv_len[s])))
            used[pg, sl] = True
        bad = as_dtype(np.full(1, fill), cache)[0]
        kc[~used], vc[~used] = bad, bad
    return kc, vc


def attend(dev, b, heads, kv_heads, hd, types, seed, fill=np.nan, mark=7.0):
    """(output rows, the padding's rows, f64 reference, bound) of one call."""
    ctx, ops = dev
    rng = np.random.default_rng(seed)
    x, cache = types
    q = as_dtype(rng.normal(0, 1, (b.num_rows, heads * hd)), x)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache, fill)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    out = d.up(as_dtype(np.full((b.num_rows, heads * hd), mark), x))
    ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, x, heads)
    ctx.sync()
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
    d.free()
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    return got[:b.T], got[b.T:], ref, attention_bound(ref, mag, top, hd, x)


def check_close(got, ref, bound, dtype):
    assert np.all(np.isfinite(got))
    worst = np.max(np.abs(got - ref) / bound) if ref.size else 0.0
    assert worst <= 1.0, worst
    # (in the 2-norm the roundings of a row's f32 sums are independent: 128 of them of
    # 2^-24, scores up to a few units; bf16: two roundings of at most 2^-8)
    assert rel_l2(got, ref) < (1e-5 if dtype == "f32" else 2.0 ** -7)


# ---- attention ---------------------------------------------------------------------------

@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 4, 128), (8, 2, 128), (7, 1, 64), (6, 2, 256), (64, 1, 64),
                                               (3, 3, 256), (16, 2, 64)])
def test_attention_single_tokens(dev, types, heads, kv_heads, hd):
    """Steps: one row each, lengths around the tile's and the pages' ends."""
    rng = np.random.default_rng(1)
    past = [0, 1, 7, 8, 30, 31, 32, 33, 127, 128, 255, 256, 300, 700]
    b = Batch(rng, [1] * len(past), past, 16)
    say(f"attention step {types} {heads}/{kv_heads}x{hd}")
    got, _, ref, bound = attend(dev, b, heads, kv_heads, hd, types, 2)
    check_close(got, ref, bound, types[0])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(4, 4, 128, 8), (8, 2, 128, 64), (12, 4, 64, 32),
                                                    (5, 1, 256, 256), (40, 1, 128, 16)])
def test_attention_ragged_rows(dev, types, heads, kv_heads, hd, page):
    """Prompts, turns, single tokens and empty sequences in one call, with rows
    behind the last sequence that stay as they were."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [70, 0, 1, 33, 5, 0, 129, 2], [0, 9, 400, 60, 1, 0, 20, 1000], page, pad=4)
    say(f"attention ragged {types} {heads}/{kv_heads}x{hd} page {page}")
    got, rest, ref, bound = attend(dev, b, heads, kv_heads, hd, types, 4)
    check_close(got, ref, bound, types[0])
    assert np.all(rest == 7.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("prefix", [1, 31, 32, 33, 100, 512, 777])
def test_attention_shared_prefix(dev, types, prefix):
    """The prefix in its own pages; the sequences' table entries of it point at
    pages of NaN."""
    rng = np.random.default_rng(prefix)
    rows = [1, 1, 3, 0, 1, 40, 1, 1]
    b = Batch(rng, rows, [prefix + p for p in (0, 5, 64, 2, 31, 10, 300, 1)], 16, prefix=prefix, pad=2)
    say(f"attention prefix {prefix} {types}")
    got, rest, ref, bound = attend(dev, b, 8, 2, 128, types, prefix + 1)
    check_close(got, ref, bound, types[0])
    assert np.all(rest == 7.0)


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 2, 64), (4, 2, 256), (24, 3, 128)])
def test_attention_prefix_of_many_rows(dev, heads, kv_heads, hd):
    rng = np.random.default_rng(8)
    b = Batch(rng, [1] * 70 + [30], [1100 + int(x) for x in rng.integers(0, 40, 71)], 32, prefix=1100)
    say(f"attention prefix many {heads}/{kv_heads}x{hd}")
    got, _, ref, bound = attend(dev, b, heads, kv_heads, hd, ("f32", "bf16"), 9)
    check_close(got, ref, bound, "f32")


@pytest.mark.parametrize("types", TYPES)
def test_attention_long(dev, types):
    """One long sequence shared by many workgroups, beside short ones."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [1, 1, 2], [20000, 3, 5000], 64)
    say(f"attention long {types}")
    got, _, ref, bound = attend(dev, b, 4, 1, 128, types, 11, fill=None)
    check_close(got, ref, bound, types[0])


def test_attention_one_position(dev):
    """The only visible position is the row's own: out = v exactly."""
    rng = np.random.default_rng(12)
    b = Batch(rng, [1, 1], [0, 0], 8)
    for types in TYPES:
        got, _, ref, _ = attend(dev, b, 4, 2, 64, types, 13)
        assert np.array_equal(got, ref)


def test_attention_most_sequences(dev):
    rng = np.random.default_rng(14)
    rows = rng.integers(0, 3, 1024)
    b = Batch(rng, rows, rng.integers(0, 60, 1024), 8)
    say("attention 1024 sequences")
    got, _, ref, bound = attend(dev, b, 2, 1, 64, ("f32", "f32"), 15)
    check_close(got, ref, bound, "f32")


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_attention_infinities_later(dev, types, what):
    """Values of later rows of the same call that are not finite do not reach the
    earlier rows, and reach their own and the later ones."""
    ctx, ops = dev
    rng = np.random.default_rng(16)
    heads, kv_heads, hd = 4, 2, 64
    b = Batch(rng, [40, 1], [10, 33], 16)
    x, cache = types
    q = as_dtype(rng.normal(0, 1, (b.T, heads * hd)), x)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache)
    pg, sl = b.cell(0, np.array([35]))
    vc[pg, sl, 0, 3] = as_dtype(np.full(1, what), cache)[0]
    pg, sl = b.cell(0, np.array([40]))
    kc[pg, sl, 1] = as_dtype(np.full(hd, what), cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    out = d.up(np.zeros((b.T, heads * hd), np.uint16 if x == "bf16" else np.float32))
    say(f"attention infinities {what} {types}")
    ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, x, heads)
    ctx.sync()
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
    d.free()
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    fine = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~fine & ~np.isnan(ref)], ref[~fine & ~np.isnan(ref)])
    with np.errstate(all="ignore"):
        bound = attention_bound(ref, mag, top, hd, x)
        # (a row that an infinity reached at a weight: compared where finite)
        ok = np.abs(got - ref) <= np.where(np.isfinite(bound), bound, np.inf)
    assert np.all(ok[fine])
    assert not fine[25:40, :2, 3].any() and fine[:25].all() and fine[40].all()


def test_attention_huge_values(dev):
    """f32 values above the largest bf16 are computed as they are."""
    ctx, ops = dev
    b = Batch(np.random.default_rng(17), [3], [0], 8)
    q = np.zeros((3, 64), np.float32)
    kc = np.zeros((b.num_pages, 8, 1, 64), np.float32)
    vc = np.full_like(kc, 3.4e38)
    d = Held(ctx, b, kc, vc, "f32", 1, 64)
    out = d.up(np.zeros_like(q))
    ops.paged_attention(d.kv, d.batch, d.up(q), 64, out, 64, "f32", 1)
    ctx.sync()
    got = out.download(np.float32).reshape(3, 64)
    d.free()
    assert np.allclose(got[0], 3.4e38, rtol=1e-6)


def test_attention_strides_and_offsets_past_32_bits(dev):
    """q and out as columns of wider rows; a page whose first element is past 2^31
    elements and 2^32 bytes of the cache."""
    ctx, ops = dev
    rng = np.random.default_rng(18)
    heads, kv_heads, hd, page = 8, 8, 128, 16
    per = page * kv_heads * hd
    pages = (1 << 31) // per + 40
    b = Batch(rng, [1, 2], [100, 200], page, pages=pages)
    b.table[0, 0], b.table[1, 1] = pages - 1, pages - 3
    dk, dv = ctx.alloc(2 * pages * per), ctx.alloc(2 * pages * per)
    small = sorted({int(p) for s in range(2) for p in b.table[s, :-(-int(b.kv_len[s]) // page)]})
    kc = {p: bf16(rng.normal(0, 1, (page, kv_heads, hd))) for p in small}
    vc = {p: bf16(rng.normal(0, 1, (page, kv_heads, hd))) for p in small}
    lib = ctx.lib
    for p in small:
        for base, src in ((dk, kc[p]), (dv, vc[p])):
            src = np.ascontiguousarray(src)
            _lib.check(lib.m1moe_copy_h2d(ctx.handle, base.addr + 2 * p * per, src.ctypes.data, src.nbytes), "copy")
    start, ln, table = ctx.to_device(b.row_start), ctx.to_device(b.kv_len), ctx.to_device(b.table)
    kv = PagedKV.make(dk, dv, "bf16", pages, page, kv_heads, hd)
    batch = PagedBatch.make(2, 3, start, ln, table, b.stride)
    qd = heads * hd
    q = rng.normal(0, 1, (3, qd + 64)).astype(np.float32)
    o = np.full((3, 2 * qd), 5.0, np.float32)
    dq, do = ctx.to_device(q), ctx.to_device(o)
    say("attention far pages, strided rows")
    ops.paged_attention(kv, batch, dq, qd + 64, do, 2 * qd, "f32", heads)
    ctx.sync()
    got = do.download(np.float32).reshape(3, 2 * qd)
    index = {p: i for i, p in enumerate(small)}
    b.table = np.vectorize(lambda p: index.get(int(p), 0))(b.table)
    ref, mag, top = attention_ref(b, np.ascontiguousarray(q[:, :qd]), np.stack([kc[p] for p in small]),
                                  np.stack([vc[p] for p in small]), heads, kv_heads, hd)
    for x in (dk, dv, start, ln, table, dq, do):
        x.free()
    assert np.all(got[:, qd:] == 5.0)
    check_close(got[:, :qd].reshape(3, heads, hd).astype(np.float64), ref,
                attention_bound(ref, mag, top, hd, "f32"), "f32")


def test_attention_equals_the_contiguous_one(dev):
    """One sequence, f32 cache: m1moe_attention_decode's result within the bound."""
    ctx, ops = dev
    rng = np.random.default_rng(19)
    heads, kv_heads, hd, L = 16, 16, 128, 200
    b = Batch(rng, [1], [L - 1], 16)
    q = rng.normal(0, 1, (1, heads * hd)).astype(np.float32)
    kc, vc = cache_of(rng, b, kv_heads, hd, "f32")
    d = Held(ctx, b, kc, vc, "f32", kv_heads, hd)
    pg, sl = b.cell(0, np.arange(L))
    dq, o1, o2 = d.up(q), d.up(np.zeros_like(q)), d.up(np.zeros_like(q))
    ops.paged_attention(d.kv, d.batch, dq, heads * hd, o1, heads * hd, "f32", heads)
    ops.attention_decode(dq, d.up(kc[pg, sl]), d.up(vc[pg, sl]), o2, heads, kv_heads, hd, L)
    ctx.sync()
    a, c = o1.download(np.float32), o2.download(np.float32)
    d.free()
    assert rel_l2(a, c) < 2e-6


@pytest.mark.parametrize("breakage", ["page_low", "page_high", "start", "short", "long", "prefix"])
def test_bad_batches_are_reported(dev, breakage):
    """A sequence out of range is skipped, a bad page is not read; the others are
    right and the next sync reports it."""
    ctx, ops = dev
    rng = np.random.default_rng(20)
    heads, kv_heads, hd = 4, 2, 64
    b = Batch(rng, [1, 2, 1], [40, 50, 30], 16, prefix=20 if breakage == "prefix" else 0)
    q = rng.normal(0, 1, (b.T, heads * hd)).astype(np.float32)
    kc, vc = cache_of(rng, b, kv_heads, hd, "f32")
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    bound = attention_bound(ref, mag, top, hd, "f32")
    bad = 1
    if breakage == "page_low":
        b.table[1, 2] = -1
    elif breakage == "page_high":
        b.table[1, 0] = b.num_pages
    elif breakage == "start":
        b.row_start = np.array([0, 1, 9, 4], np.int32)
        bad = 3            # the second and third sequences' rows
    elif breakage == "short":
        b.kv_len[1] = 1
    elif breakage == "long":
        b.kv_len[1] = b.stride * 16 + 1
    else:
        b.kv_len[1] = 21
    d = Held(ctx, b, kc, vc, "f32", kv_heads, hd)
    out = d.up(np.full((b.T, heads * hd), 3.0, np.float32))
    say(f"attention bad batch {breakage}")
    ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, "f32", heads)
    with pytest.raises(M1MoEError) as e:
        ctx.sync()
    assert e.value.code == _lib.M1MOE_ERR_DEVICE and "paged batch" in str(e.value)
    ctx.sync()   # reported once
    got = out.download(np.float32).reshape(b.T, heads, hd).astype(np.float64)
    d.free()
    keep = [0, 3] if bad == 1 else [0]
    assert np.all(np.abs(got[keep] - ref[keep]) <= bound[keep])
    if not breakage.startswith("page"):
        assert np.all(got[1:3] == 3.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("end", [30, 0, -5, 1 << 30])
def test_bad_last_start_behind_a_prefix(dev, types, end):
    """The last sequence's end lies before its start (or past the rows): it is skipped, and the
    other sequences' rows are right, those past that end too."""
    ctx, ops = dev
    rng = np.random.default_rng(74)
    heads, kv_heads, hd, prefix = 4, 2, 64, 200
    x, cache = types
    b = Batch(rng, [40, 1, 2], [prefix + 3, prefix + 50, prefix + 9], 16, prefix=prefix)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    out = d.up(as_dtype(np.full((b.T, heads * hd), 3.0), x))
    q = as_dtype(rng.normal(0, 1, (b.T, heads * hd)), x)
    say(f"attention bad last start {end} {types}")
    # (what the workspace holds: another call's)
    ops.paged_attention(d.kv, d.batch, d.up(as_dtype(f64(q)[::-1], x)), heads * hd, d.up(np.zeros_like(q)), heads * hd, x, heads)
    starts = b.row_start.copy()
    starts[3] = end
    d.start.upload(starts)
    ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, x, heads)
    with pytest.raises(M1MoEError, match="paged batch"):
        ctx.sync()
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
    d.free()
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    assert np.all(got[41:] == 3.0)
    check_close(got[:41], ref[:41], attention_bound(ref, mag, top, hd, x)[:41], x)


def test_attention_in_a_graph(dev):
    """One captured call serves later lengths: replays with other lengths, eager
    calls between them."""
    ctx, ops = dev
    rng = np.random.default_rng(21)
    heads, kv_heads, hd = 8, 2, 128
    b = Batch(rng, [1, 1, 1], [700, 20, 300], 16)
    q = rng.normal(0, 1, (3, heads * hd)).astype(np.float32)
    kc, vc = cache_of(rng, b, kv_heads, hd, "bf16")
    d = Held(ctx, b, kc, vc, "bf16", kv_heads, hd)
    dq, out = d.up(q), d.up(np.zeros_like(q))

    def call():
        ops.paged_attention(d.kv, d.batch, dq, heads * hd, out, heads * hd, "f32", heads)
    call()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()
    for lens in ([701, 21, 301], [5, 21, 64], [700, 1, 257]):
        b.kv_len = np.array(lens, np.int32)
        d.len.upload(b.kv_len)
        out.upload(np.zeros_like(q))
        say(f"attention graph replay {lens}")
        g.launch()
        ctx.sync()
        got = out.download(np.float32).reshape(3, heads, hd)
        call()
        ctx.sync()
        assert np.array_equal(got, out.download(np.float32).reshape(3, heads, hd))
        ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
        check_close(got.astype(np.float64), ref, attention_bound(ref, mag, top, hd, "f32"), "f32")
    d.free()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (2, 2, 128), (3, 1, 256)])
def test_attention_many_rows_shared_by_workgroups(dev, types, heads, kv_heads, hd):
    """Tiles of many rows, few and one whose keys several workgroups share, alone on the
    device and beside short ones."""
    rng = np.random.default_rng(60)
    for rows, past in (([130], [3000]), ([100, 1, 9, 64], [900, 5, 4000, 0])):
        b = Batch(rng, rows, past, 16)
        say(f"attention cut tiles {types} {heads}/{kv_heads}x{hd} {rows}")
        got, _, ref, bound = attend(dev, b, heads, kv_heads, hd, types, 61)
        check_close(got, ref, bound, types[0])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("slope", [0.02, 0.08, 0.3, -0.3])
def test_attention_scores_that_rise(dev, types, slope):
    """Scores that rise (or fall) with the position, by less and by more per block than what
    a softmax's reference may lag behind its maximum."""
    ctx, ops = dev
    rng = np.random.default_rng(67)
    heads, kv_heads, hd = 4, 2, 64
    x, cache = types
    b = Batch(rng, [1, 90], [900, 300], 16)
    q = as_dtype(np.full((b.T, heads * hd), 0.5) + rng.normal(0, 0.02, (b.T, heads * hd)), x)
    kc, vc = (rng.normal(0, 0.05, (b.num_pages, 16, kv_heads, hd)) for _ in range(2))
    for s in range(2):
        pos = np.arange(int(b.kv_len[s]))
        pg, sl = b.cell(s, pos)
        kc[pg, sl] += (pos * slope / 4)[:, None, None]     # (hd 0.5 / sqrt(hd) = 4)
    kc, vc = as_dtype(kc, cache), as_dtype(vc, cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    out = d.up(np.zeros((b.T, heads * hd), np.uint16 if x == "bf16" else np.float32))
    say(f"attention slope {slope} {types}")
    ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, x, heads)
    ctx.sync()
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
    d.free()
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - ref) <= attention_bound(ref, mag, top, hd, x))


@pytest.mark.parametrize("types", TYPES)
def test_attention_infinities_in_pieces(dev, types):
    """An infinity that only some of a row's pieces meet, in the prefix or behind it."""
    ctx, ops = dev
    rng = np.random.default_rng(62)
    heads, kv_heads, hd, prefix = 2, 2, 64, 600
    x, cache = types
    for where in (100, 2500):
        b = Batch(rng, [1, 40, 2], [4000, 3000, 700], 16, prefix=prefix)
        q = as_dtype(rng.normal(0, 1, (b.T, heads * hd)), x)
        kc, vc = cache_of(rng, b, kv_heads, hd, cache)
        pg, sl = b.cell(1, np.array([where]))
        vc[pg, sl, 0, 3] = as_dtype(np.full(1, np.inf), cache)[0]
        vc[pg, sl, 1, 9] = as_dtype(np.full(1, np.nan), cache)[0]
        d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
        out = d.up(np.zeros((b.T, heads * hd), np.uint16 if x == "bf16" else np.float32))
        say(f"attention infinity at {where} {types}")
        ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, x, heads)
        ctx.sync()
        got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
        d.free()
        ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
        bound = attention_bound(ref, mag, top, hd, x)
        fine = np.isfinite(ref)
        hit = slice(0, b.T) if where < prefix else slice(1, 41)
        assert np.isposinf(ref[hit, 0, 3]).all() and np.isnan(ref[hit, 1, 9]).all()
        assert (~fine).sum() == 2 * (hit.stop - hit.start)
        assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.isposinf(got[hit, 0, 3]).all()
        assert np.all(np.abs(got[fine] - ref[fine]) <= bound[fine])


@pytest.mark.parametrize("types", TYPES)
def test_attention_sequences_share_pages(dev, types):
    """Sequences whose tables name the same pages (a conversation continued twice), and a
    page named twice in one table."""
    ctx, ops = dev
    b = Batch(np.random.default_rng(68), [1, 1, 20], [600, 600, 581], 16)
    b.table[1] = b.table[0]
    b.table[2, :30] = b.table[0, :30]
    b.table[2, 31] = b.table[2, 30]
    say(f"attention shared pages {types}")
    got, _, ref, bound = attend(dev, b, 4, 2, 128, types, 69)
    check_close(got, ref, bound, types[0])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(1024, 16, 64), (256, 256, 256), (512, 8, 128)])
def test_attention_most_heads(dev, types, heads, kv_heads, hd):
    """num_heads * head_dim at its limit."""
    b = Batch(np.random.default_rng(70), [3, 1], [5, 70], 8, prefix=4)
    say(f"attention most heads {types} {heads}/{kv_heads}x{hd}")
    got, _, ref, bound = attend(dev, b, heads, kv_heads, hd, types, 71)
    check_close(got, ref, bound, types[0])


@pytest.mark.parametrize("heads,kv_heads,hd,rows,past,prefix", [
    (4, 2, 64, [60, 9, 1], [300, 900, 40], 0), (2, 2, 128, [200], [1500], 0), (8, 2, 128, [70, 5, 30], [10, 2000, 0], 0),
    (3, 1, 256, [40, 21], [700, 3], 0), (4, 4, 128, [90, 2, 1, 30], [800, 650, 640, 700], 600),
])
def test_attention_bf16_error_beyond_the_rounding(dev, heads, kv_heads, hd, rows, past, prefix):
    """bf16 rows, many of a sequence or few: what the softmax's weights lose beside the rounding of
    the output is two bf16 parts' rest, 2^-16 of each weight and of their sum."""
    b = Batch(np.random.default_rng(72), rows, past, 16, prefix=prefix)
    say(f"attention bf16 weights {heads}/{kv_heads}x{hd} {rows}")
    ctx, ops = dev
    rng = np.random.default_rng(73)
    q = bf16(rng.normal(0, 1, (b.T, heads * hd)))
    kc, vc = cache_of(rng, b, kv_heads, hd, "bf16")
    d = Held(ctx, b, kc, vc, "bf16", kv_heads, hd)
    out = d.up(np.zeros((b.T, heads * hd), np.uint16))
    ops.paged_attention(d.kv, d.batch, d.up(q), heads * hd, out, heads * hd, "bf16", heads)
    ctx.sync()
    got = f64(out.download(np.uint16)).reshape(-1, heads, hd)
    d.free()
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    before = attention_bound(ref, mag, top, hd, "f32") + 2 * 2.0 ** -16 * mag
    assert np.all(np.abs(got - ref) <= before + 2.0 ** -8 * (np.abs(ref) + before))


def test_two_graphs_share_the_partials(dev):
    """Graphs of two batches captured on one context and replayed in turn, eager calls of
    a third between them: all use the context's partials and counters."""
    ctx, ops = dev
    rng = np.random.default_rng(63)
    heads, kv_heads, hd = 4, 1, 128
    held, calls = [], []
    for rows, past, prefix in (([1, 1], [9000, 40], 0), ([70], [2000], 0), ([1, 3], [3000, 900], 500)):
        b = Batch(rng, rows, past, 32, prefix=prefix)
        q = rng.normal(0, 1, (b.T, heads * hd)).astype(np.float32)
        kc, vc = cache_of(rng, b, kv_heads, hd, "bf16")
        d = Held(ctx, b, kc, vc, "bf16", kv_heads, hd)
        dq, out = d.up(q), d.up(np.zeros_like(q))
        ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
        held.append((d, out, ref, attention_bound(ref, mag, top, hd, "f32")))
        calls.append(lambda d=d, dq=dq, out=out: ops.paged_attention(d.kv, d.batch, dq, heads * hd, out, heads * hd,
                                                                     "f32", heads))
    for c in calls:
        c()
    ctx.sync()
    first = [out.download(np.float32).copy() for _, out, _, _ in held]
    graphs = []
    for c in calls[:2]:
        ctx.graph_begin()
        c()
        graphs.append(ctx.graph_end())
    for rep in range(3):
        for _, out, _, _ in held:
            out.upload(np.zeros(out.nbytes // 4, np.float32))
        say(f"two graphs in turn {rep}")
        graphs[0].launch()
        graphs[1].launch()
        calls[2]()
        graphs[0].launch()
        ctx.sync()
        for (d, out, ref, bound), want in zip(held, first):
            got = out.download(np.float32)
            assert np.array_equal(got, want)
            check_close(got.reshape(-1, heads, hd).astype(np.float64), ref, bound, "f32")
    del graphs
    for d, _, _, _ in held:
        d.free()


def test_attention_scratch_grows_between_captures():
    """A first call inside a capture is refused, a graph from before the partials grew as
    well; sampling's first call inside one gives the same tokens."""
    rng = np.random.default_rng(64)
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    ops = DenseOps(ctx)
    heads, kv_heads, hd = 4, 2, 64
    b = Batch(rng, [1, 1], [300, 40], 16)
    q = rng.normal(0, 1, (2, heads * hd)).astype(np.float32)
    kc, vc = cache_of(rng, b, kv_heads, hd, "f32")
    d = Held(ctx, b, kc, vc, "f32", kv_heads, hd)
    dq, out = d.up(q), d.up(np.zeros_like(q))
    V = 9001
    x, u = rng.normal(0, 2, (2, 9004)).astype(np.float32), rng.random(2).astype(np.float32)
    dx, du, tok = d.up(x), d.up(u), d.up(np.zeros(2, np.int32))
    want = [sample_ref(x[r, :V], u[r])[0] for r in range(2)]

    def call():
        ops.paged_attention(d.kv, d.batch, dq, heads * hd, out, heads * hd, "f32", heads)
    say("first calls inside a capture")
    ctx.graph_begin()
    with pytest.raises(M1MoEError) as e:
        call()
    assert e.value.code == _lib.M1MOE_ERR_INVALID and "capture" in str(e.value)
    ops.sample(dx, 2, V, 9004, SampleParams.make(du), tok)
    g = ctx.graph_end()
    for _ in range(2):
        tok.upload(np.zeros(2, np.int32))
        g.launch()
        ctx.sync()
        assert tok.download(np.int32).tolist() == want
        ops.sample(dx, 2, V, 9004, SampleParams.make(du), tok)
        ctx.sync()
        assert tok.download(np.int32).tolist() == want
    call()
    ctx.graph_begin()
    call()
    g = ctx.graph_end()
    g.launch()
    ctx.sync()
    ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
    bound = attention_bound(ref, mag, top, hd, "f32")
    check_close(out.download(np.float32).reshape(2, heads, hd).astype(np.float64), ref, bound, "f32")
    b2 = Batch(rng, [40], [100], 16, prefix=64)
    q2 = rng.normal(0, 1, (40, heads * 256)).astype(np.float32)
    k2, v2 = cache_of(rng, b2, kv_heads, 256, "f32")
    d2 = Held(ctx, b2, k2, v2, "f32", kv_heads, 256)
    o2 = d2.up(np.zeros_like(q2))
    say("the partials grow")
    ops.paged_attention(d2.kv, d2.batch, d2.up(q2), heads * 256, o2, heads * 256, "f32", heads)
    ctx.sync()
    with pytest.raises(M1MoEError) as e:
        g.launch()
    assert "capture it again" in str(e.value)
    out.upload(np.zeros_like(q))
    call()
    ctx.sync()
    check_close(out.download(np.float32).reshape(2, heads, hd).astype(np.float64), ref, bound, "f32")
    ref, mag, top = attention_ref(b2, q2, k2, v2, heads, kv_heads, 256)
    check_close(o2.download(np.float32).reshape(40, heads, 256).astype(np.float64), ref,
                attention_bound(ref, mag, top, 256, "f32"), "f32")
    del g
    d.free()
    d2.free()
    ctx.close()


def test_two_contexts_in_turn(dev):
    """Calls of two contexts of one device, none waited for: each has its own partials."""
    a, ops = dev
    c = m.HIPContext(m.make_shape(64, 1, 1, 64))
    rng = np.random.default_rng(65)
    heads, hd = 4, 64
    held = []
    for ctx in (a, c):
        b = Batch(rng, [1, 20], [5000, 700], 16)
        q = rng.normal(0, 1, (b.T, heads * hd)).astype(np.float32)
        kc, vc = cache_of(rng, b, 1, hd, "f32")
        d = Held(ctx, b, kc, vc, "f32", 1, hd)
        ref, mag, top = attention_ref(b, q, kc, vc, heads, 1, hd)
        x = rng.normal(0, 2, (3, 20000)).astype(np.float32)
        u = rng.random(3).astype(np.float32)
        held.append((ctx, DenseOps(ctx), d, d.up(q), d.up(np.zeros_like(q)), ref,
                     attention_bound(ref, mag, top, hd, "f32"), d.up(x), d.up(u), d.up(np.zeros(3, np.int32)),
                     [sample_ref(x[r], u[r], top_p=0.9)[0] for r in range(3)], d.up(np.full(3, 0.9, np.float32))))
    say("two contexts in turn")
    for _ in range(3):
        for ctx, o, d, dq, out, _, _, dx, du, tok, _, dp in held:
            o.paged_attention(d.kv, d.batch, dq, heads * hd, out, heads * hd, "f32", heads)
            o.sample(dx, 3, 20000, 20000, SampleParams.make(du, top_p=dp), tok)
    for ctx, o, d, dq, out, ref, bound, _, _, tok, want, _ in held:
        ctx.sync()
        check_close(out.download(np.float32).reshape(-1, heads, hd).astype(np.float64), ref, bound, "f32")
        assert tok.download(np.int32).tolist() == want
        d.free()
    c.close()


def test_a_caller_stream(dev):
    """The operators on a stream of the caller's, captured and replayed there."""
    ctx, ops = dev
    gc.collect()
    ctx.sync()
    hip = ctypes.CDLL("libamdhip64.so")
    s = ctypes.c_void_p()
    assert hip.hipStreamCreate(ctypes.byref(s)) == 0
    try:
        if ctx.lib.m1moe_set_stream(ctx.handle, s) != _lib.M1MOE_OK:
            assert "share device" in _lib.last_error()
            pytest.skip("another context is alive on the device")
        rng = np.random.default_rng(66)
        heads, kv_heads, hd = 4, 2, 128
        b = Batch(rng, [1, 30], [2000, 10], 16)
        q = rng.normal(0, 1, (b.T, heads * hd)).astype(np.float32)
        kc, vc = cache_of(rng, b, kv_heads, hd, "bf16")
        d = Held(ctx, b, kc, vc, "bf16", kv_heads, hd)
        dq, out = d.up(q), d.up(np.zeros_like(q))
        ref, mag, top = attention_ref(b, q, kc, vc, heads, kv_heads, hd)
        bound = attention_bound(ref, mag, top, hd, "f32")

        def call():
            ops.paged_attention(d.kv, d.batch, dq, heads * hd, out, heads * hd, "f32", heads)
        say("a caller stream")
        call()
        ctx.graph_begin()
        call()
        g = ctx.graph_end()
        for _ in range(3):
            ctx.sync()
            check_close(out.download(np.float32).reshape(-1, heads, hd).astype(np.float64), ref, bound, "f32")
            out.upload(np.zeros_like(q))
            g.launch()
        ctx.sync()
        del g
        d.free()
    finally:
        ctx.lib.m1moe_set_stream(ctx.handle, None)
        assert hip.hipStreamDestroy(s) == 0


# ---- append ------------------------------------------------------------------------------

@pytest.mark.parametrize("x,cache", TYPES + [("bf16", "f32")])
@pytest.mark.parametrize("heads,kv_heads,hd,rotary,inter,norm,page", [
    (4, 4, 128, 128, False, True, 16), (8, 2, 128, 64, True, False, 8), (6, 2, 64, 48, False, True, 64),
    (3, 1, 256, 256, True, True, 32), (5, 5, 64, 16, False, False, 16), (2, 1, 256, 96, False, True, 8),
    (7, 7, 64, 0, False, True, 16), (64, 1, 128, 128, False, False, 16),
])
def test_append(dev, x, cache, heads, kv_heads, hd, rotary, inter, norm, page):
    ctx, ops = dev
    rng = np.random.default_rng(30)
    rows = [3, 0, 1, 20, 1, 0]
    b = Batch(rng, rows, [0, 5, 15, 30, 70000, 2], page, pad=3)
    qd, kvd = heads * hd, kv_heads * hd
    qkv = as_dtype(rng.normal(0, 2, (b.num_rows, qd + 2 * kvd)), x)
    qw, kw = (bf16(rng.normal(1, 0.2, hd)) if norm else None for _ in range(2))
    freq = (1e4 ** (-np.arange(max(rotary // 2, 1)) / max(rotary // 2, 1))).astype(np.float32)
    amp = 1.25
    before = as_dtype(rng.normal(0, 1, (b.num_pages, page, kv_heads, hd)), cache)
    d = Held(ctx, b, before, before, cache, kv_heads, hd)
    dx = d.up(qkv)
    size = 2 if x == "bf16" else 4
    out = d.up(as_dtype(np.full((b.num_rows, qd), 7.0), x))
    n = qd + 2 * kvd
    args = KVAppend.make(x, heads, dx, dx.addr + qd * size, dx.addr + (qd + kvd) * size, n, n, n, out, qd,
                         d.up(qw) if norm else None, d.up(kw) if norm else None, 1e-5, rotary, inter,
                         d.up(freq) if rotary else None, amp)
    say(f"append {x} {cache} {heads}/{kv_heads}x{hd} rotary {rotary} {inter} norm {norm}")
    ops.kv_append(d.kv, d.batch, args)
    ctx.sync()
    ct = np.uint16 if cache == "bf16" else np.float32
    k1, v1 = (t.download(ct).reshape(before.shape) for t in (d.k, d.v))
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(b.num_rows, heads, hd)
    d.free()
    # f32: the head's sum of squares (hd adds, half of it in the root), root, products,
    # the angle's rounding (an f32 in [-pi, pi]: 2^-23), cos, sin, amplitude, two products
    # and their sum: below (hd / 2 + 24) 2^-24 of the terms; then the output type's
    f32 = (hd / 2 + 24) * 2.0 ** -24
    one = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}
    ref, terms = append_ref(b, np.ascontiguousarray(qkv[:, :qd]), heads, hd, qw, 1e-5, rotary, inter, freq, amp)
    assert np.all(np.abs(got[:b.T] - ref) <= f32 * terms + one[x] * np.abs(ref) * 1.01 + 1e-30)
    assert np.all(got[b.T:] == 7.0)
    kref, kterms = append_ref(b, np.ascontiguousarray(qkv[:, qd:qd + kvd]), kv_heads, hd, kw, 1e-5, rotary,
                              inter, freq, amp)
    v = np.ascontiguousarray(qkv[:, qd + kvd:]).reshape(b.num_rows, kv_heads, hd)
    touched = np.zeros(before.shape[:2], bool)
    for r, (s, p) in enumerate(b.places()):
        pg, sl = b.cell(s, np.array([p]))
        touched[pg, sl] = True
        k = f64(k1[pg[0], sl[0]])
        assert np.all(np.abs(k - kref[r]) <= f32 * kterms[r] + one[cache] * np.abs(kref[r]) * 1.01 + 1e-30)
        assert np.array_equal(v1[pg[0], sl[0]], as_dtype(f64(v[r]), cache))
    assert np.array_equal(k1[~touched], before[~touched]) and np.array_equal(v1[~touched], before[~touched])


def test_append_in_place_and_kv_only(dev):
    """q rotated in place equals q rotated into another buffer; no q: only k and v."""
    ctx, ops = dev
    rng = np.random.default_rng(31)
    heads, kv_heads, hd = 4, 2, 128
    b = Batch(rng, [2, 5], [100, 3], 16)
    q, k, v = (rng.normal(0, 1, (b.T, h * hd)).astype(np.float32) for h in (heads, kv_heads, kv_heads))
    zero = np.zeros((b.num_pages, 16, kv_heads, hd), np.float32)
    freq = (1e6 ** (-np.arange(64) / 64)).astype(np.float32)
    got = []
    for mode in ("apart", "in place", "kv only"):
        d = Held(ctx, b, zero, zero, "f32", kv_heads, hd)
        dq, dk, dv, o, f = d.up(q), d.up(k), d.up(v), d.up(np.zeros_like(q)), d.up(freq)
        qd, kvd = heads * hd, kv_heads * hd
        qi, qo = {"apart": (dq, o), "in place": (dq, dq), "kv only": (None, None)}[mode]
        say(f"append {mode}")
        ops.kv_append(d.kv, d.batch, KVAppend.make("f32", heads, qi, dk, dv, qd, kvd, kvd, qo, qd, None, None, 0.0,
                                                   hd, False, f))
        ctx.sync()
        got.append(((qo or dq).download(np.float32), d.k.download(np.float32), d.v.download(np.float32)))
        d.free()
    assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[2][0], q.reshape(-1))
    for i in (1, 2):
        assert np.array_equal(got[0][1], got[i][1]) and np.array_equal(got[0][2], got[i][2])


def test_append_far_position(dev):
    """Positions near 2^24: the angle keeps its bits."""
    ctx, ops = dev
    rng = np.random.default_rng(32)
    b = Batch(rng, [1], [0], 4096)
    b.kv_len = np.array([(1 << 24) - 5], np.int32)
    b.stride = 4096
    b.table = np.zeros((1, 4096), np.int32)
    k = rng.normal(0, 1, (1, 64)).astype(np.float32)
    zero = np.zeros((b.num_pages, 4096, 1, 64), np.float32)
    freq = (1e4 ** (-np.arange(32) / 32)).astype(np.float32)
    d = Held(ctx, b, zero, zero, "f32", 1, 64)
    dk, o = d.up(k), d.up(np.zeros_like(k))
    ops.kv_append(d.kv, d.batch, KVAppend.make("f32", 1, dk, dk, dk, 64, 64, 64, o, 64, None, None, 0.0, 64, False,
                                               d.up(freq)))
    ctx.sync()
    got = o.download(np.float32).reshape(1, 1, 64)
    d.free()
    ref, terms = append_ref(b, k, 1, 64, None, 0.0, 64, False, freq, 1.0)
    assert np.all(np.abs(got - ref) <= 24 * 2.0 ** -24 * terms)


def test_append_bad_page_and_sequence(dev):
    ctx, ops = dev
    rng = np.random.default_rng(33)
    b = Batch(rng, [1, 2, 1], [40, 50, 30], 16)
    b.table[0, 2] = b.num_pages          # the page of position 40
    b.kv_len[1] = 1                      # fewer positions than rows
    x = rng.normal(0, 1, (b.T, 64)).astype(np.float32)
    zero = np.zeros((b.num_pages, 16, 1, 64), np.float32)
    d = Held(ctx, b, zero, zero, "f32", 1, 64)
    dx, o = d.up(x), d.up(np.full_like(x, 9.0))
    say("append bad page")
    ops.kv_append(d.kv, d.batch, KVAppend.make("f32", 1, dx, dx, dx, 64, 64, 64, o, 64))
    with pytest.raises(M1MoEError, match="paged batch"):
        ctx.sync()
    ctx.sync()
    k, got = d.k.download(np.float32).reshape(zero.shape), o.download(np.float32).reshape(b.T, 64)
    d.free()
    assert np.array_equal(got[0], x[0]) and np.all(got[1:3] == 9.0) and np.array_equal(got[3], x[3])
    pg, sl = b.cell(2, np.array([30]))
    assert np.array_equal(k[pg[0], sl[0], 0], x[3])
    k[pg, sl] = 0
    assert not k.any()


# ---- sampling ----------------------------------------------------------------------------

def draw(dev, x, settings, stride=None, probs=True):
    """tokens and probabilities of the rows of x under per-row dicts."""
    ctx, ops = dev
    rows, vocab = x.shape
    stride = stride or (vocab + 3) // 4 * 4
    buf = np.full((rows, stride), 99.0, np.float32)
    buf[:, :vocab] = x
    held = [ctx.to_device(buf)]

    def col(name, default, dtype):
        held.append(ctx.to_device(np.array([s.get(name, default) for s in settings], dtype)))
        return held[-1]
    params = SampleParams.make(col("u", 0.5, np.float32), col("T", 1.0, np.float32), col("top_k", 0, np.int32),
                               col("top_p", 1.0, np.float32), col("min_p", 0.0, np.float32))
    held += [ctx.to_device(np.full(rows, -7, np.int32)), ctx.to_device(np.full(rows, -7, np.float32))]
    ops.sample(held[0], rows, vocab, stride, params, held[-2], held[-1] if probs else None)
    ctx.sync()
    tok, pr = held[-2].download(np.int32), held[-1].download(np.float32)
    for h in held:
        h.free()
    return tok, pr


def check_draw(dev, x, settings, **k):
    tok, pr = draw(dev, x, settings, **k)
    for r, s in enumerate(settings):
        want, p = sample_ref(x[r], s.get("u", 0.5), s.get("T", 1.0), s.get("top_k", 0), s.get("top_p", 1.0),
                             s.get("min_p", 0.0))
        assert tok[r] == want, (r, s, tok[r], want)
        # the kept sum is of units of 2^-44: below 2^-26 of it even over 2^18 logits
        assert abs(pr[r] - p) <= 2.0 ** -23 * p, (r, s, pr[r], p)


def some_settings(rng, rows, vocab):
    out = []
    for _ in range(rows):
        s = dict(u=float(np.float32(rng.random())), T=float(rng.choice([0.0, 0.3, 0.7, 1.0, 1.7, 30.0])))
        if rng.random() < 0.5:
            s["top_k"] = int(rng.integers(1, min(vocab, 500) + 1))
        if rng.random() < 0.6:
            s["top_p"] = float(rng.random())
        if rng.random() < 0.4:
            s["min_p"] = float(rng.random() ** 3)
        out.append(s)
    return out


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 64, 255, 257, 1000, 4097, 16384, 16389, 32000, 50304, 53251, 65537,
                                   131071, 262144])
def test_sample(dev, vocab):
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 100000 else 8
    x = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    say(f"sample vocab {vocab}")
    check_draw(dev, x, some_settings(rng, rows, vocab))


@pytest.mark.parametrize("vocab", [7, 3000, 40000, 70000])
def test_sample_ties(dev, vocab):
    """Equal logits, at the cut and at the draw: few distinct values, all equal, two
    values, bf16 values."""
    rng = np.random.default_rng(vocab)
    x = [rng.integers(0, 5, (8, vocab)).astype(np.float32), np.zeros((8, vocab), np.float32),
         np.where(rng.random((8, vocab)) < 0.5, 1.0, -0.0).astype(np.float32),
         synth.bf16_to_f32(bf16(rng.normal(0, 2, (8, vocab))))]
    x = np.concatenate(x).astype(np.float32)
    say(f"sample ties {vocab}")
    check_draw(dev, x, some_settings(rng, 32, vocab))


def test_sample_odd_values(dev):
    """Masked logits (-inf, the lowest float), NaN, +inf, one candidate, none, subnormal
    and huge ranges, temperatures at the ends."""
    rng = np.random.default_rng(40)
    V = 5003
    x = rng.normal(0, 2, (16, V)).astype(np.float32)
    s = [dict(u=0.9, T=1.0) for _ in range(16)]
    x[0, 5:] = -np.inf
    x[1, rng.random(V) < 0.9] = np.finfo(np.float32).min
    x[2, ::3] = np.nan
    x[3, :] = -np.inf
    x[4, :] = np.nan
    x[5, :] = -np.inf
    x[5, 4321] = -3.0
    x[6, [7, 70, 700]] = np.inf
    s[6]["u"] = 0.5
    x[7] = rng.normal(0, 1e-42, V)
    x[8] = rng.normal(0, 1e38, V).clip(-3.4e38, 3.4e38)
    s[8]["T"] = 3e37
    x[9, 100] = 1e30
    s[10]["T"] = 1e-40
    s[11]["T"] = 3e38
    s[12]["T"] = np.nan
    s[13]["T"] = -1.0
    x[13, 17] = x[13, 3001] = 50.0
    x[14] = np.exp(rng.uniform(-80, 80, V)) * rng.choice([-1, 1], V)
    s[14]["T"] = 1e20
    x[15, :4990] = np.finfo(np.float32).min
    s[15].update(T=1e38, top_p=0.7)
    say("sample odd values")
    check_draw(dev, x, s)


def test_sample_dense_steps(dev):
    """One logit far above the others, which then share few steps of a histogram over
    all: more of them in a step than are ranked at once, with every setting's end there."""
    rng = np.random.default_rng(44)
    V = 30000
    x = rng.normal(0, 1, (12, V)).astype(np.float32)
    x[:, 777] = 1000.0
    s = [dict(u=u, T=300.0, **k) for u in (0.2, 0.95) for k in
         (dict(), dict(top_k=5), dict(top_k=300), dict(top_k=2000), dict(top_p=0.9), dict(top_k=900, top_p=0.97))]
    for i in (1, 3, 7):
        s[i]["min_p"] = float(np.exp(-1000 / 300.0) * 1.002)
    say("sample dense steps")
    check_draw(dev, x, s)


def kept_count(x, T, top_k=0, min_p=0.0):
    """How many logits of a row top-k and min-p leave (f64)."""
    x = -np.sort(-x.astype(np.float64), kind="stable")
    x = x[:top_k] if top_k else x
    return max(1, int(np.count_nonzero(np.exp((x - x[0]) / T) >= float(np.float32(min_p)))))


def test_sample_min_p_among_equal_logits(dev):
    """Two crowded values below the first logit, the border of min-p just above the one
    that top-k ends in: only the first logit stays.  And three candidates of which the border
    parts the last two."""
    x = np.concatenate([[10.0], np.full(200, 5.0), np.zeros(1000)]).astype(np.float32)
    s = [dict(u=u, top_k=k, min_p=float(np.exp(-5.0) * 1.0005)) for u in (0.0, 0.6, 0.7, 0.9, 1.0) for k in (0, 100)]
    assert all(kept_count(x, 1.0, r["top_k"], r["min_p"]) == 1 for r in s)
    say("sample min-p among equal logits")
    check_draw(dev, np.tile(x, (len(s), 1)), s)
    x = np.array([0.0, -2.005, -2.01, -10.0, -40.0], np.float32)
    s = [dict(u=u, top_k=k, min_p=float(np.exp(-2.0075))) for u in (0.5, 0.999, 1.0) for k in (3, 4)]
    assert all(kept_count(x, 1.0, r["top_k"], r["min_p"]) == 2 for r in s)
    check_draw(dev, np.tile(x, (len(s), 1)), s)


@pytest.mark.parametrize("vocab,rows", [(700, 40), (9001, 30), (50304, 1), (50304, 20), (9001, 300)])
@pytest.mark.parametrize("crowded", [False, True])
def test_sample_min_p_beside_top_k(dev, vocab, rows, crowded):
    """The border of min-p between two logits from well above the k-th to below it: in the
    same step of 2047 equal ones as the k-th, the steps beside it and others, with the order's
    beginning kept aside (top-k of at most about 1000) and not.  Crowded: the best logit is far
    above the others, which then share few steps.  One workgroup per row and several."""
    rng = np.random.default_rng(vocab + rows + crowded)
    T = 6.0
    x = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    if crowded:
        x[np.arange(rows), rng.integers(0, vocab, rows)] = 40.0
    s, same, cut = [], 0, 0
    for r in range(rows):
        y = -np.sort(-x[r].astype(np.float64))
        w = np.exp((y - y[0]) / T)
        bounds = (y[0] - np.maximum(y[-1], y[0] - 45.5 * np.log(2) * T)) / 2047
        step = np.floor((y[0] - y) / bounds)
        top_k = int(np.exp(rng.uniform(np.log(2), np.log(min(vocab - 2, 3000)))))
        # logits j - 1 and j are parted (their weights differ by more than an f32's half step
        # and what the places of an f64 exponent are off)
        away = int(rng.choice([-200, -3, -2, -1, 0, 0, 1, 2]))
        j = min(max(1, top_k + away), vocab - 1)
        while j > 1 and not w[j - 1] > w[j] * (1 + 2.0 ** -20):
            j -= 1
        min_p = float(np.float32(math.sqrt(w[j - 1] * w[j])))
        assert w[j - 1] > min_p > w[j]
        s.append(dict(u=float(np.float32(rng.choice([rng.random(), 0.999, 1.0]))), T=T, top_k=top_k, min_p=min_p))
        if rng.random() < 0.3:
            s[-1]["top_p"] = float(rng.uniform(0.8, 1.0))
        fewer = kept_count(x[r], T, top_k, min_p) < kept_count(x[r], T, top_k)
        assert fewer == (j < top_k)
        cut += fewer
        same += fewer and step[j] == step[top_k - 1]
    # (rows that min-p cuts, and those where it does so in the k-th logit's own step)
    assert rows == 1 or (cut >= rows // 4 and (same >= 2 or not crowded))
    say(f"sample min-p beside top-k {vocab} x {rows} {crowded}")
    check_draw(dev, x, s)


def test_sample_min_p_in_dense_steps(dev):
    """Settings as in test_sample_dense_steps with a border that cuts: alone, with top-p, and
    with top-k above, inside and below the k-th logit's step."""
    rng = np.random.default_rng(45)
    V, T = 30000, 300.0
    x = rng.normal(0, 1, (12, V)).astype(np.float32)
    x[:, 777] = 1000.0
    ks = [0, 0, 0, 5, 5, 300, 300, 900, 900, 2000, 2000, 40]
    at = [10, 700, 9000, 3, 9, 290, 400, 20, 880, 1500, 1990, 39]     # logits that the border leaves
    s = []
    for r in range(12):
        y = -np.sort(-x[r].astype(np.float64))
        w = np.exp((y - y[0]) / T)
        j = at[r]
        while not w[j - 1] > w[j] * (1 + 2.0 ** -20):
            j -= 1
        s.append(dict(u=(0.3, 0.95, 1.0)[r % 3], T=T, top_k=ks[r], min_p=float(np.float32(math.sqrt(w[j - 1] * w[j])))))
        assert kept_count(x[r], T, ks[r], s[-1]["min_p"]) == min(j, ks[r] or V)
    s[1]["top_p"], s[2]["top_p"] = 0.1, 0.01
    say("sample min-p in dense steps")
    check_draw(dev, x, s)


def test_sample_settings_at_their_ends(dev):
    rng = np.random.default_rng(41)
    V = 9000
    base = rng.normal(0, 2, V).astype(np.float32)
    s = [dict(u=0.0), dict(u=1.0 - 2.0 ** -24), dict(u=1.0), dict(u=2.0), dict(u=-1.0), dict(u=np.nan),
         dict(u=0.7, top_k=1), dict(u=0.7, top_k=V), dict(u=0.7, top_k=V + 5), dict(u=0.7, top_k=-3),
         dict(u=0.7, top_p=0.0), dict(u=0.7, top_p=-1.0), dict(u=0.7, top_p=1.5), dict(u=0.7, top_p=1e-30),
         dict(u=0.999, min_p=1.0), dict(u=0.999, min_p=2.0), dict(u=0.999, min_p=1e-30), dict(u=0.3, min_p=-1.0),
         dict(u=0.999, top_k=50, top_p=0.5, min_p=0.2), dict(u=1.0, top_k=3, top_p=0.9999)]
    say("sample settings at their ends")
    check_draw(dev, np.tile(base, (len(s), 1)), s, stride=9004)
    nan = np.float32(np.nan)
    check_draw(dev, np.tile(base, (2, 1)), [dict(u=0.4, top_p=nan), dict(u=0.4, min_p=nan)])


def test_sample_defaults_and_the_host_sampler(dev):
    """No settings but u; and m1moe_amd.sampling.sample_token's tokens (its f32 sums in
    order move a border by at most vocab * 2^-24: draws are kept that far from one)."""
    from m1moe_amd.sampling import sample_token
    ctx, ops = dev
    rng = np.random.default_rng(42)
    rows, V = 40, 2000
    x = rng.normal(0, 2.5, (rows, V)).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    dx, du, tok = ctx.to_device(x), ctx.to_device(u), ctx.alloc(4 * rows)
    ops.sample(dx, rows, V, V, SampleParams.make(du), tok)
    ctx.sync()
    assert [sample_ref(x[r], u[r])[0] for r in range(rows)] == tok.download(np.int32).tolist()
    for h in (dx, du, tok):
        h.free()
    got, _ = draw(dev, x, [dict(u=float(v), T=0.7, top_p=0.9) for v in u])
    same = 0
    for r in range(rows):
        near = {sample_ref(x[r], u[r] + e, 0.7, 0, 0.9)[0] for e in (-2e-4, 0.0, 2e-4)}
        if len(near) == 1:
            assert sample_token(x[r], 0.7, 0.9, u=float(u[r])) == got[r]
            same += 1
    assert same > rows // 2


def test_sample_in_a_graph(dev):
    """New random numbers and settings for a captured call."""
    ctx, ops = dev
    rng = np.random.default_rng(43)
    rows, V = 3, 6000
    x = rng.normal(0, 2.5, (rows, V)).astype(np.float32)
    dx, du, dk, tok = ctx.to_device(x), ctx.alloc(16), ctx.alloc(16), ctx.alloc(16)
    params = SampleParams.make(du, top_k=dk)
    ctx.graph_begin()
    ops.sample(dx, rows, V, V, params, tok)
    g = ctx.graph_end()
    for rep in range(3):
        u, k = rng.random(rows).astype(np.float32), rng.integers(1, 100, rows).astype(np.int32)
        du.upload(u)
        dk.upload(k)
        say(f"sample graph replay {rep}")
        g.launch()
        ctx.sync()
        assert tok.download(np.int32, rows).tolist() == [sample_ref(x[r], u[r], top_k=int(k[r]))[0]
                                                         for r in range(rows)]
    for h in (dx, du, dk, tok):
        h.free()


# ---- together ----------------------------------------------------------------------------

def test_a_batch_decodes_step_by_step(dev):
    """As a server would use them: prompts of three conversations behind a shared prefix
    appended and attended in one call, then steps of one token each, whose logits are
    made from the attention's output and sampled; every output against f64 over a cache
    kept in f64 from the stored values."""
    ctx, ops = dev
    rng = np.random.default_rng(50)
    heads, kv_heads, hd, page, V, prefix, steps = 8, 2, 64, 16, 500, 37, 4
    qd, kvd = heads * hd, kv_heads * hd
    prompts = [5, 1, 30]
    ends = [prefix + p + steps for p in prompts]
    b = Batch(rng, prompts, [prefix + steps] * 3, page, prefix=prefix)   # (tables for the final lengths)
    b.kv_len = np.array([prefix + p for p in prompts], np.int32)
    freq = (1e4 ** (-np.arange(hd // 2) / (hd // 2))).astype(np.float32)
    qw, kw = bf16(rng.normal(1, 0.1, hd)), bf16(rng.normal(1, 0.1, hd))
    head = rng.normal(0, 0.3, (V, qd)).astype(np.float32)
    embed = rng.normal(0, 1, (V, qd + 2 * kvd)).astype(np.float32)
    shape = (b.num_pages, page, kv_heads, hd)
    kc, vc = (bf16(rng.normal(0, 1, shape)) for _ in range(2))
    d = Held(ctx, b, kc, vc, "bf16", kv_heads, hd)
    dqw, dkw, df = d.up(qw), d.up(kw), d.up(freq)
    tokens = np.concatenate([rng.integers(0, V, p) for p in prompts])
    u = rng.random((steps + 1, 3)).astype(np.float32)
    for step in range(steps + 1):
        rows = prompts if step == 0 else [1, 1, 1]
        b.rows, b.row_start = rows, np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        b.T = b.num_rows = int(b.row_start[-1])
        if step:
            b.kv_len = b.kv_len + 1
        d.start.upload(b.row_start)
        d.len.upload(b.kv_len)
        batch = PagedBatch.make(3, b.T, d.start, d.len, d.table, b.stride, prefix, d.pre)
        x = embed[tokens]
        dx, dq, do = d.up(x), d.up(np.zeros((b.T, qd), np.float32)), d.up(np.zeros((b.T, qd), np.float32))
        n = qd + 2 * kvd
        ops.kv_append(d.kv, batch, KVAppend.make("f32", heads, dx, dx.addr + 4 * qd, dx.addr + 4 * (qd + kvd), n, n, n,
                                                 dq, qd, dqw, dkw, 1e-5, hd, False, df))
        ops.paged_attention(d.kv, batch, dq, qd, do, qd, "f32", heads)
        ctx.sync()
        q1 = dq.download(np.float32).reshape(b.T, qd)
        k1, v1 = (t.download(np.uint16).reshape(shape) for t in (d.k, d.v))
        kref, _ = append_ref(b, np.ascontiguousarray(x[:, qd:qd + kvd]), kv_heads, hd, kw, 1e-5, hd, False, freq, 1.0)
        for r, (s, p) in enumerate(b.places()):
            pg, sl = b.cell(s, np.array([p]))
            assert np.allclose(f64(k1[pg[0], sl[0]]), kref[r], rtol=2.0 ** -8 * 1.01, atol=1e-5)
        ref, mag, top = attention_ref(b, q1, k1, v1, heads, kv_heads, hd)
        got = do.download(np.float32).reshape(b.T, heads, hd)
        check_close(got.astype(np.float64), ref, attention_bound(ref, mag, top, hd, "f32"), "f32")
        last = b.row_start[1:] - 1
        logits = got.reshape(b.T, qd)[last] @ head.T
        dl, du, dt = d.up(logits.astype(np.float32)), d.up(u[step]), d.up(np.zeros(3, np.int32))
        settings = [dict(T=0.8, top_k=40, top_p=0.95, min_p=0.02)] * 3
        cols = [d.up(np.array([s[k] for s in settings], t)) for k, t in
                (("T", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32))]
        ops.sample(dl, 3, V, V, SampleParams.make(du, *cols), dt)
        ctx.sync()
        tokens = dt.download(np.int32)
        want = [sample_ref(logits[i].astype(np.float32), u[step, i], 0.8, 40, 0.95, 0.02)[0] for i in range(3)]
        assert tokens.tolist() == want
    assert b.kv_len.tolist() == ends
    d.free()


# ---- the decoder's sampler -----------------------------------------------------------------

def test_decoder_draws_on_the_gpu():
    """generate_sampled and forward with top_k / min_p give the tokens that the f64
    sampler draws from the same steps' logits."""
    from m1moe_amd.decoder import Decoder
    wl = synth.DECODERS["tiny_dec"]
    L, seed = wl.num_layers, 78
    shape = wl.moe.shape(L)
    with m.HIPContext(shape) as ctx:
        for layer in range(L):
            ctx.upload_layer_experts(layer, synth.layer_image(shape, seed, layer))
            ctx.upload_router(layer, synth.router(shape, seed, layer))
        dec = Decoder(ctx, wl.dec_shape(64))
        dec.upload_all(lambda w, layer: synth.dense_weight(wl, seed, w, layer))
        rng = np.random.default_rng(51)
        prompt, n = rng.integers(0, wl.vocab, 11), 12
        u = rng.random(n + 1).astype(np.float32)
        for k in (dict(temperature=0.9, top_p=0.95, top_k=20, min_p=0.01), dict(temperature=1.3), dict(temperature=0.0)):
            say(f"decoder draws {k}")
            got = dec.generate_sampled(prompt, n, u=u, **k)
            dec.reset()
            _, logits = dec.prefill(prompt, return_logits=True)
            for i in range(n + 1):
                want, _ = sample_ref(logits, u[i], k["temperature"], k.get("top_k", 0), k.get("top_p", 1.0),
                                     k.get("min_p", 0.0))
                assert got[i] == want, (k, i)
                if i < n:
                    _, logits = dec.forward(int(got[i]), return_logits=True)
        dec.reset()
        r1, r2 = np.random.default_rng(5), np.random.default_rng(5)
        tok = 3
        for _ in range(4):
            nxt, logits = dec.forward(tok, return_logits=True, temperature=0.8, top_p=0.9, rng=r1, top_k=30, min_p=0.02)
            want, _ = sample_ref(logits, r2.random(1, dtype=np.float32)[0], 0.8, 30, 0.9, 0.02)
            assert nxt == want
            tok = nxt
        with pytest.raises(ValueError):
            dec.generate_sampled(prompt, 3, 1.0, u=u)
        dec.close()
