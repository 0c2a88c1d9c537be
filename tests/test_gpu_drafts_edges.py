"""GPU: attention of trees of drafted tokens at its edges: rows without a finite score behind a shared
prefix, other head counts and sizes behind one, repeated calls.  References and bounds as in
test_gpu_drafts.py."""
import numpy as np
import pytest

import m1moe_amd as m
from m1moe_amd.decoder import DenseOps

from cases import say
from draft_cases import tree_attention_ref
from serving_cases import Batch, as_dtype, attention_bound, f64
from test_gpu_drafts import TYPES, attend, check_close, dev, trees  # noqa: F401
from test_gpu_serving import Held, cache_of

pytestmark = pytest.mark.gpu


# ---- attention behind a prefix ----------------------------------------------------------------

@pytest.mark.parametrize("prefix", [0, 40, 700])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (4, 2, 64), (6, 2, 256), (16, 2, 128)])
def test_rows_whose_scores_are_all_minus_infinity(dev, types, heads, kv_heads, hd, prefix):  # noqa: F811
    """Keys of -inf under queries of positive dims: zeros, whether the positions are a prefix or not;
    the other kv head is what it was."""
    ctx, ops = dev
    rng = np.random.default_rng(prefix + hd)
    x, cache = types
    b = Batch(rng, [1, 20, 0, 40, 3], [prefix + p for p in (700, 3, 5, 70, 0)], 16, prefix=prefix, pad=2)
    _, mask, _ = trees(rng, b)
    q = rng.normal(0, 1, (b.num_rows, heads, hd))
    share = heads // kv_heads
    q[:, :share] = np.abs(q[:, :share]) + 0.01
    q = as_dtype(q.reshape(b.num_rows, heads * hd), x)
    kc, vc = cache_of(rng, b, kv_heads, hd, cache, np.nan)
    kc[:, :, 0] = as_dtype(np.full(hd, -np.inf), cache)
    d = Held(ctx, b, kc, vc, cache, kv_heads, hd)
    out = d.up(as_dtype(np.full((b.num_rows, heads * hd), 7.0), x))
    say(f"scores of -inf {types} {heads}/{kv_heads}x{hd} prefix {prefix}")
    ops.tree_attention(d.kv, d.batch, d.up(mask), mask.shape[1], d.up(q), heads * hd, out, heads * hd, x, heads)
    ctx.sync()
    got = f64(out.download(np.uint16 if x == "bf16" else np.float32)).reshape(-1, heads, hd)
    d.free()
    with np.errstate(all="ignore"):
        ref, mag, top = tree_attention_ref(b, mask, q, kc, vc, heads, kv_heads, hd)
    bound = attention_bound(ref, mag, top, hd, x)
    assert np.all(got[:b.T, :share] == 0)
    check_close(got[:b.T, share:], ref[:, share:], bound[:, share:], x)
    assert np.all(got[b.T:] == 7.0)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(8, 2, 64, 8), (5, 1, 256, 32), (40, 1, 128, 16), (3, 3, 64, 64)])
def test_attention_prefix_of_other_heads(dev, types, heads, kv_heads, hd, page):  # noqa: F811
    rng = np.random.default_rng(heads)
    b = Batch(rng, [1, 70, 3, 0, 64, 140, 1], [300 + p for p in (0, 0, 64, 2, 31, 10, 600)], page, prefix=300, pad=2)
    _, mask, _ = trees(rng, b, 0.7)
    say(f"tree attention prefix 300 {types} {heads}/{kv_heads}x{hd}")
    got, rest, ref, bound = attend(dev, b, mask, heads, kv_heads, hd, types, heads + 1)
    check_close(got, ref, bound, types[0])
    assert np.all(rest == 7.0)


class Attention:
    """A call, tree or plain, whose operands stay on the device."""

    def __init__(self, dev, b, types, heads, kv_heads, hd, seed, tree=True):  # noqa: F811
        self.ctx, self.ops = dev
        rng = np.random.default_rng(seed)
        self.x, cache = types
        self.b, self.heads, self.n, self.tree = b, heads, heads * hd, tree
        _, mask, _ = trees(rng, b, 0.6) if tree else (0, np.zeros((b.num_rows, 1), np.uint64), 0)
        kc, vc = cache_of(rng, b, kv_heads, hd, cache)
        self.d = d = Held(self.ctx, b, kc, vc, cache, kv_heads, hd)
        self.words, self.mask = mask.shape[1], d.up(mask)
        self.q = d.up(as_dtype(rng.normal(0, 1, (b.num_rows, self.n)), self.x))
        self.zero = as_dtype(np.zeros((b.num_rows, self.n)), self.x)
        self.out = d.up(self.zero)

    def __call__(self):
        d, o = self.d, self.ops
        if self.tree:
            o.tree_attention(d.kv, d.batch, self.mask, self.words, self.q, self.n, self.out, self.n, self.x, self.heads)
        else:
            o.paged_attention(d.kv, d.batch, self.q, self.n, self.out, self.n, self.x, self.heads)

    def result(self):
        """The bits of out, and zeros in its place."""
        self.ctx.sync()
        y = self.out.download(self.zero.dtype)
        self.out.upload(self.zero)
        return y


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("heads,kv_heads,hd", [(16, 16, 128), (32, 8, 128), (8, 2, 64), (4, 2, 256)])
def test_calls_repeat_bit_for_bit(dev, types, heads, kv_heads, hd):  # noqa: F811
    """Cut tiles, shared prefixes, other batches in between and the first call of a context: one
    order of every sum, whoever ends last."""
    rng = np.random.default_rng(hd + heads)
    rows = [1, 100, 64, 17, 3, 40, 90, 16, 33]
    kinds = [Batch(rng, rows, [p + 900 for p in (20, 600, 300, 900, 5, 60, 420, 2000, 0)], 64, prefix=900, pad=3),
             Batch(rng, rows, [20, 600, 300, 2900, 5, 60, 420, 2000, 0], 64, pad=3)]
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    fresh = ctx, DenseOps(ctx)
    firsts = []
    for where in (fresh, dev):
        a, c = (Attention(where, b, types, heads, kv_heads, hd, i) for i, b in enumerate(kinds))
        say(f"repeated calls {types} {heads}/{kv_heads}x{hd}")
        a()
        want = [a.result()]
        c()
        want.append(c.result())
        for i in range(5):
            a(), c(), a()
            assert np.array_equal(a.result(), want[0]) and np.array_equal(c.result(), want[1]), i
        firsts.append(want)
        a.d.free()
        c.d.free()
    ctx.close()
    assert all(np.array_equal(x, y) for x, y in zip(*firsts))
