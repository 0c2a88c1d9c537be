"""GPU: attention of trees of drafted tokens at its edges: rows without a finite score behind a shared
prefix, other head counts and sizes behind one.  References and bounds as in test_gpu_drafts.py."""
import numpy as np
import pytest

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
