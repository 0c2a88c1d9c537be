"""GPU: captures behind a call of the largest size, which makes the workspace that smaller ones use."""
import numpy as np
import pytest

import m1moe_amd as m
from m1moe_amd.decoder import DenseOps

from cases import say
from serving_cases import Batch
from test_gpu_drafts import Product, check_product
from test_gpu_drafts_edges import Attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tree", [False, True])
def test_attention_of_fewer_rows_after_more(tree):
    """The largest batch makes the workspace: a smaller one is captured, and graphs of the larger one
    stay good."""
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    dev = ctx, DenseOps(ctx)
    rng = np.random.default_rng(5)
    large, small, step = (Attention(dev, Batch(rng, rows, [2048 + 9] * len(rows), 16, prefix=2048), ("f32", "f32"), 8, 8, 64,
                                    len(rows), tree) for rows in ([97, 96], [96, 96], [1, 1]))
    say(f"fewer rows after more, tree {tree}")
    large()
    want = [large.result()]
    graphs = []
    for c in (large, small, step):
        ctx.graph_begin()
        c()
        graphs.append(ctx.graph_end())
    for c in (small, step):
        c()
        want.append(c.result())
    for _ in range(2):
        for g, c, w in zip(graphs, (large, small, step), want):
            g.launch()
            assert np.array_equal(c.result(), w)
    del graphs
    for c in (large, small, step):
        c.d.free()
    ctx.close()


def test_q4_of_fewer_tokens_after_more():
    ctx = m.HIPContext(m.make_shape(64, 1, 1, 64))
    dev = ctx, DenseOps(ctx)
    large, small, few = (Product(dev, t, n, 1024) for t, n in ((1024, 2048), (480, 2048), (9, 96)))
    say("fewer tokens after more")
    large()
    want = [large.result()]
    graphs = []
    for p in (large, small, few):
        ctx.graph_begin()
        p()
        graphs.append(ctx.graph_end())
    for p in (small, few):
        p()
        want.append(p.result())
    for p, w in zip((large, small, few), want):
        check_product(w, p.x, p.w, p.s, p.b, p.group, "f32")
    for _ in range(2):
        for g, p, w in zip(graphs, (large, small, few), want):
            g.launch()
            assert np.array_equal(p.result(), w)
    del graphs
    for p in (large, small, few):
        p.free()
    ctx.close()
