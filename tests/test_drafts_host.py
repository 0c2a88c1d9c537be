"""Refusals of the drafted tokens' operators and of the products with 4-bit weights: every
argument check comes before the context is looked at, so they run without a GPU."""
import ctypes

import pytest

from m1moe_amd import KVAppend, PagedBatch, PagedKV, Q4Weights, _lib

A = 0x10000    # an aligned address that is never read


def kv(**k):
    d = dict(k=A, v=A, dtype="bf16", num_pages=10, page_size=16, num_kv_heads=4, head_dim=128)
    d.update(k)
    return PagedKV.make(**d)


def batch(**k):
    d = dict(num_seqs=3, num_rows=7, row_start=A, kv_len=A, pages=A, table_stride=4)
    d.update(k)
    return PagedBatch.make(**d)


def refused(rc, *words):
    assert rc == _lib.M1MOE_ERR_INVALID
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


def plan(**k):
    d = dict(seqs=3, rows=7, start=A, parents=A, words=1, mask=A, depth=A)
    d.update(k)
    return _lib.load().m1moe_tree_plan(None, d["seqs"], d["rows"], d["start"], d["parents"], d["words"], d["mask"],
                                       d["depth"])


@pytest.mark.parametrize("change,word", [
    (dict(seqs=0), "num_seqs"), (dict(seqs=1025), "num_seqs"), (dict(rows=0), "num_rows"),
    (dict(rows=(1 << 20) + 1), "num_rows"), (dict(start=None), "d_row_start"), (dict(parents=A + 2), "d_parents"),
    (dict(words=0), "mask_words"), (dict(words=5), "mask_words"), (dict(mask=None), "d_mask"),
    (dict(mask=A + 4), "d_mask"), (dict(depth=None), "d_depth"), (dict(), "context"),
])
def test_plan_refusals(change, word):
    refused(plan(**change), word)


def append(**k):
    d = dict(dtype="f32", num_heads=8, q=A, k=A, v=A, q_stride=1024, k_stride=512, v_stride=512, q_out=A + 16,
             q_out_stride=1024, rotary_dim=128, inv_freq=A)
    d.update(k)
    return KVAppend.make(**d)


def test_append_refusals():
    lib = _lib.load()
    refused(lib.m1moe_tree_append(None, kv(), batch(), append(), None), "d_depth")
    refused(lib.m1moe_tree_append(None, kv(), batch(), append(), A + 1), "d_depth")
    refused(lib.m1moe_tree_append(None, kv(page_size=3), batch(), append(), A), "page_size")
    refused(lib.m1moe_tree_append(None, kv(), batch(num_rows=0), append(), A), "num_rows")
    refused(lib.m1moe_tree_append(None, kv(), batch(), append(num_heads=6), A), "num_heads")
    refused(lib.m1moe_tree_append(None, kv(), batch(), None, A), "args")
    refused(lib.m1moe_tree_append(None, kv(), batch(), append(), A), "context")


@pytest.mark.parametrize("cache,mask,words,q,out,dtype,heads,word", [
    ("bf16", None, 1, A, A + 16, 0, 8, "d_mask"), ("bf16", A + 4, 1, A, A + 16, 0, 8, "d_mask"),
    ("bf16", A, 0, A, A + 16, 0, 8, "mask_words"), ("bf16", A, 5, A, A + 16, 0, 8, "mask_words"),
    ("bf16", A, 1, None, A + 16, 0, 8, "d_q"), ("bf16", A, 1, A, None, 0, 8, "d_out"),
    ("f32", A, 1, A, A + 16, 1, 8, "bf16 cache"), ("bf16", A, 1, A, A + 16, 0, 7, "num_heads"),
    ("bf16", A, 1, A, A, 0, 8, "overlap"), ("bf16", A, 4, A, A + 16, 0, 8, "context"),
])
def test_attention_refusals(cache, mask, words, q, out, dtype, heads, word):
    refused(_lib.load().m1moe_tree_attention(None, kv(dtype=cache), batch(), mask, words, q, 1024, out, 1024, dtype,
                                             heads), word)


def accept(caches, b, *ptrs):
    kvs = PagedKV.array(caches) if caches else None
    return _lib.load().m1moe_tree_accept(None, kvs, len(caches), b, *ptrs)


@pytest.mark.parametrize("i,word", enumerate(
    ["d_parents", "d_drafts", "d_drawn", "d_path", "d_accepted", "d_next", "d_past"]))
def test_accept_pointer_refusals(i, word):
    p = [A] * 7
    p[i] = None
    refused(accept([kv()], batch(), *p), word)
    p[i] = A + 3
    refused(accept([kv()], batch(), *p), word)


def test_accept_refusals():
    p = [A] * 7
    refused(accept([], batch(), *p), "num_caches")
    refused(accept([kv()] * 65, batch(), *p), "num_caches")
    refused(_lib.load().m1moe_tree_accept(None, None, 2, batch(), *p), "kvs")
    refused(accept([kv(), kv(k=None)], batch(), *p), "d_k")
    for change in (dict(dtype="f32"), dict(num_pages=11), dict(page_size=32), dict(num_kv_heads=2), dict(head_dim=64)):
        refused(accept([kv(), kv(**change)], batch(), *p), "cache 1")
    refused(accept([kv()], batch(kv_len=None), *p), "d_kv_len")
    refused(accept([kv()], batch(), *p), "context")


def q4(**k):
    d = dict(w=A, scales=A, biases=A, rows=40, cols=128, group=64, x=A, x_dtype=0, x_stride=128, tokens=2,
             residual=None, y=A, y_dtype=0, y_stride=40)
    d.update(k)
    w = Q4Weights.make(d["w"], d["scales"], d["biases"], d["rows"], d["cols"], d["group"])
    return _lib.load().m1moe_matmul_q4(None, w, d["x"], d["x_dtype"], d["x_stride"], d["tokens"], d["residual"],
                                       d["y"], d["y_dtype"], d["y_stride"])


@pytest.mark.parametrize("change,word", [
    (dict(w=None), "d_w"), (dict(w=A + 8), "d_w"), (dict(scales=None), "d_scales"), (dict(biases=A + 2), "d_biases"),
    (dict(rows=0), "rows"), (dict(rows=(1 << 20) + 1, y_stride=1 << 21), "rows"), (dict(cols=0), "cols"),
    (dict(cols=96), "cols"), (dict(cols=65536 + 64, x_stride=1 << 17), "cols"), (dict(group=16), "group_size"),
    (dict(group=256), "group_size"), (dict(tokens=0), "tokens"), (dict(tokens=65537), "tokens"),
    (dict(x=None), "d_x"), (dict(x=A + 4), "d_x"), (dict(x_dtype=2), "dtype"), (dict(x_stride=124), "d_x"),
    (dict(x_stride=130), "d_x"), (dict(x_dtype=1, x_stride=132), "d_x"), (dict(y_dtype=2), "y_dtype"),
    (dict(y_dtype=1), "f32 rows"), (dict(y=None), "d_y"), (dict(y_stride=36), "d_y"), (dict(y_stride=42), "d_y"),
    (dict(x_dtype=1, y_dtype=1, y_stride=44), "d_y"), (dict(residual=A + 4), "d_residual"), (dict(), "context"),
])
def test_q4_refusals(change, word):
    refused(q4(**change), word)


def test_q4_needs_weights():
    refused(_lib.load().m1moe_matmul_q4(None, None, A, 0, 128, 1, None, A, 0, 128), "weights")


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(Q4Weights) == 40 and Q4Weights.group_size.offset == 32
    assert ctypes.sizeof(PagedKV.array([kv()] * 3)) == 120
