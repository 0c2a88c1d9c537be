"""Refusals of the paged KV cache, its attention and the sampler: every argument
check comes before the context is looked at, so they run without a GPU."""
import ctypes

import pytest

from m1moe_amd import KVAppend, PagedBatch, PagedKV, SampleParams, _lib

A = 0x10000    # an aligned address that is never read


def kv(**k):
    d = dict(k=A, v=A, dtype="bf16", num_pages=10, page_size=16, num_kv_heads=4, head_dim=128)
    d.update(k)
    if isinstance(d["dtype"], int) and d["dtype"] > 1:
        c = PagedKV.make(**{**d, "dtype": "f32"})
        c.dtype = d["dtype"]
        return c
    return PagedKV.make(**d)


def batch(**k):
    d = dict(num_seqs=3, num_rows=7, row_start=A, kv_len=A, pages=A, table_stride=4)
    d.update(k)
    return PagedBatch.make(**d)


def refused(rc, *words):
    assert rc == _lib.M1MOE_ERR_INVALID
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("change,word", [
    (dict(k=0), "d_k"), (dict(v=A + 4), "d_v"), (dict(dtype=2), "dtype"), (dict(num_pages=0), "num_pages"),
    (dict(page_size=4), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=8192), "page_size"),
    (dict(head_dim=96), "head_dim"), (dict(num_kv_heads=0), "num_kv_heads"),
    (dict(num_kv_heads=513), "num_kv_heads"),
])
def test_cache_refusals(change, word):
    refused(_lib.load().m1moe_check_paged(kv(**change), batch()), word)


@pytest.mark.parametrize("change,word", [
    (dict(num_seqs=0), "num_seqs"), (dict(num_seqs=1025), "num_seqs"), (dict(num_rows=0), "num_rows"),
    (dict(num_rows=(1 << 20) + 1), "num_rows"), (dict(table_stride=0), "table_stride"),
    (dict(table_stride=(1 << 20) + 1), "table_stride"), (dict(prefix_len=-1), "prefix_len"),
    (dict(prefix_len=65, prefix_pages=A), "prefix_len"), (dict(prefix_len=8), "d_prefix_pages"),
    (dict(row_start=None), "d_row_start"), (dict(kv_len=A + 2), "d_kv_len"), (dict(pages=None), "d_pages"),
])
def test_batch_refusals(change, word):
    refused(_lib.load().m1moe_check_paged(kv(), batch(**change)), word)


def test_good_descriptions_pass():
    lib = _lib.load()
    assert lib.m1moe_check_paged(kv(), batch()) == 0
    assert lib.m1moe_check_paged(kv(page_size=4096, head_dim=64), batch(prefix_len=64, prefix_pages=A)) == 0
    refused(lib.m1moe_check_paged(None, batch()), "kv")
    refused(lib.m1moe_check_paged(kv(), None), "batch")


def append(**k):
    d = dict(dtype="f32", num_heads=8, q=A, k=A, v=A, q_stride=1024, k_stride=512, v_stride=512, q_out=A + 16,
             q_out_stride=1024, rotary_dim=128, inv_freq=A)
    d.update(k)
    return KVAppend.make(**d)


@pytest.mark.parametrize("change,word", [
    (dict(num_heads=6), "num_heads"), (dict(num_heads=0), "num_heads"), (dict(num_heads=260), "num_heads"),
    (dict(q=None), "d_q"), (dict(q_out=None), "d_q"), (dict(k=None), "d_k"), (dict(v=A + 8), "d_v"),
    (dict(q_stride=1022), "d_q"), (dict(q_stride=1026), "d_q"), (dict(k_stride=508), "d_k"),
    (dict(dtype="bf16", k_stride=516), "d_k"), (dict(q_out=A, q_out_stride=1028), "stride"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(rotary_dim=8), "rotary_dim"),
    (dict(rotary_dim=144), "rotary_dim"), (dict(rotary_dim=-16), "rotary_dim"), (dict(inv_freq=None), "d_inv_freq"),
    (dict(amplitude=float("inf")), "rope_amplitude"), (dict(q_norm=A + 2), "d_q_norm"),
])
def test_append_refusals(change, word):
    refused(_lib.load().m1moe_kv_append(None, kv(), batch(), append(**change)), word)


def test_append_needs_a_context_last():
    lib = _lib.load()
    refused(lib.m1moe_kv_append(None, kv(), batch(), append()), "context")
    refused(lib.m1moe_kv_append(None, kv(), batch(), append(q=None, q_out=None, rotary_dim=0, inv_freq=None)),
            "context")
    refused(lib.m1moe_kv_append(None, kv(), batch(), None), "args")
    a = append()
    a.interleaved = 2
    refused(lib.m1moe_kv_append(None, kv(), batch(), a), "interleaved")


@pytest.mark.parametrize("cache,q,qs,out,outs,dtype,heads,word", [
    ("bf16", None, 1024, A + 16, 1024, 0, 8, "d_q"), ("bf16", A, 1020, A + 16, 1024, 0, 8, "d_q"),
    ("bf16", A, 1024, None, 1024, 0, 8, "d_out"), ("bf16", A, 1024, A + 16, 1026, 0, 8, "d_out"),
    ("bf16", A, 1024, A + 16, 1024, 3, 8, "dtype"), ("f32", A, 1024, A + 16, 1024, 1, 8, "bf16 cache"),
    ("bf16", A, 1024, A + 16, 1024, 0, 7, "num_heads"), ("bf16", A, 1024, A, 1024, 0, 8, "overlap"),
])
def test_attention_refusals(cache, q, qs, out, outs, dtype, heads, word):
    refused(_lib.load().m1moe_paged_attention(None, kv(dtype=cache), batch(), q, qs, out, outs, dtype, heads), word)


def test_attention_needs_a_context_last():
    refused(_lib.load().m1moe_paged_attention(None, kv(), batch(), A, 1024, A + 16, 1024, 0, 8), "context")


@pytest.mark.parametrize("logits,rows,vocab,stride,tokens,probs,word", [
    (None, 1, 8, 8, A, A, "d_logits"), (A + 4, 1, 8, 8, A, A, "d_logits"), (A, 0, 8, 8, A, A, "rows"),
    (A, 65537, 8, 8, A, A, "rows"), (A, 1, 0, 8, A, A, "vocab"), (A, 1, 262145, 262148, A, A, "vocab"),
    (A, 1, 8, 4, A, A, "stride"), (A, 1, 5, 6, A, A, "stride"), (A, 1, 8, 8, None, A, "d_tokens"),
    (A, 1, 8, 8, A, A + 2, "d_probs"),
])
def test_sample_refusals(logits, rows, vocab, stride, tokens, probs, word):
    refused(_lib.load().m1moe_sample(None, logits, rows, vocab, stride, SampleParams.make(A), tokens, probs), word)


def test_sample_settings():
    lib = _lib.load()
    refused(lib.m1moe_sample(None, A, 1, 8, 8, None, A, None), "params")
    refused(lib.m1moe_sample(None, A, 1, 8, 8, SampleParams.make(None), A, None), "d_u")
    for name in ("temperature", "top_k", "top_p", "min_p"):
        refused(lib.m1moe_sample(None, A, 1, 8, 8, SampleParams.make(A, **{name: A + 1}), A, None), "d_" + name)
    refused(lib.m1moe_sample(None, A, 1, 8, 8, SampleParams.make(A), A, None), "context")


def test_struct_sizes_match_the_header():
    """Fields in the header's order and widths (offsets of the last ones)."""
    assert ctypes.sizeof(PagedKV) == 40 and PagedKV.head_dim.offset == 32
    assert ctypes.sizeof(PagedBatch) == 48 and PagedBatch.d_prefix_pages.offset == 40
    assert ctypes.sizeof(KVAppend) == 112 and KVAppend.d_inv_freq.offset == 104
    assert ctypes.sizeof(SampleParams) == 40
