"""Memory that the drafted tokens' operators write and, elsewhere in the same launch, read: refused.
On the host alone, with the stand-ins of test_drafts_calls.py."""
import pytest

from m1moe_amd import KVAppend, PagedBatch, PagedKV, _lib
from test_drafts_calls import INS, MB, OUTS, ctx, kv, lib, told  # noqa: F401

PLANE = 10 * 16 * 4 * 128 * 2
BATCH = {"d_row_start": (MB, 16), "d_kv_len": (MB + 256, 12), "d_pages": (MB + 512, 48)}


def batch(prefix=0, **at):
    d = {k: v[0] for k, v in BATCH.items()}
    d.update(at)
    return PagedBatch.make(3, 7, d["d_row_start"], d["d_kv_len"], d["d_pages"], 4, prefix, 2 * MB + 4096 if prefix else None)


def places(at, size, span):
    """(address, whether `size` bytes there are apart from the `span` bytes at `at`)"""
    return ((at, False), (at + span - 4, False), (at + span, True), (at - size + 4, False), (at - size, True))


@pytest.mark.parametrize("name", list(INS) + list(BATCH))
@pytest.mark.parametrize("plane", [64 * MB, 96 * MB, 128 * MB + PLANE])
def test_accept_inputs_and_planes(lib, ctx, name, plane):  # noqa: F811
    caches = PagedKV.array([kv(128 * MB, 64 * MB), kv(96 * MB, 128 * MB + PLANE)])
    size = BATCH[name][1] if name in BATCH else 28
    for at, ok in places(plane, size, PLANE):
        ins = {**INS, **({name: at} if name in INS else {})}
        b = batch(**({name: at} if name in BATCH else {}))
        if ok and plane == 128 * MB + PLANE and at < plane:
            continue   # (the plane before it)
        rc = lib.m1moe_tree_accept(ctx, caches, 2, b, *ins.values(), *OUTS.values())
        told(lib, rc, ok, *([] if ok else [name, "overlap"]))


@pytest.mark.parametrize("name", ["d_depth"] + list(BATCH))
def test_append_writes_nothing_that_it_reads(lib, ctx, name):  # noqa: F811
    size = BATCH[name][1] if name in BATCH else 28
    a = KVAppend.make("f32", 8, 4 * MB, 5 * MB, 6 * MB, 1024, 512, 512, 8 * MB, 1024)
    none = KVAppend.make("f32", 8, None, 5 * MB, 6 * MB, 0, 512, 512, None, 0)
    for to, span in ((64 * MB, PLANE), (128 * MB, PLANE), (8 * MB, 7 * 4096)):
        for at, ok in places(to, size, span):
            b, depth = batch(**({name: at} if name in BATCH else {})), at if name == "d_depth" else 2 * MB
            told(lib, lib.m1moe_tree_append(ctx, kv(), b, a, depth), ok, *([] if ok else [name, "overlap"]))
            told(lib, lib.m1moe_tree_append(ctx, kv(), b, none, depth), ok or span != PLANE)


@pytest.mark.parametrize("name", ["d_mask", "d_prefix_pages"] + list(BATCH))
def test_attention_writes_nothing_that_it_reads(lib, ctx, name):  # noqa: F811
    sizes = {**{k: v[1] for k, v in BATCH.items()}, "d_mask": 112, "d_prefix_pages": 8}
    at0 = {**{k: v[0] for k, v in BATCH.items()}, "d_mask": 2 * MB, "d_prefix_pages": 2 * MB + 4096}

    def call(out, prefix=0):
        return lib.m1moe_tree_attention(ctx, kv(), batch(prefix), 2 * MB, 2, 4 * MB, 1024, out, 1024, _lib.M1MOE_F32, 8)
    span = 7 * 4096
    for out, ok in ((at0[name] - span + 16, False), (at0[name], False)):
        told(lib, call(out, 20), ok, "d_out", "overlap")
    if name == "d_prefix_pages":     # (without a prefix there are none; 20 positions have two pages)
        told(lib, call(at0[name]), True)
        told(lib, call(at0[name] + 16, 20), True)


@pytest.mark.parametrize("plane,what", [(64 * MB, "d_k"), (128 * MB, "d_v")])
def test_attention_output_and_cache(lib, ctx, plane, what):  # noqa: F811
    span = 7 * 4096
    for out, ok in ((plane - span, True), (plane - span + 16, False), (plane + PLANE - 16, False), (plane + PLANE, True)):
        rc = lib.m1moe_tree_attention(ctx, kv(), batch(), 2 * MB, 2, 4 * MB, 1024, out, 1024, _lib.M1MOE_F32, 8)
        told(lib, rc, ok, *([] if ok else ["d_out", what, "overlap"]))
