"""What calls need of a context's workspaces, and the pieces of a shared prefix: the library's own
plans, which run on the host (plans_probe.cpp, linked against the built library)."""
import ctypes
import os
import subprocess

import pytest

from m1moe_amd import _lib

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "m1moe_amd", "csrc")
CUS = 256


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plans") / "libplans.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I" + CSRC, os.path.join(HERE, "plans_probe.cpp"),
                    _lib.LIB_PATH, "-Wl,-rpath," + os.path.dirname(_lib.LIB_PATH), "-o", out], check=True)
    lib = ctypes.CDLL(out)
    lib.probe_q4.restype = lib.probe_paged.restype = ctypes.c_int64
    return lib


def paged(probe, rows, heads, kv_heads, hd, bf16, prefix):
    """(floats a call makes sure of, those it uses, pieces of the prefix)"""
    splits, used = ctypes.c_int(), ctypes.c_int64()
    n = probe.probe_paged(rows, heads, kv_heads, hd, bf16, prefix, CUS, ctypes.byref(splits), ctypes.byref(used))
    return n, used.value, splits.value


def q4(probe, rows, cols, group, tokens, bf16):
    """Floats a call makes sure of, no fewer than it uses."""
    used, shared = ctypes.c_int64(), ctypes.c_int()
    n = probe.probe_q4(rows, cols, group, tokens, bf16, CUS, ctypes.byref(used), ctypes.byref(shared))
    assert used.value <= n and shared.value <= CUS
    return n


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows,cols,group", [(6144, 4096, 64), (50304, 2048, 64), (2048, 2048, 64), (2048, 1024, 32),
                                             (48, 4096, 128), (129, 352, 32), (70, 65536, 64)])
def test_products_of_fewer_tokens_need_no_more(probe, rows, cols, group, bf16):
    need = [q4(probe, rows, cols, group, t, bf16) for t in range(1, 2101)]
    assert all(a <= b for a, b in zip(need, need[1:]))
    assert need[-1] > 0
    # (nor do those of smaller weights, behind a call of more than 32 tokens)
    for n, k in ((rows // 2 + 1, cols), (rows, cols - cols // 2 // group * group), (40, group)):
        assert all(q4(probe, n, k, group, t, bf16) <= need[t - 1] for t in range(33, 700))
        assert max(q4(probe, n, k, group, t, bf16) for t in range(1, 33)) <= need[32]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (16, 16, 128), (32, 4, 128), (8, 8, 64), (40, 1, 128), (4, 2, 256)])
def test_attention_of_fewer_rows_needs_no_more(probe, heads, kv_heads, hd, bf16):
    before = None
    for prefix in (0, 1, 64, 500, 777, 1024, 4096):
        need, used, _ = zip(*(paged(probe, r, heads, kv_heads, hd, bf16, prefix) for r in range(1, 2200)))
        assert all(u <= n for u, n in zip(used, need))
        assert all(a <= b for a, b in zip(need, need[1:])), prefix
        assert before is None or all(a <= b for a, b in zip(before, need)), prefix
        before = need


# (measured: 32/8 heads, bf16, 800 rows behind 500, 2 pieces 44.9 us, 5 54.8; behind 4096, 513 rows
# 2 pieces 106, 3 and 5 87)
@pytest.mark.parametrize("rows,heads,kv_heads,bf16,prefix,splits", [
    (800, 32, 8, 1, 500, (2, 2)), (513, 32, 8, 1, 500, (2, 2)), (2100, 16, 16, 1, 500, (1, 1)),
    (513, 32, 8, 0, 500, (1, 1)), (513, 32, 8, 1, 4096, (3, 5)), (513, 32, 8, 0, 4096, (3, 5)),
    (800, 16, 16, 1, 4096, (4, 4)), (2100, 32, 8, 1, 4096, (2, 4)), (64, 32, 8, 0, 4096, (8, 8)),
    (115, 16, 16, 1, 500, (7, 7)), (1, 8, 8, 1, 63, (1, 1)), (1, 8, 8, 1, 1, (1, 1)), (1, 1, 1, 1, 1 << 20, (32, 32)),
    (1 << 20, 1, 1, 1, 4096, (1, 1))])
def test_pieces_of_a_prefix(probe, rows, heads, kv_heads, bf16, prefix, splits):
    """More pieces where that fills the card's CUs, and none that cost more than they give."""
    assert splits[0] <= paged(probe, rows, heads, kv_heads, 128, bf16, prefix)[2] <= splits[1]
