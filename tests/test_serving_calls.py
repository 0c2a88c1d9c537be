"""The C entries of the operators for several conversations on the host alone: serving.cpp,
compiled against a stand-in for the HIP runtime (serving_stub.cpp) that can be made to fail."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from m1moe_amd import KVAppend, PagedBatch, PagedKV, SampleParams, _lib

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "m1moe_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
A = 0x10000    # an aligned address that is never read


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("serving") / "libserving.so")
    subprocess.run([os.path.join(ROCM, "llvm", "bin", "clang++"), "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic",
                    "-Wno-unused-result", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include"), "-I" + CSRC,
                    "-I" + os.path.join(os.path.dirname(HERE), "include"), os.path.join(CSRC, "serving.cpp"),
                    os.path.join(HERE, "serving_stub.cpp"), "-o", out], check=True)
    lib = ctypes.CDLL(out)
    for name, res, args in _lib._PROTOTYPES:
        if name in ("m1moe_kv_append", "m1moe_paged_attention", "m1moe_sample"):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    lib.stub_ctx.restype = ctypes.c_void_p
    lib.stub_free.argtypes = [ctypes.c_void_p]
    lib.stub_live.restype = lib.stub_launches.restype = ctypes.c_long
    lib.stub_message.restype = ctypes.c_char_p
    return lib


@pytest.fixture
def ctx(lib):
    before = lib.stub_live()
    c = ctypes.c_void_p(lib.stub_ctx())
    yield c
    lib.stub_fail_memset(0)
    lib.stub_free(c)
    assert lib.stub_live() == before


def kv(**k):
    d = dict(k=A, v=A, dtype="bf16", num_pages=10, page_size=16, num_kv_heads=4, head_dim=128)
    d.update(k)
    return PagedKV.make(**d)


def batch(**k):
    d = dict(num_seqs=3, num_rows=7, row_start=A, kv_len=A, pages=A, table_stride=4)
    d.update(k)
    return PagedBatch.make(**d)


FAR = 0x10000000


def attend(lib, ctx):
    return lib.m1moe_paged_attention(ctx, kv(), batch(), A, 1024, FAR, 1024, _lib.M1MOE_F32, 8)


def sample(lib, ctx):
    return lib.m1moe_sample(ctx, A, 2, 9000, 9000, SampleParams.make(A), A, None)


@pytest.mark.parametrize("call", [attend, sample])
def test_counters_that_could_not_be_cleared_are_not_used(lib, ctx, call):
    """The memset that clears a workspace's counters fails: so does the call, what it allocated
    is given back, and the next call clears them (a launch aborts on counters that are not zero)."""
    live, launches = lib.stub_live(), lib.stub_launches()
    lib.stub_fail_memset(1)
    assert call(lib, ctx) == _lib.M1MOE_ERR_HIP and b"made to fail" in lib.stub_message()
    assert lib.stub_launches() == launches and lib.stub_live() == live
    for i in (1, 2):
        assert call(lib, ctx) == _lib.M1MOE_OK, lib.stub_message()
        assert lib.stub_launches() == launches + i
    if call is sample:
        assert lib.stub_sample_parts() == 4


B = 0x4000000    # addresses around which rows lie


def cells(base, stride, rows, n):
    """The 16-byte units of rows of n f32, stride apart."""
    return {base // 16 + r * (stride // 4) + i for r in range(rows) for i in range(n // 4)}


def test_attention_rows_that_share_memory_are_refused(lib, ctx):
    """Rows of q and of out with any offset: refused exactly if they share memory; with different
    strides, if one's rows begin before the other's end."""
    rng = np.random.default_rng(1)
    n, seen = 64, [0, 0]
    for _ in range(1500):
        rows = int(rng.integers(1, 7))
        qs, os = (4 * int(rng.integers(16, 50)) for _ in range(2))
        same = rng.random() < 0.7
        os = qs if same else os
        span = max(rows - 1, 1) * max(qs, os) + n
        out = B + 16 * int(rng.integers(-(span // 4) - 4, span // 4 + 5))
        if same and rng.random() < 0.3:      # columns of one matrix, side by side
            out = B + 4 * n if qs >= 2 * n else out
        rc = lib.m1moe_paged_attention(ctx, kv(num_kv_heads=1, head_dim=64), batch(num_rows=rows), B, qs, out, os,
                                       _lib.M1MOE_F32, 1)
        q, o = cells(B, qs, rows, n), cells(out, os, rows, n)
        clash = bool(q & o) if same or rows == 1 else max(min(q), min(o)) <= min(max(q), max(o))
        assert rc == (_lib.M1MOE_ERR_INVALID if clash else _lib.M1MOE_OK), (rows, qs, os, out - B)
        if clash and out != B:
            assert b"d_out" in lib.stub_message() and b"overlap" in lib.stub_message()
        seen[clash] += 1
    assert min(seen) > 300


@pytest.mark.parametrize("change,ok", [
    (dict(), True), (dict(q_out=B), True), (dict(q_out=B + 1024), False), (dict(q_out=B - 1024), False),
    # q, k and v columns of one matrix, q in place, or out in a column of its own
    (dict(q_stride=2560, k_stride=2560, v_stride=2560, q_out_stride=2560, k=B + 4096, v=B + 6144, q_out=B), True),
    (dict(q_stride=2560, k_stride=2560, v_stride=2560, q_out_stride=2560, k=B + 4096, v=B + 6144, q_out=B + 2048), False),
    (dict(q_stride=4096, k_stride=4096, v_stride=4096, q_out_stride=4096, k=B + 4096, v=B + 6144, q_out=B + 8192), True),
    (dict(q_stride=4096, k_stride=4096, v_stride=4096, q_out_stride=4096, k=B + 4096, v=B + 6144, q_out=B + 7680), False),
    # out over k, over v, with other strides over q's last row
    (dict(q_out=FAR, k=FAR + 4096), False), (dict(q_out=FAR, v=FAR + 6 * 4096 + 4080), False),
    (dict(q_out=FAR, v=FAR + 7 * 4096), True), (dict(q_out=B + 7 * 4096 - 16, q_out_stride=1028), False),
])
def test_append_rows_that_share_memory_are_refused(lib, ctx, change, ok):
    d = dict(dtype="f32", num_heads=8, q=B, k=A, v=A, q_stride=1024, k_stride=512, v_stride=512, q_out=FAR,
             q_out_stride=1024)
    d.update(change)
    rc = lib.m1moe_kv_append(ctx, kv(), batch(), KVAppend.make(**d))
    assert rc == (_lib.M1MOE_OK if ok else _lib.M1MOE_ERR_INVALID), lib.stub_message()
    if not ok:
        assert b"d_q_out" in lib.stub_message() and b"overlap" in lib.stub_message()
