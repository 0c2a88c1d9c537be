"""The C entries of the operators for several conversations on the host alone: serving.cpp,
compiled against a stand-in for the HIP runtime (serving_stub.cpp) that can be made to fail."""
import ctypes
import os
import subprocess

import pytest

from m1moe_amd import PagedBatch, PagedKV, SampleParams, _lib

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
