"""The C entries of the drafted tokens' operators on the host alone: drafts.cpp, compiled
against a stand-in for the HIP runtime (serving_stub.cpp, drafts_stub.cpp); which memory a call's
outputs may share with its inputs."""
import ctypes
import os
import subprocess

import pytest

from m1moe_amd import KVAppend, PagedBatch, PagedKV, Q4Weights, _lib

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "m1moe_amd", "csrc")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
NAMES = ("m1moe_tree_plan", "m1moe_tree_append", "m1moe_tree_attention", "m1moe_tree_accept", "m1moe_matmul_q4")
MB = 1 << 20


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("drafts") / "libdrafts.so")
    subprocess.run([os.path.join(ROCM, "llvm", "bin", "clang++"), "-std=c++17", "-O1", "-shared", "-fPIC", "-Wl,-Bsymbolic",
                    "-Wno-unused-result", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(ROCM, "include"), "-I" + CSRC,
                    "-I" + os.path.join(os.path.dirname(HERE), "include"), os.path.join(CSRC, "drafts.cpp"),
                    os.path.join(HERE, "serving_stub.cpp"), os.path.join(HERE, "drafts_stub.cpp"), "-o", out], check=True)
    lib = ctypes.CDLL(out)
    for name, res, args in _lib._PROTOTYPES:
        if name in NAMES:
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    lib.stub_ctx.restype = ctypes.c_void_p
    lib.stub_free.argtypes = [ctypes.c_void_p]
    lib.stub_launches.restype = lib.stub_drafts.restype = lib.stub_live.restype = ctypes.c_long
    lib.stub_message.restype = ctypes.c_char_p
    return lib


@pytest.fixture
def ctx(lib):
    c = ctypes.c_void_p(lib.stub_ctx())
    yield c
    lib.stub_free(c)


def told(lib, rc, ok, *words):
    assert rc == (_lib.M1MOE_OK if ok else _lib.M1MOE_ERR_INVALID), lib.stub_message()
    for w in words:
        assert w.encode() in lib.stub_message(), lib.stub_message()


# (seven rows in three sequences: mask 7 x 8 x words bytes, starts 16, parents and depths 28)
@pytest.mark.parametrize("change,bad", [
    (dict(), None), (dict(mask=2 * MB + 24, words=2), "d_parents"), (dict(depth=MB + 12), "d_row_start"),
    (dict(depth=MB + 16), None), (dict(depth=2 * MB + 24), "d_parents"), (dict(depth=2 * MB + 28), None),
    (dict(depth=3 * MB + 52), "d_mask"), (dict(depth=3 * MB + 56), None),
    (dict(depth=3 * MB + 52, words=1), "d_mask"), (dict(depth=3 * MB + 56, words=2), "d_mask"),
    (dict(mask=2 * MB - 56), None), (dict(mask=2 * MB - 48), "d_parents"),
])
def test_plan_outputs(lib, ctx, change, bad):
    d = dict(start=MB, parents=2 * MB, words=1, mask=3 * MB, depth=4 * MB)
    d.update(change)
    n = lib.stub_drafts()
    rc = lib.m1moe_tree_plan(ctx, 3, 7, d["start"], d["parents"], d["words"], d["mask"], d["depth"])
    told(lib, rc, bad is None, *([bad, "overlap"] if bad else []))
    assert lib.stub_drafts() == n + (bad is None)


def kv(k=64 * MB, v=128 * MB):
    return PagedKV.make(k, v, "bf16", 10, 16, 4, 128)    # planes of 160 KB


def batch():
    return PagedBatch.make(3, 7, MB, MB + 256, MB + 512, 4)


@pytest.mark.parametrize("depth,ok", [(2 * MB, True), (8 * MB + 64, False), (8 * MB + 7 * 4096 - 4, False),
                                      (8 * MB + 7 * 4096, True), (8 * MB - 28, True), (8 * MB - 24, False)])
def test_append_depths(lib, ctx, depth, ok):
    a = KVAppend.make("f32", 8, 4 * MB, 5 * MB, 6 * MB, 1024, 512, 512, 8 * MB, 1024)
    told(lib, lib.m1moe_tree_append(ctx, kv(), batch(), a, depth), ok, *([] if ok else ["d_depth"]))
    told(lib, lib.m1moe_tree_append(ctx, kv(), batch(), KVAppend.make("f32", 8, None, 5 * MB, 6 * MB, 0, 512, 512,
                                                                      None, 0), depth), True)


@pytest.mark.parametrize("mask,ok", [(2 * MB, True), (8 * MB, False), (8 * MB + 7 * 4096 - 8, False),
                                     (8 * MB + 7 * 4096, True), (8 * MB - 112, True), (8 * MB - 104, False)])
def test_attention_masks(lib, ctx, mask, ok):
    rc = lib.m1moe_tree_attention(ctx, kv(), batch(), mask, 2, 4 * MB, 1024, 8 * MB, 1024, _lib.M1MOE_F32, 8)
    told(lib, rc, ok, *([] if ok else ["d_mask"]))
    rc = lib.m1moe_tree_attention(ctx, kv(), batch(), 2 * MB, 2, 4 * MB, 1024, 4 * MB + 16, 1024, _lib.M1MOE_F32, 8)
    told(lib, rc, False, "d_out", "overlap")


INS = {"d_parents": 2 * MB, "d_drafts": 2 * MB + 256, "d_drawn": 2 * MB + 512}
OUTS = {"d_path": 3 * MB, "d_accepted": 3 * MB + 256, "d_next": 3 * MB + 512, "d_past": 3 * MB + 768}


@pytest.mark.parametrize("out", OUTS)
def test_accept_outputs(lib, ctx, out):
    size = 28 if out == "d_path" else 12
    others = {**INS, **OUTS, "d_row_start": MB, "d_kv_len": MB + 256, "d_pages": MB + 512}
    sizes = {"d_row_start": 16, "d_kv_len": 12, "d_pages": 48, "d_accepted": 12, "d_next": 12, "d_past": 12}
    for name, at in others.items():
        if name == out:
            continue
        for to, ok in ((at, False), (at + sizes.get(name, 28) - 4, False), (at + sizes.get(name, 28), True),
                       (at - size + 4, False), (at - size, True)):
            o = {**OUTS, out: to}
            rc = lib.m1moe_tree_accept(ctx, PagedKV.array([kv()]), 1, batch(), *INS.values(), *o.values())
            told(lib, rc, ok, *([] if ok else [out, name, "overlap"]))


def test_accept_planes(lib, ctx):
    plane = 10 * 16 * 4 * 128 * 2

    def call(*at):
        caches = [kv(at[i], at[i + 1]) for i in range(0, len(at), 2)]
        return lib.m1moe_tree_accept(ctx, PagedKV.array(caches), len(caches), batch(), *INS.values(), *OUTS.values())
    base = 64 * MB
    told(lib, call(*(base + i * plane for i in (3, 1, 0, 2))), True)
    told(lib, call(base, base + plane - 16), False, "overlap")
    told(lib, call(base, base + plane, base + 3 * plane, base + plane), False, "overlap")
    told(lib, call(base, base), False, "overlap")
    told(lib, call(*(base + i * plane for i in range(128))), True)


def q4(lib, ctx, **k):
    d = dict(w=16 * MB, s=17 * MB, b=18 * MB, x=20 * MB, xt=0, xs=128, t=3, r=None, y=24 * MB, yt=0, ys=40)
    d.update(k)
    w = Q4Weights.make(d["w"], d["s"], d["b"], 40, 128, 64)   # 2560 bytes, twice 160
    return lib.m1moe_matmul_q4(ctx, w, d["x"], d["xt"], d["xs"], d["t"], d["r"], d["y"], d["yt"], d["ys"])


@pytest.mark.parametrize("change,bad", [
    (dict(), None), (dict(r=24 * MB), None), (dict(r=24 * MB + 16), "d_residual"), (dict(r=24 * MB + 480), None),
    (dict(r=24 * MB + 464), "d_residual"), (dict(y=20 * MB), "d_x"), (dict(y=20 * MB + 1520), "d_x"),
    (dict(y=20 * MB + 1536), None), (dict(y=16 * MB + 2544), "d_w"), (dict(y=16 * MB + 2560), None),
    (dict(y=17 * MB + 144), "d_scales"), (dict(y=18 * MB - 464), "d_biases"), (dict(y=18 * MB - 480), None),
    # x and y columns of one matrix
    (dict(xs=168, ys=168, y=20 * MB + 512), None), (dict(xs=168, ys=168, y=20 * MB + 496), "d_x"),
    (dict(xt=1, yt=1, r=24 * MB + 240), None), (dict(xt=1, yt=1, r=24 * MB + 224), "d_residual"),
])
def test_q4_outputs(lib, ctx, change, bad):
    n = lib.stub_drafts()
    told(lib, q4(lib, ctx, **change), bad is None, *([bad, "overlap"] if bad else []))
    assert lib.stub_drafts() == n + (bad is None)


# (planes of 160 KB; 28 bytes of path, 12 of the others)
@pytest.mark.parametrize("out", OUTS)
def test_accept_outputs_and_planes(lib, ctx, out):
    plane, size = 10 * 16 * 4 * 128 * 2, 28 if out == "d_path" else 12
    caches = PagedKV.array([kv(96 * MB, 64 * MB), kv(64 * MB + plane, 128 * MB)])
    for at, ok in ((64 * MB, False), (64 * MB - size, True), (64 * MB - size + 4, False), (64 * MB + 2 * plane - 4, False),
                   (64 * MB + 2 * plane, True), (96 * MB + plane // 2, False), (128 * MB + plane - 4, False),
                   (128 * MB + plane, True), (MB + 1024, True)):
        rc = lib.m1moe_tree_accept(ctx, caches, 2, batch(), *INS.values(), *{**OUTS, out: at}.values())
        told(lib, rc, ok, *([] if ok else [out, "overlap"]))


def test_q4_counters_that_could_not_be_cleared_are_not_used(lib, ctx):
    """(the stand-in's launch ends the process if a counter is not zero)"""
    live, n = lib.stub_live(), lib.stub_drafts()
    lib.stub_fail_memset(1)
    assert q4(lib, ctx) not in (_lib.M1MOE_OK, _lib.M1MOE_ERR_INVALID)
    assert lib.stub_live() == live and lib.stub_drafts() == n
    lib.stub_fail_memset(0)
    for _ in range(2):
        told(lib, q4(lib, ctx), True)
    assert lib.stub_drafts() == n + 2 and lib.stub_live() == live + 2
