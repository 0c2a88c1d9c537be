"""What the decoder and the chat command take of the sampler: settings that reach it,
and scaled rotary frequencies.  CPU only."""
import numpy as np
import pytest

from m1moe_amd import chat, rope_frequencies


class Recorder:
    def __init__(self):
        self.calls = []

    def forward(self, token, **k):
        self.calls.append((token, k))
        return 7


def test_chat_engine_passes_top_k_and_min_p_only_when_set():
    r = Recorder()
    chat.DecoderEngine(r, 1).forward(3, 0.7, 0.9)
    chat.DecoderEngine(r, 1, top_k=40).forward(3, 0.7, 0.9)
    chat.DecoderEngine(r, 1, min_p=0.05).forward(3, 0.7, 0.9)
    assert [sorted(k) for _, k in r.calls] == [["rng", "temperature", "top_p"]] + \
        [["min_p", "rng", "temperature", "top_k", "top_p"]] * 2
    assert r.calls[1][1]["top_k"] == 40 and r.calls[2][1]["min_p"] == 0.05


def test_chat_arguments():
    a = chat.parse_args(["--top-k", "40", "--min-p", "0.05", "--top-p", "0.5"])
    assert (a["top_k"], a["min_p"], a["top_p"]) == (40, 0.05, 0.5)
    a = chat.parse_args(["--top-k", "many", "--min-p"])
    assert (a["top_k"], a["min_p"]) == (0, 0.0)


def test_rope_frequencies():
    f, amp = rope_frequencies(1e4, 128)
    i = np.arange(64)
    assert amp == 1.0 and f.dtype == np.float32
    assert np.array_equal(f, (1e4 ** (-2 * i / 128)).astype(np.float32))
    g, _ = rope_frequencies(1e4, 128, 4.0, "linear")
    assert np.array_equal(g, (1e4 ** (-2 * i / 128) / 4).astype(np.float32))
    g, _ = rope_frequencies(1e4, 128, 4.0, "base")
    assert g[0] == 1.0 and abs(g[-1] / f[-1] - 0.25) < 1e-6
    g, amp = rope_frequencies(1e4, 128, 4.0, "parts", trained_len=2048)
    turns = 2048 * (1e4 ** (-2 * i / 128)) / (2 * np.pi)
    assert np.array_equal(g[turns >= 32], f[turns >= 32])
    assert np.allclose(g[turns <= 1], f[turns <= 1] / 4, rtol=1e-6)
    mid = (turns > 1) & (turns < 32)
    assert np.all((g[mid] < f[mid]) & (g[mid] > f[mid] / 4))
    assert abs(amp - (0.1 * np.log(4) + 1)) < 1e-12
    assert rope_frequencies(1e4, 2, 4.0, "base")[0].tolist() == [1.0]


@pytest.mark.parametrize("args", [(1e4, 0), (1e4, 7), (0.0, 8), (1e4, 8, 0.5), (1e4, 8, 2.0, "other"),
                                  (1e4, 8, 2.0, "parts"), (1e4, 8, 2.0, "parts", 100, 5.0, 5.0)])
def test_rope_frequencies_refusals(args):
    with pytest.raises(ValueError):
        rope_frequencies(*args)


class FakeBuffer:
    addr = 0x1000

    def __init__(self, ctx, nbytes):
        self.ctx, self.nbytes = ctx, nbytes
        ctx.live += 1

    def upload(self, a):
        assert a.nbytes <= self.nbytes
        return self

    def download(self, dtype, count=None):
        return np.zeros(self.nbytes // 4 if count is None else count, dtype)

    def free(self):
        self.ctx.live -= 1


class FakeContext:
    """Counts its live buffers; sync fails when asked to."""
    lib, handle, live, fail_sync = None, None, 0, False

    def alloc(self, n):
        return FakeBuffer(self, n)

    def to_device(self, a):
        return FakeBuffer(self, a.nbytes)

    def sync(self):
        if self.fail_sync:
            raise RuntimeError("sync")


@pytest.mark.parametrize("where", ["", "prefill", "step", "sample", "sync", "top_k"])
@pytest.mark.parametrize("call", ["generate_sampled", "generate", "prefill"])
def test_buffers_are_freed_when_a_call_raises(monkeypatch, call, where):
    """A refused prompt, a full cache, a device error: the call's own buffers go all the same."""
    from m1moe_amd import decoder

    def step(name):
        def f(*a, **k):
            if where == name:
                raise RuntimeError(name)
        return f
    dec = decoder.Decoder.__new__(decoder.Decoder)
    dec.ctx, dec.handle = FakeContext(), None
    dec.ctx.fail_sync = where == "sync"
    dec.shape = type("Shape", (), {"vocab": 100})
    dec._tok = dec._logits = FakeBuffer(dec.ctx, 16)
    dec.reset, dec.prefill_device = lambda: None, step("prefill")
    dec.step_device = dec.step_seq = step("step")
    monkeypatch.setattr(decoder.DenseOps, "__init__", lambda self, ctx: None)
    monkeypatch.setattr(decoder.DenseOps, "sample", step("sample"))
    reached = {"generate_sampled": ("prefill", "step", "sample", "sync", "top_k"), "generate": ("step", "sync"),
               "prefill": ("prefill", "sync")}[call]
    args = {"generate_sampled": ([1, 2], 3, 0.7), "generate": ([1, 2], 3), "prefill": ([1, 2],)}[call]
    more = dict(top_k=1 << 40) if call == "generate_sampled" and where == "top_k" else {}
    before = dec.ctx.live
    if where in reached:
        with pytest.raises((RuntimeError, OverflowError, ValueError)):
            getattr(dec, call)(*args, **more)
    else:
        got = getattr(dec, call)(*args)
        assert call == "prefill" or len(got) == 4
    assert dec.ctx.live == before
