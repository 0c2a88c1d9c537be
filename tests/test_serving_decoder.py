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
