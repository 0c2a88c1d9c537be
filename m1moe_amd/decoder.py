"""Host-side mirror of the reference decoder (InferenceEngine) over the C ABI.

``Decoder.forward(token)`` is InferenceEngine.forward(token:) at temperature
0 (Sources/M1MoE/InferenceEngine.swift:125-156): embed, every layer's
attention and MoE block, final norm, lm_head, greedy token.  The whole step
runs on the GPU (m1moe_dec_step) with the token and the position in device
memory; ``forward`` adds the one host round-trip the reference's API implies
(the token in, the token out).  ``step_device`` is the same step without it,
for graph-captured loops.

The dense building blocks (RMSNorm, bf16 matvec, decode attention, argmax)
are exposed one by one in ``DenseOps`` for tests and for callers that
compose their own layers.
"""
from __future__ import annotations

import contextlib
import ctypes
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _lib
from ._lib import (DecShape, KVAppend, PagedBatch, PagedKV, SampleParams, W_EMBED, W_FINAL_NORM, W_IN_NORM, W_K, W_K_NORM, W_LM_HEAD, W_O,
                   W_PER_LAYER, W_POST_NORM, W_Q, W_Q_NORM, W_V, check, dtype_code)
from .engine import DeviceBuffer, HIPContext, _ptr
from .sampling import sample_token

WEIGHT_NAMES = {
    W_EMBED: "model.embed_tokens.weight",
    W_LM_HEAD: "lm_head.weight",
    W_FINAL_NORM: "model.norm.weight",
    W_IN_NORM: "model.layers.{}.input_layernorm.weight",
    W_POST_NORM: "model.layers.{}.post_attention_layernorm.weight",
    W_Q: "model.layers.{}.self_attn.q_proj.weight",
    W_K: "model.layers.{}.self_attn.k_proj.weight",
    W_V: "model.layers.{}.self_attn.v_proj.weight",
    W_O: "model.layers.{}.self_attn.o_proj.weight",
    W_Q_NORM: "model.layers.{}.self_attn.q_norm.weight",
    W_K_NORM: "model.layers.{}.self_attn.k_norm.weight",
}  # InferenceEngine.swift:580-599 (WeightKeys)


@dataclass(frozen=True)
class AttentionSpec:
    """AttentionSpec, ModelSpec.swift:62-75."""

    num_heads: int
    num_kv_heads: int
    head_dim: int
    rope_theta: float
    max_seq_len: int
    gpu_kv_seq_prealloc: int

    @property
    def q_dim(self) -> int:
        return self.num_heads * self.head_dim

    @property
    def kv_dim(self) -> int:
        return self.num_kv_heads * self.head_dim

    @property
    def hpkv(self) -> int:
        return self.num_heads // self.num_kv_heads


@dataclass(frozen=True)
class DecoderSpec:
    """The dense part of ModelSpec (ModelSpec.swift:14-22): vocabulary, norm
    epsilon, attention, and whether the model has per-head q/k RMSNorm (the
    reference sets it for architecture "olmoe", InferenceEngine.swift:55)."""

    architecture: str
    vocab_size: int
    rms_norm_eps: float
    attention: AttentionSpec

    @property
    def qk_norm(self) -> bool:
        return self.architecture == "olmoe"

    @staticmethod
    def from_dict(d: dict) -> "DecoderSpec":
        a = d["attention"]
        return DecoderSpec(
            architecture=str(d.get("architecture", "")),
            vocab_size=int(d["vocab_size"]),
            rms_norm_eps=float(d["rms_norm_eps"]),
            attention=AttentionSpec(int(a["num_heads"]), int(a["num_kv_heads"]),
                                    int(a["head_dim"]), float(a["rope_theta"]),
                                    int(a["max_seq_len"]), int(a["gpu_kv_seq_prealloc"])))

    def dec_shape(self, max_seq: Optional[int] = None) -> DecShape:
        """KV cache of gpu_kv_seq_prealloc positions unless max_seq is given
        (MetalContext preallocates that many, InferenceEngine.swift:353)."""
        a = self.attention
        return DecShape(self.vocab_size, a.num_heads, a.num_kv_heads, a.head_dim,
                        int(max_seq if max_seq is not None else a.gpu_kv_seq_prealloc),
                        1 if self.qk_norm else 0, a.rope_theta, self.rms_norm_eps)


def weight_count(which: int, hidden: int, s: DecShape) -> int:
    """Element count of dense tensor `which` (include/m1moe_hip.h, M1MOE_W_*)."""
    qd, kvd = s.num_heads * s.head_dim, s.num_kv_heads * s.head_dim
    return {W_EMBED: s.vocab * hidden, W_LM_HEAD: s.vocab * hidden, W_FINAL_NORM: hidden,
            W_IN_NORM: hidden, W_POST_NORM: hidden, W_Q: qd * hidden, W_K: kvd * hidden,
            W_V: kvd * hidden, W_O: hidden * qd, W_Q_NORM: s.head_dim,
            W_K_NORM: s.head_dim}[which]


def rope_frequencies(theta: float, rotary_dim: int, factor: float = 1.0, kind: str = "parts",
                     trained_len: int = 0, slow: float = 1.0, fast: float = 32.0):
    """(inv_freq f32 [rotary_dim / 2], amplitude) for KVAppend: theta^(-2i / rotary_dim),
    for contexts `factor` times the trained one: "linear" divides every frequency by it
    (position interpolation), "base" raises theta so that only the slowest pair's is (a
    scaled base), "parts" divides those of pairs with at most `slow` turns over trained_len
    positions, keeps those with `fast` or more, blends between and scales cos and sin by
    0.1 ln(factor) + 1: the formulas of the YaRN paper, whose blend is linear in the turns.
    A checkpoint whose own blend is linear in the pair's index, or with another amplitude, needs
    frequencies of its own.  No published values are at hand to compare with: parity unpinned."""
    if rotary_dim <= 0 or rotary_dim % 2 or not theta > 0 or not factor >= 1:
        raise ValueError(f"rotary_dim {rotary_dim} / theta {theta} / factor {factor}: need an even "
                         "positive rotary_dim, theta > 0 and factor >= 1")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    if kind == "base":
        if rotary_dim > 2:
            theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
        return (theta ** (-2 * i / rotary_dim)).astype(np.float32), 1.0
    f = theta ** (-2 * i / rotary_dim)
    if kind == "linear":
        return (f / factor).astype(np.float32), 1.0
    if kind != "parts":
        raise ValueError(f"unknown kind {kind!r}: linear, base or parts")
    if factor == 1:
        return f.astype(np.float32), 1.0
    if trained_len <= 0 or not 0 <= slow < fast:
        raise ValueError("kind \"parts\" needs trained_len > 0 and 0 <= slow < fast")
    keep = np.clip((trained_len * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
    return (f * keep + f / factor * (1 - keep)).astype(np.float32), 0.1 * float(np.log(factor)) + 1


class DenseOps:
    """The dense kernels one by one (asynchronous on the context stream)."""

    def __init__(self, ctx: HIPContext):
        self.ctx = ctx
        self.lib = ctx.lib

    def rmsnorm(self, x, w, out, n: int, eps: float) -> None:
        check(self.lib.m1moe_rmsnorm(self.ctx.handle, _ptr(x), _ptr(w), _ptr(out), int(n),
                                     ctypes.c_float(eps)), "m1moe_rmsnorm")

    def matvec_bf16(self, w, x, residual, y, rows: int, cols: int) -> None:
        check(self.lib.m1moe_matvec_bf16(self.ctx.handle, _ptr(w), _ptr(x), _ptr(residual),
                                         _ptr(y), int(rows), int(cols)), "m1moe_matvec_bf16")

    def attention_decode(self, q, kcache, vcache, out, num_heads: int, num_kv_heads: int,
                         head_dim: int, seq_len: int) -> None:
        check(self.lib.m1moe_attention_decode(self.ctx.handle, _ptr(q), _ptr(kcache),
                                              _ptr(vcache), _ptr(out), int(num_heads),
                                              int(num_kv_heads), int(head_dim), int(seq_len)),
              "m1moe_attention_decode")

    def argmax(self, x, n: int, idx) -> None:
        check(self.lib.m1moe_argmax(self.ctx.handle, _ptr(x), int(n), _ptr(idx)), "m1moe_argmax")

    # several conversations at once: a KV cache in pages, attention over it, sampling
    def kv_append(self, kv: PagedKV, batch: PagedBatch, args: KVAppend) -> None:
        """q/k norm, RoPE and the store of k and v for every row of the batch."""
        check(self.lib.m1moe_kv_append(self.ctx.handle, ctypes.byref(kv), ctypes.byref(batch),
                                       ctypes.byref(args)), "m1moe_kv_append")

    def paged_attention(self, kv: PagedKV, batch: PagedBatch, q, q_stride: int, out,
                        out_stride: int, dtype, num_heads: int) -> None:
        """Every row of the batch against its own sequence's positions up to its own."""
        check(self.lib.m1moe_paged_attention(
            self.ctx.handle, ctypes.byref(kv), ctypes.byref(batch), _ptr(q), q_stride, _ptr(out),
            out_stride, dtype_code(dtype), num_heads), "m1moe_paged_attention")

    def sample(self, logits, rows: int, vocab: int, stride: int, params: SampleParams, tokens,
               probs=None) -> None:
        """One token per row of f32 logits from given random numbers."""
        check(self.lib.m1moe_sample(self.ctx.handle, _ptr(logits), rows, vocab, stride,
                                    ctypes.byref(params), _ptr(tokens), _ptr(probs)),
              "m1moe_sample")


class Decoder:
    """InferenceEngine (InferenceEngine.swift:19-156) over a HIPContext that
    holds the MoE layers: dense weights resident in HBM, f32 KV cache of
    max_seq positions per layer."""

    def __init__(self, ctx: HIPContext, shape: DecShape):
        self.ctx = ctx
        self.lib = ctx.lib
        self.shape = shape
        self.hidden = ctx.shape.hidden
        self.num_layers = ctx.shape.num_layers
        h = ctypes.c_void_p()
        check(self.lib.m1moe_dec_create(ctx.handle, ctypes.byref(shape), ctypes.byref(h)),
              "m1moe_dec_create")
        self.handle = h
        self._tok = ctx.alloc(16)     # token in/out of forward()
        self._logits = ctx.alloc(4 * shape.vocab)
        self._draw = ctx.alloc(32)    # a sampled step's settings and random number

    def close(self) -> None:
        if self.handle:
            self.lib.m1moe_dec_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def upload(self, which: int, layer: int, bf16: np.ndarray) -> None:
        a = np.ascontiguousarray(bf16, dtype=np.uint16).reshape(-1)
        check(self.lib.m1moe_dec_upload(self.handle, int(which), int(layer),
                                        a.ctypes.data_as(ctypes.POINTER(ctypes.c_uint16)),
                                        ctypes.c_uint64(a.size)), "m1moe_dec_upload")

    def upload_all(self, weights) -> None:
        """weights(which, layer) -> bf16 array, for every tensor of the model."""
        for which in range(11):
            if which in (W_Q_NORM, W_K_NORM) and not self.shape.qk_norm:
                continue
            layers = range(self.num_layers) if which in W_PER_LAYER else [0]
            for layer in layers:
                self.upload(which, layer, weights(which, layer))

    @staticmethod
    @contextlib.contextmanager
    def _held():
        """hold(buffer): freed at the end of the block, also when it raises."""
        with contextlib.ExitStack() as stack:
            def hold(buf):
                stack.callback(buf.free)
                return buf
            yield hold

    def reset(self) -> None:
        """InferenceEngine.reset (InferenceEngine.swift:159-163)."""
        check(self.lib.m1moe_dec_reset(self.handle), "m1moe_dec_reset")

    def position(self) -> int:
        p = ctypes.c_int32()
        check(self.lib.m1moe_dec_position(self.handle, ctypes.byref(p)), "m1moe_dec_position")
        return int(p.value)

    def step_device(self, token_in, token_out, logits=None) -> None:
        """One step with the tokens in device memory (asynchronous)."""
        check(self.lib.m1moe_dec_step(self.handle, _ptr(token_in), _ptr(token_out),
                                      _ptr(logits)), "m1moe_dec_step")

    def step_seq(self, seq, n_prompt: int, seq_cap: int, logits=None) -> None:
        """Sequence-mode step (asynchronous): embeds seq[pos]; past the prompt
        stores the greedy token at seq[pos + 1].  n_prompt + n_gen calls after
        reset() run prompt-then-generate with no host round trip."""
        check(self.lib.m1moe_dec_step_seq(self.handle, _ptr(seq), int(n_prompt), int(seq_cap),
                                          _ptr(logits)), "m1moe_dec_step_seq")

    def prefill_device(self, tokens, T: int, token_out, logits=None) -> None:
        """The T prompt tokens (device int32) through the decoder in one batch
        per layer (asynchronous); token_out receives the greedy next token."""
        check(self.lib.m1moe_dec_prefill(self.handle, _ptr(tokens), int(T), _ptr(token_out),
                                         _ptr(logits)), "m1moe_dec_prefill")

    def prefill(self, prompt, return_logits: bool = False):
        """The prompt at once from the current position; returns the greedy
        token after its last token (and that token's logits when asked)."""
        prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        with self._held() as hold:
            d = hold(self.ctx.to_device(prompt))
            self.prefill_device(d, prompt.size, self._tok, self._logits)
            self.ctx.sync()
        nxt = int(self._tok.download(np.int32, 1)[0])
        if return_logits:
            return nxt, self._logits.download(np.float32, self.shape.vocab)
        return nxt

    def generate(self, prompt, n_gen: int):
        """Sources/bench/main.swift:136-163 at temperature 0: the prompt
        forwarded token by token, then n_gen greedy steps; returns the
        n_gen + 1 greedy tokens (the prompt's own prediction first)."""
        prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        P, cap = prompt.size, prompt.size + n_gen + 1
        with self._held() as hold:
            seq = hold(self.ctx.alloc(4 * cap))
            seq.upload(np.concatenate([prompt, np.zeros(cap - P, np.int32)]))
            self.reset()
            for _ in range(P + n_gen):
                self.step_seq(seq, P, cap)
            self.ctx.sync()
            return seq.download(np.int32)[P:]

    def _sample_params(self, buf: DeviceBuffer, u, temperature, top_k, top_p, min_p):
        """Copies n draws and the settings (one each) to buf, 4 + n words; what makes
        SampleParams of draw i."""
        words = np.zeros(4 + np.size(u), np.float32)
        words[:4] = [temperature, 0, top_p, min_p]
        words[1:2].view(np.int32)[0] = top_k
        words[4:] = u
        at = buf.upload(words).addr
        return lambda i: SampleParams.make(at + 16 + 4 * i, at, at + 4, at + 8, at + 12)

    def generate_sampled(self, prompt, n_gen: int, temperature: float, top_p: float = 1.0,
                         top_k: int = 0, min_p: float = 0.0, u=None,
                         rng: Optional[np.random.Generator] = None):
        """generate() with every token drawn on the GPU (m1moe_sample) from the
        n_gen + 1 uniform numbers u (from rng when None): the prompt in one batch, then
        a step per token, and no host round trip between them."""
        prompt = np.ascontiguousarray(prompt, dtype=np.int32)
        n, V = n_gen + 1, self.shape.vocab
        if u is None:
            u = (rng or np.random.default_rng()).random(n, dtype=np.float32)
        if np.size(u) != n:
            raise ValueError(f"{np.size(u)} random numbers for {n} tokens")
        ops = DenseOps(self.ctx)
        with self._held() as hold:
            buf, toks = hold(self.ctx.alloc(4 * (4 + n))), hold(self.ctx.alloc(4 * n))
            d = hold(self.ctx.to_device(prompt))
            params = self._sample_params(buf, u, temperature, top_k, top_p, min_p)
            self.reset()
            self.prefill_device(d, prompt.size, self._tok, self._logits)
            for i in range(n):
                if i:
                    self.step_device(toks.addr + 4 * (i - 1), self._tok, self._logits)
                ops.sample(self._logits, 1, V, (V + 3) // 4 * 4, params(i), toks.addr + 4 * i)
            self.ctx.sync()
            return toks.download(np.int32)

    def forward(self, token: int, return_logits: bool = False, temperature: float = 0.0,
                top_p: float = 1.0, rng: Optional[np.random.Generator] = None, top_k: int = 0,
                min_p: float = 0.0):
        """InferenceEngine.forward(token:temperature:topP:) (:125-156): the next
        token — greedy on the GPU at temperature <= 0, else sampled on the host
        from the step's logits as the reference does (sampling.sample_token) —
        and the f32 logits when asked.  With top_k or min_p, which the reference
        does not have, the token is drawn on the GPU (m1moe_sample) and only it
        is read back."""
        self._tok.upload(np.array([token, 0, 0, 0], dtype=np.int32))
        self.step_device(self._tok, self._tok, self._logits)
        logits = None
        if temperature > 0 and (top_k > 0 or min_p > 0):
            V = self.shape.vocab
            u = (rng or np.random.default_rng()).random(1, dtype=np.float32)
            params = self._sample_params(self._draw, u, temperature, top_k, top_p, min_p)
            DenseOps(self.ctx).sample(self._logits, 1, V, (V + 3) // 4 * 4, params(0), self._tok)
            self.ctx.sync()
            nxt = int(self._tok.download(np.int32, 1)[0])
            return (nxt, self._logits.download(np.float32, V)) if return_logits else nxt
        self.ctx.sync()
        if temperature > 0:
            logits = self._logits.download(np.float32, self.shape.vocab)
            nxt = sample_token(logits, temperature, top_p, rng=rng)
        else:
            nxt = int(self._tok.download(np.int32, 1)[0])
        if return_logits:
            if logits is None:
                logits = self._logits.download(np.float32, self.shape.vocab)
            return nxt, logits
        return nxt


__all__ = ["rope_frequencies", "AttentionSpec", "DecoderSpec", "DenseOps", "Decoder", "DeviceBuffer",
           "WEIGHT_NAMES", "weight_count"]
