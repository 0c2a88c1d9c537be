"""Batches, f64 references and buffers for the tests of the paged KV cache and
the sampler."""
from __future__ import annotations

import math

import numpy as np

from m1moe_amd import synth


def bf16(a):
    return synth.f32_to_bf16(np.asarray(a, np.float32))


def f64(a):
    """f32 or bf16 bits -> f64."""
    return (synth.bf16_to_f32(a) if a.dtype == np.uint16 else a).astype(np.float64)


def as_dtype(a, dtype):
    return bf16(a) if dtype == "bf16" else np.asarray(a, np.float32)


class Batch:
    """rows[s] new rows of sequence s behind past[s] positions (prefix
    included), pages dealt out in a random order."""

    def __init__(self, rng, rows, past, page, prefix=0, spare=3, pad=0, pages=None):
        self.rows, self.page, self.prefix, self.pad = list(rows), page, prefix, pad
        self.kv_len = np.array([r + p for r, p in zip(rows, past)], np.int32)
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.B, self.T = len(rows), int(self.row_start[-1])
        self.num_rows = self.T + pad
        need = [-(-int(n) // page) for n in self.kv_len]
        first = -(-prefix // page)
        total = sum(need) + first + spare if pages is None else pages
        order = rng.permutation(total)[:sum(need) + first] if total < 1 << 16 else \
            rng.choice(total, sum(need) + first, replace=False)
        self.num_pages = total
        self.stride = max(need + [first, 1])
        self.table = np.zeros((self.B, self.stride), np.int32)
        self.prefix_table = order[:first].astype(np.int32)
        at = first
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n

    def places(self):
        """(sequence, position) of every row."""
        return [(s, int(self.kv_len[s]) - n + i) for s, n in enumerate(self.rows) for i in range(n)]

    def cell(self, s, pos):
        """(page, slot) of the positions pos of sequence s."""
        pos = np.asarray(pos)
        pg = self.table[s][pos // self.page].copy()
        inside = pos < self.prefix
        if self.prefix:
            pg[inside] = self.prefix_table[pos[inside] // self.page]
        return pg, pos % self.page


def attention_ref(b: Batch, q, kc, vc, heads, kv_heads, hd):
    """f64 output rows, sum_p w_p |v_p| and the largest sum_d |q k| / sqrt(hd) of
    each (row, head)."""
    share = heads // kv_heads
    q64 = f64(q).reshape(-1, heads, hd)
    out = np.zeros((b.T, heads, hd))
    mag = np.zeros((b.T, heads, hd))
    top = np.zeros((b.T, heads, 1))
    for s, n in enumerate(b.rows):
        if n == 0:
            continue
        L = int(b.kv_len[s])
        pg, sl = b.cell(s, np.arange(L))
        K, V = f64(kc[pg, sl]), f64(vc[pg, sl])           # [L, kv_heads, hd]
        r0 = int(b.row_start[s])
        for i in range(n):
            P = L - n + i + 1
            for g in range(kv_heads):
                qq = q64[r0 + i, g * share:(g + 1) * share]
                with np.errstate(all="ignore"):
                    e = qq @ K[:P, g].T / math.sqrt(hd)
                    top[r0 + i, g * share:(g + 1) * share, 0] = \
                        (np.abs(qq) @ np.abs(K[:P, g]).T / math.sqrt(hd)).max(1)
                    e = np.exp(e - e.max(1, keepdims=True))
                    e /= e.sum(1, keepdims=True)
                    out[r0 + i, g * share:(g + 1) * share] = e @ V[:P, g]
                    mag[r0 + i, g * share:(g + 1) * share] = e @ np.abs(V[:P, g])
    return out, mag, top


def attention_bound(out, mag, top, hd, dtype):
    """Elementwise: a score is a sum of hd products in f32, off by at most (hd + 8)
    2^-24 of the sum of their sizes, which moves a weight and the weights' sum by as
    much each; exp2, its argument and the sums of weights and of weighted values add
    (L-independent, since sums run in blocks) 64 roundings of 2^-24.  bf16: the
    weights that multiply v are rounded (2^-8) and the output is (2^-8)."""
    bound = mag * (2 * (hd + 8) * 2.0 ** -24 * top + 64 * 2.0 ** -24)
    if dtype == "bf16":
        bound = bound + 2.0 ** -8 * mag + 2.0 ** -8 * np.abs(out)
    return bound + 1e-30


def append_ref(b: Batch, x, heads, hd, w, eps, rotary, inter, freq, amp):
    """f64 rows [T, heads, hd] normed and rotated, and the sizes |a| + |b| they are
    made of."""
    y = f64(x).reshape(-1, heads, hd)[:b.T]
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * f64(w)
    z, size = y.copy(), np.abs(y)
    h = rotary // 2
    if h:
        pos = np.array([p for _, p in b.places()], np.float64)
        ang = pos[:, None] * freq.astype(np.float64)[None]
        c, s = (np.cos(ang) * amp)[:, None], (np.sin(ang) * amp)[:, None]
        i0, i1 = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if inter else (slice(0, h), slice(h, 2 * h))
        A, B = y[..., i0], y[..., i1]
        z[..., i0], z[..., i1] = A * c - B * s, A * s + B * c
        size[..., i0] = size[..., i1] = (np.abs(A) + np.abs(B)) * abs(amp)
    return z, size


def sample_ref(x, u, T=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row in f64; the settings as f32 values."""
    T, top_p, min_p, u = (float(np.float32(v)) for v in (T, top_p, min_p, u))
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    order = np.argsort(-x, kind="stable")
    if x[order[0]] == -np.inf:
        return -1, 0.0
    if not T > 0:
        return int(order[0]), 1.0
    if top_k > 0:
        order = order[:top_k]
    xs = x[order]
    with np.errstate(invalid="ignore"):
        w = np.where(xs == xs[0], 1.0, np.exp((xs - xs[0]) / T))
    w[w < 2.0 ** -45] = 0.0
    cum = np.cumsum(w)
    keep = int(np.count_nonzero(w))
    if top_p < 1:
        keep = min(keep, int(np.searchsorted(cum, max(top_p, 0.0) * cum[-1])) + 1)
    if min_p > 0:
        keep = min(keep, max(1, int(np.count_nonzero(w >= min_p))))
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    i = min(int(np.searchsorted(cum[:keep], u * cum[keep - 1])), keep - 1)
    return int(order[i]), float(w[i] / cum[keep - 1])
