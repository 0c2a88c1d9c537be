"""Trees, f64 references and bounds for the tests of the drafted tokens' operators and of the
products with 4-bit weights."""
from __future__ import annotations

import math

import numpy as np

from serving_cases import Batch, f64


def tree_parents(rng, n, chain=0.4):
    """Every row's parent in one tree of n rows, -1 for row 0."""
    return [-1] + [i - 1 if rng.random() < chain else int(rng.integers(0, i)) for i in range(1, n)]


def ancestors(parents):
    """Of every row the rows it sees."""
    sees = []
    for i, p in enumerate(parents):
        sees.append((sees[p] if 0 <= p < i else []) + [i])
    return sees


def plan_ref(parents, words):
    """(uint64 [n][words], depths) of one tree."""
    n = len(parents)
    mask, depth = np.zeros((n, words), np.uint64), np.zeros(n, np.int32)
    for i, a in enumerate(ancestors(parents)):
        for j in a:
            mask[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
        depth[i] = len(a) - 1
    return mask, depth


def sees(mask, i, j):
    return bool(int(mask[i, j // 64]) >> (j % 64) & 1)


def tree_attention_ref(b: Batch, mask, q, kc, vc, heads, kv_heads, hd):
    """f64 output rows, sum_p w_p |v_p| and the largest sum_d |q k| / sqrt(hd) of each (row, head),
    over the positions before the tree and the rows j <= i that mask[row] names; zeros for a row
    that sees nothing."""
    share = heads // kv_heads
    q64 = f64(q).reshape(-1, heads, hd)
    out, mag, top = np.zeros((b.T, heads, hd)), np.zeros((b.T, heads, hd)), np.zeros((b.T, heads, 1))
    for s, n in enumerate(b.rows):
        if n == 0:
            continue
        L, r0 = int(b.kv_len[s]), int(b.row_start[s])
        base = L - n
        pg, sl = b.cell(s, np.arange(L))
        K, V = f64(kc[pg, sl]), f64(vc[pg, sl])
        for i in range(n):
            at = np.array(list(range(base)) + [base + j for j in range(i + 1) if sees(mask, r0 + i, j)], int)
            if len(at) == 0:
                continue
            for g in range(kv_heads):
                h = slice(g * share, (g + 1) * share)
                with np.errstate(all="ignore"):
                    e = q64[r0 + i, h] @ K[at, g].T / math.sqrt(hd)
                    top[r0 + i, h, 0] = (np.abs(q64[r0 + i, h]) @ np.abs(K[at, g]).T / math.sqrt(hd)).max(1)
                    e = np.exp(e - e.max(1, keepdims=True))
                    e /= e.sum(1, keepdims=True)
                    out[r0 + i, h] = e @ V[at, g]
                    mag[r0 + i, h] = e @ np.abs(V[at, g])
    return out, mag, top


def accept_ref(parents, drafts, drawn):
    """The path of one tree."""
    way = [0]
    while True:
        on = [i for i, p in enumerate(parents) if p == way[-1] and p < i and drafts[i] == drawn[p]]
        if not on:
            return way
        way.append(on[0])


def q4_weights(rng, rows, cols, group, sigma=0.02):
    """(words, scales, biases): any nibbles, scales and biases in bf16 bits."""
    from serving_cases import bf16
    w = rng.integers(0, 1 << 32, (rows, cols // 8), dtype=np.uint64).astype(np.uint32)
    lo = -2.5 * sigma * (1 + 0.15 * rng.normal(0, 1, (rows, cols // group)))
    step = 5 * sigma / 15 * (1 + 0.15 * rng.normal(0, 1, (rows, cols // group)))
    return w, bf16(step), bf16(lo)


def q4_dense(w, scales, biases, group):
    """f64 [rows][cols], and the sizes (nibble |scale|, |bias|) it is the sum of."""
    n = (w[:, :, None] >> np.arange(0, 32, 4, dtype=np.uint32) & 15).reshape(w.shape[0], -1).astype(np.float64)
    s, b = (np.repeat(f64(t), group, 1) for t in (scales, biases))
    return n * s + b, n * np.abs(s) + np.abs(b)


def q4_bound(x, size, y, group, dtype):
    """Elementwise.  An f32 x is taken to 22 bits (2^-22 with both roundings); a group's sum of at
    most 2 group products, cut rather than rounded where a matrix instruction adds them, is off by
    (2 group + 2) 2^-23 of the sum of their sizes, and so is the group's sum of x that the bias
    multiplies; groups, the residual and what a power of two scales come on top with one rounding
    each.  f16 parts of x end at steps of 2^-24 where the row's largest is 2^14 at least: half a
    step is 2^-39 of that one.
    bf16: the result's own rounding."""
    mag = np.abs(x) @ size.T
    groups = size.shape[1] // group
    bound = mag * (2.0 ** -22 + (2 * group + groups + 8) * 2.0 ** -23)
    bound += np.abs(x).max(1, keepdims=True) * 2.0 ** -39 * size.sum(1)[None] + np.abs(y) * 2.0 ** -22
    if dtype == "bf16":
        bound = bound + 2.0 ** -8 * np.abs(y)
    return bound + 1e-37
