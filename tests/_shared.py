"""Inputs and bars for the precision of wh_attention_shared, and a numpy form of how its kernel holds q and the weights."""
from __future__ import annotations

import numpy as np


def bar(top):
    """Relative L2 of a member's rows, with `top` the largest |score|: that of an attention in f32.

    The keys' v are independent, so errors of the weights, each relative to its weight, move the output by no more than
    their size.  A score is a sum in f32 of magnitude <= top in 2 d / 16 steps of 16 products, each off by 2^-24 of it, of
    random signs (under 4 * 2^-24 top), of limbs that hold q to 2^-22 (2^-22 top).  The exponent's argument, in powers of
    two, and the exponential add 1.45 * 2^-24 * 2 top + 2^-22; the limbs of the weights 2^-22; the sums of weights and
    products, and their joins, 300 additions of random signs, 2^-20."""
    return 2.0 ** -22 * (4 * top + 16)


def add_sink(q, k, v, share, at):
    """Makes row `at` of k the key that has `share` of the weight of a query q (one head, [d]) among the rows of k [n][d],
    with a v of 0."""
    q, n = q.astype(np.float64), k.shape[0]
    if share == 0 or n < 2:
        return
    s = np.delete(k, at, 0).astype(np.float64) @ q / np.sqrt(len(q))
    goal = s.max() + np.log(np.exp(s - s.max()).sum()) + np.log(share) - np.log1p(-share)
    k[at] = q * (goal * np.sqrt(len(q)) / (q @ q))
    v[at] = 0


def exact(q, k, v):
    """q [h][d], k and v [n][kv][d]: (out [h][d] in 64 bits, the largest |score|)."""
    h, kv = len(q), k.shape[1]
    out, top = np.zeros(q.shape), 0.0
    for j in range(kv):
        rows = slice(j * (h // kv), (j + 1) * (h // kv))
        s = q[rows].astype(np.float64) @ k[:, j].astype(np.float64).T / np.sqrt(q.shape[1])
        w = np.exp(s - s.max(1, keepdims=True))
        out[rows] = w @ v[:, j].astype(np.float64) / w.sum(1, keepdims=True)
        top = max(top, float(np.abs(s).max()))
    return out, top


def rel(got, want):
    return float(np.linalg.norm(got - want) / np.linalg.norm(want))


def _split(x, scale):
    hi = x.astype(np.float16).astype(np.float32)
    return hi, ((x - hi) * np.float32(scale)).astype(np.float16).astype(np.float64) / scale


def emulate(q, k, v, tile=32, q_limbs=2, p_limbs=2, falls=True):
    """One query row over one chunk: q and the weights in f16 limbs, all else in 64 bits.  falls: the reference follows the
    tiles down to where they are faint, and tiles with one of the highest keys beside a faint half take two turns."""
    x = np.ldexp(q, 13 - int(np.floor(np.log2(np.abs(q).max())))).astype(np.float32)
    hi, lo = _split(x, 1.0)
    s = k.astype(np.float64) @ (hi + (lo if q_limbs == 2 else 0)) * (np.abs(q).max() / np.abs(x).max()) / np.sqrt(len(q)) / np.log(2)
    m = peak = -np.inf
    l, acc = 0.0, np.zeros(v.shape[1])
    for b in range(0, len(s), tile):
        t, vt, half = s[b:b + tile], v[b:b + tile].astype(np.float64), np.arange(b, min(b + tile, len(s))) % 8 // 4
        if t.max() - m > 3:
            l, acc, m = l * 2.0 ** (m - t.max()), acc * 2.0 ** (m - t.max()), t.max()
        peak = max(peak, m)
        low = min(t[half == g].max() for g in set(half))
        counts = lambda x, ref: falls and peak - 78 <= x < ref - 30
        near = t >= t.max() - 9
        for keep in [near, ~near] if t.max() >= peak - 10 and counts(low, t.max()) else [near | True]:
            if not keep.any():
                continue
            to = max(t[keep].max(), peak - 48)
            if counts(t[keep].max(), m):
                l, acc, m = l * 2.0 ** (m - to), acc * 2.0 ** (m - to), to
            p = np.exp2(t[keep] - m + 12).astype(np.float32)
            hi, lo = _split(p, 2048.0)
            l += p.astype(np.float64).sum()
            acc = acc + (hi + (lo if p_limbs == 2 else 0)) @ vt[keep]
    return acc / l
