"""Plain 64-bit forms of the operators that verify a tree of drafted tokens, for their tests."""
from __future__ import annotations

import numpy as np

NO_TOKEN = 0xFFFFFFFF


def paths(parents) -> list:
    """Per node the list of nodes from the cache's end to it, or None where it is absent."""
    out = []
    for t, p in enumerate(int(v) for v in parents):
        if p == -1:
            out.append([t])
        else:
            out.append(out[p] + [t] if 0 <= p < t and out[p] is not None else None)
    return out


def make_parents(rng, n_tree: int, shape: str) -> np.ndarray:
    p = np.full(n_tree, -1, np.int32)
    for t in range(1, n_tree):
        if shape == "chain":
            p[t] = t - 1
        elif shape == "star":
            p[t] = 0
        elif shape == "forest":
            p[t] = int(rng.integers(-1, t))
        else:
            p[t] = int(rng.integers(max(0, t // 2 - 1), t))
    if shape == "padded":  # the last nodes, and one in the middle with all below it, are absent
        p[max(1, n_tree - n_tree // 3):] = -2
        if n_tree > 4:
            p[n_tree // 3] = n_tree + 5
    if shape == "absent":
        p[0] = -7
    return p


def rotate(x, pos, inv_freq):
    """x [..][d] rotated by pos * inv_freq in 64 bits: pairs (i, i + d / 2)."""
    a = np.float64(pos) * inv_freq.astype(np.float64)
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h].astype(np.float64), x[..., h:].astype(np.float64)
    return np.concatenate([x1 * np.cos(a) - x2 * np.sin(a), x1 * np.sin(a) + x2 * np.cos(a)], -1)


def stored(x) -> np.ndarray:
    """The f16 that the cache holds of a 64-bit value: rounded to f32, then to f16."""
    with np.errstate(over="ignore", invalid="ignore"):
        return x.astype(np.float32).astype(np.float16)


def attention(q, k, v, parents, ctx, k_cache, v_cache, inv_freq):
    """One sequence: q [t][h][d], k and v [t][kv][d] f32; caches [max_ctx][kv][d] f16, updated in place.  Returns
    out [t][h][d] in f64 and the bound of the kernel's error, per row and head.

    The bound: a score is a sum of d products of f32 accuracy.  Rotating q rounds three times and the f16 limbs hold
    2^-22 of an element: under 2^-21 together.  2 d additions in f32 add at most 2 d 2^-24 of the sum of magnitudes, S;
    the scale and the exponent's argument 2^-22 of |s| <= S, the exponential itself and P's limbs under 2^-20.  A
    relative error e of every weight moves the output by at most 2 e max|v|; the weights' sums in f32 (in tiles of 32,
    chunks and splits: under 300 terms in a row) add 300 * 2^-24 max|v|.
    """
    t, h, d = q.shape
    kv = k.shape[1]
    g = h // kv
    ps = paths(parents)
    if ctx + t > k_cache.shape[0]:
        return np.full((t, h, d), np.nan), np.zeros((t, h))
    qr = np.zeros((t, h, d))
    for i, p in enumerate(ps):
        if p is None:
            continue
        pos = ctx + len(p) - 1
        qr[i] = rotate(q[i], pos, inv_freq)
        k_cache[ctx + i] = stored(rotate(k[i], pos, inv_freq))
        v_cache[ctx + i] = stored(v[i].astype(np.float64))
    out, bound = np.zeros((t, h, d)), np.zeros((t, h))
    for i, p in enumerate(ps):
        if p is None:
            continue
        rows = np.concatenate([np.arange(ctx), ctx + np.array(p)]).astype(int)
        for head in range(h):
            kk = k_cache[rows, head // g].astype(np.float64)
            vv = v_cache[rows, head // g].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = kk @ qr[i, head] / np.sqrt(d)
                w = np.exp(s - s.max())
                out[i, head] = (w[:, None] * vv).sum(0) / w.sum()
                mag = (np.abs(kk) @ np.abs(qr[i, head])).max() / np.sqrt(d)
                e = mag * (2.0 ** -21 + 2 * d * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
                # rows with an infinite or NaN score are NaN: they have no error
                vmax = np.abs(np.where(np.isfinite(vv), vv, 0)).max()
                bound[i, head] = (2 * e + 300 * 2.0 ** -24) * vmax if np.isfinite(e) else 0
    return out, bound


def logits(x, vocab, rep, freq, pres, counts, bias, allowed, dtype):
    """One row in `dtype`, each operation rounded by itself: the processed logits and the token."""
    f = dtype
    l = x[:vocab].astype(f).copy()
    with np.errstate(invalid="ignore", over="ignore"):
        hit = counts > 0
        l[hit] = np.where(l[hit] > 0, l[hit] / f(rep), l[hit] * f(rep))
        l[hit] = l[hit] - (counts[hit].astype(f) * f(freq) + f(pres))
        for i, b in bias.items():
            l[i] = l[i] + f(b)
    if allowed is not None:
        l[~allowed] = -np.inf
    ok = l > -np.inf  # false for NaN
    token = int(np.flatnonzero(l == l[ok].max())[0]) if ok.any() else NO_TOKEN
    return l, token


def accept(tokens, parents, picked):
    """(path, next token) of one sequence."""
    ps = paths(parents)
    path, nxt = [], NO_TOKEN
    at = 0 if ps[0] is not None else None
    while at is not None:
        path.append(at)
        nxt = int(picked[at])
        at = None if nxt == NO_TOKEN else next(
            (c for c in range(at + 1, len(ps)) if parents[c] == at and int(tokens[c]) == nxt), None)
    return path, nxt
