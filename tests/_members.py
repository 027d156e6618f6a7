"""Plain 64-bit forms of the operators that run several continuations of one prompt, for their tests."""
from __future__ import annotations

import numpy as np

NO_TOKEN = 0xFFFFFFFF


def stored(x) -> np.ndarray:
    """The f16 that the cache holds of a 64-bit value: rounded to f32, then to f16."""
    with np.errstate(over="ignore", invalid="ignore"):
        return x.astype(np.float32).astype(np.float16)


def rope(x, pos, inv_freq, rot_dim, interleaved, magnitude=1.0, weight=None, eps=0.0):
    """Rows x [n][heads][d] at positions pos [n], normed and turned, and the bound of an f32 form's error.

    The bound: a norm's sum is added in at most 10 steps (2^-24 each, halved by the root), with the root, the quotient and
    two products under 10 * 2^-24 together; the turn rounds the sine or cosine, each product and their sum: 3 * 2^-24 of
    the pair.  The angle in 64 bits is off by 2^-50 of itself at most, here and there."""
    d = x.shape[-1]
    x = x.astype(np.float64)
    unit = 3 * 2.0 ** -24
    if weight is not None:
        x = x / np.sqrt((x * x).sum(-1, keepdims=True) / d + eps) * weight.astype(np.float64)
        unit += 10 * 2.0 ** -24
    angle = pos.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
    cos, sin = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    out, bound = x.copy(), np.abs(x) * unit
    i = np.arange(0, rot_dim, 2) if interleaved else np.arange(rot_dim // 2)
    j = i + (1 if interleaved else rot_dim // 2)
    out[..., i] = x[..., i] * cos - x[..., j] * sin
    out[..., j] = x[..., i] * sin + x[..., j] * cos
    pair = (np.abs(x[..., i]) + np.abs(x[..., j])) * abs(magnitude)
    bound[..., i] = bound[..., j] = pair * (unit + np.abs(angle) * 2.0 ** -50)
    return out, bound


def attention(q, k, v):
    """One member: q [h][d] f32, k and v [n][kv][d] f16 (the rows it sees).  out [h][d] in f64 and the bound of the
    kernel's error.

    The bound: q's limbs hold 2^-22 of an element; 2 d additions of the score in f32 add at most 2 d 2^-24 of the sum of
    magnitudes, S; the scale and the exponent's argument 2^-22 of |s| <= S, the exponential itself and the weight's limbs
    under 2^-20: e in all.  A weight far below the largest is off by 2^-50 of that one instead.  The sums of the weights
    and of V round at most 10 times in each of a wave's tiles (n / 128) and under 300 times where they are joined."""
    n, kv, d = k.shape
    h = q.shape[0]
    out, bound = np.zeros((h, d)), np.zeros((h, d))
    if n == 0:
        return out, bound
    for head in range(h):
        kk, vv = k[:, head // (h // kv)].astype(np.float64), v[:, head // (h // kv)].astype(np.float64)
        qq = q[head].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            s = kk @ qq / np.sqrt(d)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[head] = (w[:, None] * vv).sum(0)
            mag = (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(d)
            e = mag * (2.0 ** -21 + 2 * d * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
            va = np.abs(np.where(np.isfinite(vv), vv, 0))
            b = (2 * e + (300 + n / 8) * 2.0 ** -24) * (w[:, None] * va).sum(0) + n * 2.0 ** -50 * va.max(0) + 2.0 ** -126
            bound[head] = np.where(np.isfinite(b), b, 0)
    return out, bound


def select(logits, scores, vocab, n_out, last=None, end=NO_TOKEN, alpha=0.0, counts=None):
    """One sequence: logits [beams][..], scores [beams].  A list of (score, token, parent, count), best first; the rest
    (-inf, no token, its own place, 0)."""
    b = len(scores)
    found = []
    for j in range(b):
        score, count = np.float64(scores[j]), 0 if counts is None else int(counts[j])
        if not np.isfinite(score):
            continue
        if last is not None and int(last[j]) == end:
            found.append((-score / np.float64(max(count, 1)) ** alpha, j, 0.0, end, score, count))
            continue
        row = logits[j, :vocab].astype(np.float64)
        row = np.where(np.isnan(row), -np.inf, row)
        if row.max() in (-np.inf, np.inf):
            continue
        lse = row.max() + np.log(np.exp(row - row.max()).sum())
        for t in np.argsort(-row, kind="stable")[:n_out]:
            if row[t] > -np.inf:
                s = score + (row[t] - lse)
                found.append((-s / np.float64(count + 1) ** alpha, j, -row[t], int(t), s, count + 1))
    found.sort(key=lambda f: f[:4])
    out = [(s, t, j, c) for _, j, _, t, s, c in found[:n_out]]
    return out + [(-np.inf, NO_TOKEN, min(i, b - 1), 0) for i in range(len(out), n_out)]


def select_all(logits, scores, n_out, last=None, end=NO_TOKEN, alpha=0.0, counts=None, vocab=None):
    """Sequences: logits [n][beams][..], scores [n][beams]; arrays [n][n_out]."""
    vocab = vocab or logits.shape[-1]
    rows = [select(logits[i], scores[i], vocab, n_out, None if last is None else last[i], end, alpha,
                   None if counts is None else counts[i]) for i in range(len(scores))]
    cols = [np.array([[c[k] for c in r] for r in rows]) for k in range(4)]
    return cols[0].astype(np.float64), cols[1].astype(np.int64), cols[2].astype(np.int64), cols[3].astype(np.int64)


def histories(history, len, parents, tokens):
    """[n][beams][stride] after a choice."""
    new = history.copy()
    n, b, stride = history.shape
    for s in range(n):
        for i in range(b):
            l = int(len[s, parents[s, i]])
            new[s, i, :min(l, stride)] = history[s, parents[s, i], :min(l, stride)]
            if l < stride:
                new[s, i, l] = tokens[s, i]
    return new


def reorder(state, parents, len, pending):
    """[n][beams][max_rows][..] after the beams have followed their parents."""
    new = state.copy()
    n, b, room = state.shape[:3]
    for s in range(n):
        for i in range(b):
            rows, p = max(0, int(len[s, i]) - pending), int(parents[s, i])
            if p < b and rows <= room:
                new[s, i, :rows] = state[s, p, :rows]
    return new
