"""wh_attention_tree where numbers are at their ends."""
import numpy as np
import pytest

from tests import _tree
from tests.test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu


def exact(c):
    """The case in 64 bits, with rows of weight 0 left out: (out, bound of the error), [n][t][h][..].  The bound is that
    of _tree.attention over the keys that have a weight."""
    q, k, v = c.views()
    out, bound = np.zeros((c.n, c.t, c.h, c.d)), np.zeros((c.n, c.t, c.h, 1))
    for s in range(c.n):
        kc, vc, g = c.kc[s].copy(), c.vc[s].copy(), c.h // c.kv
        ps = _tree.paths(c.parents[s])
        for i, p in enumerate(ps):
            if p is not None:
                kc[c.lens[s] + i] = _tree.stored(_tree.rotate(k[s, i], c.lens[s] + len(p) - 1, c.inv))
                vc[c.lens[s] + i] = _tree.stored(v[s, i].astype(np.float64))
        for i, p in enumerate(ps):
            if p is None:
                continue
            rows = np.concatenate([np.arange(c.lens[s]), c.lens[s] + np.array(p)]).astype(int)
            qr = _tree.rotate(q[s, i], c.lens[s] + len(p) - 1, c.inv)
            for h in range(c.h):
                kk, vv = kc[rows, h // g].astype(np.float64), vc[rows, h // g].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    sc = kk @ qr[h] / np.sqrt(c.d)
                    if np.isnan(sc).any() or sc.max() == np.inf:
                        out[s, i, h] = np.nan
                        continue
                    some = sc > -np.inf
                    sc, kk, vv = sc[some], kk[some], vv[some]
                    w = np.exp(sc - sc.max())
                    out[s, i, h] = w @ vv / w.sum()
                mag = (np.abs(kk) @ np.abs(qr[h])).max() / np.sqrt(c.d)
                e = mag * (2.0 ** -21 + 2 * c.d * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
                bound[s, i, h] = (2 * e + 300 * 2.0 ** -24) * np.abs(vv).max()
    return out, bound


# 16 heads per KV head: a tile of 32 query rows is two nodes.  Workgroups take the 24 tiles of a KV head by one up to 1920
# rows, by two up to 5120, then by four.
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,ctx", [(300, 40), (300, 252), (5000, 40), (5000, 1000), (60000, 40), (60000, 1000)])
def test_infinite_v_under_rows_that_move_and_rows_that_do_not(gpu, rows, ctx, d):
    """Every second pair of nodes has scores that rise from key to key, so that its rows' maxima move in every tile, the
    others have queries of zero.  Infinities and NaN of the last cache rows and of the nodes, in the first elements, reach
    exactly the rows that see them, call after call."""
    n_tree, heads, kv = 48, 32, 2
    c = Case(1, n_tree, heads, kv, d, [ctx], room=rows - ctx - n_tree, shape="star", seed=rows + ctx)
    c.parents[0, 7] = -1  # roots of their own: they do not see node 0
    c.parents[0, 20:24] = -2
    u = np.zeros(d, np.float32)
    u[: d // 2] = 1
    step = _tree.rotate(u, ctx + 1, c.inv) / np.sqrt(d)
    c.kc[0, :ctx] = (np.linspace(0, 24, ctx)[:, None, None] * step).astype(np.float16)
    q, k, v = c.views()
    for t in range(n_tree):
        q[0, t] = 4 * u if t // 2 % 2 else 0
    c.vc[0, ctx - 1, 0, 0] = np.inf
    c.vc[0, ctx - 2, 1, 1] = np.nan
    v[0, 0, 0, 2] = -np.inf
    v[0, 3, 1, 3] = np.inf
    v[0, 30, 0, 3] = np.nan
    v[0, 47, 1, 0] = np.inf
    print(f"[case] infinite v under moving rows d {d} ctx {ctx} of {rows}", flush=True)
    want, bound, _, _ = c.expect()
    c.upload()
    for _ in range(8):
        c.launch()
        c.compare(f"infinite v d {d} ctx {ctx} of {rows}", c.results()[0], want, bound)


@pytest.mark.parametrize("d,heads,kv", [(64, 8, 2), (128, 8, 2), (128, 32, 2)])
@pytest.mark.parametrize("rows,ctx", [(300, 45), (300, 200), (3000, 700), (9000, 333)])
def test_infinite_keys(gpu, d, heads, kv, rows, ctx):
    """A k of infinity has a score of infinity where q has its sign, and the row is NaN; of -inf where q has the other,
    and the key has weight 0; and NaN where q is 0.  In whole tiles of the cache, in its last rows and in nodes."""
    n_tree = 12
    c = Case(1, n_tree, heads, kv, d, [ctx], room=rows - ctx - n_tree, shape="star", seed=rows + d)
    c.parents[0, 5] = -1  # it does not see node 0
    q, k, v = c.views()
    q[0, 9, 0] = 0
    q[0, 10, 1, 2:] = 2.0 ** -9  # limbs of one bit: the lo limb is 0
    c.kc[0, 3, 0, 5] = np.inf
    c.kc[0, ctx // 2, 0, d - 1] = -np.inf
    c.kc[0, ctx - 1, kv - 1, 9] = -np.inf
    k[0, 0, kv - 1, d // 2:] = 1e6  # beyond f16: stored as infinities where the rotation does not cancel them
    k[0, 0, kv - 1, :d // 2] = 0
    want, bound = exact(c)
    per = np.isnan(want).any(-1)
    assert per.any() and (~per[0]).sum() >= heads, "rows of both kinds"
    c.upload().launch()
    out, gk, _ = c.results()
    assert np.isinf(gk[0, ctx]).any()
    assert np.array_equal(np.isnan(out), np.isnan(want)), "NaN in other places"
    fine = ~np.isnan(want)
    err = np.where(fine, np.abs(np.where(fine, out - want, 0)), 0)
    print(f"[case] infinite keys d {d} {heads}/{kv} ctx {ctx} of {rows}: {err.max():.2e}, {fine.mean():.2f} finite", flush=True)
    assert (err <= bound).all(), float(err.max())
