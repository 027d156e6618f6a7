"""wh_attention_tree where numbers are at their ends."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, up
from tests.test_gpu_tree_attention import Case
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu


def exact(c, seqs=None):
    """The case in 64 bits, with rows of weight 0 left out: (out, bound of the error), [n][t][h][..], of all sequences or
    those given.  The bound is that of _tree.attention over the keys that have a weight."""
    q, k, v = c.views()
    out, bound = np.zeros((c.n, c.t, c.h, c.d)), np.zeros((c.n, c.t, c.h, 1))
    c.top = 0.0  # the largest |score|
    for s in range(c.n) if seqs is None else seqs:
        kc, vc, g, ctx = c.kc[s].copy(), c.vc[s].copy(), c.h // c.kv, c.lens[s]
        ps = _tree.paths(c.parents[s])
        there = [t for t, p in enumerate(ps) if p is not None]
        if not there:
            continue
        for t in there:
            kc[ctx + t] = _tree.stored(_tree.rotate(k[s, t], ctx + len(ps[t]) - 1, c.inv))
            vc[ctx + t] = _tree.stored(v[s, t].astype(np.float64))
        rows = ctx + there[-1] + 1
        for h in range(c.h):
            kk, vv = kc[:rows, h // g].astype(np.float64), vc[:rows, h // g].astype(np.float64)
            qr = np.stack([_tree.rotate(q[s, t, h], ctx + len(ps[t]) - 1, c.inv) for t in there])
            with np.errstate(invalid="ignore"):
                sc = qr @ kk.T / np.sqrt(c.d)
                mag = np.abs(qr) @ np.abs(kk).T / np.sqrt(c.d)
            for i, t in enumerate(there):
                see = np.concatenate([np.arange(ctx), ctx + np.array(ps[t])]).astype(int)
                x = sc[i, see]
                if np.isnan(x).any() or x.max() == np.inf:
                    out[s, t, h] = np.nan
                    continue
                some = x > -np.inf
                x, vals = x[some], vv[see][some]
                w = np.exp(x - x.max())
                out[s, t, h] = w @ vals / w.sum()
                c.top = max(c.top, float(np.abs(x).max()))
                e = mag[i, see][some].max() * (2.0 ** -21 + 2 * c.d * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20
                bound[s, t, h] = (2 * e + 300 * 2.0 ** -24) * np.abs(vals).max()
    return (out, bound) if seqs is None else (out[seqs], bound[seqs])


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
# 12 nodes of 32 heads on 2 KV heads: tiles by one, one, two and four to a workgroup, tiles of 32 keys and two at a time
@pytest.mark.parametrize("rows,ctx", [(300, 45), (300, 200), (3000, 700), (9000, 333), (60000, 333), (60000, 5000)])
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


def weights_case(n_tree, heads, kv, d, ctx, room, share, sink, seed=0, spread=1.0):
    """One sequence without rotation (inv_freq 0) in which every query row of a KV head is the same, so that one key holds
    `share` of every row's weight, with a v of 0; sink: its cache row, or -1 for node 0, which all nodes see."""
    c = Case(1, n_tree, heads, kv, d, [ctx], room=room, shape="star", seed=seed)
    c.inv[:] = 0
    q, k, v = c.views()
    u = (c.rng.standard_normal((kv, d)) * spread).astype(np.float32)
    q[0] = np.repeat(u, heads // kv, 0)
    k[0, 1:] *= 0.5
    for h in range(kv):
        keys = c.kc[0, :ctx, h].astype(np.float64) if sink < 0 else np.delete(c.kc[0, :ctx, h], sink, 0).astype(np.float64)
        rest = np.exp(keys @ u[h].astype(np.float64) / np.sqrt(d)).sum()
        if share:
            key = u[h] * (np.log(rest * share / (1 - share)) * np.sqrt(d) / float((u[h].astype(np.float64) ** 2).sum()))
            (k[0, 0] if sink < 0 else c.kc[0, sink])[h] = key
            (v[0, 0] if sink < 0 else c.vc[0, sink])[h] = 0
    return c


def weights_exact(c, nodes):
    """(out [node][kv][d] in 64 bits, largest |score|) of a weights_case; the query heads of a KV head are alike."""
    q, k, v = c.views()
    g, ctx, top = c.h // c.kv, c.lens[0], 0.0
    out = np.zeros((len(nodes), c.kv, c.d))
    for h in range(c.kv):
        kk, vv = c.kc[0, :ctx, h].astype(np.float64), c.vc[0, :ctx, h].astype(np.float64)
        u = q[0, 0, h * g].astype(np.float64) / np.sqrt(c.d)
        s = kk @ u
        for i, t in enumerate(nodes):
            path = _tree.paths(c.parents[0])[t]
            own = _tree.stored(k[0, path, h].astype(np.float64)).astype(np.float64) @ u
            w = np.exp(np.concatenate([s, own]) - max(s.max(initial=-np.inf), own.max()))
            vals = np.concatenate([vv, v[0, path, h].astype(np.float16).astype(np.float64)])
            out[i, h] = w @ vals / w.sum()
            top = max(top, float(np.abs(s).max(initial=0)), float(np.abs(own).max()))
    return out, top


def weights_bar(top):
    """Relative L2: the keys' v are independent, so errors of the weights, each relative to its weight, move the output by
    no more than their size.  A score is a sum in f32 of magnitude <= top in steps of 16 products (2 d / 16 of them, each
    off by 2^-24 of it, of random signs: under 4 * 2^-24 top), of limbs that hold q to 2^-22 (2^-22 top); the exponent's
    argument, in powers of two, and the exponential add 1.45 * 2^-24 * 2 top + 2^-22; the limbs of the weights 2^-20; the sums of weights
    and products 300 additions of random signs, 2^-20 again."""
    return 2.0 ** -22 * (4 * top + 16)


# query rows in tiles of a workgroup: one (20 rows), two, four; a chunk of thousands of keys (32 groups of 128 rows)
@pytest.mark.parametrize("share", [0, 0.9, 0.99, 0.999, 0.9999, 0.999999])
@pytest.mark.parametrize("n_tree,heads,kv,d,ctx,room", [(1, 8, 2, 64, 4000, 50), (1, 8, 2, 128, 500, 0), (5, 8, 2, 128, 300, 20),
                                                        (5, 8, 2, 64, 130000, 20), (26, 32, 8, 128, 4070, 7),
                                                        (64, 8, 1, 128, 20000, 5000), (128, 32, 1, 64, 60000, 0),
                                                        (128, 32, 1, 128, 40000, 0)])
def test_one_key_with_nearly_all_the_weight(gpu, n_tree, heads, kv, d, ctx, room, share):
    """The others carry the output, and keep the precision that f32 weights have."""
    nodes = sorted({0, n_tree // 2, n_tree - 1})
    for sink in (0, ctx // 2 + 3, ctx - 1, -1)[:4 if share else 1]:
        c = weights_case(n_tree, heads, kv, d, ctx, room, share, sink, seed=ctx)
        want, top = weights_exact(c, nodes)
        c.upload().launch()
        got = c.results()[0][0, nodes].reshape(len(nodes), kv, heads // kv, d).astype(np.float64)
        rel = float(np.linalg.norm(got - want[:, :, None]) / np.linalg.norm(np.broadcast_to(want[:, :, None], got.shape)))
        bar = weights_bar(top)
        print(f"[result] {share} of the weight on key {sink}, {n_tree} nodes {heads}/{kv}x{d} at {ctx}: {rel:.2e}, bar {bar:.2e}",
              flush=True)
        assert rel <= bar
        if n_tree == 1:
            qkv = up(np.concatenate([c.q, c.k, c.v], 1))[0]
            k0, v0, out = up(c.kc.view(np.uint16))[0], up(c.vc.view(np.uint16))[0], DeviceBuffer(4 * heads * d)
            wsz = ops.attention_workspace_bytes(heads, kv, d, ctx + 1)
            ops.attention_decode(qkv, k0, v0, ctx, heads, kv, d, c.dev["inv"], out, DeviceBuffer(wsz), wsz)
            one = down(out, np.float32, heads * d).reshape(1, kv, -1, d)
            rel = float(np.linalg.norm(one - want[:, :, None]) / np.linalg.norm(np.broadcast_to(want[:, :, None], one.shape)))
            print(f"[result] the decode step: {rel:.2e}", flush=True)
            assert rel <= bar


@pytest.mark.parametrize("spread", [3.0, 8.0])
@pytest.mark.parametrize("n_tree,heads,kv,d,ctx", [(5, 8, 2, 128, 3000), (64, 8, 1, 64, 20000), (128, 32, 1, 128, 9000)])
def test_scores_far_apart(gpu, n_tree, heads, kv, d, ctx, spread):
    """Scores whose standard deviation is 3 and 8: tiles with weights of every size, references that move up and down."""
    c = weights_case(n_tree, heads, kv, d, ctx, 20, 0, 0, seed=7, spread=spread)
    nodes = [0, n_tree - 1]
    want, top = weights_exact(c, nodes)
    c.upload().launch()
    got = c.results()[0][0, nodes].reshape(2, kv, heads // kv, d)
    err, size = np.linalg.norm(got - want[:, :, None]), np.linalg.norm(np.broadcast_to(want[:, :, None], got.shape))
    print(f"[result] scores of spread {spread}: {err / size:.2e}, bar {weights_bar(top):.2e}", flush=True)
    assert err <= weights_bar(top) * size


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n_tree,there", [(2, 1), (8, 5), (33, 32), (64, 63), (65, 64), (100, 40), (128, 65), (128, 127), (128, 1)])
def test_a_tree_that_just_fits(gpu, n_tree, there, d):
    """Absent nodes behind a tree's last one need no room in the cache.  Five sequences: one with room, one
    whose tree ends at the last row, one a row too long, one whose last node hangs below an absent one and takes a row all
    the same, one without a tree on a full cache."""
    c = Case(5, n_tree, 4, 2, d, [40] * 5, room=there - n_tree, shape="tree", seed=n_tree + there)
    rows = c.max_ctx
    assert rows == 40 + there
    c.parents[:, there:] = -2
    c.lens = [5, 40, 41, 40, rows]
    c.parents[3, there] = there + 3   # absent
    if there + 1 < n_tree:
        c.parents[3, there + 1] = there
    c.parents[4] = -2
    orphan = there + 1 < n_tree       # row there + 1 is one too many
    kc, vc = c.kc.copy(), c.vc.copy()
    q, k, v = c.views()
    want, bound = exact(c, [0, 1])
    print(f"[case] {there} of {n_tree} nodes at the cache's end, d {d}", flush=True)
    c.upload().launch()
    out, gk, gv = c.results()
    assert (np.abs(out[:2] - want) <= bound).all(), float(np.abs(out[:2] - want).max())
    assert not out[:2, there:].any(), "absent nodes' rows"
    assert np.isnan(out[2]).all()
    assert np.isnan(out[3]).all() == orphan
    assert not out[4].any()
    for s in (0, 1):
        for i, p in enumerate(_tree.paths(c.parents[s])):
            if p is not None:
                kc[s, c.lens[s] + i] = _tree.stored(_tree.rotate(k[s, i], c.lens[s] + len(p) - 1, c.inv))
                vc[s, c.lens[s] + i] = _tree.stored(v[s, i].astype(np.float64))
    keep = [0, 1, 2, 4] + ([3] if orphan else [])
    assert np.array_equal(gk[keep].view(np.uint16), kc[keep].view(np.uint16))
    assert np.array_equal(gv[keep].view(np.uint16), vc[keep].view(np.uint16))


@pytest.mark.parametrize("n,n_tree", [(1, 1), (3, 17), (70, 5), (300, 2), (1024, 1), (37, 128), (257, 33)])
def test_rows_of_many_trees(gpu, n, n_tree):
    """Trees of every length in one batch, among them none at all, on caches that the shortest of them just fit."""
    r = np.random.default_rng(n)
    there = r.integers(0, n_tree + 1, n)
    there[0] = n_tree
    c = Case(n, n_tree, 2, 1, 64, [20] * n, room=0, seed=n)
    for s in range(n):
        c.parents[s, there[s]:] = r.choice([-2, -9, 200], n_tree - there[s])
    c.lens = [int(c.max_ctx - t - (s % 3 == 0)) if t else 3 for s, t in enumerate(there)]
    over = np.array([s % 5 == 4 and t > 0 for s, t in enumerate(there)])
    c.lens = [int(c.max_ctx - t + 1) if o else n for n, t, o in zip(c.lens, there, over)]
    some = [s for s in range(n) if not over[s]]
    want, bound = exact(c, some)
    print(f"[case] {n} trees of up to {n_tree}", flush=True)
    c.upload().launch()
    out, _, _ = c.results()
    assert np.isnan(out[over]).all()
    assert (np.abs(out[some] - want) <= bound).all(), float(np.abs(out[some] - want).max())


@pytest.mark.parametrize("heads,kv,d,n_tree,lens,room", [(8, 2, 128, 5, [300], 9), (8, 2, 64, 26, [1000], 9), (8, 2, 128, 26, [4070], 0),
                                                         (32, 8, 128, 9, [700, 0, 33, 2500], 40), (8, 1, 64, 64, [3000], 4000),
                                                         (16, 1, 128, 64, [2000], 50000), (8, 8, 64, 30, [100, 5000], 9)])
def test_errors_are_those_of_f32(gpu, heads, kv, d, n_tree, lens, room):
    """Over all rows together the roundings are random: far below the bound of a single one, which a lost limb of the
    queries or the weights (2^-12) would keep."""
    c = Case(len(lens), n_tree, heads, kv, d, lens, room=room, seed=d + n_tree)
    want, _ = exact(c)
    c.upload().launch()
    got = c.results()[0]
    rel = float(np.linalg.norm(got - want) / np.linalg.norm(want))
    print(f"[result] {heads}/{kv}x{d} {n_tree} nodes at {lens}: rel-L2 {rel:.2e}, bar {weights_bar(c.top):.2e}", flush=True)
    assert rel <= weights_bar(c.top)


@pytest.mark.parametrize("d,kv,group", [(64, 2, 2), (128, 2, 2), (128, 1, 8), (64, 8, 1)])
@pytest.mark.parametrize("n_tree,ctx,room", [(20, 0, 5), (128, 37, 0), (128, 500, 0), (128, 1000, 3000), (70, 4097, 0),
                                             (33, 17500, 0), (33, 36000, 9)])
def test_every_key_is_read(gpu, d, kv, group, n_tree, ctx, room):
    """Without rotation, a query of three or eight times a key has all its weight there: each query row looks for a key of its own,
    its node's, its parent's, or one at the end of a tile, a stage or a chunk; the row is that key's v."""
    c = Case(1, n_tree, kv * group, kv, d, [ctx], room=room, shape="chain" if ctx % 2 else "forest", seed=ctx + d)
    c.inv[:] = 0
    q, k, v = c.views()
    k[:] = c.rng.standard_normal(k.shape)
    paths = _tree.paths(c.parents[0])
    ends = [e + o for e in (0, 32, 64, 128, 256, 384, 512, 768, 1024, 2048, 4096, 8192, 16384, ctx) for o in (-2, -1, 0, 1)]
    ends = [e for e in ends if 0 <= e < ctx] or [0]
    goal = np.zeros((n_tree, kv * group), int)
    for t in range(n_tree):
        for h in range(kv * group):
            pick = (t + 3 * h) % 4
            if pick == 0 or ctx == 0:
                goal[t, h] = ctx + paths[t][-1 - (t % 3 == 0 and len(paths[t]) > 1)]
            elif pick == 1:
                goal[t, h] = int(c.rng.integers(0, ctx))
            else:
                goal[t, h] = ends[(t * kv * group + h) % len(ends)]
            g = goal[t, h]
            key = c.kc[0, g, h // group] if g < ctx else k[0, g - ctx, h // group]
            q[0, t, h] = np.float32(3 if d == 128 else 8) * key.astype(np.float32)
    want, _ = exact(c)
    vals = np.concatenate([c.vc[0, :ctx], v[0].astype(np.float16)]).astype(np.float64)
    for t in range(n_tree):
        for h in range(kv * group):  # that is what the formula says, too
            assert np.abs(want[0, t, h] - vals[goal[t, h], h // group]).max() < 0.05
    c.upload().launch()
    got = c.results()[0]
    err = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
    print(f"[result] keys of {kv}x{group}x{d} at {ctx}: rel-L2 {err.max():.2e} a row, bar {weights_bar(c.top):.2e}", flush=True)
    assert err.max() <= weights_bar(c.top)
