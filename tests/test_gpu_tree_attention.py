"""wh_attention_tree against the 64-bit form: shapes, ragged batches, masks, what a row must not see, graphs."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, report, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


class Case:
    """Random inputs of one call, in host arrays."""

    def __init__(self, n_seqs, n_tree, heads, kv, d, lens, room=9, shape="tree", seed=0, pad=0, qscale=1.0):
        r = self.rng = np.random.default_rng(seed)
        self.n, self.t, self.h, self.kv, self.d = n_seqs, n_tree, heads, kv, d
        self.lens = list(lens)
        self.max_ctx = max(self.lens) + n_tree + room
        rows = n_seqs * n_tree
        f = lambda w: (r.standard_normal((rows, w + pad)) * 1.2).astype(np.float32)
        self.q, self.k, self.v = f(heads * d) * np.float32(qscale), f(kv * d), f(kv * d)
        cache = lambda: r.standard_normal((n_seqs, self.max_ctx, kv, d)).astype(np.float16)
        self.kc, self.vc = cache(), cache()
        self.parents = np.stack([_tree.make_parents(r, n_tree, shape) for _ in range(n_seqs)])
        self.inv = ops.rope_inv_freq(500000.0, d)

    def views(self):
        cut = lambda x, hh: x[:, :hh * self.d].reshape(self.n, self.t, hh, self.d)
        return cut(self.q, self.h), cut(self.k, self.kv), cut(self.v, self.kv)

    def expect(self):
        q, k, v = self.views()
        kc, vc = self.kc.copy(), self.vc.copy()
        out, bound = zip(*[_tree.attention(q[s], k[s], v[s], self.parents[s], self.lens[s], kc[s], vc[s], self.inv)
                           for s in range(self.n)])
        return np.stack(out), np.stack(bound), kc, vc

    def upload(self):
        # a guard row behind the last sequence's cache
        guard = np.full((1, self.kv, self.d), 7.5, np.float16)
        flat = lambda c: np.concatenate([c.reshape(-1, self.kv, self.d), guard]).view(np.uint16)
        self.dev = dict(q=up(self.q)[0], k=up(self.k)[0], v=up(self.v)[0], parents=up(self.parents)[0],
                        ctx=up(np.array(self.lens, np.uint32))[0], kc=up(flat(self.kc))[0], vc=up(flat(self.vc))[0],
                        inv=up(self.inv)[0])
        self.dev["out"] = DeviceBuffer(4 * self.n * self.t * self.h * self.d + 256)  # and a guard
        self.dev["out"].fill(0xEE)
        self.wsz = ops.attention_tree_workspace_bytes(self.n, self.t, self.h, self.kv, self.d, self.max_ctx)
        self.dev["ws"] = DeviceBuffer(self.wsz + 256)
        self.dev["ws"].fill(0xFF)  # NaN, and a guard
        self.guard = self.dev["ws"]
        return self

    def launch(self, stream=None):
        b = self.dev
        ops.attention_tree(b["q"], b["k"], b["v"], self.q.shape[1], self.k.shape[1], b["parents"], b["ctx"], self.n, self.t,
                           b["kc"], b["vc"], self.max_ctx, self.h, self.kv, self.d, b["inv"], b["out"], b["ws"], self.wsz,
                           stream)

    def results(self):
        out = down(self.dev["out"], np.float32, self.n * self.t * self.h * self.d).reshape(self.n, self.t, self.h, self.d)
        assert (down(self.dev["out"], np.uint8, 256, offset=out.nbytes) == 0xEE).all(), "behind the output"
        if self.dev["ws"] is self.guard:
            assert (down(self.guard, np.uint8, 256, offset=self.wsz) == 0xFF).all(), "behind the workspace"
        caches = []
        for name in ("kc", "vc"):
            c = down(self.dev[name], np.float16, (self.n * self.max_ctx + 1) * self.kv * self.d).reshape(-1, self.kv, self.d)
            assert (c[-1] == 7.5).all(), "the row behind the last sequence changed"
            caches.append(c[:-1].reshape(self.n, self.max_ctx, self.kv, self.d))
        return out, *caches

    def check(self, tag):
        want, bound, kc, vc = self.expect()
        out, gk, gv = self.results()
        self.compare(tag, out, want, bound)
        assert np.array_equal(gk.view(np.uint16), kc.view(np.uint16)), "K cache"
        assert np.array_equal(gv.view(np.uint16), vc.view(np.uint16)), "V cache"

    def compare(self, tag, out, want, bound):
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(out), np.isnan(want)), "NaN in other places"
        inf = ~fine & ~np.isnan(want)
        assert np.array_equal(out[inf], want[inf].astype(np.float32))
        err = np.where(fine, np.abs(np.where(fine, out, 0) - np.where(fine, want, 0)), 0)
        if fine.any():
            rel = float(np.linalg.norm(err) / max(np.linalg.norm(want[fine]), 1e-30))
            report(f"tree attention {tag}", rel, float(err.max()))
        assert (err <= bound[..., None]).all(), (float(err.max()), float(bound.max()))


def run(case, tag):
    print(f"[case] tree attention {tag}", flush=True)
    case.upload().launch()
    case.check(tag)


@pytest.mark.parametrize("heads,kv,d", [(32, 8, 128), (8, 8, 128), (7, 1, 128), (6, 2, 64), (16, 2, 64), (10, 2, 128),
                                        (4, 4, 64), (24, 1, 128)])
@pytest.mark.parametrize("n_tree,ctx", [(1, 0), (1, 77), (2, 1), (5, 300), (16, 33), (17, 64), (33, 1000)])
def test_heads_and_lengths(gpu, heads, kv, d, n_tree, ctx):
    run(Case(1, n_tree, heads, kv, d, [ctx], seed=n_tree * 1000 + ctx), f"{heads}/{kv}x{d} tree {n_tree} ctx {ctx}")


@pytest.mark.parametrize("ctx", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 511, 4097])
@pytest.mark.parametrize("n_tree,heads,kv,d", [(3, 4, 2, 128), (64, 8, 2, 128), (21, 8, 2, 64)])
def test_context_ends_inside_a_tile(gpu, ctx, n_tree, heads, kv, d):
    run(Case(1, n_tree, heads, kv, d, [ctx], room=0, seed=ctx), f"{heads}/{kv}x{d} tree {n_tree} ctx {ctx} no room")


@pytest.mark.parametrize("shape", ["chain", "star", "forest", "padded", "absent"])
@pytest.mark.parametrize("n_tree", [1, 31, 64, 65, 128])
@pytest.mark.parametrize("d", [64, 128])
def test_tree_shapes(gpu, shape, n_tree, d):
    run(Case(1, n_tree, 8, 2, d, [150], shape=shape, seed=n_tree), f"{shape} {n_tree} d {d}")


@pytest.mark.parametrize("heads,kv,d,n_tree", [(8, 2, 128, 6), (8, 4, 64, 40), (4, 4, 128, 17), (8, 1, 128, 9)])
@pytest.mark.parametrize("shape", ["tree", "padded"])
def test_ragged_batches(gpu, heads, kv, d, n_tree, shape):
    lens = [0, 1, 700, 33, 64, 2500, 5]
    run(Case(len(lens), n_tree, heads, kv, d, lens, shape=shape, seed=d), f"ragged {heads}/{kv}x{d} tree {n_tree} {shape}")


@pytest.mark.parametrize("heads,kv,d,n_tree", [(8, 2, 128, 5), (8, 2, 128, 12), (8, 2, 64, 30)])
@pytest.mark.parametrize("room", [0, 100, 400, 5000])
def test_room_behind_the_rows(gpu, heads, kv, d, n_tree, room):
    """The cache's size decides how the rows are cut up, not what comes out."""
    run(Case(3, n_tree, heads, kv, d, [100 - n_tree, 0, 17], room=room, shape="padded", seed=room),
        f"{heads}/{kv}x{d} tree {n_tree} room {room}")


@pytest.mark.parametrize("n,n_tree", [(300, 3), (1024, 1)])
def test_many_sequences(gpu, n, n_tree):
    rng = np.random.default_rng(3)
    lens = [int(v) for v in rng.integers(0, 90, n)]
    run(Case(n, n_tree, 4, 2, 64, lens, seed=5), f"{n} sequences")


@pytest.mark.parametrize("d", [64, 128])
def test_large_batches(gpu, d):
    """Enough nodes, heads and tiles that waves take more of them each; sequences of one chunk and of several."""
    lens = [0, 3, 40, 1500, 64, 700, 17, 130, 1, 90, 400, 33]
    run(Case(12, 81, 30, 6, d, lens, room=60, shape="padded", seed=d), f"large batch d {d}")


@pytest.mark.parametrize("pad", [1, 4, 64])
def test_row_strides(gpu, pad):
    run(Case(2, 9, 6, 2, 64, [50, 200], pad=pad, seed=pad), f"rows padded by {pad}")


def test_parts_of_one_qkv_row(gpu):
    """q, k and v as parts of [q | k | v] rows, as wh_attention_qkv lays them out."""
    c = Case(2, 7, 8, 2, 128, [90, 11], seed=8)
    whole = np.concatenate([c.q, c.k, c.v], 1)
    c.upload()
    b = c.dev
    row = up(whole)[0]
    ld = whole.shape[1]
    ops.attention_tree(row.ptr, row.ptr + 4 * 8 * 128, row.ptr + 4 * 10 * 128, ld, ld, b["parents"], b["ctx"], c.n, c.t,
                       b["kc"], b["vc"], c.max_ctx, c.h, c.kv, c.d, b["inv"], b["out"], b["ws"], c.wsz)
    c.check("one qkv row")


@pytest.mark.parametrize("qscale", [0.0, 1e-30, 1e-6, 30.0])
@pytest.mark.parametrize("d", [64, 128])
def test_query_magnitudes(gpu, qscale, d):
    """Queries of zero (equal weights), far below and far above the usual."""
    run(Case(1, 11, 8, 2, d, [333], seed=4, qscale=qscale), f"q times {qscale} d {d}")


def test_scores_beyond_f16(gpu):
    """q.k of about 1e7: far beyond f16; the largest score takes all the weight."""
    c = Case(1, 5, 4, 2, 128, [200], seed=6, qscale=1e4)
    c.kc *= np.float16(30)
    run(c, "scores beyond f16")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n_tree,ctx", [(12, 37), (70, 37), (6, 0), (12, 700), (6, 900), (100, 640)])
def test_what_a_row_does_not_see(gpu, d, n_tree, ctx):
    """NaN and infinities in stale cache rows, in absent nodes and in nodes off a
    row's path must not reach it; on its path they must."""
    c = Case(2, n_tree, 8, 2, d, [ctx, ctx + 5], shape="padded", seed=9)
    for s, n in enumerate(c.lens):
        c.kc[s, n:] = np.nan
        c.vc[s, n:] = np.inf
    q, k, v = c.views()
    for s in range(2):
        absent = [t for t, p in enumerate(_tree.paths(c.parents[s])) if p is None]
        q[s, absent] = k[s, absent] = np.nan
        v[s, absent] = -np.inf
    k[0, 1, 0, 3] = np.nan       # a node whose k is NaN for one KV head
    v[0, 2, :, 5] = np.inf       # one whose v is infinite in one dim
    v[1, 1, 1, :2] = [np.nan, -np.inf]
    v[1, 2, 0, 7] = 1e6          # beyond f16: stored as infinity
    run(c, f"unseen rows d {d} tree {n_tree} ctx {ctx}")


@pytest.mark.parametrize("n_tree", [5, 12, 30, 64])
@pytest.mark.parametrize("room", [0, 4000])
@pytest.mark.parametrize("d", [64, 128])
def test_infinities_in_the_cache_count(gpu, n_tree, room, d):
    """Infinities and NaN that the cache itself holds are seen by every row: a dim with infinities of one sign is that
    infinity, of both NaN; a NaN in k makes every row of its KV head NaN."""
    ctx = 900 if room else 100
    c = Case(1, n_tree, 8, 2, d, [ctx], room=room, seed=d + n_tree)
    c.vc[0, 3, 0, 5] = np.inf
    c.vc[0, 40, 0, 9] = -np.inf
    c.vc[0, 41, 0, 9] = -np.inf
    c.vc[0, ctx - 1, 0, 11] = np.inf
    c.vc[0, ctx - 70, 0, 11] = -np.inf
    c.vc[0, ctx - 3, 0, 20] = np.nan
    c.vc[0, 17, 0, d - 1] = np.nan
    c.kc[0, 64, 1, 2] = np.nan
    want, _, _, _ = c.expect()
    assert np.isposinf(want[0, :, 0, 5]).all() and np.isneginf(want[0, :, 1, 9]).all() and np.isnan(want[0, :, 2, 11]).all()
    run(c, f"infinities d {d} tree {n_tree} room {room}")


@pytest.mark.parametrize("heads,kv,d,n_tree", [(8, 2, 128, 6), (8, 2, 64, 20), (8, 1, 128, 30)])
def test_a_chunk_of_nothing_but_nan(gpu, heads, kv, d, n_tree):
    """The nodes lie in a chunk of their own (the cache is whole chunks), in which node 0 sees itself alone: its k is
    NaN, so are its row and every row below it, and a sibling's row is not."""
    c = Case(1, n_tree, heads, kv, d, [1024], room=3000, shape="star", seed=d)
    c.parents[0, 1] = -1  # a second root, and a node below it
    c.parents[0, 2] = 1
    c.views()[1][0, 0, :, 3] = np.nan
    want, _, _, _ = c.expect()
    assert np.isnan(want[0, 0]).all() and np.isfinite(want[0, 1:3]).all() and np.isnan(want[0, 3:]).all()
    run(c, f"chunk of NaN {heads}/{kv}x{d} tree {n_tree}")


# Caches of so many rows have their query rows cut into tiles that workgroups take by 1, 2 and 4: on 32 KV heads up to
# 70 nodes by 1 up to 768 rows, by 2 up to 2048, then by 4; on 8 KV heads 27 nodes of 3 heads by 1 up to 3840, by 2 up
# to 8192 (two sequences: half as many each).
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctx", [0, 1, 31, 64, 129, 600])
@pytest.mark.parametrize("heads,kv,n_tree,rows", [(32, 32, 70, 700), (32, 32, 70, 1500), (32, 32, 70, 2200),
                                                  (24, 8, 27, 8500)])
def test_tiles_of_a_workgroup(gpu, heads, kv, n_tree, rows, ctx, d):
    run(Case(1, n_tree, heads, kv, d, [ctx], room=rows - ctx - n_tree, shape="padded", seed=ctx + d),
        f"{heads}/{kv}x{d} tree {n_tree} ctx {ctx} of {rows}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1000, 2500, 4500])
@pytest.mark.parametrize("ctx", [0, 37, 640])
def test_unseen_rows_and_infinities_in_every_tiling(gpu, rows, ctx, d):
    c = Case(2, 27, 24, 8, d, [ctx, ctx + 5], room=rows - ctx - 32, shape="padded", seed=rows)
    for s, n in enumerate(c.lens):
        c.kc[s, n:] = np.nan
        c.vc[s, n:] = -np.inf
    q, k, v = c.views()
    for s in range(2):
        absent = [t for t, p in enumerate(_tree.paths(c.parents[s])) if p is None]
        q[s, absent] = k[s, absent] = np.nan
        v[s, absent] = np.inf
    k[0, 1, 0, 3] = np.nan
    v[0, 2, :, 5] = np.inf
    if ctx:
        c.vc[1, 3, 7, 9] = np.inf
        c.vc[1, ctx - 1, 7, 11] = -np.inf
        c.vc[1, 30, 6, d - 1] = np.nan
        c.kc[0, 20, 5, 2] = np.nan
    run(c, f"unseen rows d {d} ctx {ctx} of {rows}")


@pytest.mark.parametrize("d", [64, 128])
def test_chunks_of_one_and_of_two_workgroups_per_cu(gpu, d):
    """Chunks grow with the rows up to 1024 keys, are halved beyond, and grow again."""
    for ctx in (9000, 17500, 36000):
        run(Case(1, 2, 32, 8, d, [ctx], seed=ctx), f"2 nodes at {ctx}, d {d}")
        run(Case(1, 30, 6, 6, d, [ctx], seed=ctx), f"30 nodes at {ctx}, d {d}")


def test_largest_queries(gpu):
    """Queries of 1e36 over keys of 1e-4: the scale of a row has the whole range of f32's exponents."""
    c = Case(1, 6, 4, 2, 128, [90], seed=3, qscale=1e36)
    c.kc *= np.float16(1e-4)
    c.k *= np.float32(1e-4)
    run(c, "q times 1e36")


def test_sequence_that_does_not_fit(gpu):
    """ctx_len + n_tree > max_ctx: NaN for that sequence, nothing stored, the others as ever."""
    c = Case(4, 8, 4, 2, 128, [20, 60, 61, 30], room=0, seed=2)
    c.lens[2], c.lens[3] = 62, 0xFFFFFFF0  # max_ctx is 69
    want_k, want_v = c.kc.copy(), c.vc.copy()
    q, k, v = c.views()
    parts = [_tree.attention(q[s], k[s], v[s], c.parents[s], c.lens[s], want_k[s], want_v[s], c.inv) for s in range(4)]
    c.upload().launch()
    out, gk, gv = c.results()
    assert np.isnan(out[2:]).all()
    c.compare("does not fit", out, np.stack([p[0] for p in parts]), np.stack([p[1] for p in parts]))
    assert np.array_equal(gk.view(np.uint16), want_k.view(np.uint16))
    assert np.array_equal(gv.view(np.uint16), want_v.view(np.uint16))


@pytest.mark.parametrize("d,heads,kv", [(64, 8, 2), (128, 32, 8)])
def test_one_node_is_the_decode_step(gpu, d, heads, kv):
    """A tree of one node and wh_attention_decode agree; the angles differ by pos * 2^-24 radians at most, which moves
    a score by at most that times S = max |q| |k| / sqrt(d), an output by twice that times max |v|."""
    ctx = 200
    c = Case(1, 1, heads, kv, d, [ctx], seed=12)
    qkv = up(np.concatenate([c.q, c.k, c.v], 1))[0]
    k0, v0 = up(c.kc.view(np.uint16))[0], up(c.vc.view(np.uint16))[0]
    out = DeviceBuffer(4 * heads * d)
    wsz = ops.attention_workspace_bytes(heads, kv, d, ctx + 1)
    c.upload()
    ops.attention_decode(qkv, k0, v0, ctx, heads, kv, d, c.dev["inv"], out, DeviceBuffer(wsz), wsz)
    synchronize()
    c.launch()
    got, _, _ = c.results()
    _, bound, kc, vc = c.expect()
    s = np.linalg.norm(c.q.reshape(heads, d), axis=1).max() * np.linalg.norm(kc[0].astype(np.float64), axis=-1).max() / np.sqrt(d)
    vmax = np.abs(vc.astype(np.float64)).max()
    # the new k may also round to the neighbouring f16: 2^-10 of one key's score
    tol = 2 * bound.max() + 2 * vmax * s * (ctx * 2.0 ** -24 + 2.0 ** -10 / 10)
    assert np.abs(got.ravel() - down(out, np.float32, heads * d)).max() <= tol


def test_far_positions(gpu):
    """Position 1000000: the angle needs 64 bits.  The cache in between is zeros: keys of score 0 and v 0."""
    ctx, d, heads, kv, t = 1_000_000, 64, 2, 1, 3
    c = Case(1, t, heads, kv, d, [10], seed=14)
    live, base = 40, ctx - 40
    kc, vc = c.rng.standard_normal((2, live, kv, d)).astype(np.float16)
    row = kv * d * 2
    kb, vb = DeviceBuffer((ctx + t) * row), DeviceBuffer((ctx + t) * row)
    for b, x in ((kb, kc), (vb, vc)):
        b.fill(0)
        b.upload(x.view(np.uint16), offset=base * row)
    wsz = ops.attention_tree_workspace_bytes(1, t, heads, kv, d, ctx + t)
    out, ws = DeviceBuffer(4 * t * heads * d), DeviceBuffer(wsz)
    ops.attention_tree(up(c.q)[0], up(c.k)[0], up(c.v)[0], heads * d, kv * d, up(c.parents)[0],
                       up(np.array([ctx], np.uint32))[0], 1, t, kb, vb, ctx + t, heads, kv, d, up(c.inv)[0], out, ws, wsz)
    got = down(out, np.float32, t * heads * d).reshape(t, heads, d)
    q, k, v = (x[0] for x in c.views())
    ps = _tree.paths(c.parents[0])
    newk = np.stack([_tree.stored(_tree.rotate(k[i], ctx + len(p) - 1, c.inv)) for i, p in enumerate(ps)])
    assert np.array_equal(down(kb, np.float16, t * kv * d, offset=ctx * row).view(np.uint16), newk.ravel().view(np.uint16))
    for i, p in enumerate(ps):
        qr = _tree.rotate(q[i], ctx + len(p) - 1, c.inv)
        keys = np.concatenate([kc[:, 0], newk[p, 0]]).astype(np.float64)
        vals = np.concatenate([vc[:, 0], v[p, 0].astype(np.float16)]).astype(np.float64)
        for h in range(heads):
            s = keys @ qr[h] / np.sqrt(d)
            w = np.exp(s)
            want = (w @ vals) / (w.sum() + base)
            # every weight to 8e-5 (as in _tree.attention, S < 10), in the sum and in the total; both in tiles and chunks
            assert np.abs(got[i, h] - want).max() <= 3e-4 * (w @ np.abs(vals)).max() / (w.sum() + base)


def test_offsets_beyond_32_bits(gpu):
    """A batch whose caches pass 4 GiB: the last sequence's rows lie beyond."""
    n, t, heads, kv, d, max_ctx = 2, 4, 8, 8, 128, 1_100_000
    row = kv * d * 2
    c = Case(n, t, heads, kv, d, [30, 90], seed=15)
    assert n * max_ctx * row > 1 << 32
    kb, vb = DeviceBuffer(n * max_ctx * row), DeviceBuffer(n * max_ctx * row)
    lens = [30, max_ctx - t]
    # sequence 1: zeros but for its last 90 rows
    for b, x in ((kb, c.kc), (vb, c.vc)):
        b.fill(0)
        b.upload(x[0, :30].view(np.uint16))
        b.upload(x[1, :90].view(np.uint16), offset=(max_ctx + lens[1] - 90) * row)
    wsz = ops.attention_tree_workspace_bytes(n, t, heads, kv, d, max_ctx)
    out, ws = DeviceBuffer(4 * n * t * heads * d), DeviceBuffer(wsz)
    ops.attention_tree(up(c.q)[0], up(c.k)[0], up(c.v)[0], heads * d, kv * d, up(c.parents)[0],
                       up(np.array(lens, np.uint32))[0], n, t, kb, vb, max_ctx, heads, kv, d, up(c.inv)[0], out, ws, wsz)
    got = down(out, np.float32, n * t * heads * d).reshape(n, t, heads, d)
    q, k, v = c.views()
    zeros = [0, lens[1] - 90]
    for s in range(n):
        ps = _tree.paths(c.parents[s])
        newk = np.stack([_tree.stored(_tree.rotate(k[s, i], lens[s] + len(p) - 1, c.inv)) for i, p in enumerate(ps)])
        off = (s * max_ctx + lens[s]) * row
        assert np.array_equal(down(kb, np.float16, t * kv * d, offset=off).view(np.uint16), newk.ravel().view(np.uint16))
        live = 30 if s == 0 else 90
        for i, p in enumerate(ps):
            qr = _tree.rotate(q[s, i], lens[s] + len(p) - 1, c.inv)
            for h in range(heads):
                keys = np.concatenate([c.kc[s, :live, h], newk[p, h]]).astype(np.float64)
                vals = np.concatenate([c.vc[s, :live, h], v[s, p, h].astype(np.float16)]).astype(np.float64)
                w = np.exp(keys @ qr[h] / np.sqrt(d))
                want = (w @ vals) / (w.sum() + zeros[s])
                assert np.abs(got[s, i, h] - want).max() <= 5e-4 * (w @ np.abs(vals)).max() / (w.sum() + zeros[s])  # S < 16


def test_captured_step_follows_the_lengths(gpu):
    """Two graphs on one workspace in turn; lengths, parents and rows change between replays, with eager work between."""
    stream = Stream()
    a = Case(2, 10, 8, 2, 128, [100, 40], room=400, seed=20).upload()
    b = Case(1, 40, 8, 2, 128, [60], room=400, seed=21).upload()
    ws = DeviceBuffer(max(a.wsz, b.wsz))
    a.dev["ws"] = b.dev["ws"] = ws
    synchronize()
    graphs = []
    for c in (a, b):
        with Graph.capture(stream) as g:
            c.launch(stream)
        graphs.append(g)
    other = Case(1, 5, 4, 2, 64, [70], seed=22)
    for rep in range(3):
        for c, g in zip((a, b), graphs):
            c.lens = [int(v) for v in c.rng.integers(0, 300, c.n)]
            c.parents = np.stack([_tree.make_parents(c.rng, c.t, ("tree", "padded", "chain")[rep]) for _ in range(c.n)])
            c.q = c.rng.standard_normal(c.q.shape).astype(np.float32)
            c.dev["ctx"].upload(np.array(c.lens, np.uint32))
            c.dev["parents"].upload(c.parents)
            c.dev["q"].upload(c.q)
            # the caches as the last replay left them
            _, c.kc, c.vc = c.results()
            g.launch(stream)
            stream.synchronize()
            c.check(f"replay {rep}")
        run(other, "eager between replays")
    for g in graphs:
        g.destroy()
    stream.destroy()


def test_same_bits_again(gpu):
    c = Case(3, 20, 8, 2, 128, [900, 0, 77], seed=30).upload()
    c.launch()
    first = c.results()[0]
    for _ in range(3):
        c.dev["ws"].fill(0x55)
        c.guard = None
        c.launch()
        assert np.array_equal(c.results()[0].view(np.uint32), first.view(np.uint32))


def test_two_streams_at_once(gpu):
    """Calls on two streams with workspaces of their own, several in flight on each, do not disturb each other."""
    streams = [Stream(), Stream()]
    cases = [Case(2, 13, 8, 2, 128, [1500, 200], seed=40).upload(), Case(1, 64, 16, 4, 64, [3000], seed=41).upload()]
    synchronize()
    for _ in range(5):
        for c, s in zip(cases, streams):
            c.launch(s)
    for s in streams:
        s.synchronize()
    for i, c in enumerate(cases):
        c.check(f"stream {i}")
    for s in streams:
        s.destroy()
