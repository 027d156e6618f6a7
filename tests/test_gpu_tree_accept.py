"""wh_tree_accept and wh_kv_cache_compact against their definitions: whole numbers and rows, bit for bit."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu
NO = _tree.NO_TOKEN
u32 = lambda a: np.asarray(a).astype(np.uint32)


def run_accept(tokens, parents, picked, ctx=None, history=None, in_place=False):
    n, t = tokens.shape
    path, count, nxt = DeviceBuffer(4 * n * t), DeviceBuffer(4 * n), DeviceBuffer(4 * n)
    for b in (path, count, nxt):
        b.fill(0xEE)
    cb = up(u32(ctx))[0] if ctx is not None else None
    after = (cb if in_place else DeviceBuffer(4 * n)) if ctx is not None else None
    hb = up(u32(history))[0] if history is not None else None
    ops.tree_accept(up(u32(tokens))[0], up(parents.astype(np.int32))[0], up(u32(picked))[0], n, t, path, count, nxt, cb,
                    after, hb, history.shape[1] if history is not None else 0)
    get = lambda b, k: down(b, np.uint32, k)
    return (get(path, n * t).reshape(n, t), get(count, n), get(nxt, n), get(after, n) if after else None,
            get(hb, history.size).reshape(history.shape) if hb else None)


@pytest.mark.parametrize("t", [1, 2, 26, 63, 64, 65, 100, 128])
@pytest.mark.parametrize("shape", ["chain", "star", "tree", "forest", "padded", "absent"])
@pytest.mark.parametrize("in_place", [False, True])
def test_walk(gpu, t, shape, in_place):
    print(f"[case] accept {shape} {t} in place {in_place}", flush=True)
    r = np.random.default_rng(t)
    n = 9
    parents = np.stack([_tree.make_parents(r, t, shape) for _ in range(n)])
    tokens = r.integers(0, 6, (n, t))  # siblings often carry the same token
    picked = r.integers(0, 6, (n, t))
    for s in range(n - 1):  # mostly in agreement; the last sequence by chance only
        for i in range(1, t):
            if 0 <= parents[s, i] < i and r.random() < 0.9:
                picked[s, parents[s, i]] = tokens[s, i]
    picked[0, 0] = NO  # no token allowed at the root
    ctx = r.integers(0, 50, n)
    history = r.integers(100, 200, (n, 60))  # too short for the longest walks
    path, count, nxt, after, hist = run_accept(tokens, parents, picked, ctx, history, in_place)
    for s in range(n):
        want, last = _tree.accept(tokens[s], parents[s], picked[s])
        assert count[s] == len(want) and nxt[s] == last, s
        assert list(path[s, :len(want)]) == want and (path[s, len(want):] == NO).all(), s
        assert after[s] == ctx[s] + len(want)
        h = history[s].copy()
        for i, a in enumerate(want):
            if ctx[s] + i < 60:
                h[ctx[s] + i] = tokens[s, a]
        assert np.array_equal(hist[s], h), s


def test_walk_alone(gpu):
    """Without lengths and history; tokens that are all bits set never match."""
    parents = np.array([[-1, 0, 1]])
    path, count, nxt, _, _ = run_accept(np.array([[7, NO, 3]]), parents, np.array([[NO, 3, 9]]))
    assert count[0] == 1 and nxt[0] == NO and list(path[0]) == [0, NO, NO]
    path, count, nxt, _, _ = run_accept(np.array([[7, 5, 3]]), parents, np.array([[5, 3, 9]]))
    assert count[0] == 3 and nxt[0] == 9 and list(path[0]) == [0, 1, 2]


def compact_case(r, layers, n, max_ctx, kv, d, t):
    caches = r.integers(0, 1 << 16, (layers, 2, n, max_ctx, kv, d), dtype=np.uint16)
    path, count = np.full((n, t), NO, np.int64), np.zeros(n, np.int64)
    for s in range(n):
        count[s] = int(r.integers(0, t + 1)) if s else t
        if count[s]:
            path[s, 0] = 0
            path[s, 1:count[s]] = np.sort(r.permutation(np.arange(1, t))[:count[s] - 1])
    before = r.integers(0, max_ctx - t + 1, n)
    return caches, path, count, before


def run_compact(caches, path, count, after):
    layers, _, n, max_ctx, kv, d = caches.shape
    bufs = [[up(caches[l, j])[0] for j in range(2)] for l in range(layers)]
    ops.kv_cache_compact(ops.KvCaches([b[0] for b in bufs], [b[1] for b in bufs]), n, max_ctx, kv, d, up(u32(path))[0],
                         path.shape[1], up(u32(count))[0], up(u32(after))[0])
    return np.stack([np.stack([down(b, np.uint16, caches[0, 0].size).reshape(caches.shape[2:]) for b in two]) for two in bufs])


@pytest.mark.parametrize("layers,n,max_ctx,kv,d,t", [(1, 1, 8, 1, 8, 8), (3, 4, 40, 2, 64, 26), (70, 2, 20, 1, 64, 9),
                                                     (2, 3, 200, 8, 128, 128), (2, 1, 30, 5, 24, 17), (1, 2, 12, 40, 128, 10)])
def test_rows_move_together(gpu, layers, n, max_ctx, kv, d, t):
    print(f"[case] compact {layers} layers {n}x{max_ctx} {kv}x{d} tree {t}", flush=True)
    caches, path, count, before = compact_case(np.random.default_rng(t), layers, n, max_ctx, kv, d, t)
    want = caches.copy()
    for s in range(n):
        for i in range(count[s]):
            want[:, :, s, before[s] + i] = caches[:, :, s, before[s] + path[s, i]]
    assert np.array_equal(run_compact(caches, path, count, before + count), want)


def test_numbers_that_do_not_fit_move_nothing(gpu):
    """Counts beyond the tree or the length, lengths beyond the cache: untouched; path entries that name no later
    row of the tree or lie beyond the cache: that row stays."""
    r = np.random.default_rng(1)
    caches = r.integers(0, 1 << 16, (2, 2, 5, 20, 1, 64), dtype=np.uint16)
    path = np.tile(np.array([0, 2, 3, 5]), (5, 1))
    path[3] = [3, 0, NO, 200]  # row 0 takes row 3, the others stay
    path[4] = [0, 2, 3, 3]
    count = np.array([5, 4, 4, 4, 4])
    after = np.array([10, 3, 21, 10, 20])  # 4 is fine but row first + 3 is its own
    got = run_compact(caches, path, count, after)
    want = caches.copy()
    want[:, :, 3, 6] = caches[:, :, 3, 9]
    want[:, :, 4, 17] = caches[:, :, 4, 18]
    want[:, :, 4, 18] = caches[:, :, 4, 19]
    assert np.array_equal(got, want)


def test_rows_beyond_32_bits(gpu):
    """A cache of more than 4 GiB."""
    max_ctx, kv, d = 2_200_000, 8, 128
    row = kv * d * 2
    assert max_ctx * row > 1 << 32
    k, v = DeviceBuffer(max_ctx * row), DeviceBuffer(max_ctx * row)
    rows = np.random.default_rng(2).integers(0, 1 << 16, (2, 6, kv * d), dtype=np.uint16)
    first = max_ctx - 6
    for b, x in ((k, rows[0]), (v, rows[1])):
        b.fill(0)
        b.upload(x, offset=first * row)
    ops.kv_cache_compact(ops.KvCaches([k], [v]), 1, max_ctx, kv, d, up(u32([[0, 3, 5, NO, NO, NO]]))[0], 6, up(u32([3]))[0],
                         up(u32([first + 3]))[0])
    for b, x in ((k, rows[0]), (v, rows[1])):
        got = down(b, np.uint16, 6 * kv * d, offset=first * row).reshape(6, -1)
        assert np.array_equal(got, x[[0, 3, 5, 3, 4, 5]])
        assert not down(b, np.uint16, kv * d).any()
