"""Trees at the end of a cache: what does not fit changes nothing, alone and in a whole run."""
import numpy as np
import pytest

from tests import _tree
from tests._gpu import down, up
from tests.test_gpu_tree_accept import NO, u32
from tests.test_gpu_tree_step import MODELS, Model
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer, Graph, Stream, synchronize

pytestmark = pytest.mark.gpu


def rows_of(parents) -> int:
    return max([i + 1 for i, p in enumerate(parents) if -1 <= p < i], default=0)


@pytest.mark.parametrize("t", [1, 2, 26, 64, 65, 128])
@pytest.mark.parametrize("shape", ["chain", "star", "forest", "padded", "absent"])
def test_walk_of_trees_that_may_not_fit(gpu, t, shape):
    print(f"[case] accept in cache {shape} {t}", flush=True)
    r = np.random.default_rng(t)
    n, max_ctx = 11, 200
    parents = np.stack([_tree.make_parents(r, t, shape) for _ in range(n)])
    tokens, picked = r.integers(0, 4, (n, t)), r.integers(0, 4, (n, t))
    rows = np.array([rows_of(p) for p in parents])
    ctx = max_ctx - rows + np.array([0, 1, -1, 0, 1, -1, 0, 1, -5, 3, 0])
    ctx[-1] = 0xFFFFFFF0
    fits = ctx + rows <= max_ctx
    history = r.integers(100, 200, (n, max_ctx))
    cb, hb = up(u32(ctx))[0], up(u32(history))[0]
    path, count, nxt, after = DeviceBuffer(4 * n * t), DeviceBuffer(4 * n), DeviceBuffer(4 * n), DeviceBuffer(4 * n)
    ops.tree_accept(up(u32(tokens))[0], up(parents)[0], up(u32(picked))[0], n, t, path, count, nxt, cb, after, hb, max_ctx,
                    max_ctx=max_ctx)
    path, count, nxt = down(path, np.uint32, n * t).reshape(n, t), down(count, np.uint32, n), down(nxt, np.uint32, n)
    after, hist = down(after, np.uint32, n), down(hb, np.uint32, n * max_ctx).reshape(n, -1)
    for s in range(n):
        want, last = _tree.accept(tokens[s], parents[s], picked[s]) if fits[s] else ([], NO)
        assert count[s] == len(want) and nxt[s] == last, s
        assert list(path[s, :len(want)]) == want and (path[s, len(want):] == NO).all(), s
        assert after[s] == ctx[s] + len(want)
        h = history[s].copy()
        if want:
            h[ctx[s]:ctx[s] + len(want)] = tokens[s, want]
        assert np.array_equal(hist[s], h), s


@pytest.mark.parametrize("name", ["q4_0", "mixed"])
def test_a_captured_run_into_a_full_cache(gpu, name):
    """Trees of five nodes in a step captured for nine, until the cache is full: every row up to the last is used, then a
    step changes nothing, neither lengths, history nor caches, and a smaller tree goes on."""
    print(f"[case] full cache {name}", flush=True)
    vocab, nt, max_ctx = 300, 9, 37
    m = Model(*MODELS[name], layers=2, vocab=vocab, ctx=max_ctx, seed=3)
    stream = Stream()
    tok_b, par_b, ctx_b = DeviceBuffer(4 * nt), DeviceBuffer(4 * nt), up(np.array([0], np.uint32))[0]
    wsz = m.tree.tree_workspace_bytes(nt)
    x, lg, ws = DeviceBuffer(4 * nt * m.hidden), DeviceBuffer(4 * nt * vocab), DeviceBuffer(wsz)
    picked, path, count, nxt = DeviceBuffer(4 * nt), DeviceBuffer(4 * nt), DeviceBuffer(4), DeviceBuffer(4)
    hist = DeviceBuffer(4 * max_ctx)
    hist.fill(0xFF)
    rules = ops.LogitsRules(rows_per_seq=nt, tree_tokens=tok_b, tree_parents=par_b)
    lws = ops.logits_process_workspace_bytes(rules, nt, vocab)
    lwb, caches = DeviceBuffer(lws), m.tree.kv_caches()
    synchronize()
    with Graph.capture(stream) as replay:
        m.tree.forward_tree(tok_b, par_b, nt, ctx_b, x, lg, ws, wsz, stream)
        ops.logits_process(rules, lg, vocab, nt, vocab, None, 0, picked, lwb, lws, stream)
        ops.tree_accept(tok_b, par_b, picked, 1, nt, path, count, nxt, ctx_b, ctx_b, hist, max_ctx, stream, max_ctx=max_ctx)
        ops.kv_cache_compact(caches, 1, max_ctx, m.kv, m.d, path, nt, count, ctx_b, stream)

    def step(tokens, parents):
        pad = nt - len(tokens)
        tok_b.upload(np.array(list(tokens) + [0] * pad, np.uint32))
        par_b.upload(np.array(list(parents) + [-2] * pad, np.int32))
        replay.launch(stream)
        stream.synchronize()
        return (int(down(count, np.uint32, 1)[0]), int(down(nxt, np.uint32, 1)[0]), int(down(ctx_b, np.uint32, 1)[0]))

    state = lambda: [down(hist, np.uint32, max_ctx)] + m.rows(1, max_ctx)
    said, token, length = [], 7, 0
    for _ in range(3 * max_ctx):
        # what the decode step goes on with, one token drafted right and others wrong
        want = int(np.argmax(m.step(token, length))) if length < max_ctx else 5
        five = [token, want, (want + 1) % vocab, (want + 2) % vocab, (want + 3) % vocab]
        before = state()
        if length + 5 <= max_ctx:
            n, nxt_tok, length_now = step(five, [-1, 0, 0, 0, 1])
            assert n >= 2 and length_now == length + n
            said += [token, want][:n]
            m.step(want, length + 1)
        else:
            n, nxt_tok, length_now = step(five, [-1, 0, 0, 0, 1])
            assert (n, nxt_tok, length_now) == (0, NO, length), "does not fit"
            for a, b in zip(before, state()):
                assert np.array_equal(a, b)
            if length == max_ctx:
                break
            n, nxt_tok, length_now = step([token], [-1])
            assert n == 1 and nxt_tok == want and length_now == length + 1
            said.append(token)
        if n > 2:
            said.append(five[4])
            m.step(five[4], length + 2)
        token, length = nxt_tok, length_now
        assert list(down(hist, np.uint32, max_ctx)[:length]) == said
    assert length == max_ctx
    for a, b in zip(m.rows(0, max_ctx), m.rows(1, max_ctx)):
        step16 = np.spacing(np.abs(a).astype(np.float16)).astype(np.float64)
        assert (np.abs(a - b) <= 2 * step16 + 1e-3 * np.abs(a).max()).all()
    replay.destroy()
    stream.destroy()
