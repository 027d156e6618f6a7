"""wh_beam_select and wh_beam_reorder against their definitions."""
import numpy as np
import pytest

from tests import _members
from tests._gpu import down, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer, Graph, Stream

pytestmark = pytest.mark.gpu
NO = _members.NO_TOKEN
u32 = lambda a: np.asarray(a).astype(np.uint32)
# log-probabilities and scores are f32 at the end; lse in 64 bits but for terms that together make little of it
SCORE = 2.0 ** -23


def run(logits, scores, n_out=None, last=None, end=NO, alpha=0.0, counts=None, history=None, len_=None, pad=0, offset=0,
        in_place=False, vocab=None):
    n, b, v = logits.shape
    vocab = vocab or v
    k = n_out or b
    wide = np.full((n * b, v + pad), np.nan, np.float32)
    wide[:, :v] = logits.reshape(n * b, v)
    lb, lp = up(wide, offset=4 * offset)
    opt = lambda a: up(u32(a))[0] if a is not None else None
    sb, last_b, counts_b, hist_b, len_b = up(scores.astype(np.float32))[0], opt(last), opt(counts), opt(history), opt(len_)
    outs = [DeviceBuffer(4 * n * k) for _ in range(5)]
    for o in outs:
        o.fill(0xEE)
    if in_place:
        outs[0], outs[1], outs[3], outs[4] = sb, last_b or outs[1], counts_b or outs[3], len_b or outs[4]
    rules = ops.BeamRules(b, 0 if k == b else k, end, alpha, last_tokens=last_b, counts=counts_b, counts_out=outs[3], history=hist_b,
                          history_stride=history.shape[2] if history is not None else 0, len=len_b,
                          len_out=outs[4] if len_ is not None else None)
    need = ops.beam_select_workspace_bytes(rules, n, vocab)
    ws = DeviceBuffer(need + 64)
    ws.fill(0xFF)
    ops.beam_select(rules, lp, v + pad, n, vocab, sb, outs[0], outs[1], outs[2], ws, need)
    assert (down(ws, np.uint8, 64, need) == 0xFF).all()
    get = lambda x, t=np.uint32: down(x, t, n * k).reshape(n, k)
    return dict(scores=get(outs[0], np.float32), tokens=get(outs[1]), parents=get(outs[2]), counts=get(outs[3]),
                len=get(outs[4]) if len_ is not None else None,
                history=down(hist_b, np.uint32, history.size).reshape(history.shape) if history is not None else None)


def check(got, want):
    s, t, p, c = want
    assert np.array_equal(got["tokens"], t) and np.array_equal(got["parents"], p) and np.array_equal(got["counts"], c)
    same = got["scores"] == s
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(got["scores"] - s) <= np.abs(s) * SCORE + 2.0 ** -22)).all(), np.abs(got["scores"] - s).max()


@pytest.mark.parametrize("vocab", [1, 2, 63, 65, 511, 513, 8191, 8192, 8193, 20000, 128256])
@pytest.mark.parametrize("beams, n_out", [(1, 1), (1, 5), (4, 4), (5, 10), (8, 8), (32, 64)])
def test_sizes(gpu, vocab, beams, n_out):
    print(f"[case] select vocab {vocab} beams {beams} out {n_out}", flush=True)
    n = 1 if vocab > 10000 else 3
    r = np.random.default_rng([vocab, beams, n_out])
    logits = (r.standard_normal((n, beams, vocab)) * 3).astype(np.float32)
    scores = -(r.random((n, beams)) * 4 + 10).astype(np.float32)
    for pad, offset in ((0, 0), (3, 1)):
        got = run(logits, scores, n_out, pad=pad, offset=offset)
        check(got, _members.select_all(logits, scores, n_out))


@pytest.mark.parametrize("vocab", [7, 3000, 40000])
@pytest.mark.parametrize("beams", [1, 4, 9])
def test_equal_logits(gpu, vocab, beams):
    """Constant rows, rows of few values, and beams that are alike: the lowest beam, then the lowest token."""
    print(f"[case] select ties {vocab} {beams}", flush=True)
    r = np.random.default_rng(vocab + beams)
    scores = np.full((2, beams), -3.0, np.float32)
    for logits in (np.zeros((2, beams, vocab)), r.integers(-1, 2, (2, beams, vocab)) * 1.0,
                   np.where(r.random((2, beams, vocab)) < 0.5, 0.0, -0.0),
                   np.repeat((r.standard_normal((2, 1, vocab)) * 3).round(1), beams, 1)):
        logits = logits.astype(np.float32)
        for n_out in (beams, 2 * beams, 64):
            check(run(logits, scores, n_out), _members.select_all(logits, scores, n_out))


def test_sorted_rows(gpu):
    """The highest logits next to each other, at either end."""
    for sign in (1, -1):
        logits = (sign * np.arange(50000, dtype=np.float32) * 1e-3)[None, None].repeat(3, 1)
        scores = np.array([[-1, -1.0005, -1.5]], np.float32)
        for n_out in (3, 64):
            check(run(logits, scores, n_out), _members.select_all(logits, scores, n_out))


def test_what_is_not_allowed(gpu):
    """-inf and NaN logits, rows without any token, +inf, beams that are not there; fewer continuations than wanted."""
    r = np.random.default_rng(5)
    v, b = 9000, 6
    logits = (r.standard_normal((4, b, v)) * 2).astype(np.float32)
    logits[0][r.random((b, v)) < 0.7] = -np.inf
    logits[0, 1, :100] = np.nan
    logits[0, 2] = -np.inf
    logits[0, 3, 77] = np.inf
    logits[0, 4] = np.nan
    logits[1] = -np.inf
    logits[1, 0, [5, 8888]] = 1.0, 2.0
    logits[1, 4, 3] = -40.0
    scores = -(r.random((4, b)) * 2).astype(np.float32)
    scores[2] = -np.inf, np.nan, -1, np.inf, -np.inf, -2
    scores[3] = -np.inf
    for n_out in (b, 12):
        got = run(logits, scores, n_out)
        check(got, _members.select_all(logits, scores, n_out))
        assert (got["tokens"][3] == NO).all() and np.isneginf(got["scores"][3]).all()
    assert list(got["tokens"][1][:3]) == [8888, 5, 3] or list(got["tokens"][1][:3]) == [3, 8888, 5]


@pytest.mark.parametrize("alpha", [0.0, 0.7, 2.0, -0.5])
@pytest.mark.parametrize("in_place", [False, True])
def test_ended_beams_and_histories(gpu, alpha, in_place):
    print(f"[case] select ended {alpha} {in_place}", flush=True)
    r = np.random.default_rng(9)
    n, b, v, stride, end = 5, 7, 5000, 90, 42
    logits = (r.standard_normal((n, b, v)) * 4).astype(np.float32)
    scores = -(r.random((n, b)) * 3 + 1).astype(np.float32)
    last = r.integers(0, v, (n, b))
    last[r.random((n, b)) < 0.4] = end
    last[4] = end
    counts = r.integers(0, 60, (n, b))
    history, len_ = r.integers(0, v, (n, b, stride)), r.integers(0, 88, (n, b))
    len_[0] = [0, 1, 89, 90, 91, 500, 30]  # some beyond the history's end
    logits[last == end] = np.nan  # not read
    got = run(logits, scores, None, last, end, alpha, counts, history, len_, in_place=in_place)
    want = _members.select_all(np.where(np.isnan(logits), 0, logits), scores, b, last, end, alpha, counts)
    check(got, want)
    assert (got["counts"][4] == np.take_along_axis(counts, got["parents"].astype(int), 1)[4]).all()
    assert np.array_equal(got["len"], np.take_along_axis(len_, want[2], 1) + 1)
    assert np.array_equal(got["history"], _members.histories(history, len_, want[2], want[1]))


def test_long_histories_of_many_beams(gpu):
    r = np.random.default_rng(10)
    n, b, v, stride = 2, 32, 600, 3001
    logits = (r.standard_normal((n, b, v)) * 3).astype(np.float32)
    scores = -(r.random((n, b)) * 3).astype(np.float32)
    history, len_ = r.integers(0, v, (n, b, stride)), np.full((n, b), 2990)
    got = run(logits, scores, None, history=history, len_=len_)
    want = _members.select_all(logits, scores, b)
    check(got, want)
    assert np.array_equal(got["history"], _members.histories(history, len_, want[2], want[1]))


@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 11, 16, 17, 32])
@pytest.mark.parametrize("row_bytes", [4, 36, 16, 1024])
def test_reorder(gpu, beams, row_bytes):
    print(f"[case] reorder {beams} {row_bytes}", flush=True)
    r = np.random.default_rng([beams, row_bytes])
    n, room, states = 3, 50, 5
    arrays = r.integers(0, 1 << 32, (states, n, beams, room, row_bytes // 4), dtype=np.uint64).astype(np.uint32)
    bufs = [up(a)[0] for a in arrays]
    for pending in (0, 1, 7):
        parents = r.integers(0, beams, (n, beams))
        parents[0] = (np.arange(beams) + 1) % beams  # a ring
        len_ = r.integers(0, room + 1, (n, beams))
        len_[1, 0], len_[2, -1] = room + pending, room + pending + 1  # all rows; more than there are: stays
        parents[2, 0] = beams
        ops.beam_reorder(ops.BeamStates(bufs), n, beams, room, row_bytes, up(u32(parents))[0], up(u32(len_))[0], pending)
        arrays = np.stack([_members.reorder(a, parents, len_, pending) for a in arrays])
        for b, a in zip(bufs, arrays):
            assert np.array_equal(down(b, np.uint32, a.size).reshape(a.shape), a)


def test_reorder_many_states(gpu):
    """More states than one launch takes, in one allocation, next to each other."""
    r = np.random.default_rng(2)
    n_states, b, room, words = 300, 3, 9, 8
    a = r.integers(0, 1 << 31, (n_states, 1, b, room, words)).astype(np.uint32)
    buf = up(a)[0]
    step = a[0].nbytes
    parents, len_ = np.array([[2, 2, 0]]), np.array([[9, 4, 6]])
    ops.beam_reorder(ops.BeamStates([buf.ptr + i * step for i in range(n_states)]), 1, b, room, 4 * words, up(u32(parents))[0],
                     up(u32(len_))[0], 0)
    want = np.stack([_members.reorder(x, parents, len_, 0) for x in a])
    assert np.array_equal(down(buf, np.uint32, a.size).reshape(a.shape), want)


def test_graph(gpu):
    """Both calls captured, everything in place, replayed step by step."""
    r = np.random.default_rng(3)
    n, b, v, stride = 2, 4, 10000, 30
    s = Stream()
    logits = DeviceBuffer(4 * n * b * v)
    scores, tokens, parents, counts, len_b = (DeviceBuffer(4 * n * b) for _ in range(5))
    hist, rows = DeviceBuffer(4 * n * b * stride), DeviceBuffer(16 * n * b * stride)
    end = 7
    rules = ops.BeamRules(b, 0, end, 0.6, last_tokens=tokens, counts=counts, counts_out=counts, history=hist, history_stride=stride,
                          len=len_b, len_out=len_b)
    need = ops.beam_select_workspace_bytes(rules, n, v)
    ws, states = DeviceBuffer(need), ops.BeamStates([rows])
    with Graph.capture(s) as g:
        ops.beam_select(rules, logits, v, n, v, scores, scores, tokens, parents, ws, need, s)
        ops.beam_reorder(states, n, b, stride, 16, parents, len_b, 1, s)
    hs = dict(scores=np.full((n, b), -np.inf, np.float32), tokens=np.full((n, b), 1), counts=np.zeros((n, b), int),
              len=np.zeros((n, b), int), hist=r.integers(0, 9, (n, b, stride)), rows=r.integers(0, 99, (n, b, stride, 4)).astype(np.uint32))
    hs["scores"][:, 0] = 0  # a search begins with one beam
    for buf, name in ((scores, "scores"), (tokens, "tokens"), (counts, "counts"), (len_b, "len"), (hist, "hist"), (rows, "rows")):
        a = hs[name]
        buf.upload(a if a.dtype == np.float32 else u32(a))
    for step in range(12):
        x = (r.standard_normal((n, b, v)) * 3).astype(np.float32)
        x[:, :, end] += 7.0
        logits.upload(x)
        g.launch(s)
        s.synchronize()
        want = _members.select_all(x, hs["scores"], b, hs["tokens"], end, 0.6, hs["counts"])
        hs["hist"] = _members.histories(hs["hist"], hs["len"], want[2], want[1])
        hs["len"] = np.take_along_axis(hs["len"], want[2], 1) + 1
        hs["rows"] = _members.reorder(hs["rows"], want[2], hs["len"], 1)
        got = down(scores, np.float32, n * b).reshape(n, b)
        assert (np.abs(got - want[0]) <= np.abs(want[0]) * SCORE + 2.0 ** -22).all()
        hs["scores"], hs["tokens"], hs["counts"] = got, want[1], want[3]
        for buf, name in ((tokens, "tokens"), (counts, "counts"), (len_b, "len"), (hist, "hist"), (rows, "rows")):
            assert np.array_equal(down(buf, np.uint32, hs[name].size), u32(hs[name]).ravel()), (step, name)
    assert (hs["tokens"] == end).any()
