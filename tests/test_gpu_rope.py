"""wh_qk_norm_rope against 64 bits."""
import numpy as np
import pytest

from tests import _members
from tests._gpu import down, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu
u32 = lambda a: np.asarray(a).astype(np.uint32)


def case(groups=1, per=3, new=1, heads=8, kv=2, d=128, rot=0, inter=False, magnitude=1.0, q_norm=False, k_norm=False, base=1000,
         lens=None, room=40, pad=0, offset=0, in_place=False, no_base=False, no_len=False, seed=0, base_lens=None):
    r = np.random.default_rng([seed, groups, per, new, heads, d])
    n = groups * per
    rot_dim = rot or d
    lens = np.array(lens if lens is not None else r.integers(new, room + 1, n))
    base_lens = np.zeros(groups, int) if no_base else np.array(base_lens if base_lens is not None else r.integers(0, base + 1, groups))
    if no_len:
        lens[:] = new
    width = (heads + 2 * kv) * d + pad
    rows = r.standard_normal((n * new, width)).astype(np.float32) * 1.5
    inv = (1.0 / 10000.0 ** (np.arange(0, rot_dim, 2) / rot_dim)).astype(np.float32)
    qw, kw = (1 + 0.3 * r.standard_normal((2, d))).astype(np.float32)
    # buffers at an odd element, so that no address is a multiple of 8 by itself
    xb, x = up(rows, offset=4 * offset)
    cache = r.integers(0, 1 << 16, (2, n, room, kv, d), dtype=np.uint16)  # what is not written stays, whatever it is
    caches = [up(c)[0] for c in cache]
    qwb, kwb, invb = up(qw)[0], up(kw)[0], up(inv)[0]
    rules = ops.RopeRules(invb, rot, inter, magnitude, qwb if q_norm else None, kwb if k_norm else None, 1e-6)
    q, k, v = x, x + 4 * heads * d, x + 4 * (heads + kv) * d
    ldo = width if in_place else heads * d + 3
    qo, ko = (None, None) if in_place else (DeviceBuffer(4 * n * new * ldo), DeviceBuffer(4 * n * new * (kv * d + 1)))
    for b in (qo, ko):
        if b:
            b.fill(0xEE)
    lenb, baseb = up(u32(lens))[0], up(u32(base_lens))[0]
    ops.qk_norm_rope(rules, q, k, v, width, width, None if no_base else baseb, None if no_len else lenb, groups, per, new, heads, kv,
                     d, q if in_place else qo, ldo, k if in_place else ko, width if in_place else kv * d + 1, caches[0], caches[1], room)
    if in_place:
        got = down(xb, np.float32, rows.size, 4 * offset).reshape(rows.shape)
        gq, gk = got[:, :heads * d], got[:, heads * d:(heads + kv) * d]
        assert np.array_equal(got[:, (heads + kv) * d:], rows[:, (heads + kv) * d:])
    else:
        gq = down(qo, np.float32, n * new * ldo).reshape(-1, ldo)
        assert (gq[:, heads * d:].view(np.uint32) == 0xEEEEEEEE).all()
        gq = gq[:, :heads * d]
        gk = down(ko, np.float32, n * new * (kv * d + 1)).reshape(-1, kv * d + 1)[:, :kv * d]
    index = (lens[:, None] - new + np.arange(new)).reshape(-1)
    pos = np.maximum(index, 0) + np.repeat(base_lens, per * new)
    want_q, bound_q = _members.rope(rows[:, :heads * d].reshape(-1, heads, d), pos, inv, rot_dim, inter, magnitude or 1.0,
                                    qw if q_norm else None, 1e-6)
    want_k, bound_k = _members.rope(rows[:, heads * d:(heads + kv) * d].reshape(-1, kv, d), pos, inv, rot_dim, inter, magnitude or 1.0,
                                    kw if k_norm else None, 1e-6)
    vals = rows[:, (heads + kv) * d:(heads + 2 * kv) * d].reshape(-1, kv, d)
    have = [down(c, np.float16, cache[0].size).reshape(cache[0].shape) for c in caches]
    expect = cache.copy()
    gq, gk = gq.reshape(-1, heads, d), gk.reshape(-1, kv, d)
    for row, i in enumerate(index):
        m = row // new
        if i < 0:
            assert not gq[row].any() and not gk[row].any(), row
            continue
        if i >= room:
            assert np.isnan(gq[row]).all(), row
        else:
            assert (np.abs(gq[row] - want_q[row]) <= bound_q[row]).all(), (row, np.abs(gq[row] - want_q[row]).max())
            expect[1, m, i] = vals[row].astype(np.float16).view(np.uint16)
            err = np.abs(have[0][m, i].astype(np.float64) - want_k[row])
            assert (err <= bound_k[row] + np.abs(want_k[row]) * 2.0 ** -11 * (1 + 2.0 ** -10) + 2.0 ** -25).all(), (row, err.max())
            if pos.max() < 10 ** 6:  # in 64 bits, the norm too: the row is the formula's
                far = have[0][m, i] != _members.stored(want_k[row])
                assert far.mean() <= 2.0 ** -9, far.mean()  # but for sums that lie on the border of two f32
            expect[0, m, i] = have[0][m, i].view(np.uint16)
        assert (np.abs(gk[row] - want_k[row]) <= bound_k[row]).all(), row
    assert np.array_equal(np.stack(have).view(np.uint16), expect), "rows that no token has, and V"


@pytest.mark.parametrize("d", [2, 6, 64, 80, 96, 126, 128, 130, 192, 256])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_head_sizes_and_parts(gpu, d, inter, norm):
    for rot in sorted({0, 2, d // 2 & ~1, d - 2 & ~1} - {0} | {0}):
        print(f"[case] rope d {d} rot {rot} inter {inter} norm {norm}", flush=True)
        case(d=d, rot=rot, inter=inter, q_norm=norm, k_norm=norm, magnitude=1.25, seed=rot)


@pytest.mark.parametrize("heads, kv", [(1, 1), (2, 1), (7, 7), (32, 8), (40, 5), (3, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_heads(gpu, heads, kv, d):
    print(f"[case] rope heads {heads} kv {kv} d {d}", flush=True)
    case(heads=heads, kv=kv, d=d, q_norm=True, per=5)
    case(heads=heads, kv=kv, d=d, k_norm=True, per=2, groups=3, pad=5, offset=1)


@pytest.mark.parametrize("d", [64, 128, 192])
def test_prompts_of_mixed_lengths(gpu, d):
    """Absent tokens in front, tokens behind the cache's end, and enough rows for the many-heads form."""
    print(f"[case] rope prompts d {d}", flush=True)
    case(groups=3, per=2, new=37, lens=[0, 1, 36, 37, 41, 60], room=45, d=d, inter=True, rot=d // 2, pad=1)
    case(groups=1, per=5, new=900, lens=[0, 1, 899, 900, 1001], room=950, heads=9, kv=3, d=d, k_norm=True, q_norm=True)


def test_in_place_and_defaults(gpu):
    case(in_place=True, pad=7, offset=1, q_norm=True, k_norm=True)
    case(in_place=True, new=600, room=700, heads=10, kv=5)  # many heads
    case(no_base=True, no_len=True, new=5)
    case(magnitude=0.0)  # counts as 1

def test_far_positions(gpu):
    case(base_lens=[2 ** 31], per=4)
    case(base_lens=[131072], per=4, inter=True)


def test_values_apart(gpu):
    """Infinities and NaN stay in their pair; the part that does not turn is passed on as it is."""
    d, heads, kv = 64, 4, 2
    x = np.ones((1, (heads + 2 * kv) * d), np.float32)
    x[0, 20] = np.inf              # head 0, not turned
    x[0, d + 40] = np.nan          # head 1, not turned
    x[0, 2 * d + 13] = np.inf      # head 2, turned with 5
    x[0, heads * d + 3] = -np.inf  # key head 0, turned with 11
    inv = np.linspace(0, 0.7, 8).astype(np.float32)
    xb, invb, out = up(x)[0], up(inv)[0], DeviceBuffer(4 * heads * d)
    caches = [DeviceBuffer(2 * kv * d) for _ in range(2)]
    ops.qk_norm_rope(ops.RopeRules(invb, 16), xb, xb.ptr + 4 * heads * d, xb.ptr + 4 * (heads + kv) * d, x.shape[1], x.shape[1],
                     None, None, 1, 1, 1, heads, kv, d, out, heads * d, None, 0, caches[0], caches[1], 1)
    q = down(out, np.float32, heads * d).reshape(heads, d)
    assert q[0, 20] == np.inf and np.isfinite(np.delete(q[0], 20)).all()
    assert np.isnan(q[1, 40]) and np.isfinite(np.delete(q[1], 40)).all()
    assert not np.isfinite(q[2, [5, 13]]).any() and np.isfinite(np.delete(q[2], [5, 13])).all()
    assert np.isfinite(q[3]).all() and (q[3, 16:] == 1).all()
    k = down(caches[0], np.float16, kv * d).reshape(kv, d)
    assert not np.isfinite(k[0, 3]) and np.isfinite(np.delete(k[0], [3, 11])).all()
    assert (down(caches[1], np.float16, kv * d) == 1).all()


def test_norms_of_tiny_heads(gpu):
    """Heads whose mean square is no normal f32 number, and heads of zeros, without an epsilon.

    Squares of 1e-19 are off by 2^-150, 7e-8 of them, as is each of the sum's steps in f32: with the other roundings of the
    norm and the turn under 2^-19 of the pair.  Keys are normed in 64 bits."""
    d, heads, kv = 64, 3, 2
    x = np.full((1, (heads + 2 * kv) * d), 1e-19, np.float32) * np.tile([1, -1], (heads + 2 * kv) * d // 2).astype(np.float32)
    x[0, d:2 * d] = 0            # query head 1
    x[0, heads * d:heads * d + d] = 0  # key head 0
    inv, w = np.linspace(0.1, 0.7, d // 2).astype(np.float32), np.linspace(0.5, 1.5, d).astype(np.float32)
    xb, invb, wb, out, kout = up(x)[0], up(inv)[0], up(w)[0], DeviceBuffer(4 * heads * d), DeviceBuffer(4 * kv * d)
    for eps in (0.0, 1e-6):
        rules = ops.RopeRules(invb, 0, False, 1.0, wb, wb, eps)
        ops.qk_norm_rope(rules, xb, xb.ptr + 4 * heads * d, xb.ptr + 4 * (heads + kv) * d, x.shape[1], x.shape[1], None, None, 1, 1, 1,
                         heads, kv, d, out, heads * d, kout, kv * d, None, None, 0)
        with np.errstate(invalid="ignore"):
            want_q, _ = _members.rope(x[:, :heads * d].reshape(1, heads, d), np.array([0]), inv, d, False, 1.0, w, eps)
            want_k, _ = _members.rope(x[:, heads * d:(heads + kv) * d].reshape(1, kv, d), np.array([0]), inv, d, False, 1.0, w, eps)
        q, k = down(out, np.float32, heads * d).reshape(heads, d), down(kout, np.float32, kv * d).reshape(kv, d)
        for got, want, bar in ((q, want_q[0], 2.0 ** -19), (k, want_k[0], 2.0 ** -23)):
            assert np.array_equal(np.isnan(got), np.isnan(want)), eps
            assert (np.abs(got - want) <= bar * np.abs(want))[~np.isnan(want)].all(), eps


def test_outputs_that_are_not_wanted(gpu):
    """Each output by itself is what it is beside the others."""
    heads, kv, d, n, room = 6, 2, 96, 5, 4
    width = (heads + 2 * kv) * d
    x = np.random.default_rng(0).standard_normal((n, width)).astype(np.float32)
    xb, inv = up(x)[0], up(np.linspace(0.1, 0.9, d // 2).astype(np.float32))[0]
    base, lens = up(u32([7]))[0], up(u32([1, 4, 2, 5, 0]))[0]  # one that does not fit, one that is absent
    sizes = (4 * n * heads * d, 4 * n * kv * d, 2 * n * room * kv * d, 2 * n * room * kv * d)

    def call(q, k, cache):
        bufs = [DeviceBuffer(s) for s in sizes]
        for b in bufs:
            b.fill(0xEE)
        ops.qk_norm_rope(ops.RopeRules(inv), xb, xb.ptr + 4 * heads * d, xb.ptr + 4 * (heads + kv) * d, width, width, base, lens, 1, n, 1,
                         heads, kv, d, bufs[0] if q else None, heads * d, bufs[1] if k else None, kv * d, bufs[2] if cache else None,
                         bufs[3] if cache else None, room if cache else 0)
        return [down(b, np.uint8, s) for b, s in zip(bufs, sizes)]

    every, without = call(True, True, True), call(True, True, False)
    untouched = [np.full(s, 0xEE, np.uint8) for s in sizes]
    for want in (dict(q=True, k=False, cache=True), dict(q=False, k=True, cache=True), dict(q=False, k=False, cache=True),
                 dict(q=True, k=False, cache=False), dict(q=False, k=True, cache=False), dict(q=False, k=False, cache=False)):
        got = call(**want)
        have = (want["q"], want["k"], want["cache"], want["cache"])
        full = every if want["cache"] else without
        for g, f, u, h in zip(got, full, untouched, have):
            assert np.array_equal(g, f if h else u), want
