"""wh_attention_shared: an infinity of V counts with any weight above 0, however small, and is NaN with a weight of 0, in
whichever tile, chunk or part of the rows its key lies."""
import numpy as np
import pytest

from tests import _members
from tests.test_gpu_shared_attention import WIDE, Case

pytestmark = pytest.mark.gpu

# heads, kv, d, members, max_prefix, max_own: few query rows, members whose own rows are in one and in several chunks, many
FORMS = [(4, 1, 64, 3, 900, 400), (4, 1, 128, 3, 900, 400), (40, 1, 128, 2, 300, 500)] + WIDE


@pytest.mark.parametrize("heads, kv, d, per, max_prefix, max_own", FORMS)
@pytest.mark.parametrize("n", [70, 900, 2111])
def test_infinities_of_any_weight(gpu, heads, kv, d, per, max_prefix, max_own, n):
    """Every query row is c u with c from 1 to 60: key `top` is 4 u, far above the others, the keys `far` are -4 u, whose
    weights are e^-8 of it for the first row and e^-480 for the last.  One key is u times -inf."""
    g, own = heads // kv, min(max_own, 300)
    n = min(n, max_prefix)
    r = np.random.default_rng([n, per])
    u = np.where(r.random(d) < 0.5, -1, 1).astype(np.float32)
    for top in (5, n - 1, n + own - 1):
        c = Case(heads, kv, d, per, [n], [own] * per, max_prefix=max_prefix, max_own=max_own, seed=n)
        c.q.reshape(per, heads, d)[:] = np.linspace(1, 60, per * heads).reshape(per, heads)[:, :, None] * u / np.sqrt(d)
        key = lambda i: (c.kp, c.vp, 0, i) if i < n else (c.ko, c.vo, slice(None), i - n)  # of every member, where it is an own one

        def put(i, k, dim, x):
            ka, va, who, row = key(i)
            ka[who, row] = k
            if dim is not None:
                va[who, row, :, dim] = x

        put(top, 4 * u, None, 0)
        far = sorted({0, 33, 64, n // 2, n - 2, n + 1, n + own // 2, n + own - 2} - {top})
        for j, i in enumerate(far):
            put(i, -4 * u, j, np.inf if j % 2 else -np.inf)
        none = n // 3
        put(none, np.where(u > 0, -np.inf, np.inf), 20, np.inf)
        print(f"[case] shared infinities {heads}/{kv}x{d} {per} members at {n}, top {top}", flush=True)
        c.upload().call()
        got = c.out()
        for j in range(len(far)):
            assert (got[:, :, j] == (np.inf if j % 2 else -np.inf)).all(), (top, far[j])
        assert np.isnan(got[:, :, 20]).all(), top
        rest = [i for i in range(d) if i != 20 and i >= len(far)]
        keep = np.delete(np.arange(n), none)
        for m in sorted({0, per // 2, per - 1}):
            want, bound = _members.attention(c.q[m].reshape(heads, d), np.concatenate([c.kp[0, keep], c.ko[m, :own]]),
                                             np.concatenate([c.vp[0, keep], c.vo[m, :own]]))
            assert (np.abs(got[m] - want)[:, rest] <= bound[:, rest]).all(), (top, m)


@pytest.mark.parametrize("d", [64, 128])
def test_no_weight_above_0(gpu, d):
    """Rows whose every score is -inf are 0 / 0; a part of them in which all are has no say but for what 0 makes NaN."""
    for n, own in ((200, 30), (30, 200), (1000, 300)):
        c = Case(2, 1, d, 2, [n], [own, own])
        c.q[:] = np.abs(c.q) + 0.1
        c.kp[:] = -np.inf
        c.vp[0, n // 2, 0, 3] = np.inf
        c.ko[1, :own] = -np.inf
        c.upload().call()
        got = c.out()
        assert np.isnan(got[1]).all()
        assert np.isnan(got[0, :, 3]).all()
        want, bound = _members.attention(c.q[0].reshape(2, d), c.ko[0, :own], c.vo[0, :own])
        rest = [i for i in range(d) if i != 3]
        assert (np.abs(got[0] - want)[:, rest] <= bound[:, rest]).all()
