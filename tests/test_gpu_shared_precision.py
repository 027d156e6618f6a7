"""wh_attention_shared: the precision of its rows together, in every form of the kernel and at the lengths where weights far
below the largest make the output."""
import numpy as np
import pytest

from tests import _shared
from tests.test_gpu_shared_attention import Case

pytestmark = pytest.mark.gpu

# heads, kv, d, members, prefix rows, max_own: 32 query rows to a workgroup in chunks of 128 keys and of more than 1000 (5
# tiles of 32 rows), 64 and 128 to a workgroup in chunks of 750 to 7500
FORMS = [(4, 1, 64, 4, 40, 20), (4, 1, 128, 4, 3000, 20), (64, 32, 128, 72, 4000, 3), (64, 32, 64, 72, 5000, 3),
         (64, 32, 128, 16, 6000, 4), (8, 1, 128, 200, 20000, 1300), (8, 1, 128, 1000, 60000, 3), (8, 1, 64, 1000, 60000, 3)]


def alike(heads, kv, d, per, n, max_own, share, at, seed=0, spread=1.3):
    """A case whose query rows of a KV head are u, -u and 0 by turns of the members, so that a key that has `share` of the
    weight for u has next to none for -u; two own rows each."""
    c = Case(heads, kv, d, per, [n], [2] * per, max_own=max_own, seed=seed)
    r = np.random.default_rng([seed, n])
    u = (r.standard_normal((kv, d)) * spread).astype(np.float32)
    sign = np.array([1, -1, 1, 0])[np.arange(per) % 4].astype(np.float32)
    c.q[:, :heads * d] = (sign[:, None, None, None] * u[None, :, None]).repeat(heads // kv, 2).reshape(per, -1)
    for j in range(kv):
        _shared.add_sink(u[j], c.kp[0, :, j], c.vp[0, :, j], share, at)
    return c


def check(c, members, what):
    got = c.out().astype(np.float64)
    for m in members:
        g = m // c.per
        k = np.concatenate([c.kp[g, :c.prefix[g]], c.ko[m, :c.own[m]]])
        v = np.concatenate([c.vp[g, :c.prefix[g]], c.vo[m, :c.own[m]]])
        want, top = _shared.exact(c.q[m, :c.heads * c.d].reshape(c.heads, c.d), k, v)
        err, bar = _shared.rel(got[m], want), _shared.bar(top)
        print(f"[result] {what}, member {m}: {err:.2e}, bar {bar:.2e}", flush=True)
        assert err <= bar, (what, m, err, bar)


@pytest.mark.parametrize("heads, kv, d, per, n, max_own", FORMS)
@pytest.mark.parametrize("share", [0.9, 0.999999, 1 - 1e-9])
def test_one_key_with_nearly_all_the_weight(gpu, heads, kv, d, per, n, max_own, share):
    """The others carry the output, and keep the precision that f32 weights have; the sink at the start, in the middle and at
    the end of a chunk."""
    for at in (0, n // 2 + 3, n - 1)[:2 if kv * n > 50000 else 3]:
        c = alike(heads, kv, d, per, n, max_own, share, at)
        print(f"[case] shared sink {share} at {at}, {heads}/{kv}x{d} {per} members at {n}", flush=True)
        c.upload().call()
        check(c, [0, 1, 3, per - 2], f"{share} of the weight on key {at}, {heads}/{kv}x{d} {per} members at {n}")


@pytest.mark.parametrize("share", [0.9, 0.999999, 1 - 1e-9])
@pytest.mark.parametrize("heads, kv, d, per, own", [(8, 2, 128, 3, 900), (8, 1, 64, 260, 1500), (40, 1, 64, 260, 300)])
def test_one_own_key_with_nearly_all_the_weight(gpu, heads, kv, d, per, own, share):
    """The same among a member's own rows."""
    c = Case(heads, kv, d, per, [50], [own] * per)
    q = c.q.reshape(per, kv, heads // kv, d)
    q[:] = q[:, :, :1]
    for m in range(per):
        for j in range(kv):
            _shared.add_sink(q[m, j, 0], c.ko[m, :, j], c.vo[m, :, j], share, m * 7 % own)
    print(f"[case] shared own sink {share}, {heads}/{kv}x{d} {per} members of {own} rows", flush=True)
    c.upload().call()
    check(c, sorted({0, 1, 2, per // 2, per - 1}), f"{share} of the weight on an own key, {heads}/{kv}x{d} {per} members of {own}")


@pytest.mark.parametrize("heads, kv, d, per, n, max_own", FORMS[1:])
@pytest.mark.parametrize("spread", [3.0, 8.0, 30.0])
def test_scores_far_apart(gpu, heads, kv, d, per, n, max_own, spread):
    """Scores whose standard deviation is 3, 8 and 30: weights of every size, references that move up and down."""
    c = alike(heads, kv, d, per, min(n, 20000), max_own, 0, 0, seed=3, spread=spread)
    print(f"[case] shared spread {spread}, {heads}/{kv}x{d} {per} members at {n}", flush=True)
    c.upload().call()
    check(c, [0, 1, 3, per - 2], f"scores of spread {spread}, {heads}/{kv}x{d} {per} members at {n}")


@pytest.mark.parametrize("heads, kv, d, per, n, max_own", FORMS)
def test_errors_are_those_of_f32(gpu, heads, kv, d, per, n, max_own):
    """Over a member's rows together the roundings are random: far below the bound of a single one, which a lost limb of the
    queries or the weights would keep."""
    c = Case(heads, kv, d, per, [n], [2] * per, max_own=max_own, seed=9)
    c.upload().call()
    check(c, sorted({0, 1, per // 2, per - 1}), f"{heads}/{kv}x{d} {per} members at {n}")
