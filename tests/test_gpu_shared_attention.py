"""wh_attention_shared against 64 bits."""
import numpy as np
import pytest

from tests import _members
from tests._gpu import down, report, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer, Graph, Stream

pytestmark = pytest.mark.gpu
u32 = lambda a: np.asarray(a).astype(np.uint32)


class Case:
    """Inputs on the device; rows behind the lengths are NaN and infinities."""

    def __init__(self, heads, kv, d, per, prefix, own, max_prefix=None, max_own=None, pad=0, offset=0, scale=1.3, seed=0):
        """prefix: a length per group; own: one per member."""
        r = np.random.default_rng([seed, heads, kv, d, per, len(prefix)])
        self.heads, self.kv, self.d, self.per, self.groups = heads, kv, d, per, len(prefix)
        self.n = self.groups * per
        assert len(own) == self.n
        self.prefix, self.own = list(prefix), list(own)
        self.max_prefix = max(prefix) if max_prefix is None else max_prefix
        self.max_own = max(own) if max_own is None else max_own
        self.ldq = heads * d + pad
        self.q = (r.standard_normal((self.n, self.ldq)) * scale).astype(np.float32)
        self.kp, self.vp = (r.standard_normal((self.groups, self.max_prefix, kv, d)).astype(np.float16) for _ in range(2))
        self.ko, self.vo = (r.standard_normal((self.n, self.max_own, kv, d)).astype(np.float16) for _ in range(2))
        for i, l in enumerate(self.prefix):
            self.kp[i, l:], self.vp[i, l:] = np.nan, np.inf
        for i, l in enumerate(self.own):
            self.ko[i, l:], self.vo[i, l:] = np.inf, np.nan
        self.offset = offset

    def upload(self):
        self.qb, self.qp = up(self.q, offset=4 * self.offset)
        self.bufs = [up(a)[0] for a in (self.kp, self.vp, self.ko, self.vo)]
        self.lens = [up(u32(self.prefix))[0], up(u32(self.own))[0]]
        self.outb = DeviceBuffer(4 * (self.n * self.heads * self.d + 2 * self.offset))
        self.outb.fill(0xEE)
        self.need = ops.attention_shared_workspace_bytes(self.groups, self.per, self.heads, self.kv, self.d, self.max_prefix, self.max_own)
        self.ws = DeviceBuffer(self.need + 256)
        self.ws.fill(0xFF)
        return self

    def call(self, stream=None):
        kp, vp, ko, vo = self.bufs
        some = lambda rows, *a: a if rows else (None,) * len(a)
        pl, kp, vp = some(self.max_prefix, self.lens[0], kp, vp)
        ol, ko, vo = some(self.max_own, self.lens[1], ko, vo)
        ops.attention_shared(self.qp, self.ldq, pl, ol, self.groups, self.per, kp, vp, self.max_prefix, ko, vo, self.max_own,
                             self.heads, self.kv, self.d, self.outb.ptr + 4 * self.offset, self.ws, self.need, stream)

    def out(self):
        all_ = down(self.outb, np.float32, self.n * self.heads * self.d + 2 * self.offset)
        assert (all_[:self.offset].view(np.uint32) == 0xEEEEEEEE).all()
        assert (all_[self.offset + self.n * self.heads * self.d:].view(np.uint32) == 0xEEEEEEEE).all()
        assert (down(self.ws, np.uint8, 256, self.need) == 0xFF).all(), "the workspace's end"
        return all_[self.offset:self.offset + self.n * self.heads * self.d].reshape(self.n, self.heads, self.d)

    def member(self, m):
        g = m // self.per
        k = np.concatenate([self.kp[g, :self.prefix[g]], self.ko[m, :self.own[m]]])
        v = np.concatenate([self.vp[g, :self.prefix[g]], self.vo[m, :self.own[m]]])
        return _members.attention(self.q[m, :self.heads * self.d].reshape(self.heads, self.d), k, v)

    def check(self, members=None):
        got, num, den = self.out().astype(np.float64), 0.0, 0.0
        for m in range(self.n) if members is None else members:
            want, bound = self.member(m)
            err = np.abs(got[m] - want)
            assert (err <= bound).all(), (m, self.prefix[m // self.per], self.own[m], err.max(), (err / np.maximum(bound, 1e-300)).max())
            num, den = num + (err ** 2).sum(), den + (want ** 2).sum()
        report(f"shared {self.heads}/{self.kv}x{self.d} {self.groups}x{self.per}", np.sqrt(num / den) if den else 0.0, 0.0)


HEADS = [(4, 4, 64), (8, 2, 64), (40, 1, 64), (32, 8, 128), (14, 2, 128), (33, 1, 128), (6, 6, 128)]


@pytest.mark.parametrize("heads, kv, d", HEADS)
def test_lengths(gpu, heads, kv, d):
    """Groups whose prefixes and members' rows end anywhere, none at all among them."""
    print(f"[case] shared lengths {heads} {kv} {d}", flush=True)
    prefix = [0, 1, 31, 32, 33, 127, 128, 129, 300]
    own = [0, 1, 2, 31, 32, 33, 64, 127, 128, 129, 161, 200, 0, 5, 90, 0, 1, 40]
    c = Case(heads, kv, d, 2, prefix, own, max_prefix=310, max_own=203).upload()
    c.call()
    c.check()
    assert not c.out()[0].any()  # no row at all


@pytest.mark.parametrize("heads, kv, d", [(4, 1, 64), (16, 2, 128)])
@pytest.mark.parametrize("per", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 24, 33, 64, 100])
def test_members(gpu, heads, kv, d, per):
    """One group of any size: tiles of query rows that are full, or nearly empty."""
    print(f"[case] shared members {heads} {kv} {d} {per}", flush=True)
    r = np.random.default_rng(per)
    c = Case(heads, kv, d, per, [777], list(r.integers(0, 70, per)), max_prefix=800, max_own=75, pad=3, offset=1).upload()
    c.call()
    c.check(range(0, per, max(1, per // 9)))


@pytest.mark.parametrize("heads, kv, d", [(8, 2, 64), (16, 2, 128)])
def test_long(gpu, heads, kv, d):
    """Prefixes in many chunks, and own rows in several; caches much larger than what is in them."""
    print(f"[case] shared long {heads} {kv} {d}", flush=True)
    c = Case(heads, kv, d, 3, [9001, 40], [1500, 3, 700, 0, 2111, 64], max_prefix=20000, max_own=5000).upload()
    c.call()
    c.check()
    c = Case(heads, kv, d, 40, [4099], [7] * 40).upload()
    c.call()
    c.check([0, 17, 39])


# heads, kv, d, members, max_prefix, max_own: workgroups of 64 and of 128 query rows, one and two to a CU, the last one's rows
# not all there, and (5 tiles of 32) workgroups of 32 rows, two to a CU
WIDE = [(4, 1, 128, 43, 60000, 400), (4, 1, 128, 43, 96000, 20), (4, 1, 128, 52, 50000, 60), (8, 2, 128, 60, 120000, 30),
        (4, 1, 128, 39, 140000, 20), (8, 1, 64, 52, 64000, 30), (8, 1, 64, 23, 50000, 20)]


@pytest.mark.parametrize("heads, kv, d, per, max_prefix, max_own", WIDE)
def test_many_rows(gpu, heads, kv, d, per, max_prefix, max_own):
    """Members whose query rows share the prefix's stages, at lengths that end anywhere in a stage, none and one."""
    print(f"[case] shared many rows {heads} {kv} {d} {per} {max_prefix}", flush=True)
    r = np.random.default_rng(per)
    for n in (0, 1, 64, 95, 2111, max_prefix):
        own = [int(v) for v in r.integers(0, 20, per)]
        own[0] = 0
        c = Case(heads, kv, d, per, [n], own, max_prefix=max_prefix, max_own=max_own, seed=n).upload()
        c.call()
        c.check([0, 8, 19, per - 1] if n > 3000 else None)


@pytest.mark.parametrize("heads, kv, d, per, max_prefix, max_own", WIDE)
def test_infinities_of_many_rows(gpu, heads, kv, d, per, max_prefix, max_own):
    for n in (75, 1000):
        c = Case(heads, kv, d, per, [n], [2] * per, max_prefix=max_prefix, max_own=max_own)
        c.vp[0, 5, 0, 3] = np.inf
        c.vp[0, 40, 0, 9] = -np.inf
        c.vp[0, n - 1, 0, 11] = np.nan
        c.kp[0, 37, 0] = np.where(c.q[1, :d] > 0, -np.inf, np.inf)  # member 1, head 0: score -inf; any other row's is NaN
        c.upload().call()
        got = c.out()
        assert got[1, 0, 3] == np.inf and np.isneginf(got[1, 0, 9]) and np.isnan(got[1, 0, 11])
        g = heads // kv
        others = [(m, h) for m in range(per) for h in range(g) if (m, h) != (1, 0)]
        assert all(np.isnan(got[m, h]).all() for m, h in others)
        rest = [i for i in range(d) if i not in (3, 9, 11)]
        keep = np.delete(np.arange(n), 37)
        want, bound = _members.attention(c.q[1, :d][None], np.concatenate([c.kp[0, keep, :1], c.ko[1, :2, :1]]),
                                         np.concatenate([c.vp[0, keep, :1], c.vo[1, :2, :1]]))
        assert (np.abs(got[1, 0] - want[0])[rest] <= bound[0, rest]).all()


# heads, kv, d, groups, members each, max_prefix: chunks shared by the lengths, in workgroups of 32, 64 and 128 query rows,
# more groups than chunks per group, as many groups as a wave has lanes, and one more
GROUPS = [(8, 2, 64, 7, 3, 24000), (4, 1, 128, 2, 16, 84000), (4, 1, 128, 3, 31, 28000), (8, 1, 64, 33, 2, 10000), (6, 1, 128, 64, 1, 5200),
          (6, 1, 128, 65, 1, 5200), (16, 16, 64, 12, 1, 2000)]


@pytest.mark.parametrize("heads, kv, d, groups, per, max_prefix", GROUPS)
def test_groups_of_any_length(gpu, heads, kv, d, groups, per, max_prefix):
    """Prefixes of equal lengths, of lengths far apart, empty ones among them, and of lengths that do not fit."""
    print(f"[case] shared groups {heads} {kv} {d} {groups} {per} {max_prefix}", flush=True)
    r = np.random.default_rng(groups)
    own = [int(v) for v in r.integers(0, 9, groups * per)]
    c = Case(heads, kv, d, per, [max_prefix] * groups, own, max_prefix=max_prefix).upload()
    some = sorted({0, 1, groups // 2, groups - 1})
    falling = [int(v) for v in np.exp(np.linspace(np.log(max_prefix), 0, groups))]
    for lens in ([300] * groups, falling, falling[::-1], [int(v) for v in r.integers(0, 2000, groups)], [0] * groups,
                 [0] * (groups - 1) + [max_prefix], [max_prefix] + [128] * (groups - 1)):
        lens = [min(l, max_prefix) for l in lens]
        c.prefix = lens
        c.lens[0].upload(u32(lens))
        c.call()
        c.check(sorted({g * per + m for g in some for m in {0, per - 1}}))
    lens[groups // 2] = max_prefix + 1
    c.lens[0].upload(u32(lens))
    c.call()
    assert np.isnan(c.out()[groups // 2 * per:(groups // 2 + 1) * per]).all()
    c.check([m for m in (0, groups * per - 1) if m // per != groups // 2])


@pytest.mark.parametrize("heads, kv, d, groups, per", [(8, 4, 64, 1, 64), (16, 8, 128, 3, 11), (16, 8, 128, 1, 32), (32, 8, 64, 5, 13)])
def test_own_rows_of_any_length(gpu, heads, kv, d, groups, per):
    """As many members as are taken by the length of their own rows, and one more: rows of one number, none, one, too many."""
    print(f"[case] shared own rows {heads} {kv} {d} {groups} {per}", flush=True)
    r, n, most = np.random.default_rng(per), groups * per, 700
    c = Case(heads, kv, d, per, [70] * groups, [most] * n).upload()
    far = np.zeros(n, int)
    far[n // 3] = most
    for own in (np.full(n, 129), np.zeros(n, int), np.ones(n, int), far, r.integers(0, most + 1, n), np.arange(n) * most // n,
                np.arange(n)[::-1] * most // n, np.where(np.arange(n) == n - 1, most + 1, 33)):
        c.own = [int(v) for v in own]
        c.lens[1].upload(u32(c.own))
        c.call()
        if max(c.own) > most:
            assert np.isnan(c.out()[-1]).all()
        c.check([m for m in (0, 1, n // 3, n // 2, n - 2, n - 1) if c.own[m] <= most])


def test_prefix_or_own_rows_alone(gpu):
    for d in (64, 128):
        c = Case(8, 2, d, 3, [200], [0, 0, 0]).upload()
        assert c.max_own == 0
        c.call()
        c.check()
        c = Case(8, 2, d, 3, [0], [1, 300, 33]).upload()
        assert c.max_prefix == 0
        c.call()
        c.check()
        c = Case(8, 2, d, 3, [0], [0, 0, 0]).upload()
        c.call()
        assert not c.out().any()


def test_lengths_that_do_not_fit(gpu):
    """The members' rows are NaN, the others as they were."""
    for d in (64, 128):
        c = Case(8, 2, d, 2, [50, 60], [4, 9, 8, 7]).upload()
        c.lens[0].upload(u32([61, 60]))
        c.lens[1].upload(u32([4, 9, 0xFFFFFFFF, 7]))
        c.call()
        got = c.out()
        assert np.isnan(got[:3]).all()
        c.check([3])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("share", [0.9, 0.999, 0.999999])
def test_weights_beside_a_dominant_key(gpu, d, share):
    """The first key has nearly all the weight and next to no v (the usual first token): the others make the output, and
    keep f32's precision."""
    print(f"[case] shared sink {d} {share}", flush=True)
    for n in (40, 3000):
        c = Case(4, 1, d, 4, [n], [20] * 4, scale=0.4)
        for m in range(4):
            c.q[m, :] = 0.02 * c.q[m] + 0.25  # all rows alike along one direction
        extra = np.log(share / (1 - share) * n)
        c.kp[0, 0] = (extra / (0.25 * d) * np.sqrt(d))
        c.vp[0, 0] = 0
        c.upload().call()
        c.check()


@pytest.mark.parametrize("d", [64, 128])
def test_infinities(gpu, d):
    """What the members see of them, as the formula has it; the others see nothing of it."""
    n = 300
    c = Case(4, 1, d, 3, [n], [40, 40, 40])
    c.vo[0, 7, 0, 3] = np.inf      # member 0 alone
    c.vp[0, 150, 0, 9] = -np.inf   # all
    c.vp[0, 20, 0, 11] = np.nan
    c.ko[1, 33, 0] = np.where(c.q[1, :d] > 0, -np.inf, np.inf)  # member 1, head 0: score -inf, weight 0
    c.ko[2, 5, 0, 2] = np.nan      # member 2: NaN
    c.upload().call()
    got = c.out()
    assert (got[0, :, 3] == np.inf).all() and np.isfinite(got[1, 0, 3])
    assert np.isneginf(got[0, :, 9]).all() and np.isneginf(got[1, 0, 9])
    assert np.isnan(got[0, :, 11]).all() and np.isnan(got[1, 0, 11])
    assert np.isnan(got[2]).all()
    rest = [i for i in range(d) if i not in (3, 9, 11)]
    want, bound = c.member(0)
    assert (np.abs(got[0] - want)[:, rest] <= bound[:, rest]).all()
    keep = np.delete(np.arange(40), 33)
    want, bound = _members.attention(c.q[1, :d][None], np.concatenate([c.kp[0], c.ko[1, keep]]), np.concatenate([c.vp[0], c.vo[1, keep]]))
    assert (np.abs(got[1, 0] - want[0])[rest] <= bound[0, rest]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_scores_of_every_size(gpu, d):
    """Tiny and huge queries, equal scores, and scores that rise from key to key."""
    for scale in (1e-30, 1e-3, 20.0, 3e4):
        c = Case(4, 2, d, 2, [260], [33, 0], scale=scale).upload()
        c.call()
        c.check()
    c = Case(4, 2, d, 2, [260], [33, 0])
    c.q[:] = 0
    c.upload().call()
    c.check()
    c = Case(4, 2, d, 2, [700], [90, 3], scale=0.1)
    c.q[:] = np.abs(c.q) + 0.5
    c.kp[:] = (np.linspace(-4, 4, 700)[:, None, None] + 0.01 * c.kp.astype(np.float32)[0]).astype(np.float16)
    c.upload().call()
    c.check()


def test_graph_follows_the_lengths(gpu):
    """A captured call, replayed with other lengths and queries on another stream than the uploads'."""
    c = Case(16, 4, 128, 4, [900], [100, 100, 90, 3], max_own=128).upload()
    s = Stream()
    with Graph.capture(s) as g:
        c.call(s)
    for own, prefix in (([100, 100, 90, 3], 900), ([1, 128, 0, 64], 333), ([2, 2, 2, 2], 1), ([5, 5, 5, 128], 0)):
        c.own, c.prefix = own, [prefix]
        full = Case(16, 4, 128, 4, [900], [128] * 4)
        c.kp, c.vp, c.ko, c.vo = full.kp, full.vp, full.ko, full.vo
        c.q = (np.random.default_rng(prefix).standard_normal(c.q.shape)).astype(np.float32)
        for b, a in zip(c.bufs + c.lens + [c.qb], (c.kp, c.vp, c.ko, c.vo, u32([prefix]), u32(own), c.q)):
            b.upload(a)
        g.launch(s)
        s.synchronize()
        c.check()
    first = c.out()
    c.call()
    assert np.array_equal(first, c.out()), "the same call twice, the same bits"


def test_captured_groups_of_other_lengths(gpu):
    """Chunks and the members' order follow the lengths of each replay."""
    c = Case(16, 4, 64, 13, [9000] * 5, [90] * 65, max_prefix=9000, max_own=90).upload()  # the groups share chunks
    d = Case(16, 8, 128, 16, [500] * 3, [300] * 48).upload()                             # longest own rows first
    s = Stream()
    with Graph.capture(s) as g:
        c.call(s)
        d.call(s)
    r = np.random.default_rng(3)
    for prefix in ([9000, 1, 700, 0, 130], [0] * 5, [9000] * 5):
        for case, most in ((c, 90), (d, 300)):
            case.prefix = [min(v, case.max_prefix) for v in prefix[:case.groups]]
            case.own = [int(v) for v in r.integers(0, most + 1, case.n)]
            case.lens[0].upload(u32(case.prefix))
            case.lens[1].upload(u32(case.own))
        g.launch(s)
        s.synchronize()
        c.check([0, 14, 27, 51, 64])
        d.check([0, 15, 16, 47])
        first = c.out(), d.out()
        c.call()
        d.call()
        assert np.array_equal(first[0], c.out()) and np.array_equal(first[1], d.out())


def test_two_streams_at_once(gpu):
    """Calls that overlap, each with its own workspace."""
    cases = [Case(16, 4, 128, 9, [4000, 50], [700] * 18, seed=i).upload() for i in range(2)]
    streams = [Stream(), Stream()]
    for _ in range(20):
        for c, s in zip(cases, streams):
            c.call(s)
    for c, s in zip(cases, streams):
        s.synchronize()
        c.check([0, 8, 17])
