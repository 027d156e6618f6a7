"""wh_qk_norm_rope: heads whose squares are no f32 numbers, and calls beyond one launch dimension."""
import numpy as np
import pytest

from tests import _members
from tests._gpu import down, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [2, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("rows", [1, 700])
def test_norms_of_values_of_any_size(gpu, d, rows):
    """Query and key heads of huge and of tiny values are normed as the formula has it, beside heads of ordinary ones."""
    heads, kv = 9, 3
    r = np.random.default_rng([d, rows])
    x = r.standard_normal((rows, heads + 2 * kv, d)).astype(np.float32)
    for h, size in ((0, 1e25), (1, 1e-25), (3, 2e19), (4, 3e-20), (5, 1e-40), (6, 5e37), (heads, 1e25), (heads + 1, 1e-25)):
        x[:, h] = (x[:, h].astype(np.float64) * size).astype(np.float32)
    x[:, 7, 0] = 3e38  # one element makes the norm
    inv = np.linspace(0.1, 0.7, d // 2).astype(np.float32)
    qw, kw = (1 + 0.3 * r.standard_normal((2, d))).astype(np.float32)
    width = (heads + 2 * kv) * d
    xb, out, kout = up(x.reshape(rows, -1))[0], DeviceBuffer(4 * rows * heads * d), DeviceBuffer(4 * rows * kv * d)
    print(f"[case] norms of any size d {d} rows {rows}", flush=True)
    for eps in (0.0, 1e-6):
        rules = ops.RopeRules(up(inv)[0], 0, False, 1.0, up(qw)[0], up(kw)[0], eps)
        ops.qk_norm_rope(rules, xb, xb.ptr + 4 * heads * d, xb.ptr + 4 * (heads + kv) * d, width, width, None, None, 1, 1, rows, heads, kv,
                         d, out, heads * d, kout, kv * d, None, None, 0)
        q, k = down(out, np.float32, rows * heads * d).reshape(rows, heads, d), down(kout, np.float32, rows * kv * d).reshape(rows, kv, d)
        for got, inp, w in ((q, x[:, :heads], qw), (k, x[:, heads:heads + kv], kw)):
            want, bound = _members.rope(inp, np.arange(rows), inv, d, False, 1.0, w, eps)
            # 2^-149: an output below the normal f32 numbers (values of 1e-40 beside an epsilon)
            assert (np.abs(got - want) <= bound + 2.0 ** -148).all(), (eps, np.abs(got - want).max())


def test_infinities_and_nan_of_a_normed_head(gpu):
    """An infinity leaves 0 of the others and is NaN itself; a NaN is the head's."""
    d, heads, kv = 64, 3, 1
    x = np.ones((1, heads + 2 * kv, d), np.float32)
    x[0, 0, 5], x[0, 1, 9], x[0, heads, 7] = np.inf, np.nan, -np.inf
    inv, w = up(np.zeros(d // 2, np.float32))[0], up(np.ones(d, np.float32))[0]
    xb, out, kout = up(x.reshape(1, -1))[0], DeviceBuffer(4 * heads * d), DeviceBuffer(4 * kv * d)
    ops.qk_norm_rope(ops.RopeRules(inv, 0, False, 1.0, w, w, 1e-6), xb, xb.ptr + 4 * heads * d, xb.ptr + 4 * (heads + kv) * d,
                     (heads + 2 * kv) * d, (heads + 2 * kv) * d, None, None, 1, 1, 1, heads, kv, d, out, heads * d, kout, kv * d, None, None, 0)
    q, k = down(out, np.float32, heads * d).reshape(heads, d), down(kout, np.float32, kv * d).reshape(kv, d)
    pair = lambda i: [i, i + d // 2]
    for got, i in ((q[0], 5), (k[0], 7)):
        assert np.isnan(got[i]) and not np.delete(got, pair(i)).any()
    assert np.isnan(q[1]).all()
    assert (np.abs(q[2] - 1) <= 2.0 ** -20).all()


def test_more_rows_than_a_launch_dimension_takes(gpu):
    """2^26 rows and some of two heads of two elements: 64 threads to a row are more than 2^32 in all."""
    rows, period = (1 << 26) + 37, 4099
    r = np.random.default_rng(0)
    pattern = r.standard_normal((period, 6)).astype(np.float32)
    x = DeviceBuffer.from_array(np.tile(pattern, (-(-rows // period), 1))[:rows])
    inv = np.array([0.37], np.float32)
    out = DeviceBuffer(8 * rows)
    out.fill(0xEE)
    print(f"[case] rope of {rows} rows", flush=True)
    ops.qk_norm_rope(ops.RopeRules(up(inv)[0]), x, x.ptr + 8, x.ptr + 16, 6, 6, None, None, 1, 1, rows, 1, 1, 2, out, 2, None, 0, None, None, 0)
    got = down(out, np.float32, 2 * rows).reshape(rows, 1, 2)
    some = np.unique(np.concatenate([np.arange(0, rows, 997), np.arange(300), np.arange(rows - 300, rows), (1 << 24) + np.arange(-300, 300)]))
    want, bound = _members.rope(pattern[some % period, None, :2], some, inv, 2, False)
    assert (np.abs(got[some] - want) <= bound).all()
    assert not (got.view(np.uint32) == 0xEEEEEEEE).any()
