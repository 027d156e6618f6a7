"""The bar of tests/_shared.py tells two f16 limbs from one, and a reference that follows the tiles from one that does not."""
import numpy as np
import pytest

from tests import _shared


def inputs(d, n, share=0.0, at=0, seed=0):
    r = np.random.default_rng([seed, d, n])
    q = (r.standard_normal(d) * 1.3).astype(np.float32)
    k, v = (r.standard_normal((n, d)).astype(np.float16) for _ in range(2))
    _shared.add_sink(q, k, v, share, at)
    want, top = _shared.exact(q[None], k[:, None], v[:, None])
    return q, k, v, want[0], _shared.bar(top)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [33, 300, 3000, 40000])
def test_one_limb_fails_the_bar(d, n):
    q, k, v, want, bar = inputs(d, n)
    assert _shared.rel(_shared.emulate(q, k, v), want) <= bar / 8
    assert _shared.rel(_shared.emulate(q, k, v, p_limbs=1), want) > 2 * bar
    assert _shared.rel(_shared.emulate(q, k, v, q_limbs=1), want) > 2 * bar


@pytest.mark.parametrize("n, tile", [(40, 32), (3000, 32), (8000, 64), (40000, 64)])
@pytest.mark.parametrize("share", [0.9, 0.999999, 1 - 1e-9, 1 - 1e-12])
def test_weights_beside_a_dominant_key(n, tile, share):
    for at in (0, n // 2 + 3, n - 1):
        q, k, v, want, bar = inputs(64, n, share, at)
        assert _shared.rel(_shared.emulate(q, k, v, tile), want) <= bar / 8
        assert _shared.rel(_shared.emulate(q, k, v, tile, p_limbs=1), want) > 2 * bar
        if at == 0 and n >= 3000 and 1 - share < 1e-8:  # a weight of (1 - share) / n is off by 2^-48
            assert _shared.rel(_shared.emulate(q, k, v, tile, falls=False), want) > 2 * bar
