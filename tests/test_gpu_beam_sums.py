"""wh_beam_select: how near a row's log sum exp comes to 64 bits."""
import numpy as np
import pytest

from tests._gpu import down, up
from woolly_amd import ops
from woolly_amd.device import DeviceBuffer

pytestmark = pytest.mark.gpu


def rows(vocab, r):
    normal = r.standard_normal(vocab)
    yield "normal of 1", normal
    yield "normal of 3", 3 * normal
    yield "normal of 10", 10 * normal
    yield "equal but one", np.where(np.arange(vocab) == vocab // 2, np.log(vocab), 0.0)
    yield "a slope", -np.arange(vocab) / vocab * 30
    yield "far from 0", normal + 1000
    yield "few allowed", np.where(np.arange(vocab) % 97 == 5, 2 * normal, -np.inf)


@pytest.mark.parametrize("vocab", [7, 1000, 4099, 32000, 128256])
@pytest.mark.parametrize("pad", [0, 1])
def test_log_sum_exp(gpu, vocab, pad):
    """The score of the best continuation, with scores that bring it near 0, where f32 shows what the sum is off by.

    The bound: a term e^d, d <= 0, has its distance d in f32 (2^-24 |d|), that times log2 e in f32 (2^-24 |d|, and 2^-26 |d| of
    the constant) and its exponential (2^-23); a thread adds at most 8 of them (7 * 2^-24), the rest is in 64 bits.  Terms
    at d make at most the share min(1, N e^d) of N logits' sum, so |d| counts up to log N + 1: 2^-22 of that, and 2^-21."""
    r = np.random.default_rng(vocab)
    named = list(rows(vocab, r))
    logits = np.full((len(named), vocab + pad), np.inf, np.float32)
    logits[:, :vocab] = np.stack([x for _, x in named])
    x = logits[:, :vocab].astype(np.float64)
    top = x.max(1)
    best = -np.log(np.exp(x - top[:, None]).sum(1))  # its log-probability
    scores = (-best).astype(np.float32)
    rules, n = ops.BeamRules(1), len(named)
    out, tokens, parents = (DeviceBuffer(4 * n) for _ in range(3))
    need = ops.beam_select_workspace_bytes(rules, n, vocab)
    print(f"[case] beam sums {vocab}", flush=True)
    ops.beam_select(rules, up(logits)[0], vocab + pad, n, vocab, up(scores)[0], out, tokens, parents, DeviceBuffer(need), need)
    assert np.array_equal(down(tokens, np.uint32, n), x.argmax(1))
    err = np.abs(down(out, np.float32, n) - (scores.astype(np.float64) + best))
    bound = 2.0 ** -22 * (np.log(vocab) + 1) + 2.0 ** -21
    print("[result] " + ", ".join(f"{name} {e:.1e}" for (name, _), e in zip(named, err)) + f", bound {bound:.1e}", flush=True)
    assert (err <= bound).all(), err.max()
