"""Sampling where most of the weight is far from the largest logit: tens of thousands of tokens of nearly equal weight, and random numbers next to the
borders between two of them."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from test_gpu_sample import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


def near_borders(rng, row, temperature, n):
    """n random numbers whose share of the weight ends close to a border between two tokens, but not closer than the arithmetic allows: a weight is
    within 2^-32 of itself and half of 2^-44 of the largest (vocabularies up to 2^17 tokens), and so is a sum of them; twice that."""
    w = np.exp((row.astype(np.float64) - float(row.max())) / float(np.float32(temperature)))
    mass = np.cumsum(w.astype(np.longdouble))
    u = rng.random(1 << 20, np.float32)
    at = u.astype(np.longdouble) * mass[-1]
    i = np.searchsorted(mass, at, side="right")
    off = np.minimum(at - np.where(i > 0, mass[np.maximum(i - 1, 0)], -1), mass[np.minimum(i, row.size - 1)] - at)
    allowed = 2 * (2.0 ** -32 * mass[-1] + row.size * 2.0 ** -45)
    order = np.argsort(np.where(off > allowed, off, np.inf))
    return u[order[:n]]


@pytest.mark.parametrize("near, far", [(3.9, 4.1), (1.0, 4.5), (5.0, 5.5), (7.3, 9.9), (11.0, 20.0)])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_two_levels(ctx, near, far, temperature):
    """One largest logit; a part of the vocabulary `near`, the rest `far` temperatures below, one behind the other: an error that equal weights share
    adds up, and moves the borders of the ones against the others'."""
    rng = np.random.default_rng(int(near * 10))
    vocab, n = 128256, 64
    share = 1 / (1 + np.exp(far - near))  # so that both have the same weight
    row = np.float32(2.5) - np.where(np.arange(vocab) < vocab * share, near, far).astype(np.float32) * np.float32(temperature)
    row[rng.integers(vocab)] = 2.5
    u = near_borders(rng, row, temperature, n)
    tok, lp = run(ctx, np.broadcast_to(row, (n, vocab)), u, temperature)
    for r in range(n):
        want, wlp = kit.sample(row, temperature, u=u[r])
        assert tok[r] == want, (r, tok[r], want, u[r])
        # the result's rounding, 2^-32 of the sum, and half a unit of 2^-44 for each of the weights, which equal ones share: 128,256 of 2^-45 are 3.6e-9
        assert abs(lp[r] - wlp) <= 2.0 ** -23 * abs(wlp) + 2.0 ** -32 + vocab * 2.0 ** -45


@pytest.mark.parametrize("low, high", [(-9.0, -4.0), (-16.0, -3.0), (-30.0, -12.0)])
def test_a_spread_tail(ctx, low, high):
    rng = np.random.default_rng(int(-low))
    vocab, n = 100003, 64
    row = np.sort(rng.uniform(low, high, vocab)).astype(np.float32)
    row[7] = 0.0
    u = near_borders(rng, row, 1.0, n)
    tok, _ = run(ctx, np.broadcast_to(row, (n, vocab)), u, 1.0)
    assert tok.tolist() == [kit.sample(row, 1.0, u=x)[0] for x in u]
