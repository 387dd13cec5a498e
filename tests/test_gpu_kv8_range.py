"""Attention over the 8-bit cache with values of any magnitude: whole blocks and open ones, few rows and portions."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from test_gpu_kv8 import Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("before, count", [(0, 40), (300, 1), (300, 64), (100, 200), (256, 128)])
@pytest.mark.parametrize("spread", [1e-30, 1e-24, 1e-12, 1e12, 1e25, 1e33])
def test_small_and_large_values(ctx, before, count, spread):
    rng = np.random.default_rng(count)
    c = Cache(ctx, 1, 700, 2, 64)
    change = lambda k, v: np.multiply(v, np.float32(spread), out=v)  # noqa: E731
    if before:
        c.append(rng, [before], change=change)
    call = c.append(rng, [count], change=change)
    c.check(rng, call, [count], 8)
    c.kv.free()


@pytest.mark.parametrize("spread", [1e-28, 1.0, 1e33])
@pytest.mark.parametrize("step", [-0.2, 0.05, 0.15, 0.2, 0.5])
def test_scores_that_climb(ctx, spread, step):
    """Every block's scores stand above (or below) the ones before it, so that a row's largest score is behind most of the time."""
    rng = np.random.default_rng(7)

    def change(k, v):
        at = np.arange(len(k))[:, None, None] // 64
        k *= np.float32(0.1)
        k[:, :, :1] = step * 8 * at * np.sqrt(np.float32(64))
        v *= np.float32(spread)
    c = Cache(ctx, 1, 700, 1, 64)
    call = c.append(rng, [640 + 30], change=change)
    q = np.abs(rng.standard_normal((670, 4, 64))).astype(np.float32) * np.float32(0.1)
    q[:, :, 0] = 1.0
    _, out = c.attend(rng, call, 4, q=q)
    k, v = kit.held(c.k[0]), kit.held(c.v[0])
    for j in (0, 63, 64, 200, 383, 500, 639, 640, 669):
        want, tol = kit.attend(q[j:j + 1], k, v, j)
        assert (np.abs(out[j] - want[0]) <= tol[0]).all(), (j, np.abs(out[j] - want[0]).max(), tol[0].min())
    c.drop()
    c.kv.free()
