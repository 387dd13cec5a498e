"""Portions among many sequences: every sequence's attention looked at, and the kernel for portions where the call has one, however many sequences the
cache has room for."""
import numpy as np
import pytest

import loom_b200
from test_gpu_kv8 import Cache, check_some

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dim, heads", [(40, 2), (40, 8), (128, 6)])
def test_portions_of_most_of_200_sequences(ctx, dim, heads):
    rng = np.random.default_rng(dim + heads)
    n = 200
    c = Cache(ctx, n, 700, 2, dim)
    counts = np.where(rng.random(n) < 0.2, 0, rng.integers(1, 300, n))
    call = c.append(rng, counts)
    check_some(c, rng, call, counts, heads, 1)
    c.drop()
    counts = np.where(rng.random(n) < 0.2, 0, rng.integers(1, 200, n))  # from every place of a block
    call = c.append(rng, counts)
    check_some(c, rng, call, counts, heads, 1)
    c.drop()
    c.kv.free()


@pytest.mark.parametrize("others", [0, 1])
@pytest.mark.parametrize("rows", [70, 200])
def test_one_portion_in_a_cache_of_many(ctx, others, rows):
    rng = np.random.default_rng(rows + others)
    n = 256
    c = Cache(ctx, n, 1300, 1, 128)
    before = np.where(np.arange(n) == 100, 1000, 30 * others)
    c.append(rng, before)
    c.drop()
    counts = np.where(np.arange(n) == 100, rows, others)
    call = c.append(rng, counts)
    launches = ctx.launch_count
    check_some(c, rng, call, counts, 4, 3)
    assert ctx.launch_count - launches == 2  # few rows, and portions
    c.drop()
    c.kv.free()


def test_a_step_of_few_sequences_is_one_launch(ctx):
    rng = np.random.default_rng(3)
    c = Cache(ctx, 16, 300, 1, 128)
    c.append(rng, np.full(16, 100))
    call = c.append(rng, np.ones(16, int))  # (with starts)
    launches = ctx.launch_count
    check_some(c, rng, call, np.ones(16, int), 4, 1)
    assert ctx.launch_count - launches == 1
    c.drop()
    c.kv.free()
