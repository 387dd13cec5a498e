"""Attention whose work does not fit into its counters -- sequences that share rows, which only starts that go back can say: reported and not done."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from loom_b200 import LoomB200Error, cabi

pytestmark = pytest.mark.gpu


def test_more_work_than_the_counters_hold():
    """Heads of more than 128 dimensions, whose portions the kernel for few rows has too."""
    seqs, max_len, rows, heads, dim = 4096, 4096, 64, 4224, 130
    blocks = (max_len - rows) // 64 + 1
    assert seqs // 2 * (rows * heads // 8) * blocks >= 2 ** 32
    ctx = loom_b200.Context(0)
    try:
        kv = cabi.KV8(ctx, seqs, max_len, 1, dim)
        starts = ctx.to_device(np.append(np.tile(np.array([0, rows], np.int32), seqs // 2), np.int32(rows)))
        lengths = ctx.to_device(np.full(seqs, max_len - rows, np.int32))
        rng = np.random.default_rng(0)
        host = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        q, out = ctx.to_device(host), ctx.to_device(np.full((rows, heads, dim), 3.5, np.float32))
        kv.attend(rows, heads, lengths, q, out, starts=starts)
        with pytest.raises(LoomB200Error) as e:
            ctx.sync()
        assert e.value.code == cabi.ERR_INVALID and "more work" in str(e.value)
        assert (ctx.download(out, (rows, heads, dim), np.float32) == 3.5).all()
        # the next call is as ever
        k = rng.standard_normal((70, 1, dim)).astype(np.float32)
        one = np.full(seqs + 1, 70, np.int32)
        one[0] = 0
        zero, starts, dev = ctx.to_device(np.zeros(seqs, np.int32)), ctx.to_device(one), ctx.to_device(k)
        kv.append(70, zero, dev, dev, starts=starts)
        kv.attend(70, 2, zero, q, out, starts=starts)
        got = ctx.download(out, (rows, heads, dim), np.float32).ravel()[:140 * dim].reshape(70, 2, dim)
        want, tol = kit.attend(host.reshape(-1, 2, dim)[:70], kit.held(k), kit.held(k), 0)
        assert (np.abs(got - want) <= tol).all()
        ctx.sync()
    finally:
        ctx.close()
