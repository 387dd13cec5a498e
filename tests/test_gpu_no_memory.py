"""A handle that does not fit into the GPU's memory is refused, and the context goes on as before."""
import numpy as np
import pytest

import loom_b200
from loom_b200 import LoomB200Error, cabi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("make", [lambda ctx: cabi.KV8(ctx, 4096, 1 << 24, 64, 256), lambda ctx: cabi.Adapters(ctx, 4096, 1 << 23, 1 << 23, 256, cabi.DTYPE_F32)])
def test_a_handle_that_does_not_fit(make):
    ctx = loom_b200.Context(0)
    try:
        with pytest.raises(LoomB200Error) as e:
            make(ctx)
        assert e.value.code == cabi.ERR_CUDA and "memory" in str(e.value)
        a = cabi.Adapters(ctx, 1, 5, 6, 2, cabi.DTYPE_F32)
        a.put(0, np.ones((2, 6), np.float32), np.ones((5, 2), np.float32))
        x, slot, out = ctx.to_device(np.ones((1, 6), np.float32)), ctx.to_device(np.zeros(1, np.int32)), ctx.to_device(np.zeros((1, 5), np.float32))
        a.apply(1, slot, x, out)
        assert (ctx.download(out, (1, 5), np.float32) == 12).all()
        ctx.sync()
    finally:
        ctx.close()
