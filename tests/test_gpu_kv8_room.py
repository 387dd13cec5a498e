"""Attention of long portions for which their sequence has no room, beside sequences that have: zeros, and no wait for them."""
import numpy as np
import pytest
import torch

import loom_b200
import servingkit as kit
from loom_b200 import LoomB200Error, cabi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("many", [2000, 33])
def test_a_portion_without_room(dim, many):
    rng = np.random.default_rng(many)
    ctx = loom_b200.Context(0)
    try:
        kv_heads, heads, seqs = 4, 32, 200
        kv = cabi.KV8(ctx, seqs, 300, kv_heads, dim)
        counts = np.ones(seqs, int)
        counts[[3, 150]] = many, many // 2
        lengths = np.where(counts == 1, 20, 290).astype(np.int32)
        rows, starts = int(counts.sum()), np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        at = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        old = rng.standard_normal((int(lengths.sum()), kv_heads, dim)).astype(np.float32)
        new = rng.standard_normal((rows, kv_heads, dim)).astype(np.float32)
        q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        d = {n: ctx.to_device(a) for n, a in dict(zero=np.zeros(seqs, np.int32), at=at, old=old, new=new, q=q, starts=starts, lengths=lengths).items()}
        out = ctx.to_device(np.full((rows + 1, heads, dim), 3.5, np.float32))
        kv.append(len(old), d["zero"], d["old"], d["old"], starts=d["at"])
        kv.append(rows, d["lengths"], d["new"], d["new"], starts=d["starts"])
        stream = torch.cuda.ExternalStream(ctx.stream)
        took = []
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record(stream)
            kv.attend(rows, heads, d["lengths"], d["q"], out, starts=d["starts"])
            b.record(stream)
            b.synchronize()
            took.append(a.elapsed_time(b))
        got = ctx.download(out, (rows + 1, heads, dim), np.float32)
        with pytest.raises(LoomB200Error) as e:
            ctx.sync()
        assert e.value.code == cabi.ERR_INVALID and "8-bit cache" in str(e.value)
        assert (got[rows] == 3.5).all()
        for s in range(seqs):
            if counts[s] > 1:
                assert (got[starts[s]:starts[s + 1]] == 0).all()
            elif s % 17 == 0:
                mine = np.concatenate([old[at[s]:at[s + 1]], new[starts[s]:starts[s + 1]]])
                want, tol = kit.attend(q[starts[s]:starts[s + 1]], kit.held(mine), kit.held(mine), 20)
                assert (np.abs(got[starts[s]] - want[0]) <= tol[0]).all()
        assert min(took) < 2.0, took  # ms: 3000 rows of zeros are 49 MB, one thread takes 200
    finally:
        ctx.close()
