"""Low-rank adapters against the plain form, token by token: numbers of tokens around every tile, odd sizes, ranks of one and many, slots in any
order, empty and out of range, rows with strides, in place, and recorded frames."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from loom_b200 import cabi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


def bf16(a):
    return (cabi.to_bf16(a).astype(np.uint32) << 16).view(np.float32)


class Set:
    def __init__(self, ctx, rng, slots, rows, cols, ranks, dtype, max_rank=None):
        self.ctx, self.rows, self.cols = ctx, rows, cols
        self.a = cabi.Adapters(ctx, slots, rows, cols, max_rank or max(max(ranks), 1), dtype)
        self.host = []
        for s, r in enumerate(ranks):
            down, up = rng.standard_normal((r, cols)).astype(np.float32), rng.standard_normal((rows, r)).astype(np.float32)
            scale = np.float32(rng.uniform(-2, 2))
            if dtype == cabi.DTYPE_BF16:
                down, up = bf16(down), bf16(up)
            if r:
                self.a.put(s, down, up, scale)
            self.host.append((down, up, float(scale)))

    def run(self, x, slot, base, in_place=False, ldx=None, offset=0):
        ctx, n = self.ctx, x.shape[0]
        ldx = self.cols if ldx is None else ldx
        flat = np.full(offset + n * ldx + 4, np.nan, np.float32)
        for i in range(n):
            flat[offset + i * ldx:][:self.cols] = x[i]
        bx, bs = ctx.to_device(flat), ctx.to_device(np.asarray(slot, np.int32))
        bb = None if base is None else ctx.to_device(base)
        guard = np.full((n + 1) * self.rows, 7.25, np.float32)  # a row behind the last stays as it is
        out = bb if in_place else ctx.to_device(guard)
        self.a.apply(n, bs, bx + 4 * offset, out, base=bb, ldx=ldx)
        got = ctx.download(out, (n if in_place else n + 1, self.rows), np.float32)
        if not in_place:
            assert (got[n] == 7.25).all()
        ctx.sync()
        for b in {bx, bs, bb, out} - {None}:
            ctx.free(b)
        return got[:n]

    def check(self, x, slot, base, **how):
        got = self.run(x, slot, base, **how)
        for i in range(x.shape[0]):
            s = slot[i]
            if 0 <= s < len(self.host) and self.host[s][0].shape[0]:
                want, tol = kit.adapter(x[i], *self.host[s], None if base is None else base[i])
                assert (np.abs(got[i] - want) <= tol).all(), (i, s, np.abs(got[i] - want).max(), (np.abs(got[i] - want) / tol).max())
            else:
                assert np.array_equal(got[i], np.zeros(self.rows, np.float32) if base is None else base[i])
        return got


DTYPES = [cabi.DTYPE_BF16, cabi.DTYPE_F32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 64, 255, 256, 257, 400])
def test_numbers_of_tokens(ctx, dtype, tokens):
    rng = np.random.default_rng(tokens)
    s = Set(ctx, rng, 5, 200, 136, [8, 16, 3, 20, 0], dtype)
    slot = rng.integers(-1, 6, tokens)  # none, the empty one and one past the last among them
    s.check(rng.standard_normal((tokens, 136)).astype(np.float32), slot, rng.standard_normal((tokens, 200)).astype(np.float32))
    s.check(rng.standard_normal((tokens, 136)).astype(np.float32), np.full(tokens, 1), None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (16, 31), (17, 32), (33, 33), (50, 1000), (777, 64), (1024, 2052)])
@pytest.mark.parametrize("tokens", [5, 300])
def test_sizes(ctx, dtype, rows, cols, tokens):
    rng = np.random.default_rng(rows * cols)
    s = Set(ctx, rng, 3, rows, cols, [1, 9, 32], dtype)
    s.check(rng.standard_normal((tokens, cols)).astype(np.float32), rng.integers(0, 3, tokens), rng.standard_normal((tokens, rows)).astype(np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_ranks(ctx, dtype):
    rng = np.random.default_rng(3)
    s = Set(ctx, rng, 9, 90, 300, [1, 7, 8, 15, 17, 63, 64, 65, 256], dtype)
    for tokens in (9, 270):
        s.check(rng.standard_normal((tokens, 300)).astype(np.float32), np.arange(tokens) % 9, rng.standard_normal((tokens, 90)).astype(np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_tokens_than_a_launch_takes(ctx, dtype):
    rng = np.random.default_rng(9)
    a = Set(ctx, rng, 3, 13, 20, [5, 0, 17], dtype)
    n = 2 * 4096 + 7
    x, base = rng.standard_normal((n, 20)).astype(np.float32), rng.standard_normal((n, 13)).astype(np.float32)
    slot = rng.integers(-1, 4, n)
    a.check(x, slot, base, ldx=23, offset=1)
    a.check(x, slot, base, in_place=True)
    a.a.free()


def test_a_slot_put_again(ctx):
    rng = np.random.default_rng(4)
    s = Set(ctx, rng, 2, 40, 50, [16, 12], cabi.DTYPE_BF16)
    x, base = rng.standard_normal((6, 50)).astype(np.float32), rng.standard_normal((6, 40)).astype(np.float32)
    slot = [0, 1, 0, 1, 0, 1]
    s.check(x, slot, base)
    down, up = bf16(rng.standard_normal((3, 50)).astype(np.float32)), bf16(rng.standard_normal((40, 3)).astype(np.float32))
    s.a.put(0, cabi.to_bf16(down), cabi.to_bf16(up), 0.5, cabi.DTYPE_BF16)  # a smaller rank: nothing of the former is left
    s.host[0] = (down, up, 0.5)
    s.check(x, slot, base)
    s.a.put(1, None, None)
    s.host[1] = (down[:0], up[:, :0], 0.0)
    got = s.check(x, slot, base)
    assert np.array_equal(got[1::2], base[1::2])


@pytest.mark.parametrize("tokens", [7, 300])
def test_in_place_and_strides(ctx, tokens):
    rng = np.random.default_rng(5)
    s = Set(ctx, rng, 4, 130, 70, [4, 8, 16, 24], cabi.DTYPE_BF16)
    x, base, slot = rng.standard_normal((tokens, 70)).astype(np.float32), rng.standard_normal((tokens, 130)).astype(np.float32), rng.integers(-1, 4, tokens)
    plain = s.check(x, slot, base)
    assert np.array_equal(s.run(x, slot, base, in_place=True).view(np.uint32), plain.view(np.uint32))
    for ldx, offset in ((70, 1), (71, 0), (72, 4), (100, 3)):
        assert np.array_equal(s.run(x, slot, base, ldx=ldx, offset=offset).view(np.uint32), plain.view(np.uint32))


def test_odd_values_stay_in_their_row(ctx):
    rng = np.random.default_rng(6)
    s = Set(ctx, rng, 2, 64, 96, [8, 8], cabi.DTYPE_BF16)
    x, base = rng.standard_normal((20, 96)).astype(np.float32), rng.standard_normal((20, 64)).astype(np.float32)
    slot = np.arange(20) % 2
    clean = s.run(x, slot, base)
    x[3, 5], x[8, 9], x[9] = np.nan, np.inf, np.float32(3e38)
    got = s.run(x, slot, base)
    rest = [i for i in range(20) if i not in (3, 8, 9)]
    assert np.isnan(got[3]).all() and not np.isfinite(got[8]).any()
    assert np.array_equal(got[rest].view(np.uint32), clean[rest].view(np.uint32))


def test_more_slots_than_tokens_and_a_frame():
    rng = np.random.default_rng(8)
    ctx = loom_b200.Context(0)
    try:
        s = Set(ctx, rng, 700, 48, 32, [2] * 700, cabi.DTYPE_F32)
        x, base = rng.standard_normal((64, 32)).astype(np.float32), rng.standard_normal((64, 48)).astype(np.float32)
        slot = rng.integers(0, 700, 64)
        s.check(x, slot, base)
        bx, bs, bb, out = ctx.to_device(x), ctx.to_device(slot.astype(np.int32)), ctx.to_device(base), ctx.alloc(64 * 48 * 4)
        s.a.apply(64, bs, bx, out, base=bb)
        want = ctx.download(out, (64, 48), np.uint32)
        ctx.graph_begin()
        s.a.apply(64, bs, bx, out, base=bb)
        frame = ctx.graph_end()
        for _ in range(3):
            ctx.zero(out, 64 * 48 * 4)
            ctx.graph_launch(frame)
            assert np.array_equal(ctx.download(out, (64, 48), np.uint32), want)
        other = rng.integers(0, 700, 64)  # other requests in the same frame
        ctx.upload(bs, other.astype(np.int32))
        ctx.graph_launch(frame)
        got = ctx.download(out, (64, 48), np.float32)
        for i in range(64):
            y, tol = kit.adapter(x[i], *s.host[other[i]], base[i])
            assert (np.abs(got[i] - y) <= tol).all()
        ctx.graph_free(frame)
    finally:
        ctx.close()
