"""The 8-bit cache: what it holds bit for bit, however the rows came, and attention over it against the plain form in 64 bits."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from loom_b200 import LoomB200Error, cabi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


class Cache:
    """A cache and, on the host, every row that each sequence was given."""

    def __init__(self, ctx, seqs, max_len, kv_heads, dim):
        self.ctx, self.kv, self.dim, self.heads, self.seqs = ctx, cabi.KV8(ctx, seqs, max_len, kv_heads, dim), dim, kv_heads, seqs
        self.k = [np.zeros((0, kv_heads, dim), np.float32) for _ in range(seqs)]
        self.v = [np.zeros((0, kv_heads, dim), np.float32) for _ in range(seqs)]
        self.held = []

    def dev(self, a):
        self.held.append(self.ctx.to_device(a))
        return self.held[-1]

    def drop(self):
        self.ctx.sync()
        for b in self.held:
            self.ctx.free(b)
        self.held = []

    def lengths(self):
        return np.array([len(k) for k in self.k], np.int32)

    def append(self, rng, counts, spread=1.0, change=None, step=False, pad=0):
        """counts[s] random rows to every sequence.  step: one row each without starts; pad: floats between rows.  Returns starts and lengths on
        the device and the number of rows, for the calls that follow."""
        counts = np.asarray(counts)
        rows, width = int(counts.sum()), self.heads * self.dim
        k, v = rng.standard_normal((rows, self.heads, self.dim)).astype(np.float32) * np.float32(spread), rng.standard_normal((rows, self.heads, self.dim)).astype(np.float32)
        if change:
            change(k, v)
        lengths = self.dev(self.lengths())
        starts = None if step else self.dev(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        wide = [np.full((rows, width + pad), np.nan, np.float32) for _ in "kv"]
        wide[0][:, :width], wide[1][:, :width] = k.reshape(rows, -1), v.reshape(rows, -1)
        self.kv.append(rows, lengths, self.dev(wide[0]), self.dev(wide[1]), starts=starts, ld=width + pad)
        at = 0
        for s, n in enumerate(counts):
            self.k[s], self.v[s] = np.concatenate([self.k[s], k[at:at + n]]), np.concatenate([self.v[s], v[at:at + n]])
            at += n
        return starts, lengths, rows

    def read(self, starts, lengths, rows):
        out = [self.dev(np.full((rows, self.heads, self.dim), 9.5, np.float32)) for _ in "kv"]
        self.kv.read(rows, lengths, *out, starts=starts)
        return [self.ctx.download(o, (rows, self.heads, self.dim), np.float32) for o in out]

    def check_rows(self, call, counts):
        got = self.read(*call)
        at = 0
        for s, n in enumerate(counts):
            for g, mine in zip(got, (self.k[s], self.v[s])):
                want = kit.held(mine, exact=False)[len(mine) - n:]
                assert np.array_equal(g[at:at + n], want, equal_nan=True), (s, n)
            at += n

    def attend(self, rng, call, heads, scale=0.0, q=None, pad=0):
        starts, lengths, rows = call
        width = heads * self.dim
        q = rng.standard_normal((rows, heads, self.dim)).astype(np.float32) if q is None else q
        wide = np.full((rows, width + pad), np.nan, np.float32)
        wide[:, :width] = q.reshape(rows, -1)
        out = self.dev(np.full((rows + 1, heads, self.dim), 3.5, np.float32))
        self.kv.attend(rows, heads, lengths, self.dev(wide), out, starts=starts, scale=scale, ldq=width + pad)
        got = self.ctx.download(out, (rows + 1, heads, self.dim), np.float32)
        assert (got[rows] == 3.5).all()
        return q, got[:rows]

    def check(self, rng, call, counts, heads, scale=0.0, pad=0, want_rows=None):
        q, got = self.attend(rng, call, heads, scale, pad=pad)
        at = 0
        for s, n in enumerate(counts):
            if n:
                want, tol = kit.attend(q[at:at + n], kit.held(self.k[s]), kit.held(self.v[s]), len(self.k[s]) - n, scale or None)
                off = np.abs(got[at:at + n] - want)
                assert (off <= tol).all(), (s, n, len(self.k[s]), off.max(), (off / tol).max())
            at += n
        self.drop()
        return q, got


@pytest.mark.parametrize("dim", [1, 8, 20, 32, 40, 64, 72, 80, 96, 128, 160, 200, 224, 256])
def test_head_dimensions(ctx, dim):
    rng = np.random.default_rng(dim)
    c = Cache(ctx, 3, 400, 2, dim)
    counts = [130, 64, 7]
    call = c.append(rng, counts)
    c.check_rows(call, counts)
    c.check(rng, call, counts, 6)
    call = c.append(rng, [1, 1, 1], step=True)
    c.check_rows(call, [1, 1, 1])
    c.check(rng, call, [1, 1, 1], 6)
    call = c.append(rng, [0, 63, 60])
    c.check_rows(call, [0, 63, 60])
    c.check(rng, call, [0, 63, 60], 2)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 20])
def test_query_heads(ctx, group):
    rng = np.random.default_rng(group)
    c = Cache(ctx, 2, 600, 3, 64)
    c.append(rng, [300, 129])
    c.drop()
    call = c.append(rng, [1, 1], step=True)
    c.check(rng, call, [1, 1], 3 * group)
    call = c.append(rng, [5, 37])
    c.check(rng, call, [5, 37], 3 * group)


@pytest.mark.parametrize("length", [0, 1, 2, 31, 62, 63, 64, 65, 127, 128, 129, 191, 192, 1000])
def test_lengths(ctx, length):
    """One row, a step and portions at every place of a block."""
    rng = np.random.default_rng(length)
    for counts in ([1], [2], [63], [64], [65], [130]):
        c = Cache(ctx, 1, length + 140, 2, 32)
        if length:
            c.append(rng, [length])
            c.drop()
        call = c.append(rng, counts)
        c.check_rows(call, counts)
        c.check(rng, call, counts, 4)


def test_a_long_sequence(ctx):
    rng = np.random.default_rng(1)
    c = Cache(ctx, 1, 20000, 1, 128)
    c.append(rng, [19000])
    c.drop()
    call = c.append(rng, [1], step=True)
    c.check(rng, call, [1], 4)
    call = c.append(rng, [40])
    c.check(rng, call, [40], 4)


def test_many_sequences_of_all_lengths(ctx):
    rng = np.random.default_rng(2)
    n = 200
    c = Cache(ctx, n, 700, 2, 40)
    counts = np.where(rng.random(n) < 0.2, 0, rng.integers(1, 300, n))
    call = c.append(rng, counts)
    c.check_rows(call, counts)
    c.check(rng, call, counts[:0], 2)
    call = c.append(rng, np.ones(n, int), step=True)
    c.check_rows(call, np.ones(n, int))
    c.check(rng, call, np.ones(n, int), 8)


def test_however_the_rows_came(ctx):
    """Row by row, in portions or at once: the same cache bit for bit, and the same attention of the last row."""
    rng = np.random.default_rng(3)
    k, v = rng.standard_normal((333, 2, 48)).astype(np.float32), rng.standard_normal((333, 2, 48)).astype(np.float32)
    q = rng.standard_normal((1, 4, 48)).astype(np.float32)
    results = []
    for cuts in (list(range(334)), [0, 333], [0, 1, 64, 65, 190, 192, 300, 333], [0, 63, 127, 128, 332, 333], [0, 332, 333]):
        c = Cache(ctx, 1, 333, 2, 48)
        for a, b in zip(cuts, cuts[1:]):
            def put(kk, vv, a=a, b=b):
                kk[:], vv[:] = k[a:b], v[a:b]
            c.append(rng, [b - a], change=put)
            c.drop()
        whole = [c.dev(np.array(x, np.int32)) for x in ([0, 333], [0])]
        rows = c.read(whole[0], whole[1], 333)
        last = [c.dev(np.array(x, np.int32)) for x in ([0, 1], [332])]
        results.append((rows[0].view(np.uint32), rows[1].view(np.uint32), c.attend(rng, (last[0], last[1], 1), 4, q=q)[1].view(np.uint32)))
        c.drop()
    for r in results[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(r, results[0]))


def test_cut_back_and_go_on(ctx):
    """A sequence cut back into the block in front of its last one, then given other rows (what a rejected draft does)."""
    rng = np.random.default_rng(4)
    for length, back in ((200, 190), (200, 128), (195, 130), (130, 64), (64, 63), (64, 1), (128, 65), (70, 3)):
        c = Cache(ctx, 1, 400, 2, 32)
        c.append(rng, [length])
        c.drop()
        c.k[0], c.v[0] = c.k[0][:back], c.v[0][:back]
        call = c.append(rng, [1], step=True)
        c.check(rng, call, [1], 2)
        call = c.append(rng, [100])
        c.check_rows(call, [100])
        c.check(rng, call, [100], 2)


def test_strides_and_scale(ctx):
    rng = np.random.default_rng(5)
    for pad in (1, 3, 4, 96):
        c = Cache(ctx, 2, 300, 2, 24)
        counts = [150, 70]
        call = c.append(rng, counts, pad=pad)
        c.check_rows(call, counts)
        c.check(rng, call, counts, 4, scale=0.7, pad=pad)


def test_values_at_their_ends(ctx):
    rng = np.random.default_rng(6)

    def change(k, v):
        k[:64] = 0.0                       # a block of zeros
        k[64:128, 0] *= np.float32(1e30)   # large, small and tiny blocks
        v[64:128, 1] *= np.float32(1e-30)
        v[128:192, 0] = np.float32(1e-42)
        k[130, 0, 3] = np.float32(50.0)    # an outlier
        v[192:256] = np.where(v[192:256] > 0, np.float32(1.0), np.float32(-1.0))
        k[200, 1] = np.float32(0.5) * k[192:256, 1].max() / 127  # half a step
    c = Cache(ctx, 1, 300, 2, 16)
    call = c.append(rng, [290], change=change)
    c.check_rows(call, [290])


def test_what_is_not_finite_stays_in_its_block_and_head(ctx):
    rng = np.random.default_rng(7)

    def change(k, v):
        k[70, 0, 3] = np.nan    # block 1 of head 0
        v[130, 1, 2] = np.inf   # block 2 of head 1
        k[200, 1, 0] = -np.inf  # block 3 of head 1, open
    c = Cache(ctx, 1, 300, 2, 16)
    call = c.append(rng, [205], change=change)
    got_k, got_v = c.read(*call)
    assert np.isnan(got_k[64:128, 0]).all() and np.isfinite(got_k[64:128, 1]).all() and np.isfinite(got_k[:64]).all() and np.isfinite(got_k[128:192]).all()
    assert np.isnan(got_v[128:192, 1]).all() and np.isfinite(got_v[128:192, 0]).all()
    _, out = c.attend(rng, call, 4)
    bad = ~np.isfinite(out).all(2)  # heads 0, 1 read head 0
    assert not bad[:64].any()
    assert bad[64:, :2].all()
    assert not bad[:128, 2:].any() and bad[128:, 2:].all()
    c.drop()
    # a query that is not finite: its own row alone
    c = Cache(ctx, 1, 300, 2, 16)
    call = c.append(rng, [100])
    q = rng.standard_normal((100, 4, 16)).astype(np.float32)
    q[50, 1, 3], q[60, 2, 0] = np.nan, np.inf
    _, out = c.attend(rng, call, 4, q=q)
    bad = ~np.isfinite(out).all(2)
    assert bad[50, 1] and bad[60, 2] and bad.sum() == 2
    c.drop()


def test_zero_and_large_queries(ctx):
    rng = np.random.default_rng(8)
    c = Cache(ctx, 1, 300, 1, 16)
    call = c.append(rng, [200])
    q = rng.standard_normal((200, 2, 16)).astype(np.float32)
    q[:50] = 0.0
    q[50:100] *= np.float32(1e-30)
    q[100:150] *= np.float32(30.0)
    _, out = c.attend(rng, call, 2, q=q)
    want, tol = kit.attend(q, kit.held(c.k[0]), kit.held(c.v[0]), 0)
    assert (np.abs(out - want) <= tol).all(), (np.abs(out - want) / tol).max()
    c.drop()


def test_rows_without_room(ctx):
    """Rows past max_len are not taken, the call's other sequences are; sync says so once."""
    rng = np.random.default_rng(9)
    c = Cache(ctx, 3, 100, 1, 16)
    c.append(rng, [90, 90, 90])
    c.drop()
    counts = [10, 11, 5]
    k = rng.standard_normal((26, 1, 16)).astype(np.float32)
    starts, lengths = c.dev(np.array([0, 10, 21, 26], np.int32)), c.dev(c.lengths())
    c.kv.append(26, lengths, c.dev(k), c.dev(k), starts=starts)
    with pytest.raises(LoomB200Error) as e:
        ctx.sync()
    assert e.value.code == cabi.ERR_INVALID and "8-bit cache" in str(e.value)
    ctx.sync()
    for s in (0, 2):
        at = [0, 10, 21][s]
        c.k[s], c.v[s] = np.concatenate([c.k[s], k[at:at + counts[s]]]), np.concatenate([c.v[s], k[at:at + counts[s]]])
    q = rng.standard_normal((26, 2, 16)).astype(np.float32)
    out = c.dev(np.full((26, 2, 16), 3.5, np.float32))
    c.kv.attend(26, 2, lengths, c.dev(q), out, starts=starts)
    got = ctx.download(out, (26, 2, 16), np.float32)
    with pytest.raises(LoomB200Error):
        ctx.sync()
    assert (got[10:21] == 0).all()
    for s, a in ((0, 0), (2, 21)):
        want, tol = kit.attend(q[a:a + counts[s]], kit.held(c.k[s]), kit.held(c.v[s]), 90)
        assert (np.abs(got[a:a + counts[s]] - want) <= tol).all()
    c.drop()


def test_starts_that_do_not_ascend_or_pass_the_rows(ctx):
    rng = np.random.default_rng(10)
    c = Cache(ctx, 4, 100, 1, 8)
    k = rng.standard_normal((20, 1, 8)).astype(np.float32)
    starts, lengths = c.dev(np.array([-3, 5, 2, 8, 99], np.int32)), c.dev(np.zeros(4, np.int32))  # sequences: rows 0-4, none, 2-7, 8-19
    c.kv.append(20, lengths, c.dev(k), c.dev(k), starts=starts)
    ctx.sync()
    out = c.dev(np.zeros((20, 1, 8), np.float32))
    c.kv.attend(20, 1, lengths, c.dev(k), out, starts=starts)
    got = ctx.download(out, (20, 1, 8), np.float32)
    want, tol = kit.attend(k[8:], k[8:].astype(np.float64), k[8:].astype(np.float64), 0)
    assert (np.abs(got[8:] - want) <= tol).all()
    ctx.sync()
    c.drop()


def check_some(c, rng, call, counts, heads, most=40, scale=0.0):
    """A call's rows against the plain implementation: the first and last ones of every sequence, and some between them."""
    q, got = c.attend(rng, call, heads, scale)
    at = 0
    for s, n in enumerate(counts):
        first = len(c.k[s]) - n
        k, v = kit.held(c.k[s]), kit.held(c.v[s])
        for j in sorted({0, n - 1, *rng.integers(0, n, min(n, most)).tolist()} if n else {}):
            want, tol = kit.attend(q[at + j:at + j + 1], k, v, first + j, scale or None)
            off = np.abs(got[at + j] - want[0])
            assert (off <= tol[0]).all(), (s, j, n, first, (off / tol[0]).max())
        at += n
    return q, got


@pytest.mark.parametrize("heads, kv_heads, dim", [(20, 5, 128), (6, 2, 72), (7, 1, 96), (16, 16, 32), (9, 3, 50), (64, 1, 128)])
@pytest.mark.parametrize("before, count", [(0, 65), (1000, 257), (63, 128), (640, 49), (2900, 300)])
def test_portions(ctx, heads, kv_heads, dim, before, count):
    rng = np.random.default_rng(before + count + dim)
    c = Cache(ctx, 1, before + count, kv_heads, dim)
    if before:
        c.append(rng, [before], spread=2.0)
    call = c.append(rng, [count])
    check_some(c, rng, call, [count], heads, 12)
    c.drop()


def test_more_tiles_than_ctas(ctx):
    """Portions of which a CTA takes several, and single rows beside them; again, bit for bit."""
    rng = np.random.default_rng(20)
    c = Cache(ctx, 5, 1700, 8, 64)
    c.append(rng, [100, 0, 37, 64, 200])
    counts = [1500, 1, 400, 0, 90]
    call = c.append(rng, counts)
    q, got = check_some(c, rng, call, counts, 48, 15)
    for _ in range(3):
        assert np.array_equal(c.attend(rng, call, 48, q=q)[1], got)
    c.drop()


@pytest.mark.parametrize("dim", [32, 128])
def test_query_heads_that_are_many(ctx, dim):
    """One row a sequence, without starts, of more heads than the kernel for few rows takes."""
    rng = np.random.default_rng(dim)
    c = Cache(ctx, 4, 700, 1, dim)
    c.append(rng, [600, 3, 64, 255])
    call = c.append(rng, [1, 1, 1, 1], step=True)
    c.check(rng, call, [1, 1, 1, 1], 150)


def test_a_portion_with_rows_that_are_not_finite(ctx):
    """Keys, values and queries; what is not finite reaches the rows that see it, and no others."""
    rng = np.random.default_rng(21)

    def change(k, v):
        k[300, 0, 3] = np.nan
        v[310, 1, 2] = np.inf
        k[20, 1, 5] = np.inf
    c = Cache(ctx, 1, 1000, 2, 64)
    c.append(rng, [650])
    call = c.append(rng, [330], change=change)  # positions 650 .. 979, blocks 10 .. 15; 960 on are open
    q = rng.standard_normal((330, 8, 64)).astype(np.float32)
    q[7, 2, 1] = np.nan
    _, out = c.attend(rng, call, 8, q=q)
    bad = ~np.isfinite(out).all(2)
    want = np.zeros((330, 8), bool)
    want[7, 2] = True
    pos = np.arange(330) + 650
    want[pos >= (650 + 300) // 64 * 64, :4] = True  # a whole block reads as not-a-numbers
    want[pos >= (650 + 20) // 64 * 64, 4:] = True
    want[pos >= 960, 4:] = True
    assert np.array_equal(bad, want), np.argwhere(bad != want)[:5]
    for h in (0, 3):
        for j in (0, 100, 240):
            o, tol = kit.attend(q[j:j + 1], kit.held(c.k[0]), kit.held(c.v[0]), 650 + j)
            assert (np.abs(out[j, h] - o[0, h]) <= tol[0, h]).all()
    c.drop()


def test_open_rows_that_are_not_finite(ctx):
    rng = np.random.default_rng(22)

    def change(k, v):
        k[40, 0, 3] = np.nan
        v[50, 1, 2] = -np.inf
    c = Cache(ctx, 1, 200, 2, 64)
    c.append(rng, [64])
    call = c.append(rng, [60], change=change)
    q, out = c.attend(rng, call, 8)
    bad = ~np.isfinite(out).all(2)
    want = np.zeros((60, 8), bool)
    want[40:, :4] = True
    want[50:, 4:] = True
    assert np.array_equal(bad, want)
    for j in (0, 39, 49):
        o, tol = kit.attend(q[j:j + 1], kit.held(c.k[0]), kit.held(c.v[0]), 64 + j)
        good = ~bad[j]
        assert (np.abs(out[j, good] - o[0, good]) <= tol[0, good]).all()
    c.drop()


@pytest.mark.parametrize("spread", [1e-30, 1e-4, 1e4, 1e15])
def test_portions_of_small_and_large_values(ctx, spread):
    """Keys by `spread`, queries by its inverse: the same scores, whatever power of two stands in between."""
    rng = np.random.default_rng(23)
    c = Cache(ctx, 1, 400, 1, 64)
    call = c.append(rng, [200], change=lambda k, v: np.multiply(k, np.float32(spread), out=k))
    q = (rng.standard_normal((200, 4, 64)) / spread).astype(np.float32)
    _, got = c.attend(rng, call, 4, q=q)
    for j in (0, 63, 64, 150, 199):
        o, tol = kit.attend(q[j:j + 1], kit.held(c.k[0]), kit.held(c.v[0]), j)
        assert (np.abs(got[j] - o[0]) <= tol[0]).all()
    c.drop()


@pytest.mark.parametrize("n, dim", [(300, 64), (700, 32)])
def test_hundreds_of_sequences(ctx, n, dim):
    """Single rows, few rows and portions, over more sequences than a CTA's threads look at together."""
    rng = np.random.default_rng(n)
    c = Cache(ctx, n, 400, 2, dim)
    call = c.append(rng, rng.integers(0, 130, n))
    counts = np.where(rng.random(n) < 0.1, 0, rng.integers(1, 12, n))
    counts[[5, n // 2, n - 1]] = 100, 40, 70
    call = c.append(rng, counts)
    assert call[2] > 2 * n
    check_some(c, rng, call, counts, 16, 1)
    c.check_rows(call, counts)
    counts = np.ones(n, int)
    counts[7] = 30  # few rows a sequence on the average, and many of one
    call = c.append(rng, counts)
    check_some(c, rng, call, counts, 16, 1)
    c.drop()


def test_one_row_of_several_sequences(ctx):
    """Starts that go back, so that one row is three sequences' (more blocks than the call's rows can touch where they ascend)."""
    rng = np.random.default_rng(31)
    c = Cache(ctx, 6, 200, 2, 32)
    starts, lengths = c.dev(np.array([0, 1, 0, 1, 0, 1, 1], np.int32)), c.dev(np.zeros(6, np.int32))
    row = rng.standard_normal((1, 2, 32)).astype(np.float32)
    c.kv.append(1, lengths, c.dev(row), c.dev(row), starts=starts)
    for s in range(0, 6, 2):
        one = np.zeros(7, np.int32)
        one[s + 1:] = 1
        got = c.read(c.dev(one), lengths, 1)
        assert np.array_equal(got[0], row) and np.array_equal(got[1], row), s
    # a hundred rows three times: blocks that are whole, and open rows
    k = rng.standard_normal((100, 2, 32)).astype(np.float32)
    starts = c.dev(np.array([0, 100, 0, 100, 0, 100, 100], np.int32))
    c.kv.append(100, lengths, c.dev(k), c.dev(-k), starts=starts)
    for s in range(0, 6, 2):
        one = np.zeros(7, np.int32)
        one[s + 1:] = 100
        got = c.read(c.dev(one), lengths, 100)
        assert np.array_equal(got[0], kit.held(k, exact=False)) and np.array_equal(got[1], kit.held(-k, exact=False)), s
    c.drop()


def test_frames_and_repeats():
    """A recorded step replayed with new lengths, beside another frame of the same cache: the same bits as eager calls."""
    rng = np.random.default_rng(11)
    ctx = loom_b200.Context(0)
    try:
        runs = []
        for recorded in (False, True):
            r2 = np.random.default_rng(12)
            c = Cache(ctx, 5, 2000, 2, 128)
            c.append(r2, [1500, 3, 700, 64, 1])
            c.drop()
            base = c.lengths()
            steps = [[r2.standard_normal((5, 2, 128)).astype(np.float32) for _ in "kv"] + [r2.standard_normal((5, 8, 128)).astype(np.float32)] for _ in range(6)]
            lengths, k, v, q, out = c.dev(base), c.dev(steps[0][0]), c.dev(steps[0][1]), c.dev(steps[0][2]), c.dev(np.zeros((5, 8, 128), np.float32))

            def call():
                c.kv.append(5, lengths, k, v)
                c.kv.attend(5, 8, lengths, q, out)
            frames = []
            if recorded:
                for _ in range(2):
                    ctx.graph_begin()
                    call()
                    frames.append(ctx.graph_end())
            got = []
            for i, (kk, vv, qq) in enumerate(steps):
                for buf, a in ((lengths, base + i), (k, kk), (v, vv), (q, qq)):
                    ctx.upload(buf, a.astype(np.int32) if buf == lengths else a)
                for _ in range(2):  # (a step again is the same step)
                    ctx.graph_launch(frames[i % 2]) if recorded else call()
                got.append(ctx.download(out, (5, 8, 128), np.uint32))
            runs.append(got)
            for f in frames:
                ctx.graph_free(f)
            c.drop()
            c.kv.free()
        assert all(np.array_equal(a, b) for a, b in zip(*runs))
    finally:
        ctx.close()


def test_portions_in_frames():
    """A recorded call of up to 200 rows, replayed with other starts and lengths: portions, single rows, nothing; the same bits as eager calls."""
    ctx = loom_b200.Context(0)
    try:
        runs = []
        for recorded in (False, True):
            rng = np.random.default_rng(13)
            c = Cache(ctx, 3, 1000, 2, 64)
            c.append(rng, [300, 0, 64])
            c.drop()
            q, out = c.dev(rng.standard_normal((200, 8, 64)).astype(np.float32)), c.dev(np.zeros((200, 8, 64), np.float32))
            k = c.dev(rng.standard_normal((200, 2, 64)).astype(np.float32))
            lengths, starts = c.dev(c.lengths()), c.dev(np.zeros(4, np.int32))

            def call():
                c.kv.append(200, lengths, k, k, starts=starts)
                c.kv.attend(200, 8, lengths, q, out, starts=starts)
            frame = None
            if recorded:
                ctx.graph_begin()
                call()
                frame = ctx.graph_end()
            held, got = c.lengths(), []
            for counts in ([150, 49, 1], [1, 1, 1], [0, 0, 0], [0, 200, 0], [13, 12, 170], [200, 0, 0]):
                ctx.upload(lengths, held)
                ctx.upload(starts, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
                for _ in range(2):  # (a step again is the same step)
                    ctx.graph_launch(frame) if recorded else call()
                got.append(ctx.download(out, (200, 8, 64), np.uint32))
                held = (held + np.array(counts)).astype(np.int32)
            ctx.sync()
            if frame:
                ctx.graph_free(frame)
            runs.append(got)
            c.drop()
            c.kv.free()
        assert all(np.array_equal(a, b) for a, b in zip(*runs))
    finally:
        ctx.close()
