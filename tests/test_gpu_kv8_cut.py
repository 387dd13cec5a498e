"""Sequences of the 8-bit cache that are cut back again and again: which rows they go on from, bit for bit, and attention over them."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from loom_b200 import cabi

pytestmark = pytest.mark.gpu
BLOCK = kit.BLOCK


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


class Sequence:
    """What one sequence's rows are: those of the blocks that were written last, of an even and of an odd number, as they came; a cut into any
    other block goes on from its rows as the 8-bit form holds them."""

    def __init__(self, heads, dim):
        self.rows = [np.zeros((0, heads, dim), np.float32) for _ in "kv"]
        self.places, self.whole = [None, None], {}

    def __len__(self):
        return len(self.rows[0])

    def cut(self, length):
        b, left = divmod(length, BLOCK)
        for i, r in enumerate(self.rows):
            r = r[:length].copy()
            if left and self.places[b & 1] != b:
                r[b * BLOCK:] = self.whole[b][i][:left]
            self.rows[i] = r

    def append(self, new):
        first, last = len(self) // BLOCK, (len(self) + len(new[0]) - 1) // BLOCK
        self.rows = [np.concatenate([r, x]) for r, x in zip(self.rows, new)]
        for b in range(first, last + 1):
            if (b + 1) * BLOCK <= len(self):
                self.whole[b] = [kit.held(r[b * BLOCK:(b + 1) * BLOCK], exact=False) for r in self.rows]
        for b in range(max(first, last - 1), last + 1):
            self.places[b & 1] = b


class Run:
    def __init__(self, ctx, seqs, max_len, kv_heads, dim):
        self.ctx, self.kv, self.kv_heads, self.dim = ctx, cabi.KV8(ctx, seqs, max_len, kv_heads, dim), kv_heads, dim
        self.seqs = [Sequence(kv_heads, dim) for _ in range(seqs)]

    def step(self, rng, counts, heads, starts=True, call=None):
        """counts[s] new rows each; compares what the cache holds of them, all that it holds, and the attention of first, middle and last rows.
        call: stands in for append and attend."""
        ctx, n = self.ctx, int(np.sum(counts))
        new = [rng.standard_normal((n, self.kv_heads, self.dim)).astype(np.float32) for _ in "kv"]
        q = rng.standard_normal((n, heads, self.dim)).astype(np.float32)
        edges = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        before = [len(s) for s in self.seqs]
        host = dict(lengths=np.array(before, np.int32), starts=edges, k=new[0], v=new[1], q=q)
        dev = {name: ctx.to_device(a) for name, a in host.items()}
        out = ctx.to_device(np.zeros((n, heads, self.dim), np.float32))
        given = dict(starts=dev["starts"]) if starts else {}
        if call:
            got = call(n, host)
        else:
            self.kv.append(n, dev["lengths"], dev["k"], dev["v"], **given)
            self.kv.attend(n, heads, dev["lengths"], dev["q"], out, **given)
            got = ctx.download(out, (n, heads, self.dim), np.float32)
        for s, seq in enumerate(self.seqs):
            if counts[s]:
                seq.append([x[edges[s]:edges[s + 1]] for x in new])
        total = [len(s) for s in self.seqs]
        everything, none = np.concatenate([[0], np.cumsum(total)]).astype(np.int32), np.zeros(len(total), np.int32)
        dev["all"], dev["none"] = ctx.to_device(everything), ctx.to_device(none)
        back = [ctx.to_device(np.zeros((sum(total), self.kv_heads, self.dim), np.float32)) for _ in "kv"]
        self.kv.read(sum(total), dev["none"], *back, starts=dev["all"])
        held = [ctx.download(b, (sum(total), self.kv_heads, self.dim), np.float32) for b in back]
        ctx.sync()
        for b in (*dev.values(), out, *back):
            ctx.free(b)
        for s, seq in enumerate(self.seqs):
            if not counts[s]:
                continue  # (what a cut without new rows leaves is seen with the next ones)
            for h, mine in zip(held, seq.rows):
                assert np.array_equal(h[everything[s]:everything[s + 1]], kit.held(mine, exact=False)), (s, before[s], counts[s])
            for j in sorted({0, counts[s] // 2, counts[s] - 1}):
                r = edges[s] + j
                want, tol = kit.attend(q[r:r + 1], kit.held(seq.rows[0]), kit.held(seq.rows[1]), before[s] + j)
                assert (np.abs(got[r] - want[0]) <= tol[0]).all(), (s, before[s], j)


@pytest.mark.parametrize("dim", [20, 128, 200])
def test_two_cuts_across_blocks(ctx, dim):
    """330 positions, back to 260, on by one, back to 200: rows 192 to 199 are no longer there as they came."""
    rng = np.random.default_rng(dim)
    for whole, cuts in ((330, [(260, 1), (200, 1), (199, 70)]), (130, [(70, 1), (60, 4), (50, 90)]), (130, [(70, 58), (128, 3), (100, 1)]),
                        (500, [(20, 10), (10, 200), (3, 1)]), (1000, [(901, 1), (130, 130), (129, 2), (128, 1), (65, 64)])):
        c = Run(ctx, 1, 1100, 2, dim)
        c.step(rng, [whole], 4)
        for back, more in cuts:
            c.seqs[0].cut(back)
            c.step(rng, [more], 4, starts=more > 1)
        c.kv.free()


@pytest.mark.parametrize("seed", range(6))
def test_cuts_in_any_order(ctx, seed):
    rng = np.random.default_rng(seed)
    n = 5
    c = Run(ctx, n, 420, [1, 3][seed % 2], [32, 64, 96][seed % 3])
    c.step(rng, rng.integers(1, 300, n), 6)
    for _ in range(12):
        for s in c.seqs:
            if rng.random() < 0.7:
                s.cut(int(rng.integers(0, len(s) + 1)))
        room = [c.kv.max_len - len(s) for s in c.seqs]
        counts = [min(r, int(rng.choice([0, 1, 1, 5, 63, 64, 130]))) for r in room]
        if sum(counts):
            c.step(rng, counts, 6)


def test_cuts_in_a_recorded_frame():
    """One recorded append and attention, replayed for every step of a sequence that goes forth and back."""
    rng = np.random.default_rng(9)
    ctx = loom_b200.Context(0)
    try:
        rows, heads, kv_heads, dim = 70, 4, 2, 64
        c = Run(ctx, 1, 700, kv_heads, dim)
        c.step(rng, [330], heads)
        d = dict(lengths=ctx.to_device(np.zeros(1, np.int32)), starts=ctx.to_device(np.zeros(2, np.int32)), k=ctx.to_device(np.zeros((rows, kv_heads, dim), np.float32)),
                 v=ctx.to_device(np.zeros((rows, kv_heads, dim), np.float32)), q=ctx.to_device(np.zeros((rows, heads, dim), np.float32)))
        out = ctx.to_device(np.zeros((rows, heads, dim), np.float32))
        ctx.graph_begin()
        c.kv.append(rows, d["lengths"], d["k"], d["v"], starts=d["starts"])
        c.kv.attend(rows, heads, d["lengths"], d["q"], out, starts=d["starts"])
        frame = ctx.graph_end()

        def replay(n, host):
            for name, a in host.items():
                full = np.zeros((rows, *a.shape[1:]), a.dtype) if a.ndim == 3 else a
                full[:len(a)] = a
                ctx.upload(d[name], full)
            ctx.graph_launch(frame)
            return ctx.download(out, (rows, heads, dim), np.float32)[:n]
        for back, more in ((260, 1), (200, 1), (201, 70), (140, 2), (30, 70), (100, 1), (101, 1), (0, 70)):
            c.seqs[0].cut(back)
            c.step(rng, [more], heads, call=replay)
        ctx.graph_free(frame)
    finally:
        ctx.close()


def test_a_cut_into_a_block_that_is_not_finite(ctx):
    """Its rows are gone: what they go on from reads as not-a-numbers, in that head and side alone, until the block begins anew."""
    rng = np.random.default_rng(3)
    kv, zero = cabi.KV8(ctx, 1, 400, 2, 32), ctx.to_device(np.zeros(1, np.int32))
    k, v = (rng.standard_normal((330, 2, 32)).astype(np.float32) for _ in "kv")
    k[70, 1, 5] = np.inf

    def append(kk, vv, at):
        starts, lengths = ctx.to_device(np.array([0, len(kk)], np.int32)), ctx.to_device(np.array([at], np.int32))
        kv.append(len(kk), lengths, ctx.to_device(kk), ctx.to_device(vv), starts=starts)

    def held(n):
        out = [ctx.to_device(np.zeros((n, 2, 32), np.float32)) for _ in "kv"]
        kv.read(n, zero, *out, starts=ctx.to_device(np.array([0, n], np.int32)))
        return [ctx.download(o, (n, 2, 32), np.float32) for o in out]
    append(k, v, 0)
    append(k[90:91], v[90:91], 90)  # block 1, whose place block 5 has: 64 .. 89 from the codes
    got_k, got_v = held(91)
    assert np.isnan(got_k[64:90, 1]).all() and np.isfinite(got_k[:, 0]).all() and np.isfinite(got_k[:64]).all() and np.isfinite(got_v).all()
    assert np.array_equal(got_k[90], k[90]) and np.array_equal(got_v[90], v[90])
    assert np.array_equal(got_k[64:90, 0], kit.held(k, exact=False)[64:90, 0])
    fresh = rng.standard_normal((70, 2, 32)).astype(np.float32)
    append(fresh, fresh, 64)  # cut to the block's beginning
    got_k, _ = held(134)
    assert np.array_equal(got_k[64:], kit.held(np.concatenate([k[:64], fresh]), exact=False)[64:])
    ctx.sync()
    kv.free()
