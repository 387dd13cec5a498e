"""Sampling against the plain form, one row at a time: sizes around every cluster and slice, settings at their ends, rows with ties, masks,
infinities and not-a-numbers, strides, repeats and recorded frames.  Tokens are equal; log probabilities to two float32 roundings and the
weights' own unit (vocab 2^-43 of the kept weight)."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit

pytestmark = pytest.mark.gpu
FMIN = np.finfo(np.float32).min


@pytest.fixture(scope="module")
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


def run(ctx, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, stride=None, offset=0):
    """logits [rows, vocab] put `stride` floats apart, `offset` floats into a buffer of not-a-numbers."""
    rows, vocab = logits.shape
    stride = vocab if stride is None else stride
    flat = np.full(offset + rows * stride + 8, np.nan, np.float32)
    for r in range(rows):
        flat[offset + r * stride:][:vocab] = logits[r]
    full = lambda v, kind: None if v is None else ctx.to_device(np.broadcast_to(np.asarray(v, kind), (rows,)))  # noqa: E731
    buf = ctx.to_device(flat)
    args = [full(u, np.float32), full(temperature, np.float32), full(top_k, np.int32), full(top_p, np.float32), full(min_p, np.float32)]
    tok, lp = ctx.to_device(np.full(rows, -77, np.int32)), ctx.to_device(np.full(rows, 55, np.float32))
    ctx.sample(rows, vocab, buf + 4 * offset, args[0], tok, temperature=args[1], top_k=args[2], top_p=args[3], min_p=args[4], logprob=lp, stride=stride)
    out = ctx.download(tok, (rows,), np.int32), ctx.download(lp, (rows,), np.float32)
    ctx.sync()
    for a in (buf, tok, lp, *args):
        if a is not None:
            ctx.free(a)
    return out


def check(ctx, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **where):
    rows, vocab = logits.shape
    tok, lp = run(ctx, logits, u, temperature, top_k, top_p, min_p, **where)
    full = lambda v: np.broadcast_to(np.asarray(v), (rows,))  # noqa: E731
    u, t, k, p, m = full(u), full(temperature), full(top_k), full(top_p), full(min_p)
    for r in range(rows):
        want, wlp = kit.sample(logits[r], t[r], k[r], p[r], m[r], u[r])
        assert tok[r] == want, (r, tok[r], want, t[r], k[r], p[r], m[r], u[r])
        assert np.isnan(wlp) == np.isnan(lp[r])
        if not np.isnan(wlp):
            assert abs(lp[r] - wlp) <= 2.0 ** -23 * abs(wlp) + vocab * 2.0 ** -43 + 1e-30, (r, lp[r], wlp)


def settings(rng, rows):
    return dict(u=rng.random(rows, np.float32), temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5], rows), top_k=rng.choice([0, 1, 2, 7, 40, 300], rows),
                top_p=rng.choice([1.0, 0.99, 0.9, 0.5, 0.05], rows), min_p=rng.choice([0.0, 0.0, 0.01, 0.2], rows))


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 32, 33, 100, 511, 1025, 4096, 8191, 8192, 8193, 16385, 32003, 65537, 128256, 131073, 250001, 655360])
def test_sizes(ctx, vocab):
    rng = np.random.default_rng(vocab)
    rows = 12 if vocab < 50000 else 5
    logits = rng.standard_normal((rows, vocab)).astype(np.float32) * rng.choice([0.5, 2.0, 5.0], (rows, 1)).astype(np.float32)
    check(ctx, logits, **settings(rng, rows))


def test_many_rows(ctx):
    rng = np.random.default_rng(0)
    logits = rng.standard_normal((700, 1500)).astype(np.float32) * 3
    check(ctx, logits, **settings(rng, 700))


@pytest.mark.parametrize("levels", [1, 2, 3, 17])
@pytest.mark.parametrize("vocab", [50, 2000, 40000])
def test_ties(ctx, levels, vocab):
    """Few different logits: the limits fall into ties, some of more values than one CTA ranks; equal weights make every sum exact."""
    rng = np.random.default_rng(levels * vocab)
    logits = rng.integers(0, levels, (24, vocab)).astype(np.float32)
    logits[::2] *= 0.0  # all equal
    logits[::4] *= -1.0  # and of either sign
    n = 24
    check(ctx, logits, rng.random(n, np.float32), rng.choice([0.0, 0.5, 1.0], n), rng.choice([0, 1, 3, vocab // 2, vocab - 1, vocab, vocab + 5], n),
          rng.choice([1.0, 0.5, 0.25, 0.125], n), rng.choice([0.0, 1.0], n))


@pytest.mark.parametrize("vocab", [3000, 128256])
def test_masked_rows(ctx, vocab):
    rng = np.random.default_rng(7)
    base = rng.standard_normal(vocab).astype(np.float32) * 2
    rows = []
    for fill in (-np.inf, FMIN, -1e9, np.nan):
        for left in (0, 1, 2, 50, vocab // 2):
            row = np.full(vocab, fill, np.float32)
            at = rng.choice(vocab, left, replace=False)
            row[at] = base[at]
            rows.append(row)
    logits = np.stack(rows)
    n = len(rows)
    for k, p, m in ((0, 1.0, 0.0), (40, 1.0, 0.0), (0, 0.9, 0.0), (40, 0.9, 0.0), (vocab - 1, 0.999, 0.0), (0, 1.0, 0.05), (7, 0.5, 0.05)):
        check(ctx, logits, rng.random(n, np.float32), 0.8, k, p, m)
    check(ctx, logits, 0.5, 0.0)


@pytest.mark.parametrize("vocab", [40, 20000])
def test_infinities(ctx, vocab):
    rng = np.random.default_rng(3)
    logits = rng.standard_normal((8, vocab)).astype(np.float32)
    logits[0, [3, 17, 30]] = np.inf
    logits[1, 5] = np.inf
    logits[2] = np.inf
    logits[3, ::2] = -np.inf
    logits[4, 1:] = -np.inf
    logits[5] = -np.inf
    logits[6] = np.nan
    logits[7, 9], logits[7, 8] = np.inf, np.nan
    for u in (0.0, 0.4, 0.999):
        for t in (0.0, 0.5, np.inf):
            for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 0.7, 0.0), (3, 0.6, 0.3)):
                check(ctx, logits, u, t, k, p, m)


def test_settings_at_their_ends(ctx):
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((6, 5000)).astype(np.float32) * 4
    u = np.array([0.0, 1e-45, 0.25, 0.5, 0.99999, 0.99999994], np.float32)
    for t in (1e-38, 1e-10, 1e-3, 50.0, 1e30, 3e38):
        for k, p, m in ((0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.5, 0.0), (100, 0.5, 0.5)):
            check(ctx, logits, u, t, k, p, m)
    for p in (0.0, 1e-45, 1e-9, 0.99999994, 1.0, 2.0, np.inf, -1.0):
        check(ctx, logits, u, 1.0, 0, p, 0.0)
    for m in (1e-30, 0.999, 1.0, 5.0, -1.0):
        check(ctx, logits, u, 1.0, 0, 1.0, m)
    for k in (-5, 0, 1, 4999, 5000, 2 ** 31 - 1):
        check(ctx, logits, u, 1.0, k)
    # settings that are not numbers: no temperature is the largest logit, the others are off; a random number of 1 or more is the
    # last token with any weight (all have some here), one below 0 or that is none the first
    nan = np.float32(np.nan)
    assert np.array_equal(run(ctx, logits, u, nan)[0], logits.argmax(1))
    assert np.array_equal(run(ctx, logits, u, 1.0, 0, nan, nan)[0], run(ctx, logits, u)[0])
    assert run(ctx, logits, [-1.0, nan, 1.0, 7.0, np.inf, 0.0])[0].tolist() == [0, 0, 4999, 4999, 4999, 0]


@pytest.mark.parametrize("vocab,stride,offset", [(1000, 1000, 1), (1001, 1003, 0), (33000, 33001, 3), (128256, 128256, 2), (7, 300, 0)])
def test_strides(ctx, vocab, stride, offset):
    rng = np.random.default_rng(stride)
    logits = rng.standard_normal((4, vocab)).astype(np.float32) * 3
    check(ctx, logits, rng.random(4, np.float32), 0.9, 50, 0.95, 0.0, stride=stride, offset=offset)
    check(ctx, logits, rng.random(4, np.float32), 0.9, 0, 0.95, 0.0, stride=stride, offset=offset)


def test_repeats_and_recorded_frame():
    """Two frames and eager calls on one context: the same tokens bit for bit; a frame reads its buffers anew at every replay."""
    rng = np.random.default_rng(5)
    ctx = loom_b200.Context(0)
    try:
        sets = []
        for vocab in (32000, 128256):
            rows = 9
            logits = rng.standard_normal((rows, vocab)).astype(np.float32) * 3
            d = dict(rows=rows, vocab=vocab, host=logits, logits=ctx.to_device(logits), u=ctx.to_device(rng.random(rows, np.float32)), tok=ctx.alloc(rows * 4), lp=ctx.alloc(rows * 4),
                     p=ctx.to_device(np.full(rows, 0.95, np.float32)), k=ctx.to_device(np.full(rows, 200, np.int32)))
            d["call"] = lambda d=d: ctx.sample(d["rows"], d["vocab"], d["logits"], d["u"], d["tok"], top_k=d["k"], top_p=d["p"], logprob=d["lp"])
            d["get"] = lambda d=d: (ctx.download(d["tok"], (d["rows"],), np.int32), ctx.download(d["lp"], (d["rows"],), np.uint32))
            sets.append(d)
        frames, want = [], []
        for d in sets:
            d["call"]()
            want.append(d["get"]())
            ctx.graph_begin()
            d["call"]()
            frames.append(ctx.graph_end())
        for _ in range(20):
            for i in (0, 1):
                ctx.zero(sets[i]["tok"], 36)
                ctx.graph_launch(frames[i])
            for i in (0, 1):
                got = sets[i]["get"]()
                assert np.array_equal(got[0], want[i][0]) and np.array_equal(got[1], want[i][1])
        fresh = rng.standard_normal((9, 32000)).astype(np.float32) * 3
        u = rng.random(9, np.float32)
        ctx.upload(sets[0]["logits"], fresh)
        ctx.upload(sets[0]["u"], u)
        ctx.graph_launch(frames[0])
        assert sets[0]["get"]()[0].tolist() == [kit.sample(fresh[r], 1.0, 200, 0.95, 0.0, u[r])[0] for r in range(9)]
        for f in frames:
            ctx.graph_free(f)
    finally:
        ctx.close()
