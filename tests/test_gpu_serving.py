"""Sampling on decoders, and the operators of a serving step behind one another: rows into the 8-bit cache, attention over it, the shared
projection, the requests' adapters, logits, the next tokens."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import loom_b200
import servingkit as kit
import stackkit
from loom_b200 import LoomB200Error, cabi, models
from oracle import oracle as orc

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


def ternary_decoder(ctx, rng, batch, vocab=300):
    L, H, heads, kvh, hd, inter, msl = 2, 128, 4, 2, 32, 256, 96
    dec = cabi.Decoder(ctx, L, H, heads, kvh, hd, inter, vocab, 1e-5, 10000.0, cabi.ACT_SILU, msl)
    if batch > 1:
        dec.set_batch(batch)
    for b in range(L):
        ws = []
        for r, c in ((H, H), (kvh * hd, H), (kvh * hd, H), (H, H), (inter, H), (inter, H), (H, inter)):
            words, scale = orc.pack_f32((rng.standard_normal(r * c) * 0.02).astype(np.float32), r, c)
            ws.append(ctx.upload_ternary(words, r, c, scale))
        dec.set_block(b, ws)
    dec.set_embeddings(ctx.to_device((rng.standard_normal((vocab, H)) * 0.3).astype(np.float32)))
    return dec


def stack_decoder(ctx, rng, batch, vocab=120):
    cfg = stackkit.config(72, vocab, [stackkit.gla(2, 16, 24, 4.0, stackkit.dense(96)), stackkit.latent(3, 24, 16, 32, 0.3, stackkit.dense(96))])
    return models.build(ctx, cfg, stackkit.Weights(stackkit.random_weights(cfg, 3)), models.LoadOptions(cabi.DTYPE_F32, 96, batch=batch))


SETTINGS = dict(temperature=[0.7, 1.0, 0.0, 1.3, 0.9], top_k=[0, 40, 0, 5, 0], top_p=[0.9, 1.0, 1.0, 0.8, 0.95], min_p=[0.0, 0.05, 0.0, 0.0, 0.1])


def drawn(logits, u, **s):
    return [kit.sample(row, *(np.broadcast_to(s[k], (len(logits),))[i] for k in ("temperature", "top_k", "top_p", "min_p")), u[i]) for i, row in enumerate(logits)]


@pytest.mark.parametrize("make", [ternary_decoder, stack_decoder])
def test_sequences_draw_from_their_own_logits(ctx, make):
    rng = np.random.default_rng(0)
    dec = make(ctx, rng, 5)
    vocab = dec.dims.vocab
    try:
        logits = np.empty((5, vocab), np.float32)
        for i in range(5):
            dec.select(i)
            prompt = rng.integers(0, vocab, 3 + 9 * i).astype(np.int32)
            logits[i] = dec.extend(prompt, [len(prompt) - 1])[0]
        for step in range(8):
            u = rng.random(5, np.float32)
            tokens, logprob = dec.sample(u, **SETTINGS)
            want = drawn(logits, u, **SETTINGS)
            assert tokens.tolist() == [w[0] for w in want]
            assert np.allclose(logprob, [w[1] for w in want], rtol=2.0 ** -22, atol=1e-9)
            one, lp = dec.sample(u[3], 1.3, 5, 0.8, seq=3)  # the same of one sequence
            assert one[0] == tokens[3] and lp[0] == logprob[3]
            logits = dec.step_batch(tokens)
    finally:
        dec.close()


@pytest.mark.parametrize("make", [ternary_decoder, stack_decoder])
def test_one_sequence(ctx, make):
    """Prompts by either path (few tokens, a block), then steps whose frame is recorded; sampling changes nothing for greedy decoding."""
    rng = np.random.default_rng(1)
    dec = make(ctx, rng, 1)
    vocab = dec.dims.vocab
    try:
        with pytest.raises(LoomB200Error) as e:
            dec.sample([0.5], 1.0)
        assert e.value.code == cabi.ERR_INVALID and "no prompt" in str(e.value)
        for n in (1, 5, 40):
            prompt = rng.integers(0, vocab, n).astype(np.int32)
            greedy, _ = dec.generate(prompt, 6)
            dec.reset()  # (a forward of one token goes on with what is there)
            logits = dec.forward(prompt)
            token, lp = dec.sample([0.3])
            assert (token[0], 0) == (kit.sample(logits, u=0.3)[0], 0)
            mine = []
            for _ in range(6):  # a temperature of 0 is the greedy loop
                token, lp = dec.sample([0.9], 0.0)
                assert lp[0] == 0.0
                mine.append(int(token[0]))
                logits = dec.extend(token, [0])[0]
            assert mine == greedy.tolist()
            for _ in range(4):
                u = rng.random(1, np.float32)
                token, _ = dec.sample(u, 0.9, 50, 0.95, 0.02)
                assert token[0] == kit.sample(logits, 0.9, 50, 0.95, 0.02, u[0])[0]
                logits = dec.extend(token, [0])[0]
        with pytest.raises(LoomB200Error):
            dec.sample([0.5], seq=1)
    finally:
        dec.close()


def test_command_line_samples(tmp_path):
    cfg = stackkit.config(72, 120, [stackkit.gla(2, 16, 24, 4.0, stackkit.dense(96))])
    model = str(tmp_path / "model")
    stackkit.save(model, cfg, stackkit.random_weights(cfg, 2))
    base = [sys.executable, "-m", "loom_b200", "generate", "--model", model, "--dtype", "float32", "--max-new", "7", "--tokens", "3,4,5"]

    def lines(*more):
        r = subprocess.run(base + list(more), cwd=ROOT, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr
        return [json.loads(x)["tokens"] for x in r.stdout.splitlines()]

    greedy = lines()
    assert lines("--temperature", "1.0", "--top-k", "1") == greedy
    a, b = lines("--temperature", "1.5", "--tokens", "9,8", "--seed", "5"), lines("--temperature", "1.5", "--tokens", "9,8", "--seed", "5")
    assert a == b and len(a) == 2 and all(len(r) == 7 for r in a)
    assert a != lines("--temperature", "1.5", "--tokens", "9,8", "--seed", "6")


def test_a_serving_step(ctx):
    """Six requests with adapters of their own: a prompt portion and three steps, each stage against its plain form on the same input."""
    rng = np.random.default_rng(2)
    n, kv_heads, group, dim, vocab = 6, 2, 4, 32, 500
    width, heads = kv_heads * group * dim, kv_heads * group
    master = (rng.standard_normal(vocab * width) * 0.02).astype(np.float32)
    words, scale = orc.pack_f32(master, vocab, width)
    w = ctx.upload_ternary(words, vocab, width, scale)
    adapters, host = cabi.Adapters(ctx, 3, vocab, width, 8, cabi.DTYPE_F32), []
    for i in range(3):
        down, up = (rng.standard_normal((4 + i, width)) / 16).astype(np.float32), rng.standard_normal((vocab, 4 + i)).astype(np.float32)
        adapters.put(i, down, up, 0.5)
        host.append((down, up, 0.5))
    slot = np.array([2, -1, 0, 0, 1, 2], np.int32)
    cache = cabi.KV8(ctx, n, 200, kv_heads, dim)
    lengths = np.zeros(n, np.int32)
    past = [[np.zeros((0, kv_heads, dim), np.float32)] * 2 for _ in range(n)]
    try:
        for step in range(4):
            counts = np.array([70, 1, 0, 64, 33, 5]) if step == 0 else np.ones(n, int)
            rows = int(counts.sum())
            starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
            k, v = (rng.standard_normal((rows, kv_heads, dim)).astype(np.float32) for _ in "kv")
            q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
            dev = {name: ctx.to_device(a) for name, a in dict(starts=starts, lengths=lengths, k=k, v=v, q=q, slot=np.repeat(slot, counts).astype(np.int32),
                                                             u=rng.random(rows, np.float32)).items()}
            att, qi, amax, base, logits, tok = (ctx.alloc(s) for s in (rows * width * 4, rows * width, rows * 4, rows * vocab * 4, rows * vocab * 4, rows * 4))
            cache.append(rows, dev["lengths"], dev["k"], dev["v"], starts=dev["starts"])
            cache.attend(rows, heads, dev["lengths"], dev["q"], att, starts=dev["starts"])
            ctx.quantize_activation(rows, width, att, qi, amax)
            ctx.ternary_linear(w, rows, qi, amax, base)
            adapters.apply(rows, dev["slot"], att, logits, base=base)
            ctx.sample(rows, vocab, logits, dev["u"], tok, temperature=None, top_k=None)
            ctx.sync()
            got = {name: ctx.download(b, shape, kind) for name, b, shape, kind in (("att", att, (rows, heads, dim), np.float32), ("base", base, (rows, vocab), np.float32),
                   ("logits", logits, (rows, vocab), np.float32), ("tok", tok, (rows,), np.int32), ("u", dev["u"], (rows,), np.float32))}
            at = 0
            for s in range(n):
                m = counts[s]
                past[s] = [np.concatenate([p, x[at:at + m]]) for p, x in zip(past[s], (k, v))]
                if m:
                    want, tol = kit.attend(q[at:at + m], kit.held(past[s][0]), kit.held(past[s][1]), lengths[s])
                    assert (np.abs(got["att"][at:at + m] - want) <= tol).all()
                for r in range(at, at + m):
                    if slot[s] < 0:
                        assert np.array_equal(got["logits"][r], got["base"][r])
                    else:
                        want, tol = kit.adapter(got["att"][r].ravel(), *host[slot[s]], got["base"][r])
                        assert (np.abs(got["logits"][r] - want) <= tol).all()
                    assert got["tok"][r] == kit.sample(got["logits"][r], u=got["u"][r])[0]
                at += m
            lengths = (lengths + counts).astype(np.int32)
            for b in (*dev.values(), att, qi, amax, base, logits, tok):
                ctx.free(b)
    finally:
        cache.free()
        adapters.free()


def test_two_contexts_at_once():
    """Two contexts with streams of their own, every call of one beside a call of the other: each has what it has alone.  (Portions begin with a
    block, so that a call again is the same call.)"""
    rng = np.random.default_rng(3)
    kv_heads, heads, dim, seqs, rows, vocab = 2, 8, 64, 4, 260, 40000
    counts = np.array([200, 1, 59, 0])
    host = dict(starts=np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), lengths=np.array([128, 700, 0, 64], np.int32),
                k=rng.standard_normal((rows, kv_heads * dim)).astype(np.float32), q=rng.standard_normal((rows, heads * dim)).astype(np.float32),
                logits=(4 * rng.standard_normal((8, vocab))).astype(np.float32), u=rng.random(8, np.float32), slot=rng.integers(-1, 2, rows).astype(np.int32))
    down, up = rng.standard_normal((9, heads * dim)).astype(np.float32), rng.standard_normal((333, 9)).astype(np.float32)

    class One:
        def __init__(self):
            self.ctx = ctx = loom_b200.Context(0)
            self.dev = {n: ctx.to_device(a) for n, a in host.items()}
            self.kv, self.ad = cabi.KV8(ctx, seqs, 1000, kv_heads, dim), cabi.Adapters(ctx, 2, 333, heads * dim, 9)
            self.ad.put(0, down, up, 0.25)
            old = ctx.to_device(np.random.default_rng(4).standard_normal((892, kv_heads * dim)).astype(np.float32))
            zero, starts = ctx.to_device(np.zeros(seqs, np.int32)), ctx.to_device(np.array([0, 128, 828, 828, 892], np.int32))
            self.kv.append(892, zero, old, old, starts=starts)
            self.att, self.out, self.tok, self.lp = (ctx.to_device(np.zeros(n, np.float32)) for n in (rows * heads * dim, rows * 333, 8, 8))
            ctx.sync()
            for b in (old, zero, starts):
                ctx.free(b)

        def calls(self):
            d = self.dev
            return [lambda: self.kv.append(rows, d["lengths"], d["k"], d["k"], starts=d["starts"]),
                    lambda: self.kv.attend(rows, heads, d["lengths"], d["q"], self.att, starts=d["starts"]),
                    lambda: self.ad.apply(rows, d["slot"], self.att, self.out),
                    lambda: self.ctx.sample(8, vocab, d["logits"], d["u"], self.tok, logprob=self.lp)]

        def results(self):
            return [self.ctx.download(b, (n,), np.uint32) for b, n in ((self.att, rows * heads * dim), (self.out, rows * 333), (self.tok, 8), (self.lp, 8))]

        def close(self):
            self.ctx.sync()
            self.kv.free()
            self.ad.free()
            self.ctx.close()
    one, two = One(), One()
    try:
        for c in one.calls():
            c()
        alone = one.results()
        for _ in range(20):
            for c, d in zip(one.calls(), two.calls()):
                c()
                d()
        for o in (one, two):
            assert all(np.array_equal(a, b) for a, b in zip(o.results(), alone))
            o.ctx.sync()
    finally:
        one.close()
        two.close()
