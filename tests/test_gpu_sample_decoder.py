"""What sampling on a decoder draws from: only logits of the position that a sequence is at."""
import numpy as np
import pytest

import loom_b200
import servingkit as kit
from loom_b200 import LoomB200Error, cabi
from test_gpu_serving import stack_decoder, ternary_decoder

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ctx():
    c = loom_b200.Context(0)
    yield c
    c.close()


def refused(dec, word="no logits", **how):
    with pytest.raises(LoomB200Error) as e:
        dec.sample([0.5] * (1 if "seq" in how else dec.batch), 1.0, **how)
    assert e.value.code == cabi.ERR_INVALID and word in str(e.value)


def test_a_cache_that_was_uploaded_or_cut(ctx):
    rng = np.random.default_rng(0)
    dec = ternary_decoder(ctx, rng, 1)
    try:
        refused(dec, "no prompt")
        prompt = rng.integers(0, 300, 9).astype(np.int32)
        dec.forward(prompt)
        dec.sample([0.5], 1.0)
        k, v = dec.cache(0)
        dec.set_kv_offset(9)  # where it is
        dec.sample([0.5], 1.0)
        dec.set_kv_offset(6)
        refused(dec)
        logits = dec.extend(prompt[6:7], [0])[0]
        assert dec.sample([0.3], 0.8)[0][0] == kit.sample(logits, 0.8, u=0.3)[0]
        dec.upload_cache(0, 7, k[:7], v[:7])  # the same position, by other rows
        refused(dec)
        dec.extend(prompt[7:])
        dec.sample([0.5], 1.0)
        dec.reset()
        refused(dec, "no prompt")
    finally:
        dec.close()


@pytest.mark.parametrize("make", [ternary_decoder, stack_decoder])
def test_every_way_forward_leaves_logits(ctx, make):
    """Prompts without a place that is wanted, steps, greedy loops: what is drawn is what the same tokens' logits give."""
    rng = np.random.default_rng(1)
    dec, other = make(ctx, np.random.default_rng(5), 3), make(ctx, np.random.default_rng(5), 1)
    vocab = dec.dims.vocab
    try:
        seen = []
        for i, n in enumerate((1, 7, 40)):
            dec.select(i)
            seen.append(rng.integers(0, vocab, n).tolist())
            dec.extend(seen[i])
            if i < 2:
                refused(dec, "no prompt")

        def compare():
            u = rng.random(3, np.float32)
            got = dec.sample(u, 0.9)[0].tolist()
            for i in range(3):
                other.reset()
                logits = other.extend(seen[i], [len(seen[i]) - 1])[0]
                assert got[i] == kit.sample(logits, 0.9, u=u[i])[0]
        compare()
        tokens = rng.integers(0, vocab, 3).astype(np.int32)
        dec.step_batch(tokens, want_logits=False)
        seen = [s + [int(t)] for s, t in zip(seen, tokens)]
        compare()
        dec.continue_batch(2)
        for s, t in zip(seen, dec.generated_tokens_batch(2)):
            s += t.tolist()
        compare()
        dec.select(0)
        dec.reset()
        refused(dec, "no prompt", seq=0)
        dec.sample([0.5], 1.0, seq=2)
    finally:
        dec.close()
        other.close()
