"""The greedy loop of one sequence after passes of others: it goes on from its own next token."""
import numpy as np
import pytest

import loom_b200
from test_gpu_serving import stack_decoder, ternary_decoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("make", [ternary_decoder, stack_decoder])
def test_a_greedy_loop_after_other_sequences(make):
    ctx = loom_b200.Context(0)
    rng = np.random.default_rng(1)
    dec, alone = make(ctx, np.random.default_rng(5), 3), make(ctx, np.random.default_rng(5), 1)
    try:
        prompts = [rng.integers(0, dec.dims.vocab, n).astype(np.int32) for n in (1, 7, 40)]
        want = []
        for p in prompts:
            want.append(alone.generate(p, 12)[0].tolist())
        for i, p in enumerate(prompts):
            dec.select(i)
            dec.forward(p, want_logits=False)
        fed = [[], [], []]
        for i, steps in ((0, 2), (1, 1), (None, 2), (1, 3), (2, 1), (0, 1), (None, 1), (2, 4)):
            if i is None:
                dec.continue_batch(steps)
                for f, t in zip(fed, dec.generated_tokens_batch(steps)):
                    f += t.tolist()
            else:
                dec.select(i)
                dec.continue_greedy(steps)
                fed[i] += dec.generated_tokens(steps).tolist()
            for f, w in zip(fed, want):
                assert f == w[:len(f)], (i, steps)
    finally:
        dec.close()
        alone.close()
        ctx.close()
