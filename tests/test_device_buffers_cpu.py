"""Sampling, adapters and the 8-bit cache take buffers on the device only: arrays and tensors of the host, other types and gaps are refused, before
their addresses reach a kernel."""
import numpy as np
import pytest
import torch

from loom_b200 import cabi


class OnDevice:
    """A tensor that says it is on a GPU."""

    is_cuda = True

    def __init__(self, dtype, at=4096, contiguous=True):
        self.dtype, self.at, self.whole = dtype, at, contiguous

    def data_ptr(self):
        return self.at

    def is_contiguous(self):
        return self.whole

    def stride(self):
        return (1, 2)


F, I = OnDevice(torch.float32, 4096), OnDevice(torch.int32, 8192)


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, a)) or 0


@pytest.fixture()
def calls(monkeypatch):
    library = Library()
    monkeypatch.setattr(cabi, "lib", lambda: library)
    ctx = cabi.Context.__new__(cabi.Context)
    ctx.__dict__.update(h=1, device=0)

    def make(kind, **sizes):
        o = kind.__new__(kind)
        o.__dict__.update(ctx=ctx, h=2, **sizes)
        return o
    kv, ad = make(cabi.KV8, kv_heads=2, head_dim=8), make(cabi.Adapters, rows=5, cols=6)
    yield library.calls, {
        "sample": (lambda **b: ctx.sample(2, 9, **b), dict(logits=F, uniform=F, tokens=I, temperature=F, top_k=I, top_p=F, min_p=F, logprob=F)),
        "apply": (lambda **b: ad.apply(2, **b), dict(slot=I, x=F, out=F, base=F)),
        "append": (lambda **b: kv.append(2, **b), dict(lengths=I, k=F, v=F, starts=I)),
        "read": (lambda **b: kv.read(2, **b), dict(lengths=I, k=F, v=F, starts=I)),
        "attend": (lambda **b: kv.attend(2, 4, **b), dict(lengths=I, q=F, out=F, starts=I)),
    }
    kv.h = ad.h = ctx.h = None  # (nothing to free)


@pytest.mark.parametrize("name", ["sample", "apply", "append", "read", "attend"])
def test_buffers(calls, name):
    seen, entries = calls
    call, good = entries[name]
    call(**good)
    call(**{n: b.at for n, b in good.items()})
    assert len(seen) == 2 and seen[0] == seen[1]  # addresses or tensors: the same call
    assert [a for a in seen[0][1] if a in (4096, 8192)].count(8192) == sum(b is I for b in good.values())
    for n, b in good.items():
        floats = b is F
        for bad in (np.zeros(4, np.float32 if floats else np.int32), torch.zeros(4), [1, 2], OnDevice(torch.int64), OnDevice(torch.float64), OnDevice(torch.bfloat16),
                    OnDevice(torch.int32 if floats else torch.float32)):
            with pytest.raises(TypeError):
                call(**{**good, n: bad})
        with pytest.raises(ValueError):
            call(**{**good, n: OnDevice(b.dtype, contiguous=False)})
    assert len(seen) == 2
