"""What Matrix.put and Adapters.put hand to the library: the element type is the values' own, and sizes are checked, whatever the caller says."""
import ctypes as C

import numpy as np
import pytest
import torch

from loom_b200 import cabi


class Library:
    """Takes the two calls and notes what they would read."""

    def __init__(self):
        self.seen = []

    def loom_b200_adapters_put(self, ctx, a, slot, rank, scale, down, up, dtype, on_device):
        read = lambda p, n: None if on_device or not p else bytes(C.string_at(p, n * (2 if dtype else 4)))  # noqa: E731
        self.seen.append((rank, dtype, on_device, read(down, rank * 6), read(up, rank * 5)))
        return 0

    def loom_b200_matrix_put(self, ctx, m, group, row0, rows, src, dtype, on_device):
        self.seen.append((rows, dtype, on_device, None if on_device else bytes(C.string_at(src, rows * 6 * (2 if dtype else 4)))))
        return 0


class Device:
    h, device = 1, 0

    def _check(self, rc):
        assert rc == 0


class OnDevice:
    """A tensor that says it is on a GPU."""

    is_cuda = True

    def __init__(self, shape, dtype="torch.bfloat16", index=0, contiguous=True):
        self.shape, self.dtype, self.device, self._c = shape, dtype, type("D", (), dict(index=index))(), contiguous

    def data_ptr(self):
        return 4096

    def is_contiguous(self):
        return self._c

    def contiguous(self):
        assert self._c
        return self

    def stride(self):
        return (1, 2)


@pytest.fixture()
def calls(monkeypatch):
    library = Library()
    monkeypatch.setattr(cabi, "lib", lambda: library)

    def make(kind, **sizes):
        o = kind.__new__(kind)
        o.__dict__.update(ctx=Device(), h=None, **sizes)
        return o
    return library, make(cabi.Adapters, slots=2, rows=5, cols=6, max_rank=4, dtype=cabi.DTYPE_BF16), make(cabi.Matrix, rows=5, cols=6, groups=1, dtype=cabi.DTYPE_BF16)


def pair(kind, rank=3):
    rng = np.random.default_rng(0)
    return rng.standard_normal((rank, 6)).astype(kind), rng.standard_normal((5, rank)).astype(kind)


def test_the_type_is_the_arrays(calls):
    library, adapters, matrix = calls
    down, up = pair(np.float32)
    adapters.put(0, down, up)
    assert library.seen[-1] == (3, cabi.DTYPE_F32, 0, down.tobytes(), up.tobytes())
    bits = [cabi.to_bf16(a) for a in (down, up)]
    for given in ((), (cabi.DTYPE_BF16,)):
        adapters.put(0, *bits, 1.0, *given)
        assert library.seen[-1] == (3, cabi.DTYPE_BF16, 0, bits[0].tobytes(), bits[1].tobytes())
    adapters.put(0, *pair(np.float64))
    assert library.seen[-1][1:4] == (cabi.DTYPE_F32, 0, pair(np.float64)[0].astype(np.float32).tobytes())
    adapters.put(0, down.T.copy().T, up[:, ::-1])  # rows that do not follow one another
    assert library.seen[-1][3:] == (down.tobytes(), up[:, ::-1].tobytes())
    matrix.put(bits[0])
    assert library.seen[-1] == (3, cabi.DTYPE_BF16, 0, bits[0].tobytes())
    matrix.put(down)
    assert library.seen[-1] == (3, cabi.DTYPE_F32, 0, down.tobytes())


def test_tensors(calls):
    library, adapters, matrix = calls
    down, up = (torch.from_numpy(a) for a in pair(np.float32))
    adapters.put(0, down, up)  # on the host
    assert library.seen[-1] == (3, cabi.DTYPE_F32, 0, down.numpy().tobytes(), up.numpy().tobytes())
    half = down.bfloat16()
    adapters.put(0, half, up.bfloat16())
    assert library.seen[-1][:4] == (3, cabi.DTYPE_BF16, 0, half.view(torch.int16).numpy().tobytes())
    matrix.put(half)
    assert library.seen[-1][:3] == (3, cabi.DTYPE_BF16, 0)
    adapters.put(0, OnDevice((3, 6)), OnDevice((5, 3)))
    assert library.seen[-1][:3] == (3, cabi.DTYPE_BF16, 1)
    matrix.put(OnDevice((3, 6), "torch.float32"), cabi.DTYPE_F32)
    assert library.seen[-1][:3] == (3, cabi.DTYPE_F32, 1)


def test_an_empty_slot(calls):
    library, adapters, _ = calls
    adapters.put(1, None, None)
    adapters.put(1, np.zeros((0, 6), np.float32), np.zeros((5, 0), np.float32))
    assert [s[0] for s in library.seen] == [0, 0]


@pytest.mark.parametrize("change", ["dtype", "bits as floats", "two types", "two places", "int", "half", "other device", "strides", "shape", "one"])
def test_refusals(calls, change):
    library, adapters, matrix = calls
    down, up = pair(np.float32)
    bits = cabi.to_bf16(down)
    bad = {"dtype": (down, up, 1.0, cabi.DTYPE_BF16), "bits as floats": (bits, cabi.to_bf16(up), 1.0, cabi.DTYPE_F32), "two types": (bits, up),
           "two places": (OnDevice((3, 6), "torch.float32"), up), "int": (down.astype(np.int32), up.astype(np.int32)),
           "half": (OnDevice((3, 6), "torch.float16"), OnDevice((5, 3), "torch.float16")), "other device": (OnDevice((3, 6), index=1), OnDevice((5, 3), index=1)),
           "strides": (OnDevice((3, 6), contiguous=False), OnDevice((5, 3))), "shape": (down, up.T), "one": (down, None)}[change]
    with pytest.raises(ValueError):
        adapters.put(0, *bad)
    if change not in ("two types", "two places", "shape", "one"):
        with pytest.raises(ValueError):
            matrix.put(bad[0], *bad[3:])
    with pytest.raises(ValueError):
        matrix.put(down, rows=4)
    assert not library.seen
