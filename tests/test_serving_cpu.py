"""Sampling, adapters and the 8-bit cache: calls that are refused before they reach a device, and the plain forms against each other."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import servingkit as kit
from loom_b200 import build, cabi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = cabi.ERR_INVALID, cabi.ERR_UNSUPPORTED
P = 4096  # an address that nothing reads


@pytest.fixture(scope="module")
def fakes(tmp_path_factory):
    build.build()
    out = str(tmp_path_factory.mktemp("h") / "refusal_harness.so")
    flags = [f for f in build.NVCC_FLAGS if f not in ("-Xptxas", "-v")]
    subprocess.run([build.nvcc(), *flags, "-shared", "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, os.path.join(ROOT, "tests", "refusal_harness.cu"), "-o", out], check=True)
    h = C.CDLL(out)
    for name in ("t_context", "t_adapters", "t_kv8"):
        getattr(h, name).restype = C.c_void_p
    ctx, other, rec = h.t_context(0), h.t_context(0), h.t_context(1)
    vp = C.c_void_p
    return dict(L=cabi.lib(), ctx=ctx, other=other, rec=rec, ad=h.t_adapters(vp(ctx), 4, 48, 32, 8), kv=h.t_kv8(vp(ctx), 3, 2, 16))


def refused(f, rc, code, word, ctx=None):
    assert rc == code
    text = (f["L"].loom_b200_last_error(f["ctx"] if ctx is None else ctx) or b"").decode()
    assert word in text, text


def test_sample_refusals(fakes):
    f, s = fakes, fakes["L"].loom_b200_sample
    ok = dict(ctx=f["ctx"], rows=2, vocab=10, logits=P, stride=10, t=None, k=None, p=None, m=None, u=P, out=P, lp=None)
    call = lambda **w: s(*{**ok, **w}.values())  # noqa: E731
    assert call(ctx=None) == INVALID
    refused(f, call(rows=0), INVALID, "0 rows")
    refused(f, call(vocab=0), INVALID, "of 0 logits")
    refused(f, call(logits=None), INVALID, "NULL")
    refused(f, call(u=None), INVALID, "NULL")
    refused(f, call(out=None), INVALID, "NULL")
    refused(f, call(stride=9), INVALID, "stride 9")
    refused(f, call(vocab=655361, stride=655361), UNSUPPORTED, "655360")


def test_adapter_refusals(fakes):
    f, L, out = fakes, fakes["L"], C.c_void_p()
    create = lambda *a: L.loom_b200_adapters_create(f["ctx"], *a, C.byref(out))  # noqa: E731
    assert L.loom_b200_adapters_create(None, 1, 1, 1, 1, 1, C.byref(out)) == INVALID
    refused(f, L.loom_b200_adapters_create(f["ctx"], 1, 1, 1, 1, 1, None), INVALID, "out is NULL")
    for bad in ((0, 8, 8, 8, 1), (1, 0, 8, 8, 1), (1, 8, 0, 8, 1), (1, 8, 8, 0, 1)):
        refused(f, create(*bad), INVALID, "slots")
    refused(f, create(1, 8, 8, 8, 2), INVALID, "dtype 2")
    refused(f, create(1, 8, 8, 257, 1), UNSUPPORTED, "rank 257")
    refused(f, create(4097, 8, 8, 8, 1), UNSUPPORTED, "4097 slots")
    refused(f, L.loom_b200_adapters_create(f["rec"], 1, 8, 8, 8, 1, C.byref(out)), INVALID, "recorded", f["rec"])
    put = lambda *a, ctx=f["ctx"]: L.loom_b200_adapters_put(ctx, f["ad"], *a)  # noqa: E731
    refused(f, put(4, 8, 1.0, P, P, 0, 1), INVALID, "slot 4")
    refused(f, put(-1, 8, 1.0, P, P, 0, 1), INVALID, "slot -1")
    refused(f, put(0, 9, 1.0, P, P, 0, 1), INVALID, "rank 9")
    refused(f, put(0, 8, 1.0, None, P, 0, 1), INVALID, "NULL")
    refused(f, put(0, 8, 1.0, P, P, 5, 1), INVALID, "dtype 5")
    refused(f, put(0, 8, 1.0, P, P, 0, 1, ctx=f["other"]), INVALID, "another context", f["other"])
    ok = dict(ctx=f["ctx"], a=f["ad"], tokens=3, slot=P, x=P, ldx=32, base=None, out=P)
    call = lambda **w: L.loom_b200_adapters_apply(*{**ok, **w}.values())  # noqa: E731
    refused(f, call(tokens=0), INVALID, "0 tokens")
    refused(f, call(ldx=31), INVALID, "31 floats")
    refused(f, call(tokens=(1 << 22) + 1), UNSUPPORTED, "tokens")
    for name in ("a", "slot", "x", "out"):
        refused(f, call(**{name: None}), INVALID, "NULL")
    refused(f, call(ctx=f["other"]), INVALID, "another context", f["other"])
    assert L.loom_b200_adapters_info(None, None, None, None, None, None) == INVALID


def test_cache_refusals(fakes):
    f, L, out = fakes, fakes["L"], C.c_void_p()
    create = lambda *a: L.loom_b200_kv8_create(f["ctx"], *a, C.byref(out))  # noqa: E731
    assert L.loom_b200_kv8_create(None, 1, 1, 1, 1, C.byref(out)) == INVALID
    refused(f, L.loom_b200_kv8_create(f["ctx"], 1, 1, 1, 1, None), INVALID, "out is NULL")
    for bad in ((0, 64, 1, 8), (1, 0, 1, 8), (1, 64, 0, 8), (1, 64, 1, 0)):
        refused(f, create(*bad), INVALID, "sequences")
    refused(f, create(1, 64, 1, 257), UNSUPPORTED, "257")
    refused(f, create(4097, 64, 1, 8), UNSUPPORTED, "4097")
    refused(f, L.loom_b200_kv8_create(f["rec"], 1, 64, 1, 8, C.byref(out)), INVALID, "recorded", f["rec"])
    append = dict(ctx=f["ctx"], c=f["kv"], rows=3, starts=None, lengths=P, k=P, v=P, ld=32)
    attend = dict(ctx=f["ctx"], c=f["kv"], rows=3, heads=4, starts=None, lengths=P, q=P, ldq=64, scale=0.0, out=P)
    read = dict(ctx=f["ctx"], c=f["kv"], rows=3, starts=None, lengths=P, k=P, v=P)
    for entry, ok in (("append", append), ("attend", attend), ("read", read)):
        call = lambda **w: getattr(L, "loom_b200_kv8_" + entry)(*{**ok, **w}.values())  # noqa: E731
        refused(f, call(rows=0), INVALID, "0 rows")
        refused(f, call(rows=4), INVALID, "4 rows without starts")
        refused(f, call(lengths=None), INVALID, "NULL")
        refused(f, call(c=None), INVALID, "NULL")
        refused(f, call(ctx=f["other"]), INVALID, "another context", f["other"])
        assert call(ctx=None) == INVALID
    refused(f, L.loom_b200_kv8_append(*{**append, "ld": 31}.values()), INVALID, "31 floats")
    refused(f, L.loom_b200_kv8_attend(*{**attend, "heads": 3}.values()), INVALID, "3 query heads over 2")
    refused(f, L.loom_b200_kv8_attend(*{**attend, "ldq": 63}.values()), INVALID, "63 floats")
    refused(f, L.loom_b200_kv8_attend(*{**attend, "scale": float("nan")}.values()), INVALID, "scale")
    refused(f, L.loom_b200_kv8_attend(*{**attend, "starts": P, "rows": 1 << 29}.values()), INVALID, "rows")


def test_decoder_sample_without_a_decoder():
    assert cabi.lib().loom_b200_decoder_sample(None, -1, None, None, None, None, P, P, None) == INVALID


def test_plain_sampling_is_the_distribution():
    """The plain sampler over a fine comb of random numbers gives every token its share."""
    rng = np.random.default_rng(0)
    row = rng.standard_normal(9).astype(np.float32) * 2
    n = 20000
    got = np.bincount([kit.sample(row, 0.9, 7, 0.97, 0.01, (i + 0.5) / n)[0] for i in range(n)], minlength=9) / n
    w = np.exp((row.astype(np.float64) - row.max()) / np.float64(np.float32(0.9)))
    order = np.argsort(-row, kind="stable")[:7]
    mass = np.cumsum(w[order]) / w[order].sum()
    kept = order[:int(np.searchsorted(mass, np.float32(0.97))) + 1]
    kept = kept[w[kept] >= np.float32(0.01)]
    share = np.zeros(9)
    share[kept] = w[kept] / w[kept].sum()
    assert np.abs(got - share).max() <= 1.01 / n  # (a share of n points begins and ends between two of them)


def test_plain_cache_rows_are_within_half_a_step():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((150, 2, 24)).astype(np.float32)
    held = kit.held(x)
    for b in (0, 64):
        for h in range(2):
            blk = x[b:b + 64, h].astype(np.float64)
            assert np.abs(held[b:b + 64, h] - blk).max() <= np.abs(blk).max() / 127 / 2 * (1 + 1e-12)
    assert np.array_equal(held[128:], x[128:])
