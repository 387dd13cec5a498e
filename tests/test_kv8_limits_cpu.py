"""Calls on the 8-bit cache whose work does not fit into the counters: refused before they reach a device."""
import ctypes as C
import os
import subprocess

import pytest

from loom_b200 import build, cabi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # an address that nothing reads


@pytest.fixture(scope="module")
def fakes(tmp_path_factory):
    build.build()
    out = str(tmp_path_factory.mktemp("h") / "kv8_limits_harness.so")
    flags = [f for f in build.NVCC_FLAGS if f not in ("-Xptxas", "-v")]
    subprocess.run([build.nvcc(), *flags, "-shared", "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, os.path.join(ROOT, "tests", "kv8_limits_harness.cu"), "-o", out], check=True)
    h = C.CDLL(out)
    h.t_context.restype = h.t_kv8.restype = C.c_void_p
    return h, cabi.lib(), C.c_void_p(h.t_context())


def work(blocks, group, counts, pos, kv_heads, tile=8, open_cost=6):
    """What the list of work of a kernel for few rows counts up to."""
    total = 0
    for n, at in zip(counts, pos):
        load = (at + n - 1) // 64 + 1 + (open_cost if (at + n) % 64 else 0)
        total += kv_heads * -(-n * group // tile) * load
    return total


@pytest.mark.parametrize("kv_heads", [5, 8, 15])
def test_open_blocks_count(fakes, kv_heads):
    """Short sequences whose open block is most of their work: 64 rows of 4095 heads for a KV head each."""
    h, lib, ctx = fakes
    cache = C.c_void_p(h.t_kv8(ctx, 4096, 64, kv_heads, 1))
    rows, group = 1 << 18, 4095  # 64 rows a sequence fill it; 63 leave an open block
    counts = [63] * 4096
    real = work(1, group, counts, [0] * 4096, kv_heads)
    assert real >= 2 ** 32
    rc = lib.loom_b200_kv8_attend(ctx, cache, rows, kv_heads * group, P, P, P, kv_heads * group, 0.0, P)
    assert rc == cabi.ERR_UNSUPPORTED and b"fewer rows" in lib.loom_b200_last_error(ctx)


def test_tiles_of_a_portion_for_every_sequence(fakes):
    h, lib, ctx = fakes
    cache = C.c_void_p(h.t_kv8(ctx, 4096, 64, 8, 1))
    rows, group = 1 << 15, 512
    assert 8 * 2 * (rows * group / 8 + 8 * 4096) < 2 ** 31 <= 8 * 4096 * rows * group / 128
    rc = lib.loom_b200_kv8_attend(ctx, cache, rows, 8 * group, P, P, P, 8 * group, 0.0, P)
    assert rc == cabi.ERR_UNSUPPORTED and b"fewer rows" in lib.loom_b200_last_error(ctx)


def test_the_longest_sequence(fakes):
    _, lib, ctx = fakes
    out = C.c_void_p()
    rc = lib.loom_b200_kv8_create(ctx, 1, (1 << 29) + 1, 1, 8, C.byref(out))
    assert rc == cabi.ERR_UNSUPPORTED and b"536870912 at most" in lib.loom_b200_last_error(ctx)
    assert ((1 << 29) // 64 + 1 + 6) * 2 * 148 < 2 ** 32  # a tile's load times parts, as many as CTAs
