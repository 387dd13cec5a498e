"""Rows that an 8-bit cache does not take are reported, but not in the place of a wait that ran out before."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import loom_b200
from loom_b200 import LoomB200Error, build, cabi

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def status_of(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("h") / "status_harness.so")
    flags = [f for f in build.NVCC_FLAGS if f not in ("-Xptxas", "-v")]
    subprocess.run([build.nvcc(), *flags, "-shared", "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, os.path.join(ROOT, "tests", "status_harness.cu"), "-o", out], check=True)
    h = C.CDLL(out)
    h.t_status.restype = C.c_void_p
    h.t_status.argtypes = [C.c_void_p]
    return h.t_status


def test_a_wait_that_ran_out_stays(status_of):
    ctx = loom_b200.Context(0)
    try:
        kv = cabi.KV8(ctx, 2, 64, 1, 8)
        rows = ctx.to_device(np.ones((2, 1, 8), np.float32))
        lengths, out = ctx.to_device(np.full(2, 64, np.int32)), ctx.to_device(np.ones((2, 1, 8), np.float32))
        calls = [lambda: kv.append(2, lengths, rows, rows), lambda: kv.read(2, lengths, out, out), lambda: kv.attend(2, 1, lengths, rows, out)]
        for call in calls:
            for before, code in ((0, cabi.ERR_INVALID), (1, cabi.ERR_TIMEOUT)):
                ctx.upload(status_of(ctx.h), np.array([before], np.int32))
                call()
                with pytest.raises(LoomB200Error) as e:
                    ctx.sync()
                assert e.value.code == code, before
                ctx.sync()
    finally:
        ctx.close()
