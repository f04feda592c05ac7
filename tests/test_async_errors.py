"""An error that a kernel leaves after its call has returned (a wait that ran
out inside matmul_q8) comes from the next call that waits, once, whichever
that is: no token is taken from logits that were never finished."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

import titania_b200 as tb
from titania_b200 import _lib, build

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def wait_out(tmp_path_factory):
    """Enqueues a kernel whose one wait runs out after about a second (wait_out.cu)."""
    so = str(tmp_path_factory.mktemp("wait_out") / "wait_out.so")
    subprocess.run([build.NVCC, *build.ARCH, *build.FLAGS, "-shared", "-cudart", "static", "-o", so,
                    os.path.join(HERE, "wait_out.cu")], check=True, capture_output=True)
    f = ctypes.CDLL(so).wait_out
    f.argtypes, f.restype = [ctypes.c_void_p], ctypes.c_int
    return f


def test_the_helper_builds(wait_out):
    assert wait_out


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["sync", "read", "write", "argmax", "matmul", "read_q8", "write_q8", "sample",
                                  "sampler_state", "score"])
def test_the_next_call_that_waits_reports(b200, wait_out, name):
    x, q = b200.alloc(256), b200.q8(4, 64)
    w, out = b200.upload(tb.Tensor([8, 64], np.full((8, 64), 0x3F80, np.uint16))), b200.alloc(4 * 8)
    sampler, scorer = tb.DeviceSampler(b200, 1, 256, 1.0, 5, 0.9, [1]), tb.LogProbs(b200, 1, 256, 3)
    call = {
        "sync": b200.sync,
        "read": lambda: b200.read(x),
        "write": lambda: b200.write(x, np.ones(256, np.float32)),
        "argmax": lambda: b200.argmax(x),
        "matmul": lambda: b200.matmul(out, w, x),
        "read_q8": lambda: b200.read_q8(q),
        "write_q8": lambda: b200.write_q8(q, np.ones((4, 64), np.int8), np.ones(4, np.float32)),
        "sample": lambda: sampler.sample(x),
        "sampler_state": sampler.states,
        "score": lambda: scorer.score(x, [1]),
    }[name]
    call()
    b200.sync()
    assert wait_out(b200._h) == 0
    spare = b200.alloc(4)  # neither making nor freeing a handle takes the report away
    del spare
    with pytest.raises(tb.DeviceError, match="timed out") as e:
        call()
    assert e.value.code == _lib.TB200_ERR_TIMEOUT
    call()  # once
    b200.sync()
