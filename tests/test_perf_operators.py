"""The workloads of perf/operators.py: what a pass over the framework returns can
be read in torch's own order, without waiting for the device."""

import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def workloads():
    torch = pytest.importorskip("torch")
    spec = importlib.util.spec_from_file_location("perf_operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    yield m
    torch.cuda.synchronize()
    torch.cuda.set_stream(torch.cuda.default_stream())


def leaves(v):
    return [x for k in sorted(v) for x in leaves(v[k])] if isinstance(v, dict) else (
        [x for e in v for x in leaves(e)] if isinstance(v, list) else [v])


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    {"op": "norm", "rows": 3, "cols": 200, "residual": True}, {"op": "quantize", "rows": 3, "cols": 200},
    {"op": "matmul", "rows": 2, "cols": 200, "channels": 30}, {"op": "logprobs", "rows": 3, "vocab": 700, "top": 4}],
    ids=lambda c: c["op"])
def test_outputs_are_in_torchs_order(workloads, case):
    """With the device's stream busy for a tenth of a second before the pass, what torch copies right after the pass
    is what it wrote, not what was there before."""
    import torch

    state = workloads.prepare(case, 5)
    before = [x.clone() for x in leaves(state["out"])]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(state["dev"].stream)):
        torch.cuda._sleep(200_000_000)
    out = leaves(workloads.run(state))
    copies = [x.clone() for x in out]
    torch.cuda.synchronize()
    for b, c, x in zip(before, copies, out):
        assert torch.equal(c, x) and not torch.equal(b, x)
