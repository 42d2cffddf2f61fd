"""perf/operators.py: the framework's side of the cases keeps in step with torch's
stream, which makes their inputs and takes their memory back."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = [
    {"kind": "norm", "rows": 300, "n": 2048, "residual": True, "f32": True, "wtype": "f32"},
    {"kind": "linear", "tokens": 200, "in": 2048, "out": 1024, "scales": "f32", "y": "f32"},
    {"kind": "up", "h": 512, "E": 16, "K": 4, "ff": 256, "tokens": 500, "skew": "none"},
    {"kind": "down", "h": 512, "E": 16, "K": 4, "ff": 256, "tokens": 500, "skew": "none", "y": "f32"},
    {"kind": "mix", "tokens": 400, "h": 2048, "K": 8, "x": "f32", "residual": True},
]


@pytest.fixture(scope="module")
def cases():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, root)
    try:
        import perf.operators as o
    finally:
        sys.path.remove(root)
    o.own = True
    yield o
    o.own = False
    if o.OPEN:
        o.OPEN["batch"].finish()
        o.OPEN["gpu"].close()
        o.OPEN.clear()


def outputs(v):
    return [t.view(torch.uint8) for _, t in sorted(v.items())] if isinstance(v, dict) else [v.view(torch.uint8)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["kind"])
def test_a_pass_right_after_its_inputs_and_a_state_dropped_in_flight(cases, case):
    s = cases.prepare(case, 1)
    torch.cuda.synchronize()
    want = cases.run(s)
    torch.cuda.synchronize()
    want = [t.clone() for t in outputs(want)]
    del s
    busy = torch.randn(8192, 8192, device="cuda")
    for _ in range(3):
        for _ in range(4):
            busy = busy @ busy * 1e-4                 # torch's stream is behind when the pass is issued
        s = cases.prepare(case, 1)
        got = cases.run(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outputs(got)))
        for _ in range(20):
            got = cases.run(s)
        kept = got                                    # outputs outlive the state, whole
        del s, got
        other = [torch.full((1 << 20,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(64)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outputs(kept)))
        assert all(bool((t == 0x55).all()) for t in other)
        del other, kept
