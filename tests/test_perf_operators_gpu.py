"""perf/operators.py calls the library on inputs that another stream is still making. In a process of its own: torch
brings its own HIP runtime, which has to be loaded before the library."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import torch
from perf import operators as O

case = {"kind": "linear", "rows": 8, "n": 96, "k": 64}
state, other = O.prepare(case, 1), O.prepare(case, 2)
fresh = lambda s: {**s, "y": torch.zeros_like(s["y"])}
want = O.run(fresh(other)).clone()
O.own = True
O.run(fresh(state))  # (the library is loaded)
torch.cuda.set_stream(torch.cuda.default_stream())
torch.cuda.synchronize()
torch.cuda._sleep(100_000_000)  # some 50 ms of the default stream, then the other inputs
for name in ("x", "sx", "w", "sw"):
    state[name].copy_(other[name])
got = O.run(state)
torch.cuda.synchronize()
off = (got.float() - want.float()).abs().max() / want.float().abs().max()
assert off <= 2.0 ** -10, float(off)
print("same inputs", flush=True)
"""


def test_a_first_call_waits_for_its_inputs():
    r = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True,
                       text=True, timeout=100)
    assert r.returncode == 0 and "same inputs" in r.stdout, r.stdout + r.stderr
