"""The low-bit operators whose very first call in a process is a captured one: loading a library and asking how many blocks the GPU holds come inside
the capture then.  A process of its own, so that no kernel has been used before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

SCRIPT = """
import sys
import torch
from llmengine_b200.kernels.ops import CudaOps
from llmengine_b200.weights.quantize import quantize_e4m3, quantize_int4

F8, dev = torch.float8_e4m3fn, torch.device("cuda:0")
ops = CudaOps(dev)
if sys.argv[1] != "auto":
    ops.low_bit_form(sys.argv[1])
x, gain = torch.randn(300, 512, device=dev), torch.ones(512, device=dev)
w = torch.randn(264, 512, device=dev)
x8, xs = quantize_e4m3(x)
w8, ws = quantize_e4m3(w)
packed, scales, zero = quantize_int4(w, 64, True)
xb = x.to(torch.bfloat16)
calls = []
for m in (1, 13, 40, 300):
    q, s, out8, out4 = torch.zeros(m, 512, dtype=F8, device=dev), torch.zeros(m, device=dev), torch.zeros(m, 264, device=dev), torch.zeros(m, 264, dtype=torch.bfloat16, device=dev)
    g = torch.zeros(m, 256, dtype=F8, device=dev)
    calls += [(lambda m=m, q=q, s=s: ops.rmsnorm_e4m3(x[:m], gain, 1e-6, q, s), (q, s)), (lambda m=m, q=q, s=s: ops.rows_e4m3(xb[:m], q, s), (q, s)),
              (lambda m=m, g=g, s=s: ops.swiglu_e4m3(xb[:m], g, s), (g, s)), (lambda m=m, o=out8: ops.linear_e4m3(x8[:m], xs[:m], w8, ws, o), (out8,)),
              (lambda m=m, o=out4: ops.linear_int4(xb[:m], packed, scales, o, zeros=zero), (out4,))]
torch.cuda.synchronize()
got = []
for call, outs in calls:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    graph.replay()
    torch.cuda.synchronize()
    got.append([o.float().clone() for o in outs])
for (call, outs), first in zip(calls, got):
    for o in outs:
        o.view(torch.uint8).zero_()
    call()
    for o, f in zip(outs, first):
        assert torch.equal(o.float(), f) and f.abs().max() > 0
print("FIRST CALLS CAPTURED", len(got))
"""


@pytest.mark.parametrize("form", ["auto", "wide", "pair"])
def test_first_calls_are_captured(form):
    env = dict(os.environ, PYTHONPATH=os.path.dirname(HERE) + os.pathsep + os.environ.get("PYTHONPATH", ""))
    done = subprocess.run([sys.executable, "-c", SCRIPT, form], env=env, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "FIRST CALLS CAPTURED 20" in done.stdout, done.stdout[-2000:] + done.stderr[-3000:]
