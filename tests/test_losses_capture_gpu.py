"""A call of the losses may be the first of its kind on a device and be captured: nothing has to be called before a capture.
In a process of its own, in which no kernel of theirs has run."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = r"""
import sys
sys.path.insert(0, %(root)r)
import torch
from graph_rws_b200.layers import distillation_loss, linear_cross_entropy

def body(x, w, y, reduction, grad):
    loss = linear_cross_entropy(x, w, y, reduction=reduction)
    return (loss.detach(),) + torch.autograd.grad(loss, (x, w), grad)

def soft(z, t, ids, grad):
    loss = distillation_loss(z, t, ids, temperature=2.0)
    return (loss.detach(),) + torch.autograd.grad(loss, z, grad)

calls = []
for dtype in (torch.bfloat16, torch.float16, torch.float32):
    for n, d, V in ((100, 72, 1003), (700, 136, 1003), (40, 16, 9)):
        x = torch.randn(n, d, device="cuda").to(dtype).requires_grad_(True)
        w = torch.randn(d, V, device="cuda").to(dtype).requires_grad_(True)
        y = torch.randint(0, V, (n,), device="cuda")
        for reduction in ("mean", "none"):
            grad = torch.ones((n,) if reduction == "none" else (), device="cuda")
            calls.append(lambda a=(x, w, y, reduction, grad): body(*a))
    for n, V in ((2000, 47), (300, 3000), (2, 100000)):
        z = torch.randn(n, V, device="cuda").to(dtype).requires_grad_(True)
        t, ids = torch.randn(n, 5, device="cuda"), torch.randint(0, V, (n, 5), device="cuda")
        calls.append(lambda a=(z, t, ids, torch.ones((), device="cuda")): soft(*a))
torch.cuda.synchronize()
graphs = []
for call in calls:
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    graphs.append((g, out))
for (g, out), call in zip(graphs, calls):
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, call()))
print("FIRST-CALLS-CAPTURED-OK", len(calls))
"""


def test_first_calls_may_be_captured():
    out = subprocess.run([sys.executable, "-c", CHILD % {"root": ROOT}], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-4000:]
    assert "FIRST-CALLS-CAPTURED-OK" in out.stdout
