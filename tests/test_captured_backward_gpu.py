"""A backward captured into a graph while an eager graph of the same leaves lives: refused, the process goes on, and the
capture works once that graph is gone.  In processes of their own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

_COMMON = """
import torch
from dmad_b200 import ops
from dmad_b200.models.layers import head_attention_core
dev = "cuda"
torch.manual_seed(0)
w = torch.rand(64, device=dev, requires_grad=True)
if NORM:
    leaves = [torch.randn(40, 4, 64, device=dev).bfloat16().requires_grad_(True),
              torch.randn(40, 2, 64, device=dev).bfloat16().requires_grad_(True), w]
    forward = lambda: ops.qk_head_norm_rope(leaves[0], leaves[1], w, w)
else:
    leaves = [torch.randn(40, 3 * 2 * 64, device=dev).bfloat16().requires_grad_(True), w]
    forward = lambda: (head_attention_core(leaves[0], w, w, None, None, 1, 40, 2),)
outs = forward()
g = [torch.randn_like(o).detach() for o in outs]
step = lambda: torch.autograd.grad(forward(), leaves, g)
del outs
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    want = step()
torch.cuda.current_stream().wait_stream(side)
torch.cuda.synchronize()

def capture():
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    return graph, got

def check(graph, got):
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
"""

_REFUSED = _COMMON + """
alive = forward()  # on the default stream
try:
    capture()
    raise SystemExit("not refused")
except RuntimeError as e:
    assert "same leaves" in str(e), e
torch.cuda.synchronize()
# the eager graph is as it was
assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, leaves, g), want))
del alive
check(*capture())
ops.check_device_status()
print("as it should")
"""

_SAME_STREAM = _COMMON + """
with torch.cuda.stream(side):
    alive = forward()
torch.cuda.synchronize()
check(*capture())
assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, leaves, g), want))
print("as it should")
"""


def _run(code, norm):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", f"NORM = {norm}\n" + code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "as it should" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.parametrize("norm", [True, False])
def test_refused_beside_an_eager_graph(norm):
    _run(_REFUSED, norm)


@pytest.mark.parametrize("norm", [True, False])
def test_graph_recorded_on_the_captured_stream(norm):
    _run(_SAME_STREAM, norm)
