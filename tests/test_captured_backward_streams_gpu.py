"""A backward captured while an eager graph of the same leaves, recorded on a third stream, lives: that stream joins the
capture, and the replays are right."""
import pytest

from tests.test_captured_backward_gpu import _COMMON, _run

pytestmark = pytest.mark.gpu

_THIRD_STREAM = _COMMON + """
third = torch.cuda.Stream()
third.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(third):
    alive = forward()
torch.cuda.synchronize()
check(*capture())
assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, leaves, g), want))
print("as it should")
"""


@pytest.mark.parametrize("norm", [True, False])
def test_graph_recorded_on_a_third_stream(norm):
    _run(_THIRD_STREAM, norm)
