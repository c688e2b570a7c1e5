"""The 4-bit H3 network on the kernels against the same network on the CPU restatement."""
import copy

import pytest
import torch

from tests.test_fp4_models_cpu import _h3_inputs
from tests.test_fp4_models_gpu import _tiny_h3_for_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_h3_in_four_bits_matches_the_cpu(fmt):
    from dmad_b200 import ops
    m = _tiny_h3_for_gpu().bfloat16().eval().requires_grad_(False)
    m.quantize_fp4_(fmt)
    g = copy.deepcopy(m).cuda()
    for a, b in zip(m.modules(), g.modules()):  # the same codes
        if getattr(a, "fp4", None) is not None:
            assert torch.equal(a.fp4.data, b.fp4.data.cpu()) and torch.equal(a.fp4.scales, b.fp4.scales.cpu())
    v, a, pe, kw = _h3_inputs()
    with torch.no_grad():
        want = m(v, a, pe, **kw)
        got = g(v.cuda(), a.cuda(), pe.cuda(), **{k: t.cuda() for k, t in kw.items()})
    ops.check_device_status()
    for o, r in zip(got, want):
        # the two differ by last bits of bf16 between the projections; a number near a border of two codes then takes the
        # other one.  At worst that is as if each side had drawn its 4-bit rounding by itself: 0.1 of a projection's input
        # in the mean square, twice, and the blocks add them to a stream that has none.  A scale or a row out of place
        # changes a projection by its own size.
        assert (o.float().cpu() - r.float()).norm() <= 0.2 * r.float().norm()
