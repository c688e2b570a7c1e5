"""4-bit products at the edges: kernels that end right after they begin, factors at both ends of fp32, sums that are
exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu
dev = "cuda"


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def test_one_tile_a_pair_back_to_back_on_two_streams():
    """One tile a pair and one K step a tile: the second CTA of a pair is done as soon as it can be, while the leader's
    last arrivals in its shared memory are on their way; the next kernel takes that memory at once."""
    ops = _ops()
    torch.manual_seed(0)
    w = ops.quantize_fp4(torch.randn(16512, 32, device=dev), "mxfp4")
    xs = [ops.quantize_fp4(torch.randn(256, 32, device=dev), "mxfp4") for _ in range(2)]
    wv = ops.dequantize_fp4(w, torch.float32).double()
    # codes are multiples of half a scale: 32 products and their fp32 sums, then half a bf16 step
    want = [ops.dequantize_fp4(x, torch.float32).double() @ wv.t() for x in xs]
    size = [ops.dequantize_fp4(x, torch.float32).double().abs() @ wv.abs().t() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(40):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.fp4_linear(xs[i], w))
    torch.cuda.synchronize()
    ops.check_device_status()
    for g, r, s in zip(got, want, size):
        assert ((g[0].double() - r).abs() <= 2.0 ** -8 * r.abs() + 40 * 2.0 ** -23 * s).all()
        assert all(torch.equal(g[0], o) for o in g)
