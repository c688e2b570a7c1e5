"""The 8-bit operators together inside the models on the GPU: integer inference, kept activations, checkpoints, captures."""
import copy
import os
import subprocess
import sys

import pytest
import torch

from tests.test_fp4_models_cpu import _h3_inputs, _tiny_h3

pytestmark = pytest.mark.gpu


def _wan():
    from dmad_b200.models.wan import WanConfig, WanModel
    torch.manual_seed(0)
    net = WanModel(WanConfig(dim=256, ffn_dim=544, num_heads=2, num_layers=2, text_dim=64, freq_dim=64))
    torch.nn.init.normal_(net.head.head.weight, std=0.05)
    return net.cuda().to(torch.bfloat16).train()


def _step(net):
    g = torch.Generator().manual_seed(4)
    x, t = torch.randn(1, 16, 2, 16, 16, generator=g).cuda(), torch.rand(1, 1, generator=g).cuda()
    y = net(x, t, torch.randn(1, 8, 64, generator=g).cuda())
    y.float().square().mean().backward()
    return y.detach(), torch.cat([p.grad.float().reshape(-1) for p in net.parameters() if p.grad is not None])


def test_wan_training_with_kept_codes():
    """act8, 8-bit checkpoints, and both: the same forward pass (its products on other kernels: bf16), near gradients."""
    from dmad_b200 import ops
    y0, g0 = _step(_wan())
    for act8, blocks in ((True, 0), (False, 2), (True, 1)):
        net = _wan()
        net.checkpoint_blocks, net.checkpoint_policy = blocks, "block_int8"
        assert net.enable_act8(act8) == 2 * 7
        y, g = _step(net)
        # act8's forward products round as the library's do, but sum in another order
        assert (y - y0).norm() <= (2e-2 if act8 else 0.0) * y0.norm()
        assert 0 < (g - g0).norm() <= 5e-2 * g0.norm()
    torch.cuda.synchronize()
    ops.check_device_status()


def test_wan_gradients_match_the_cpu_with_act8():
    net = _wan()
    cpu = copy.deepcopy(net).cpu().float()
    net.enable_act8()
    y, g = _step(net)
    gen = torch.Generator().manual_seed(4)
    x, t = torch.randn(1, 16, 2, 16, 16, generator=gen), torch.rand(1, 1, generator=gen)
    yc = cpu(x, t, torch.randn(1, 8, 64, generator=gen))
    yc.square().mean().backward()
    gc = torch.cat([p.grad.reshape(-1) for p in cpu.parameters() if p.grad is not None])
    assert (y.float().cpu() - yc).norm() <= 5e-2 * yc.norm() and (g.cpu() - gc).norm() <= 1e-1 * gc.norm()


def test_kept_memory():
    """What a feed-forward keeps between forward and backward: 1.03 bytes an element of its two inputs, not two and of the
    GELU's output besides."""
    from dmad_b200.models.layers import SegLinear, enable_act8
    torch.manual_seed(0)
    R, D, Fd = 4096, 512, 2048
    net = torch.nn.ModuleList([SegLinear(D, [("0", Fd)]), SegLinear(Fd, [("2", D)])]).cuda().to(torch.bfloat16)
    x = torch.randn(R, D, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    kept = []
    for on in (False, True):
        enable_act8(net, on)
        xin = x * 1.0
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = net[1](net[0](xin), act="gelu_tanh")
        del xin
        kept.append(torch.cuda.memory_allocated() - before - y.numel() * 2)
        y.sum().backward()
        del y
    codes = R * (D + Fd) * 33 // 32
    # without codes xin stays (counted before), the GELU's input and output are kept
    assert kept[0] >= 2 * R * Fd * 2 and kept[1] <= codes - R * D * 2 + (1 << 20)


def test_h3_in_8_bits():
    from dmad_b200 import ops
    m = _tiny_h3().bfloat16().eval().requires_grad_(False)
    v, a, pe, kw = _h3_inputs()
    c = copy.deepcopy(m)
    c.quantize_int8_()
    with torch.no_grad():
        want = c(v, a, pe, **kw)
        g = m.cuda()
        # the coded layers on the GPU, head size 32 on the CPU path only: compare layer by layer
        for lin, ref in zip((x for x in g.modules() if hasattr(x, "quantize_int8_") and hasattr(x, "seg_slices")),
                            (x for x in c.modules() if hasattr(x, "quantize_int8_") and hasattr(x, "seg_slices"))):
            lin.quantize_int8_()
            assert torch.equal(lin.int8.data.cpu(), ref.int8.data) and torch.equal(lin.int8.scale.cpu(), ref.int8.scale)
            x = torch.randn(37, lin.in_features).bfloat16()
            y, yr = lin(x.cuda()).cpu().float(), ref(x).float()
            # one rounding of the same number: a step of bf16 where fp32's roundings before it decide
            assert ((y - yr).abs() <= 2.0 ** -7 * yr.abs() + 1e-6).all()
    assert all(torch.isfinite(t).all() for t in want)
    ops.check_device_status()


def test_attention_to_mlp_run():
    """A block's feed-forward as serving and training run it: integers, kept codes and the coded checkpoint side by side."""
    from dmad_b200 import ops
    torch.manual_seed(1)
    x = torch.randn(300, 512, device="cuda", dtype=torch.bfloat16)
    w1 = (torch.randn(2 * 768, 512, device="cuda") * 512 ** -0.5).bfloat16()
    w2 = (torch.randn(512, 768, device="cuda") * 768 ** -0.5).bfloat16()
    with torch.no_grad():
        h = ops.int8_linear(x, ops.quantize_int8(w1))
        served = ops.int8_linear((h[:, :768] * torch.nn.functional.silu(h[:, 768:])), ops.quantize_int8(w2))
    xt, t1, t2 = (t.clone().requires_grad_(True) for t in (x, w1, w2))
    y = ops.linear_act8(ops.linear_act8(xt, t1), t2, None, "swiglu")
    y.backward(torch.randn_like(y))
    x64 = x.double()
    h64 = x64 @ w1.double().t()
    ref = (h64[:, :768] * h64[:, 768:] / (1 + torch.exp(-h64[:, 768:]))) @ w2.double().t()
    assert (y.double() - ref).norm() <= 2.0 ** -7 * ref.norm()      # two bf16 operands in a row
    assert (served.double() - ref).norm() <= 2.0 ** -5 * ref.norm()  # four coded operands, each off by up to 2^-8 of its row's largest
    q = ops.quantize_int8(xt.detach(), 32)
    # A block's step is 2^(floor(log2 max) - 6); an element is off by half of one, and by less than one where 127.5 .. 128
    # steps become 127: by 2^-6 of the block's largest at most.  (In norm: 2^-5 / sqrt(12) = 0.9 % of normal numbers, whose
    # 32 have a largest from 2 to 4.)
    err = (ops.dequantize_int8(q).double() - x64).abs().view(300, 16, 32)
    assert (err <= 2.0 ** -6 * x64.abs().view(300, 16, 32).amax(2, keepdim=True)).all()
    assert all(t.grad is not None and t.grad.isfinite().all() for t in (xt, t1, t2))


_COMMON = """
import torch
from dmad_b200 import ops
dev = "cuda"
torch.manual_seed(0)
leaves = [torch.randn(40, 64, device=dev).bfloat16().requires_grad_(True), torch.randn(32, 64, device=dev).bfloat16().requires_grad_(True),
          torch.randn(32, device=dev).requires_grad_(True)]
forward = lambda: ops.linear_act8(*leaves, "gelu_tanh")
y = forward()
g = torch.randn_like(y).detach()
del y
step = lambda: torch.autograd.grad(forward(), leaves, g)
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
assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(alive, leaves, g), want))
del alive
check(*capture())
print("done")
"""

_OTHER = _COMMON + """
with torch.cuda.stream(torch.cuda.Stream()):
    alive = forward()  # on a stream that joins the capture
check(*capture())
del alive
check(*capture())
print("done")
"""


@pytest.mark.parametrize("code", [_REFUSED, _OTHER], ids=["default", "other"])
def test_captured_backward_beside_a_living_graph(code):
    env = dict(os.environ, PYTHONPATH=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "done" in r.stdout, r.stderr[-2000:]
