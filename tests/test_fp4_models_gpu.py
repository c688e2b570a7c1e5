"""The 4-bit projections, the fused q / k norm and the attention together, as an H3 block runs them."""
import copy

import pytest
import torch

from tests.test_fp4_models_cpu import _h3_inputs
from tests.test_head_norm_cpu import complex_oracle

pytestmark = pytest.mark.gpu
dev = "cuda"


def _attention(x, q, k, v):
    p = torch.softmax(torch.einsum("lhd,mhd->hlm", q, k) / q.shape[-1] ** 0.5, -1)
    return torch.einsum("hlm,mhd->lhd", p, v)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("L", [1, 77, 700])
def test_attention_block_stage_by_stage(fmt, L):
    """Each stage of the running block against 64 bits on that stage's own input."""
    from dmad_b200 import ops
    from dmad_b200.models.h3 import _H3Attention
    torch.manual_seed(L)
    D, H = 512, 4
    att = _H3Attention(D, H, 1e-6).to(dev, torch.bfloat16).eval().requires_grad_(False)
    for p in (att.norm_q.weight, att.norm_k.weight):
        p.normal_(1, 0.2)
    att.fused_qk_norm = True
    out = getattr(att.to_out, "0")
    for lin in (att.qkv, out):
        lin.quantize_fp4_(fmt)
    seen = {}
    att.qkv.register_forward_hook(lambda m, i, o: seen.update(x=i[0], qkv=o))
    out.register_forward_hook(lambda m, i, o: seen.update(att=i[0], y=o))
    ang = torch.randn(L, D // H // 2, device=dev)
    x = torch.randn(L, D, device=dev).bfloat16()
    y = att(x, ang.cos(), ang.sin(), L)
    ops.check_device_status()
    assert torch.equal(y, seen["y"])

    def linear_ok(inp, lin, got):
        xv = ops.dequantize_fp4(ops.quantize_fp4(inp, fmt), torch.float32).double()
        wv, b = ops.dequantize_fp4(lin.fp4, torch.float32).double(), lin.bias.double()
        ref, size = xv @ wv.t() + b, xv.abs() @ wv.abs().t() + b.abs()
        # half a bf16 step, and a truncation of the running size at each of the products
        assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (D + 8) * 2.0 ** -23 * size).all()

    linear_ok(seen["x"], att.qkv, seen["qkv"])
    linear_ok(seen["att"], out, seen["y"])
    h = seen["qkv"].view(L, 3, H, D // H)
    at = torch.arange(L, device=dev)
    q, k = (complex_oracle(h[:, i], w, ang.cos(), ang.sin(), at, D // H, True, 1e-6)
            for i, w in ((0, att.norm_q.weight), (1, att.norm_k.weight)))
    ref = _attention(x, q, k, h[:, 2].double())
    # bf16 q, k (logits off by 2 x 2^-8 of |q| |k| / sqrt(hd) < 14, so p by 11%, which averages out over keys), p and o
    assert (seen["att"].view(L, H, -1).double() - ref).norm() <= 2e-2 * ref.norm()


@pytest.mark.parametrize("B,L,H,hd,rope", [(1, 300, 4, 128, True), (2, 129, 3, 64, True), (1, 65, 2, 128, False)])
def test_head_attention_core_gradients(B, L, H, hd, rope):
    from dmad_b200.models.layers import head_attention_core
    torch.manual_seed(hd)
    qkv = torch.randn(B * L, 3 * H * hd, device=dev).bfloat16().requires_grad_(True)
    wq, wk = ((1 + 0.2 * torch.randn(hd, device=dev)).requires_grad_(True) for _ in range(2))
    ang = torch.randn(L, hd // 2, device=dev)
    cos, sin = (ang.cos(), ang.sin()) if rope else (None, None)
    g = torch.randn(B * L, H * hd, device=dev).bfloat16()
    o = head_attention_core(qkv, wq, wk, cos, sin, B, L, H)
    got = (o, *torch.autograd.grad(o, (qkv, wq, wk), g))
    x = qkv.detach().double().requires_grad_(True)
    ws = [w.detach().double().requires_grad_(True) for w in (wq, wk)]
    h = x.view(B * L, 3, H, hd)
    at = torch.arange(B * L, device=dev) % L
    q, k = (complex_oracle64(h[:, i], ws[i], cos, sin, at, hd if rope else 0) for i in range(2))
    ref = torch.cat([_attention(None, q[b * L:(b + 1) * L], k[b * L:(b + 1) * L], h[b * L:(b + 1) * L, 2])
                     for b in range(B)]).reshape(B * L, H * hd)
    want = (ref, *torch.autograd.grad(ref, (x, *ws), g.double()))
    for a, b in zip(got, want):
        # at most five bf16 roundings in a row (q / k, p, o, ds, dq / dk), 2^-8 each, on tensors of the result's size
        assert (a.double() - b).norm() <= 5 * 2.0 ** -8 * b.norm()


def complex_oracle64(x, w, cos, sin, at, rot):
    return complex_oracle(x, w, cos, sin, at, rot, True, 1e-6)


def test_h3_fused_qk_norm_matches_the_cpu():
    m = _tiny_h3_for_gpu()
    v, a, pe, kw = _h3_inputs()
    ref = m(v, a, pe, **kw)
    g = copy.deepcopy(m).to(dev, torch.bfloat16)
    g.enable_fused_qk_norm()
    out = g(v.cuda(), a.cuda(), pe.cuda(), **{k: t.cuda() for k, t in kw.items()})
    for o, r in zip(out, ref):
        assert (o.float().cpu() - r).norm() <= 5e-2 * r.norm()  # the bound of the unfused model's own test


def _tiny_h3_for_gpu():
    from dmad_b200.models.h3 import H3Config, H3Model
    torch.manual_seed(0)
    m = H3Model(H3Config(dim=256, num_heads=2, ffn_dim=512, num_layers=2, refiner_layers=1, text_dim=32, time_embed_dim=32))
    for p in m.parameters():
        p.data.normal_(0, 0.03)
    return m


def test_h3_dmad_trains_with_the_fused_norm():
    from tests.test_h3_gpu import _h3_train_cfg, _nonzero_outputs

    from dmad_b200 import ops
    from dmad_b200.distill.h3_dmad import H3DMAD
    cfg = _h3_train_cfg()
    cfg.fused_qk_norm = True
    m = H3DMAD(cfg, "cuda", dtype=torch.bfloat16)
    assert all(b.attn.fused_qk_norm for n in (m.student, m.fake) for b in n.transformer_blocks)
    _nonzero_outputs(m)
    before = [p.detach().clone() for p in m.s_params]
    for _ in range(2):
        out = m.train_iteration()
        for stage in out.values():
            assert all(torch.isfinite(torch.tensor(float(v))) for v in stage.values()), out
    ops.check_device_status()
    assert any(not torch.equal(a, b) for a, b in zip(before, m.s_params))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_h3_in_four_bits_runs_and_repeats(fmt):
    m = _tiny_h3_for_gpu().to(dev, torch.bfloat16).eval().requires_grad_(False)
    m.quantize_fp4_(fmt)
    v, a, pe, kw = _h3_inputs()
    kw = {k: t.cuda() for k, t in kw.items()}
    with torch.no_grad():
        one = m(v.cuda(), a.cuda(), pe.cuda(), **kw)
        two = m(v.cuda(), a.cuda(), pe.cuda(), **kw)
    assert all(torch.isfinite(o).all() and torch.equal(o, t) for o, t in zip(one, two))


_FIRST = """
import torch
from dmad_b200 import ops
x = torch.randn(3, 256, device="cuda").bfloat16()
big = torch.randn(300, 256, device="cuda").bfloat16()
q = torch.randn(3, 2, 64, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):  # the first kernels of the process
    w = ops.quantize_fp4(big)
    y, z = ops.fp4_linear(x, w), ops.fp4_linear(big, w)
    h = ops.qk_head_norm_rope(q, q)
g.replay()
torch.cuda.synchronize()
w2 = ops.quantize_fp4(big)
assert torch.equal(y, ops.fp4_linear(x, w2)) and torch.equal(z, ops.fp4_linear(big, w2))
assert torch.equal(h[0], ops.qk_head_norm_rope(q, q)[0])
ops.check_device_status()
print("captured first")
"""


def test_first_calls_of_a_process_under_capture():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stdout + r.stderr


def test_training_step_of_the_norm_in_a_graph():
    """Forward and backward captured and replayed on new numbers, beside an eager graph of the same leaves."""
    from dmad_b200 import ops
    q = torch.randn(40, 4, 64, device=dev).bfloat16().requires_grad_(True)
    k = torch.randn(40, 2, 64, device=dev).bfloat16().requires_grad_(True)
    w = torch.rand(64, device=dev, requires_grad=True)
    ang = torch.randn(40, 32, device=dev)
    c, s = ang.cos(), ang.sin()
    gq, gk = torch.randn_like(q).detach(), torch.randn_like(k).detach()

    def step():
        return torch.autograd.grad(ops.qk_head_norm_rope(q, k, w, w, c, s), (q, k, w), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    alive = ops.qk_head_norm_rope(q, k, w, w, c, s)
    for seed in range(2):
        with torch.no_grad():
            torch.manual_seed(seed)
            gq.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.isfinite(t).all() for t in torch.autograd.grad(alive, (q, k, w), (gq, gk)))


def test_results_do_not_depend_on_the_stream_or_repetition():
    """The few-rows kernel splits K over clusters: the same sums every time, on any stream, beside other work."""
    from dmad_b200 import ops
    torch.manual_seed(0)
    for M, N, K in ((1, 640, 5120), (100, 1000, 2048), (200, 256, 4096)):
        x = torch.randn(M, K, device=dev).bfloat16()
        w = ops.quantize_fp4(torch.randn(N, K, device=dev), "nvfp4")
        want = ops.fp4_linear(x, w)
        streams = [torch.cuda.Stream() for _ in range(3)]
        torch.cuda.synchronize()
        got = []
        for i in range(12):
            with torch.cuda.stream(streams[i % 3]):
                got.append(ops.fp4_linear(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
    ops.check_device_status()
