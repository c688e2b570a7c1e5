"""8-bit integer layers, 8-bit kept activations and 8-bit checkpoints inside the models, on the CPU."""
import copy

import pytest
import torch
import torch.nn.functional as F

from dmad_b200 import ops
from dmad_b200.models.layers import SegLinear, enable_act8, quantize_fp4_, quantize_int8_
from dmad_b200.models.sac import checkpoint_block
from tests.test_fp4_models_cpu import _h3_inputs, _linear, _tiny_h3


def test_layer_multiplies_the_coded_weight():
    lin, x = _linear(), torch.randn(3, 5, 64).bfloat16()
    w, b = lin.weight.detach().clone(), lin.bias.detach()
    lin.quantize_int8_()
    with torch.no_grad():
        y = lin(x)
        assert torch.equal(y, ops.int8_linear(x, ops.quantize_int8(w), b))
        assert torch.equal(lin.forward_rows(x, 45, 80), y[..., 45:80]) and lin.forward_rows(x, 90, 95).shape == (3, 5, 0)
        assert torch.equal(lin.effective_weight(), ops.dequantize_int8(ops.quantize_int8(w)))
        assert torch.equal(lin(x, act="gelu_tanh"), lin(ops.gelu_tanh(x)))
    assert [n for n, _ in lin.named_parameters()] == ["bias"]


def test_spectral_norm_and_lora_are_folded_in():
    lin = _linear(1, torch.float32).eval()
    lin.enable_spectral_norm()
    lin.enable_lora(4)
    lin.lora_B.data.normal_(0, 0.1)
    want = (lin.effective_weight() + lin.lora_delta_weight()).detach()
    lin.quantize_int8_()
    assert torch.equal(ops.dequantize_int8(lin.int8, torch.float32), ops.dequantize_int8(ops.quantize_int8(want), torch.float32))
    with torch.no_grad():
        assert lin(torch.randn(2, 64)).dtype == torch.bfloat16  # an fp32 layer computes in bf16


def test_quantised_layers_move_but_are_not_saved_loaded_or_trained():
    lin = _linear().quantize_int8_()
    scale = lin.int8.scale.clone()
    lin.to(torch.bfloat16).half().to("cpu")
    assert lin.int8.scale.dtype == torch.float32 and torch.equal(lin.int8.scale, scale)
    with torch.no_grad():
        assert lin(torch.randn(2, 64).half()).dtype == torch.float16
    for f in (lin.state_dict, lambda: lin.load_state_dict({}), lambda: lin.enable_lora(4), lin.enable_spectral_norm,
              lin.quantize_int8_, lambda: lin.quantize_fp4_("nvfp4"), lambda: lin.seg_weight("q")):
        with pytest.raises(RuntimeError, match="8-bit"):
            f()
    with pytest.raises(RuntimeError, match="forward only"):
        lin(torch.randn(2, 64).half().requires_grad_(True))
    net = torch.nn.Sequential(_linear(), torch.nn.Linear(4, 4), _linear(2))
    assert quantize_int8_(net) == 2 and quantize_int8_(net) == 0
    with pytest.raises(RuntimeError, match="8-bit"):
        quantize_fp4_(net)


def test_h3_in_8_bits_is_the_network_of_the_coded_weights():
    m = _tiny_h3().bfloat16().eval().requires_grad_(False)
    ref = copy.deepcopy(m)
    assert m.quantize_int8_() == 3 * 4 and all(b.attn.fused_qk_norm for b in m.transformer_blocks)
    for lin, old in zip((x for x in m.modules() if isinstance(x, SegLinear)), (x for x in ref.modules() if isinstance(x, SegLinear))):
        assert torch.equal(lin.effective_weight(), ops.dequantize_int8(ops.quantize_int8(old.weight)))
    v, a, pe, kw = _h3_inputs()
    with torch.no_grad():
        got, want = m(v, a, pe, **kw), ref(v, a, pe, **kw)
    for x, y in zip(got, want):  # two blocks of products with operands off by 2^-8 at most
        assert torch.isfinite(x).all() and (x - y).norm() <= 0.05 * y.norm()


def test_act8_layer():
    lin, x = _linear(3, torch.float32), torch.randn(6, 64, requires_grad=True)
    plain = copy.deepcopy(lin)
    assert enable_act8(lin) == 1
    for act in (None, "gelu_tanh"):
        y = lin(x, act=act)
        assert torch.equal(y, ops.linear_act8(x, lin.weight, lin.bias, act))
        with torch.no_grad():
            assert torch.equal(lin(x, act=act), plain(x, act=act))
        ref = plain(x, act=act)
        g = torch.randn_like(y)
        for p, q in zip(torch.autograd.grad(y, (x, lin.weight, lin.bias), g), torch.autograd.grad(ref, (x, plain.weight, plain.bias), g)):
            assert (p - q).norm() <= 2.0 ** -6 * q.norm()  # the kept input is off by 2^-7 of its block's largest at most
    h = torch.randn(6, 128)
    with torch.no_grad():
        assert torch.equal(lin(h, act="swiglu"), F.linear(h[:, :64] * F.silu(h[:, 64:]), lin.weight, lin.bias))
    with pytest.raises(ValueError):
        lin(x, act="relu")
    lin.enable_lora(4)
    assert torch.equal(lin(x, act="gelu_tanh"), lin(ops.gelu_tanh(x)))  # a layer with an adapter keeps its input as it is
    enable_act8(lin, False)
    assert not lin.act8


def _wan():
    from dmad_b200.models.wan import WanConfig, WanModel
    torch.manual_seed(0)
    net = WanModel(WanConfig(dim=64, ffn_dim=160, num_heads=2, num_layers=2, text_dim=32, text_len=8))
    torch.nn.init.normal_(net.head.head.weight, std=0.05)
    return net


def _wan_step(net):
    g = torch.Generator().manual_seed(1)
    x, t, c = torch.randn(1, 16, 2, 8, 8, generator=g), torch.tensor([[0.4]]), torch.randn(1, 8, 32, generator=g)
    y = net(x, t, c)
    y.square().sum().backward()
    return y.detach(), {n: p.grad for n, p in net.named_parameters() if p.grad is not None}


def _h3_step(net):
    torch.manual_seed(7)
    v, a, pe, kw = _h3_inputs()
    o = net(v, a, pe, **kw)
    (o[0].square().sum() + o[1].square().sum()).backward()
    return torch.cat([t.reshape(-1) for t in o]).detach(), {n: p.grad for n, p in net.named_parameters() if p.grad is not None}


def _near(a, b, rel):
    # over all parameters: a single one's gradient may be next to zero
    assert set(a) == set(b)
    d = sum((a[n] - b[n]).square().sum() for n in a).sqrt()
    assert d <= rel * sum(b[n].square().sum() for n in b).sqrt()


@pytest.mark.parametrize("make,step", [(_wan, _wan_step), (_tiny_h3, _h3_step)])
def test_networks_with_act8(make, step):
    net = make().train()
    ref = copy.deepcopy(net)
    layers = sum(isinstance(m, SegLinear) for m in (net.blocks if hasattr(net, "blocks") else net.transformer_blocks).modules())
    assert net.enable_act8() == layers
    (y, g), (yr, gr) = step(net), step(ref)
    assert (y - yr).norm() <= 1e-5 * yr.norm()  # the forward pass is the same, in fp32 sums of another order
    _near(g, gr, 0.02)
    assert any(not torch.equal(g[n], gr[n]) for n in g)


@pytest.mark.parametrize("make,step", [(_wan, _wan_step), (_tiny_h3, _h3_step)])
def test_networks_with_8_bit_checkpoints(make, step):
    net = make().train()
    ref = copy.deepcopy(net)
    net.checkpoint_blocks, net.checkpoint_policy = 2, "block_int8"
    (y, g), (yr, gr) = step(net), step(ref)
    assert torch.equal(y, yr)
    _near(g, gr, 0.02)
    assert any(not torch.equal(g[n], gr[n]) for n in g)


def test_checkpoint_block_keeps_codes_only_and_differentiates_at_them():
    w = torch.randn(40, 40, requires_grad=True)
    x0 = torch.randn(6, 40, requires_grad=True)
    kept = []

    def block(x, s):
        kept.append(x)
        return torch.tanh(x @ w) * s

    x = x0 * 1.0
    s = torch.tensor(2.0, requires_grad=True)
    y = checkpoint_block(block, x, s, policy="block_int8")
    assert torch.equal(y, torch.tanh(x @ w) * s) and len(kept) == 1
    g = torch.randn(6, 40)
    got = torch.autograd.grad(y, (x0, w, s), g, retain_graph=True)
    xq = ops.dequantize_int8(ops.quantize_int8(x.detach(), 32), torch.float32)
    assert len(kept) == 2 and torch.equal(kept[1], xq)
    xr = xq.requires_grad_(True)
    want = torch.autograd.grad(torch.tanh(xr @ w) * s, (xr, w, s), g)
    assert all(torch.allclose(p, q, rtol=1e-5, atol=1e-5) for p, q in zip(got, want))
    again = torch.autograd.grad(y, (x0, w, s), g)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    with torch.no_grad():
        assert torch.equal(checkpoint_block(block, x, s, policy="block_int8"), y)
    with pytest.raises(ValueError, match="block_int8"):
        checkpoint_block(block, x, s, policy="block_fp8")


def test_checkpoint_block_with_an_input_that_needs_no_gradient():
    w = torch.randn(32, 32, requires_grad=True)
    x = torch.randn(4, 32)
    y = checkpoint_block(lambda v: torch.tanh(v @ w), x, policy="block_int8")
    d, = torch.autograd.grad(y.sum(), w)
    xq = ops.dequantize_int8(ops.quantize_int8(x, 32), torch.float32)
    ref, = torch.autograd.grad(torch.tanh(xq @ w).sum(), w)
    assert torch.allclose(d, ref, rtol=1e-5, atol=1e-6)


def test_command_lines(tmp_path):
    from dmad_b200.cli.h3_inference import main, parse_args
    outs = main(["--config", "tiny", "--random-init", "--prompt", "x", "--output-dir", str(tmp_path), "--steps", "1",
                 "--height", "64", "--width", "64", "--num-frames", "22", "--text-tokens", "8", "--linear-int8"])
    assert torch.isfinite(outs[0][0].float()).all()
    for bad in (["--linear-int8", "--low-vram", "8"], ["--linear-int8", "--weights-fp4", "nvfp4"]):
        with pytest.raises(SystemExit):
            parse_args(["--output-dir", "o", *bad])
    from dmad_b200.cli.wan_sample import main as wan
    pj = tmp_path / "p.json"
    pj.write_text('["a"]')
    wan(["--tiny", "--distilled", "--prompt_json", str(pj), "--num_frames", "5", "--num_steps", "1",
         "--output_dir", str(tmp_path / "w"), "--linear_int8"])
    assert (tmp_path / "w" / "00000-0.latent.pt").exists()


def test_trainer_configurations():
    from dmad_b200.distill.wan_dmad import WanDMAD, WanDMADConfig
    from dmad_b200.models.wan import WanConfig
    m = WanDMAD(WanDMADConfig(net=WanConfig(dim=64, ffn_dim=96, num_heads=2, num_layers=1, text_dim=32, text_len=8), act8=True,
                              checkpoint_student_policy="block_int8"), dtype=torch.float32)
    assert all(lin.act8 for n in (m.net, m.net_fake_score) for b in n.blocks for lin in b.linears())
    assert m.net.checkpoint_policy == "block_int8"
