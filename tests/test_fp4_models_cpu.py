"""4-bit layers and the fused q / k norm inside the models, on the CPU."""
import copy

import pytest
import torch

from dmad_b200 import ops
from dmad_b200.models.layers import SegLinear, head_attention_core, quantize_fp4_


def _linear(seed=0, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    return SegLinear(64, [("q", 48), ("k", 32)], flat_name="qk").to(dtype)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_layer_multiplies_the_coded_weight(fmt):
    lin, x = _linear(), torch.randn(3, 5, 64).bfloat16()
    w, b = lin.weight.detach().clone(), lin.bias.detach()
    lin.quantize_fp4_(fmt)
    with torch.no_grad():
        y = lin(x)
        assert torch.equal(y, ops.fp4_linear(x, ops.quantize_fp4(w, fmt), b))
        assert torch.equal(lin.forward_rows(x, 48, 80), y[..., 48:80])
        assert torch.equal(lin.effective_weight(), ops.dequantize_fp4(ops.quantize_fp4(w, fmt)))
    assert [n for n, _ in lin.named_parameters()] == ["bias"]


def test_spectral_norm_and_lora_are_folded_in():
    lin = _linear(1, torch.float32).eval()
    lin.enable_spectral_norm()
    lin.enable_lora(4)
    lin.lora_B.data.normal_(0, 0.1)
    want = (lin.effective_weight() + lin.lora_delta_weight()).detach()
    lin.quantize_fp4_("nvfp4")
    assert torch.equal(ops.dequantize_fp4(lin.fp4, torch.float32),
                       ops.dequantize_fp4(ops.quantize_fp4(want, "nvfp4"), torch.float32))
    with torch.no_grad():
        assert lin(torch.randn(2, 64)).dtype == torch.bfloat16  # an fp32 layer computes in bf16


def test_quantised_layers_move_but_are_not_saved_loaded_or_trained():
    lin = _linear().quantize_fp4_("nvfp4")
    rs = lin.fp4.row_scale.clone()
    lin.to(torch.bfloat16).half().to("cpu")
    assert lin.fp4.row_scale.dtype == torch.float32 and torch.equal(lin.fp4.row_scale, rs)
    for f in (lin.state_dict, lambda: lin.load_state_dict({}), lambda: lin.enable_lora(4), lin.enable_spectral_norm,
              lambda: lin.quantize_fp4_("nvfp4")):
        with pytest.raises(RuntimeError, match="4-bit"):
            f()
    with pytest.raises(RuntimeError, match="forward only"):
        lin(torch.randn(2, 64).bfloat16().requires_grad_(True))


def _tiny_h3():
    from dmad_b200.models.h3 import H3Config, H3Model
    torch.manual_seed(0)
    m = H3Model(H3Config(dim=64, num_heads=2, ffn_dim=96, num_layers=2, refiner_layers=1, text_dim=32, time_embed_dim=32))
    for p in m.parameters():
        p.data.normal_(0, 0.05)
    return m


def _h3_inputs():
    from dmad_b200.inference.h3 import H3Geometry, build_packed_sequence, build_row_timesteps, latent_shape_of
    shape = latent_shape_of(64, 64, 22, H3Geometry())
    lay = build_packed_sequence(torch.ones(9, dtype=torch.long), shape["latent_frames"], shape["latent_height"],
                                shape["latent_width"], shape["audio_latents"])
    ts, ti = build_row_timesteps(lay, torch.tensor(0.7), torch.tensor(0.4))
    kw = dict(timestep=ts, timestep_indices=ti, token_tags=lay.token_tags, position_ids=lay.position_ids,
              video_indices=lay.video_indices, audio_indices=lay.audio_indices, text_indices=lay.text_indices)
    return torch.randn(shape["video_tokens"]), torch.randn(shape["audio_tokens"]), torch.randn(1, 9, 32), kw


def test_h3_fused_qk_norm_is_the_same_network():
    """fp32 on the CPU: the same sums in another order, forward and gradients."""
    m = _tiny_h3()
    f = copy.deepcopy(m)
    f.enable_fused_qk_norm()
    v, a, pe, kw = _h3_inputs()
    outs = [net(v, a, pe, **kw) for net in (m, f)]
    for x, y in zip(*outs):
        assert (x - y).norm() <= 1e-5 * x.norm()
    for net, o in zip((m, f), outs):
        (o[0].square().sum() + o[1].square().sum()).backward()
    for (n, p), q in zip(m.named_parameters(), f.parameters()):
        if p.grad is not None:
            assert (p.grad - q.grad).norm() <= 1e-4 * p.grad.norm() + 1e-7, n


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_h3_in_four_bits_is_the_network_of_the_coded_weights(fmt):
    """Every projection replaced, and only those; the weights' values are the codes'."""
    m = _tiny_h3().bfloat16().eval().requires_grad_(False)
    ref = copy.deepcopy(m)
    n = m.quantize_fp4_(fmt)
    assert n == 3 * 4 and all(b.attn.fused_qk_norm for b in m.transformer_blocks)
    for lin, old in zip((x for x in m.modules() if isinstance(x, SegLinear)),
                        (x for x in ref.modules() if isinstance(x, SegLinear))):
        assert torch.equal(lin.effective_weight(), ops.dequantize_fp4(ops.quantize_fp4(old.weight, fmt)))
    v, a, pe, kw = _h3_inputs()
    with torch.no_grad():
        assert all(torch.isfinite(o).all() for o in m(v, a, pe, **kw))


def test_head_attention_core_matches_its_parts():
    torch.manual_seed(0)
    B, L, H, hd = 2, 6, 2, 8
    qkv = torch.randn(B * L, 3 * H * hd)
    wq, wk = torch.rand(2, hd)
    ang = torch.randn(L, hd // 2)
    o = head_attention_core(qkv, wq, wk, ang.cos(), ang.sin(), B, L, H)
    x = qkv.double().view(B * L, 3, H, hd)
    from tests.test_head_norm_cpu import complex_oracle
    at = torch.arange(B * L) % L
    q = complex_oracle(x[:, 0], wq, ang.cos(), ang.sin(), at, hd, True, 1e-6).view(B, L, H, hd)
    k = complex_oracle(x[:, 1], wk, ang.cos(), ang.sin(), at, hd, True, 1e-6).view(B, L, H, hd)
    p = torch.softmax(torch.einsum("blhd,bmhd->bhlm", q, k) / hd ** 0.5, -1)
    ref = torch.einsum("bhlm,bmhd->blhd", p, x[:, 2].view(B, L, H, hd)).reshape(B * L, H * hd)
    assert (o - ref).abs().max() <= 1e-5


def test_command_lines(tmp_path):
    from dmad_b200.cli.h3_inference import main, parse_args
    outs = main(["--config", "tiny", "--random-init", "--prompt", "x", "--output-dir", str(tmp_path), "--steps", "1",
                 "--height", "64", "--width", "64", "--num-frames", "22", "--text-tokens", "8", "--weights-fp4", "mxfp4"])
    assert torch.isfinite(outs[0][0].float()).all()
    with pytest.raises(SystemExit):
        parse_args(["--output-dir", "o", "--weights-fp4", "nvfp4", "--low-vram", "8"])
    from dmad_b200.cli.wan_sample import main as wan
    pj = tmp_path / "p.json"
    pj.write_text('["a"]')
    wan(["--tiny", "--distilled", "--prompt_json", str(pj), "--num_frames", "5", "--num_steps", "1",
         "--output_dir", str(tmp_path / "w"), "--weights_fp4", "nvfp4"])
    assert (tmp_path / "w" / "00000-0.latent.pt").exists()


def test_quantize_helper_counts_and_skips():
    net = torch.nn.Sequential(_linear(), torch.nn.Linear(4, 4), _linear(2))
    assert quantize_fp4_(net) == 2 and quantize_fp4_(net) == 0
