"""The trainers with kept 8-bit activations and 8-bit checkpoints: whole steps, and a warning where no layer keeps codes."""
import copy
import warnings

import pytest
import torch

from dmad_b200 import ops
from dmad_b200.distill.h3_dmad import H3DMAD, H3DMADConfig
from dmad_b200.distill.wan_dmad import WanDMAD, WanDMADConfig
from dmad_b200.models.h3 import H3Config
from dmad_b200.models.layers import act8_layers
from dmad_b200.models.wan import WanConfig


@pytest.fixture
def calls(monkeypatch):
    seen, real = [], ops.linear_act8
    monkeypatch.setattr(ops, "linear_act8", lambda *a, **k: seen.append(1) or real(*a, **k))
    return seen


def _h3(**kw):
    cfg = H3DMADConfig(model=H3Config(dim=64, num_heads=1, ffn_dim=96, num_layers=2, refiner_layers=1, text_dim=16,
                                      time_embed_dim=32), height=64, width=64, num_frames=22, student_lora_rank=4,
                       text_tokens=4, critic_freeze_blocks=0, **kw)
    return H3DMAD(cfg, "cpu", dtype=torch.float32)


def _wan(**kw):
    net = WanConfig(dim=64, ffn_dim=128, num_heads=1, num_layers=2, text_dim=16)
    return WanDMAD(WanDMADConfig(net=net, sn_power_iters=2, **kw), device="cpu", dtype=torch.float32)


def _batch():
    g = torch.Generator().manual_seed(2)
    return {"latents": torch.randn(1, 16, 2, 4, 4, generator=g), "real_latents": torch.randn(1, 16, 2, 4, 4, generator=g),
            "context": torch.randn(1, 8, 16, generator=g)}


@pytest.mark.parametrize("make,kw", [
    (_h3, {}), (_h3, {"gradient_checkpointing": False}), (_h3, {"fake_train_type": "full", "shard_weights": True}),
    (_wan, {"checkpoint_student_blocks": 2, "checkpoint_critic_blocks": 2}),
    (_wan, {"student_lora_rank": 4, "checkpoint_critic_blocks": 2})])
def test_a_warning_where_no_layer_keeps_codes(make, kw, calls):
    with pytest.warns(UserWarning, match="act8 reaches no layer"):
        m = make(act8=True, **kw)
    m.train_iteration() if make is _h3 else [m.training_step(_batch(), it) for it in range(2)]
    assert not calls


@pytest.mark.parametrize("make,kw", [
    (_h3, {"gradient_checkpointing": False, "fake_train_type": "full"}), (_h3, {"fake_train_type": "full"}), (_wan, {}),
    (_wan, {"student_lora_rank": 4}), (_wan, {"checkpoint_student_blocks": 2, "checkpoint_critic_blocks": 1}),
    (_wan, {"checkpoint_student_blocks": 2, "checkpoint_critic_blocks": 2, "checkpoint_critic_blocks_student_phase": 0}),
    (_wan, {"critic_spectral_norm": False, "generator_spectral_norm": False, "dp_optimizer": "replicated"})])
def test_steps_with_kept_codes(make, kw, calls):
    with warnings.catch_warnings():
        warnings.simplefilter("error", UserWarning)
        m = make(act8=True, **kw)
    if make is _h3:
        assert act8_layers(m.student.transformer_blocks) == 0 < act8_layers(m.fake.transformer_blocks)
        out = m.train_iteration()
        values = [v for d in out.values() for v in d.values()]
        moved = m.fake.parameters()
    else:
        before = [p.detach().clone() for p in m.net_fake_score.parameters()]
        values = [v for it in range(2) for v in m.training_step(_batch(), it).values()]
        moved = [p for p, b in zip(m.net_fake_score.parameters(), before) if not torch.equal(p, b)]
        assert moved
    assert calls and all(torch.isfinite(torch.as_tensor(v)).all() for v in values)
    assert all(p.isfinite().all() for p in moved)


def _critic_step(kw):
    m = _wan(**kw)
    torch.manual_seed(3)
    m.training_step(_batch(), 1)
    return torch.cat([p.detach().reshape(-1) for p in m.net_fake_score.parameters()])


def test_policies_of_the_critic():
    """A critic step with 8-bit checkpoints, and with act8 in the blocks that are not checkpointed: AdamW's first step moves
    each weight by the rate at most, and the same way unless its gradient is small."""
    assert not _wan().is_student_phase(1)
    base, start = _critic_step({}), torch.cat([p.detach().reshape(-1) for p in _wan().net_fake_score.parameters()])
    assert not torch.equal(base, start)
    for kw in ({"checkpoint_critic_blocks": 2, "checkpoint_critic_policy": "block_int8"}, {"act8": True},
               {"act8": True, "checkpoint_critic_blocks": 1, "checkpoint_critic_policy": "block_int8"}):
        got = _critic_step(kw)
        assert not torch.equal(got, base)
        assert ((got - start) * (base - start) > 0).float().sum() > 0.9 * (base != start).float().sum()
    for policy in ("block_wise", "mm_only"):  # the recomputed products are the same numbers
        assert torch.equal(_critic_step({"act8": True, "checkpoint_critic_blocks": 2, "checkpoint_critic_policy": policy}),
                           _critic_step({"checkpoint_critic_blocks": 2, "checkpoint_critic_policy": policy}))
