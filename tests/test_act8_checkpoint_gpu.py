"""Kept 8-bit activations beside activation checkpoints on the GPU, where other threads compute the blocks again."""
import pytest
import torch

from tests.test_int8_models_gpu import _step, _wan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("policy", ["block_wise", "mm_only", "block_int8"])
@pytest.mark.parametrize("blocks", [1, 2])
def test_checkpointed_blocks_keep_no_codes(policy, blocks, monkeypatch):
    from dmad_b200 import ops
    net = _wan()
    net.enable_act8()
    net.checkpoint_blocks, net.checkpoint_policy = blocks, policy
    calls, real = [], ops.linear_act8
    monkeypatch.setattr(ops, "linear_act8", lambda *a, **k: calls.append(1) or real(*a, **k))
    y, g = _step(net)
    assert len(calls) == 7 * (2 - blocks)
    ref = _wan()
    ref.checkpoint_blocks, ref.checkpoint_policy = blocks, policy
    yr, gr = _step(ref)
    assert len(calls) == 7 * (2 - blocks)
    if blocks == 2:  # the same kernels throughout (but attention's dQ is summed in any order, and then rounded: a step of bf16)
        assert torch.equal(y, yr) and (g - gr).norm() <= 2.0 ** -7 * gr.norm()
    else:
        assert (y - yr).norm() <= 2e-2 * yr.norm() and 0 < (g - gr).norm() <= 5e-2 * gr.norm()
