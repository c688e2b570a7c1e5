"""Kept 8-bit activations beside activation checkpoints: blocks that are computed again run as plain ones."""
import copy

import pytest
import torch

from dmad_b200 import ops
from dmad_b200.models.sac import checkpoint_block, inside_checkpoint
from tests.test_fp4_models_cpu import _tiny_h3
from tests.test_int8_models_cpu import _h3_step, _wan, _wan_step
from tests.test_sac_cpu import _CountMM

NETS = [(_wan, _wan_step), (_tiny_h3, _h3_step)]


@pytest.fixture
def calls(monkeypatch):
    """The layers that keep codes, one entry a call."""
    seen, real = [], ops.linear_act8
    monkeypatch.setattr(ops, "linear_act8", lambda *a, **k: seen.append(1) or real(*a, **k))
    return seen


def _blocks(net):
    return net.blocks if hasattr(net, "blocks") else net.transformer_blocks


@pytest.mark.parametrize("make,step", NETS)
@pytest.mark.parametrize("policy", ["block_wise", "mm_only", "block_int8"])
def test_checkpointed_blocks_run_without_codes(make, step, policy, calls):
    net = make().train()
    net.checkpoint_blocks, net.checkpoint_policy = len(_blocks(net)), policy
    ref = copy.deepcopy(net)
    net.enable_act8()
    with _CountMM() as products:
        y, g = step(net)
    with _CountMM() as products_ref:
        yr, gr = step(ref)
    assert not calls and products.n == products_ref.n
    assert torch.equal(y, yr) and set(g) == set(gr) and all(torch.equal(g[n], gr[n]) for n in g)


@pytest.mark.parametrize("make,step", NETS)
def test_the_other_blocks_keep_codes(make, step, calls):
    net = make().train()
    net.enable_act8()
    net.checkpoint_blocks = len(_blocks(net)) - 1
    step(net)
    last = _blocks(net)[-1]
    assert len(calls) == sum(getattr(m, "act8", False) for m in last.modules()) > 0
    calls.clear()
    net.eval()  # (a network that is evaluated checkpoints nothing)
    step(net)
    assert len(calls) == sum(getattr(m, "act8", False) for m in _blocks(net).modules())


def test_the_mark_ends_with_the_block():
    x = torch.ones(3, requires_grad=True)

    def fails(v):
        assert inside_checkpoint()
        raise KeyError("x")

    def nested(v):
        y = checkpoint_block(lambda u: u.exp(), v)
        assert inside_checkpoint()
        return y

    with pytest.raises(KeyError):
        checkpoint_block(fails, x)
    assert not inside_checkpoint()
    checkpoint_block(nested, x).sum().backward()
    assert not inside_checkpoint() and torch.equal(x.grad, torch.ones(3).exp())
