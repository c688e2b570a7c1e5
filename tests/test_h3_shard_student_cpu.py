"""The student's gradients through a critic with sharded block weights, with more blocks than gathered copies."""
import pytest
import torch

from dmad_b200.distill.h3_dmad import H3DMAD, H3DMADConfig
from dmad_b200.models.h3 import H3Config


def _student_gradients(shard, fake_train_type, layers):
    cfg = H3DMADConfig(model=H3Config(dim=64, num_heads=1, ffn_dim=96, num_layers=layers, refiner_layers=1, text_dim=16,
                                      time_embed_dim=32), height=64, width=64, num_frames=22, student_lora_rank=4,
                       text_tokens=4, fake_train_type=fake_train_type, critic_freeze_blocks=2, shard_weights=shard)
    m = H3DMAD(cfg, "cpu", dtype=torch.float32, seed=0)
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():  # adapters and heads that are not zero
        for p in [*m.heads.parameters(), m.student.proj_out.weight, *(p for n, p in m.student.named_parameters() if "lora_B" in n)]:
            p.copy_(0.1 * torch.randn(p.shape, generator=g))
    torch.manual_seed(11)
    grads, step = [], m.opt_s.step
    m.opt_s.step = lambda: (grads.extend(p.grad.reshape(-1).clone() for p in m.s_params), step())
    m.student_stage()
    assert m.fake.training
    return torch.cat(grads)


@pytest.mark.parametrize("fake_train_type", ["full", "lora"])
@pytest.mark.parametrize("layers", [4, 9])
def test_sharded_critic_gives_the_student_the_same_gradients(fake_train_type, layers):
    want = _student_gradients(False, fake_train_type, layers)
    assert want.norm() > 0
    # one rank: the same products of the same numbers
    assert torch.equal(_student_gradients(True, fake_train_type, layers), want)
