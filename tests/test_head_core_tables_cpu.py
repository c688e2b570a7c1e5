"""Tables of other lengths than the sequence in the fused per-head attention core."""
import pytest
import torch

from dmad_b200.models.layers import head_attention_core


def check_tables(device, dtype, hd):
    torch.manual_seed(0)
    B, L, H = 3, 10, 2
    qkv = torch.randn(B * L, 3 * H * hd, device=device).to(dtype)
    w = torch.rand(2, hd, device=device)
    ang = torch.randn(L + 6, hd // 2, device=device)
    c, s = ang.cos(), ang.sin()
    want = head_attention_core(qkv, *w, c[:L].contiguous(), s[:L].contiguous(), B, L, H)
    # every sequence of the batch counts its positions from zero, whatever the table's length
    assert torch.equal(head_attention_core(qkv, *w, c, s, B, L, H), want)
    one = torch.cat([head_attention_core(qkv[b * L:(b + 1) * L], *w, c, s, 1, L, H) for b in range(B)])
    if device == "cpu":
        assert (one - want).abs().max() <= 1e-5
    with pytest.raises(ValueError, match="L = 10"):
        head_attention_core(qkv, *w, c[:L - 1], s[:L - 1], B, L, H)


def test_longer_and_shorter_tables():
    check_tables("cpu", torch.float32, 8)
