"""qk_head_norm_rope on the CPU: the restatement against complex numbers in 64 bits and differences, and every
refusal."""
import pytest
import torch

from dmad_b200 import ops
from dmad_b200.ops.head_norm import qk_head_norm_rope_reference


def _case(R, hq, hk, hd, rot, T, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(R, hq, hd, generator=g, dtype=dtype), torch.randn(R, hk, hd, generator=g, dtype=dtype)
    wq, wk = 1 + 0.3 * torch.randn(2, hd, generator=g, dtype=dtype)
    ang = torch.randn(T, rot // 2, generator=g, dtype=torch.float64)
    return q, k, wq, wk, ang.cos(), ang.sin()


def complex_oracle(x, w, cos, sin, at, rot, interleaved, eps):
    """The op in fp64 with each pair of elements as one complex number."""
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (w.double() if w is not None else 1.0)
    if rot:
        h = y[..., :rot]
        a, b = (h[..., ::2], h[..., 1::2]) if interleaved else h.chunk(2, -1)
        z = torch.complex(a, b) * torch.complex(cos.double(), sin.double())[at][:, None]
        r = torch.stack([z.real, z.imag], -1).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
        y = torch.cat([r, y[..., rot:]], -1)
    return y


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("R,hq,hk,hd,rot,T,pos", [(1, 1, 1, 8, 8, 1, False), (5, 4, 2, 16, 6, 3, False),
                                                  (4, 3, 3, 24, 24, 9, True)])
def test_reference_matches_complex_numbers(R, hq, hk, hd, rot, T, pos, interleaved):
    q, k, wq, wk, c, s = _case(R, hq, hk, hd, rot, T)
    at = torch.randint(0, T, (R,)) if pos else torch.arange(R) % T
    qo, ko = qk_head_norm_rope_reference(q, k, wq, wk, c, s, at if pos else None, 1e-6, interleaved)
    for o, x, w in ((qo, q, wq), (ko, k, wk)):
        ref = complex_oracle(x, w, c, s, at, rot, interleaved, 1e-6)
        assert (o - ref).abs().max() <= 64 * 2.0 ** -53 * ref.abs().max()


def test_reference_gradients_are_differences():
    q, k, wq, wk, c, s = _case(2, 2, 1, 8, 4, 2)
    args = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
    assert torch.autograd.gradcheck(lambda *a: qk_head_norm_rope_reference(*a, c, s, None, 1e-6, False), args)


def test_empty_rows_and_missing_parts():
    q, k = torch.randn(0, 2, 16), torch.randn(0, 1, 16)
    qo, ko = ops.qk_head_norm_rope(q, k)
    assert qo.shape == q.shape and ko.shape == k.shape
    q, k = torch.randn(3, 2, 16).bfloat16(), torch.randn(3, 1, 16).bfloat16()
    qo, _ = ops.qk_head_norm_rope(q, k)
    ref = complex_oracle(q, None, None, None, None, 0, True, 1e-6)
    # one rounding (half a step, 2^-8) over fp32 arithmetic of a few 2^-24
    assert ((qo.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -18) * ref.abs()).all()


def test_position_outside_the_table_is_nan_in_the_rotated_part():
    q, k, wq, wk, c, s = _case(3, 2, 1, 16, 8, 4, dtype=torch.float32)
    qo, _ = ops.qk_head_norm_rope(q, k, wq, wk, c, s, torch.tensor([0, 4, -1]))
    assert torch.isfinite(qo[0]).all() and torch.isnan(qo[1:, :, :8]).all() and torch.isfinite(qo[1:, :, 8:]).all()


def test_refusals():
    q, k, wq, wk, c, s = _case(3, 2, 1, 16, 8, 4, dtype=torch.float32)
    p = torch.zeros(3, dtype=torch.long)
    f = ops.qk_head_norm_rope
    bad = [lambda: f(q[0], k), lambda: f(q, k[:2]), lambda: f(q, k[..., :8]), lambda: f(q, k.half()),
           lambda: f(q.double(), k.double()), lambda: f(q[..., :12], k[..., :12]), lambda: f(q[:, :0], k),
           lambda: f(torch.randn(3, 1, 264), torch.randn(3, 1, 264)), lambda: f(q, k, wq[:8], wk),
           lambda: f(q, k, wq, wk.int()), lambda: f(q, k, wq, wk, c), lambda: f(q, k, wq, wk, None, s),
           lambda: f(q, k, wq, wk, positions=p), lambda: f(q, k, wq, wk, c[:0], s[:0]), lambda: f(q, k, wq, wk, c, s[:2]),
           lambda: f(q, k, wq, wk, torch.ones(4, 9), torch.ones(4, 9)), lambda: f(q, k, wq, wk, c.int(), s.int()),
           lambda: f(q, k, wq, wk, c.clone().requires_grad_(True), s), lambda: f(q, k, wq, wk, c, s, p[:2]),
           lambda: f(q, k, wq, wk, c, s, p.float())]
    for g in bad:
        with pytest.raises(ValueError):
            g()
