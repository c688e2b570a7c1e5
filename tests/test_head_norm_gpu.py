"""qk_head_norm_rope kernels against complex numbers in 64 bits: forward, gradients, layouts, positions, streams."""
import pytest
import torch

from tests.test_head_norm_cpu import complex_oracle

pytestmark = pytest.mark.gpu
dev = "cuda"


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def _case(R, hq, hk, hd, rot, T, dtype, wdtype, seed=0, grad=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    qkv = torch.randn(R, (hq + 2 * hk) * hd, device=dev, generator=g).to(dtype)
    q, k = qkv[:, :hq * hd].view(R, hq, hd), qkv[:, hq * hd:(hq + hk) * hd].view(R, hk, hd)
    w = None
    if wdtype is not None:
        w = [(1 + 0.3 * torch.randn(hd, device=dev, generator=g)).to(wdtype) for _ in range(2)]
    c = s = None
    if rot:
        ang = 3 * torch.randn(T, rot // 2, device=dev, generator=g)
        c, s = ang.cos(), ang.sin()
    return q, k, w, c, s


def _oracle(q, k, w, c, s, at, rot, pairs, grads):
    ins = [t.detach().double().requires_grad_(True) for t in (q, k)]
    ws = [t.detach().double().requires_grad_(True) for t in w] if w else [None, None]
    outs = [complex_oracle(x, v, c, s, at, rot, pairs, 1e-6) for x, v in zip(ins, ws)]
    got = torch.autograd.grad(outs, ins + [v for v in ws if v is not None], [g.double() for g in grads])
    return outs, got


SHAPES = [(1, 1, 1, 8, 8, 1), (1, 40, 40, 128, 128, 64), (3, 4, 2, 32, 32, 3), (37, 6, 6, 64, 32, 5), (130, 5, 1, 80, 40, 130),
          (65, 8, 1, 96, 96, 13), (33, 3, 2, 256, 128, 33), (9, 7, 3, 128, 0, 1), (11, 2, 2, 128, 6, 4), (5, 2, 1, 56, 12, 5)]


@pytest.mark.parametrize("R,hq,hk,hd,rot,T", SHAPES)
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                          (torch.float32, None)])
def test_forward_and_gradients(R, hq, hk, hd, rot, T, pairs, dtype, wdtype):
    ops = _ops()
    q, k, w, c, s = _case(R, hq, hk, hd, rot, T, dtype, wdtype, seed=R + hd)
    positions = at = None
    if rot:
        at = torch.randint(0, T, (R,), device=dev) if R % 2 else torch.arange(R, device=dev) % T
        positions = (at if R % 4 == 1 else at.int()) if R % 2 else None
    gq, gk = torch.randn(q.shape, device=dev).to(dtype), torch.randn(k.shape, device=dev).to(dtype)
    leaves = [t.detach().requires_grad_(True) for t in (q, k)] + ([t.requires_grad_(True) for t in w] if w else [])
    wq, wk = w if w else (None, None)
    out = ops.qk_head_norm_rope(leaves[0], leaves[1], wq, wk, c, s, positions, 1e-6, pairs)
    got = torch.autograd.grad(out, leaves, (gq, gk))
    ops.check_device_status()
    ref, gref = _oracle(q, k, w, c, s, at, rot, pairs, (gq, gk))
    half = torch.finfo(dtype).eps / 2
    for o, r in zip(out, ref):
        assert o.is_contiguous() and o.dtype == dtype
        # one rounding, and ~30 fp32 operations on terms no larger than the head's largest element (|rot| = 1)
        size = r.abs().amax(-1, keepdim=True) * 2
        assert ((o.double() - r).abs() <= half * r.abs() + 64 * 2.0 ** -24 * size + 2.0 ** -25).all()
    for gt, r, x, g in zip(got[:2], gref[:2], (q, k), (gq, gk)):
        # dx = r (gy w - n c): two terms, each at most r * |w| * |g| * sqrt(hd)
        rr = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        size = rr * g.double().norm(dim=-1, keepdim=True) * 4
        assert ((gt.double() - r).abs() <= half * r.abs() + (64 + hd) * 2.0 ** -24 * size + 2.0 ** -25).all()
    if w:
        hw = torch.finfo(wdtype).eps / 2
        for gt, r, g in zip(got[2:], gref[2:], (gq, gk)):
            # sums over rows and heads: one rounding, fp32 additions of terms |g| * |n| <= |g| sqrt(hd)
            size = g.double().norm(dim=-1).sum() * hd ** 0.5
            assert gt.dtype == wdtype
            assert ((gt.double() - r).abs() <= hw * r.abs() + 64 * 2.0 ** -24 * size).all()


def test_long_rows_and_many_blocks():
    """More rows than one pass of the persistent grid, and weight gradients summed over all of them."""
    ops = _ops()
    q, k, w, c, s = _case(20000, 3, 2, 128, 128, 777, torch.bfloat16, torch.float32, seed=4)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, *w)]
    gq, gk = torch.randn(q.shape, device=dev).bfloat16(), torch.randn(k.shape, device=dev).bfloat16()
    out = ops.qk_head_norm_rope(*leaves, c, s)
    got = torch.autograd.grad(out, leaves, (gq, gk))
    again = torch.autograd.grad(ops.qk_head_norm_rope(*leaves, c, s), leaves, (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # no atomics: the same sums each time
    ref, gref = _oracle(q, k, w, c, s, torch.arange(20000, device=dev) % 777, 128, True, (gq, gk))
    for o, r in zip((*out, *got[:2]), (*ref, *gref[:2])):
        assert ((o.double() - r).abs() <= 2.0 ** -8 * r.abs() + 2.0 ** -16).all()
    for o, r in zip(got[2:], gref[2:]):
        # 60000 terms of size about 1: a few hundred additions a thread and a tree above them
        assert ((o.double() - r).abs() <= 1000 * 2.0 ** -24 * 60000 ** 0.5 * 4).all()


def test_gradient_is_the_difference_quotient():
    ops = _ops()
    q, k, w, c, s = _case(2, 2, 1, 16, 8, 2, torch.float32, torch.float32, seed=1)
    gq, gk = torch.randn(q.shape, device=dev), torch.randn(k.shape, device=dev)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, *w)]
    grads = torch.autograd.grad(ops.qk_head_norm_rope(*leaves, c, s), leaves, (gq, gk))
    for i, (t, g) in enumerate(zip(leaves, grads)):
        d = torch.randn_like(t)
        h = 2.0 ** -7

        def f(sign):
            a = [u.detach() for u in leaves]
            a[i] = a[i] + sign * h * d
            qo, ko = ops.qk_head_norm_rope(*a, c, s)
            return (qo.double() * gq.double()).sum() + (ko.double() * gk.double()).sum()

        num = (f(1) - f(-1)) / (2 * h)
        # central difference: h^2 / 6 times a third derivative of order |d|^3 / |x|^3 and fp32 noise / h
        assert (num - (g.double() * d.double()).sum()).abs() <= 2e-2 * (1 + num.abs())


def test_odd_strides_expanded_gradients_and_one_side():
    ops = _ops()
    base = torch.randn(7, 5, 3 * 64, device=dev).bfloat16()
    q, k = base[:, :, 1:65], base[::1, :2, 64:128]  # q starts off 16 bytes
    w = torch.rand(64, device=dev)
    qo, ko = ops.qk_head_norm_rope(q, k, w, None)
    for o, x, v in ((qo, q, w), (ko, k, None)):
        ref = complex_oracle(x, v, None, None, None, 0, True, 1e-6)
        assert ((o.double() - ref).abs() <= (2.0 ** -8 + 2.0 ** -18) * ref.abs() + 2.0 ** -25).all()
    ql = q.detach().requires_grad_(True)
    qo, ko = ops.qk_head_norm_rope(ql, k)
    qo.sum().backward()  # an expanded gradient, and none at all for ko
    want, = torch.autograd.grad(complex_oracle(z := q.detach().double().requires_grad_(True), None, None, None, None, 0,
                                               True, 1e-6).sum(), z)
    # |dx| <= r sqrt(hd) * 2; a row of ones cancels, so the rounding is of that size's fp32 terms and the result's bf16
    rr = (q.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    assert ((ql.grad.double() - want).abs() <= 2.0 ** -8 * want.abs() + 128 * 2.0 ** -24 * rr * 8 * 4).all()


def test_empty_positions_status_streams_and_graphs():
    ops = _ops()
    w = torch.ones(64, device=dev).requires_grad_(True)
    e = torch.empty(0, 2, 64, device=dev, requires_grad=True)
    out = ops.qk_head_norm_rope(e, e, w, w)
    g = torch.autograd.grad(out, (e, w), (torch.empty_like(e), torch.empty_like(e)))
    assert g[0].shape == e.shape and torch.equal(g[1], torch.zeros(64, device=dev))
    q, k, ws, c, s = _case(6, 2, 2, 64, 32, 8, torch.bfloat16, torch.float32)
    qo, ko = ops.qk_head_norm_rope(q, k, *ws, c, s, torch.tensor([0, 1, 8, -1, 2, 3], device=dev))
    assert torch.isnan(qo[2:4, :, :32]).all() and torch.isfinite(qo[2:4, :, 32:]).all()
    assert torch.isfinite(qo[[0, 1, 4, 5]]).all()
    with pytest.raises(RuntimeError, match="bounds"):
        ops.check_device_status()
    ops.check_device_status()
    pos = torch.arange(6, device=dev)
    want = ops.qk_head_norm_rope(q, k, *ws, c, s, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.qk_head_norm_rope(q, k, *ws, c, s, pos)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.qk_head_norm_rope(q, k, *ws, c, s, pos)
    pos.copy_(pos.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    want = ops.qk_head_norm_rope(q, k, *ws, c, s, pos)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_on_the_gpu():
    ops = _ops()
    q, k, w, c, s = _case(3, 2, 1, 16, 8, 4, torch.bfloat16, torch.float32)
    p = torch.zeros(3, dtype=torch.long, device=dev)
    f = ops.qk_head_norm_rope
    for g in (lambda: f(q[0], k), lambda: f(q, k[:2]), lambda: f(q, k.half()), lambda: f(q.double(), k.double()),
              lambda: f(q[..., :12], k[..., :12]), lambda: f(q, k.cpu()), lambda: f(q, k, w[0][:8]),
              lambda: f(q, k, w[0].cpu(), w[1]), lambda: f(q, k, *w, c), lambda: f(q, k, *w, positions=p),
              lambda: f(q, k, *w, c[:0], s[:0]), lambda: f(q, k, *w, torch.ones(4, 9, device=dev), torch.ones(4, 9, device=dev)),
              lambda: f(q, k, *w, c.clone().requires_grad_(True), s), lambda: f(q, k, *w, c, s, p[:2]),
              lambda: f(q, k, *w, c, s, p.float()), lambda: f(q, k, *w, c.cpu(), s.cpu())):
        with pytest.raises(ValueError):
            g()


def test_autograd_corner_cases():
    """One weight without a gradient, an unused output, gradients twice through one graph, no second derivative, and an
    input changed between forward and backward."""
    ops = _ops()
    q, k, w, c, s = _case(5, 2, 1, 64, 64, 5, torch.bfloat16, torch.float32)
    ql, kl, wl = q.detach().requires_grad_(True), k.detach(), w[0].detach().requires_grad_(True)
    qo, ko = ops.qk_head_norm_rope(ql, kl, wl, w[1].detach(), c, s)
    assert qo.requires_grad and ko.requires_grad
    g = torch.randn(qo.shape, device=dev).bfloat16()
    a = torch.autograd.grad(qo, (ql, wl), g, retain_graph=True)
    b = torch.autograd.grad(qo, (ql, wl), g)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    ref, gref = _oracle(q, k, w, c, s, torch.arange(5, device=dev), 64, True, (g, torch.zeros_like(ko)))
    assert (a[0].double() - gref[0]).norm() <= 2.0 ** -8 * gref[0].norm()
    assert (a[1].double() - gref[2]).norm() <= 2.0 ** -16 * gref[2].norm()
    qo, _ = ops.qk_head_norm_rope(ql, kl, wl, w[1].detach(), c, s)
    first, = torch.autograd.grad(qo, ql, g, create_graph=True)
    assert torch.equal(first, a[0])
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(first.float().sum(), ql)
    x = q.clone().requires_grad_(True)
    qo, _ = ops.qk_head_norm_rope(x, kl, wl, w[1].detach(), c, s)
    with torch.no_grad():
        x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(qo, x, g)
    with torch.no_grad():
        assert not ops.qk_head_norm_rope(ql, kl, wl)[0].requires_grad
