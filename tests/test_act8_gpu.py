"""linear_act8 on the GPU against fp64, its codes, layouts, streams, graphs and refusals."""
import pytest
import torch

from tests import _int8_oracle as oracle

pytestmark = pytest.mark.gpu
dev = "cuda"
ACTS = (None, "gelu_tanh", "swiglu")


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def _act64(h, act):
    if act == "gelu_tanh":
        return 0.5 * h * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (h + 0.044715 * h ** 3)))
    if act == "swiglu":
        v, u = h.chunk(2, dim=-1)
        return v * u / (1 + torch.exp(-u))
    return h


def _kept64(x, act):
    if act == "swiglu":
        return torch.cat([oracle.values(h, 32) for h in x.chunk(2, dim=-1)], dim=-1)
    return oracle.values(x, 32)


def _inputs(R, N, F, act, dtype, bias, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, F * (2 if act == "swiglu" else 1), generator=g) * torch.exp(0.5 * torch.randn(R, 1, generator=g))
    x[:, ::50] *= 8
    w = torch.randn(N, F, generator=g) * F ** -0.5
    gy = torch.randn(R, N, generator=g)
    b = torch.randn(N, generator=g).to(bias).to(dev).requires_grad_(True) if bias is not None else None
    return x.to(dtype).to(dev).requires_grad_(True), w.to(dtype).to(dev).requires_grad_(True), b, gy.to(dtype).to(dev)


def _check(got, x, w, b, g, act):
    """Elementwise bounds.  Each output is rounded once to its type (eps / 2), act(x) once as an operand (eps / 2 of each
    term); fp32 sums lose 2^-23 of their size at each term, the activation and its derivative 2^-16 of their terms' sizes
    (2^z and 1 / v to 2^-22, the exponent z, up to 2^7, in fp32)."""
    dtype = x.dtype
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x, w, g = x.detach().double(), w.detach().double(), g.double()
    y, grads = got[0].detach().double(), got[1:]
    R, F = x.shape[0], w.shape[1]

    def near(a, want, slack, unit=u):
        err = (a.double() - want).abs()
        assert a.shape == want.shape and (err <= unit * want.abs() * (1 + 2.0 ** -6) + slack + tiny).all(), (err / (want.abs() + slack)).max()

    a = _act64(x, act)
    base = x.abs() if act != "swiglu" else x[:, :F].abs() * (1 + x[:, F:].abs())
    rounding = 0.0 if act is None else u
    want, size = a @ w.t(), (a.abs() * rounding + (2.0 ** -16 if act else 0.0) * base + 2.0 ** -23 * (F + 8) * a.abs() + tiny) @ w.abs().t()
    if b is not None:
        want, size = want + b.detach().double(), size + 2.0 ** -23 * b.detach().double().abs()
    near(y, want, size)
    xk = _kept64(x, act).requires_grad_(True)
    ak = _act64(xk, act)
    da = g @ w
    dx, = torch.autograd.grad(ak, xk, da)
    ak, xk = ak.detach(), xk.detach()
    err = 2.0 ** -23 * (w.shape[0] + 8) * (g.abs() @ w.abs()) + (2.0 ** -16 if act else 0.0) * da.abs()
    if act == "swiglu":
        v, t = xk[:, :F].abs(), xk[:, F:].abs()
        err = torch.cat([err * (1 + t), err * v * (2 + t)], dim=1)
    elif act:
        err = err * (2 + xk.abs()) ** 2
    near(grads[0], dx, err)
    kb = xk.abs() if act != "swiglu" else xk[:, :F].abs() * (1 + xk[:, F:].abs())
    near(grads[1], g.t() @ ak, g.abs().t() @ (ak.abs() * (rounding + 2.0 ** -23 * (R + 8)) + (2.0 ** -16 if act else 0.0) * kb + tiny))
    if b is not None:
        near(grads[2], g.sum(0), 2.0 ** -23 * (R + 8) * g.abs().sum(0), torch.finfo(b.dtype).eps / 2)


def _run(ops, x, w, b, g, act):
    y = ops.linear_act8(x, w, b, act)
    return (y, *torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], g))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, torch.float32), (torch.float16, None), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("R,N,F", [(1, 1, 1), (1, 256, 512), (3, 130, 33), (77, 640, 2048), (129, 257, 100), (300, 1543, 777),
                                   (1000, 96, 1536), (2049, 1536, 1544), (4096, 1536, 4608), (5000, 2304, 2056)])
def test_against_64_bits(R, N, F, act, dtype, bias):
    ops = _ops()
    x, w, b, g = _inputs(R, N, F, act, dtype, bias, R + N + F)
    got = _run(ops, x, w, b, g, act)
    torch.cuda.synchronize()
    ops.check_device_status()
    assert all(t.dtype == dtype for t in got[:3]) and (b is None or got[3].dtype == bias)
    _check(got, x, w, b, g, act)


@pytest.mark.parametrize("act", ACTS)
def test_the_same_again_and_only_what_is_wanted(act):
    ops = _ops()
    x, w, b, g = _inputs(700, 520, 200, act, torch.bfloat16, torch.float32, 1)
    full = _run(ops, x, w, b, g, act)
    for again in (_run(ops, x, w, b, g, act), _run(ops, x, w, b, g, act)):
        assert all(torch.equal(p, q) for p, q in zip(full, again))
    y = ops.linear_act8(x, w, b, act)
    for t, want in zip((x, w, b), full[1:]):
        got, = torch.autograd.grad(y, t, g, retain_graph=True)
        # without dx, act(x') is decoded by another kernel: the same formula on the same codes
        assert torch.equal(got, want)
    for k in range(3):  # leaves without a gradient
        ts = [t.detach().requires_grad_(i != k) for i, t in enumerate((x, w, b))]
        y = ops.linear_act8(*ts, act)
        got = torch.autograd.grad(y, [t for t in ts if t.requires_grad], g)
        assert all(torch.equal(p, q) for p, q in zip(got, [f for i, f in enumerate(full[1:]) if i != k]))
    with torch.no_grad():
        assert torch.equal(ops.linear_act8(x, w, b, act), full[0])
    assert not ops.linear_act8(x.detach(), w.detach(), b.detach(), act).requires_grad


@pytest.mark.parametrize("act", ACTS)
def test_layouts(act):
    ops = _ops()
    H = 2 if act == "swiglu" else 1
    base = torch.randn(60, 400, device=dev, dtype=torch.bfloat16)
    wide = torch.randn(90, 160, device=dev, dtype=torch.bfloat16)
    tall = torch.randn(200, 60, device=dev, dtype=torch.bfloat16)
    F = 64
    for xv in (base[:, :H * F], base[:, 3:3 + H * F], base[::2, 8:8 + H * F], base[0, :H * F].expand(9, H * F),
               tall.t()[:, :H * F], base[:, :H * F].unflatten(0, (6, 10)),
               base[0, :H * F]):
        for wv in (wide[:, :F], wide[:, 5:5 + F], tall[:, :50].t()[:, :F]):
            xs, ws = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
            xc, wc = xv.detach().contiguous().clone().requires_grad_(True), wv.detach().contiguous().clone().requires_grad_(True)
            ys, yc = ops.linear_act8(xs, ws, None, act), ops.linear_act8(xc, wc, None, act)
            assert torch.equal(ys, yc) and ys.shape == (*xv.shape[:-1], wv.shape[0])
            gy = torch.randn_like(yc)
            for gv in (gy, gy.transpose(0, -1).contiguous().transpose(0, -1), torch.ones((), device=dev, dtype=gy.dtype).expand(gy.shape)):
                a = torch.autograd.grad(ys, (xs, ws), gv, retain_graph=True)
                b = torch.autograd.grad(yc, (xc, wc), gv.contiguous(), retain_graph=True)
                assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[0].is_contiguous() and a[1].is_contiguous()


@pytest.mark.parametrize("act", ACTS)
def test_empty(act):
    ops = _ops()
    H = 2 if act == "swiglu" else 1
    x = torch.zeros(0, 3, 40 * H, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(8, 40, device=dev, dtype=torch.bfloat16, requires_grad=True)
    b = torch.randn(8, device=dev, requires_grad=True)
    y = ops.linear_act8(x, w, b, act)
    d = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
    assert y.shape == (0, 3, 8) and d[0].shape == x.shape and not d[1].any() and not d[2].any()
    x = torch.randn(5, 40 * H, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w0 = torch.zeros(0, 40, device=dev, dtype=torch.bfloat16, requires_grad=True)
    y = ops.linear_act8(x, w0, None, act)
    d = torch.autograd.grad(y, (x, w0), torch.zeros_like(y))
    assert y.shape == (5, 0) and not d[0].any() and d[1].shape == (0, 40)


@pytest.mark.parametrize("act", ACTS)
def test_far_values_and_non_finite_blocks(act):
    ops = _ops()
    H = 2 if act == "swiglu" else 1
    F = 96
    x = torch.randn(300, H * F, device=dev, dtype=torch.bfloat16)
    x[0, :F] = torch.linspace(-300, 300, F, device=dev)
    x[1] = 0
    x[2, :F] = torch.linspace(-1, 1, F, device=dev) * 2.0 ** -100
    if act == "swiglu":
        x[0, F:] = torch.linspace(200, -200, F, device=dev)
    x = x.requires_grad_(True)
    w = torch.randn(40, F, device=dev, dtype=torch.bfloat16, requires_grad=True)
    g = torch.randn(300, 40, device=dev, dtype=torch.bfloat16)
    got = _run(ops, x, w, None, g, act)
    assert all(t.isfinite().all() for t in got)
    _check(got, x, w, None, g, act)
    bad = x.detach().clone()
    bad[7, 40] = float("nan")
    bad = bad.requires_grad_(True)
    y, dx, dw = _run(ops, bad, w, None, g, act)
    keep = [r for r in range(300) if r != 7]
    assert y[7].isnan().all() and torch.equal(y[keep], got[0][keep])
    if act is not None:  # (the derivative along a SwiGLU's value is a function of its gate alone, and the other way round)
        at = F + 32 if act == "swiglu" else 32
        assert dx[7, at:at + 32].isnan().all() and torch.equal(dx[keep], got[1][keep]) and torch.equal(dx[7, :32], got[1][7, :32])
    else:
        assert torch.equal(dx, got[1])
    assert dw[:, 32:64].isnan().all() and torch.equal(dw[:, :32], got[2][:, :32]) and torch.equal(dw[:, 64:], got[2][:, 64:])


def test_what_is_kept():
    ops = _ops()
    x = torch.randn(64, 128, device=dev, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(32, 128, device=dev, dtype=torch.bfloat16, requires_grad=True)
    wg = torch.randn(32, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    for act, weight in ((None, w), ("gelu_tanh", w), ("swiglu", wg)):
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t):
            ops.linear_act8(x, weight, None, act)
        codes = [t for t in saved if t is not None and t.dtype == torch.int8]
        rest = [t for t in saved if t is not None and t.dtype not in (torch.int8, torch.uint8)]
        ref = ops.quantize_int8(x.detach(), 32)
        assert len(codes) == 1 and torch.equal(codes[0].view(ref.data.shape), ref.data)
        assert all(t.shape == weight.shape for t in rest)


def test_streams():
    ops = _ops()
    x, w, b, g = _inputs(500, 300, 160, "gelu_tanh", torch.bfloat16, torch.float32, 2)
    want = _run(ops, x, w, b, g, "gelu_tanh")
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(4):
                got.append(_run(ops, x, w, b, g, "gelu_tanh"))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for t in got for p, q in zip(t, want))


def test_captured_steps():
    ops = _ops()
    x, w, b, g = _inputs(500, 300, 160, "swiglu", torch.bfloat16, torch.float32, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(ops, x, w, b, g, "swiglu")
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(ops, x, w, b, g, "swiglu")
        graphs.append((graph, [t.detach() for t in out]))
        del out
    first = x.detach().clone()
    for scale in (1.0, -0.5):
        with torch.no_grad():
            x.copy_(first * scale)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = [t.detach() for t in _run(ops, x, w, b, g, "swiglu")]
        assert all(torch.equal(p, q) for _, out in graphs for p, q in zip(out, want))
    ops.check_device_status()


def test_differentiable_once_and_refusals():
    ops = _ops()
    x = torch.randn(4, 32, device=dev, dtype=torch.bfloat16)
    w = torch.randn(8, 32, device=dev, dtype=torch.bfloat16)
    for bad in (lambda: ops.linear_act8(x, w, None, "relu"), lambda: ops.linear_act8(x.float(), w.float()),
                lambda: ops.linear_act8(x, w.half()), lambda: ops.linear_act8(x, w[0]), lambda: ops.linear_act8(x[:, :31], w),
                lambda: ops.linear_act8(x, w, None, "swiglu"), lambda: ops.linear_act8(x, w, torch.zeros(7, device=dev)),
                lambda: ops.linear_act8(x, w, torch.zeros(8)), lambda: ops.linear_act8(x, w.cpu()),
                lambda: ops.linear_act8(x, w, torch.zeros(8, device=dev).double()), lambda: ops.linear_act8(x[:, :0], w[:, :0]),
                lambda: ops.linear_act8(x[0, 0], w)):
        with pytest.raises(ValueError):
            bad()
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.linear_act8(d, w)
    x.requires_grad_(True)
    dx, = torch.autograd.grad(ops.linear_act8(x, w).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


def test_steps_one_behind_the_other():
    """Steps whose kernels overlap, over memory that the steps before have just freed: the results of steps that are waited
    for."""
    ops = _ops()
    cases = []
    for i, (R, N, F, act) in enumerate([(300, 1280, 2048, None), (1001, 777, 1543, "gelu_tanh"), (64, 96, 200, "swiglu"), (2500, 2600, 1300, None),
                                        (3000, 512, 4104, "gelu_tanh"), (1500, 1000, 3001, "swiglu")]):
        x, w, b, g = _inputs(R, N, F, act, torch.bfloat16, torch.float32, i)
        torch.cuda.synchronize()
        out = _run(ops, x, w, b, g, act)
        torch.cuda.synchronize()
        cases.append(((x, w, b, g, act), [t.detach() for t in out]))
    wrong = torch.zeros((), device=dev, dtype=torch.int64)
    for i in torch.randint(0, len(cases), (150,), generator=torch.Generator().manual_seed(2)).tolist():
        args, want = cases[i]
        for t, ref in zip(_run(ops, *args), want):
            wrong += (t.detach() != ref).sum()
    assert int(wrong) == 0
    ops.check_device_status()


def test_frozen_weight_and_shared_leaves():
    ops = _ops()
    x, w, b, g = _inputs(200, 64, 96, None, torch.bfloat16, torch.float32, 4)
    full = _run(ops, x, w, b, g, None)
    frozen = ops.linear_act8(x, w.detach())
    assert torch.equal(torch.autograd.grad(frozen, x, g)[0], full[1])
    # one input through two layers of one weight: the gradients add up
    y = ops.linear_act8(x, w, b) + ops.linear_act8(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), g)
    assert all(torch.equal(p, 2 * q) for p, q in zip(got, full[1:]))
