"""8-bit integer kernels: the quantiser's bytes against the CPU restatement, the products against 64 bits, streams, graphs
and refusals."""
import pytest
import torch

from tests import _int8_oracle as oracle

pytestmark = pytest.mark.gpu
dev = "cuda"


def _ops():
    from dmad_b200 import ops
    assert ops.native_available()
    return ops


def _matrix(R, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-6, 6, (R, 1), generator=g).float())
    x[:, ::7] *= 16
    if R > 3:
        x[1] = 0
        x[2, K // 2:] = 0
        x[3] = torch.randint(-127, 128, (K,), generator=g).float() / 2  # quotients on halves
        x[3, 0] = 127.0
    return x.to(dtype)


def _same(q, ref):
    assert torch.equal(q.data.cpu(), ref.data)
    assert torch.equal(torch.nan_to_num(q.scale.cpu().float(), nan=-1.0), torch.nan_to_num(ref.scale.float(), nan=-1.0))


@pytest.mark.parametrize("block", [0, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 16), (1, 5120), (3, 33), (130, 48), (5, 1543), (4, 2049), (2, 16400), (2, 33000),
                                 (2, 40000)])
def test_quantize_gives_the_cpu_bytes(R, K, dtype, block):
    ops = _ops()
    x = _matrix(R, K, dtype, R * 7 + K)
    q, ref = ops.quantize_int8(x.to(dev), block), ops.quantize_int8(x, block)
    _same(q, ref)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(ops.dequantize_int8(q, t).cpu(), ops.dequantize_int8(ref, t))


@pytest.mark.parametrize("K", [64, 70])
@pytest.mark.parametrize("block", [0, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_extremes(dtype, block, K):
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    x = torch.zeros(9, K)
    x[1, :40] = torch.randn(40, generator=g) * 2.0 ** -130
    x[2, 3] = 2.0 ** -133
    x[3], x[4], x[5] = (torch.randn(K, generator=g) for _ in range(3))
    x[3, 5], x[4, 40], x[5, 0] = float("inf"), float("nan"), -float("inf")
    x[6] = (torch.rand(K, generator=g) - 0.5) * 6e38
    x[7, 0], x[7, 1:] = 1.0, 2.0 ** -140
    x[8] = -0.0
    x = x.to(dtype)
    q, ref = ops.quantize_int8(x.to(dev), block), ops.quantize_int8(x, block)
    _same(q, ref)
    same = lambda a, b: torch.equal(torch.nan_to_num(a, nan=5.0), torch.nan_to_num(b, nan=5.0))
    for t in (torch.float32, torch.bfloat16):
        assert same(ops.dequantize_int8(q, t).cpu(), ops.dequantize_int8(ref, t))


def test_nearly_half_quotients_are_decided_exactly():
    ops = _ops()
    s = torch.tensor(3.3333333 / 127, dtype=torch.float32)
    x = ((torch.arange(-126, 126).double() + 0.5) * s.double()).float()
    x = torch.cat([x, torch.nextafter(x, torch.tensor(9.0)), torch.nextafter(x, torch.tensor(-9.0)), torch.tensor([3.3333333])])
    x = torch.stack([x * 2.0 ** p * m for p in range(-100, 100, 7) for m in (1.0, 0.7312345, 1.9999999)])
    for v in (x, x[:, 1:]):
        q = ops.quantize_int8(v.to(dev), 0)
        assert torch.equal(q.data[:, :v.shape[1]].cpu().double(), oracle.rows(v)[0])


@pytest.mark.parametrize("block", [0, 32])
def test_quantize_strides(block):
    ops = _ops()
    big = torch.randn(40, 320).to(torch.bfloat16)
    gpu = big.to(dev)
    for view in (lambda b: b[:, 16:144], lambda b: b[::3, 1:100], lambda b: b[1:].t(), lambda b: b[:, :64].unsqueeze(0),
                 lambda b: b[0].expand(5, 320), lambda b: b.view(4, 10, 320)[:, 2:5], lambda b: b[:, :1]):
        _same(ops.quantize_int8(view(gpu), block), ops.quantize_int8(view(big).contiguous(), block))


def _check_linear(ops, M, N, K, dtype, bias, seed=0, out=None):
    x = _matrix(M, K, torch.float32, seed).clamp(-2000, 2000).to(dtype)
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(seed + 1)).mul(K ** -0.5).to(dtype)
    b = torch.randn(N).to(bias) if bias is not None else None
    bg = b.to(dev) if b is not None else None
    xq, wq = ops.quantize_int8(x.to(dev)), ops.quantize_int8(w.to(dev))
    y = ops.int8_linear(x.to(dev), wq, bg, out)
    assert torch.equal(ops.int8_linear(xq, wq, bg, out_dtype=out or dtype), y)
    torch.cuda.synchronize()
    ops.check_device_status()
    prod = (xq.data[:, :K].double() @ wq.data[:, :K].double().t()) * xq.scale.double()[:, None] * wq.scale.double()
    ref = prod if b is None else prod + bg.double()
    t = out or dtype
    # half a step of the output and fp16's smallest one; in fp32 a half each for the sum, the row factor and the last step
    # (the column factor and the bias in one)
    bound = torch.finfo(t).eps / 2 * ref.abs() * (1 + 2.0 ** -20) + torch.finfo(t).smallest_normal * torch.finfo(t).eps \
        + 3 * 2.0 ** -24 * (prod.abs() + ref.abs())
    assert y.shape == (M, N) and y.dtype == t
    assert ((y.double() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, torch.float32), (torch.float16, None), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 128), (1, 1536, 5120), (3, 130, 33), (33, 1543, 1000), (128, 256, 4096),
                                   (129, 520, 100), (256, 5120, 640), (333, 1543, 1000), (1000, 4096, 160), (2049, 4104, 96),
                                   (700, 9000, 1001), (1500, 3001, 257)])
def test_linear(M, N, K, dtype, bias):
    _check_linear(_ops(), M, N, K, dtype, bias, seed=M + N + K)


def test_linear_long_sums_and_other_output_types():
    ops = _ops()
    _check_linear(ops, 5, 70, 60000, torch.bfloat16, None, out=torch.float16)
    _check_linear(ops, 600, 2500, 20000, torch.float16, torch.float16, out=torch.bfloat16)
    # the longest sum, all at the codes' ends: 133144 * 127^2 is below 2^31, one more is not
    K = 133144
    x = ops.Int8Tensor(torch.full((300, K + 8), 127, dtype=torch.int8, device=dev), torch.ones(300, device=dev), 0, (300, K))
    w = ops.Int8Tensor(torch.full((40, K + 8), -127, dtype=torch.int8, device=dev), torch.ones(40, device=dev), 0, (40, K))
    y = ops.int8_linear(x, w)
    assert (y.float() == torch.tensor(-127.0 * 127 * K).to(torch.bfloat16).float().to(dev)).all()


@pytest.mark.parametrize("M", [4, 700])
def test_linear_factors_at_the_ends_of_fp32(M):
    ops = _ops()
    g = torch.Generator().manual_seed(1)
    K, N = 160, 9000
    x = ops.quantize_int8(torch.randn(M, K, generator=g).to(dev))
    w = ops.quantize_int8(torch.randn(N, K, generator=g).to(dev))
    prod = x.data[:, :K].double() @ w.data[:, :K].double().t()
    sx = torch.exp2(torch.linspace(-125, 118, M)).to(dev)
    for size in (2.0 ** -120, 1.0, 2.0 ** 110):
        xs, ws = ops.Int8Tensor(x.data, sx, 0, x.shape), ops.Int8Tensor(w.data, w.scale * size, 0, w.shape)
        y = ops.int8_linear(xs, ws)
        ref = prod * sx.double()[:, None] * ws.scale.double()
        big = ref.abs() > 3.3e38
        assert (y[big].isinf() | (y[big].abs() > 3.2e38)).all()
        ok = ref.abs() < 3.2e38
        err = (y.double() - ref).abs()
        # half a step of bf16, its smallest number, three roundings in fp32
        assert (err[ok] <= 2.0 ** -8 * ref.abs()[ok] * (1 + 2.0 ** -14) + 2.0 ** -133).all()
    sx[0] = float("nan")
    y = ops.int8_linear(ops.Int8Tensor(x.data, sx, 0, x.shape), w)
    assert y[0].isnan().all() and not y[1:].isnan().any()


def test_linear_ignores_what_is_stored_past_the_columns():
    ops = _ops()
    for M, N in ((3, 200), (900, 5000)):
        x, w = ops.quantize_int8(torch.randn(M, 100, device=dev)), ops.quantize_int8(torch.randn(N, 100, device=dev))
        y = ops.int8_linear(x, w)
        x.data[:, 100:], w.data[:, 100:] = 55, -77
        assert torch.equal(ops.int8_linear(x, w), y)


def test_linear_empty_and_rows():
    ops = _ops()
    w = ops.quantize_int8(torch.randn(300, 64, device=dev))
    x = torch.randn(2, 5, 64, device=dev, dtype=torch.bfloat16)
    y = ops.int8_linear(x, w)
    assert y.shape == (2, 5, 300)
    assert ops.int8_linear(x[:0], w).shape == (0, 5, 300) and ops.int8_linear(x, w.row_slice(7, 7)).shape == (2, 5, 0)
    assert torch.equal(ops.int8_linear(x, w.row_slice(5, 261)), y[..., 5:261])
    one = ops.int8_linear(x[0, 0], w)
    assert one.shape == (300,) and torch.equal(one, y[0, 0])
    wide = torch.randn(10, 200, device=dev, dtype=torch.bfloat16)
    assert torch.equal(ops.int8_linear(wide[:, 3:67], w), ops.int8_linear(wide[:, 3:67].contiguous(), w))
    assert torch.equal(ops.int8_linear(wide[:, 0].expand(64, 10).t(), w), ops.int8_linear(wide[:, :1].repeat(1, 64), w))


def test_a_row_with_an_infinity_gives_a_row_of_nan():
    ops = _ops()
    for M, N in ((8, 256), (600, 9000)):
        x = torch.randn(M, 64, device=dev, dtype=torch.bfloat16)
        w = ops.quantize_int8(torch.randn(N, 64, device=dev))
        y = ops.int8_linear(x, w)
        x[3, 7] = float("inf")
        z = ops.int8_linear(x, w)
        assert z[3].isnan().all() and torch.equal(z[:3], y[:3]) and torch.equal(z[4:], y[4:])


def test_streams_and_graphs():
    ops = _ops()
    w = ops.quantize_int8(torch.randn(4096, 1024, device=dev))
    xs = [torch.randn(M, 1024, device=dev, dtype=torch.bfloat16) for M in (3, 700)]
    want = [ops.int8_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [(ops.int8_linear(x, w), ref) for x, ref in zip(xs, want) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)
    x = xs[1].clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.int8_linear(x, w)
            z = ops.dequantize_int8(ops.quantize_int8(x, 32))
        graphs.append((g, y, z))
    for scale in (1.0, -3.0):
        x.copy_(xs[1] * scale)
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        ref, refz = ops.int8_linear(x, w), ops.dequantize_int8(ops.quantize_int8(x, 32))
        assert all(torch.equal(y, ref) and torch.equal(z, refz) for _, y, z in graphs)
    ops.check_device_status()


def test_refusals():
    ops = _ops()
    x = torch.randn(4, 64, device=dev, dtype=torch.bfloat16)
    w = ops.quantize_int8(torch.randn(8, 64, device=dev))
    I = ops.Int8Tensor
    for bad in (lambda: ops.quantize_int8(x.double()), lambda: ops.quantize_int8(x[:, :0]), lambda: ops.quantize_int8(x, 16),
                lambda: ops.quantize_int8(x[0, 0]), lambda: ops.int8_linear(x.float(), w), lambda: ops.int8_linear(x[:, :32], w),
                lambda: ops.int8_linear(x[0, 0], w),
                lambda: ops.int8_linear(x.cpu(), w), lambda: ops.int8_linear(x, w.to("cpu")),
                lambda: ops.int8_linear(x, w, torch.zeros(8)), lambda: ops.int8_linear(x, w, torch.zeros(7, device=dev)),
                lambda: ops.int8_linear(x, I(w.data.cpu(), w.scale, 0, (8, 64))),
                lambda: ops.int8_linear(x, I(w.data, w.scale.cpu(), 0, (8, 64))),
                lambda: ops.int8_linear(x, I(w.data, w.scale.double(), 0, (8, 64))),
                lambda: ops.int8_linear(x, I(w.data.view(torch.uint8), w.scale, 0, (8, 64))),
                lambda: ops.int8_linear(x, I(w.data.t(), w.scale, 0, (8, 64))),
                lambda: ops.int8_linear(x, I(w.data[:, :32], w.scale, 0, (8, 64))),
                lambda: ops.int8_linear(x, I(w.data, w.scale[:7], 0, (8, 64))),
                lambda: ops.int8_linear(ops.quantize_int8(x, 32), w), lambda: ops.int8_linear(x, ops.quantize_int8(x, 32)),
                lambda: ops.int8_linear(I(w.data[:4], w.scale[:4], 0, (4, 60)), w),
                lambda: ops.dequantize_int8(I(w.data, w.scale, 32, (8, 64))),
                lambda: ops.dequantize_int8(I(w.data, w.scale, 0, (8, 32))), lambda: ops.dequantize_int8(w, torch.int8)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="forward only"):
        ops.int8_linear(x.requires_grad_(True), w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("K", [1, 15, 17, 31, 500, 513, 529, 1039, 4111])
def test_rows_that_start_anywhere(K, dtype):
    """Every offset of a row's start, read and written back, and nothing written beside the rows."""
    ops = _ops()
    for start in range(0, 18):
        wide = _matrix(7, K + 40, dtype, K + start)
        x, xg = wide[:, start:start + K], wide.to(dev)[:, start:start + K]
        for block in (0, 32):
            q, ref = ops.quantize_int8(xg, block), ops.quantize_int8(x.contiguous(), block)
            _same(q, ref)
            assert torch.equal(ops.dequantize_int8(q, dtype).cpu(), ops.dequantize_int8(ref, dtype))
    w = ops.quantize_int8(torch.randn(40, K, device=dev))
    line = torch.randn(K + 40, device=dev).to(torch.bfloat16)
    for start in range(0, 18):  # one row: coded within the product
        x = line[start:start + K]
        assert torch.equal(ops.int8_linear(x, w), ops.int8_linear(ops.quantize_int8(x), w, None, torch.bfloat16))


def test_offsets_past_32_bits():
    ops = _ops()
    R, K = 70000, 32768  # 2.3e9 elements
    x = torch.zeros(R, K, dtype=torch.bfloat16, device=dev)
    rows = [0, 1, 65535, 65536, 65537, R - 1]
    part = torch.randn(len(rows), K, device=dev).to(torch.bfloat16)
    x[rows] = part
    for block in (0, 32):
        q = ops.quantize_int8(x, block)
        ref = ops.quantize_int8(part, block)
        assert torch.equal(q.data[rows], ref.data) and torch.equal(q.scale[rows], ref.scale)
        assert torch.equal(ops.dequantize_int8(q)[rows], ops.dequantize_int8(ref))
        del q
    del x
    torch.cuda.empty_cache()
    w = ops.quantize_int8(torch.randn(K, 64, device=dev))
    x = torch.randn(R, 64, device=dev, dtype=torch.bfloat16)
    y = ops.int8_linear(x, w)  # 2.3e9 outputs
    for r in (0, 65535, 65536, R - 200):
        assert torch.equal(y[r:r + 200], ops.int8_linear(x[r:r + 200].contiguous(), w))
    del y
    torch.cuda.empty_cache()


def test_calls_one_behind_the_other():
    """Calls whose kernels overlap, over memory that the calls before have just freed: the results of calls that are waited for."""
    ops = _ops()
    g = torch.Generator().manual_seed(9)
    shapes = [(1, 700, 500), (40, 1000, 4000), (200, 300, 5000), (300, 2500, 1001), (1200, 5200, 640), (2600, 2600, 2600)]
    args = [(torch.randn(M, K, generator=g).to(torch.bfloat16).to(dev), ops.quantize_int8(torch.randn(N, K, generator=g).to(dev)),
             torch.randn(N, generator=g).to(dev)) for M, N, K in shapes]
    want = []
    for x, w, b in args:
        torch.cuda.synchronize()
        want.append((ops.int8_linear(x, w, b), ops.dequantize_int8(ops.quantize_int8(x, 32))))
    torch.cuda.synchronize()
    order = torch.randint(0, len(shapes), (300,), generator=g).tolist()
    wrong = torch.zeros((), device=dev, dtype=torch.int64)
    for i in order:
        x, w, b = args[i]
        y, z = ops.int8_linear(x, w, b), ops.dequantize_int8(ops.quantize_int8(x, 32))
        wrong += (y != want[i][0]).sum() + (z != want[i][1]).sum()
        del y, z
    assert int(wrong) == 0
    kept = [(i, ops.int8_linear(*args[i])) for i in order[:100]]
    assert all(torch.equal(y, want[i][0]) for i, y in kept)
