"""Measured cases of the 8-bit operators: the coding of activations and weights in 8-bit integers, the product of
8-bit integers with a scale for each token and each output channel, and the linear layer that keeps its input for the
backward pass in 8 bits.

``run`` computes a case in its plain form (elementary torch operations in fp32, rounded once at the end), or,
with ``own`` set, by the calls of ``dmad_b200.ops`` that a program makes.

Layouts of the codes, whole numbers from -127 to 127 along the last dimension:

* rows (``block`` 0): one scale a row, s = max|x| / 127 in fp32 (1 for a row of zeros, never below 2^-126); the code is
  x / s rounded to the nearest whole number, halves to the even one, and the value s times the code;
* blocks of 32 columns: one power of two a block, s = 2^(floor(log2 max|x|) - 6) (never below 2^-127), kept as its
  biased exponent; codes that round to +-128 become +-127.

The linear layer with an activation, y = act(h) W^T + b, keeps h in blocks of 32 (those of the two halves of a SwiGLU's
[value | gate] each counted from the half's start), and its gradients are those at the kept values.  Sizes are those of
this package's packed audio-video sequence (37966 rows, hidden 5120, SwiGLU width 15360), its Wan 1.3B block (32760
rows, 1536 / 8960), its SDXL text context (4 x 77 rows of 2048) and generic ragged ones.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _code(name, rows, cols, block, dtype):
    return {"name": name, "op": "code", "rows": rows, "cols": cols, "block": block, "dtype": dtype}


def _linear(name, rows, out, cols, dtype, bias):
    return {"name": name, "op": "linear", "rows": rows, "out": out, "cols": cols, "dtype": dtype, "bias": bias}


def _act8(name, rows, out, cols, act, dtype, bias):
    # cols: the columns that the product sums over; a SwiGLU's input has twice as many
    return {"name": name, "op": "act8", "rows": rows, "out": out, "cols": cols, "act": act, "dtype": dtype, "bias": bias}


def listed():
    return [
        # one token's hidden state, coded and read back
        _code("code_token", 1, 5120, 0, "bf16"),
        # a ragged fp32 matrix whose rows end inside a block
        _code("code_ragged", 1001, 1543, 32, "fp32"),
        # the hidden states of one packed audio-video sequence, as a checkpoint of a block's input
        _code("code_sequence", 37966, 5120, 32, "bf16"),
        # one token through the fused q/k/v projection: the weight's bytes and the launches are all there is
        _linear("linear_token", 1, 15360, 5120, "bf16", True),
        # a prompt's 256 rows through the second feed-forward projection: few tiles, a long K
        _linear("linear_prompt", 256, 5120, 15360, "bf16", True),
        # sizes that no tile divides, fp16, no bias
        _linear("linear_ragged", 333, 1543, 1000, "fp16", False),
        # the packed sequence through the SwiGLU projection, the largest product of the block
        _linear("linear_sequence", 37966, 30720, 5120, "bf16", True),
        # a training step's key/value projection of a batch of text contexts: the smallest of the trained layers
        _act8("act8_context", 308, 1280, 2048, "", "bf16", False),
        # sizes that no tile divides, fp16, with the activation in front
        _act8("act8_ragged", 1001, 777, 1543, "gelu_tanh", "fp16", True),
        # the fused q/k/v projection of the Wan 1.3B block over a full clip
        _act8("act8_clip", 32760, 4608, 1536, "", "bf16", True),
        # its feed-forward's second projection with the GELU in front of it
        _act8("act8_clip_gelu", 32760, 1536, 8960, "gelu_tanh", "bf16", True),
        # the packed sequence through the SwiGLU and its projection
        _act8("act8_sequence", 37966, 5120, 15360, "swiglu", "bf16", True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("code", "linear", "act8"))
    if op == "code":
        rows, cols = _log(rng, 1, 37966), _log(rng, 16, 30720)
        while rows * cols > 37966 * 5120:
            rows //= 2
        c = _code("", rows, cols, rng.choice((0, 32)), rng.choice(("bf16", "fp16", "fp32")))
    elif op == "linear":
        rows, out, cols = _log(rng, 1, 37966), _log(rng, 64, 30720), _log(rng, 64, 15360)
        while rows * out * cols > 37966 * 30720 * 5120:
            rows //= 2
        c = _linear("", rows, out, cols, rng.choice(("bf16", "fp16")), rng.random() < 0.5)
    else:
        rows, out, cols = _log(rng, 1, 37966), _log(rng, 64, 15360), _log(rng, 64, 15360)
        while rows * out * cols > 37966 * 5120 * 15360:
            rows //= 2
        c = _act8("", rows, out, cols, rng.choice(("", "gelu_tanh", "swiglu")), rng.choice(("bf16", "fp16")),
                  rng.random() < 0.5)
    del c["name"]
    return c


# ----------------------------------------------------------------------------------------------- inputs


def _activations(rows, cols, dtype, g):
    """Rows of different sizes with a few channels that stand out, as hidden states have them."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    x *= torch.where(torch.rand(1, cols, device="cuda", generator=g) < 0.01, 8.0, 1.0)
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "code":
        return {"case": case, "x": _activations(case["rows"], case["cols"], dtype, g)}
    w = torch.randn(case["out"], case["cols"], device="cuda", generator=g) * 0.02
    bias = torch.randn(case["out"], device="cuda", generator=g).to(dtype) if case["bias"] else None
    if case["op"] == "linear":
        codes, scale = _encode_rows(w.to(dtype))
        data = torch.nn.functional.pad(codes.to(torch.int8), (0, -case["cols"] % 32))
        # the weight as a program keeps it: codes in rows padded to 32 bytes, and the rows' scales
        return {"case": case, "x": _activations(case["rows"], case["cols"], dtype, g), "bias": bias, "data": data,
                "scale": scale}
    width = case["cols"] * (2 if case["act"] == "swiglu" else 1)
    s = {"case": case, "x": _activations(case["rows"], width, dtype, g), "w": w.to(dtype), "bias": bias,
         "g": torch.randn(case["rows"], case["out"], device="cuda", generator=g).to(dtype)}
    for n in ("x", "w", "bias"):
        if s[n] is not None:
            s[n] = s[n].detach().requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------- plain forms


def _pow2(e):
    """2^e in fp32 for whole numbers -127 <= e <= 127, from the number's bits (a power function may round)."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _encode_rows(x):
    """(codes as fp32 whole numbers [R, K], scales [R] fp32) of rows x."""
    amax = x.float().abs().amax(-1)
    scale = torch.where(amax > 0, (amax / 127).clamp(min=2.0 ** -126), 1.0)
    # the quotient in fp64: next to a half, one in fp32 can round onto it
    codes = torch.round(x.double() / scale.double()[:, None]).clamp(-127, 127).float()
    return codes, scale


def _coded_blocks(x):
    """The values in fp32 that rows x have in blocks of 32 columns."""
    rows, cols = x.shape
    xb = torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)
    amax = xb.abs().amax(-1)
    exponent = torch.frexp(amax)[1] - 7  # frexp's mantissa is in [1/2, 1)
    exponent = torch.where(amax > 0, exponent, -127).clamp(-127, 127)[..., None]
    codes = torch.round(xb * _pow2(-exponent)).clamp(-127, 127)
    return (codes * _pow2(exponent)).view(rows, -1)[:, :cols]


def _plain_act8(s):
    act, dtype, n = s["case"]["act"], s["x"].dtype, s["case"]["cols"]
    h, w, g = s["x"].detach().float(), s["w"].detach().float(), s["g"].float()
    k = math.sqrt(2.0 / math.pi)

    def gelu(v):
        return 0.5 * v * (1.0 + torch.tanh(k * (v + 0.044715 * v * v * v)))

    def silu(v):
        return v / (1.0 + torch.exp(-v))

    if act == "gelu_tanh":
        a = gelu(h)
    elif act == "swiglu":
        a = h[:, :n] * silu(h[:, n:])
    else:
        a = h
    y = a @ w.t()
    if s["bias"] is not None:
        y += s["bias"].detach().float()
    out = {"y": y.to(dtype)}
    del y, a
    da = g @ w
    if act == "gelu_tanh":
        v = _coded_blocks(h)
        t = torch.tanh(k * (v + 0.044715 * v * v * v))
        dx = da * (0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * v * v))
        a = gelu(v)
    elif act == "swiglu":
        v, u = _coded_blocks(h[:, :n]), _coded_blocks(h[:, n:])
        p = 1.0 / (1.0 + torch.exp(-u))
        dx = torch.cat([da * u * p, da * v * p * (1.0 + u * (1.0 - p))], dim=1)
        a = v * u * p
    else:
        dx, a = da, _coded_blocks(h)
    out["dx"] = dx.to(dtype)
    del dx, da
    out["dw"] = (g.t() @ a).to(dtype)
    if s["bias"] is not None:
        out["db"] = g.sum(0).to(dtype)
    return out


def _plain(s):
    case, x = s["case"], s["x"]
    if case["op"] == "act8":
        return _plain_act8(s)
    if case["op"] == "code":
        if case["block"]:
            return _coded_blocks(x).to(x.dtype)
        codes, scale = _encode_rows(x)
        return (codes * scale[:, None]).to(x.dtype)
    codes, scale = _encode_rows(x)
    y = codes @ s["data"][:, :case["cols"]].float().t()
    y = y * scale[:, None] * s["scale"]
    if s["bias"] is not None:
        y += s["bias"].float()
    return y.to(x.dtype)


# ----------------------------------------------------------------------------------------------- one pass


def run(state):
    if not own:
        return _plain(state)
    from dmad_b200 import ops

    case, x = state["case"], state["x"]
    if case["op"] == "code":
        return ops.dequantize_int8(ops.quantize_int8(x, block=case["block"]), x.dtype)
    if case["op"] == "linear":
        w = ops.Int8Tensor(state["data"], state["scale"], 0, (case["out"], case["cols"]))
        return ops.int8_linear(x, w, state["bias"])
    y = ops.linear_act8(x, state["w"], state["bias"], act=case["act"] or None)
    names = [n for n in ("x", "w", "bias") if state[n] is not None]
    grads = torch.autograd.grad(y, [state[n] for n in names], state["g"])
    return {"y": y.detach(), **{{"x": "dx", "w": "dw", "bias": "db"}[n]: t for n, t in zip(names, grads)}}


def work(case):
    e = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    rows, cols = case["rows"], case["cols"]
    n = rows * cols
    if case["op"] == "code":
        # x in, the codes and scales out, and the values that they stand for out
        return {"bytes": n * (2 * e + 1) + (n // 32 if case["block"] else 4 * rows), "flops": 3 * n}
    out, bias = case["out"], case["out"] * e if case["bias"] else 0
    if case["op"] == "linear":
        return {"bytes": n * e + out * cols + 4 * out + rows * out * e + bias, "flops": 2 * n * out}
    # forward: x, weight and bias in, y and the codes out; backward: the gradient, the codes and the weight in, those of
    # x, weight and bias out
    h = n * (2 if case["act"] == "swiglu" else 1)
    return {"bytes": h * (2 * e + 2) + h // 16 + 2 * rows * out * e + 3 * out * cols * e + 2 * bias, "flops": 6 * n * out}


# ----------------------------------------------------------------------------------------------- in 64 bits


def _two(p):
    """2^p in fp64 for whole numbers p, by the exponent's bits."""
    return ((p.to(torch.int64) + 1023) << 52).view(torch.float64)


def _nearest(t):
    """The whole number nearest to t, the even one of two that are as near."""
    low = torch.floor(t)
    rest = t - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
    return low + up


def _rows64(x):
    """(codes, scales) of rows x from the definition: the scale is a number of fp32, all else in fp64."""
    x = x.double()
    size = x.abs().amax(1)
    s = torch.maximum((size / 127).float().double(), torch.tensor(2.0 ** -126, dtype=torch.float64, device=x.device))
    s = torch.where(size > 0, s, 1.0)
    return _nearest(x / s[:, None]).clamp(-127, 127), s


def _blocks64(x):
    """Values of x in blocks of 32 columns from the definition, in fp64."""
    x = x.double()
    out = torch.empty_like(x)
    for lo in range(0, x.shape[1], 8192):
        part = x[:, lo:lo + 8192]
        whole = part.shape[1] // 32 * 32
        for a, b, width in ((0, whole, 32), (whole, part.shape[1], part.shape[1] - whole)):
            if a == b:
                continue
            v = part[:, a:b].reshape(x.shape[0], -1, width)
            top = v.abs().amax(-1)
            p = torch.floor(torch.log2(top.clamp(min=2.0 ** -200)))
            p = torch.where(_two(p + 1) <= top, p + 1, torch.where(_two(p) > top, p - 1, p))  # where log2 is next to a whole number
            s = _two((p - 6).clamp(min=-127))[..., None]
            out[:, lo + a:lo + b] = (_nearest(v / s).clamp(-127, 127) * s).reshape(x.shape[0], b - a)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    n = case["cols"]
    if case["op"] == "code":
        if case["block"]:
            return _blocks64(s["x"])
        codes, scale = _rows64(s["x"])
        return codes * scale[:, None]
    if case["op"] == "linear":
        codes, scale = _rows64(s["x"])
        w = s["data"][:, :n].double() * s["scale"].double()[:, None]
        y = (codes @ w.t()) * scale[:, None]
        return y if s["bias"] is None else y + s["bias"].double()

    def layer(h, w, b):
        if case["act"] == "gelu_tanh":
            # (1 + tanh t) / 2 is the logistic function of 2 t
            h = h * torch.sigmoid((8.0 / math.pi) ** 0.5 * (h + 0.044715 * h ** 3))
        elif case["act"] == "swiglu":
            h = h[:, :n] * h[:, n:] * torch.sigmoid(h[:, n:])
        y = h @ w.t()
        return y if b is None else y + b

    ins = [s[k].detach().double() if s[k] is not None else None for k in ("x", "w", "bias")]
    y = layer(*ins)
    halves = [ins[0][:, :n], ins[0][:, n:]] if case["act"] == "swiglu" else [ins[0]]
    ins[0] = torch.cat([_blocks64(h) for h in halves], dim=1)
    del halves
    ins = [t.requires_grad_(True) if t is not None else None for t in ins]
    grads = torch.autograd.grad(layer(*ins), [t for t in ins if t is not None], s["g"].double())
    return {"y": y, **dict(zip(("dx", "dw", "db"), grads))}
