"""Measured cases of the 4-bit inference path's operators: block-scaled 4-bit quantisation, the product of
4-bit operands, and the per-head norm of queries and keys with the position rotation.

``run`` computes a case in its plain form (elementary torch operations in fp32, rounded once at the end), or,
with ``own`` set, by the calls of ``dmad_b200.ops`` that a program makes.

Formats (both store two e2m1 codes a byte, the even column in the low four bits, rows padded to 16 bytes):

* ``mxfp4``: blocks of 32 columns share a power of two, 2^(floor(log2 max|x|) - 2), kept as its biased exponent;
* ``nvfp4``: blocks of 16 columns share an e4m3 scale of max|x| / 6, relative to a power of two of the row, the
  smallest for which no block's scale passes 448.

Block scales are stored in tiles of 128 rows x 4 blocks: [row tiles, block tiles, 512], byte
(row % 32) * 16 + (row / 32) * 4 + block of a tile.  Sizes are those of this package's packed audio-video
sequence (37966 rows of 40 heads of 128, hidden 5120, SwiGLU width 15360), its Wan 1.3B block (1536 / 8960)
and generic ragged ones.
"""
import math

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BLOCK = {"mxfp4": 32, "nvfp4": 16}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _quantize(name, op, rows, cols, fmt, dtype):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "fmt": fmt, "dtype": dtype}


def _linear(name, rows, out, cols, fmt, dtype, bias):
    return {"name": name, "op": "linear", "rows": rows, "out": out, "cols": cols, "fmt": fmt, "dtype": dtype, "bias": bias}


def _headnorm(name, rows, hq, hk, hd, rot, layout, dtype, wdtype, positions, grad):
    return {"name": name, "op": "headnorm", "rows": rows, "hq": hq, "hk": hk, "hd": hd, "rot": rot, "layout": layout,
            "dtype": dtype, "wdtype": wdtype, "positions": positions, "grad": grad}


def listed():
    return [
        # one token's hidden state, coded and read back
        _quantize("quant_token", "quantize", 1, 5120, "nvfp4", "bf16"),
        # a ragged fp32 matrix whose rows end inside a block: weights of a layer with odd widths
        _quantize("quant_ragged", "quantize", 1001, 1543, "mxfp4", "fp32"),
        # the hidden states of one packed audio-video sequence
        _quantize("quant_sequence", "quantize", 37966, 5120, "nvfp4", "bf16"),
        # one token through the fused q/k/v projection: the weight's bytes and the launches are all there is
        _linear("linear_token", 1, 15360, 5120, "nvfp4", "bf16", True),
        # a prompt's 256 rows through the second feed-forward projection: few tiles, a long K
        _linear("linear_prompt", 256, 5120, 15360, "mxfp4", "bf16", True),
        # sizes that no tile divides, fp16, no bias
        _linear("linear_ragged", 333, 1543, 1000, "nvfp4", "fp16", False),
        # the Wan 1.3B block's first feed-forward projection over a full clip
        _linear("linear_clip", 32760, 8960, 1536, "mxfp4", "bf16", True),
        # the packed sequence through the SwiGLU projection, the largest product of the block
        _linear("linear_sequence", 37966, 30720, 5120, "nvfp4", "bf16", True),
        # one new token of 40 heads at its place in the position table
        _headnorm("headnorm_token", 1, 40, 40, 128, 128, "pairs", "bf16", "bf16", True, False),
        # grouped heads with the half-split rotation of part of the head, as text decoders have them
        _headnorm("headnorm_grouped", 4097, 64, 8, 128, 64, "halves", "fp16", "fp32", True, False),
        # the packed sequence's queries and keys
        _headnorm("headnorm_sequence", 37966, 40, 40, 128, 128, "pairs", "bf16", "bf16", False, False),
        # the same in a training step: outputs and all gradients
        _headnorm("headnorm_train", 37966, 40, 40, 128, 128, "pairs", "bf16", "fp32", False, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "headnorm"))
    fmt = rng.choice(("mxfp4", "nvfp4"))
    if op == "quantize":
        rows, cols = _log(rng, 1, 37966), _log(rng, 16, 15360)
        while rows * cols > 37966 * 5120:
            rows //= 2
        c = _quantize("", op, rows, cols, fmt, rng.choice(("bf16", "fp16", "fp32")))
    elif op == "linear":
        rows, out, cols = _log(rng, 1, 37966), _log(rng, 64, 30720), _log(rng, 64, 15360)
        while rows * out * cols > 37966 * 30720 * 5120:
            rows //= 2
        c = _linear("", rows, out, cols, fmt, rng.choice(("bf16", "fp16")), rng.random() < 0.5)
    else:
        hd = rng.choice((32, 64, 80, 96, 128, 256))
        hk = _log(rng, 1, 40)
        hq = hk * rng.choice((1, 1, 2, 4, 8))
        rows = _log(rng, 1, 37966)
        while rows * (hq + hk) * hd > 37966 * 80 * 128:
            rows //= 2
        rot = hd if rng.random() < 0.6 else rng.choice((0, hd // 2))
        c = _headnorm("", rows, hq, hk, hd, rot, rng.choice(("pairs", "halves")), rng.choice(("bf16", "fp16", "fp32")),
                      rng.choice(("bf16", "fp32")), rng.random() < 0.5, rng.random() < 0.5)
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
    if case["op"] == "quantize":
        return {"case": case, "x": _activations(case["rows"], case["cols"], dtype, g)}
    if case["op"] == "linear":
        w = torch.randn(case["out"], case["cols"], device="cuda", generator=g) * 0.02
        codes, scales, row_scale = _encode(w.to(dtype), case["fmt"])
        bias = torch.randn(case["out"], device="cuda", generator=g).to(dtype) if case["bias"] else None
        # the weight as a program keeps it: packed codes, tiled block scales, row scales
        return {"case": case, "x": _activations(case["rows"], case["cols"], dtype, g), "bias": bias,
                "data": _pack(codes), "scales": _tile(scales), "row_scale": row_scale}
    rows, hq, hk, hd, rot = (case[k] for k in ("rows", "hq", "hk", "hd", "rot"))
    qkv = torch.randn(rows, (hq + 2 * hk) * hd, device="cuda", generator=g).to(dtype)  # a fused projection's output
    q = qkv[:, :hq * hd].view(rows, hq, hd)
    k = qkv[:, hq * hd:(hq + hk) * hd].view(rows, hk, hd)
    wq, wk = (1 + 0.2 * torch.randn(2, hd, device="cuda", generator=g)).to(DTYPES[case["wdtype"]]).unbind()
    s = {"case": case, "q": q, "k": k, "wq": wq.contiguous(), "wk": wk.contiguous(), "cos": None, "sin": None,
         "positions": None}
    places = rows
    if case["positions"]:
        places = 2 * rows + 4096
        s["positions"] = torch.randint(0, places, (rows,), device="cuda", generator=g)
    if rot:
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(places, device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["positions"] = None
    if case["grad"]:
        s["gq"] = torch.randn(rows, hq, hd, device="cuda", generator=g).to(dtype)
        s["gk"] = torch.randn(rows, hk, hd, device="cuda", generator=g).to(dtype)
        for n in ("q", "k", "wq", "wk"):
            s[n] = s[n].detach().requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------- plain forms


def _pow2(e):
    """2^e in fp32 for whole numbers -127 <= e <= 127, from the number's bits (a power function may round)."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _encode(x, fmt):
    """(codes [R, K] uint8, block scales [R, blocks] uint8, row scales [R] fp32 or None) of rows x."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    blocks = -(-cols // block)
    xb = torch.nn.functional.pad(x.float(), (0, blocks * block - cols)).view(rows, blocks, block)
    amax = xb.abs().amax(-1)
    if fmt == "mxfp4":
        exponent = torch.frexp(amax)[1] - 3  # frexp's mantissa is in [1/2, 1)
        exponent = torch.where(amax > 0, exponent, -127).clamp(-127, 127)
        stored = (exponent + 127).to(torch.uint8)
        v = xb.abs() * _pow2(-exponent)[..., None]
        row_scale = None
    else:
        m, e = torch.frexp(amax.amax(-1))
        e = torch.where(m > 1.3125 / 2, e - 11, e - 12).clamp(-126, 126)  # 6 * 448 = 1.3125 * 2^11
        row_scale = torch.where(amax.amax(-1) > 0, _pow2(e), 1.0)
        scale = (amax / row_scale[:, None] / 6).to(torch.float8_e4m3fn)
        stored = scale.view(torch.uint8)
        s = scale.float()[..., None]
        v = torch.where(s > 0, xb.abs() / row_scale[:, None, None] / s, 0.0)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(max=6)  # halves go to the even code
    code = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4)).to(torch.uint8)
    code = torch.where(torch.signbit(xb), code + 8, code)
    return code.view(rows, blocks * block)[:, :cols], stored, row_scale


def _pack(codes):
    rows, cols = codes.shape
    c = torch.nn.functional.pad(codes, (0, -cols % 32))
    return (c[:, 0::2] | (c[:, 1::2] << 4)).contiguous()


def _tile(scales):
    rows, blocks = scales.shape
    s = torch.nn.functional.pad(scales, (0, -blocks % 4, 0, -rows % 128))
    s = s.view(-1, 4, 32, s.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return s.reshape(s.shape[0], s.shape[1], 512)


def _untile(tiles, rows, blocks):
    s = tiles.view(tiles.shape[0], tiles.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)
    return s.reshape(tiles.shape[0] * 128, -1)[:rows, :blocks]


def _unpack(data, cols):
    return torch.stack([data & 15, data >> 4], dim=-1).view(data.shape[0], -1)[:, :cols]


def _values(codes, scales, row_scale, fmt):
    """What codes and scales stand for, in fp32."""
    rows, cols = codes.shape
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)[codes.long()]
    if fmt == "mxfp4":
        s = _pow2(scales.int() - 127)
    else:
        s = scales.contiguous().view(torch.float8_e4m3fn).float() * row_scale[:, None]
    return level * s.repeat_interleave(BLOCK[fmt], dim=1)[:, :cols]


def _rotate(x, cos, sin, layout, rot):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if layout == "pairs" else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    r = torch.stack([ra, rb], dim=-1).flatten(-2) if layout == "pairs" else torch.cat([ra, rb], dim=-1)
    return torch.cat([r, x[..., rot:]], dim=-1)


def _plain_headnorm(s):
    case = s["case"]
    rot, eps = case["rot"], 1e-6
    cos = sin = None
    if rot:
        at = s["positions"] if s["positions"] is not None else torch.arange(case["rows"], device="cuda") % s["cos"].shape[0]
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    outs, grads = [], []
    for x0, w0, g0 in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        x, w = x0.detach().float(), w0.detach().float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        n = x * r
        y = n * w
        outs.append((_rotate(y, cos, sin, case["layout"], rot) if rot else y).to(x0.dtype))
        if g0 is not None:
            gy = _rotate(g0.float(), cos, -sin, case["layout"], rot) if rot else g0.float()
            gn = gy * w
            grads.append(((gn - n * (gn * n).mean(-1, keepdim=True)) * r).to(x0.dtype))
            grads.append((gy * n).sum((0, 1)).to(w0.dtype))
    if not grads:
        return {"q": outs[0], "k": outs[1]}
    return {"q": outs[0], "k": outs[1], "dq": grads[0], "dk": grads[2], "dwq": grads[1], "dwk": grads[3]}


def _plain(s):
    case = s["case"]
    if case["op"] == "headnorm":
        return _plain_headnorm(s)
    fmt, x = case["fmt"], s["x"]
    xv = _values(*_encode(x, fmt), fmt)
    if case["op"] == "quantize":
        return xv.to(torch.float32 if x.dtype == torch.float16 else x.dtype)
    scales = _untile(s["scales"], case["out"], -(-case["cols"] // BLOCK[fmt]))
    y = xv @ _values(_unpack(s["data"], case["cols"]), scales, s["row_scale"], fmt).t()
    if s["bias"] is not None:
        y += s["bias"].float()
    return y.to(x.dtype)


# ----------------------------------------------------------------------------------------------- one pass


def run(state):
    if not own:
        return _plain(state)
    from dmad_b200 import ops

    case = state["case"]
    if case["op"] == "quantize":
        x = state["x"]
        # every value of either format is a bf16 number; fp16 is too narrow for the largest
        return ops.dequantize_fp4(ops.quantize_fp4(x, case["fmt"]),
                                  torch.float32 if x.dtype == torch.float16 else x.dtype)
    if case["op"] == "linear":
        w = ops.Fp4Tensor(state["data"], state["scales"], state["row_scale"], case["fmt"], (case["out"], case["cols"]))
        return ops.fp4_linear(state["x"], w, state["bias"])
    args = [state[n] for n in ("q", "k", "wq", "wk")]
    q, k = ops.qk_head_norm_rope(*args, state["cos"], state["sin"], positions=state["positions"], eps=1e-6,
                                 interleaved=case["layout"] == "pairs")
    if not case["grad"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), args, (state["gq"], state["gk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    e = size[case["dtype"]]
    if case["op"] == "headnorm":
        n = case["rows"] * (case["hq"] + case["hk"]) * case["hd"]
        table = 2 * case["rows"] * case["rot"] // 2 * 4 + (8 * case["rows"] if case["positions"] else 0)
        # forward: x in, y out; with gradients: g in, dx out as well
        return {"bytes": n * e * (4 if case["grad"] else 2) + table + 4 * case["hd"] * size[case["wdtype"]],
                "flops": n * (20 if case["grad"] else 7)}
    fmt = case["fmt"]
    coded = 0.5 + 1 / BLOCK[fmt]
    n = case["rows"] * case["cols"]
    if case["op"] == "quantize":
        # x in, the codes and scales out, and the values that they stand for out
        return {"bytes": n * (e + coded + (2 if e == 2 and case["dtype"] == "bf16" else 4)), "flops": 4 * n}
    return {"bytes": n * e + case["out"] * case["cols"] * coded + case["rows"] * case["out"] * e
            + (case["out"] * e if case["bias"] else 0),
            "flops": 2 * n * case["out"]}


# ----------------------------------------------------------------------------------------------- in 64 bits


def _two(p):
    """2^p in fp64 for whole numbers p, by the exponent's bits."""
    return ((p.to(torch.int64) + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """v >= 0 rounded to the nearest e4m3 number, halves to the even one: steps of 2^(e - 3), 2^-9 below 2^-6."""
    e = torch.floor(torch.log2(v.clamp(min=2.0 ** -30)))
    step = _two(e.clamp(min=-6.0) - 3)
    return torch.round(v / step) * step


def _coded(x, fmt):
    """The values that the 4-bit form of x stands for, from the definition, in fp64."""
    rows, cols = x.shape
    block = BLOCK[fmt]
    x = x.double()
    out = torch.empty_like(x)
    whole = cols // block * block
    parts = [(0, whole, block)] if whole else []
    if whole < cols:
        parts.append((whole, cols, cols - whole))
    size = x.abs().amax(1)
    # the smallest power of two with size / (6 * 448) below it
    g = _two(torch.ceil(torch.log2(size.clamp(min=2.0 ** -200) / 2688.0)))
    g = torch.where(size / 2688.0 > g, 2 * g, torch.where(size / 2688.0 <= g / 2, g / 2, g))[:, None]
    for lo, hi, width in parts:
        b = x[:, lo:hi].reshape(rows, -1, width)
        top = b.abs().amax(-1)
        if fmt == "mxfp4":
            p = torch.floor(torch.log2(top.clamp(min=2.0 ** -200)))
            p = torch.where(_two(p + 1) <= top, p + 1, torch.where(_two(p) > top, p - 1, p))
            s = _two((p - 2).clamp(min=-127))
        else:
            s = _e4m3(top / (6 * g)) * g
        t = torch.where(s[..., None] > 0, b.abs() / s[..., None], 0.0)
        v = torch.zeros_like(t)
        at = 0.0
        # a half goes to the neighbour with the even code: down at 1/4, 5/4, 5/2 and 5, up at 3/4, 7/4 and 7/2
        for border, nxt, up in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True),
                                (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
            v += (nxt - at) * ((t >= border) if up else (t > border))
            at = nxt
        out[:, lo:hi] = (torch.sign(b) * v * s[..., None]).view(rows, hi - lo)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _coded(s["x"], case["fmt"])
    if case["op"] == "linear":
        rows, cols, block = case["out"], case["cols"], BLOCK[case["fmt"]]
        code = torch.empty(rows, s["data"].shape[1] * 2, dtype=torch.long, device="cuda")
        code[:, 0::2], code[:, 1::2] = s["data"] % 16, s["data"] // 16
        low, sign = code[:, :cols] % 8, 1.0 - 2.0 * (code[:, :cols] // 8).double()
        w = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")[low] * sign
        r = torch.arange(rows, device="cuda")[:, None]
        b = torch.arange(cols, device="cuda")[None] // block
        byte = s["scales"][r // 128, b // 4, (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4].double()
        if case["fmt"] == "mxfp4":
            w *= _two(byte - 127)
        else:
            e, m = torch.floor(byte / 8), byte % 8
            w *= torch.where(e > 0, (8 + m) * _two(e - 10), m * 2.0 ** -9) * s["row_scale"].double()[:, None]
        y = _coded(s["x"], case["fmt"]) @ w.t()
        return y if s["bias"] is None else y + s["bias"].double()
    rot, rows, hd = case["rot"], case["rows"], case["hd"]
    turn = None
    if rot:
        at = s["positions"] if s["positions"] is not None else torch.arange(rows, device="cuda")
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]
    ins = [s[n].detach().double().requires_grad_(case["grad"]) for n in ("q", "k", "wq", "wk")]
    outs = []
    for x, w in ((ins[0], ins[2]), (ins[1], ins[3])):
        y = x / (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * w
        if rot:
            # each pair of coordinates is a complex number, turned by its position's angle
            h = y[..., :rot]
            z = h.reshape(rows, -1, rot // 2, 2) if case["layout"] == "pairs" else h.reshape(rows, -1, 2, rot // 2).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = z.reshape(h.shape) if case["layout"] == "pairs" else z.transpose(-1, -2).reshape(h.shape)
            y = torch.cat([z, y[..., rot:]], dim=-1)
        outs.append(y)
    if not case["grad"]:
        return {"q": outs[0], "k": outs[1]}
    dq, dk, dwq, dwk = torch.autograd.grad(outs, ins, [s["gq"].double(), s["gk"].double()])
    return {"q": outs[0].detach(), "k": outs[1].detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
