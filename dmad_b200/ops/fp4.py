"""Block-scaled 4-bit floating point: quantisation, its inverse, and the linear layer on 4-bit operands.

Formats (``fmt``), both of e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives):

* ``"mxfp4"``: blocks of 32 columns share the power of two ``2^(floor(log2 max|x|) - 2)`` (the OCP
  microscaling rule), stored as a biased exponent byte;
* ``"nvfp4"``: blocks of 16 columns share an e4m3 scale, ``max|x| / 6`` relative to a factor of the row.  The
  quantiser's row factor is the smallest power of two for which no block's scale passes 448; a stored
  weight may have any positive fp32 factors (one tensor-wide factor repeated, for instance).

All roundings are to the nearest, halves to the even code; values above 6 scales become 6 (mxfp4 can clip the
largest of a block by up to a quarter), and zero is +0.  A block that holds an infinity or a NaN reads back as NaN.  The CPU
path is a PyTorch restatement that gives the same bytes.

Forward only: the codes have no derivative, so inputs that require a gradient are refused while gradients are
recorded, and dual tensors (forward mode) always.  It stands beside the int8 weights of the low-VRAM path (``inference.lowmem.int8_rows``): weights
take 4.25 (mxfp4) or 4.5 (nvfp4) bits an element and the product runs on the tensor core's 4-bit kind.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import ext
from .tangent import carries_tangent

FP4_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@dataclass
class Fp4Tensor:
    """A matrix [R, K] in 4 bits (leading dimensions of ``shape`` are flattened into R).

    ``data`` uint8 [R, ceil(K / 32) * 16]: two codes a byte, the even column in the low bits, zeros past K.
    ``scales`` uint8 [ceil(R / 128), ceil(blocks / 4), 512]: tiles of 128 rows x 4 blocks, byte
    ``(row % 32) * 16 + (row % 128 // 32) * 4 + block % 4``; zeros past R and past the last block.
    ``row_scale`` fp32 [R] (nvfp4; None for mxfp4)."""

    data: torch.Tensor
    scales: torch.Tensor
    row_scale: torch.Tensor | None
    fmt: str
    shape: tuple

    @property
    def device(self):
        return self.data.device

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def nbytes(self) -> int:
        return self.data.numel() + self.scales.numel() + (4 * self.rows if self.row_scale is not None else 0)

    def row_slice(self, start: int, stop: int) -> "Fp4Tensor":
        """Rows [start, stop) of a matrix, sharing its storage; ``start`` is a multiple of 128, the rows of a tile of
        scales.  (The scales of the rows behind ``stop`` in its last tile stay; nothing reads them.)"""
        if len(self.shape) != 2 or start % 128 or not 0 <= start <= stop <= self.shape[0]:
            raise ValueError(f"row_slice: rows [{start}, {stop}) of shape {tuple(self.shape)} (a matrix, start a multiple of 128)")
        rs = None if self.row_scale is None else self.row_scale[start:stop]
        return Fp4Tensor(self.data[start:stop], self.scales[start // 128:start // 128 - (start - stop) // 128], rs, self.fmt,
                         (stop - start, self.shape[1]))

    def to(self, device) -> "Fp4Tensor":
        rs = None if self.row_scale is None else self.row_scale.to(device)
        return Fp4Tensor(self.data.to(device), self.scales.to(device), rs, self.fmt, self.shape)


def _block(fmt: str) -> int:
    if fmt not in FP4_BLOCK:
        raise ValueError(f"fmt must be one of {sorted(FP4_BLOCK)}, got {fmt!r}")
    return FP4_BLOCK[fmt]


def fp4_storage_shapes(rows: int, cols: int, fmt: str) -> tuple[tuple, tuple]:
    """Shapes of ``data`` and ``scales`` of a [rows, cols] matrix."""
    blocks = -(-cols // _block(fmt))
    return (rows, -(-cols // 32) * 16), (-(-rows // 128), -(-blocks // 4), 512)


def _columns(shape, what: str):
    """A ValueError for the shape of a single number, which has no columns."""
    if len(shape) < 1:
        raise ValueError(f"{what} must have at least one dimension, got shape {tuple(shape)}")


def _check(q: Fp4Tensor, name: str):
    _columns(q.shape, name)
    blk = _block(q.fmt)
    cols, rows = int(q.shape[-1]), 1
    for s in q.shape[:-1]:
        rows *= int(s)
    d, s = fp4_storage_shapes(rows, cols, q.fmt)
    if q.data.dtype != torch.uint8 or tuple(q.data.shape) != d:
        raise ValueError(f"{name}.data must be uint8 {d} for shape {tuple(q.shape)}, got {q.data.dtype} {tuple(q.data.shape)}")
    if q.scales.dtype != torch.uint8 or tuple(q.scales.shape) != s:
        raise ValueError(f"{name}.scales must be uint8 {s} for blocks of {blk}, got {q.scales.dtype} {tuple(q.scales.shape)}")
    if q.fmt == "nvfp4" and (q.row_scale is None or q.row_scale.dtype != torch.float32
                             or tuple(q.row_scale.shape) != (rows,)):
        raise ValueError(f"{name}.row_scale must be fp32 ({rows},) for nvfp4")
    if q.fmt == "mxfp4" and q.row_scale is not None:
        raise ValueError(f"{name}: mxfp4 has no row_scale")
    if any(t is not None and t.device != q.data.device for t in (q.scales, q.row_scale)):
        raise ValueError(f"{name}: data, scales and row_scale are on different devices")
    return rows, cols


def _no_grad(what: str, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is forward only: 4-bit codes have no gradient (call it under torch.no_grad)")
    if carries_tangent(*tensors):
        raise RuntimeError(f"{what} is forward only: 4-bit codes have no forward-mode derivative (unpack the dual tensor)")


# ----------------------------------------------------------------------------- reference math


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for integers -127 <= e <= 127, exact."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _exponent(bits: torch.Tensor) -> torch.Tensor:
    return (bits >> 23) - 127


def _tile_scales(s: torch.Tensor) -> torch.Tensor:
    R, nb = s.shape
    s = torch.nn.functional.pad(s, (0, -nb % 4, 0, -R % 128))
    s = s.reshape(-1, 4, 32, s.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return s.reshape(s.shape[0], s.shape[1], 512).contiguous()


def _untile_scales(t: torch.Tensor, R: int, nb: int) -> torch.Tensor:
    s = t.reshape(t.shape[0], t.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)
    return s.reshape(t.shape[0] * 128, t.shape[1] * 4)[:R, :nb]


def quantize_fp4_reference(x: torch.Tensor, fmt: str):
    """(data, scales, row_scale) of rows x [R, K]."""
    blk = _block(fmt)
    R, K = x.shape
    nb = -(-K // blk)
    xb = torch.nn.functional.pad(x.float(), (0, nb * blk - K)).reshape(R, nb, blk)
    bits = xb.abs().contiguous().view(torch.int32).amax(-1) if xb.numel() else torch.zeros(R, nb, dtype=torch.int32, device=x.device)
    bad = bits >= 0x7F800000  # infinities and NaN order above every finite number
    xb = torch.where(bad[..., None], torch.zeros_like(xb), xb)
    row_scale = None
    if fmt == "mxfp4":
        e = (_exponent(bits) - 2).clamp(min=-127)
        scale = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
        v = xb.abs() * _pow2(torch.where(bad, torch.zeros_like(e), -e))[..., None]
    else:
        top = torch.where(bad, torch.zeros_like(bits), bits).amax(-1)
        e = (_exponent(top) - 11 + ((top & 0x7FFFFF) > 0x280000).int()).clamp(min=-126)  # 6 * 448 = 1.3125 * 2^11
        row_scale = torch.where(top > 0, _pow2(e), torch.ones(R, device=x.device))
        inv = torch.where(top > 0, _pow2(-e), torch.ones(R, device=x.device))[:, None]
        amax = torch.where(bad, torch.zeros_like(bits), bits).view(torch.float32)
        s8 = (amax * inv / 6).to(torch.float8_e4m3fn)
        s = s8.float()[..., None]
        v = torch.where(s > 0, xb.abs() * inv[..., None] / s.clamp(min=2.0 ** -9), torch.zeros_like(xb))
        scale = torch.where(bad, torch.full_like(bits, 0x7F), s8.view(torch.uint8).int()).to(torch.uint8)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    v = (torch.round(v / step) * step).clamp(max=6.0)  # round: halves to even multiples = even codes
    code = torch.where(v < 2, 2 * v, torch.where(v < 4, v + 2, v / 2 + 4)).to(torch.uint8)
    code = torch.where((xb < 0) & (code > 0), code + 8, code)  # zero has one code
    code = torch.where(bad[..., None], torch.zeros_like(code), code).reshape(R, nb * blk)[:, :K]
    code = torch.nn.functional.pad(code, (0, -K % 32))
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), _tile_scales(scale), row_scale


def dequantize_fp4_reference(q: Fp4Tensor) -> torch.Tensor:
    """fp32 values [R, K]."""
    R, K = _check(q, "q")
    blk = FP4_BLOCK[q.fmt]
    code = torch.stack([q.data & 15, q.data >> 4], dim=-1).reshape(R, q.data.shape[1] * 2)[:, :K].long()
    lv = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=q.device)[code]
    sc = _untile_scales(q.scales, R, -(-K // blk))
    if q.fmt == "mxfp4":
        s = torch.where(sc == 255, torch.full(sc.shape, float("nan"), device=q.device),
                        _pow2(sc.int().clamp(max=254) - 127))
    else:
        s = sc.contiguous().view(torch.float8_e4m3fn).float() * q.row_scale[:, None]
    return lv * s.repeat_interleave(blk, dim=1)[:, :K]


# ----------------------------------------------------------------------------- ops


def quantize_fp4(x: torch.Tensor, fmt: str = "nvfp4") -> Fp4Tensor:
    """The 4-bit form of ``x`` [..., K] (bf16, fp16 or fp32), quantised along the last dimension."""
    nv = _block(fmt) == 16
    _no_grad("quantize_fp4", x)
    if x.is_cuda:  # the same checks are the extension's
        return Fp4Tensor(*ext().fp4_quantize(x, nv), fmt, tuple(x.shape))
    if x.dtype not in _DTYPES:
        raise ValueError(f"quantize_fp4: x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"quantize_fp4: the last dimension must hold at least one column, got {tuple(x.shape)}")
    K = x.shape[-1]
    return Fp4Tensor(*quantize_fp4_reference(x.detach().reshape(x.numel() // K, K), fmt), fmt, tuple(x.shape))


def dequantize_fp4(q: Fp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``q`` [..., K].  fp32 holds them all exactly, bf16 all those of the quantiser's (four
    significant bits of a scale by two of a code) above bf16's subnormals; fp16 rounds and can overflow."""
    if dtype not in _DTYPES:
        raise ValueError(f"dequantize_fp4: dtype must be bf16, fp16 or fp32, got {dtype}")
    _no_grad("dequantize_fp4", q.row_scale)
    _columns(q.shape, "dequantize_fp4: q")
    if not q.data.is_cuda:
        return dequantize_fp4_reference(q).to(dtype).reshape(q.shape)
    out = ext().fp4_dequantize(q.data, q.scales, q.row_scale, math.prod(q.shape[:-1]), q.shape[-1], _block(q.fmt) == 16,
                               _DTYPES.index(dtype))
    return out if len(q.shape) == 2 else out.view(q.shape)


def fp4_linear(x: torch.Tensor | Fp4Tensor, w: Fp4Tensor, bias: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x W^T + bias`` with both operands in 4 bits: ``x`` [..., K] (bf16 or fp16, quantised here to the
    weight's format, or an ``Fp4Tensor`` of that format), ``w`` [N, K], ``bias`` [N] (fp32, bf16 or fp16).

    fp32 accumulation, one rounding to ``out_dtype`` (bf16 or fp16; x's type, bf16 for a quantised x).
    """
    if len(w.shape) != 2:
        raise ValueError(f"fp4_linear: w must be a matrix, got shape {tuple(w.shape)}")
    if out_dtype not in (None, torch.bfloat16, torch.float16):
        raise ValueError(f"fp4_linear: out_dtype must be bf16 or fp16, got {out_dtype}")
    _columns(x.shape, "fp4_linear: x")
    N, K = w.shape
    nv = _block(w.fmt) == 16
    coded = isinstance(x, Fp4Tensor)
    if coded and x.fmt != w.fmt:
        raise ValueError(f"fp4_linear: x is {x.fmt}, w is {w.fmt}")
    _no_grad("fp4_linear", x.row_scale if coded else x, w.row_scale, bias)
    if w.data.is_cuda:  # the same checks are the extension's
        out = -1 if out_dtype is None else _DTYPES.index(out_dtype)
        if not coded:
            return ext().fp4_linear(x, w.data, w.scales, w.row_scale, bias, N, K, nv, out)
        if x.shape[-1] != K:
            raise ValueError(f"fp4_linear: x has {x.shape[-1]} columns, w has {K}")
        y = ext().fp4_matmul(x.data, x.scales, x.row_scale, math.prod(x.shape[:-1]), w.data, w.scales, w.row_scale, bias,
                             N, K, nv, out)
        return y if len(x.shape) == 2 else y.view(*x.shape[:-1], N)
    if not coded and x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"fp4_linear: x must be bf16 or fp16, got {x.dtype}")
    if x.shape[-1] != K:
        raise ValueError(f"fp4_linear: x has {x.shape[-1]} columns, w has {K}")
    if x.device != w.device or (bias is not None and bias.device != w.device):
        raise ValueError("fp4_linear: x, w and bias must be on one device")
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype not in _DTYPES):
        raise ValueError(f"fp4_linear: bias must be bf16, fp16 or fp32 ({N},), got {bias.dtype} {tuple(bias.shape)}")
    xq = x if coded else quantize_fp4(x.detach(), w.fmt)
    y = dequantize_fp4_reference(xq) @ dequantize_fp4_reference(w).t()
    y = y if bias is None else y + bias.detach().float()
    return y.to(out_dtype or (torch.bfloat16 if coded else x.dtype)).reshape(*xq.shape[:-1], N)
