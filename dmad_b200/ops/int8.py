"""8-bit integers: the coding of activations and weights, its inverse, and the linear layer on 8-bit operands.

Codes are whole numbers from -127 to 127 along the last dimension, in one of two layouts (``block``):

* 0, rows: one fp32 scale a row, ``s = max|x| / 127`` (1 for a row of zeros; 2^-126 at least, and at
  most the largest whose 127-fold is finite).  What ``int8_linear``
  multiplies: a scale for each token and for each output channel;
* 32, blocks of 32 columns: one power of two a block, ``s = 2^(floor(log2 max|x|) - 6)`` (2^-127 at least), stored as a
  biased exponent byte; codes of +-128 become +-127.  What activations are kept in for a backward pass
  (``linear_act8``, the ``block_int8`` checkpoint policy): small channels beside large ones keep their digits, and every
  value is a bf16 number.

A code is ``x / s`` rounded to the nearest whole number, halves to the even one, decided exactly.  A row or block that
holds an infinity or a NaN reads back as NaN.  The CPU path is a PyTorch restatement that gives the same bytes.

Forward only: the codes have no derivative, so inputs that require a gradient are refused while gradients are recorded, and
dual tensors (forward mode) always.  ``inference.lowmem.int8_rows`` codes the weights that the low-VRAM path streams; those
are decoded before each product, these are multiplied as they are.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import ext
from .tangent import carries_tangent

INT8_BLOCKS = (0, 32)
INT8_MAX_K = 133144  # 2^31 / 127^2: the longest sum that int32 holds
INT8_MIN_SCALE, INT8_MAX_SCALE = 2.0 ** -126, float.fromhex("0x1.020406p121")
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


@dataclass
class Int8Tensor:
    """A matrix [R, K] in 8 bits (leading dimensions of ``shape`` are flattened into R).

    ``data`` int8 [R, ceil(K / 32) * 32], from -127 to 127 (what is stored past K is not used).  ``scale``: fp32 [R] (``block`` 0), or uint8 [R, ceil(K / 32)],
    the exponent plus 127 of each block's power of two, 255 for NaN (``block`` 32)."""

    data: torch.Tensor
    scale: torch.Tensor
    block: int
    shape: tuple

    @property
    def device(self):
        return self.data.device

    @property
    def rows(self) -> int:
        return self.data.shape[0]

    @property
    def nbytes(self) -> int:
        return self.data.numel() + self.scale.numel() * self.scale.element_size()

    def row_slice(self, start: int, stop: int) -> "Int8Tensor":
        """Rows [start, stop) of a matrix, sharing its storage."""
        if len(self.shape) != 2 or not 0 <= start <= stop <= self.shape[0]:
            raise ValueError(f"row_slice: rows [{start}, {stop}) of shape {tuple(self.shape)} (a matrix)")
        return Int8Tensor(self.data[start:stop], self.scale[start:stop], self.block, (stop - start, self.shape[1]))

    def to(self, device) -> "Int8Tensor":
        return Int8Tensor(self.data.to(device), self.scale.to(device), self.block, self.shape)


def _block(block) -> bool:
    """Whether ``block`` means blocks of 32."""
    if block not in INT8_BLOCKS:
        raise ValueError(f"block must be 0 (one scale a row) or 32, got {block!r}")
    return block == 32


def _columns(shape, what: str):
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"{what}: the last dimension must hold at least one column, got {tuple(shape)}")


def _check(q: Int8Tensor, name: str):
    blocks = _block(q.block)
    _columns(q.shape, name)
    rows, cols = math.prod(int(s) for s in q.shape[:-1]), int(q.shape[-1])
    d, s = (rows, -(-cols // 32) * 32), (rows, -(-cols // 32)) if blocks else (rows,)
    want = torch.uint8 if blocks else torch.float32
    if q.data.dtype != torch.int8 or tuple(q.data.shape) != d:
        raise ValueError(f"{name}.data must be int8 {d} for shape {tuple(q.shape)}, got {q.data.dtype} {tuple(q.data.shape)}")
    if q.scale.dtype != want or tuple(q.scale.shape) != s:
        raise ValueError(f"{name}.scale must be {want} {s} for block {q.block}, got {q.scale.dtype} {tuple(q.scale.shape)}")
    if q.scale.device != q.data.device:
        raise ValueError(f"{name}: data and scale must be on one device")
    return rows, cols


def _no_grad(what: str, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} is forward only: 8-bit codes have no gradient (call it under torch.no_grad)")
    if carries_tangent(*tensors):
        raise RuntimeError(f"{what} is forward only: 8-bit codes have no forward-mode derivative (unpack the dual tensor)")


# ----------------------------------------------------------------------------- reference math


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 for integers -127 <= e <= 127, exact."""
    e = e.to(torch.int32)
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def quantize_int8_reference(x: torch.Tensor, block: int = 0):
    """(data, scale) of rows x [R, K]."""
    R, K = x.shape
    pad = -K % 32
    xp = torch.nn.functional.pad(x.float(), (0, pad))
    if _block(block):
        xp = xp.reshape(R, (K + pad) // 32, 32)
    bits = xp.abs().contiguous().view(torch.int32).amax(-1)
    bad = bits >= 0x7F800000  # infinities and NaN order above every finite number
    xp = torch.where(bad[..., None], torch.zeros_like(xp), xp)
    if _block(block):
        e = ((bits >> 23) - 6).clamp(min=0)
        scale = torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)
        codes = torch.round(xp * _pow2(torch.where(bad, torch.zeros_like(e), 127 - e))[..., None]).clamp(-127, 127)
    else:
        s = (torch.where(bad, torch.zeros_like(bits), bits).view(torch.float32) / 127).clamp(INT8_MIN_SCALE, INT8_MAX_SCALE)
        s = torch.where(bits == 0, torch.ones_like(s), s)
        codes = torch.round(xp.double() / s.double()[..., None])  # in fp64, where no quotient rounds onto a half
        scale = torch.where(bad, torch.full_like(s, float("nan")), s)
    return codes.to(torch.int8).reshape(R, K + pad), scale


def _scales(q: Int8Tensor) -> torch.Tensor:
    """fp32 scales that broadcast over ``data``'s rows (or over its blocks of 32)."""
    if not _block(q.block):
        return q.scale[:, None]
    s = q.scale.int()
    return torch.where(s == 255, torch.full(s.shape, float("nan"), device=q.device), _pow2(s.clamp(max=254) - 127))[..., None]


def dequantize_int8_reference(q: Int8Tensor) -> torch.Tensor:
    """fp32 values [R, K]."""
    R, K = _check(q, "q")
    v = q.data.float()
    if _block(q.block):
        v = v.reshape(R, v.shape[1] // 32, 32)
    return (v * _scales(q)).reshape(q.data.shape)[:, :K]


# ----------------------------------------------------------------------------- ops


def quantize_int8(x: torch.Tensor, block: int = 0) -> Int8Tensor:
    """The 8-bit form of ``x`` [..., K] (bf16, fp16 or fp32), coded along the last dimension with one scale a row
    (``block`` 0) or a power of two for each 32 columns (``block`` 32)."""
    blocks = _block(block)
    _no_grad("quantize_int8", x)
    if x.is_cuda:  # the same checks are the extension's
        return Int8Tensor(*ext().int8_quantize(x, blocks), block, tuple(x.shape))
    if x.dtype not in _DTYPES:
        raise ValueError(f"quantize_int8: x must be bf16, fp16 or fp32, got {x.dtype}")
    _columns(x.shape, "quantize_int8")
    K = x.shape[-1]
    return Int8Tensor(*quantize_int8_reference(x.detach().reshape(x.numel() // K, K), block), block, tuple(x.shape))


def dequantize_int8(q: Int8Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``q`` [..., K], code times scale, rounded to ``dtype``.  bf16 holds those of blocks exactly (above its
    subnormals)."""
    if dtype not in _DTYPES:
        raise ValueError(f"dequantize_int8: dtype must be bf16, fp16 or fp32, got {dtype}")
    _no_grad("dequantize_int8", q.scale)
    _columns(q.shape, "dequantize_int8: q")
    if not q.data.is_cuda:
        return dequantize_int8_reference(q).to(dtype).reshape(q.shape)
    out = ext().int8_dequantize(q.data, q.scale, math.prod(q.shape[:-1]), q.shape[-1], _block(q.block), _DTYPES.index(dtype))
    return out if len(q.shape) == 2 else out.view(q.shape)


def int8_linear(x: torch.Tensor | Int8Tensor, w: Int8Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``x W^T + bias`` with both operands in 8-bit integers: ``x`` [..., K] (bf16 or fp16, coded here with one scale a
    row, or an ``Int8Tensor`` of that layout), ``w`` [N, K] with one scale a row, ``bias`` [N] (fp32, bf16 or fp16).

    The sums are exact (int32, so K <= 133144); scales, bias and one rounding to ``out_dtype`` (bf16 or fp16; x's type, bf16
    for a coded x) follow in fp32.  A row of ``x`` with an infinity or a NaN gives a row of NaN.
    """
    if len(w.shape) != 2:
        raise ValueError(f"int8_linear: w must be a matrix, got shape {tuple(w.shape)}")
    if out_dtype not in (None, torch.bfloat16, torch.float16):
        raise ValueError(f"int8_linear: out_dtype must be bf16 or fp16, got {out_dtype}")
    N, K = w.shape
    coded = isinstance(x, Int8Tensor)
    if _block(w.block) or (coded and _block(x.block)):
        raise ValueError("int8_linear: x and w have one scale a row (block 0)")
    _no_grad("int8_linear", x.scale if coded else x, w.scale, bias)
    if w.data.is_cuda:  # the same checks are the extension's
        out = -1 if out_dtype is None else _DTYPES.index(out_dtype)
        if not coded:
            return ext().int8_linear(x, w.data, w.scale, bias, N, K, out)
        _columns(x.shape, "int8_linear: x")
        if x.shape[-1] != K:
            raise ValueError(f"int8_linear: x has {x.shape[-1]} columns, w has {K}")
        y = ext().int8_matmul(x.data, x.scale, math.prod(x.shape[:-1]), w.data, w.scale, bias, N, K, out)
        return y if len(x.shape) == 2 else y.view(*x.shape[:-1], N)
    _columns(x.shape, "int8_linear: x")
    if not coded and x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"int8_linear: x must be bf16 or fp16, got {x.dtype}")
    if x.shape[-1] != K:
        raise ValueError(f"int8_linear: x has {x.shape[-1]} columns, w has {K}")
    if K > INT8_MAX_K:
        raise ValueError(f"int8_linear: {K} columns: int32 sums hold {INT8_MAX_K} at most")
    if x.device != w.device or (bias is not None and bias.device != w.device):
        raise ValueError("int8_linear: x, w and bias must be on one device")
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype not in _DTYPES):
        raise ValueError(f"int8_linear: bias must be bf16, fp16 or fp32 ({N},), got {bias.dtype} {tuple(bias.shape)}")
    xq = x if coded else quantize_int8(x.detach())
    _check(xq, "x")
    _check(w, "w")
    y = xq.data[:, :K].double() @ w.data[:, :K].double().t()  # whole numbers below 2^53
    y = y * xq.scale.double()[:, None] * w.scale.double()
    y = y if bias is None else y + bias.detach().double()
    return y.to(out_dtype or (torch.bfloat16 if coded else x.dtype)).reshape(*xq.shape[:-1], N)
