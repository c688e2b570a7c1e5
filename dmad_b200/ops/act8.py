"""The linear layer that keeps its input in 8 bits for the backward pass, with an activation in front of it.

    y = act(x) W^T + bias,      dW = g^T act(x'),   dx = (g W) act'(x'),   db = sum of g over the rows

``x'`` are the values of ``x`` coded in 8-bit integers, blocks of 32 columns sharing a power of two (``ops.quantize_int8(x,
32)``; a SwiGLU's two halves are coded each from its start).  The forward pass is that of ``x`` itself; the backward pass
needs 1.03 bytes an element of ``x`` instead of the two of ``x`` and, with an activation, the two of ``act(x)`` besides.
A code is off by at most half a step, 2^-7 of its block's largest element (a step where it is clipped, next to 2^7 steps),
so gradients differ from those at ``x`` by that much; the sums themselves are fp32.

``SegLinear.act8`` and the feed-forward networks of the Wan and H3 blocks use it (``enable_act8``); the ``block_int8``
checkpoint policy keeps whole blocks' inputs in the same code.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from . import ext
from .int8 import Int8Tensor, dequantize_int8_reference, quantize_int8_reference
from .tangent import carries_tangent

ACTS = (None, "gelu_tanh", "swiglu")
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _act(h: torch.Tensor, act):
    """act(h) in h's type; a SwiGLU's h is [value | gate]."""
    if act == "gelu_tanh":
        return F.gelu(h, approximate="tanh")
    if act == "swiglu":
        v, u = h.chunk(2, dim=-1)
        return v * F.silu(u)
    return h


def _gelu_slope(v: torch.Tensor):
    """The derivative of gelu_tanh, 1 or 0 for far values of either sign (the library's is NaN where v v overflows)."""
    s = (v * v).clamp(max=1024.0)  # above, p (1 - p) is 0
    u = (2 / math.pi) ** 0.5 * v * (1 + 0.044715 * s)
    p = torch.sigmoid(2 * u)
    return p + p * (1 - p) * v * (2 * (2 / math.pi) ** 0.5) * (1 + 3 * 0.044715 * s)


def _swiglu_backward(da: torch.Tensor, h: torch.Tensor):
    """da times the derivatives of value * silu(gate), for far values too: da value is not formed, which may overflow where
    the gate's slope is 0."""
    v, u = h.chunk(2, dim=-1)
    p = torch.sigmoid(u)
    return torch.cat([da * (u * p), da * (p + u * p * (1 - p)) * v], dim=-1)


def _kept(x2: torch.Tensor, act):
    """Codes of rows x2, a SwiGLU's halves as rows of their own."""
    rows = x2.reshape(-1, x2.shape[1] // 2) if act == "swiglu" else x2
    return quantize_int8_reference(rows, 32)


class _LinearAct8Reference(torch.autograd.Function):
    """Plain math in fp32, rounded once; CPU."""

    @staticmethod
    def forward(ctx, x, w, bias, act, keep):
        x2 = x.reshape(-1, x.shape[-1])
        y = _act(x2.float(), act) @ w.float().t()
        if bias is not None:
            y = y + bias.float()
        ctx.save_for_backward(w, *(_kept(x2, act) if keep else (None, None)))
        ctx.cfg = (act, x.shape, None if bias is None else bias.dtype)
        return y.to(x.dtype).reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        w, data, scale = ctx.saved_tensors
        act, shape, bias_type = ctx.cfg
        g2 = g.reshape(g.shape[:-1].numel(), w.shape[0]).float()
        dx = dw = db = None
        if data is not None:
            v = dequantize_int8_reference(Int8Tensor(data, scale, 32, (data.shape[0], w.shape[1]))).reshape(g2.shape[0], shape[-1])
        if ctx.needs_input_grad[0]:
            da = g2 @ w.float()
            if act == "gelu_tanh":
                da = da * _gelu_slope(v)
            elif act == "swiglu":
                da = _swiglu_backward(da, v)
            dx = da.to(g.dtype).reshape(shape)
        if ctx.needs_input_grad[1]:
            dw = (g2.t() @ _act(v, act)).to(w.dtype)
        if bias_type is not None and ctx.needs_input_grad[2]:
            db = g2.sum(0).to(bias_type)
        return dx, dw, db, None, None


def linear_act8(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, act: str | None = None) -> torch.Tensor:
    """``act(x) W^T + bias``, differentiable once in ``x``, ``w`` and ``bias``; ``x`` is kept in 8 bits.

    ``x`` [..., F] (bf16 or fp16; on the CPU also fp32; any strides), [..., 2 F] as ``[value | gate]`` for ``act``
    "swiglu" (``value * silu(gate)``); "gelu_tanh" and None are the others.  ``w`` [N, F] of x's type, ``bias`` [N] (fp32,
    bf16 or fp16).  ``act(x)`` is rounded to x's type, as the operand of the product, which the tensor core sums in fp32.
    Where nothing needs a gradient, nothing is kept.  Gradients that depend on a block of 32
    columns of ``x`` with an infinity or a NaN are NaN.
    """
    if act not in ACTS:
        raise ValueError(f"linear_act8: act must be one of {ACTS}, got {act!r}")
    if carries_tangent(x, w, bias):
        raise RuntimeError("linear_act8 has no forward-mode derivative (unpack the dual tensor)")
    if x.is_cuda:  # the checks are the extension's
        return ext().linear_act8(x, w, bias, ACTS.index(act))
    if x.dtype not in _DTYPES:
        raise ValueError(f"linear_act8: x must be bf16, fp16 or fp32, got {x.dtype}")
    if w.dim() != 2 or w.dtype != x.dtype or w.shape[1] < 1:
        raise ValueError(f"linear_act8: w must be a matrix of x's type, got {w.dtype} {tuple(w.shape)}")
    cols = w.shape[1] * (2 if act == "swiglu" else 1)
    if x.dim() < 1 or x.shape[-1] != cols:
        raise ValueError(f"linear_act8: x {tuple(x.shape)} must have {cols} columns for w {tuple(w.shape)}")
    if bias is not None and (tuple(bias.shape) != (w.shape[0],) or bias.dtype not in _DTYPES):
        raise ValueError(f"linear_act8: bias must be bf16, fp16 or fp32 ({w.shape[0]},), got {bias.dtype} {tuple(bias.shape)}")
    if any(t is not None and t.device != x.device for t in (w, bias)):
        raise ValueError("linear_act8: x, w and bias must be on one device")
    keep = torch.is_grad_enabled() and (w.requires_grad or (act is not None and x.requires_grad))
    return _LinearAct8Reference.apply(x, w, bias, act, keep)
