"""Per-head RMSNorm of queries and keys with the position rotation in the same pass.

    out = Rot(x / sqrt(mean(x^2) + eps) * w)        for every row and head

The norm of the H3 attention (``norm_q`` / ``norm_k`` over the head size) and of text decoders with grouped
heads; the Wan blocks' norm over the whole hidden size is ``ops.qk_norm_rope``.  One kernel reads the q and k
columns of a fused projection where they are and writes the rotated heads, rounding once; the separate
``rms_norm`` and ``rope`` calls read and write them twice and round in between.
"""
from __future__ import annotations

import torch

from . import ext
from .tangent import carries_tangent

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _rotate(y, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        r = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([r, y[..., rot:]], dim=-1)


def qk_head_norm_rope_reference(q, k, wq=None, wk=None, cos=None, sin=None, positions=None, eps=1e-6,
                                interleaved=True):
    """Plain differentiable math in fp32 (fp64 inputs: in fp64), rounded once."""
    outs = []
    if cos is not None:
        R, T = q.shape[0], cos.shape[0]
        at = positions.long() if positions is not None else torch.arange(R, device=q.device) % T
        bad = (at < 0) | (at >= T)
        nan = torch.where(bad, float("nan"), 0.0)[:, None]
        at = at.clamp(0, T - 1)
    for x, w in ((q, wq), (k, wk)):
        ct = torch.float64 if x.dtype == torch.float64 else torch.float32
        xf = x.to(ct)
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.to(ct)
        if cos is not None:
            y = _rotate(y, (cos[at] + nan).to(ct), (sin[at] + nan).to(ct), interleaved)
        outs.append(y.to(x.dtype))
    return tuple(outs)


def _check(q, k, wq, wk, cos, sin, positions):
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"qk_head_norm_rope: q and k must be [R, heads, hd] with one R and hd, got {tuple(q.shape)} "
                         f"and {tuple(k.shape)}")
    if q.dtype != k.dtype or q.dtype not in _DTYPES:
        raise ValueError(f"qk_head_norm_rope: q and k must share bf16, fp16 or fp32, got {q.dtype} and {k.dtype}")
    R, hd = q.shape[0], q.shape[2]
    if hd % 8 or not 8 <= hd <= 256 or q.shape[1] < 1 or k.shape[1] < 1:
        raise ValueError(f"qk_head_norm_rope: the head size must be a multiple of 8 up to 256 and q and k have heads, "
                         f"got {tuple(q.shape)} and {tuple(k.shape)}")
    for name, w in (("wq", wq), ("wk", wk)):
        if w is not None and (tuple(w.shape) != (hd,) or w.dtype not in _DTYPES):
            raise ValueError(f"qk_head_norm_rope: {name} must be bf16, fp16 or fp32 ({hd},), got {w.dtype} {tuple(w.shape)}")
    if (cos is None) != (sin is None) or (positions is not None and cos is None):
        raise ValueError("qk_head_norm_rope: cos and sin come together, and positions with them")
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1 or 2 * cos.shape[1] > hd:
            raise ValueError(f"qk_head_norm_rope: cos and sin must be [T, rot / 2] with T >= 1 and rot <= {hd}, got "
                             f"{tuple(cos.shape)} and {tuple(sin.shape)}")
        if not (cos.is_floating_point() and sin.is_floating_point()) or cos.requires_grad or sin.requires_grad:
            raise ValueError("qk_head_norm_rope: cos and sin are constant floating-point tables (no gradient)")
    if positions is not None and (tuple(positions.shape) != (R,) or positions.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"qk_head_norm_rope: positions must be int32 or int64 ({R},), got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    if any(t is not None and t.device != q.device for t in (k, wq, wk, cos, sin, positions)):
        raise ValueError("qk_head_norm_rope: all tensors must be on one device")


def qk_head_norm_rope(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor | None = None, wk: torch.Tensor | None = None,
                      cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                      positions: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = True):
    """``(Rot(rmsnorm(q) * wq), Rot(rmsnorm(k) * wk))`` per head, contiguous; differentiable once in q, k, wq and wk
    (reverse mode; dual tensors are refused on CUDA).

    ``q`` [R, Hq, hd], ``k`` [R, Hk, hd] (bf16, fp16 or fp32; any row and head strides, e.g. column ranges of one
    fused projection; hd a multiple of 8 up to 256; Hq and Hk independent).  ``wq`` / ``wk`` [hd] (None: ones).
    ``cos`` / ``sin`` [T, rot / 2] turn the first ``rot`` elements of each head, as pairs (2i, 2i + 1) when
    ``interleaved``, else (i, i + rot / 2); row r uses table row ``positions[r]``, or r % T without ``positions``.  A
    position outside [0, T) turns its row's rotated elements to NaN and, on CUDA, records status 6 for
    ``check_device_status``.
    """
    if not q.is_cuda:
        _check(q, k, wq, wk, cos, sin, positions)
        return qk_head_norm_rope_reference(q, k, wq, wk, cos, sin, positions, eps, interleaved)
    # on CUDA the same checks are the extension's
    if carries_tangent(q, k, wq, wk, cos, sin):
        raise RuntimeError("qk_head_norm_rope: the CUDA kernels have no forward-mode derivative (unpack the dual tensor)")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, wq, wk)):
        return ext().head_norm_rope(q, k, wq, wk, cos, sin, positions, eps, interleaved)
    return ext().head_norm_rope_fwd(q, k, wq, wk, cos, sin, positions, eps, interleaved)
