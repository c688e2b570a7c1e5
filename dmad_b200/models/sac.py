"""Activation checkpointing policies for transformer blocks.

Parity: train/wan/rcm/utils/selective_activation_checkpoint.py:26-74.

* ``"block_wise"``: the whole block is recomputed in the backward; only its inputs are kept.
* ``"mm_only"``: the outputs of the matrix products are kept from the forward and everything else
  (normalisation, modulation, RoPE, activations, gates) is recomputed.  The kept ops are the
  library GEMMs (``aten.mm`` / ``addmm`` / ``bmm``), this package's tcgen05 flash-attention forward
  (``dmad::flash_attn_fwd``, output and LSE) and LoRA-fused linear (``dmad::lora_linear_fwd``).  The
  fused context-parallel attention (exchange + attention in one autograd function) is recomputed whole,
  as the reference recomputes its all-to-all.
* ``"block_int8"`` (not in the reference): as ``"block_wise"``, with the block's first input, its hidden states, kept in
  8-bit integers of which 32 columns share a power of two (``ops.quantize_int8(x, 32)``): half the memory, and gradients at
  the decoded input.  The forward pass is not changed.

Layers that keep their inputs in 8 bits (``SegLinear.act8``) run as plain ones inside of a block under any of the policies, in
its forward pass and in its recomputation: what they would keep is thrown away, and ``mm_only`` keeps library products only.
"""
from __future__ import annotations

import functools
import threading

import torch
from torch.utils.checkpoint import CheckpointPolicy, checkpoint, create_selective_checkpoint_contexts

from .. import ops

POLICIES = ("block_wise", "mm_only", "block_int8")


@functools.lru_cache(maxsize=1)
def _saved_ops():
    from ..ops import attention as _attn  # noqa: F401  (registers dmad::flash_attn_fwd)
    from ..ops import linear as _lin  # noqa: F401  (registers dmad::lora_linear_fwd)

    aten = torch.ops.aten
    return frozenset({aten.mm.default, aten.addmm.default, aten.bmm.default, aten.baddbmm.default,
                      torch.ops.dmad.flash_attn_fwd.default, torch.ops.dmad.lora_linear_fwd.default})


def _mm_only_policy(ctx, op, *args, **kwargs):
    return CheckpointPolicy.MUST_SAVE if op in _saved_ops() else CheckpointPolicy.PREFER_RECOMPUTE


def mm_only_context():
    return create_selective_checkpoint_contexts(_mm_only_policy)


class _Held:
    """A tensor that is there until ``code`` and decoded from 8 bits after it."""

    def __init__(self, x):
        self.x, self.codes, self.dtype, self.grad = x, None, x.dtype, x.requires_grad

    def code(self):
        self.codes, self.x = ops.quantize_int8(self.x.detach(), 32), None

    def get(self):
        return self.x if self.codes is None else ops.dequantize_int8(self.codes, self.dtype).requires_grad_(self.grad)


def _checkpoint_int8(fn, x, *args):
    held = _Held(x)
    # the recomputation only has to give the tensors that the block saved: its input needs no history
    y = checkpoint(lambda *rest: fn(held.get(), *rest), *args, use_reentrant=False)
    if torch.is_grad_enabled():
        held.code()
    return y


_inside = threading.local()  # (a backward pass recomputes in threads of its own)


def inside_checkpoint() -> bool:
    """Whether the calling thread is in a block that ``checkpoint_block`` runs, the first time or again."""
    return getattr(_inside, "depth", 0) > 0


def _marked(fn):
    def run(*args):
        _inside.depth = getattr(_inside, "depth", 0) + 1
        try:
            return fn(*args)
        finally:  # a recomputation ends in an exception, once it has what the backward pass wants
            _inside.depth -= 1

    return run


def checkpoint_block(fn, *args, policy: str = "block_wise"):
    """``fn(*args)`` under activation checkpointing with the given policy (non-reentrant)."""
    fn = _marked(fn)
    if policy == "mm_only":
        return checkpoint(fn, *args, use_reentrant=False, context_fn=mm_only_context)
    if policy == "block_int8":
        return _checkpoint_int8(fn, *args)
    if policy != "block_wise":
        raise ValueError(f"unknown checkpoint policy {policy!r} (one of {POLICIES})")
    return checkpoint(fn, *args, use_reentrant=False)
