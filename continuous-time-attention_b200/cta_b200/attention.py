"""Softmax attention of prompts with its gradients.

``prompt_attention`` is the attention of the PDE Transformers' layers
(``cta_b200.transformers``, ``attention="fused"``) and of packed prefill
batches, whose output the mixer (``cta_b200.serving_vllm``) refines: padded
[B, L, heads, dim] with a key mask, or packed [T, heads, dim] with offsets;
causal or not; grouped key/value heads; float32, bfloat16, float16.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad

from . import ops

__all__ = ["prompt_attention"]


class _PromptAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask_words, cu_seqlens, causal, scale):
        q, k, v, cu, sizes, code, scale = ops._attention_inputs(q, k, v, cu_seqlens, mask_words, scale)
        out = ops._new(q)
        # what rounding the output loses: delta of rows with few keys needs it
        low = torch.empty_like(out) if code != 0 else None
        lse = ops._attention_forward(q, k, v, out, 0 if low is None else low.data_ptr(), cu, mask_words, causal, scale,
                                     sizes, code, True, True)
        ctx.save_for_backward(q, k, v, out, low, lse, mask_words, cu)
        ctx.plan = (causal, scale, sizes, code)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        # the forward has checked what was saved
        q, k, v, out, low, lse, mask_words, cu = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        dq, dk, dv = ops._attention_backward(grad_out, q, k, v, out, 0 if low is None else low.data_ptr(), lse, cu,
                                             mask_words, *ctx.plan, need_q, need_k or need_v)
        return dq, dk if need_k else None, dv if need_v else None, None, None, None, None


def _tangents(*tensors: torch.Tensor) -> bool:
    """Whether one carries a forward-mode tangent: such a call goes through the function, which refuses it.
    Outside of a dual level, a look at its number (unpack_dual takes 0.4 us a tensor)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def prompt_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    causal: bool = False,
    scale: Optional[float] = None,
    key_mask: Optional[torch.Tensor] = None,
    mask_words: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """softmax(scale * q k^T) v over the keys each row sees, differentiable in q, k, v.

    Padded: q [B, L, heads, dim], k and v [B, L, kv_heads, dim]; ``key_mask``
    [B, L] (any mask dtype, non-zero = valid) hides padding, or ``mask_words``,
    its form from ``ops.attention_mask``, made once for several layers.  Packed:
    [T, heads, dim] with ``cu_seqlens`` (device int32, sequences + 1 offsets from 0, not decreasing).  ``causal``:
    row i sees keys j <= i of its sequence.  ``scale`` defaults to dim**-0.5.

    A row that sees no key is zero and has no gradient, as are packed rows
    behind the last sequence.  Masked keys and such rows may hold anything,
    infinities and NaN included; a NaN or infinity in the k or v of a valid token may
    also reach earlier rows of its sequence, one in the q or the output gradient of
    a row the gradients of later keys.  Forward-mode differentiation raises."""
    words = mask_words
    if key_mask is not None:
        if words is not None:
            raise ValueError("give key_mask or mask_words, not both")
        if q.dim() != 4 or cu_seqlens is not None or key_mask.shape != q.shape[:2]:
            raise ValueError("key_mask must be (B, L) for padded q, k, v")
        if key_mask.get_device() != q.get_device():
            raise ValueError(f"key_mask on {key_mask.device}, expected {q.device}")
        words = ops.attention_mask(key_mask)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or _tangents(q, k, v):
        return _PromptAttention.apply(q, k, v, words, cu_seqlens, bool(causal), scale)
    return ops.attention_forward(q, k, v, causal=causal, scale=scale, mask_words=words, cu_seqlens=cu_seqlens,
                                 need_lse=False)[0]
