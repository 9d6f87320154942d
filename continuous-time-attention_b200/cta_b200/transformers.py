"""PDE-refined Transformer models whose refinement runs on the fused kernels.

Drop-in for ``PDETransformerClassifier`` and ``PDETransformerLM`` of the
reference's src/models/transformers.py (:35-142 and :220-320): same
constructor arguments, same submodules and parameter names
(``pde_layers.{layer}.{step}.alpha``, so reference state_dicts load unchanged),
same forward.  The Transformer parts are stock PyTorch modules, exactly as in
the reference; the only change is that the ``pde_steps`` refinement layers
after each Transformer layer run as ONE fused launch forward and one backward
(:124-133, :309-317), with no layout transposes for ``pde_layout="bld"``.

``attention="fused"`` (default ``"torch"``: the stock modules, as above) runs the
layers' attention on ``cta_b200.attention.prompt_attention``: same parameters,
no L x L mask or scores in memory, forward or backward.  Two things differ from
the stock modules: the attention weights themselves are not dropped out (the
layers' other dropouts stay), and a row that sees no valid token (left padding
under the causal mask) gets zeros from its attention, where softmax over nothing
gives NaN.  The language model's ``attention_window=W, attention_sinks=S`` (fused
only) limit each token's attention to the last W tokens and the first S valid ones.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .attention import prompt_attention
from .pde_layers import (
    _DiffusionFamilyLayer,
    _TwoCoefficientLayer,
    create_pde_layer,
    diffusion_pde_stack,
    diffusion_stack_pool,
    pde_stack_forward,
)

__all__ = ["generate_causal_mask", "PDETransformerClassifier", "PDETransformerLM"]


def generate_causal_mask(seq_len: int, device: torch.device) -> torch.Tensor:
    """Additive (seq_len, seq_len) mask, -inf above the diagonal (transformers.py:13-32)."""
    return torch.triu(torch.full((seq_len, seq_len), float("-inf"), device=device, dtype=torch.float32), diagonal=1)


def _refine(x: torch.Tensor, pde_list: nn.ModuleList, layout: str, attention_mask: torch.Tensor) -> torch.Tensor:
    if not all(isinstance(l, _DiffusionFamilyLayer) for l in pde_list):
        grad = torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in pde_list.parameters()))
        kinds = {getattr(l, "KIND", None) for l in pde_list}
        if not grad and len(kinds) == 1 and all(isinstance(l, _TwoCoefficientLayer) for l in pde_list):
            # inference: the whole stack in one launch (per 4 layers); x is [B, L, D] here
            return pde_stack_forward(x, pde_list, attention_mask=attention_mask, layout="bld")
        # training (or mixed kinds): one step per layer, as the reference loops
        x_t = x.transpose(1, 2).contiguous() if layout == "bdl" else x
        for layer in pde_list:
            x_t = layer(x_t, attention_mask=attention_mask)
        return x_t.transpose(1, 2).contiguous() if layout == "bdl" else x_t
    if layout == "bdl":
        x_t = x.transpose(1, 2).contiguous()
        x_t = diffusion_pde_stack(x_t, pde_list, attention_mask=attention_mask)
        return x_t.transpose(1, 2).contiguous()
    return diffusion_pde_stack(x, pde_list, attention_mask=attention_mask)


def _key_words(attention_mask: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """The mask as the fused attention takes it; its words alone do not tell a length from the next."""
    if attention_mask.shape != x.shape[:2]:
        raise ValueError(f"attention_mask must be {tuple(x.shape[:2])}, got {tuple(attention_mask.shape)}")
    return ops.attention_mask(attention_mask)


class _FusedSelfAttention(nn.MultiheadAttention):
    """The layers' attention module (same parameters and names), running fused."""

    reach = {}  # window and sinks, where the model has them

    def forward(self, x, mask_words, causal):  # type: ignore[override]
        B, L, E = x.shape
        qkv = F.linear(x, self.in_proj_weight, self.in_proj_bias).view(B, L, 3, self.num_heads, E // self.num_heads)
        q, k, v = qkv.unbind(2)
        return self.out_proj(prompt_attention(q, k, v, causal=causal, mask_words=mask_words, **self.reach)
                             .reshape(B, L, E))


class _FusedAttentionLayer(nn.TransformerEncoderLayer):
    """A post-norm encoder layer (same parameters and names) whose attention runs fused, as a
    call of its ``self_attn``, so that hooks there see it."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self._fuse()

    def __setstate__(self, state):
        super().__setstate__(state)
        self._fuse()  # saved whole by a version that kept the stock module

    def _fuse(self):
        # the stock module with another forward: the parameters are drawn once, as in a stock layer
        self.self_attn.__class__ = _FusedSelfAttention

    def forward(self, x, mask_words, causal):  # type: ignore[override]
        x = self.norm1(x + self.dropout1(self.self_attn(x, mask_words, causal)))
        return self.norm2(x + self._ff_block(x))


def _encoder_layers(attention, embed_dim, num_heads, hidden_dim, num_layers, dropout):
    if attention not in ("torch", "fused"):
        raise ValueError(f"attention must be 'torch' or 'fused', got {attention!r}")
    cls = _FusedAttentionLayer if attention == "fused" else nn.TransformerEncoderLayer
    return nn.ModuleList(
        [
            cls(d_model=embed_dim, nhead=num_heads, dim_feedforward=hidden_dim, dropout=dropout, batch_first=True)
            for _ in range(num_layers)
        ]
    )


class PDETransformerClassifier(nn.Module):
    """Sequence classifier with PDE refinement after every layer (transformers.py:35-142)."""

    attention = "torch"  # of objects saved whole before there was a choice

    def __init__(
        self,
        vocab_size,
        embed_dim,
        num_heads,
        hidden_dim,
        num_layers,
        num_classes,
        pde_type="diffusion",
        pde_steps=1,
        pde_layout: str = "bld",
        max_length=512,
        dropout=0.1,
        attention: str = "torch",
        **pde_kwargs,
    ):
        super().__init__()
        self.embedding = nn.Embedding(vocab_size, embed_dim)
        self.pos_encoder = nn.Parameter(torch.randn(1, max_length, embed_dim))
        self.dropout = nn.Dropout(dropout)
        self.attention = attention
        self.transformer_layers = _encoder_layers(attention, embed_dim, num_heads, hidden_dim, num_layers, dropout)
        self.pde_layout = pde_layout
        self.pde_layers = nn.ModuleList(
            [
                nn.ModuleList(
                    [create_pde_layer(pde_type, embed_dim, layout=pde_layout, **pde_kwargs) for _ in range(pde_steps)]
                )
                for _ in range(num_layers)
            ]
        )
        self.fc = nn.Linear(embed_dim, num_classes)

    def forward(self, input_ids, attention_mask):
        x = self.embedding(input_ids)
        seq_len = x.size(1)
        x = x + self.pos_encoder[:, :seq_len, :]
        x = self.dropout(x)
        fused = self.attention == "fused"
        if fused:
            words = _key_words(attention_mask, x)
        else:
            padding_mask = attention_mask == 0
        n = len(self.transformer_layers)
        for i, (transformer_layer, pde_list) in enumerate(zip(self.transformer_layers, self.pde_layers)):
            if fused:
                x = transformer_layer(x, words, False)
            else:
                x = transformer_layer(x, src_key_padding_mask=padding_mask)
            if (i == n - 1 and self.pde_layout == "bld" and len(pde_list) > 0 and x.size(1) >= 3
                    and all(isinstance(l, _DiffusionFamilyLayer) and not l.causal for l in pde_list)):
                # the last refinement and the masked mean pool in one pass
                return self.fc(diffusion_stack_pool(x, pde_list, attention_mask))
            x = _refine(x, pde_list, self.pde_layout, attention_mask)
        expanded_mask = attention_mask.unsqueeze(-1).expand(x.size())
        sum_embeddings = torch.sum(x * expanded_mask, dim=1)
        sum_mask = torch.clamp(attention_mask.sum(dim=1, keepdim=True), min=1)
        return self.fc(sum_embeddings / sum_mask)


class PDETransformerLM(nn.Module):
    """Language model with causal PDE refinement after every layer (transformers.py:220-320)."""

    attention = "torch"  # of objects saved whole before there was a choice

    def __init__(
        self,
        vocab_size,
        embed_dim,
        num_heads,
        hidden_dim,
        num_layers,
        pde_type="diffusion",
        pde_steps=1,
        pde_layout: str = "bld",
        max_length=512,
        dropout=0.1,
        attention: str = "torch",
        attention_window: Optional[int] = None,
        attention_sinks: int = 0,
        **pde_kwargs,
    ):
        super().__init__()
        ops._window(attention_window, attention_sinks)
        if attention_window is not None and attention != "fused":
            raise ValueError("attention_window needs attention='fused'")
        self.embedding = nn.Embedding(vocab_size, embed_dim)
        self.pos_encoder = nn.Parameter(torch.randn(1, max_length, embed_dim))
        self.dropout = nn.Dropout(dropout)
        self.attention = attention
        self.transformer_layers = _encoder_layers(attention, embed_dim, num_heads, hidden_dim, num_layers, dropout)
        if attention_window is not None:
            for layer in self.transformer_layers:
                layer.self_attn.reach = {"window": attention_window, "sinks": attention_sinks}
        self.pde_layout = pde_layout
        self.pde_layers = nn.ModuleList(
            [
                nn.ModuleList(
                    [
                        create_pde_layer(pde_type, embed_dim, layout=pde_layout, causal=True, **pde_kwargs)
                        for _ in range(pde_steps)
                    ]
                )
                for _ in range(num_layers)
            ]
        )
        self.fc = nn.Linear(embed_dim, vocab_size)

    def forward(self, input_ids, attention_mask):
        x = self.embedding(input_ids)
        seq_len = x.size(1)
        x = x + self.pos_encoder[:, :seq_len, :]
        x = self.dropout(x)
        fused = self.attention == "fused"
        if fused:
            words = _key_words(attention_mask, x)
        else:
            padding_mask = torch.zeros_like(attention_mask, dtype=torch.float32)
            padding_mask = padding_mask.masked_fill(attention_mask == 0, float("-inf"))
            causal_mask = generate_causal_mask(seq_len, device=x.device)
        for transformer_layer, pde_list in zip(self.transformer_layers, self.pde_layers):
            if fused:
                x = transformer_layer(x, words, True)
            else:
                x = transformer_layer(x, src_mask=causal_mask, src_key_padding_mask=padding_mask)
            x = _refine(x, pde_list, self.pde_layout, attention_mask)
        return self.fc(x)
