"""Spatial self-attention layer (reference: modeling/attention.py:35-84)."""
from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from dm_hip import ops
from modeling.layers import GroupNorm, Linear


class Attention2D(nn.Module):
    """Attention over the pixels of a feature map, and two extensions that the reference does not have (both off by default,
    which leaves parameters and results as they are):

    top_blocks: on maps of more than 64 * top_blocks pixels every pixel attends only to the `top_blocks` runs of 64 neighbouring
        positions whose mean key it scores highest (ops.sparse_attention), instead of to all.
    n_context: the pixels also attend to context tokens of this width (a multiple of 64), forward's `context` [B, T, n_context],
        of which the first context_len[b] are valid; their keys and values come from a projection of their own
        (`context_proj`) and stand behind the pixels' in the same softmax."""

    def __init__(self, n_dim: int, n_heads: Optional[int] = None, n_dim_head: Optional[int] = None,
                 norm_groups: int = 32, dropout: float = 0.0, top_blocks: Optional[int] = None,
                 n_context: Optional[int] = None):
        super().__init__()
        assert n_dim_head is not None or n_heads is not None
        if n_dim_head is None:
            assert n_dim % n_heads == 0
            n_dim_head = n_dim // n_heads
        elif n_heads is None:
            assert n_dim % n_dim_head == 0
            n_heads = n_dim // n_dim_head
        self.n_heads = n_heads
        self.n_dim_head = n_dim_head
        self.n_dim_inner = n_heads * n_dim_head
        self._dropout = float(dropout)
        self.register_buffer("dropout_p", torch.tensor(dropout))

        self.norm = GroupNorm(norm_groups, n_dim)
        self.qkv_proj = Linear(n_dim, 3 * self.n_dim_inner)
        self.out_proj = Linear(self.n_dim_inner, n_dim)
        if n_context is not None:
            if n_context <= 0 or n_context % 64:
                raise ValueError(f"Attention2D: the context's width must be a multiple of 64, not {n_context}")
            if dropout > 0:
                raise ValueError("Attention2D: no dropout on the attention weights with a context")
        self.context_proj = Linear(n_context, 2 * self.n_dim_inner) if n_context is not None else None
        self.top_blocks = None
        self.attend_to(top_blocks)

    def attend_to(self, top_blocks: Optional[int]):
        """Every pixel attends to `top_blocks` blocks of 64 positions (1 to 64); None: to all."""
        if top_blocks is not None:
            if not 1 <= top_blocks <= 64:
                raise ValueError(f"Attention2D: 1 to 64 blocks, not {top_blocks}")
            if self._dropout > 0:
                raise ValueError("Attention2D: no dropout on the attention weights of chosen blocks")
        self.top_blocks = top_blocks

    def _attention_with_context(self, tokens, context, context_len):
        """q of the pixels over the keys of pixels and context tokens; without top_blocks all blocks are attended to."""
        B, L, _ = tokens.shape
        T = context.shape[1]
        heads = (B, T, 2, self.n_heads, self.n_dim_head)
        kv = self.context_proj(context.to(torch.bfloat16).transpose(1, 2).unsqueeze(2))     # [B, 2*inner, 1, T] pixel-major
        ck, cv = kv.permute(0, 2, 3, 1).reshape(heads).unbind(2)
        q, k, v = tokens.view(B, L, 3, self.n_heads, self.n_dim_head).unbind(2)
        k, v = torch.cat([k, ck], 1), torch.cat([v, cv], 1)
        k_len = None if context_len is None else (context_len.clamp(0, T) + L).to(torch.int32)
        n = -(-(L + T) // ops.BLOCK)
        if self.top_blocks is None and n > 64:
            raise RuntimeError(f"Attention2D: {L} pixels and {T} context tokens are more than 64 blocks of {ops.BLOCK}: choose top_blocks")
        top = min(n, self.top_blocks or n)
        blocks = ops.block_select(q, ops.block_keys(k, k_len), top, k_len)
        return ops.block_attention(q, k, v, blocks, k_len=k_len).reshape(B, L, self.n_dim_inner)

    def _attention_with_dropout(self, tokens):
        """Attention with dropout on the attention weights (modeling/attention.py:75-78, 92-96: softmax, dropout,
        times v). No configuration of the reference trains with it, so it is not a kernel of the library: the weights
        are materialised ([B, heads, L, L], fp32 softmax) and the two products are library batched GEMMs. The mask
        comes from torch's generator - the reference's comes from inside its fused attention kernel, a stream no
        other implementation can reproduce; only the distribution is the same."""
        B, L, _ = tokens.shape
        q, k, v = tokens.view(B, L, 3, self.n_heads, self.n_dim_head).permute(2, 0, 3, 1, 4)   # each [B, heads, L, d]
        w = torch.softmax(torch.matmul(q, k.transpose(-1, -2)).float() * self.n_dim_head ** -0.5, dim=-1)
        w = F.dropout(w, p=self._dropout, training=True).to(tokens.dtype)
        return torch.matmul(w, v).transpose(1, 2).reshape(B, L, self.n_dim_inner)

    def forward(self, x: torch.Tensor, context: Optional[torch.Tensor] = None, context_len: Optional[torch.Tensor] = None):
        if context is not None:
            if self.context_proj is None:
                raise RuntimeError("Attention2D: a context needs n_context")
            if context.dim() != 3 or context.shape[0] != x.shape[0] or context.shape[2] != self.context_proj.in_features:
                raise RuntimeError(f"Attention2D: the context must be [{x.shape[0]}, tokens, {self.context_proj.in_features}], "
                                   f"got {tuple(context.shape)}")
        B, C, H, W = x.shape
        L = H * W
        x = ops.as_nhwc(x)
        # the residual branch reads x through the norm's fork, so that its gradient is added inside the norm's backward
        # kernel instead of by a separate accumulation pass
        h, x, _ = self.norm(x, fork=True)                 # [B, C, H, W] pixel-major == tokens [B, L, C]
        qkv = self.qkv_proj(h)                            # [B, 3*inner, H, W] == tokens [B, L, (3, heads, d)]
        tokens = qkv.permute(0, 2, 3, 1).reshape(B, L, 3 * self.n_dim_inner)
        if self.training and self._dropout > 0:
            att = self._attention_with_dropout(tokens)
        elif context is not None and context.shape[1] > 0:
            att = self._attention_with_context(tokens, context, context_len)
        elif self.top_blocks is not None and L > ops.BLOCK * self.top_blocks:
            att = ops.sparse_attention(tokens, self.n_heads, self.n_dim_head, self.top_blocks)
        else:
            att = ops.attention(tokens, self.n_heads, self.n_dim_head)  # [B, L, inner]
        att = att.view(B, H, W, self.n_dim_inner).permute(0, 3, 1, 2)   # pixel-major view, no copy
        return self.out_proj(att, res=x)
