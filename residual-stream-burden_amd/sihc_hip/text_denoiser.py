"""A SiHC denoiser conditioned on a text, whose conditioning runs on the HIP operators.

The class-conditional denoiser of `e2e` (behaviour of tongtongliang/residual-stream-burden
sihc/models/sihc/sublayer.py:30-128) with what a prompt needs: its token ids are looked up as states
(`embedding_lookup`, scaled by the square root of their width, no gradient for the padding token),
every block's attention update also attends them (`cross_attention`, each image with its prompt's
own length, 0 for the unconditional half of classifier-free guidance), and the carrier passes a
group norm with SiLU (`group_norm_act`) before the head. Routing and the other bodies are those
of `e2e`. The reference has no text conditioning.

    model = TextSiHCDenoiser(hidden=1152, heads=16, vocab=32768).to("cuda", torch.bfloat16)
    out = model(images, t, labels, tokens, lengths)     # tokens [B, L] int32, lengths [B] int32
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from .conditioning import cross_attention, embedding_lookup, group_norm_act
from .e2e import RMSNorm, SiHCDenoiser


class CrossAttention(nn.Module):
    """Queries from the workspace, keys and values from the states; `kv_heads` of them are shared by
    groups of heads."""

    def __init__(self, dim: int, heads: int, kv_heads: int, state_dim: int):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads
        self.norm = RMSNorm(dim)
        self.q = nn.Linear(dim, dim)
        self.kv = nn.Linear(state_dim, 2 * kv_heads * self.head_dim)
        self.q_norm, self.k_norm = RMSNorm(self.head_dim), RMSNorm(self.head_dim)
        self.proj = nn.Linear(dim, dim)

    def forward(self, z: Tensor, states: Tensor, lengths: Tensor, attend) -> Tensor:
        b, n, c = z.shape
        q = self.q_norm(self.q(self.norm(z)).reshape(b, n, self.heads, self.head_dim))
        k, v = self.kv(states).reshape(b, -1, 2, self.kv_heads, self.head_dim).unbind(2)
        return self.proj(attend(q, self.k_norm(k), v, lengths).reshape(b, n, c))


class GroupNormAct(nn.Module):
    def __init__(self, dim: int, groups: int, eps: float = 1e-6):
        super().__init__()
        self.weight, self.bias = nn.Parameter(torch.ones(dim)), nn.Parameter(torch.zeros(dim))
        self.groups, self.eps, self.norm = groups, eps, group_norm_act

    def forward(self, x: Tensor) -> Tensor:
        return self.norm(x.contiguous(), self.weight, self.bias, self.groups, self.eps, "silu")


class TextSiHCDenoiser(SiHCDenoiser):
    def __init__(self, hidden: int = 1152, heads: int = 16, vocab: int = 32768, state_dim: int = 768,
                 kv_heads: Optional[int] = None, padding_idx: int = 0, groups: int = 32, max_tokens: int = 256,
                 depth: int = 28, stages: tuple[int, ...] = (8, 12, 8), **kwargs):
        super().__init__(hidden=hidden, heads=heads, depth=depth, stages=stages, **kwargs)
        self.padding_idx, self.state_dim = padding_idx, state_dim
        self.tokens = nn.Parameter(torch.zeros(vocab, state_dim))
        self.positions = nn.Parameter(torch.zeros(max_tokens, state_dim))
        self.state_norm = RMSNorm(state_dim)
        self.cross = nn.ModuleList(CrossAttention(hidden, heads, kv_heads or heads, state_dim) for _ in range(depth))
        self.final_norm = GroupNormAct(hidden, groups)
        # replaceable, as the routing hooks: the operators, their host-side value checks left out
        self.lookup = lambda *a: embedding_lookup(*a, validate=False)
        self.attend = lambda *a: cross_attention(*a, validate=False)

    # The states travel with the workspace, beside the prefix tokens: calls on several threads, and bodies
    # that are computed again in the backward, each have their own.
    def _context(self, y_emb, dtype, text):
        return super()._context(y_emb, dtype, text), text

    def _update(self, block, part, z, mod, context, index):
        prefix, text = context
        dz, prefix = super()._update(block, part, z, mod, prefix, index)
        if part == 0 and text is not None:
            dz = dz + mod[2].unsqueeze(1) * self.cross[index](z, *text, self.attend)
        return dz, (prefix, text)

    def forward(self, x: Tensor, t: Tensor, y: Tensor, tokens: Optional[Tensor] = None,
                lengths: Optional[Tensor] = None) -> Tensor:
        """tokens [B, L] (int32 or int64), lengths [B] int32 (None: all L); no tokens: labels alone."""
        if tokens is None:
            return self._denoise(x, t, y)
        if tokens.shape[1] > self.positions.shape[0]:
            raise ValueError(f"at most {self.positions.shape[0]} tokens, got {tokens.shape[1]}")
        states = self.lookup(self.tokens, tokens, math.sqrt(self.state_dim), self.padding_idx)
        states = self.state_norm(states + self.positions[:tokens.shape[1]])
        return self._denoise(x, t, y, (states, lengths))


__all__ = ["TextSiHCDenoiser"]
