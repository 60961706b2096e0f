"""A decoder's cross attention at any width: modules on ops.cross_attention and ops.add_rms_norm, beside the policies' own 128-wide fused decoders
(models/decoder.py, baselines/matnet.py).  Parameter names are those of the reference's MultiHeadCrossAttention (`Wq`, `Wkv`, `out_proj`:
rrnco/baselines/MatNet/encoder.py:95-116) and of its RMSNorm (`weight`: rrnco/models/nn/attn_freenet.py:13-26)."""
from __future__ import annotations

import torch
import torch.nn as nn

from ..ops import add_rms_norm, cross_attention


class CrossAttention(nn.Module):
    """Queries [B, Lq, embed_dim] attend to an encoder's states [B, Lk, kv_dim]: out_proj(attention(Wq x, Wkv states)).

    num_kv_heads < num_heads shares each key head among a group of query heads.  `precompute` gives the keys and values of the states once,
    for the many steps of a decoder; forward takes either.  The attention runs in the type of the keys (under torch.autocast, or with keys and values made
    in another precision than the queries')."""

    def __init__(self, embed_dim: int, num_heads: int, num_kv_heads: int | None = None, kv_dim: int | None = None, bias: bool = False):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if num_heads < 1 or num_kv_heads < 1 or embed_dim % num_heads or num_heads % num_kv_heads or (embed_dim // num_heads) % 8 or embed_dim // num_heads > 128:
            raise ValueError("CrossAttention: heads of a multiple of 8 up to 128 columns, num_heads a multiple of num_kv_heads")
        self.embed_dim, self.num_heads, self.num_kv_heads, self.head_dim = embed_dim, num_heads, num_kv_heads, embed_dim // num_heads
        self.Wq = nn.Linear(embed_dim, embed_dim, bias=bias)
        self.Wkv = nn.Linear(embed_dim if kv_dim is None else kv_dim, 2 * num_kv_heads * self.head_dim, bias=bias)
        self.out_proj = nn.Linear(embed_dim, embed_dim, bias=bias)

    def precompute(self, states):
        """-> (keys, values) [B, Lk, num_kv_heads, head_dim], slices of one projection."""
        return self.Wkv(states).unflatten(-1, (2, self.num_kv_heads, self.head_dim)).unbind(2)

    def forward(self, x, states=None, mask=None, kv_lens=None, cache=None):
        """mask: bool [B, Lq, Lk] or [B, 1, Lq, Lk] / [B, H, Lq, Lk], True where a state may be seen; kv_lens [B]; cache: what `precompute` gave."""
        if (states is None) == (cache is None):
            raise ValueError("CrossAttention: the states or their precomputed keys and values")
        k, v = self.precompute(states) if cache is None else cache
        if mask is not None and mask.dim() == 3:
            mask = mask.unsqueeze(1)
        q = self.Wq(x).unflatten(-1, (self.num_heads, self.head_dim))
        return self.out_proj(cross_attention(q.to(k.dtype), k, v, mask=mask, kv_lens=kv_lens).flatten(2).to(q.dtype))


class CrossAttentionLayer(nn.Module):
    """Norm before, residual after, the next layer's norm joined with the addition: (y, h) -> attention(y) -> h' = h + attention, y' = RMSNorm(h').

    forward takes the normed stream y and the residual stream h (`start` makes both from a first x) and returns the next ones, so that a stack of
    layers reads and writes the stream once a layer.  The streams keep their type, also where the attention runs in another (torch.autocast)."""

    def __init__(self, embed_dim: int, num_heads: int, num_kv_heads: int | None = None, kv_dim: int | None = None, bias: bool = False, eps: float = 1e-5):
        super().__init__()
        self.attention = CrossAttention(embed_dim, num_heads, num_kv_heads, kv_dim, bias)
        self.norm = nn.Module()
        self.norm.weight = nn.Parameter(torch.ones(embed_dim))
        self.eps = eps

    @staticmethod
    def start(x, weight=None, eps: float = 1e-5):
        return add_rms_norm(x, None, weight, eps)

    def forward(self, y, h, states=None, mask=None, kv_lens=None, cache=None):
        return add_rms_norm(self.attention(y, states, mask, kv_lens, cache).to(h.dtype), h, self.norm.weight, self.eps)
