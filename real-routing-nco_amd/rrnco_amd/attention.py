"""Cross attention of a decoder's queries to an encoder's states on csrc/rr_xattn.hip, beside the policy's own fused glimpse (rrnco/models/decoder.py:281-323,
128 wide, 8 heads, float32): any numbers of queries, keys and heads, float32 / float16 / bfloat16, masks, ragged lengths, gradients."""
from __future__ import annotations

from . import _lib as L


def cross_attention(query, key, value, mask=None, kv_lens=None, scale=None, return_lse: bool = False):
    """softmax(scale * query key^T over the keys that may be seen) value -> [B, Lq, H, D] in the inputs' type.

    query [B, Lq, H, D]; key, value [B, Lk, Hk, D], H a multiple of Hk (query head h reads key head h // (H / Hk)), D a multiple of 8 up to 128;
    float32, float16 or bfloat16, any strides: slices of one cache row and start-major views are read in place, only tensors whose heads do not
    lie on 16 bytes are copied.
    mask: bool, broadcastable [B, H, Lq, Lk], True where a key may be seen (an environment's action mask [S * B, N] is `mask.view(S, B, N).transpose(0, 1)[:, None]`).
    kv_lens [B] int32 / int64: only the first kv_lens[b] keys exist (values outside 0 .. Lk count as the nearer end); what lies behind is never read.
    scale: > 0, D ** -0.5 if None.
    A query that sees no key gives zeros and takes part in no gradient.  A key that a query may not see never shows in its result, whatever it holds
    (non-finite values too); scores, softmax and sums are in float32, the weights are rounded to the inputs' type before the product with the values.
  In the backward the weights are rounded to it before their product too, the scores' gradients to two values of it (in float16 all times powers of two, so that small ones on long states
  keep their bits and large ones stay finite), and the sum of out * its gradient is taken of the stored out, except in 16 bits on at most 64 keys.
    return_lse: also the logarithm of the sum of exponentials [B, H, Lq] float32 (-inf where nothing is seen; no gradient through it).
    Differentiable once in query, key and value (backward; forward-mode tangents are refused); no atomics, the same inputs give the same bits."""
    out, lse = (L._native or L.native()).cross_attention(query, key, value, mask, kv_lens, scale, return_lse)
    return (out, lse) if return_lse else out
