"""A choice from logits with given random numbers on csrc/rr_draw.hip, beside rr_select's keyed generator (rrnco/models/decoding.py:272-298, 311-361)."""
from __future__ import annotations

from . import _lib as L


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=0.0, min_p=0.0, mask=None):
    """One choice for every row of logits [..., V] from the random numbers uniforms [...] -> (index [...] int64, logp [...] float32).

    The row's distribution is softmax(logits / temperature) over the keys that mask (bool, broadcastable to the logits, True = may be drawn) leaves,
    filtered in this order:  top_k keeps the logits that are not under the k-th largest, top_p those of them that have less than top_p of their mass
    strictly above, min_p those whose probability is at least min_p times the largest.  Equal logits stay or go together, so a filter may keep copies
    of its last value.  index is the first key, in index order, at which the running sum of the kept weights exceeds uniform * their sum; logp its
    log-probability among them.  Weights and sums are held in 64 bits (exact to 1e-14 of the largest): the
    same numbers give the same choices as any other such evaluation, unless a border lies within that of a number.  Rows of more than 1 024 keys take top_p's masses in whole steps of 2^-45
    of the largest weight, so that the order of adding does not matter; weights under 2^-46 of it count as nothing there.
    temperature 0 takes the largest logit, the lowest index among equals, with logp 0.  0 (and 1 for top_p, V and more for top_k) switches a filter off.
    temperature, top_k, top_p, min_p: a number, or a tensor with one for each row (out of range: temperatures that are not positive count as 0,
    top_k below 1 and top_p outside (0, 1) as off, min_p above 1 as 1).
    logits float32 / float16 / bfloat16, rows of up to 2^24 keys by any row stride; NaN and -inf are never drawn; a row with nothing left gives
    index 0 and logp -inf.  uniforms float32 in [0, 1) (a number outside counts as the nearer end, NaN as 0).  No gradient."""
    return (L._native or L.native()).sample(logits, uniforms, temperature, top_k, top_p, min_p, mask)
