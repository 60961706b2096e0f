"""Residual addition + root-mean-square norm (RMSNorm rrnco/models/nn/attn_freenet.py:13-26 behind a skip connection) on csrc/rr_norm.hip,
for any width up to 16 384 in float32, float16 or bfloat16, with its gradient, and a form that hands the result on in 8 bits."""
from __future__ import annotations

from . import _lib as L


def add_rms_norm(x, residual=None, weight=None, eps: float = 1e-5):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight  over the last axis -> (y, h), both of x's type.

    x, residual [..., E], E up to 16 384, float32 / float16 / bfloat16 with any strides (a last axis that is not contiguous is copied);
    weight [E] in x's type or float32, None for ones.  The norm is taken of the sum before it is rounded to h.  residual=None: h is x.
    eps >= 0; with eps = 0 a row whose root mean square is 2^-128 or less has no reciprocal in float32, and gives inf or NaN, as a row of zeros does.
    Differentiable once in x, residual and weight (backward; forward-mode tangents are refused); the sums of the backward have a fixed order."""
    return (L._native or L.native()).add_rms_norm(x, residual, weight, eps)


def add_rms_norm_fp8(x, residual=None, weight=None, eps: float = 1e-5):
    """add_rms_norm with y handed on in 8 bits: -> (q, scale, h), y ~ q * scale of its group.

    q [..., E] float8_e4m3fn; scale [..., ceil(E / 128)] float32, one for every 128 columns (the last group may be shorter): the group's
    largest |y| / 448 (2^-126 at the least), or 1 where the group is all zeros.  Inference only: refused where a gradient would be asked for."""
    return (L._native or L.native()).add_rms_norm_fp8(x, residual, weight, eps)
