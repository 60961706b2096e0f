"""Residual addition + root-mean-square norm (RMSNorm rrnco/models/nn/attn_freenet.py:13-26 behind a skip connection) on csrc/rr_norm.hip,
for any width up to 16 384 in float32, float16 or bfloat16, with its gradient, and a form that hands the result on in 8 bits."""
from __future__ import annotations

import torch

from . import _lib as L

MAX_WIDTH = 16384


def _rows(t, E):
    """[..., E] -> [rows, E] with unit column stride; a view where the strides allow it."""
    t = t.reshape(-1, E)
    return t if t.stride(1) == 1 or E == 1 else t.contiguous()


def _checked(x, residual, weight, eps):
    if x.dtype not in L.DTYPE_CODE:
        raise TypeError(f"add_rms_norm: float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"add_rms_norm: a last axis of 1 .. {MAX_WIDTH}, got shape {tuple(x.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("add_rms_norm: the residual has the input's shape, type and device")
    if weight is not None and (weight.shape != x.shape[-1:] or weight.dtype not in (x.dtype, torch.float32) or weight.device != x.device):
        raise ValueError("add_rms_norm: the weight is [width], of the input's type or float32, on its device")
    if not eps >= 0:
        raise ValueError(f"add_rms_norm: eps >= 0, got {eps}")
    L.require_gpu(x)


def _forward(x, residual, weight, eps, want_rstd):
    E = x.shape[-1]
    x2, r2 = _rows(x, E), None if residual is None else _rows(residual, E)
    w = None if weight is None else weight.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty_like(y) if residual is not None else None
    rows = x2.shape[0]
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_rstd else None
    if rows:
        with L.on_device(x) as st:
            L.check(L.lib().rr_add_rms_norm(L.DTYPE_CODE[x.dtype], x2.data_ptr(), x2.stride(0), None if r2 is None else r2.data_ptr(),
                                            0 if r2 is None else r2.stride(0), None if w is None else w.data_ptr(),
                                            int(w is not None and w.dtype == torch.float32), y.data_ptr(), None if h is None else h.data_ptr(),
                                            None if rstd is None else rstd.data_ptr(), None, None, rows, E, eps, st), "rr_add_rms_norm")
    return y, (x if h is None else h), rstd


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _forward(x, residual, weight, eps, True)
        ctx.save_for_backward(x, residual, weight, rstd)
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        x, residual, weight, rstd = ctx.saved_tensors
        nx, nr, nw = ctx.needs_input_grad[:3]
        E, rows, dev = x.shape[-1], rstd.shape[0], x.device
        if dy is None:                                              # only the sum was used
            return dh if nx else None, dh if nr else None, torch.zeros_like(weight) if nw else None, None
        dx, dw = torch.empty(x.shape, dtype=x.dtype, device=dev), torch.empty(weight.shape, dtype=weight.dtype, device=dev) if nw else None
        if rows == 0:
            return dx if nx else None, dx if nr else None, None if dw is None else dw.zero_(), None
        x2, r2, dy2 = _rows(x, E), None if residual is None else _rows(residual, E), _rows(dy, E)
        dh2, w = None if dh is None else _rows(dh, E), None if weight is None else weight.contiguous()
        lib = L.lib()
        parts = lib.rr_add_rms_norm_parts(rows, E)
        ws = torch.empty(parts * E, dtype=torch.float32, device=dev) if nw else None
        with L.on_device(x) as st:
            L.check(lib.rr_add_rms_norm_bwd(L.DTYPE_CODE[x.dtype], x2.data_ptr(), x2.stride(0), None if r2 is None else r2.data_ptr(),
                                            0 if r2 is None else r2.stride(0), None if w is None else w.data_ptr(),
                                            int(w is not None and w.dtype == torch.float32), dy2.data_ptr(), dy2.stride(0),
                                            None if dh2 is None else dh2.data_ptr(), 0 if dh2 is None else dh2.stride(0), rstd.data_ptr(), dx.data_ptr(),
                                            None if dw is None else dw.data_ptr(), None if ws is None else ws.data_ptr(), parts, rows, E, st),
                    "rr_add_rms_norm_bwd")
        return dx if nx else None, dx if nr else None, dw, None


def add_rms_norm(x, residual=None, weight=None, eps: float = 1e-5):
    """h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight  over the last axis -> (y, h), both of x's type.

    x, residual [..., E], E up to 16 384, float32 / float16 / bfloat16 with any strides (a last axis that is not contiguous is copied);
    weight [E] in x's type or float32, None for ones.  The norm is taken of the sum before it is rounded to h.  residual=None: h is x.
    Differentiable once in x, residual and weight; the sums of the backward have a fixed order."""
    _checked(x, residual, weight, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad) or (weight is not None and weight.requires_grad)):
        out = _AddRMSNorm.apply(x, residual, weight, float(eps))
        return out if residual is not None else (out, x)
    y, h, _ = _forward(x, residual, weight, float(eps), False)
    return y, h


def add_rms_norm_fp8(x, residual=None, weight=None, eps: float = 1e-5):
    """add_rms_norm with y handed on in 8 bits: -> (q, scale, h), y ~ q * scale of its group.

    q [..., E] float8_e4m3fn; scale [..., ceil(E / 128)] float32, one for every 128 columns (the last group may be shorter): the group's
    largest |y| / 448, or 1 where the group is all zeros.  Inference only: refused where a gradient would be asked for."""
    _checked(x, residual, weight, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad) or (weight is not None and weight.requires_grad)):
        raise RuntimeError("add_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    E = x.shape[-1]
    x2, r2 = _rows(x, E), None if residual is None else _rows(residual, E)
    w = None if weight is None else weight.contiguous()
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(*x.shape[:-1], (E + 127) // 128, dtype=torch.float32, device=x.device)
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x2.shape[0]:
        with L.on_device(x) as st:
            L.check(L.lib().rr_add_rms_norm(L.DTYPE_CODE[x.dtype], x2.data_ptr(), x2.stride(0), None if r2 is None else r2.data_ptr(),
                                            0 if r2 is None else r2.stride(0), None if w is None else w.data_ptr(),
                                            int(w is not None and w.dtype == torch.float32), None, None if h is None else h.data_ptr(), None,
                                            q.data_ptr(), scale.data_ptr(), x2.shape[0], E, float(eps), st), "rr_add_rms_norm")
    return q, scale, (x if h is None else h)
