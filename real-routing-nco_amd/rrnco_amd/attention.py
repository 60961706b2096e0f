"""Cross attention of a decoder's queries to an encoder's states on csrc/rr_xattn.hip, beside the policy's own fused glimpse (rrnco/models/decoder.py:281-323,
128 wide, 8 heads, float32): any numbers of queries, keys and heads, float32 / float16 / bfloat16, masks, ragged lengths, gradients."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

MAX_HEAD_DIM = 128


def _placed(t):
    """The kernels read 16 bytes of a head at a time: a unit last stride, the base and every other stride on 16 bytes; anything else is copied."""
    per = 16 // t.element_size()
    sb, sl, sh, sd = t.stride()
    if sd != 1 or (sb | sl | sh) % per or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)      # (contiguous() would hand back a tensor whose base is off the grid)
    return t


def _strides(t):
    return tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()))


def _checked(q, k, v, mask, kv_lens, scale):
    if q.dtype not in L.DTYPE_CODE or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"cross_attention: query, key and value of one type out of float32, float16, bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"cross_attention: query [B, Lq, H, D], key and value [B, Lk, Hk, D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    if D % 8 or not 8 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"cross_attention: a head dim that is a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
    if Hk < 1 or H % Hk:
        raise ValueError(f"cross_attention: the query's heads are a multiple of the key's, got {H} and {Hk}")
    if k.device != q.device or v.device != q.device:
        raise ValueError("cross_attention: query, key and value are on one device")
    if mask is not None:
        if mask.dtype != torch.bool or mask.dim() != 4 or mask.device != q.device:
            raise ValueError("cross_attention: mask is a bool tensor of four axes (batch, head, query, key) on the query's device, True where a key may be seen")
        if any(n not in (1, m) for n, m in zip(mask.shape, (B, H, Lq, Lk))):
            raise ValueError(f"cross_attention: mask {tuple(mask.shape)} does not broadcast to {(B, H, Lq, Lk)}")
    if kv_lens is not None and (kv_lens.dtype not in (torch.int32, torch.int64) or kv_lens.shape != (B,) or kv_lens.device != q.device):
        raise ValueError("cross_attention: kv_lens is [B], int32 or int64, on the query's device")
    if not 0.0 < scale < 3e38:
        raise ValueError(f"cross_attention: scale > 0, got {scale}")
    L.require_gpu(q)


def _io(q, k, v, mask, kv_lens, scale):
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    io = L.XAttnIO()
    io.q, io.k, io.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    io.q_stride, io.k_stride, io.v_stride = _strides(q), _strides(k), _strides(v)
    if mask is not None:
        if mask.shape[3] != Lk or (Lk > 1 and mask.stride(3) != 1):
            mask = mask.expand(*mask.shape[:3], Lk).contiguous()
        io.mask, io.mask_stride = mask.data_ptr(), _strides(mask)
    if kv_lens is not None:
        kv_lens = kv_lens.contiguous()
        io.kv_lens, io.lens_int64 = kv_lens.data_ptr(), int(kv_lens.dtype == torch.int64)
    io.dtype, io.B, io.Lq, io.Lk, io.Hk, io.G, io.D, io.scale = L.DTYPE_CODE[q.dtype], B, Lq, Lk, Hk, H // Hk, D, scale
    return io, (q, k, v, mask, kv_lens)                  # the tensors that the pointers belong to


def _workspace(io, backward, device):
    n = L.lib().rr_cross_attn_workspace(io.B, io.Lq, io.Lk, io.Hk, io.G, io.D, backward)
    if n < 0:
        raise ValueError("cross_attention: more rows, keys or heads than 32-bit counts hold")
    ws = None
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        io.workspace, io.workspace_bytes = ws.data_ptr(), n
    return ws


def _forward(q, k, v, mask, kv_lens, scale, want_lse):
    B, Lq, H, D = q.shape
    out = torch.empty(B, Lq, H, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, Lq, dtype=torch.float32, device=q.device) if want_lse else None
    if out.numel() == 0:
        return out, lse
    if k.numel() == 0:                                   # nothing to see
        return out.zero_(), None if lse is None else lse.fill_(float("-inf"))
    io, keep = _io(_placed(q), _placed(k), _placed(v), mask, kv_lens, scale)
    io.out = out.data_ptr()
    if lse is not None:
        io.lse = lse.data_ptr()
    with L.on_device(q) as st:
        ws = _workspace(io, 0, q.device)
        L.check(L.lib().rr_cross_attn(C.byref(io), st), "rr_cross_attn")
    del keep, ws
    return out, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, kv_lens, scale):
        out, lse = _forward(q, k, v, mask, kv_lens, scale, True)
        ctx.save_for_backward(q, k, v, mask, kv_lens, out, lse)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        q, k, v, mask, kv_lens, out, lse = ctx.saved_tensors
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)]
        if out.numel() == 0 or k.numel() == 0:
            grads = [t.zero_() for t in grads]
        else:
            dout = _placed(dout)
            io, keep = _io(_placed(q), _placed(k), _placed(v), mask, kv_lens, ctx.scale)
            delta = torch.empty_like(lse)
            io.out, io.lse, io.dout, io.dout_stride, io.delta = out.data_ptr(), lse.data_ptr(), dout.data_ptr(), _strides(dout), delta.data_ptr()
            io.dq, io.dk, io.dv = (t.data_ptr() for t in grads)
            with L.on_device(q) as st:
                ws = _workspace(io, 1, q.device)
                L.check(L.lib().rr_cross_attn_bwd(C.byref(io), st), "rr_cross_attn_bwd")
            del keep, ws
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None, None, None)


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
    return_lse: also the logarithm of the sum of exponentials [B, H, Lq] float32 (-inf where nothing is seen; no gradient through it).
    Differentiable once in query, key and value; no atomics, the same inputs give the same bits."""
    scale = float(query.shape[-1]) ** -0.5 if scale is None and query.shape[-1] else float(scale or 0.0)
    _checked(query, key, value, mask, kv_lens, scale)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        out, lse = _CrossAttention.apply(query, key, value, mask, kv_lens, scale)
    else:
        out, lse = _forward(query, key, value, mask, kv_lens, scale, return_lse)
    return (out, lse) if return_lse else out
