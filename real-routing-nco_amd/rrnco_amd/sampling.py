"""A choice from logits with given random numbers on csrc/rr_draw.hip, beside rr_select's keyed generator (rrnco/models/decoding.py:272-298, 311-361)."""
from __future__ import annotations

import torch

from . import _lib as L

MAX_CHOICES = 1 << 24


def _setting(name, v, R, dev, low, high, dtype):
    """A number for all rows -> (number, None); a tensor [rows] -> (0, tensor in the kernel's type)."""
    if torch.is_tensor(v):
        if v.numel() != R or v.device != dev or v.dtype.is_complex or v.dtype == torch.bool:
            raise ValueError(f"sample: {name} is a number or a tensor of one number for each of the {R} rows on the logits' device")
        return 0, v.reshape(R).to(dtype).contiguous()
    if not low <= v <= high:
        raise ValueError(f"sample: {name} in {low} .. {high}, got {v}")
    return v, None


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=0.0, min_p=0.0, mask=None):
    """One choice for every row of logits [..., V] from the random numbers uniforms [...] -> (index [...] int64, logp [...] float32).

    The row's distribution is softmax(logits / temperature) over the keys that mask (bool, broadcastable to the logits, True = may be drawn) leaves,
    filtered in this order:  top_k keeps the logits that are not under the k-th largest, top_p those of them that have less than top_p of their mass
    strictly above, min_p those whose probability is at least min_p times the largest.  Equal logits stay or go together, so a filter may keep copies
    of its last value.  index is the first key, in index order, at which the running sum of the kept weights exceeds uniform * their sum; logp its
    log-probability among them.  Weights and sums are held in 64 bits: the same numbers give the same choices as any other exact evaluation.
    temperature 0 takes the largest logit, the lowest index among equals, with logp 0.  0 (and 1 for top_p, V and more for top_k) switches a filter off.
    temperature, top_k, top_p, min_p: a number, or a tensor with one for each row (out of range: temperatures that are not positive count as 0,
    top_k below 1 and top_p outside (0, 1) as off, min_p above 1 as 1).
    logits float32 / float16 / bfloat16, rows of up to 2^24 keys by any row stride; NaN and -inf are never drawn; a row with nothing left gives
    index 0 and logp -inf.  uniforms float32 in [0, 1) (a number outside counts as the nearer end, NaN as 0).  No gradient."""
    if logits.dtype not in L.DTYPE_CODE:
        raise TypeError(f"sample: logits float32, float16 or bfloat16, got {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_CHOICES:
        raise ValueError(f"sample: logits [..., V] with V in 1 .. {MAX_CHOICES}, got shape {tuple(logits.shape)}")
    lead, V, dev = logits.shape[:-1], logits.shape[-1], logits.device
    if uniforms.shape != lead or uniforms.dtype != torch.float32 or uniforms.device != dev:
        raise ValueError(f"sample: uniforms float32 of shape {tuple(lead)} on the logits' device, got {uniforms.dtype} {tuple(uniforms.shape)}")
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != dev:
            raise ValueError("sample: mask is a bool tensor on the logits' device, True where a key may be drawn")
        if mask.dim() > logits.dim() or any(m not in (1, n) for m, n in zip(mask.shape[::-1], logits.shape[::-1])):
            raise ValueError(f"sample: mask {tuple(mask.shape)} does not broadcast to the logits' {tuple(logits.shape)}")
    x = logits.detach().reshape(-1, V)
    R = x.shape[0]
    if R > 0x7fffffff:
        raise ValueError("sample: at most 2^31 - 1 rows")
    t, row_t = _setting("temperature", temperature, R, dev, 0.0, 1e29, torch.float32)
    k, row_k = _setting("top_k", top_k, R, dev, 0, 1 << 40, torch.int32)
    p, row_p = _setting("top_p", top_p, R, dev, 0.0, 1.0, torch.float32)
    mp, row_mp = _setting("min_p", min_p, R, dev, 0.0, 1.0, torch.float32)
    L.require_gpu(logits)
    if V > 1 and x.stride(1) != 1:
        x = x.contiguous()
    if mask is not None:
        mask = mask.expand(logits.shape).reshape(-1, V)
        if V > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
    u = uniforms.reshape(-1).contiguous()
    index, logp = torch.empty(lead, dtype=torch.int64, device=dev), torch.empty(lead, dtype=torch.float32, device=dev)
    opt = lambda s: None if s is None else s.data_ptr()                                       # noqa: E731
    if R:
        lib = L.lib()
        n = lib.rr_draw_workspace(R, V)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        with L.on_device(logits) as st:
            L.check(lib.rr_draw(L.DTYPE_CODE[x.dtype], x.data_ptr(), x.stride(0), opt(mask), 0 if mask is None else mask.stride(0), u.data_ptr(),
                                    index.data_ptr(), logp.data_ptr(), R, V, float(t), min(int(k), V), float(p), float(mp), opt(row_t), opt(row_k), opt(row_p),
                                    opt(row_mp), opt(ws), n, st), "rr_draw")
    return index, logp
