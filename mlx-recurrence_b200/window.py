"""Sliding-window attention with sinks: the sequence mixer that hybrid models
interleave with the recurrences of this package. Like them it keeps a state of
constant size: the last ``window`` keys and values plus the first ``sinks``.

    y_i = sum_j softmax_j(scale q_i . k_j) v_j
    over the j of i's own sequence with j <= i and (i - j < window or j < sinks)

``window_attention`` takes [B, L, H, Dh], ``window_attention_packed`` a packed
batch [T, H, Dh] with sequence borders, ``*_with_state`` also return the caches
that ``window_attention_step`` decodes with. Not in the reference. Unlike the
scans, whose y is float32 because it carries the state, y comes in the inputs'
dtype (float32 inputs: float32). Kernels: ``csrc/window_*.cu``.
"""

from __future__ import annotations

import math
import operator

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._chassis import common_dtype, prep, prep_cu, wants_grad

MAX_SINKS = 64
HEAD_DIMS = (32, 64, 96, 128)


def _check(q, k, v, window, sinks, scale, dims, layout):
    if q.dim() != dims or k.dim() != dims or v.shape != k.shape:
        raise ValueError(f"q, k, v must be {layout}, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    Hq, Dh = q.shape[-2:]
    Hkv = k.shape[-2]
    if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != Dh or Hkv == 0 or Hq == 0 or Hq % Hkv != 0:
        raise ValueError(f"q, k, v must be {layout} with Hq a multiple of Hkv, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if Dh not in HEAD_DIMS:
        raise ValueError(f"Dh={Dh} must be one of {HEAD_DIMS}")
    window, sinks = operator.index(window), operator.index(sinks)
    if window < 1:
        raise ValueError(f"window must be positive, got {window}")
    if not 0 <= sinks <= MAX_SINKS:
        raise ValueError(f"sinks must be in 0..{MAX_SINKS}, got {sinks}")
    scale = Dh ** -0.5 if scale is None else float(scale)
    if not (0.0 < scale <= 2e38):  # times log2(e) it must stay finite
        raise ValueError(f"scale must be positive and at most 2e38, got {scale}")
    return window, sinks, scale


def _rows(t, dt, packed_dims):
    """t in dtype ``dt`` as [T, H, Dh] rows the kernels can read in place:
    dense last axis, 16-byte aligned start and strides (a slice of a fused
    projection qualifies); anything else is copied. Returns (tensor, token
    stride, head stride)."""
    if t.dtype != dt:
        t = t.to(dt)
    if not packed_dims:
        B, L = t.shape[:2]
        if B > 1 and L > 1 and t.stride(0) != L * t.stride(1):
            t = t.contiguous()
        elif B > 1 and L == 1:
            t = t.contiguous()
        t = t.flatten(0, 1)
    n = 16 // t.element_size()
    T, H, Dh = t.shape
    hs = t.stride(1) if H > 1 else Dh
    ts = t.stride(0) if T > 1 else H * hs
    if t.stride(2) != 1 or ts < n or hs < n or ts % n or hs % n or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        ts, hs = H * Dh, Dh
    return t, ts, hs


def _dense16(t, dt):
    t = prep(t.detach() if t.requires_grad else t, dt)
    return t.clone() if t.data_ptr() % 16 else t


def _kernel_args(q, k, v, dt, packed_dims, cu, meta):
    """q, k, v as the kernels read them, and the kernels' shared arguments: strides and addresses are of these very
    tensors, which the caller keeps until it has launched."""
    S, L, window, sinks, scale = meta
    (q, qt, qh), (k, kt, kh), (v, vt, vh) = (_rows(t, dt, packed_dims) for t in (q, k, v))
    T, Hq, Dh = q.shape
    return (q, k, v), (qt, qh, kt, kh, vt, vh, _lib.addr(cu), S, L, _lib.DTYPE_CODE[dt], T, Hq, k.shape[1], Dh, window,
                       sinks, scale)


def _attend(q, k, v, cu, window, sinks, scale, want_lse):
    packed = q.dim() == 3
    dev = _lib.require_cuda(q, k, v)
    dt = common_dtype(q, k, v)
    if packed:
        cu = prep_cu(cu, dev)
        S, L = cu.numel() - 1, 0
    else:
        S, L = q.shape[:2]
    meta = S, L, window, sinks, scale
    (q_, k_, v_), args = _kernel_args(q, k, v, dt, packed, cu, meta)
    T, Hq, Dh = q_.shape
    y = torch.empty((T, Hq, Dh), dtype=dt, device=dev)
    lse = torch.empty((Hq, T), dtype=torch.float32, device=dev) if want_lse else None
    y_low = torch.empty_like(y) if want_lse and dt != torch.float32 else None  # what rounding y drops
    _lib.call_on(dev, "mr_window_attn_fwd", q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), *args, y.data_ptr(),
                 _lib.addr(y_low), _lib.addr(lse))
    return y if packed else y.view(q.shape), meta, (q_, k_, v_, cu, y, y_low, lse)


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu, window, sinks, scale):
        y, ctx.meta, saved = _attend(q, k, v, cu, window, sinks, scale, True)
        ctx.save_for_backward(*saved)
        ctx.shapes = (q.shape, k.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        # Under checkpointing and saved-tensor hooks these are other tensors than the forward's, maybe of other strides:
        # nothing of the forward's addresses or layout is used here.
        q_, k_, v_, cu, y, y_low, lse = ctx.saved_tensors
        dev, dt = q_.device, q_.dtype
        if cu is not None:
            cu = cu.contiguous()
        (q_, k_, v_), args = _kernel_args(q_, k_, v_, dt, True, cu, ctx.meta)
        T, Hq, Dh = q_.shape
        Hkv = k_.shape[1]
        gy, y, lse = _dense16(gy, dt), _dense16(y, dt), lse.contiguous()
        y_low = None if y_low is None else _dense16(y_low, dt)
        gq = torch.empty((T, Hq, Dh), dtype=dt, device=dev)
        gk, gv = (torch.empty((T, Hkv, Dh), dtype=dt, device=dev) for _ in range(2))
        nws = _lib.load().mr_window_attn_bwd_workspace_bytes(_lib.DTYPE_CODE[dt], T, Hq, Hkv, Dh, ctx.meta[3])
        ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=dev)
        _lib.call_on(dev, "mr_window_attn_bwd", gy.data_ptr(), y.data_ptr(), _lib.addr(y_low), lse.data_ptr(),
                     q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), *args, gq.data_ptr(), gk.data_ptr(), gv.data_ptr(),
                     ws.data_ptr(), ws.numel())
        sq, sk = ctx.shapes
        if len(sq) == 4:
            gq, gk, gv = gq.view(sq), gk.view(sk), gv.view(sk)
        return gq, gk, gv, None, None, None, None


def _dispatch(q, k, v, cu, window, sinks, scale):
    if wants_grad(q, k, v):
        return _WindowAttention.apply(q, k, v, cu, window, sinks, scale)
    return _attend(q, k, v, cu, window, sinks, scale, False)[0]


def window_attention(q, k, v, window, sinks=0, scale=None):
    """Causal sliding-window attention with sinks over a dense batch.

    Args:
        q:      [B, L, Hq, Dh]; Dh 32, 64, 96 or 128.
        k, v:   [B, L, Hkv, Dh]; Hq a multiple of Hkv (consecutive query heads
                share a key/value head, whose gradient sums over them).
        window: how many tokens back a query sees, itself included (>= 1).
        sinks:  how many first tokens of the sequence stay visible (0..64).
        scale:  factor of the scores, > 0 (default Dh ** -0.5).

    Returns:
        y: [B, L, Hq, Dh] in the inputs' common dtype (float32, bfloat16 or
        float16); differentiable in q, k, v. Scores, softmax statistics and
        sums are float32; for 16-bit inputs the probabilities, and in the
        backward the scores' gradients, are rounded to the inputs' dtype for
        the tensor cores' products. A key that a query does not see has no influence on
        its row, even if it holds infinities or NaN. Slices of a fused
        projection are read in place.
    """
    window, sinks, scale = _check(q, k, v, window, sinks, scale, 4, "[B, L, H, Dh]")
    return _dispatch(q, k, v, None, window, sinks, scale)


def window_attention_packed(q, k, v, cu_seqlens, window, sinks=0, scale=None):
    """:func:`window_attention` over a packed batch: q [T, Hq, Dh], k, v
    [T, Hkv, Dh], and ``cu_seqlens`` as in :func:`rglru_scan_packed` (rows
    behind the last border come out as zeros, gradients too)."""
    window, sinks, scale = _check(q, k, v, window, sinks, scale, 3, "[T, H, Dh]")
    return _dispatch(q, k, v, cu_seqlens, window, sinks, scale)


def _caches(k, v, dt, cu, window, sinks):
    packed = k.dim() == 3
    dev = k.device
    S, L = (cu.numel() - 1, 0) if packed else k.shape[:2]
    (k_, *ks), (v_, *vs) = (_rows(t.detach(), dt, packed) for t in (k, v))
    T, Hkv, Dh = k_.shape
    slots = sinks + window
    ck, cv = (torch.empty((S, slots, Hkv, Dh), dtype=dt, device=dev) for _ in range(2))
    cu_ = prep_cu(cu, dev) if packed else None
    _lib.call_on(dev, "mr_window_cache", k_.data_ptr(), v_.data_ptr(), *ks, *vs, _lib.addr(cu_), S, L,
                 _lib.DTYPE_CODE[dt], T, Hkv, Dh, slots, sinks, ck.data_ptr(), cv.data_ptr())
    return ck, cv


def window_attention_with_state(q, k, v, window, sinks=0, scale=None):
    """:func:`window_attention` that also returns the caches a decode loop
    starts from: cache_k, cache_v [B, sinks + window, Hkv, Dh] in y's dtype.
    Token t lies in slot t (t < sinks) or sinks + (t - sinks) % window; unused
    slots are zero. The caches are state, not differentiable."""
    y = window_attention(q, k, v, window, sinks, scale)
    return (y, *_caches(k, v, y.dtype, None, operator.index(window), operator.index(sinks)))


def window_attention_packed_with_state(q, k, v, cu_seqlens, window, sinks=0, scale=None):
    """:func:`window_attention_packed` that also returns every sequence's caches
    [S, sinks + window, Hkv, Dh] (see :func:`window_attention_with_state`)."""
    y = window_attention_packed(q, k, v, cu_seqlens, window, sinks, scale)
    return (y, *_caches(k, v, y.dtype, cu_seqlens, operator.index(window), operator.index(sinks)))


def window_attention_step(q, k, v, cache_k, cache_v, pos, sinks=0, scale=None):
    """One decode step on the caches, which are advanced in place.

    Args:
        q:      [B, Hq, Dh], k, v: [B, Hkv, Dh]: the new token's.
        cache_k, cache_v: [B, sinks + window, Hkv, Dh], contiguous, in the
                dtype of q, k, v (:func:`window_attention_with_state`; zeros
                for an empty state). Their extent sets the window.
        pos:    [B] int64 or int32 on the same device: the new token's
                position, counted from 0 (the number of tokens before it). One
                tensor serves every layer; the caller advances it. A row with
                pos < 0 is free: its caches stay as they are and its y is 0.
        sinks, scale: as in :func:`window_attention`.

    Returns:
        y: [B, Hq, Dh] in the inputs' dtype. Not differentiable. (Its products
        take the probabilities' rounding along, unlike the other forms'.)
    """
    dims = "[B, H, Dh]"
    B, Hq, Dh = q.shape if q.dim() == 3 else (0, 0, 0)
    _, sinks, scale = _check(q, k, v, 1, sinks, scale, 3, dims)
    Hkv = k.shape[1]
    dev = _lib.require_cuda(q, k, v, cache_k, cache_v)
    dt = common_dtype(q, k, v)
    if (cache_k.dim() != 4 or cache_k.shape[0] != B or cache_k.shape[1] <= sinks or cache_k.shape[2:] != (Hkv, Dh)
            or cache_v.shape != cache_k.shape):
        raise ValueError(f"caches must both be [B, sinks + window, Hkv, Dh] = [{B}, > {sinks}, {Hkv}, {Dh}], got "
                         f"{tuple(cache_k.shape)} and {tuple(cache_v.shape)}")
    if (cache_k.dtype != dt or cache_v.dtype != dt or not cache_k.is_contiguous() or not cache_v.is_contiguous()
            or (B and (cache_k.data_ptr() % 16 or cache_v.data_ptr() % 16))):
        raise ValueError(f"caches must be contiguous, 16-byte aligned {dt} tensors (updated in place), got "
                         f"{cache_k.dtype} and {cache_v.dtype}")
    if abs(cache_k.data_ptr() - cache_v.data_ptr()) < cache_k.numel() * cache_k.element_size():
        raise ValueError("cache_k and cache_v must not overlap")
    if not isinstance(pos, torch.Tensor) or tuple(pos.shape) != (B,) or pos.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"pos must be an int64 or int32 tensor of shape [{B}]")
    if pos.device != dev:
        raise ValueError(f"pos must be on {dev}, got {pos.device}")
    q_, k_, v_ = _dense16(q, dt), _dense16(k, dt), _dense16(v, dt)
    pos = pos.contiguous()
    y = torch.empty((B, Hq, Dh), dtype=dt, device=dev)
    _lib.call_on(dev, "mr_window_step", q_.data_ptr(), k_.data_ptr(), v_.data_ptr(), cache_k.data_ptr(),
                 cache_v.data_ptr(), pos.data_ptr(), pos.dtype == torch.int64, _lib.DTYPE_CODE[dt], B, Hq, Hkv, Dh,
                 cache_k.shape[1], sinks, scale, y.data_ptr())
    return y


def window_attention_reference(q, k, v, window, sinks=0, scale=None):
    """Masked softmax attention in plain torch over [B, L, H, Dh]. Differentiable, any device."""
    B, L, Hq, Dh = q.shape
    ft = torch.promote_types(q.dtype, torch.float32)
    k, v = (t.to(ft).repeat_interleave(Hq // k.shape[2], dim=2).transpose(1, 2) for t in (k, v))
    i, j = torch.arange(L, device=q.device)[:, None], torch.arange(L, device=q.device)[None]
    see = (j <= i) & ((i - j < window) | (j < sinks))
    s = q.to(ft).transpose(1, 2) @ k.transpose(2, 3) * (Dh ** -0.5 if scale is None else scale)
    return (torch.softmax(s.masked_fill(~see, -math.inf), dim=-1) @ v).transpose(1, 2)
