"""Causal attention over a sliding window and the first few tokens (sinks).

The softmax attention that stacks of recurrent layers mix in: its state is
bounded too, by the window.  ``window_attention`` takes prompts and chunks of
prompts, ``window_attention_step`` one token against a ring cache.  Layouts,
errors and streams are those of ``gdn_chunk_fwd``; everything runs in the
sm_100a library through its C ABI.
"""

from __future__ import annotations

import operator

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _DTYPES, _check_device, _empty, _launch, _refuse_tangents, _status_ptr

__all__ = ["window_attention", "window_attention_step"]


def _check_tensors(tensors):
    """Types, layouts and gradients of the tensors; their common type is the first's."""
    grad = torch.is_grad_enabled()
    dtype = None
    for name, t in tensors:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if dtype is None:
            dtype = t.dtype
        elif t.dtype != dtype:
            raise ValueError(f"{name} must have q's dtype (got {t.dtype}, q has {dtype})")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
        if grad and t.requires_grad:
            raise NotImplementedError("windowed attention has no backward: call it under torch.no_grad()")
    _refuse_tangents("windowed attention", *(t for _, t in tensors))
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise NotImplementedError(f"gdn_b200 takes fp16 or bf16 q/k/v (got {dtype})")


def _check_sizes(D, window, sinks, scale):
    """Head size, window and sinks; returns the scale."""
    if D != 64 and D != 128:
        raise NotImplementedError(f"the head size must be 64 or 128 (got {D})")
    if window < 1 or sinks < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0 (got {window}, {sinks})")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"scale must be positive (got {scale})")
    return scale


def _check_devices(tensors, dev):
    """All CUDA tensors on ``dev``, the device of the first."""
    for name, t in tensors:
        if t.device != dev or not t.is_cuda:
            _check_device(name, t, dev, "q")


def _check_ints(name, t, B):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape ({B},)")


def window_attention(q, k, v, window, sinks=0, *, scale=None, lengths=None):
    """Causal softmax attention over the last ``window`` tokens and the first ``sinks``.

    Args:
        q: [B, T, H, D] fp16/bf16, D 64 or 128 (last dim contiguous, rows
            16-byte aligned)
        k, v: [B, S, HK, D] same dtype, S >= T, H a multiple of HK: query head
            h reads key head h // (H // HK); like q they may be expanded
            (stride 0) over the batch or the heads
        window: tokens a row sees, itself included (>= 1)
        sinks: first tokens that stay visible behind the window
        scale: factor of q k^T, positive; None = 1/sqrt(D)
        lengths: optional [B] int32 on q's device, the number of tokens of each
            right-padded sequence (clamped to 0..S); keys behind it are hidden
            and rows behind it are 0
    Returns:
        o [B, T, H, D] in q's dtype

    Row i sits at position S - T + i: with S == T a whole prompt, with S > T a
    chunk of one whose keys so far are all in k and v.  Hidden keys and values
    may hold anything, NaN and infinities included.  Inference only.
    """
    tensors = (("q", q), ("k", k), ("v", v))
    _check_tensors(tensors)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q must be [B, T, H, D], k and v [B, S, HK, D]")
    B, T, H, D = q.shape
    S, HK = k.shape[1], k.shape[2]
    if k.shape != (B, S, HK, D) or k.shape != v.shape:
        raise ValueError(f"k and v must be [{B}, S, HK, {D}] (got {tuple(k.shape)} and {tuple(v.shape)})")
    if not (B and T and H and D and S and HK):
        raise ValueError("q, k and v must not be empty")
    if H % HK != 0:
        raise ValueError(f"the number of query heads ({H}) must be a multiple of the key heads ({HK})")
    if S < T:
        raise ValueError(f"fewer keys ({S}) than query rows ({T})")
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    if (sq[1] == 0 and T > 1) or ((sk[1] == 0 or sv[1] == 0) and S > 1):
        name = "q" if sq[1] == 0 and T > 1 else "k" if sk[1] == 0 else "v"
        raise ValueError(f"{name} must not be expanded along its rows (stride 0); over the batch or the heads it may be")
    window, sinks = operator.index(window), operator.index(sinks)
    scale = _check_sizes(D, window, sinks, scale)
    dev = q.device
    if lengths is not None:
        _check_ints("lengths", lengths, B)
        _check_device("lengths", lengths, dev, "q")
    _check_devices(tensors, dev)
    o = _empty(q, q.dtype)
    so = o.stride()
    args = _lib.WINDOW_ATTN_ARGS.pack(
        # beyond the keys neither window nor sinks change anything
        _lib.ABI_VERSION, B, T, S, H, HK, D, _DTYPES[q.dtype], min(window, S), min(sinks, S), scale, 0,
        q.data_ptr(), sq[0], sq[1], sq[2], k.data_ptr(), sk[0], sk[1], sk[2], v.data_ptr(), sv[0], sv[1], sv[2],
        o.data_ptr(), so[0], so[1], so[2], 0 if lengths is None else lengths.data_ptr(),
        _status_ptr(dev))
    _launch(_lib.load().gdn_window_attn_sm100, "gdn_window_attn_sm100", args, dev)
    return o


def window_attention_step(q, k, v, k_cache, v_cache, positions, window, sinks=0, *, scale=None):
    """One token of ``window_attention``, against a ring cache that it extends.

    Args:
        q: [B, H, D] fp16/bf16, D 64 or 128
        k, v: [B, HK, D] the token's own key and value
        k_cache, v_cache: [B, capacity, HK, D], capacity >= window + sinks;
            the token is written into its slot
        positions: [B] int32 on q's device: the token's position (0 for the
            first); negative: the row is off, o is 0, the cache stays as it is
        window, sinks, scale: as in ``window_attention``
    Returns:
        o [B, H, D] in q's dtype

    Position j lives in slot j while j < capacity, then in slot
    ``sinks + (j - sinks) % (capacity - sinks)``: the sinks stay, the rest is a
    ring.  Slots without a visible token may hold anything.  Two sequences must
    not share cache memory.  Inference only.
    """
    tensors = (("q", q), ("k", k), ("v", v), ("k_cache", k_cache), ("v_cache", v_cache))
    _check_tensors(tensors)
    if q.dim() != 3 or k.dim() != 3 or k_cache.dim() != 4:
        raise ValueError("q must be [B, H, D], k and v [B, HK, D], the caches [B, capacity, HK, D]")
    B, H, D = q.shape
    HK, cap = k.shape[1], k_cache.shape[1]
    if k.shape != (B, HK, D) or k.shape != v.shape:
        raise ValueError(f"k and v must be [{B}, HK, {D}] (got {tuple(k.shape)} and {tuple(v.shape)})")
    if k_cache.shape != (B, cap, HK, D) or k_cache.shape != v_cache.shape:
        raise ValueError(f"the caches must be [{B}, capacity, {HK}, {D}] (got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)})")
    if not (B and H and D and HK and cap):
        raise ValueError("q, k, v and the caches must not be empty")
    if H % HK != 0:
        raise ValueError(f"the number of query heads ({H}) must be a multiple of the key heads ({HK})")
    window, sinks = operator.index(window), operator.index(sinks)
    scale = _check_sizes(D, window, sinks, scale)
    if window + sinks > cap:
        raise ValueError(f"the cache's capacity ({cap}) must hold window + sinks ({window + sinks}) tokens")
    skc, svc = k_cache.stride(), v_cache.stride()
    for name, s in (("k_cache", skc), ("v_cache", svc)):
        if (s[0] == 0 and B > 1) or (s[1] == 0 and cap > 1) or (s[2] == 0 and HK > 1):
            raise ValueError(f"{name} is written to and must not be an expanded tensor")
    _check_ints("positions", positions, B)
    dev = q.device
    _check_devices(tensors, dev)
    _check_device("positions", positions, dev, "q")
    o = _empty(q, q.dtype)
    sq, sk, sv, so = q.stride(), k.stride(), v.stride(), o.stride()
    args = _lib.WINDOW_STEP_ARGS.pack(
        _lib.ABI_VERSION, B, H, HK, D, cap, window, sinks, _DTYPES[q.dtype], scale,
        q.data_ptr(), sq[0], sq[1], k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1],
        k_cache.data_ptr(), skc[0], skc[1], skc[2], v_cache.data_ptr(), svc[0], svc[1], svc[2],
        o.data_ptr(), so[0], so[1], positions.data_ptr())
    _launch(_lib.load().gdn_window_step_sm100, "gdn_window_step_sm100", args, dev)
    increment_version((k_cache, v_cache))
    return o
