"""Causal attention over a sliding window and the first few tokens (sinks).

The softmax attention that stacks of recurrent layers mix in: its state is
bounded too, by the window.  ``window_attention`` takes prompts and chunks of
prompts, ``window_attention_step`` one token against a ring cache.  Layouts,
errors and streams are those of ``gdn_chunk_fwd``; everything runs in the
sm_100a library through its C ABI.
"""

from __future__ import annotations

import math

import torch

from . import _lib, ops
from .ops import _DTYPES, _launch

__all__ = ["window_attention", "window_attention_step"]


def _check(tensors, window, sinks, scale, D):
    q = tensors["q"]
    for name, t in tensors.items():
        if t.dtype != q.dtype:
            raise ValueError(f"{name} must have q's dtype (got {t.dtype}, q has {q.dtype})")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise NotImplementedError(f"gdn_b200 takes fp16 or bf16 q/k/v (got {q.dtype})")
    if D not in (64, 128):
        raise NotImplementedError(f"the head size must be 64 or 128 (got {D})")
    if int(window) < 1 or int(sinks) < 0:
        raise ValueError(f"window must be at least 1 and sinks at least 0 (got {window}, {sinks})")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"scale must be positive (got {scale})")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors.values()):
        raise NotImplementedError("windowed attention has no backward: call it under torch.no_grad()")
    return scale


def _check_devices(tensors, dev):
    for name, t in tensors.items():
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (got device {t.device})")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, q is on {dev}")


def _check_tensors(**tensors):
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")


def _check_ints(name, t, B):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape ({B},)")


def window_attention(q, k, v, window, sinks=0, *, scale=None, lengths=None):
    """Causal softmax attention over the last ``window`` tokens and the first ``sinks``.

    Args:
        q: [B, T, H, D] fp16/bf16, D 64 or 128 (last dim contiguous, rows
            16-byte aligned)
        k, v: [B, S, HK, D] same dtype, S >= T, H a multiple of HK: query head
            h reads key head h // (H // HK)
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
    _check_tensors(q=q, k=k, v=v)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q must be [B, T, H, D], k and v [B, S, HK, D]")
    B, T, H, D = q.shape
    S, HK = k.shape[1], k.shape[2]
    if tuple(k.shape) != (B, S, HK, D) or k.shape != v.shape:
        raise ValueError(f"k and v must be [{B}, S, HK, {D}] (got {tuple(k.shape)} and {tuple(v.shape)})")
    if 0 in q.shape or 0 in k.shape:
        raise ValueError("q, k and v must not be empty")
    if H % HK != 0:
        raise ValueError(f"the number of query heads ({H}) must be a multiple of the key heads ({HK})")
    if S < T:
        raise ValueError(f"fewer keys ({S}) than query rows ({T})")
    scale = _check({"q": q, "k": k, "v": v}, window, sinks, scale, D)
    if lengths is not None:
        _check_ints("lengths", lengths, B)
    dev = q.device
    _check_devices({"q": q, "k": k, "v": v} if lengths is None else {"q": q, "k": k, "v": v, "lengths": lengths}, dev)
    lib = _lib.load()
    o = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    a = _lib.WindowAttnArgs()
    a.abi_version = _lib.ABI_VERSION
    a.B, a.T, a.S, a.H, a.HK, a.D = B, T, S, H, HK, D
    a.dtype = _DTYPES[q.dtype]
    # beyond the keys neither changes anything
    a.window, a.sinks = min(int(window), S), min(int(sinks), S)
    a.scale = scale
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_stride", t.stride()[:3])
    if lengths is not None:
        a.lengths = lengths.data_ptr()
    # The status word is made outside of graph captures: one made inside would
    # live, and be cleared, with the graph.
    if dev.index in ops._status_words or not torch.cuda.is_current_stream_capturing():
        a.status = ops._status_word(dev).data_ptr()
    _launch(lib.gdn_window_attn_sm100, "gdn_window_attn_sm100", a, dev)
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
    _check_tensors(q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache)
    if q.dim() != 3 or k.dim() != 3 or k_cache.dim() != 4:
        raise ValueError("q must be [B, H, D], k and v [B, HK, D], the caches [B, capacity, HK, D]")
    B, H, D = q.shape
    HK, cap = k.shape[1], k_cache.shape[1]
    if tuple(k.shape) != (B, HK, D) or k.shape != v.shape:
        raise ValueError(f"k and v must be [{B}, HK, {D}] (got {tuple(k.shape)} and {tuple(v.shape)})")
    if tuple(k_cache.shape) != (B, cap, HK, D) or k_cache.shape != v_cache.shape:
        raise ValueError(f"the caches must be [{B}, capacity, {HK}, {D}] (got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)})")
    if 0 in q.shape or 0 in k_cache.shape:
        raise ValueError("q, k, v and the caches must not be empty")
    if H % HK != 0:
        raise ValueError(f"the number of query heads ({H}) must be a multiple of the key heads ({HK})")
    tensors = {"q": q, "k": k, "v": v, "k_cache": k_cache, "v_cache": v_cache}
    scale = _check(tensors, window, sinks, scale, D)
    window, sinks = int(window), int(sinks)
    if window + sinks > cap:
        raise ValueError(f"the cache's capacity ({cap}) must hold window + sinks ({window + sinks}) tokens")
    for name in ("k_cache", "v_cache"):
        if any(n > 1 and s == 0 for n, s in zip(tensors[name].shape, tensors[name].stride())):
            raise ValueError(f"{name} is written to and must not be an expanded tensor")
    _check_ints("positions", positions, B)
    dev = q.device
    tensors["positions"] = positions
    _check_devices(tensors, dev)
    lib = _lib.load()
    o = torch.empty(B, H, D, dtype=q.dtype, device=dev)
    a = _lib.WindowStepArgs()
    a.abi_version = _lib.ABI_VERSION
    a.B, a.H, a.HK, a.D = B, H, HK, D
    a.capacity, a.window, a.sinks = cap, window, sinks
    a.dtype = _DTYPES[q.dtype]
    a.scale = scale
    for name, t in (("q", q), ("k", k), ("v", v), ("o", o)):
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_stride", t.stride()[:2])
    for name, t in (("k", k_cache), ("v", v_cache)):
        setattr(a, name + "_cache", t.data_ptr())
        setattr(a, name + "c_stride", t.stride()[:3])
    a.positions = positions.data_ptr()
    _launch(lib.gdn_window_step_sm100, "gdn_window_step_sm100", a, dev)
    return o
