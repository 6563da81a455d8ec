"""Gated linear recurrence over the sequence, with gradients and a single-token form.

The elementwise sibling of the Gated DeltaNet recurrence: the state is a vector
per head instead of a matrix, and every channel has its own decay.  Layouts,
gates, fp32 states and errors are those of ``gdn_chunk_fwd``; everything runs
in the sm_100a library through its C ABI.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import _DTYPES, _launch

__all__ = ["gated_scan", "gated_scan_step"]


def _gate_flags(g_activation):
    if g_activation is None:
        return 0
    if g_activation != "logsigmoid":
        raise ValueError(f"g_activation must be None or 'logsigmoid' (got {g_activation!r})")
    return _lib.FLAG_G_LOGSIGMOID


def _check(x, g, state, state_name, output_dtype, dims):
    for name, t in (("x", x), ("g", g), (state_name, state)):
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    if x.dim() != len(dims):
        raise ValueError(f"x must be [{', '.join(dims)}] (got shape {tuple(x.shape)})")
    if g.shape != x.shape:
        raise ValueError(f"g shape {tuple(g.shape)} != x shape {tuple(x.shape)}")
    if 0 in x.shape:
        raise ValueError(f"x must not be empty (got shape {tuple(x.shape)})")
    for name, t in (("x", x), ("g", g)):
        if t.dtype not in _DTYPES:
            raise NotImplementedError(f"{name} must be fp16, bf16 or fp32 (got {t.dtype})")
        if t.stride(-1) != 1 and t.shape[-1] != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
    shape = (x.shape[0],) + tuple(x.shape[-2:])
    if state is not None and tuple(state.shape) != shape:
        raise ValueError(f"{state_name} must be [B, H, D] = {shape} (got {tuple(state.shape)})")
    out_dtype = x.dtype if output_dtype is None else output_dtype
    if out_dtype != x.dtype and out_dtype != torch.float32:
        raise ValueError(f"output_dtype must be x's dtype or torch.float32 (got {out_dtype})")
    dev = x.device
    for name, t in (("x", x), ("g", g), (state_name, state)):
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (got device {t.device})")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, x is on {dev}")
    return out_dtype


def _set(a, name, t):
    """Pointer and (b, t, h) strides of a [B, T, H, D] tensor, or of a [B, H, D] one (T = 1)."""
    st = t.stride()
    setattr(a, name, t.data_ptr())
    stride = (st[0], st[1], st[2]) if t.dim() == 4 else (st[0], 0, st[1])
    setattr(a, ("do" if name == "d_o" else name) + "_stride", stride)


def _args(x, g, out_dtype, flags):
    a = _lib.GatedScanArgs()
    a.abi_version = _lib.ABI_VERSION
    if x.dim() == 4:
        a.B, a.T, a.H, a.D = x.shape
    else:
        a.B, a.H, a.D = x.shape
        a.T = 1
    a.x_dtype, a.g_dtype, a.o_dtype = _DTYPES[x.dtype], _DTYPES[g.dtype], _DTYPES[out_dtype]
    a.flags = flags
    _set(a, "x", x)
    _set(a, "g", g)
    return a


def _forward(x, g, h0, flags, out_dtype, want_ht, want_states):
    lib = _lib.load()
    dev = x.device
    o = torch.empty(x.shape, dtype=out_dtype, device=dev)
    a = _args(x, g, out_dtype, flags)
    _set(a, "o", o)
    ht = states = None
    if h0 is not None:
        a.h0 = h0.data_ptr()
    if want_ht:
        ht = torch.empty(x.shape[0], *x.shape[-2:], dtype=torch.float32, device=dev)
        a.ht = ht.data_ptr()
    if want_states:
        states = torch.empty(int(lib.gdn_gated_scan_states_bytes(ctypes.byref(a))) // 4, dtype=torch.float32, device=dev)
        a.states = states.data_ptr()
    _launch(lib.gdn_gated_scan_fwd_sm100, "gdn_gated_scan_fwd_sm100", a, dev)
    return o, ht, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, h0, flags, out_dtype, want_ht):
        o, ht, states = _forward(x, g, h0, flags, out_dtype, want_ht, True)
        ctx.save_for_backward(x, g, states)
        ctx.flags, ctx.out_dtype, ctx.has_h0 = flags, out_dtype, h0 is not None
        ctx.set_materialize_grads(False)
        return o, ht

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, dht):
        if d_o is None and dht is None:
            return None, None, None, None, None, None
        x, g, states = ctx.saved_tensors
        lib = _lib.load()
        a = _args(x, g, ctx.out_dtype, ctx.flags)
        a.states = states.data_ptr()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dg = torch.empty(g.shape, dtype=g.dtype, device=x.device)
        _set(a, "dx", dx)
        _set(a, "dg", dg)
        dh0 = None
        if d_o is not None:
            if d_o.stride(-1) != 1:  # e.g. the expanded gradient of a sum
                d_o = d_o.contiguous()
            _set(a, "d_o", d_o)
        if dht is not None:
            dht = dht.contiguous()
            a.dht = dht.data_ptr()
        if ctx.has_h0 and ctx.needs_input_grad[2]:
            dh0 = torch.empty(x.shape[0], *x.shape[2:], dtype=torch.float32, device=x.device)
            a.dh0 = dh0.data_ptr()
        _launch(lib.gdn_gated_scan_bwd_sm100, "gdn_gated_scan_bwd_sm100", a, x.device)
        return (dx if ctx.needs_input_grad[0] else None, dg if ctx.needs_input_grad[1] else None, dh0, None, None, None)


def gated_scan(x, g, initial_state=None, *, g_activation=None, output_dtype=None, output_final_state=True):
    """Gated linear recurrence ``h_t = a_t h_{t-1} + x_t``, one chain per channel.

    Args:
        x: [B, T, H, D] fp16, bf16 or fp32 (last dim contiguous), any D and T >= 1
        g: [B, T, H, D] log decay (<= 0), ``a = exp(g)``, in fp32 or x's dtype
            (another dtype is cast to fp32); -inf resets the chain
        initial_state: optional [B, H, D] state h_0 (fp32 is used)
        g_activation: 'logsigmoid' if g holds logits (``a = sigmoid(g)``)
        output_dtype: dtype of o: x's (default) or torch.float32
        output_final_state: return the final state (else None)
    Returns:
        (o [B, T, H, D] = every h_t, h_T [B, H, D] fp32 or None)

    The state and all sums are fp32.  Differentiable (once) in x, g and
    initial_state; the backward recomputes the states in fp32 from x and g and
    states kept every 32 (fp32 x) or 64 rows.  Results repeat bit for bit.
    Launches on the current stream of x's device without synchronising.
    """
    out_dtype = _check(x, g, initial_state, "initial_state", output_dtype, ("B", "T", "H", "D"))
    flags = _gate_flags(g_activation)
    if g.dtype != torch.float32 and g.dtype != x.dtype:
        g = g.float()
    h0 = None if initial_state is None else initial_state.to(torch.float32).contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or (h0 is not None and h0.requires_grad)):
        return _GatedScan.apply(x, g, h0, flags, out_dtype, bool(output_final_state))
    o, ht, _ = _forward(x, g, h0, flags, out_dtype, output_final_state, False)
    return o, ht


def gated_scan_step(x, g, state, *, g_activation=None, output_dtype=None):
    """One token of ``gated_scan``: the state is updated in place, its new value returned as o.

    Args:
        x, g: [B, H, D], as in ``gated_scan`` without the time dimension
        state: [B, H, D] fp32, contiguous; overwritten with ``a * state + x``
        g_activation, output_dtype: as in ``gated_scan``
    Returns:
        o [B, H, D] in x's dtype or output_dtype

    For inference: tensors that require gradients are refused while gradients
    are recorded.
    """
    if state is None:
        raise TypeError("state must be a torch.Tensor")
    out_dtype = _check(x, g, state, "state", output_dtype, ("B", "H", "D"))
    flags = _gate_flags(g_activation)
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 tensor: it is updated in place")
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or state.requires_grad):
        raise NotImplementedError("gated_scan_step has no backward: use gated_scan, or torch.no_grad()")
    if g.dtype != torch.float32 and g.dtype != x.dtype:
        g = g.float()
    lib = _lib.load()
    o = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    a = _args(x, g, out_dtype, flags)
    _set(a, "o", o)
    a.h0 = a.ht = state.data_ptr()
    _launch(lib.gdn_gated_scan_fwd_sm100, "gdn_gated_scan_fwd_sm100", a, x.device)
    return o
