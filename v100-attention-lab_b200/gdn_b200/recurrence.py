"""Gated linear recurrence over the sequence, with gradients and a single-token form.

The elementwise sibling of the Gated DeltaNet recurrence: the state is a vector
per head instead of a matrix, and every channel has its own decay.  Layouts,
gates, fp32 states and errors are those of ``gdn_chunk_fwd``; everything runs
in the sm_100a library through its C ABI.
"""

from __future__ import annotations

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .ops import _DTYPES, _check_device, _empty, _launch, _refuse_tangents, _status_ptr

__all__ = ["gated_scan", "gated_scan_step"]


def _gate_flags(g_activation):
    if g_activation is None:
        return 0
    if g_activation != "logsigmoid":
        raise ValueError(f"g_activation must be None or 'logsigmoid' (got {g_activation!r})")
    return _lib.FLAG_G_LOGSIGMOID


def _check(x, g, state, state_name, output_dtype, dims):
    for name, t in (("x", x), ("g", g), (state_name, state)):
        if not isinstance(t, torch.Tensor) and (t is not None or name != "initial_state"):
            raise TypeError(f"{name} must be a torch.Tensor")
    _refuse_tangents("the gated recurrence", x, g, state)
    shape, dtype = x.shape, x.dtype
    if len(shape) != len(dims):
        raise ValueError(f"x must be [{', '.join(dims)}] (got shape {tuple(shape)})")
    if g.shape != shape:
        raise ValueError(f"g shape {tuple(g.shape)} != x shape {tuple(shape)}")
    if 0 in shape:
        raise ValueError(f"x must not be empty (got shape {tuple(shape)})")
    for name, t in (("x", x), ("g", g)):
        if t.dtype not in _DTYPES:
            raise NotImplementedError(f"{name} must be fp16, bf16 or fp32 (got {t.dtype})")
        if t.stride(-1) != 1 and shape[-1] != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
    if state is not None and state.shape != (shape[0], shape[-2], shape[-1]):
        raise ValueError(f"{state_name} must be [B, H, D] = {(shape[0], shape[-2], shape[-1])} (got {tuple(state.shape)})")
    out_dtype = dtype if output_dtype is None else output_dtype
    if out_dtype != dtype and out_dtype != torch.float32:
        raise ValueError(f"output_dtype must be x's dtype or torch.float32 (got {out_dtype})")
    for name, t in (("x", x), ("g", g), (state_name, state)):
        if t is not None:
            _check_device(name, t, x.device, "x")
    return out_dtype


def _at(t):
    """Pointer and (b, t, h) strides of a [B, T, H, D] tensor, of a [B, H, D] one (T = 1) or of none."""
    if t is None:
        return 0, 0, 0, 0
    s = t.stride()
    return (t.data_ptr(), s[0], s[1], s[2]) if len(s) == 4 else (t.data_ptr(), s[0], 0, s[1])


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _pack(x, g, o_dtype, flags, h0=None, o=None, ht=None, states=None, d_o=None, dht=None, dx=None, dg=None, dh0=None):
    shape = x.shape
    return _lib.GATED_SCAN_ARGS.pack(
        _lib.ABI_VERSION, shape[0], shape[1] if len(shape) == 4 else 1, shape[-2], shape[-1],
        _DTYPES[x.dtype], _DTYPES[g.dtype], _DTYPES[o_dtype], flags, 0,
        *_at(x), *_at(g), _ptr(h0), *_at(o), _ptr(ht), _ptr(states), *_at(d_o), _ptr(dht), *_at(dx), *_at(dg), _ptr(dh0),
        _status_ptr(x.device))


def _forward(x, g, h0, flags, out_dtype, want_ht, want_states):
    lib = _lib.load()
    dev, shape = x.device, x.shape
    o = _empty(x, out_dtype)
    ht = torch.empty((shape[0], shape[2], shape[3]), dtype=torch.float32, device=dev) if want_ht else None
    states = None
    if want_states:
        nbytes = int(lib.gdn_gated_scan_states_bytes(_pack(x, g, out_dtype, flags)))
        states = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
    _launch(lib.gdn_gated_scan_fwd_sm100, "gdn_gated_scan_fwd_sm100",
            _pack(x, g, out_dtype, flags, h0=h0, o=o, ht=ht, states=states), dev)
    return o, ht, states


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, h0, flags, out_dtype, want_ht):
        o, ht, states = _forward(x, g, h0, flags, out_dtype, want_ht, True)
        ctx.save_for_backward(x, g, states)
        ctx.flags, ctx.out_dtype = flags, out_dtype
        ctx.set_materialize_grads(False)
        return o, ht

    @staticmethod
    def backward(ctx, d_o, dht):
        # The wrapper that refuses a second derivative costs 20 us of host time;
        # without create_graph nothing is recorded, and none can be asked for.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, d_o, dht)


def _backward(ctx, d_o, dht):
    if d_o is None and dht is None:
        return None, None, None, None, None, None
    _refuse_tangents("the gated recurrence's backward", d_o, dht)
    x, g, states = ctx.saved_tensors
    dev = x.device
    dx, dg = _empty(x, x.dtype), _empty(x, g.dtype)
    need_x, need_g, need_h0 = ctx.needs_input_grad[:3]
    dh0 = torch.empty((x.shape[0],) + x.shape[2:], dtype=torch.float32, device=dev) if need_h0 else None
    if d_o is not None and d_o.stride(-1) != 1:  # e.g. the expanded gradient of a sum
        d_o = d_o.contiguous()
    if dht is not None:
        dht = dht.contiguous()
    _launch(_lib.load().gdn_gated_scan_bwd_sm100, "gdn_gated_scan_bwd_sm100",
            _pack(x, g, ctx.out_dtype, ctx.flags, states=states, d_o=d_o, dht=dht, dx=dx, dg=dg, dh0=dh0), dev)
    return dx if need_x else None, dg if need_g else None, dh0, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


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

    The state and all sums are fp32.  Differentiable (once, in reverse mode) in
    x, g and initial_state; the backward recomputes the states in fp32 from x and g and
    states kept every 64 (fp32 x) or 128 rows.  Results repeat bit for bit.
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
    out_dtype = _check(x, g, state, "state", output_dtype, ("B", "H", "D"))
    flags = _gate_flags(g_activation)
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 tensor: it is updated in place")
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad or state.requires_grad):
        raise NotImplementedError("gated_scan_step has no backward: use gated_scan, or torch.no_grad()")
    if g.dtype != torch.float32 and g.dtype != x.dtype:
        g = g.float()
    o = _empty(x, out_dtype)
    B, H, D = x.shape
    sx, sg, at = x.stride(), g.stride(), state.data_ptr()
    args = _lib.GATED_SCAN_ARGS.pack(
        _lib.ABI_VERSION, B, 1, H, D, _DTYPES[x.dtype], _DTYPES[g.dtype], _DTYPES[out_dtype], flags, 0,
        x.data_ptr(), sx[0], 0, sx[1], g.data_ptr(), sg[0], 0, sg[1], at, o.data_ptr(), H * D, 0, D, at, 0,
        0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _launch(_lib.load().gdn_gated_scan_fwd_sm100, "gdn_gated_scan_fwd_sm100", args, x.device)
    increment_version(state)
    return o
