"""Requests that the recurrent and windowed operators refuse by name (no GPU needed)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import gdn_b200

BF = torch.bfloat16


def z(*s, dt=BF):
    return torch.zeros(*s, dtype=dt)


def calls():
    """Every entry with valid shapes: name, function, tensors."""
    x, g, h = z(2, 5, 3, 8), z(2, 5, 3, 8, dt=torch.float32), z(2, 3, 8, dt=torch.float32)
    qkv = [z(1, 4, 4, 64), z(1, 8, 2, 64), z(1, 8, 2, 64)]
    one = [z(1, 4, 64), z(1, 2, 64), z(1, 2, 64), z(1, 16, 2, 64), z(1, 16, 2, 64)]
    pos = torch.zeros(1, dtype=torch.int32)
    gdn = [z(2, 3, 128), z(2, 3, 128), z(2, 3, 128), z(2, 3), z(2, 3), z(2, 3, 128, 128, dt=torch.float32)]
    return [("gated_scan", gdn_b200.gated_scan, [x, g, h]),
            ("gated_scan_step", gdn_b200.gated_scan_step, [x[:, 0], g[:, 0], h]),
            ("window_attention", lambda *t: gdn_b200.window_attention(*t, 4), qkv),
            ("window_attention_step", lambda *t: gdn_b200.window_attention_step(*t, pos, 8, 4), one),
            ("gdn_step", gdn_b200.gdn_step, gdn)]


@pytest.mark.parametrize("which", range(5))
def test_forward_mode_gradients_are_refused(which):
    """A dual tensor's tangent would be dropped without a word."""
    name, f, tensors = calls()[which]
    for i, t in enumerate(tensors):
        with fwd.dual_level():
            dual = tensors[:i] + [fwd.make_dual(t, torch.ones_like(t))] + tensors[i + 1:]
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*dual)
            with pytest.raises(ValueError, match="CUDA|one device"):  # no dual among them: the next check
                f(*tensors)


def test_the_alignment_status_names_the_entries_rules():
    from gdn_b200 import _build, _lib
    _build.build()
    text = _lib.status_string(_lib.ERR_ALIGNMENT)
    assert "16-byte" in text and "gdn_step: 8-byte" in text and "gated_scan: whole elements" in text


def test_expanded_rows_are_refused():
    q, k, v = calls()[2][2]
    for i, name in enumerate("qkv"):
        t = [q, k, v]
        t[i] = t[i][:, :1].expand(t[i].shape)
        with pytest.raises(ValueError, match=f"{name} .*expanded"):
            gdn_b200.window_attention(*t, 4)


def test_a_scale_of_zero_is_refused():
    """0 stands for "not given" in the C structs, so the call would answer with a scale of 1."""
    t = calls()[4][2]
    for scale in (0.0, 0, -0.0):
        with pytest.raises(ValueError, match="scale"):
            gdn_b200.gdn_step(*t, scale=scale)


@pytest.mark.parametrize("scale", [1e-50, -1e-46, 1e39, float("inf"), -float("inf"), float("nan")])
def test_scales_outside_fp32_are_refused(scale):
    """1e-50 would be packed as 0, which stands for 1; 1e39 would raise OverflowError."""
    with pytest.raises(ValueError, match="scale"):
        gdn_b200.gdn_step(*calls()[4][2], scale=scale)
