"""Layouts that cost no copy: dimensions of one element with any stride, inputs
that are expanded over the batch or the heads."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_gdn_step_of_one_request_from_a_packed_projection(dt):
    """A batch of one: its batch stride is never taken, so it need not be a multiple of anything."""
    import gdn_b200
    H = 3
    row = torch.randn(1, 3 * H * 128 + 2 * H + 1, device="cuda").to(dt)  # q, k, v and the gates of one token
    assert row.stride(0) % 4
    row = torch.as_strided(row, row.shape, (row.shape[1], 1))
    q, k, v = (row[:, i * H * 128:(i + 1) * H * 128].view(1, H, 128) for i in range(3))
    beta, g = torch.rand(1, H, device="cuda"), -torch.rand(1, H, device="cuda")
    s0 = torch.randn(1, H, 128, 128, device="cuda")
    s1 = s0.clone()
    got = gdn_b200.gdn_step(q, k, v, beta, g, s0)
    want = gdn_b200.gdn_step(*(t.clone().view(1, H, 128) for t in (q, k, v)), beta, g, s1)
    assert torch.equal(got, want) and torch.equal(s0, s1)
    # one head of many requests: the head stride is never taken
    wide = torch.randn(4, 3 * 128, device="cuda").to(dt)
    q, k, v = (torch.as_strided(wide, (4, 1, 128), (384, 127, 1), 128 * i) for i in range(3))
    s0 = torch.randn(4, 1, 128, 128, device="cuda")
    s1 = s0.clone()
    beta = torch.rand(4, 1, device="cuda")
    got = gdn_b200.gdn_step(q, k, v, beta, None, s0)
    want = gdn_b200.gdn_step(*(t.contiguous() for t in (q, k, v)), beta, None, s1)
    assert torch.equal(got, want) and torch.equal(s0, s1)


@pytest.mark.parametrize("shape", [(3, 200, 300, 4, 2, 64), (2, 130, 130, 6, 6, 128), (80, 256, 256, 4, 2, 64)], ids=str)
def test_window_attention_of_expanded_inputs(shape):
    """One prompt's keys for a whole batch, one key head for all: as copies of them, bit for bit."""
    import gdn_b200
    B, T, S, H, HK, D = shape
    r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    q, k, v = r(B, T, H, D), r(B, S, HK, D), r(B, S, HK, D)
    lengths = torch.randint(S - T, S + 1, (B,), device="cuda", dtype=torch.int32)
    over = {"batch": lambda t: t[:1].expand(t.shape), "heads": lambda t: t[:, :, :1].expand(t.shape),
            "both": lambda t: t[:1, :, :1].expand(t.shape), "none": lambda t: t}
    for eq, ek, ev in (("none", "batch", "batch"), ("batch", "none", "none"), ("heads", "heads", "both"),
                       ("both", "both", "heads"), ("none", "none", "batch")):
        a, b, c = over[eq](q), over[ek](k), over[ev](v)
        got = gdn_b200.window_attention(a, b, c, 90, 3, lengths=lengths)
        want = gdn_b200.window_attention(a.contiguous(), b.contiguous(), c.contiguous(), 90, 3, lengths=lengths)
        gdn_b200.check_status()
        assert torch.equal(got, want), (eq, ek, ev)


def test_rows_that_are_expanded_are_named():
    """One row as a whole sequence is refused, by name."""
    import gdn_b200
    r = lambda *s: torch.randn(*s, device="cuda").bfloat16()
    q, k, v = r(1, 40, 2, 64), r(1, 40, 2, 64), r(1, 40, 2, 64)
    for i in range(3):
        t = [q, k, v]
        t[i] = t[i][:, :1].expand(t[i].shape)
        with pytest.raises(ValueError, match=f"{'qkv'[i]} .*expanded"):
            gdn_b200.window_attention(*t, 8)
