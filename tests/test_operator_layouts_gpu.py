"""Layouts that cost no copy: dimensions of one element with any stride."""

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
