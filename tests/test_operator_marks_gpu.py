"""What autograd is told (of states that are overwritten, of gradients that are not there), and captured tokens."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_an_overwritten_state_is_noticed_by_autograd():
    """A state or cache that a recorded graph has saved and a step overwrites: its backward raises."""
    import gdn_b200
    B, H, D = 2, 3, 128
    r = lambda *s: torch.randn(*s, device="cuda")

    def saved(shape, dtype=torch.float32):
        s = r(*shape).to(dtype).requires_grad_() * 1
        return s, (s * s).sum()

    x, g = r(B, H, D), -torch.rand(B, H, D, device="cuda")
    h, loss = saved((B, H, D))
    with torch.no_grad():
        gdn_b200.gated_scan_step(x, g, h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()

    q = r(B, H, D).bfloat16()
    s, loss = saved((B, H, D, D))
    with torch.no_grad():
        gdn_b200.gdn_step(q, q, q, torch.rand(B, H, device="cuda"), None, s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()

    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    for which in range(2):
        c = [r(B, 9, H, D).bfloat16() for _ in range(2)]
        c[which], loss = saved((B, 9, H, D), torch.bfloat16)
        with torch.no_grad():
            gdn_b200.window_attention_step(q, q, q, *c, pos, 8, 1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_steps_under_inference_mode():
    """Tensors made there have no version to count; those made before have."""
    import gdn_b200
    B, H, D = 1, 2, 128
    old = torch.zeros(B, H, D, device="cuda")
    before = old._version
    with torch.inference_mode():
        q = torch.randn(B, H, D, device="cuda").bfloat16()
        beta = torch.rand(B, H, device="cuda")
        new, S = torch.zeros(B, H, D, device="cuda"), torch.zeros(B, H, D, D, device="cuda")
        kc, vc = (torch.zeros(B, 4, H, D, device="cuda", dtype=q.dtype) for _ in range(2))
        for state in (old, new):
            gdn_b200.gated_scan_step(q, -q.abs(), state)
        gdn_b200.gdn_step(q, q, q, beta, None, S)
        gdn_b200.window_attention_step(q, q, q, kc, vc, torch.zeros(B, dtype=torch.int32, device="cuda"), 4)
        assert torch.equal(old, new)
    assert old._version > before


def test_a_dual_gradient_is_refused_by_the_backward():
    """The backward is linear in the outputs' gradient, whose tangent would be dropped without a word."""
    import gdn_b200
    import torch.autograd.forward_ad as fwd
    x = torch.randn(1, 20, 1, 8, device="cuda", requires_grad=True)
    o, _ = gdn_b200.gated_scan(x, -torch.rand_like(x).detach())
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(o, x, fwd.make_dual(torch.ones_like(o).detach(), torch.ones_like(o).detach()))


def test_captured_tokens_of_the_recurrences():
    """One captured token of gdn_step and gated_scan_step, replayed along a sequence."""
    import gdn_b200
    B, H, D, n = 2, 3, 128, 12
    gen = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    q, k, v = (torch.nn.functional.normalize(r(n, B, H, D), dim=-1).bfloat16() for _ in range(3))
    beta, g, z = r(n, B, H), r(n, B, H) + 2, r(n, B, H, D) + 2
    kw = dict(beta_activation="sigmoid", g_activation="logsigmoid")
    S0, h0 = 0.1 * r(B, H, D, D), r(B, H, D)

    def token(i, S, h):
        return (gdn_b200.gdn_step(i[0], i[1], i[2], i[3], i[4], S, **kw),
                gdn_b200.gated_scan_step(i[2], i[5], h, g_activation="logsigmoid"))

    rows = [[t[j] for t in (q, k, v, beta, g, z)] for j in range(n)]
    S, h = S0.clone(), h0.clone()
    want = [token(i, S, h) for i in rows]
    slots = [torch.zeros_like(t) for t in rows[0]]
    Sg, hg = S0.clone(), h0.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = token(slots, Sg, hg)
    Sg.copy_(S0), hg.copy_(h0)
    for j in range(n):
        for s, t in zip(slots, rows[j]):
            s.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want[j])), j
    assert torch.equal(Sg, S) and torch.equal(hg, h)
