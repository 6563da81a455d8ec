"""The gated linear recurrence against its definition in 64 bits.

Tolerances come from the arithmetic.  With eps = 2^-24: the base-2 exponential
is off by 4 eps, its argument's rounding adds |g| eps (|g| <= 7 here), and for
logits 1 + e, its reciprocal and the product with e add 4: a gate, or its
gradient's factor 1 - a, is off by (8 + |g|) eps at most, 15.  Every row adds
the roundings of its products and sums, once in the row itself and once in
the maps that carry the state across it: 18 eps of the row's magnitude in all.
So an error bound follows the recurrence itself,

    E_t = a_t E_{t-1} + 18 eps S_t,   S_t = a_t S_{t-1} + |x_t|,

backwards the same with |do_t|; products add their factors' errors.  Storing in
a type adds half a step of it.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 18 * 2.0 ** -24


def scan64(a, x, h0):
    """All h_t of h_t = a_t h_{t-1} + x_t, step by step."""
    h, out = h0, []
    for t in range(a.shape[1]):
        h = a[:, t] * h + x[:, t]
        out.append(h)
    return torch.stack(out, 1)


def bound64(a, s):
    """E_t = a_t E_{t-1} + EPS s_t from E = 0."""
    return scan64(a, EPS * s, torch.zeros_like(s[:, 0]))


def stored(t, ref):
    return torch.finfo(t.dtype).eps / 2 * ref.abs() + torch.finfo(t.dtype).smallest_normal


def check(name, got, ref, err):
    off = (got.detach().double() - ref).abs()
    tol = err * (1 + torch.finfo(got.dtype).eps) + stored(got, ref)
    assert torch.isfinite(got).all(), name
    worst = (off / tol).max().item()
    assert worst <= 1, (name, worst)


def make(B, T, H, D, x=torch.bfloat16, g=torch.float32, logits=False, seed=0, h0=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    z = r(B, T, H, D) + 2
    gt = (z if logits else torch.nn.functional.logsigmoid(z)).to(g)
    return r(B, T, H, D).to(x), gt, (r(B, H, D) if h0 else None), r(B, T, H, D), r(B, H, D)


def reference(x, g, h0, logits):
    a = torch.sigmoid(g.double()) if logits else g.double().exp()
    h0 = torch.zeros_like(a[:, 0]) if h0 is None else h0.double()
    h = scan64(a, x.double(), h0)
    s = scan64(a, x.double().abs(), h0.abs())
    return a, h0, h, s, bound64(a, s)


SIZES = [
    (1, 1, 1, 1), (2, 1, 3, 128), (1, 2, 1, 4), (3, 7, 2, 5), (2, 16, 2, 8), (2, 17, 1, 100), (1, 63, 2, 64),
    (1, 64, 2, 64), (2, 65, 3, 36), (1, 130, 1, 33), (2, 513, 2, 99), (1, 1025, 4, 128), (1, 2111, 1, 7),
    (9, 200, 5, 60),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("types", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")], ids=str)
@pytest.mark.parametrize("logits", [False, True])
def test_forward_and_gradients(size, types, logits):
    import gdn_b200
    T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
    x, g, h0, do, dh = make(*size, T[types[0]], T[types[1]], logits, seed=sum(size), h0=size[1] % 2 == 1)
    act = "logsigmoid" if logits else None
    a, h0r, h, s, e = reference(x, g, h0, logits)
    o, hT = gdn_b200.gated_scan(x, g, h0, g_activation=act)
    check("o", o, h, e)
    check("hT", hT, h[:, -1], e[:, -1])
    o32, none = gdn_b200.gated_scan(x, g, h0, g_activation=act, output_dtype=torch.float32, output_final_state=False)
    assert none is None
    check("o32", o32, h, e)

    for out32 in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, g)] + ([h0.clone().requires_grad_()] if h0 is not None else [])
        o, hT = gdn_b200.gated_scan(*leaves[:2], leaves[2] if h0 is not None else None, g_activation=act,
                                    output_dtype=torch.float32 if out32 else None)
        check("o of the recorded call", o, h, e)
        dot = do.to(o.dtype)
        grads = torch.autograd.grad((o, hT), leaves, (dot, dh))
        d = dot.double().clone()
        d[:, -1] += dh.double()
        ar = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
        zero = torch.zeros_like(a[:, 0])
        lam = scan64(ar, d.flip(1), zero).flip(1)
        # do_T and dh_T enter as two terms (a do_T + a dh_T in the maps), so their magnitudes add
        d = dot.double().abs()
        d[:, -1] += dh.double().abs()
        ls = scan64(ar, d.flip(1), zero)
        le = bound64(ar, ls).flip(1)
        ls = ls.flip(1)
        hp = torch.cat([h0r[:, None], h[:, :-1]], 1)
        hpe = torch.cat([zero[:, None], e[:, :-1]], 1)
        mu, mue = a * lam, a * le + EPS * a * ls
        slope = torch.sigmoid(-g.double()) if logits else torch.ones_like(a)
        dg = mu * hp * slope
        dge = (mu.abs() * hpe + mue * hp.abs() + mue * hpe + EPS * (mu * hp).abs()) * slope
        check("dx", grads[0], lam, le)
        check("dg", grads[1], dg, dge)
        if h0 is not None:
            check("dh0", grads[2], mu[:, 0], mue[:, 0])


@pytest.mark.parametrize("logits", [False, True])
def test_gradients_against_differences(logits):
    """L = sum(w o) + sum(w2 h_T) is linear in x and h0 and, in one g_t, linear in a_t.

    A central difference over +-d is off by d^2/6 of the third derivative (at most e^d |dL/dg| for
    exp, |dL/da| / 8 for the sigmoid) and by the outputs' own errors over d."""
    import gdn_b200
    x, g, h0, w, w2 = make(1, 150, 1, 6, torch.float32, torch.float32, logits, seed=3)
    act = "logsigmoid" if logits else None
    leaves = [t.clone().requires_grad_() for t in (x, g, h0)]
    o, hT = gdn_b200.gated_scan(*leaves, g_activation=act)
    dx, dg, dh0 = torch.autograd.grad((o, hT), leaves, (w, w2))

    def parts(x, g, h0):
        o, hT = gdn_b200.gated_scan(x, g, h0, g_activation=act)
        return (w * o).double().sum((1, 2)) + (w2 * hT).double().sum(1)  # one loss per channel

    d = 2.0 ** -5
    for t in (0, 1, 63, 64, 99, 149):
        for n, (leaf, grad) in enumerate(((x, dx), (g, dg))):
            moved = []
            for s in (d, -d):
                m = leaf.clone()
                m[:, t] += s
                args = [x, g, h0]
                args[n] = m
                a, _, h, mag, e = reference(*args, logits)
                moved.append((parts(*args), (w.double().abs() * (e + 2.0 ** -22 * h.abs())).sum((1, 2))
                              + (w2.double().abs() * (e[:, -1] + 2.0 ** -22 * h[:, -1].abs())).sum(1)))
            diff = (moved[0][0] - moved[1][0]) / (2 * d)
            tol = (moved[0][1] + moved[1][1]) / (2 * d) + 1e-5 * grad[:, t, 0].double().abs()
            if n:
                slope = a[:, t, 0] * (1 - a[:, t, 0]) if logits else a[:, t, 0]
                third = grad[:, t, 0].double().abs() * ((1 / slope / 8) if logits else 1.04)
                tol = tol + d * d / 6 * third * 1.1
            assert ((diff - grad[:, t, 0].double()).abs() <= tol).all(), (t, n)


def test_single_gradients_and_broadcast_gates():
    """Only some leaves, only one output's gradient, a gate shared by a head's channels."""
    import gdn_b200
    x, g, h0, do, dh = make(2, 90, 2, 12, seed=4)
    gh = g[..., :1].clone().requires_grad_()
    o, hT = gdn_b200.gated_scan(x, gh.expand_as(x).contiguous(), h0)
    (dgh,) = torch.autograd.grad(o, gh, do.to(o.dtype))
    full = gh.detach().expand_as(x).contiguous().requires_grad_()
    o2, _ = gdn_b200.gated_scan(x, full, h0)
    (dg,) = torch.autograd.grad(o2, full, do.to(o.dtype))
    # a sum of 12 terms in fp32, each half a step off at most per addition
    assert ((dgh - dg.sum(-1, keepdim=True)).abs() <= 24 * 2.0 ** -24 * dg.abs().sum(-1, keepdim=True)).all()
    # the final state's gradient alone equals a zero gradient of o
    xl = x.clone().requires_grad_()
    o, hT = gdn_b200.gated_scan(xl, g, h0)
    (d1,) = torch.autograd.grad(hT, xl, dh, retain_graph=True)
    (d2,) = torch.autograd.grad((o, hT), xl, (torch.zeros_like(o), dh))
    assert torch.equal(d1, d2)
    # the gradient of a sum arrives expanded (stride 0)
    xl = x.clone().requires_grad_()
    o, _ = gdn_b200.gated_scan(xl, g, h0)
    (d3,) = torch.autograd.grad(o.sum(), xl)
    xl2 = x.clone().requires_grad_()
    o, _ = gdn_b200.gated_scan(xl2, g, h0)
    (d4,) = torch.autograd.grad(o, xl2, torch.ones_like(o))
    assert torch.equal(d3, d4)
    # no gradient recorded: no state kept, same values
    with torch.no_grad():
        o5, _ = gdn_b200.gated_scan(xl, g, h0)
    assert not o5.requires_grad and torch.equal(o5, o)


def test_second_derivative_is_refused():
    import gdn_b200
    x, g, h0, do, _ = make(1, 20, 1, 8, torch.float32, seed=4)
    xl = x.requires_grad_()
    (d0,) = torch.autograd.grad(gdn_b200.gated_scan(xl, g, h0)[0], xl, do)
    (d1,) = torch.autograd.grad(gdn_b200.gated_scan(xl, g, h0)[0], xl, do.requires_grad_(), create_graph=True)
    assert torch.equal(d0, d1)
    with pytest.raises(RuntimeError, match="twice"):
        d1.sum().backward()


def test_strides_and_views():
    """Heads cut from a wider tensor, a base that no vector fits, time slices, expanded batches."""
    import gdn_b200
    x, g, h0, _, _ = make(2, 70, 6, 32, seed=5)
    for cut in (lambda t: t[:, :, 1:4], lambda t: t[:, 3:60], lambda t: t[:, ::3], lambda t: t[..., 1:30],
                lambda t: t[:1].expand(2, -1, -1, -1), lambda t: t[:, :, ::2, 4:24]):
        xc, gc = cut(x), cut(g)
        want = gdn_b200.gated_scan(xc.contiguous(), gc.contiguous())
        got = gdn_b200.gated_scan(xc, gc)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        xl, gl = xc.detach().requires_grad_(), gc.detach().requires_grad_()
        xd, gd = xc.contiguous().requires_grad_(), gc.contiguous().requires_grad_()
        one = torch.ones_like(want[0])
        for u, v in zip(torch.autograd.grad(gdn_b200.gated_scan(xl, gl)[0], (xl, gl), one),
                        torch.autograd.grad(gdn_b200.gated_scan(xd, gd)[0], (xd, gd), one)):
            assert torch.equal(u, v)


@pytest.mark.parametrize("size", [(40, 300, 4, 128), (3, 1400, 2, 512), (2, 300, 3, 200)], ids=str)
def test_wide_and_head_first_layouts(size):
    """Many chains, heads wider than a CTA's columns, and storage with the heads before the time."""
    import gdn_b200
    x, g, h0, do, dh = make(*size, seed=9)
    a, h0r, h, s, e = reference(x, g, h0, False)
    want = None
    for first in (lambda t: t, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)):
        xl, gl = first(x).requires_grad_(), first(g).requires_grad_()
        o, hT = gdn_b200.gated_scan(xl, gl, h0)
        check("o", o, h, e)
        check("hT", hT, h[:, -1], e[:, -1])
        got = (o.detach(), hT.detach()) + torch.autograd.grad((o, hT), (xl, gl), (do.to(o.dtype), dh))
        want = want or got
        assert all(torch.equal(u, w) for u, w in zip(got, want))


def test_one_tensor_as_both_inputs():
    import gdn_b200
    z = -torch.rand(1, 80, 1, 64, device="cuda")
    zl = z.clone().requires_grad_()
    (both,) = torch.autograd.grad(gdn_b200.gated_scan(zl, zl)[0].sum(), zl)
    x, g = z.clone().requires_grad_(), z.clone().requires_grad_()
    dx, dg = torch.autograd.grad(gdn_b200.gated_scan(x, g)[0].sum(), (x, g))
    assert torch.equal(both, dx + dg)


def test_resets_and_extreme_gates():
    """-inf resets the chain, 0 keeps it, saturated logits do either; gradients stay finite."""
    import gdn_b200
    x, g, h0, do, dh = make(1, 200, 1, 64, torch.float32, seed=6)
    g[:, 50] = -torch.inf
    g[:, 100:120] = 0
    g[:, 150] = -1e30
    a, h0r, h, s, e = reference(x, g, h0, False)
    o, hT = gdn_b200.gated_scan(x, g, h0)
    check("o", o, h, e)
    assert torch.equal(o[:, 50], x[:, 50]) and torch.equal(o[:, 150], x[:, 150])
    z = torch.where(g == 0, 1000.0, torch.where(g < -1e20, -1000.0, g))
    z[:, 60], z[:, 61] = torch.inf, -torch.inf
    leaves = [x.clone().requires_grad_(), z.clone().requires_grad_()]
    a, _, h, s, e = reference(x, z, h0, True)
    o, hT = gdn_b200.gated_scan(*leaves, h0, g_activation="logsigmoid")
    check("o", o, h, e)
    dx, dz = torch.autograd.grad((o, hT), leaves, (do.to(o.dtype), dh))
    assert torch.isfinite(dx).all() and torch.isfinite(dz).all()
    assert (dz[:, 100:120] == 0).all() and (dz[:, 50] == 0).all() and (dz[:, 60:62] == 0).all()


def test_step_continues_the_sequence():
    import gdn_b200
    for logits in (False, True):
        x, g, h0, _, _ = make(3, 40, 2, 100, g=torch.bfloat16 if logits else torch.float32, logits=logits, seed=7)
        act = "logsigmoid" if logits else None
        want, hT = gdn_b200.gated_scan(x, g, h0, g_activation=act)
        o, state = gdn_b200.gated_scan(x[:, :30], g[:, :30], h0, g_activation=act)
        a, h0r, h, s, e = reference(x, g, h0, logits)
        for t in range(30, 40):
            o = gdn_b200.gated_scan_step(x[:, t], g[:, t], state, g_activation=act)
            check("step", o, h[:, t], e[:, t])
        check("state", state, h[:, -1], e[:, -1])
    with pytest.raises(ValueError, match="in place"):
        gdn_b200.gated_scan_step(x[:, 0], g[:, 0], state.half())
    with pytest.raises(NotImplementedError, match="backward"):
        gdn_b200.gated_scan_step(x[:, 0].clone().requires_grad_(), g[:, 0], state)


def test_repeats_bit_for_bit_and_in_a_graph():
    import gdn_b200
    x, g, h0, do, dh = make(2, 3000, 2, 128, g=torch.bfloat16, logits=True, seed=8)
    do = do.to(x.dtype)
    leaves = [t.clone().requires_grad_() for t in (x, g, h0)]

    def step():
        o, hT = gdn_b200.gated_scan(*leaves, g_activation="logsigmoid")
        return (o.detach(), hT.detach()) + torch.autograd.grad((o, hT), leaves, (do, dh))

    first = step()
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for t in captured:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(first, captured))


def test_streams_at_once():
    import gdn_b200
    sets = [make(2, 2000, 2, 64, seed=20 + i) for i in range(4)]
    want = [gdn_b200.gated_scan(s[0], s[1], s[2]) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(gdn_b200.gated_scan(s[0], s[1], s[2]))
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])


def test_offsets_past_32_bits():
    """A view whose rows lie 2^31 elements apart."""
    import gdn_b200
    far = torch.empty((1 << 31) + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(far, (1, 2, 1, 64), (0, 1 << 31, 64, 1))
    x.copy_(torch.randn(1, 2, 1, 64, device="cuda"))
    g = torch.full((1, 2, 1, 64), -0.5, device="cuda")
    o, hT = gdn_b200.gated_scan(x, g)
    w, wT = gdn_b200.gated_scan(x.contiguous(), g)
    assert torch.equal(o, w) and torch.equal(hT, wT)


def test_first_call_of_a_thread():
    """A thread that has made no CUDA call yet has no current context; a first backward runs on such a thread."""
    import subprocess
    import sys
    import textwrap
    from conftest import ROOT
    code = """
    import sys, threading
    sys.path.insert(0, "v100-attention-lab_b200")
    import torch, gdn_b200
    x = torch.nn.functional.normalize(torch.randn(1, 64, 2, 128, device="cuda"), dim=-1).bfloat16()
    g = -torch.rand(1, 64, 2, 128, device="cuda")
    b = torch.rand(1, 64, 2, device="cuda")
    want = gdn_b200.gated_scan(x, g)[0], gdn_b200.window_attention(x, x, x, 9), gdn_b200.gdn_chunk_fwd(x, x, x, b, -b)[0]
    xl = x.clone().requires_grad_()
    torch.autograd.grad(gdn_b200.gated_scan(xl, g)[0].sum(), xl)
    for i, f in enumerate((lambda: gdn_b200.gated_scan(x, g)[0], lambda: gdn_b200.window_attention(x, x, x, 9),
                           lambda: gdn_b200.gdn_chunk_fwd(x, x, x, b, -b)[0])):
        got = []
        t = threading.Thread(target=lambda: got.append(f()))
        t.start()
        t.join()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[i]), i
    """
    subprocess.run([sys.executable, "-c", textwrap.dedent(code)], check=True, cwd=ROOT, timeout=300)
