"""The gated recurrence with gates near 1, whose memory is thousands of rows.

With eps = 2^-24.  A gate that is near 1 (log decay up to 2^-9 from 0, logits above
4) is one fp32 rounding, half an eps there, and less than eps / 2 more from its
exact value, so that a row's decay is off by eps.  A row's product and sum are
rounded once where the row is computed and once in the map that carries the
state across it (eps each), the map's product of gates once more, and the maps of
warps, tiles and clusters add less than eps per row.  So

    E_t = a_t E_{t-1} + 5 eps S_t,   S_t = a_t S_{t-1} + |x_t|

bounds the error.  Inputs are positive, so that S is the state itself and not a sum
that cancels: a state that loses or repeats a tile is then off by far more
(a tile of 128 rows is 1 % of 9000; the bound is 5 eps T / 2 = 0.13 %).
"""

import pytest
import torch

from test_recurrence_gpu import scan64, stored

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def check(name, got, ref, err):
    assert torch.isfinite(got).all(), name
    off = (got.detach().double() - ref).abs()
    worst = (off / (err * (1 + torch.finfo(got.dtype).eps) + stored(got, ref))).max().item()
    assert worst <= 1, (name, worst)


def bound(a, s):
    return scan64(a, 5 * EPS * s, torch.zeros_like(s[:, 0]))


GATES = ["zero", "-1e-5", "-1e-4..-1e-3", "z 7..14", "z 40"]


def gates(kind, shape, gen):
    r = torch.rand(*shape, device="cuda", generator=gen)
    if kind == "zero":
        return torch.zeros(shape, device="cuda"), False
    if kind == "-1e-5":
        return -1e-5 * (1 + 0.1 * r[:, :1]).expand(shape).contiguous(), False  # constant along the sequence
    if kind == "-1e-4..-1e-3":
        return -torch.exp(torch.log(torch.tensor(1e-4)).item() + 2.3 * r), False
    return (7 + 7 * r, True) if kind == "z 7..14" else (torch.full(shape, 40.0, device="cuda"), True)


@pytest.mark.parametrize("kind", GATES)
@pytest.mark.parametrize("types", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32")], ids=str)
@pytest.mark.parametrize("D", [64, 33])
def test_long_memory(kind, types, D):
    """Forward and gradients over several strides of a cluster, the composed gates still near 1."""
    import gdn_b200
    B, N, H = 1, 9001, 1
    gen = torch.Generator(device="cuda").manual_seed(len(kind) + D)
    g, logits = gates(kind, (B, N, H, D), gen)
    g = g.to(T[types[1]])
    x = (0.5 + torch.rand(B, N, H, D, device="cuda", generator=gen)).to(T[types[0]])
    h0 = 1000 * (1 + torch.rand(B, H, D, device="cuda", generator=gen))
    # gradients small enough that dg, their sum times the state, stays within fp16
    do = (2e-4 * (0.5 + torch.rand(B, N, H, D, device="cuda", generator=gen))).to(T[types[0]])
    dh = 0.2 * (1 + torch.rand(B, H, D, device="cuda", generator=gen))
    a = torch.sigmoid(g.double()) if logits else g.double().exp()
    slope = torch.sigmoid(-g.double()) if logits else torch.ones_like(a)
    h = scan64(a, x.double(), h0.double())
    e = bound(a, h)
    leaves = [t.clone().requires_grad_() for t in (x, g, h0)]
    o, hT = gdn_b200.gated_scan(*leaves, g_activation="logsigmoid" if logits else None, output_dtype=torch.float32)
    check("o", o, h, e)
    check("hT", hT, h[:, -1], e[:, -1])
    dx, dg, dh0 = torch.autograd.grad((o, hT), leaves, (do.float(), dh))
    gdn_b200.check_status()
    d = do.double()
    d[:, -1] += dh.double()
    ar = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    lam = scan64(ar, d.flip(1), torch.zeros_like(d[:, 0]))
    le = bound(ar, lam).flip(1)
    lam = lam.flip(1)
    hp = torch.cat([h0.double()[:, None], h[:, :-1]], 1)
    hpe = torch.cat([torch.zeros_like(e[:, :1]), e[:, :-1]], 1)
    mu, mue = a * lam, a * le + 2 * EPS * a * lam
    check("dx", dx, lam, le)
    # the factor 1 - a: exponential (with its argument's rounding, |z| eps), sum, reciprocal and product
    dge = (mu * hpe + mue * hp + mue * hpe + (2 + (8 + g.double().abs() if logits else 0)) * EPS * mu * hp) * slope
    check("dg", dg, mu * hp * slope, dge)
    check("dh0", dh0, mu[:, 0], mue[:, 0])


@pytest.mark.parametrize("rows", [1, 40])
def test_gates_near_one_are_rounded_once(rows):
    """With x = 0 and h_0 = 1 a row's gate is its output: 2^-25 of rounding below 1, and little more.

    Log decays: g^3 / 6 (2^-29.6) and a rounding of g (2^-33).  Logits above 4: 1 - a is below 0.018 and
    within (10 + z) eps of itself, z < 18.  A constant gate's error counts once per row of memory."""
    import gdn_b200
    n = 1 << 16
    for logits, g in ((False, -(2.0 ** -(9 + 20 * torch.rand(n, device="cuda")))), (True, 4.01 + 13.9 * torch.rand(n, device="cuda"))):
        gates = torch.full((1, rows, 1, n), 1e3 if logits else 0.0, device="cuda")  # the other rows keep the state
        gates[:, 0] = g
        o, _ = gdn_b200.gated_scan(torch.zeros_like(gates), gates, torch.ones(1, 1, n, device="cuda"),
                                   g_activation="logsigmoid" if logits else None)
        ref = torch.sigmoid(g.double()) if logits else g.double().exp()
        more = (28 * EPS * (1 - ref) if logits else 2.0 ** -29.5)
        worst = ((o[0, -1, 0].double() - ref).abs() / (2.0 ** -25 + more)).max().item()
        assert worst <= 1, (logits, worst)
