"""Windowed attention at the ends of its types' ranges: one key far above the
rest, values whose plain sum would pass fp32, infinities that a row sees.

Tolerances as in test_windowed_gpu.py, but for what a probability may lose: fp16
has a grid of 2^-24 below 2^-14, so one that is stored times 2^s, as a share of
the largest, is off by half a step (2^-11) of itself or by 2^-25-s, whichever is
more; the two terms of the single-token form by 2^-25-s at most.  s is 11 in
the prompt kernel and 14 in the single-token one.  Each key counts that times the
largest value; a subnormal output adds 2^-25.
"""

import math

import pytest
import torch

from test_windowed_gpu import TYPES, attention64, compare, half_step, make, slot, visible

pytestmark = pytest.mark.gpu


def tolerance(o, mag, reach, dt, D, n, scale, vmax, step):
    u = half_step(dt)
    e = (D + 4) * 2.0 ** -23 * reach * scale + 2.0 ** -20
    tol = ((2.0 ** -16 if step else u) + 2 * e + n * 2.0 ** -23) * mag + u * o.abs() + torch.finfo(dt).smallest_normal * u
    if dt == torch.float16:
        tol = tol + n * vmax * (2.0 ** -39 if step else 2.0 ** -36)
    return tol * (1 + 2 * u)


def sink_above(B, S, HK, H, D, gap, dt, seed):
    """Queries for which key 0 scores ``gap`` (nats) above the others' mean; its value is 0, theirs are positive."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    scale = 1 / math.sqrt(D)
    q, k = 0.3 * r(B, S, H, D), 0.3 * r(B, S, HK, D)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:, 0] = 0.0
    k[:, 0, :, 0] = gap / (8.0 * scale)
    v = 0.5 + r(B, S, HK, D).abs()
    v[:, 0] = 0.0
    return q.to(dt), k.to(dt), v.to(dt)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("gap", [10.0, 14.5, 15.0, 17.0, 18.0])
@pytest.mark.parametrize("D,H,HK", [(64, 2, 1), (128, 3, 3)])
def test_a_sink_far_above_the_window(dt, gap, D, H, HK):
    import gdn_b200
    S, window, sinks = 1300, 1024, 1
    q, k, v = sink_above(1, S, HK, H, D, gap, TYPES[dt], 3)
    o = gdn_b200.window_attention(q, k, v, window, sinks)
    gdn_b200.check_status()
    scale = 1 / math.sqrt(D)
    ref, mag, reach = attention64(q[0], k[0], v[0], visible(S, S, window, sinks, S), scale)
    vmax = v.abs().max().item()
    compare("o", o[0], ref, tolerance(ref, mag, reach, q.dtype, D, window + sinks, scale, vmax, False))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("gap", [10.0, 14.5, 15.0, 17.0, 18.0])
@pytest.mark.parametrize("D,H,HK", [(64, 2, 1), (128, 20, 2)])
def test_a_sink_far_above_the_window_one_token(dt, gap, D, H, HK):
    import gdn_b200
    window, sinks = 1024, 1
    cap = window + sinks
    q, k, v = sink_above(1, cap, HK, H, D, gap, TYPES[dt], 4)
    kc, vc = k.clone(), v.clone()
    p = cap - 1
    pos = torch.tensor([p], dtype=torch.int32, device="cuda")
    kc[:, p], vc[:, p] = float("nan"), float("nan")
    o = gdn_b200.window_attention_step(q[:, p], k[:, p], v[:, p], kc, vc, pos, window, sinks)
    scale = 1 / math.sqrt(D)
    see = torch.ones(1, cap, dtype=torch.bool, device="cuda")
    ref, mag, reach = attention64(q[0, p:], k[0], v[0], see, scale)
    tol = tolerance(ref, mag, reach, q.dtype, D, cap, scale, v.abs().max().item(), True)
    compare("o", o, ref, tol)


def near_the_end(size):
    """Values up to 3e38 and scores that rise along the keys, so that a running reference lags behind the maximum."""
    S, H, HK, D, window, sinks = size
    q, k, v = make(1, S, S, H, HK, D, torch.bfloat16, 5)
    q, k = q.abs(), (k.abs() * torch.linspace(0.1, 1, S, device="cuda")[None, :, None, None]).bfloat16()
    v = (3e38 * (1 - 0.1 * torch.rand(1, S, HK, D, device="cuda"))).bfloat16()
    return q, k, v, attention64(q[0], k[0], v[0], visible(S, S, window, sinks, S), 1 / math.sqrt(D))


END = [(300, 2, 1, 64, 200, 4), (700, 2, 2, 128, 5000, 0)]


@pytest.mark.parametrize("size", END, ids=str)
def test_bf16_values_near_the_end_of_the_range(size):
    """Averages of values up to 3e38 are finite, whatever the sum of the unnormalised terms would be."""
    import gdn_b200
    S, H, HK, D, window, sinks = size
    q, k, v, (ref, mag, reach) = near_the_end(size)
    o = gdn_b200.window_attention(q, k, v, window, sinks)
    gdn_b200.check_status()
    compare("o", o[0], ref, tolerance(ref, mag, reach, q.dtype, D, min(S, window + sinks), 1 / math.sqrt(D), 3e38, False))


@pytest.mark.parametrize("size", END, ids=str)
def test_bf16_values_near_the_end_of_the_range_one_token(size):
    import gdn_b200
    S, H, HK, D, window, sinks = size
    q, k, v, (ref, mag, reach) = near_the_end(size)
    cap, p = window + sinks, S - 1
    kc, vc = (torch.zeros(1, cap, HK, D, device="cuda", dtype=q.dtype) for _ in range(2))
    for j in list(range(min(sinks, p))) + list(range(max(0, p - window + 1), p)):
        kc[:, slot(j, cap, sinks)], vc[:, slot(j, cap, sinks)] = k[:, j], v[:, j]
    pos = torch.tensor([p], dtype=torch.int32, device="cuda")
    o = gdn_b200.window_attention_step(q[:, p], k[:, p], v[:, p], kc, vc, pos, window, sinks)
    n = min(S, window + sinks)
    compare("o", o, ref[p:], tolerance(ref[p:], mag[p:], reach[p:], q.dtype, D, n, 1 / math.sqrt(D), 3e38, True))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("size", [(2, 4, 2, 64, 20, 2), (1, 20, 1, 128, 700, 4), (3, 6, 2, 128, 90, 0)], ids=str)
def test_infinities_that_one_token_sees(dt, size):
    """inf and -inf come out as such, both or a NaN as NaN, in their columns and heads alone."""
    import gdn_b200
    B, H, HK, D, window, sinks = size
    cap = window + sinks + 3
    q, k, v = make(B, 1, 1, H, HK, D, TYPES[dt], 6)
    kc, vc = make(B, cap, cap, HK, HK, D, TYPES[dt], 7)[1:]
    p = 3 * cap + 1
    seen = list(range(sinks)) + list(range(p - window + 1, p + 1))
    slots = [slot(j, cap, sinks) for j in seen]
    hidden = sorted(set(range(cap)) - set(slots))
    pos = torch.full((B,), p, dtype=torch.int32, device="cuda")
    clean = gdn_b200.window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, pos, window, sinks)
    inf = float("inf")
    vc[:, hidden] = float("nan")
    v[:, 0, 0, 9], v[:, 0, 0, 21] = inf, inf          # the token's own value
    vc[:, slots[0], 0, 5] = inf
    vc[:, slots[3], 0, 6], vc[:, slots[-2], 0, 6] = -inf, -inf
    vc[:, slots[4], 0, 7], vc[:, slots[-3], 0, 7] = inf, -inf
    vc[:, slots[5], 0, 8] = float("nan")
    vc[:, slots[1], 0, 21] = -inf
    o = gdn_b200.window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, pos, window, sinks)
    G = H // HK
    assert torch.equal(o[:, G:], clean[:, G:])
    rest = [d for d in range(D) if d not in (5, 6, 7, 8, 9, 21)]
    assert torch.equal(o[..., rest], clean[..., rest])
    got = o[:, :G]
    assert (got[..., 5] == inf).all() and (got[..., 9] == inf).all()
    assert (got[..., 6] == -inf).all()
    assert got[..., [7, 8, 21]].isnan().all()


def test_scores_that_are_not_finite_one_token():
    """A NaN or infinite query or key makes NaN of the heads that meet it, and of no others."""
    import gdn_b200
    B, H, HK, D, window, sinks = 2, 40, 2, 64, 300, 2
    cap = window + sinks
    q, k, v = make(B, 1, 1, H, HK, D, torch.bfloat16, 8)
    kc, vc = make(B, cap, cap, HK, HK, D, torch.bfloat16, 9)[1:]
    pos = torch.full((B,), cap - 1, dtype=torch.int32, device="cuda")
    clean = gdn_b200.window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, pos, window, sinks)
    q[0, 0, 3], q[0, 0, 18, 5] = float("nan"), float("nan")  # two heads of key head 0, in either group of 16
    kc[1, 150, 1, 7] = float("nan")                           # all heads of key head 1
    vc[0, 100, 0, 9] = float("inf")
    o = gdn_b200.window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, pos, window, sinks)
    bad = torch.zeros(B, H, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[0, 18] = True
    bad[1, 20:] = True
    assert o[bad].isnan().all()
    want = clean.clone()
    want[0, :20, 9] = float("inf")
    assert torch.equal(o[~bad], want[~bad])
