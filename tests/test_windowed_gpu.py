"""Windowed attention with sinks, and the single-token operators, against their
definitions in 64 bits.

Tolerances.  u is half a step of the operands' type.  Every probability is off by
at most u (its rounding for the second product) plus e, the error of its exponent
and exponential: (D + 4) 2^-23 of |q| max|k| scale for a score summed in fp32, and
2^-20 for the exponential and the running rescalings.  The numerator is then off
by (u + 2 e + n 2^-23) sum_j w_j |v_j|, with n the keys summed in fp32, and the
output's own rounding adds u |o|.  fp16 adds 2^-24 of max |v| per key for
probabilities below its normal range.  In the single-token form the
probabilities keep two terms, so u^2 (and nothing below the normal range but
2^-48) takes the place of u.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def visible(T, S, window, sinks, length, device="cuda"):
    p = torch.arange(S - T, S, device=device)[:, None]
    j = torch.arange(S, device=device)[None]
    return (j <= p) & (j < length) & ((p - j < window) | (j < sinks)) & (p < length)


def attention64(q, k, v, see, scale):
    """One sequence: q [T, H, D], k, v [S, HK, D], see [T, S] -> o, sum_j w_j |v_j|, |q| max|k| per row."""
    T, H, D = q.shape
    G = H // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    o, mag, reach = (torch.zeros(T, H, D, dtype=torch.float64, device=q.device) for _ in range(3))
    for h in range(H):
        kh, vh = k[:, h // G], v[:, h // G]
        z = (q[:, h] @ torch.where(see.any(0)[:, None], kh, 0).T) * scale
        w = torch.softmax(z.masked_fill(~see, -math.inf), -1)
        w = torch.where(see, w, 0)
        vz = torch.where(see.any(0)[:, None], vh, 0)
        o[:, h], mag[:, h] = w @ vz, w @ vz.abs()
        kn = torch.where(see.any(0), kh.norm(dim=-1), 0)
        reach[:, h] = (q[:, h].norm(dim=-1, keepdim=True) * kn.max()).expand(-1, D)
    return o, mag, reach


def tolerance(o, mag, reach, dt, D, n, scale, vmax, two_terms=False):
    u = half_step(dt)
    e = (D + 4) * 2.0 ** -23 * reach * scale + 2.0 ** -20
    tol = ((u * u if two_terms else u) + 2 * e + n * 2.0 ** -23) * mag + u * o.abs() + torch.finfo(dt).smallest_normal * u
    if dt == torch.float16:
        tol = tol + n * vmax * (2.0 ** -48 if two_terms else 2.0 ** -24)
    return tol * (1 + 2 * u)


def compare(name, got, o, tol):
    assert torch.isfinite(got).all(), name
    worst = ((got.double() - o).abs() / tol).max().item()
    assert worst <= 1, (name, worst)


def make(B, T, S, H, HK, D, dt, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dt)
    return r(B, T, H, D), r(B, S, HK, D), r(B, S, HK, D)


# B, T, S, H, HK, D, window, sinks
SIZES = [
    (1, 1, 1, 1, 1, 128, 1, 0),
    (1, 1, 200, 2, 1, 128, 64, 4),
    (2, 7, 7, 3, 1, 64, 3, 0),
    (1, 63, 63, 2, 2, 128, 1000, 0),
    (1, 128, 128, 1, 1, 128, 128, 1),
    (1, 129, 129, 2, 2, 64, 128, 4),
    (2, 130, 257, 4, 2, 128, 100, 5),
    (1, 257, 400, 3, 3, 128, 129, 128),
    (1, 500, 500, 6, 2, 64, 1, 130),
    (2, 513, 1100, 8, 2, 128, 300, 4),
    (1, 777, 777, 5, 1, 128, 4096, 0),
    (1, 1030, 1030, 2, 1, 64, 127, 300),
    (1, 640, 3000, 2, 1, 128, 1500, 64),
    (1, 300, 333, 2, 1, 64, 1, 10000),
    (2, 70, 4000, 1, 1, 128, 3, 65),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_window_attention(size, dt):
    import gdn_b200
    B, T, S, H, HK, D, window, sinks = size
    q, k, v = make(B, T, S, H, HK, D, TYPES[dt], sum(size))
    scale = 1 / math.sqrt(D)
    o = gdn_b200.window_attention(q, k, v, window, sinks)
    gdn_b200.check_status()
    for b in range(B):
        ref, mag, reach = attention64(q[b], k[b], v[b], visible(T, S, window, sinks, S), scale)
        tol = tolerance(ref, mag, reach, q.dtype, D, min(S, window + sinks), scale, v.abs().max().item())
        compare("o", o[b], ref, tol)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("sizes", [(3, 300, 300, 4, 2, 128, 90, 4), (4, 200, 450, 3, 1, 64, 150, 0)], ids=str)
def test_padded_batches(dt, fill, sizes):
    """Keys and queries behind each sequence's end hold anything; those rows are 0."""
    import gdn_b200
    B, T, S, H, HK, D, window, sinks = sizes
    q, k, v = make(B, T, S, H, HK, D, TYPES[dt], 5)
    lengths = torch.tensor([S, 0, S - T + 129, S - 1][:B], dtype=torch.int32, device="cuda")
    for b in range(B):
        n = int(lengths[b])
        k[b, n:], v[b, n:] = fill, fill
        q[b, max(0, n - (S - T)):] = fill
    o = gdn_b200.window_attention(q, k, v, window, sinks, lengths=lengths, scale=0.2)
    gdn_b200.check_status()
    for b in range(B):
        n = int(lengths[b])
        live = max(0, n - (S - T))
        assert (o[b, live:] == 0).all()
        if live:
            see = visible(T, S, window, sinks, n)[:live]
            ref, mag, reach = attention64(q[b, :live], k[b], v[b], see, 0.2)
            vmax = v[b, :n].abs().max().item()
            compare("o", o[b, :live], ref, tolerance(ref, mag, reach, q.dtype, D, min(S, window + sinks), 0.2, vmax))


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("what", ["nan", "inf", "-inf", "mixed", "key"])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(dt, what):
    import gdn_b200
    B, T, S, H, HK, D, window, sinks = 1, 700, 700, 4, 2, 128, 200, 6
    q, k, v = make(B, T, S, H, HK, D, TYPES[dt], 9)
    clean = gdn_b200.window_attention(q, k, v, window, sinks)
    at = [8, 129, 391, 699]
    fills = {"nan": [float("nan")] * 4, "inf": [float("inf")] * 4, "-inf": [-float("inf")] * 4,
             "mixed": [float("inf"), -float("inf"), float("nan"), float("inf")], "key": [float("nan")] * 4}[what]
    for j, f in zip(at, fills):
        (k if what == "key" else v)[0, j, 0, 5] = f
    o = gdn_b200.window_attention(q, k, v, window, sinks)
    gdn_b200.check_status()
    see = visible(T, S, window, sinks, S)
    ref, mag, reach = attention64(q[0], torch.nan_to_num(k[0]), torch.nan_to_num(v[0], 0, 0, 0), see, 1 / math.sqrt(D))
    tol = tolerance(ref, mag, reach, q.dtype, D, window + sinks, 1 / math.sqrt(D), 8.0)
    hit = see[:, at]  # [T, 4]
    touched = hit.any(1)
    for h in range(H):
        got = o[0, :, h]
        if h // 2 == 1:  # the other key head
            assert torch.equal(got, clean[0, :, h])
            continue
        compare("untouched", got[~touched], ref[~touched, h], tol[~touched, h])
        if what == "key":
            assert torch.isnan(got[touched]).all()
            continue
        rest = [d for d in range(D) if d != 5]
        compare("other columns", got[:, rest], ref[:, h][:, rest], tol[:, h][:, rest])
        f = torch.tensor(fills, device="cuda")
        pos = (hit & (f == math.inf)).any(1)
        neg = (hit & (f == -math.inf)).any(1)
        nan = (hit & f.isnan()).any(1) | (pos & neg)
        col = got[:, 5]
        assert torch.equal(col.isnan(), nan)
        assert torch.equal(col == math.inf, pos & ~nan) and torch.equal(col == -math.inf, neg & ~nan)


def test_many_items_per_cta_with_poisoned_ones():
    """More work items than SMs, some of them done twice: each as if it were alone, bit for bit."""
    import gdn_b200
    B, T, H, HK, D = 10, 900, 8, 8, 64
    q, k, v = make(B, T, T, H, HK, D, torch.bfloat16, 12)
    for b, j, h in ((0, 899, 0), (3, 450, 2), (3, 451, 2), (7, 0, 5), (9, 130, 7)):
        v[b, j, h, j % D] = float("nan") if j % 2 else float("inf")
    k[5, 600, 1] = float("nan")
    o = gdn_b200.window_attention(q, k, v, 170, 3)
    gdn_b200.check_status()
    for b in range(B):
        one = gdn_b200.window_attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], 170, 3)
        assert torch.equal(one[0].view(torch.int16), o[b].view(torch.int16)), b


def test_large_scores_and_growing_maxima():
    """Scores that rise along the keys move the running reference again and again."""
    import gdn_b200
    B, T, S, H, HK, D = 1, 600, 600, 2, 2, 128
    q, k, v = make(B, T, S, H, HK, D, torch.float16, 3)
    q, k = q.abs(), (k.abs() * torch.linspace(0.1, 3, S, device="cuda")[None, :, None, None]).half()
    o = gdn_b200.window_attention(q, k, v, 400, 3)
    ref, mag, reach = attention64(q[0], k[0], v[0], visible(T, S, 400, 3, S), 1 / math.sqrt(D))
    compare("o", o[0], ref, tolerance(ref, mag, reach, q.dtype, D, 403, 1 / math.sqrt(D), v.abs().max().item()))


def test_strided_views():
    import gdn_b200
    B, T, H, D = 2, 150, 4, 64
    packed = torch.randn(B, T, H + 4, D, device="cuda").bfloat16()
    q, k, v = packed[:, :, :H], packed[:, :, H:H + 2], packed[:, :, H + 2:]
    want = gdn_b200.window_attention(q.contiguous(), k.contiguous(), v.contiguous(), 40, 2)
    assert torch.equal(gdn_b200.window_attention(q, k, v, 40, 2), want)
    head_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(gdn_b200.window_attention(head_first, k, v, 40, 2), want)
    with pytest.raises(ValueError, match="16-byte"):
        gdn_b200.window_attention(packed.flatten()[4:4 + B * T * D].view(B, T, 1, D), k[:, :, :1], v[:, :, :1], 40)


# ------------------------------------------------------------------ one token
def slot(j, cap, sinks):
    return j if j < cap else sinks + (j - sinks) % (cap - sinks)


# B, H, HK, D, window, sinks, spare slots, tokens
STEPS = [
    (1, 1, 1, 128, 1, 0, 0, 4),
    (2, 4, 4, 64, 5, 2, 0, 20),
    (1, 8, 1, 128, 16, 4, 1, 60),
    (3, 6, 2, 128, 33, 1, 7, 100),
    (2, 24, 1, 64, 40, 0, 0, 90),
    (1, 20, 2, 128, 17, 64, 3, 120),
]


@pytest.mark.parametrize("size", STEPS, ids=str)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_window_step_by_step(size, dt):
    """Every token of a sequence, from an uninitialised (NaN) cache past several turns of the ring."""
    import gdn_b200
    B, H, HK, D, window, sinks, spare, n = size
    cap = window + sinks + spare
    q, k, v = make(B, n, n, H, HK, D, TYPES[dt], sum(size))
    kc, vc = (torch.full((B, cap, HK, D), float("nan"), device="cuda", dtype=q.dtype) for _ in range(2))
    scale = 1 / math.sqrt(D)
    full = [attention64(q[b], k[b], v[b], visible(n, n, window, sinks, n), scale) for b in range(B)]
    late = torch.arange(B, device="cuda", dtype=torch.int32) * 3  # sequences start apart
    for t in range(n + 3 * B):
        pos = t - late
        pos = torch.where(pos < n, pos, -1).to(torch.int32)
        i = pos.clamp(min=0).long()
        rows = torch.arange(B, device="cuda")
        before = kc.clone(), vc.clone()
        o = gdn_b200.window_attention_step(q[rows, i], k[rows, i], v[rows, i], kc, vc, pos, window, sinks)
        for b in range(B):
            p = int(pos[b])
            if p < 0:
                assert (o[b] == 0).all()
                assert torch.equal(kc[b].view(torch.int16), before[0][b].view(torch.int16))
                assert torch.equal(vc[b].view(torch.int16), before[1][b].view(torch.int16))
                continue
            s = slot(p, cap, sinks)
            before[0][b, s], before[1][b, s] = k[b, p], v[b, p]
            assert torch.equal(kc[b].view(torch.int16), before[0][b].view(torch.int16))
            assert torch.equal(vc[b].view(torch.int16), before[1][b].view(torch.int16))
            ref, mag, reach = (x[p] for x in full[b])
            tol = tolerance(ref, mag, reach, q.dtype, D, window + sinks, scale, v.abs().max().item(), two_terms=True)
            compare((b, p), o[b], ref, tol)


@pytest.mark.parametrize("size", [(1, 16, 4, 128, 1024, 4), (2, 8, 8, 64, 2000, 64), (16, 32, 4, 128, 515, 0)], ids=str)
def test_window_step_long(size):
    import gdn_b200
    B, H, HK, D, window, sinks = size
    cap = window + sinks + 5
    q, k, v = make(B, 1, 1, H, HK, D, torch.bfloat16, 1)
    kc, vc = make(B, cap, cap, HK, HK, D, torch.bfloat16, 2)[1:]
    pos = torch.randint(0, 9 * cap, (B,), device="cuda", dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    o = gdn_b200.window_attention_step(q[:, 0], k[:, 0], v[:, 0], kc, vc, pos, window, sinks)
    for b in range(B):
        p = int(pos[b])
        seen = list(range(min(sinks, p + 1)))
        seen += list(range(max(len(seen), p - window + 1), p + 1))
        idx = torch.tensor([slot(j, cap, sinks) for j in seen], device="cuda")
        see = torch.ones(1, len(seen), dtype=torch.bool, device="cuda")
        ref, mag, reach = attention64(q[b], kc[b, idx], vc[b, idx], see, 1 / math.sqrt(D))
        tol = tolerance(ref, mag, reach, q.dtype, D, len(seen), 1 / math.sqrt(D), 8.0, two_terms=True)
        compare(b, o[b][None], ref, tol)


def test_window_step_cache_views_past_32_bits():
    """A cache cut out of a pool: slots 2^31 elements apart, a head stride of its own."""
    import gdn_b200
    D, window = 64, 2
    far = torch.zeros((1 << 31) + (1 << 10), dtype=torch.bfloat16, device="cuda")
    view = torch.as_strided(far, (1, 2, 1, D), (1 << 31, 1 << 31, 128, 1))
    q, k, v = make(1, 3, 3, 2, 1, D, torch.bfloat16, 4)
    vc = torch.zeros(1, 2, 1, D, device="cuda", dtype=torch.bfloat16)
    near, vn = torch.zeros_like(vc), torch.zeros_like(vc)
    for p in range(3):
        pos = torch.tensor([p], dtype=torch.int32, device="cuda")
        a = gdn_b200.window_attention_step(q[:, p], k[:, p], v[:, p], view, vc, pos, window)
        b = gdn_b200.window_attention_step(q[:, p], k[:, p], v[:, p], near, vn, pos, window)
        assert torch.equal(a, b) and torch.equal(view, near)


# ------------------------------------------------------------------ gdn_step
@pytest.mark.parametrize("BH", [(1, 1), (2, 3), (5, 16)], ids=str)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("prep", [False, True])
def test_gdn_step(BH, dt, prep):
    """Sums of 128 terms in fp32: 2^-24 per term and a few more of each magnitude."""
    import gdn_b200
    B, H = BH
    gen = torch.Generator(device="cuda").manual_seed(7)
    r = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    q, k, v = (r(B, H, 128).to(TYPES[dt]) for _ in range(3))
    if not prep:
        q, k = (torch.nn.functional.normalize(t.float(), dim=-1).to(t.dtype) for t in (q, k))
    beta, g, state = r(B, H), r(B, H), r(B, H, 128, 128)
    if not prep:
        beta, g = beta.sigmoid(), torch.nn.functional.logsigmoid(g)
    kw = dict(use_qk_l2norm_in_kernel=True, beta_activation="sigmoid", g_activation="logsigmoid") if prep else {}
    for g_arg in (g, None):
        if g_arg is None and prep:
            kw["g_activation"] = None
        s0 = state.clone()
        o = gdn_b200.gdn_step(q, k, v, beta, g_arg, s0, scale=0.7, output_dtype=torch.float32, **kw)
        s1 = state.clone()
        o16 = gdn_b200.gdn_step(q, k, v, beta, g_arg, s1, scale=0.7, **kw)
        assert torch.equal(s0, s1) and torch.equal(o16, o.to(q.dtype))
        Q, K, V, b = q.double(), k.double(), v.double(), beta.double()
        a = torch.ones_like(b) if g_arg is None else (torch.sigmoid(g.double()) if prep else g.double().exp())
        if prep:
            Q, K = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (Q, K))
            b = b.sigmoid()
        h = a[..., None, None] * state.double()
        hk = (h * K[..., None, :]).sum(-1)
        u = b[..., None] * (V - hk)
        new = h + u[..., None] * K[..., None, :]
        ref = 0.7 * (new * Q[..., None, :]).sum(-1)
        e = 150 * 2.0 ** -24  # 128 terms, the decay (4), the norms of q and k (128 / 2 terms under a root, and 4)
        e = 2 * e if prep else e
        hka = (h.abs() * K.abs()[..., None, :]).sum(-1)
        ue = e * b[..., None] * (V.abs() + hka)
        newe = e * h.abs() + (ue + e * u.abs())[..., None] * K.abs()[..., None, :]
        kq = (K.abs() * Q.abs()).sum(-1, keepdim=True)
        oe = 0.7 * (e * (h.abs() * Q.abs()[..., None, :]).sum(-1) + (ue + e * u.abs()) * kq)
        assert ((s0.double() - new).abs() <= newe + 2.0 ** -24 * new.abs()).all()
        assert ((o.double() - ref).abs() <= oe + 2.0 ** -24 * ref.abs()).all()


def test_gdn_step_strided_heads():
    import gdn_b200
    x = torch.randn(3, 6, 3, 128, device="cuda").half()
    q, k, v = (x[:, 1:5, i] for i in range(3))
    beta, g = torch.rand(3, 9, device="cuda")[:, 2:6], -torch.rand(3, 9, device="cuda")[:, 2:6]
    s0 = torch.randn(3, 4, 128, 128, device="cuda")
    s1 = s0.clone()
    o0 = gdn_b200.gdn_step(q, k, v, beta, g, s0)
    o1 = gdn_b200.gdn_step(*(t.contiguous() for t in (q, k, v, beta, g)), s1)
    assert torch.equal(o0, o1) and torch.equal(s0, s1)


# ------------------------------------------------------------------ together
def test_prompt_then_tokens_through_all_mixers():
    """A stack's three mixers: a prompt through the long forms, then token by token, as in serving.

    Each token's output must match the long form over the whole sequence: the GDN forward within its
    own bar (1e-3 of the largest output, plus bf16 storage), the others within one step of bf16."""
    import gdn_b200
    from gpu_util import make as make_gdn
    from gpu_util import STORE_ROUNDING, TOL
    B, P, N, H, HK, D, window, sinks = 2, 200, 12, 4, 2, 128, 64, 4
    T = P + N
    q, k, v, beta, g, h0 = make_gdn(B, T, H, seed=11, dtype=torch.bfloat16, h0_std=0.1)
    kk, vk = k[:, :, :HK].contiguous(), v[:, :, :HK].contiguous()
    z = torch.randn(B, T, H, D, device="cuda") + 2
    with torch.no_grad():
        full = (gdn_b200.gdn_chunk_fwd(q, k, v, beta, g, initial_state=h0)[0],
                gdn_b200.gated_scan(v, z, g_activation="logsigmoid")[0],
                gdn_b200.window_attention(q, kk, vk, window, sinks))
        cap = window + sinks + 3
        _, S = gdn_b200.gdn_chunk_fwd(q[:, :P], k[:, :P], v[:, :P], beta[:, :P], g[:, :P], initial_state=h0)
        _, h = gdn_b200.gated_scan(v[:, :P], z[:, :P], g_activation="logsigmoid")
        kc, vc = (torch.full((B, cap, HK, D), float("nan"), device="cuda", dtype=q.dtype) for _ in range(2))
        keep = list(range(sinks)) + list(range(P - window, P))
        slots = [slot(j, cap, sinks) for j in keep]
        kc[:, slots], vc[:, slots] = kk[:, keep], vk[:, keep]

        def token(t, pos):
            return (gdn_b200.gdn_step(q[:, t], k[:, t], v[:, t], beta[:, t], g[:, t], S),
                    gdn_b200.gated_scan_step(v[:, t], z[:, t], h, g_activation="logsigmoid"),
                    gdn_b200.window_attention_step(q[:, t], kk[:, t], vk[:, t], kc, vc, pos, window, sinks))

        for t in range(P, T):
            got = token(t, torch.full((B,), t, dtype=torch.int32, device="cuda"))
            bars = (TOL + 2 * STORE_ROUNDING[torch.bfloat16], 2.0 ** -7, 2.0 ** -7)
            for name, a, b, bar in zip(("gdn", "scan", "window"), got, full, bars):
                b = b[:, t]
                assert (a.float() - b.float()).abs().max() <= bar * b.float().abs().max(), (name, t)


def test_steps_in_a_graph():
    """One captured token, replayed along a sequence: positions move on the device."""
    import gdn_b200
    B, H, HK, D, window, sinks, n = 2, 4, 2, 128, 20, 2, 70
    cap = window + sinks
    q, k, v = make(B, n, n, H, HK, D, torch.bfloat16, 2)
    want_k, want_v = (torch.zeros(B, cap, HK, D, device="cuda", dtype=q.dtype) for _ in range(2))
    want = [gdn_b200.window_attention_step(q[:, t], k[:, t], v[:, t], want_k, want_v,
                                           torch.full((B,), t, dtype=torch.int32, device="cuda"), window, sinks)
            for t in range(n)]
    kc, vc = torch.zeros_like(want_k), torch.zeros_like(want_v)
    qs, ks, vs = (torch.zeros_like(t[:, 0]) for t in (q, k, v))
    pos = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pos += 1
        out = gdn_b200.window_attention_step(qs, ks, vs, kc, vc, pos, window, sinks)
    pos.fill_(-1)
    kc.zero_(), vc.zero_()
    for t in range(n):
        qs.copy_(q[:, t]), ks.copy_(k[:, t]), vs.copy_(v[:, t])
        graph.replay()
        assert torch.equal(out, want[t]), t
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_window_attention_repeats_streams_and_graph():
    import gdn_b200
    sets = [make(1, 900, 900, 4, 2, 128, torch.bfloat16, s) for s in range(3)]
    want = [gdn_b200.window_attention(*s, 300, 4) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(gdn_b200.window_attention(*s, 300, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gdn_b200.window_attention(*sets[0], 300, 4)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want[0])
    gdn_b200.check_status()
