"""What is measured of the recurrent and windowed operators: cases, inputs, the
plain form of each operator and its definition in 64 bits.

Kinds of a case (``op``):
  scan        gated_scan forward:  h_t = a_t h_{t-1} + x_t
  scan_train  gated_scan forward and backward (gradients of x, g and h0)
  scan_step   gated_scan_step: one token, the state updated in place
  win         window_attention over a prompt or a chunk of one
  win_step    window_attention_step: one token against a ring cache
  gdn_step    gdn_step: one token of the Gated DeltaNet recurrence

``run`` calls the framework where ``own`` is true, and elementary torch
operations in 32 bits where it is false.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # a batch of requests, one token each, through one recurrent layer of 2048 channels; gates as logits
        dict(name="scan_step_b64", op="scan_step", B=64, H=16, D=128, x="bf16", gt="bf16", act=True),
        # the forward benchmark's shape (2 x 4096 tokens, 16 heads of 128), log decays in fp32
        dict(name="scan_2x4096", op="scan", B=2, T=4096, H=16, D=128, x="bf16", gt="f32", act=False),
        # one very long document (the long-sequence configuration), gate logits as a projection leaves them
        dict(name="scan_1x65536", op="scan", B=1, T=65536, H=16, D=128, x="bf16", gt="bf16", act=True),
        # a training step's recurrence: gate logits in the projections' type
        dict(name="scan_train_8x2048", op="scan_train", B=8, T=2048, H=16, D=128, x="bf16", gt="bf16", act=True),
        # odd everything: channels that fill no vector, a length that fills no tile, fp32
        dict(name="scan_train_3x1531", op="scan_train", B=3, T=1531, H=5, D=99, x="f32", gt="f32", act=False),
        # a prompt of the forward benchmark's shape, every head with its own keys
        dict(name="win_2x4096", op="win", B=2, T=4096, S=4096, H=16, HK=16, D=128, x="bf16", window=1024, sinks=4,
             ragged=False),
        # a long prompt with shared key heads and a wide window
        dict(name="win_1x16384", op="win", B=1, T=16384, S=16384, H=32, HK=8, D=128, x="f16", window=4096, sinks=64,
             ragged=False),
        # one chunk of a padded batch of prompts: odd lengths, shared heads of 64, some rows beyond their sequence
        dict(name="win_chunk_3x501", op="win", B=3, T=501, S=2777, H=12, HK=4, D=64, x="bf16", window=700, sinks=4,
             ragged=True),
        # one token of one request: latency
        dict(name="win_step_b1", op="win_step", B=1, H=16, HK=4, D=128, x="bf16", cap=1028, window=1024, sinks=4),
        # one token each of a full batch, the rings wrapped many times
        dict(name="win_step_b64", op="win_step", B=64, H=32, HK=8, D=128, x="bf16", cap=4160, window=4096, sinks=4),
        # one token of one request through one GDN layer: latency
        dict(name="gdn_step_b1", op="gdn_step", B=1, H=16, x="bf16", act=True),
        # one token each of a full batch
        dict(name="gdn_step_b128", op="gdn_step", B=128, H=32, x="bf16", act=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan_step", "scan", "scan", "scan_train", "win", "win", "win_step", "win_step", "gdn_step"])
    if op == "gdn_step":
        return dict(op=op, B=_log(rng, 1, 128), H=rng.choice([1, 2, 8, 16, 32]), x=rng.choice(["bf16", "f16"]),
                    act=rng.random() < 0.5)
    if op in ("scan", "scan_train", "scan_step"):
        x = rng.choice(["bf16", "bf16", "f16", "f32"])
        c = dict(op=op, B=_log(rng, 1, 64 if op == "scan_step" else 8), H=rng.randint(1, 16),
                 D=rng.choice([64, 128, 128, rng.randint(1, 160)]), x=x, gt=rng.choice(["f32", x]),
                 act=rng.random() < 0.5)
        if op != "scan_step":
            most = (1 << 24 if op == "scan_train" else 1 << 26) // (c["B"] * c["H"] * c["D"])
            c["T"] = _log(rng, 1, max(2, min(65536, most)))
        return c
    x = rng.choice(["bf16", "f16"])
    HK = rng.choice([1, 2, 4, 8])
    H = HK * rng.choice([1, 2, 3, 4, 8])
    D = rng.choice([64, 128, 128])
    window, sinks = _log(rng, 16, 4096), rng.choice([0, 1, 4, 64])
    if op == "win_step":
        return dict(op=op, B=_log(rng, 1, 64), H=H, HK=HK, D=D, x=x, cap=window + sinks + rng.choice([0, 1, 60]),
                    window=window, sinks=sinks)
    B = _log(rng, 1, 4)
    T = _log(rng, 1, max(2, min(16384, (16384 * 32) // (B * H))))
    S = T + rng.choice([0, 0, rng.randint(1, 2000)])
    return dict(op=op, B=B, T=T, S=S, H=H, HK=HK, D=D, x=x, window=window, sinks=sinks, ragged=rng.random() < 0.4)


def _pairs(c):
    """Visible (row, key) pairs of one head, summed over full sequences."""
    S, T, w, s = c["S"], c["T"], c["window"], c["sinks"]
    p = torch.arange(S - T, S, dtype=torch.int64)
    first = (p - w + 1).clamp(min=0)
    return c["B"] * int((p - first + 1 + torch.minimum(first, torch.tensor(s))).sum())


def work(case):
    c = case
    op = c["op"]
    if op == "gdn_step":
        n = c["B"] * c["H"]
        return {"bytes": n * (2 * 128 * 128 * 4 + 4 * 128 * 2 + 8), "flops": n * 7 * 128 * 128}
    if op in ("scan", "scan_train", "scan_step"):
        n = c["B"] * c["H"] * c["D"]
        sx, sg = _SIZE[c["x"]], _SIZE[c["gt"]]
        if op == "scan_step":
            return {"bytes": n * (2 * sx + sg + 8), "flops": 3 * n}
        e = n * c["T"]
        if op == "scan":
            return {"bytes": e * (2 * sx + sg) + 8 * n, "flops": 3 * e}
        # x, g, do in; o, dx, dg out; h0, dh_T in; h_T, dh0 out
        return {"bytes": e * (4 * sx + 2 * sg) + 16 * n, "flops": 10 * e}
    s = _SIZE[c["x"]]
    if op == "win_step":
        n = c["window"] + c["sinks"]
        b = c["B"] * (2 * c["HK"] * n * c["D"] + 2 * c["H"] * c["D"] + 2 * c["HK"] * c["D"]) * s
        return {"bytes": b, "flops": 4 * c["B"] * c["H"] * n * c["D"]}
    keys = c["S"] if c["S"] - c["T"] <= c["window"] else c["T"] + c["window"] + c["sinks"]
    b = c["B"] * (2 * c["H"] * c["T"] + 2 * c["HK"] * min(keys, c["S"])) * c["D"] * s
    return {"bytes": b, "flops": 4 * c["H"] * c["D"] * _pairs(c)}


def _inputs(case, seed):
    """All inputs of a case as tensors on the GPU, from the seed alone."""
    c, op = case, case["op"]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    dt = _TYPES[c["x"]]
    st = {"case": dict(c)}
    if op == "gdn_step":
        B, H = c["B"], c["H"]
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)
        st["q"], st["k"], st["v"] = unit(rand(B, H, 128)).to(dt), unit(rand(B, H, 128)).to(dt), rand(B, H, 128).to(dt)
        st["beta"], st["g"] = rand(B, H), rand(B, H) + 2.0
        if not c["act"]:
            st["beta"] = torch.sigmoid(st["beta"])
            st["g"] = torch.nn.functional.logsigmoid(st["g"])
        st["state"] = 0.1 * rand(B, H, 128, 128)
        return st
    if op in ("scan", "scan_train", "scan_step"):
        shape = (c["B"], c["H"], c["D"]) if op == "scan_step" else (c["B"], c["T"], c["H"], c["D"])
        z = rand(*shape) + 2.0
        if not c["act"]:
            z = -torch.log1p(torch.exp(-z))
        st["g"] = z.to(_TYPES[c["gt"]])
        del z
        st["x"] = rand(*shape).to(dt)
        h = rand(c["B"], c["H"], c["D"])
        if op == "scan_step":
            st["state"] = h
            return st
        st["h0"] = h
        if op == "scan_train":
            st["do"], st["dh"] = rand(*shape).to(dt), rand(c["B"], c["H"], c["D"])
            for n in ("x", "g", "h0"):
                st[n].requires_grad_(True)
        return st
    B, H, HK, D = c["B"], c["H"], c["HK"], c["D"]
    if op == "win":
        st["q"] = rand(B, c["T"], H, D).to(dt)
        st["k"], st["v"] = rand(B, c["S"], HK, D).to(dt), rand(B, c["S"], HK, D).to(dt)
        st["lengths"] = None
        if c["ragged"]:
            lo = max(0, c["S"] - c["T"] - 1)
            st["lengths"] = torch.randint(lo, c["S"] + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
        return st
    st["q"], st["k"], st["v"] = rand(B, H, D).to(dt), rand(B, HK, D).to(dt), rand(B, HK, D).to(dt)
    st["k_cache"], st["v_cache"] = rand(B, c["cap"], HK, D).to(dt), rand(B, c["cap"], HK, D).to(dt)
    # every request is past its window, most past their ring's end
    st["positions"] = torch.randint(c["window"] + c["sinks"], 9 * c["cap"], (B,), device="cuda", generator=gen,
                                    dtype=torch.int32)
    return st


def prepare(case, seed):
    if own:
        path = os.path.join(_ROOT, "v100-attention-lab_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
    return _inputs(case, seed)


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    import gdn_b200 as fw
    c = st["case"]
    op = c["op"]
    act = "logsigmoid" if c.get("act") else None
    if op == "gdn_step":
        o = fw.gdn_step(st["q"], st["k"], st["v"], st["beta"], st["g"], st["state"], g_activation=act,
                        beta_activation="sigmoid" if act else None)
        return {"o": o, "state": st["state"]}
    if op == "scan_step":
        o = fw.gated_scan_step(st["x"], st["g"], st["state"], g_activation=act)
        return {"o": o, "state": st["state"]}
    if op == "scan":
        o, h = fw.gated_scan(st["x"], st["g"], st["h0"], g_activation=act)
        return {"o": o, "h": h}
    if op == "scan_train":
        o, h = fw.gated_scan(st["x"], st["g"], st["h0"], g_activation=act)
        dx, dg, dh0 = torch.autograd.grad((o, h), (st["x"], st["g"], st["h0"]), (st["do"], st["dh"]))
        return {"o": o.detach(), "h": h.detach(), "dx": dx, "dg": dg, "dh0": dh0}
    if op == "win":
        return {"o": fw.window_attention(st["q"], st["k"], st["v"], c["window"], c["sinks"], lengths=st["lengths"])}
    o = fw.window_attention_step(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["positions"],
                                 c["window"], c["sinks"])
    return {"o": o, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


# ---------------------------------------------------------------- plain forms


def _scan_plain(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 1 by doubling, from h = 0 (both overwritten)."""
    T, s = x.shape[1], 1
    while s < T:
        x[:, s:] = x[:, s:] + a[:, s:] * x[:, :-s]
        a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return x


def _decay(g, act):
    g = g.detach().float()
    return 1.0 / (1.0 + torch.exp(-g)) if act else torch.exp(g)


def _run_plain(st):
    c = st["case"]
    op = c["op"]
    if op == "gdn_step":
        g, beta = st["g"], st["beta"]
        a = _decay(g, c["act"])[..., None, None]
        if c["act"]:
            beta = 1.0 / (1.0 + torch.exp(-beta))
        q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
        h = a * st["state"]
        u = beta[..., None] * (v - (h * k[..., None, :]).sum(-1))
        h = h + u[..., :, None] * k[..., None, :]
        st["state"].copy_(h)
        return {"o": (h * q[..., None, :]).sum(-1).to(st["q"].dtype), "state": st["state"]}
    if op == "scan_step":
        h = _decay(st["g"], c["act"]) * st["state"] + st["x"].float()
        st["state"].copy_(h)
        return {"o": h.to(st["x"].dtype), "state": st["state"]}
    if op in ("scan", "scan_train"):
        a = _decay(st["g"], c["act"])
        x = st["x"].detach().float().clone()
        h0 = st["h0"].detach()
        x[:, 0] += a[:, 0] * h0
        h = _scan_plain(a.clone() if op == "scan_train" else a, x)
        out = {"o": h.to(st["x"].dtype), "h": h[:, -1].clone()}
        if op == "scan":
            return out
        # lambda_t = do_t + a_{t+1} lambda_{t+1}: the same recurrence, backwards in time
        lam = st["do"].float().flip(1)
        lam[:, 0] += st["dh"]
        ar = torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1)
        lam = _scan_plain(ar, lam).flip(1)
        mu = a * lam
        dg = mu * torch.cat([h0[:, None], h[:, :-1]], 1)
        if c["act"]:
            dg = dg * (1.0 - a)
        return out | {"dx": lam.to(st["x"].dtype), "dg": dg.to(st["g"].dtype), "dh0": mu[:, 0].clone()}
    H, HK, D, w, s = c["H"], c["HK"], c["D"], c["window"], c["sinks"]
    G = H // HK
    scale = 1.0 / math.sqrt(D)
    if op == "win":
        q, k, v = st["q"], st["k"], st["v"]
        B, T, S = c["B"], c["T"], c["S"]
        o = torch.empty_like(q)
        length = st["lengths"] if st["lengths"] is not None else torch.full((B,), S, device=q.device)
        for i in range(0, T, 512):
            n = min(512, T - i)
            p = torch.arange(S - T + i, S - T + i + n, device=q.device)
            first = max(0, S - T + i - w + 1)
            end = S - T + i + n
            j = torch.arange(first, end, device=q.device)
            if s and first:
                j = torch.cat([torch.arange(min(s, first), device=q.device), j])
            kj, vj = k[:, j].float(), v[:, j].float()
            qi = q[:, i:i + n].float().view(B, n, HK, G, D)
            see = (j <= p[:, None]) & ((p[:, None] - j < w) | (j < s))
            see = see[None] & (j < length[:, None])[:, None] & (p < length[:, None])[:, :, None]
            z = torch.einsum("bnhgd,bjhd->bhgnj", qi, kj) * scale
            z = z.masked_fill(~see[:, None, None], -math.inf)
            m = z.amax(-1, keepdim=True).clamp(min=-1e30)
            e = torch.exp(z - m)
            y = torch.einsum("bhgnj,bjhd->bnhgd", e, vj)
            y = y / e.sum(-1).clamp(min=1e-30).permute(0, 3, 1, 2)[..., None]
            o[:, i:i + n] = y.reshape(B, n, H, D).to(q.dtype)
        return {"o": o}
    B, cap, pos = c["B"], c["cap"], st["positions"].long()
    slot = torch.where(pos < cap, pos, s + (pos - s) % (cap - s))
    rows = torch.arange(B, device=pos.device)
    st["k_cache"][rows, slot] = st["k"]
    st["v_cache"][rows, slot] = st["v"]
    j = torch.arange(cap, device=pos.device)
    # the newest position that each slot can hold
    last = torch.where(j < s, j, j + torch.div(pos[:, None] - j, cap - s, rounding_mode="floor") * (cap - s))
    see = torch.where(j < s, j <= pos[:, None], (last >= s) & (pos[:, None] - last < w))
    q = st["q"].float().view(B, HK, G, D)
    z = torch.einsum("bhgd,bjhd->bjhg", q, st["k_cache"].float()) * scale
    z = z.masked_fill(~see[:, :, None, None], -math.inf)
    e = torch.exp(z - z.amax(1, keepdim=True))
    o = torch.einsum("bjhg,bjhd->bhgd", e, st["v_cache"].float()) / e.sum(1)[..., None]
    return {"o": o.reshape(B, H, D).to(st["q"].dtype), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


# ---------------------------------------------------------------- definitions in 64 bits


def exact(case, seed):
    """What ``run`` returns for fresh inputs, step by step and row by row in 64 bits."""
    c, op = case, case["op"]
    st = _inputs(case, seed)
    f = lambda n: st[n].detach().double()
    gate = lambda: torch.sigmoid(f("g")) if c["act"] else f("g").exp()
    if op == "gdn_step":
        beta = torch.sigmoid(f("beta")) if c["act"] else f("beta")
        h = f("state") * gate()[:, :, None, None]
        u = (f("v") - torch.matmul(h, f("k").unsqueeze(-1)).squeeze(-1)) * beta.unsqueeze(-1)
        h = torch.baddbmm(h.flatten(0, 1), u.flatten(0, 1).unsqueeze(2), f("k").flatten(0, 1).unsqueeze(1)).view_as(h)
        return {"o": torch.matmul(h, f("q").unsqueeze(-1)).squeeze(-1), "state": h}
    if op == "scan_step":
        h = torch.addcmul(f("x"), gate(), f("state"))
        return {"o": h, "state": h}
    if op in ("scan", "scan_train"):
        B, T, H, D = st["x"].shape
        n = B * T * H * D
        if n > 1 << 28:
            return None
        a, hs, h = gate(), torch.empty(B, T, H, D, dtype=torch.float64, device="cuda"), f("h0")
        x = st["x"].detach()
        for t in range(T):
            h = torch.addcmul(x[:, t].double(), a[:, t], h, out=hs[:, t])
        out = {"o": hs, "h": h}
        if op == "scan":
            return out
        do, mu = st["do"], f("dh")
        dx, dg = torch.empty_like(hs), torch.empty_like(hs)
        for t in range(T - 1, -1, -1):
            lam = torch.add(do[:, t].double(), mu, out=dx[:, t])
            before = hs[:, t - 1] if t else f("h0")
            mu = a[:, t] * lam
            torch.mul(mu, before, out=dg[:, t])
        if c["act"]:
            dg *= torch.sigmoid(-f("g"))
        return out | {"dx": dx, "dg": dg, "dh0": mu}
    H, HK, D, w, s, B = c["H"], c["HK"], c["D"], c["window"], c["sinks"], c["B"]
    G = H // HK
    if op == "win":
        T, S = c["T"], c["S"]
        if 4 * H * D * _pairs(c) > 4e12:
            return None
        o = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
        step = 128
        for b in range(B):
            L = S if st["lengths"] is None else int(st["lengths"][b])
            for t0 in range(0, T, step):
                t1 = min(T, t0 + step, L - (S - T))  # rows at or behind the sequence's end stay zero
                if t1 <= t0:
                    continue
                p = torch.arange(S - T + t0, S - T + t1, device="cuda")
                lo = max(0, int(p[0]) - w + 1)
                js = torch.cat([torch.arange(0, min(s, lo), device="cuda"),
                                torch.arange(lo, min(L, int(p[-1]) + 1), device="cuda")])
                hide = (js[None] > p[:, None]) | ((p[:, None] - js[None] >= w) & (js[None] >= s))
                for hk in range(HK):
                    q = st["q"][b, t0:t1, hk * G:(hk + 1) * G].double().transpose(0, 1)
                    z = q @ st["k"][b, js, hk].double().T / math.sqrt(D)
                    z[:, hide] = -math.inf
                    o[b, t0:t1, hk * G:(hk + 1) * G] = (torch.softmax(z, -1) @ st["v"][b, js, hk].double()).transpose(0, 1)
        return {"o": o}
    cap = c["cap"]
    o = torch.empty(B, H, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        p = int(st["positions"][b])
        seen = list(range(min(s, p + 1)))
        seen += list(range(max(len(seen), p - w + 1), p))
        slots = torch.tensor([j if j < cap else s + (j - s) % (cap - s) for j in seen], device="cuda", dtype=torch.long)
        k = torch.cat([st["k_cache"][b, slots], st["k"][b][None]]).double()
        v = torch.cat([st["v_cache"][b, slots], st["v"][b][None]]).double()
        q = st["q"][b].double().view(HK, G, D)
        z = torch.einsum("hgd,jhd->hgj", q, k) / math.sqrt(D)
        o[b] = torch.einsum("hgj,jhd->hgd", torch.softmax(z, -1), v).reshape(H, D)
    return {"o": o, "k_cache": None, "v_cache": None}
