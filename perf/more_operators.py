"""A feed-forward block of experts on quantized weights: the choice of each token's experts, their gate and up
projections with the activation, and their down projection with the weighted sum and the residual.

listed() names the cases, draw() gives more of the same ranges, prepare() builds what a program holds before a call
(expert weights in device memory, activations, the routing of the step), run() is one pass, work() the bytes and
operations no pass can do without, exact() the results in 64 bits.  With `own` false run() is plain torch; with it true
it calls the package's entry points.

An expert tensor is [experts][rows][blocks], rows of GGUF blocks.  Products take the activation as the format's 8-bit
codes (Q8_0 blocks of 32 for q8_0, Q8_K blocks of 256 for the K formats), as the dense projections do.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
UNIT = {"q8_0": (32, 34), "q4_k": (256, 144), "q5_k": (256, 176), "q6_k": (256, 210)}
GGML = {"q8_0": 8, "q4_k": 12, "q5_k": 13, "q6_k": 14}


def listed():
    return [
        # one token's choice among many small experts: the smallest call, where latency is all
        dict(name="route_m1", kind="route", experts=128, top=8, m=1, score="softmax", bias=False, groups=1, top_groups=1,
             best=1, norm=True, scale=1.0, masked=0.0),
        # a prefill chunk routed by sigmoid scores with a bias for balance, four of eight groups of experts a token
        dict(name="route_groups_m4096", kind="route", experts=256, top=8, m=4096, score="sigmoid", bias=True, groups=8,
             top_groups=4, best=2, norm=True, scale=2.5, masked=0.0),
        # a ragged batch with some experts switched off for some tokens, for padding tokens all of them
        dict(name="route_masked_m777", kind="route", experts=60, top=4, m=777, score="softmax", bias=False, groups=1,
             top_groups=1, best=1, norm=False, scale=1.0, masked=0.3),
        # one user's token through the eight of 128 small experts that it chose
        dict(name="gate_up_m1", kind="gate_up", type="q4_k", experts=128, top=8, m=1, n_embd=2560, n_ff=768, bias=False,
             f="silu"),
        # three users of a model of eight large experts
        dict(name="gate_up_large_m3", kind="gate_up", type="q4_k", experts=8, top=2, m=3, n_embd=4096, n_ff=14336,
             bias=False, f="silu"),
        # forty tokens of a small model with biases
        dict(name="gate_up_small_m40", kind="gate_up", type="q8_0", experts=32, top=4, m=40, n_embd=576, n_ff=1536,
             bias=True, f="gelu"),
        # a prompt's chunk: 32 tokens an expert
        dict(name="gate_up_m512", kind="gate_up", type="q4_k", experts=128, top=8, m=512, n_embd=2560, n_ff=768,
             bias=False, f="silu"),
        # a long prompt's chunk: 256 tokens an expert, bound by the products
        dict(name="gate_up_m4096", kind="gate_up", type="q4_k", experts=128, top=8, m=4096, n_embd=2560, n_ff=768,
             bias=False, f="silu"),
        # the way back for one user's token
        dict(name="down_m1", kind="down", type="q6_k", experts=128, top=8, m=1, n_embd=2560, n_ff=768, bias=False,
             residual=True),
        # twelve users of the eight large experts
        dict(name="down_large_m12", kind="down", type="q4_k", experts=8, top=2, m=12, n_embd=4096, n_ff=14336, bias=False,
             residual=True),
        # a ragged prompt through experts with biases, five bits a weight
        dict(name="down_m333", kind="down", type="q5_k", experts=64, top=6, m=333, n_embd=2560, n_ff=1024, bias=True,
             residual=False),
        # the way back of the long chunk
        dict(name="down_m4096", kind="down", type="q6_k", experts=128, top=8, m=4096, n_embd=2560, n_ff=768, bias=False,
             residual=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "gate_up", "gate_up", "down", "down"])
    m = _log_int(rng, 1, 4096)
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = max(2, _log_int(rng, 4, 256) // groups)
        top_groups = rng.randint(1, groups)
        return dict(kind=kind, experts=groups * per, top=rng.randint(1, min(10, top_groups * per)), m=m,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups,
                    top_groups=top_groups, best=rng.choice([1, 2]), norm=rng.random() < 0.6,
                    scale=rng.choice([1.0, 1.0, 2.5]), masked=rng.choice([0.0, 0.0, 0.2]))
    t = rng.choice(sorted(UNIT))
    unit = UNIT[t][0]
    experts = _log_int(rng, 4, 256)
    top = rng.randint(1, min(10, experts))

    def rows(lo, hi, whole):
        n = _log_int(rng, lo, hi)
        return unit * max(1, round(n / unit)) if whole else n

    # the rows that the product contracts over are whole blocks; what it gives may be of any length
    n_embd = rows(256, 4096, kind == "gate_up")
    # at most the weights of eight large experts, and the operations of the longest chunk
    n_ff = rows(256, max(300, min(14336, 8 * 14336 * 4096 // (experts * n_embd))), kind == "down")
    m = min(m, max(1, 4096 * 8 * 2560 * 768 // (top * n_embd * n_ff)))
    c = dict(kind=kind, type=t, experts=experts, top=top, m=m, n_embd=n_embd, n_ff=n_ff, bias=rng.random() < 0.4)
    if kind == "gate_up":
        return dict(c, f=rng.choice(["silu", "silu", "gelu"]))
    return dict(c, residual=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEV)


def _half(t):
    return t.to(torch.float16).view(torch.uint8)


def _blocks(qt, rows, n, std, g):
    """Rows of blocks as a quantizer writes them: codes near a bell, block scales that vary by a factor of two, minima
    that centre the block, and the variance of a trained projection."""
    if qt == "q8_0":
        nb = n // 32
        q = (_normal((rows, nb, 32), g) * 42).round_().clamp_(-127, 127).to(torch.int8)
        d = std / 42 * (0.7 + 0.7 * torch.rand((rows, nb, 1), generator=g, device=DEV))
        return torch.cat([_half(d), q.view(torch.uint8)], 2).view(rows, -1)
    nb = n // 256
    if qt in ("q4_k", "q5_k"):
        top, spread = (15, 2.9) if qt == "q4_k" else (31, 5.8)
        sc = torch.randint(24, 64, (rows, nb, 8), generator=g, device=DEV)
        mn = (sc + torch.randint(-4, 5, (rows, nb, 8), generator=g, device=DEV)).clamp_(0, 63)
        q = (_normal((rows, nb, 4, 2, 32), g) * spread + top / 2).round_().clamp_(0, top).to(torch.uint8)
        d = std / (spread * 43) * (0.7 + 0.7 * torch.rand((rows, nb, 1), generator=g, device=DEV))
        head = torch.cat([sc[..., :4] | (sc[..., 4:] >> 4 << 6), mn[..., :4] | (mn[..., 4:] >> 4 << 6),
                          (sc[..., 4:] & 15) | ((mn[..., 4:] & 15) << 4)], 2).to(torch.uint8)
        parts = [_half(d), _half(top / 2 * d), head]
        if qt == "q5_k":
            fifth = torch.zeros((rows, nb, 32), dtype=torch.uint8, device=DEV)
            for j in range(8):
                fifth |= (q[:, :, j // 2, j % 2] >> 4) << j
            parts.append(fifth)
            q = q & 15
        return torch.cat(parts + [(q[:, :, :, 0] | (q[:, :, :, 1] << 4)).view(rows, nb, 128)], 2).view(rows, -1)
    sc = torch.randint(40, 128, (rows, nb, 16), generator=g, device=DEV)
    sc = sc * (1 - 2 * torch.randint(0, 2, (rows, nb, 16), generator=g, device=DEV))
    q = ((_normal((rows, nb, 2, 4, 32), g) * 10).round_().clamp_(-32, 31) + 32).to(torch.uint8)
    d = std / (10 * 87) * (0.7 + 0.7 * torch.rand((rows, nb, 1), generator=g, device=DEV))
    ql = torch.cat([(q[:, :, :, 0] & 15) | (q[:, :, :, 2] << 4), (q[:, :, :, 1] & 15) | (q[:, :, :, 3] << 4)], 3)
    qh = (q[:, :, :, 0] >> 4) | (q[:, :, :, 1] >> 4 << 2) | (q[:, :, :, 2] >> 4 << 4) | (q[:, :, :, 3] >> 4 << 6)
    return torch.cat([ql.reshape(rows, nb, 128), qh.reshape(rows, nb, 64), sc.to(torch.int8).view(torch.uint8),
                      _half(d)], 2).view(rows, -1)


def _experts(qt, experts, rows, n, g):
    unit, size = UNIT[qt]
    total = experts * rows
    out = torch.empty((total, n // unit * size), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // n)
    for r in range(0, total, step):
        k = min(step, total - r)
        out[r:r + k] = _blocks(qt, k, n, 1 / math.sqrt(n), g)
    return out.view(experts, rows, -1)


def _scores(case, g):
    """Router scores: a bell, some experts more popular than others; masked experts of a token at minus infinity, for
    some tokens every expert."""
    m, n = case["m"], case["experts"]
    s = _normal((m, n), g) + 0.5 * _normal((1, n), g)
    off = case.get("masked", 0.0)
    if off:
        dead = torch.rand((m, n), generator=g, device=DEV) < off
        dead |= torch.rand((m, 1), generator=g, device=DEV) < off / 4
        s = s.masked_fill(dead, -math.inf)
    return s


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "edgexpu-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import edgexpu_amd

    edgexpu_amd.hip().check(edgexpu_amd.hip().init(torch.cuda.current_device()), "init")
    return edgexpu_amd


def _inputs(case, seed):
    g = _gen(seed)
    s = dict(case=case, scores=_scores(case, g))
    if case["kind"] == "route":
        s["bias"] = 0.1 * _normal((case["experts"],), g) if case["bias"] else None
        return s
    t, e, h, f, m, k = (case[n] for n in ("type", "experts", "n_embd", "n_ff", "m", "top"))
    if case["kind"] == "gate_up":
        big = (torch.rand((1, h), generator=g, device=DEV) < 0.01).float() * 7 + 1
        s.update(x=_normal((m, h), g) * big, gate=_experts(t, e, f, h, g), up=_experts(t, e, f, h, g),
                 b_gate=0.1 * _normal((e, f), g) if case["bias"] else None,
                 b_up=0.1 * _normal((e, f), g) if case["bias"] else None)
        return s
    a = _normal((m, k, f), g)
    s.update(act=a / (1 + torch.exp(-a)) * _normal((m, k, f), g), down=_experts(t, e, h, f, g),
             bias=0.1 * _normal((e, h), g) if case["bias"] else None,
             residual=_normal((m, h), g) if case["residual"] else None)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    product = case["kind"] != "route"
    if own:
        E = s["E"] = _package()
        s["plan"] = E.MoePlan(case["experts"], case["top"], case["m"], case["n_embd"] if product else 32,
                              case["n_ff"] if product else 32)
        if product:  # the products of a step follow its routing
            E.moe_route(s["plan"], s["scores"])
    elif product:
        s["ids"], s["weights"] = _route(s["scores"], None, dict(case, score="softmax", groups=1, norm=True, scale=1.0))
    return s


# ------------------------------------------------------------------ plain forms


def _route(scores, bias, case):
    """The choice in 64 bits, where values next to a border decide; weights rounded once."""
    m, n = scores.shape
    s = scores.to(torch.float64)
    live = torch.isfinite(s)
    if case["score"] == "sigmoid":
        p = torch.where(live, 1 / (1 + torch.exp(-s)), 0.0)
    else:
        s = s.masked_fill(~live, -math.inf)
        top = s.amax(1, keepdim=True)
        e = torch.where(live, torch.exp(s - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
        total = e.sum(1, keepdim=True)
        p = e / torch.where(total > 0, total, 1.0)
    c = p if bias is None else p + bias.to(torch.float64)
    c = c.masked_fill(~(live & torch.isfinite(c)), -math.inf)
    if case["groups"] > 1:
        k = case["groups"]
        g = c.view(m, k, n // k).sort(dim=2, descending=True)[0][..., :case["best"]]
        rank = torch.where(torch.isinf(g), 0.0, g).sum(2).masked_fill(torch.isinf(g[..., 0]), -math.inf)
        stay = rank.sort(dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        keep = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, stay, True)
        c = c.masked_fill(~keep.repeat_interleave(n // k, 1), -math.inf)
    v, ids = c.sort(dim=1, descending=True, stable=True)
    v, ids = v[:, :case["top"]], ids[:, :case["top"]]
    none = torch.isinf(v)
    w = p.gather(1, ids).masked_fill(none, 0.0)
    if case["norm"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    return ids.to(torch.int32).masked_fill(none, -1), (w * case["scale"]).to(torch.float32)


def _f32(b):
    return b.contiguous().view(torch.float16).to(torch.float32)


def _unpack32(qt, w, n):
    """[rows, n] weights of uint8 rows in 32 bits."""
    rows = w.shape[0]
    if qt == "q8_0":
        b = w.view(rows, n // 32, 34)
        return (_f32(b[..., :2]) * b[..., 2:].contiguous().view(torch.int8).to(torch.float32)).view(rows, n)
    nb = n // 256
    if qt == "q6_k":
        b = w.view(rows, nb, 210)
        ql, qh = b[..., :128].view(rows, nb, 2, 2, 32), b[..., 128:192].view(rows, nb, 2, 32)
        q = torch.stack([(ql[:, :, :, 0] & 15) | ((qh & 3) << 4), (ql[:, :, :, 1] & 15) | ((qh >> 2 & 3) << 4),
                         (ql[:, :, :, 0] >> 4) | ((qh >> 4 & 3) << 4), (ql[:, :, :, 1] >> 4) | (qh >> 6 << 4)], 3)
        q = q.view(rows, nb, 16, 16).to(torch.float32) - 32
        sc = b[..., 192:208].contiguous().view(torch.int8).to(torch.float32)
        return ((_f32(b[..., 208:]) * sc).unsqueeze(3) * q).view(rows, n)
    b = w.view(rows, nb, UNIT[qt][1])
    lo, mid, hi = b[..., 4:8], b[..., 8:12], b[..., 12:16]
    sc = torch.cat([lo & 63, (hi & 15) | (lo >> 6 << 4)], 2).to(torch.float32)
    mn = torch.cat([mid & 63, (hi >> 4) | (mid >> 6 << 4)], 2).to(torch.float32)
    qs = b[..., -128:].view(rows, nb, 4, 1, 32)
    q = torch.cat([qs & 15, qs >> 4], 3).view(rows, nb, 8, 32)
    if qt == "q5_k":
        bit = torch.arange(8, device=DEV, dtype=torch.uint8).view(1, 1, 8, 1)
        q = q | ((b[..., 16:48].unsqueeze(2) >> bit & 1) << 4)
    d, dm = _f32(b[..., :2]), _f32(b[..., 2:4])
    return ((d * sc).unsqueeze(3) * q.to(torch.float32) - (dm * mn).unsqueeze(3)).view(rows, n)


def _div(a, b):
    """a / b in 32 bits, rounded once."""
    return (a.to(torch.float64) / b.to(torch.float64)).to(torch.float32)


def _codes32(qt, x):
    """The activation as the product sees it: the format's 8-bit codes times the block's scale."""
    unit = UNIT[qt][0]
    b = x.reshape(-1, unit)
    top = b.abs().amax(1, keepdim=True)
    full = torch.full_like(top, 127.0)
    inv = torch.where(top > 0, _div(full, torch.where(top > 0, top, 1.0)), 0.0)
    q = (b * inv).round().clamp_(-127, 127)
    if qt == "q8_0":
        d = _div(top, full).to(torch.float16).to(torch.float32)
    else:
        d = torch.where(top > 0, _div(torch.ones_like(inv), torch.where(top > 0, inv, 1.0)), 0.0)
    return (q * d).view(x.shape)


def _by_expert(ids, experts):
    """(expert, its pairs): the pairs sorted by their expert, those of none left out."""
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat + 1, minlength=experts + 1).tolist()
    at = counts[0]
    for e in range(experts):
        if counts[e + 1]:
            yield e, order[at:at + counts[e + 1]]
        at += counts[e + 1]


def _plain_gate_up(s):
    c = s["case"]
    t, k, n = c["type"], c["top"], c["n_embd"]
    a = _codes32(t, s["x"])
    act = torch.zeros((c["m"] * k, c["n_ff"]), device=DEV)
    for e, pairs in _by_expert(s["ids"], c["experts"]):
        rows = a[pairs // k]
        g, u = rows @ _unpack32(t, s["gate"][e], n).t(), rows @ _unpack32(t, s["up"][e], n).t()
        if s["b_gate"] is not None:
            g, u = g + s["b_gate"][e], u + s["b_up"][e]
        if c["f"] == "silu":
            f = g / (1 + torch.exp(-g))
        else:
            f = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
        act[pairs] = f * u
    return act.view(c["m"], k, -1)


def _plain_down(s):
    c = s["case"]
    t, m, k, n = c["type"], c["m"], c["top"], c["n_ff"]
    a = _codes32(t, s["act"]).view(m * k, n)
    y = torch.zeros((m * k, c["n_embd"]), device=DEV)
    for e, pairs in _by_expert(s["ids"], c["experts"]):
        r = a[pairs] @ _unpack32(t, s["down"][e], n).t()
        if s["bias"] is not None:
            r = r + s["bias"][e]
        y[pairs] = r * s["weights"].view(-1)[pairs].unsqueeze(1)
    out = y.view(m, k, -1).sum(1)
    return out if s["residual"] is None else out + s["residual"]


# ------------------------------------------------------------------ a pass


def run(s):
    c = s["case"]
    if c["kind"] == "route":
        if own:
            return s["E"].moe_route(s["plan"], s["scores"], score=c["score"], bias=s["bias"], n_groups=c["groups"],
                                    top_groups=c["top_groups"], group_best=c["best"], normalise=c["norm"],
                                    scale=c["scale"])
        return _route(s["scores"], s["bias"], c)
    if c["kind"] == "gate_up":
        if own:
            return s["E"].moe_gate_up(s["plan"], s["gate"], s["up"], GGML[c["type"]], s["x"], b_gate=s["b_gate"],
                                      b_up=s["b_up"], activation=c["f"])
        return _plain_gate_up(s)
    if own:
        return s["E"].moe_down(s["plan"], s["down"], GGML[c["type"]], s["act"], bias=s["bias"], residual=s["residual"])
    return _plain_down(s)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    m, k, n = case["m"], case["top"], case["experts"]
    if case["kind"] == "route":
        # two exponentials' worth of arithmetic a score, one comparison a score and choice
        return {"bytes": 4 * m * n + 8 * m * k + (4 * n if case["bias"] else 0), "flops": m * n * (20 + k)}
    # the experts that m tokens reach when each takes k of n at random
    reached = n * (1 - (1 - k / n) ** m)
    unit, size = UNIT[case["type"]]
    h, f = case["n_embd"], case["n_ff"]
    if case["kind"] == "gate_up":
        w = 2 * f * (h // unit * size + (4 if case["bias"] else 0))
        return {"bytes": int(reached * w) + 4 * m * h + 4 * m * k * f + 4 * m * k, "flops": 4 * m * k * h * f}
    w = h * (f // unit * size + (4 if case["bias"] else 0))
    return {"bytes": int(reached * w) + 4 * m * k * f + 4 * m * h * (2 if case["residual"] else 1) + 8 * m * k,
            "flops": 2 * m * k * h * f}


# ------------------------------------------------------------------ the results in 64 bits


def _exact_route(scores, bias, case):
    """Token by token on the host: the definition, read aloud."""
    s = scores.to(torch.float64).cpu().numpy()
    b = None if bias is None else bias.to(torch.float64).cpu().numpy()
    m, n = s.shape
    ids, ws = np.full((m, case["top"]), -1, np.int32), np.zeros((m, case["top"]), np.float64)
    per = n // case["groups"]
    for t in range(m):
        live = np.isfinite(s[t])
        p = np.zeros(n)
        if case["score"] == "sigmoid":
            p[live] = 1 / (1 + np.exp(-s[t][live]))
        elif live.any():
            p[live] = np.exp(s[t][live] - s[t][live].max())
            p /= p.sum()
        c = p if b is None else p + b
        c = np.where(live & np.isfinite(c), c, -np.inf)
        if case["groups"] > 1:
            rank = []
            for g in range(case["groups"]):
                v = sorted((x for x in c[g * per:(g + 1) * per] if x > -np.inf), reverse=True)[:case["best"]]
                rank.append((-sum(v) if v else np.inf, g))
            for _, g in sorted(rank)[case["top_groups"]:]:
                c[g * per:(g + 1) * per] = -np.inf
        pick = [e for e in np.argsort(-c, kind="stable")[:case["top"]] if c[e] > -np.inf]
        w = p[pick]
        if case["norm"] and w.sum() > 0:
            w = w / w.sum()
        ids[t, :len(pick)], ws[t, :len(pick)] = pick, w * case["scale"]
    return torch.from_numpy(ids).to(DEV), torch.from_numpy(ws).to(DEV)


def _places(qt):
    """For element e of a K block: (byte, shift, mask, up) of each part of its code."""
    e = np.arange(256)
    if qt == "q6_k":
        half, r, l = e // 128, e % 128 // 32, e % 32
        return [(64 * half + 32 * (r % 2) + l, 4 * (r // 2), 15, 0), (128 + 32 * half + l, 2 * r, 3, 4)]
    first = 16 if qt == "q4_k" else 48
    parts = [(first + 32 * (e // 64) + e % 32, 4 * (e // 32 % 2), 15, 0)]
    return parts if qt == "q4_k" else parts + [(16 + e % 32, e // 32, 1, 4)]


def _unpack64(qt, w, n):
    """[rows, n] weights of uint8 rows in 64 bits, element by element from the format's table."""
    unit, size = UNIT[qt]
    b = w.reshape(-1, size)

    def half(at):
        return b[:, at:at + 2].contiguous().view(torch.float16).to(torch.float64)

    if qt == "q8_0":
        return (half(0) * b[:, 2:].contiguous().view(torch.int8).to(torch.float64)).view(-1, n)
    code = torch.zeros((b.shape[0], 256), dtype=torch.int32, device=DEV)
    for byte, shift, mask, up in _places(qt):
        v = b[:, torch.as_tensor(byte, device=DEV)].to(torch.int32)
        code |= (v >> torch.as_tensor(np.broadcast_to(shift, 256).astype(np.int32), device=DEV) & mask) << up
    if qt == "q6_k":
        sc = b[:, 192:208].contiguous().view(torch.int8).to(torch.float64).repeat_interleave(16, 1)
        return (half(208) * sc * (code.to(torch.float64) - 32)).view(-1, n)
    head = b[:, 4:16].to(torch.int32)
    sc, mn = [], []
    for j in range(8):
        if j < 4:
            sc.append(head[:, j] & 63)
            mn.append(head[:, j + 4] & 63)
        else:
            sc.append((head[:, j + 4] & 15) | (head[:, j - 4] >> 6 << 4))
            mn.append((head[:, j + 4] >> 4) | (head[:, j] >> 6 << 4))
    sc = torch.stack(sc, 1).to(torch.float64).repeat_interleave(32, 1)
    mn = torch.stack(mn, 1).to(torch.float64).repeat_interleave(32, 1)
    return (half(0) * sc * code.to(torch.float64) - half(2) * mn).view(-1, n)


def _codes64(qt, x):
    """The codes, decided in the 32-bit steps of the format's definition, times their scales in 64 bits; on the host."""
    unit = UNIT[qt][0]
    b = x.cpu().numpy().reshape(-1, unit)
    top = np.abs(b).max(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.where(top > 0, np.float32(127) / top, np.float32(0))
        d = (top / np.float32(127)).astype(np.float16).astype(np.float64) if qt == "q8_0" else np.where(
            top > 0, np.float32(1) / inv, np.float32(0)).astype(np.float64)
    q = np.clip(np.rint(b * inv), -127, 127).astype(np.float64)
    return torch.from_numpy((q * d).reshape(x.shape)).to(DEV)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "route":
        return _exact_route(s["scores"], s["bias"], case)
    ids, weights = _exact_route(s["scores"], None, dict(case, score="softmax", groups=1, norm=True, scale=1.0))
    t, m, k = case["type"], case["m"], case["top"]
    weights = weights.to(torch.float32).to(torch.float64)  # (an input of the product)
    flat = ids.view(-1).long()
    if case["kind"] == "gate_up":
        a = _codes64(t, s["x"])
        out = torch.zeros((m * k, case["n_ff"]), dtype=torch.float64, device=DEV)
    else:
        a = _codes64(t, s["act"]).view(m * k, -1)
        out = torch.zeros((m, case["n_embd"]), dtype=torch.float64, device=DEV)
        if s["residual"] is not None:
            out += s["residual"]
    for e in sorted(set(flat.tolist()) - {-1}):
        pairs = (flat == e).nonzero().view(-1)
        if case["kind"] == "gate_up":
            g, u = (a[pairs // k] @ _unpack64(t, s[w][e], case["n_embd"]).t() for w in ("gate", "up"))
            if s["b_gate"] is not None:
                g, u = g + s["b_gate"][e], u + s["b_up"][e]
            if case["f"] == "silu":
                f = g * torch.sigmoid(g)
            else:
                f = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
            out[pairs] = f * u
            continue
        y = a[pairs] @ _unpack64(t, s["down"][e], case["n_ff"]).t()
        if s["bias"] is not None:
            y = y + s["bias"][e]
        # (a token takes an expert once, so no two rows of this sum are the same)
        out[pairs // k] += y * weights.view(-1)[pairs].unsqueeze(1)
    return out.view(m, k, -1) if case["kind"] == "gate_up" else out
