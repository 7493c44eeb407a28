"""The feed-forward of experts in 64 bits, plainly, and how far f32 sums may be from it.

u = 2^-24 is half a step of f32.  A row's dot is a sum of block terms dx (d I - dmin M) with exact integers I and M
(rounded to f32 where they pass 2^24): at most six roundings a term, so 6 u of the term's |dx d I| + |dx dmin M|, which
S = sum |w x| bounds; products inside a block summed in f32 (at most 16 steps) 16 u S more; nb terms summed in any order
and joined over at most 16 waves (nb + 16) u S.  Together (nb + 38) u S; 40 here.
"""
import numpy as np

import npref as R

U = 2.0 ** -24


def codes(qtype, x):
    """Quantized rows [rows, bytes] of f32 [rows, n]."""
    q = R.quantize_q8_k if qtype in (12, 13, 14) else R.quantize_q8_0
    return q(np.ascontiguousarray(x, dtype=np.float32).reshape(-1)).reshape(x.shape[0], -1)


def dots(qtype, w, xq):
    """(value, tolerance) [rows of xq, rows of w]."""
    k = qtype in (12, 13, 14)
    val, mag = (R.kq_q8k_gemm_f64 if k else R.g32_q80_gemm_f64)(qtype, w, xq)
    nb = xq.shape[1] // (292 if k else 34)
    return val, (nb + 40) * U * mag


def silu(v):
    """Value and a bound of the slope."""
    e = np.exp(-np.abs(v))
    s = np.where(v >= 0, 1 / (1 + e), e / (1 + e))
    return v * s, 1.1


def gelu(v):
    u = 2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)
    e = np.exp(-np.abs(u))
    return v * np.where(u >= 0, 1 / (1 + e), e / (1 + e)), 1.13


def gate_up(qtype, x, w_gate, w_up, ids, b_gate=None, b_up=None, act="silu"):
    """act [m, k, n_ff] and its tolerance; w_* [experts, n_ff, row bytes]."""
    m, k = ids.shape
    n_ff = w_gate.shape[1]
    out, tol = np.zeros((m, k, n_ff)), np.zeros((m, k, n_ff))
    xq = codes(qtype, x)
    for e in sorted(set(ids.reshape(-1).tolist())):
        if not 0 <= e < w_gate.shape[0]:
            continue
        t, j = np.nonzero(ids == e)
        (g, dg), (v, dv) = dots(qtype, w_gate[e], xq[t]), dots(qtype, w_up[e], xq[t])
        if b_gate is not None:
            g, dg = g + b_gate[e], dg + U * (np.abs(g) + np.abs(b_gate[e]))
        if b_up is not None:
            v, dv = v + b_up[e], dv + U * (np.abs(v) + np.abs(b_up[e]))
        f, slope = silu(g) if act == "silu" else gelu(g)
        # the exponential: its argument is off by 4 u of itself (gelu; silu: none), itself by 4 u; a division, two
        # products and a sum besides: 12 u in all, and where 1 + exp overflows f32 nothing is left of f
        arg = np.abs(g) if act == "silu" else np.abs(2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))
        df = slope * dg + np.abs(f) * (12 + 4 * arg) * U + 2e-38 * (1 + np.abs(g))
        out[t, j] = f * v
        tol[t, j] = df * np.abs(v) + np.abs(f) * dv + df * dv + 2 * U * np.abs(f * v) + 1e-44
    return out, tol


def down(qtype, act, w, ids, weights, bias=None, residual=None):
    """out [m, n_embd] and its tolerance; act [m, k, n_ff]."""
    m, k = ids.shape
    n = w.shape[1]
    parts, tols, size = np.zeros((m, k, n)), np.zeros((m, k, n)), np.zeros((m, k, n))
    for e in sorted(set(ids.reshape(-1).tolist())):
        if not 0 <= e < w.shape[0]:
            continue
        t, j = np.nonzero(ids == e)
        y, dy = dots(qtype, w[e], codes(qtype, act[t, j]))
        big = np.abs(y)
        if bias is not None:
            y, big = y + bias[e], big + np.abs(bias[e])
        g = weights[t, j].astype(np.float64)[:, None]
        parts[t, j], tols[t, j], size[t, j] = g * y, np.abs(g) * dy, np.abs(g) * big
    out, big = parts.sum(1), size.sum(1)
    if residual is not None:
        out, big = out + residual, big + np.abs(residual)
    return out, tols.sum(1) + (k + 4) * U * big + 1e-44


def route(scores, k, score="softmax", bias=None, n_groups=1, top_groups=1, best=1, normalise=True, scale=1.0):
    """ids [m, k] and weights in 64 bits, token by token."""
    m, n = scores.shape
    ids, ws, per = np.full((m, k), -1, np.int32), np.zeros((m, k)), n // n_groups
    for t in range(m):
        s = scores[t].astype(np.float64)
        live = np.isfinite(s)
        p = np.zeros(n)
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                p[live] = 1 / (1 + np.exp(-s[live]))
        elif live.any():
            p[live] = np.exp(s[live] - s[live].max())
            p /= p.sum()
        c = p if bias is None else p + bias.astype(np.float64)
        c = np.where(live & np.isfinite(c), c, -np.inf)
        if n_groups > 1:
            rank = []
            for g in range(n_groups):
                v = sorted((x for x in c[g * per:(g + 1) * per] if x > -np.inf), reverse=True)[:best]
                rank.append((-sum(v) if v else np.inf, g))
            for _, g in sorted(rank)[top_groups:]:
                c[g * per:(g + 1) * per] = -np.inf
        pick = [e for e in np.argsort(-c, kind="stable")[:k] if c[e] > -np.inf]
        w = p[pick]
        if normalise and w.sum() > 0:
            w = w / w.sum()
        ids[t, :len(pick)], ws[t, :len(pick)] = pick, w * scale
    return ids, ws
