"""Plain forms in 64 bits of the rotation, the paged cache's layout and attention over it."""
import numpy as np
import torch

import edgexpu_amd as E

EPS16 = torch.finfo(torch.float16).eps / 2
EPS32 = torch.finfo(torch.float32).eps / 2


def decode(pool, qtype, layers, pages, kv, page, dim):
    """The pool's values [layer, page, K or V, head, token, dim] in 64 bits."""
    b = pool.cpu().numpy().reshape(layers, pages, 2, kv, -1)
    shape = (layers, pages, 2, kv, page, dim)
    if qtype != E.Q8_0:
        t = np.float32 if qtype == E.F32 else np.float16
        return np.ascontiguousarray(b).view(t).reshape(shape).astype(np.float64)
    n = page * dim
    codes = np.ascontiguousarray(b[..., :n]).view(np.int8).reshape(shape[:-1] + (dim // 32, 32))
    d = np.ascontiguousarray(b[..., n:]).view(np.float16).reshape(shape[:-1] + (dim // 32, 1))
    return (codes.astype(np.float64) * d.astype(np.float64)).reshape(shape)


def random_pool(rng, qtype, layers, pages, kv, page, dim, std=1.0):
    """A pool's bytes with values near a bell."""
    x = rng.standard_normal((layers, pages, 2, kv, page, dim)) * std
    if qtype != E.Q8_0:
        t = np.float32 if qtype == E.F32 else np.float16
        return torch.from_numpy(x.astype(t).reshape(-1).view(np.uint8).copy())
    codes = np.clip(np.rint(x / std * 45), -127, 127).astype(np.int8).reshape(layers, pages, 2, kv, -1).view(np.uint8)
    d = (std / 45 * rng.uniform(0.5, 2, (layers, pages, 2, kv, page * dim // 32))).astype(np.float16).view(np.uint8)
    return torch.from_numpy(np.concatenate([codes, d], -1).reshape(-1).copy())


def values(pool_values, layer, pages, n):
    """K and V [heads, n, dim] of a sequence's first n tokens."""
    p = pool_values[layer][pages]
    return [np.concatenate(list(p[:, j].transpose(0, 2, 1, 3)), 0)[:n].transpose(1, 0, 2) if n else
            np.zeros((p.shape[2], 0, p.shape[4])) for j in (0, 1)]


def attend(q, k, v, first, scale, qtype):
    """(out, tolerance) [new, heads, dim] of q [new, heads, dim] at the positions from `first` on.

    The tolerance: with S the largest sum of |scale q_i k_i| and n keys, a score is off by at most
    (dim + 8) eps32 S (sums of dim products, q in parts that miss 2^-22 = 4 eps32 of it, two scalings), its
    exponent's argument by 2 eps32 S more, so a weight by twice that relatively (its own and the
    maximum's); exp2 and the weight's parts add 8 eps32, the two sums (n + 8) eps32 each.  Numerator and
    denominator both carry these, hence the factor 2.

    F16 and Q8_0 weights are two f16 parts of p = 2^(s - m + 7), the largest of a row between 2^7 and 2^15; the second
    part rounds to steps of 2^-24 at the finest, so a weight is off by up to 2^-25, 2^-32 of the row's largest, whatever
    its own size.  With Q8_0 the parts are of p d / D, D at most twice the largest scale d, which makes it 2^-31 of the
    largest weight times the largest value, and n such terms add up."""
    m, H, dim = q.shape
    kv = k.shape[0]
    q = torch.from_numpy(q).double()
    out, tol = np.zeros((m, H, dim)), np.zeros((m, H, dim))
    for h in range(H):
        kh, vh = torch.from_numpy(k[h // (H // kv)]), torch.from_numpy(v[h // (H // kv)])
        for t in range(m):
            n = first + t + 1
            s = (kh[:n] @ q[t, h]) * scale
            w = torch.exp(s - s.max())
            w = w / w.sum()
            out[t, h] = (w @ vh[:n]).numpy()
            big = float((kh[:n].abs() @ q[t, h].abs()).max()) * abs(scale)
            rel = 2 * ((dim + 12) * 2 * EPS32 * big + (8 + 2 * (n + 8)) * EPS32)
            floor = 0.0 if qtype == E.F32 else n * 2.0 ** -31 * float(w.max() * vh[:n].abs().max())
            tol[t, h] = ((w @ vh[:n].abs()) * rel).numpy() + floor + 1e-30
    return out, tol


def rotated(x, weight, eps, pos, n_rot, base=10000.0, scale=1.0, factors=None, interleaved=False):
    """x [tokens, heads, dim] normed and rotated in 64 bits."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    if n_rot:
        i = np.arange(n_rot // 2)
        f = scale * np.power(np.longdouble(base), np.longdouble(-2) * i / n_rot)
        if factors is not None:
            f = f / np.asarray(factors, np.float32).astype(np.longdouble)
        a = np.asarray(pos, np.longdouble)[:, None] * f
        c, s = np.cos(a).astype(np.float64)[:, None], np.sin(a).astype(np.float64)[:, None]
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + n_rot // 2)
        y = x.copy()
        y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., lo] * s + x[..., hi] * c
        x = y
    return x


def rotated_tol(x, weight, eps):
    """How far 32 bits may be: the norm's scale and two products 6 eps32, sine and cosine (angle rounded once in turns:
    pi eps32, functions 4 eps32), two products and a sum 4 eps32, of the larger of a pair (here of the head's largest)."""
    big = np.abs(rotated(x, weight, eps, None, 0)).max(-1, keepdims=True)
    return big * 24 * EPS32 + 1e-37
