"""How many bits attention keeps: few keys and queries with few nonzero values, so that what sums may lose is far below
what one f16 part of a query or a weight would; rows whose heaviest key has a value of zero; Q8_0 scales far apart."""
import numpy as np
import pytest
import torch

import edgexpu_amd as E
import kv_plain as P

pytestmark = pytest.mark.gpu

EPS = P.EPS32
LOG2E = 1.4426950408889634
TERMS = 4  # nonzero values of a query
TILE = 32


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def encode(x, qtype, page, scales=None):
    """Pool bytes of values [2, heads, n, dim] in pages one after the other, and what they decode to.  Q8_0: x are the
    codes, scales [2, heads, n, dim / 32]."""
    two, kv, n, dim = x.shape
    pages = -(-n // page)

    def paged(a):  # [2, heads, n, ...] -> [pages, 2, heads, page, ...]
        a = np.concatenate([a, np.zeros(a.shape[:2] + (pages * page - n,) + a.shape[3:], a.dtype)], 2)
        return np.moveaxis(a.reshape((two, kv, pages, page) + a.shape[3:]), 2, 0)

    if qtype != E.Q8_0:
        t = x.astype(np.float16 if qtype == E.F16 else np.float32)
        return torch.from_numpy(np.ascontiguousarray(paged(t)).reshape(-1).view(np.uint8).copy()), t.astype(np.float64)
    d = scales.astype(np.float16)
    codes = np.ascontiguousarray(paged(x.astype(np.int8))).reshape(pages, 2, kv, -1).view(np.uint8)
    raw = np.concatenate([codes, np.ascontiguousarray(paged(d)).reshape(pages, 2, kv, -1).view(np.uint8)], -1)
    with np.errstate(invalid="ignore"):
        return torch.from_numpy(raw.reshape(-1).copy()), x.astype(np.float64) * np.repeat(d.astype(np.float64), 32, -1)


def queries(rng, new, heads, dim, std=1.0):
    """TERMS nonzero values a row, in channels spread over the head."""
    q = np.zeros((new, heads, dim), np.float32)
    at = np.arange(TERMS) * dim // TERMS
    q[..., at] = rng.standard_normal((new, heads, TERMS)) * std
    return q


def run(pool, qtype, kv, dim, page, n, q, scale):
    new, heads, _ = q.shape
    c = E.KvCache(qtype, 1, kv, dim, page, -(-n // page), 1, pool=pool.cuda())
    s = c.new()
    c.extend([s], [n])
    b = E.KvBatch(c, heads, 1, new)
    b.set([s], [new])
    return E.attention(b, 0, dev(q.reshape(new, -1)), scale).cpu().numpy().reshape(new, heads, dim)


def expect(q, k, v, scale, qtype, terms=TERMS, scales=None):
    """(out, tolerance, weights) of q [new, heads, dim] at the last positions of k, v [kv heads, n, dim], all in 64 bits.

    With B the largest sum of |scale q_i k_i| of a row in base-2 units (terms products) and eps = 2^-24, a weight is off
    relatively by
      ln2 eps ((2 terms + 16) B     products of q's two parts (4 eps of it lost), sums, a block's scale; terms 0: one
                                    product, by a power of two, and nothing of it
               + 2 B                the factor of the scores, rounded twice
               + 2 (2 B + 32))      its exponent's argument, s - m and the reference's offset
      + 4 eps                       exp2 and its two parts' 22 bits, 2 + 2
      + 12 eps                      the joins of waves and pieces, a sum's rescaling
      + 6 eps                       Q8_0: times a scale, and its value's parts (22 bits)
    A weight passes through at most 64 + 4 n / 32 sums (32 products and two parts of a tile, then twice a tile and the
    joins) in the numerator, 8 n / 32 + 32 in the denominator; a tile is 32 keys.  The division adds 3 eps.

    The parts' finest step adds 2^-22 of the largest weight of its tile, 2^-34 of it where it is the largest so far With
    Q8_0 it is that of weight times value scale for a block (single tokens and few; `scales` [kv heads, n, dim / 32]
    where they differ), and 2^-22 of a block's largest value comes on top."""
    m, H, dim = q.shape
    kv, n, _ = k.shape
    out, tol, weights = np.zeros((m, H, dim)), np.zeros((m, H, dim)), []
    for h in range(H):
        kh, vh = k[h // (H // kv)], v[h // (H // kv)]
        for t in range(m):
            seen = n - m + t + 1
            qt = q[t, h].astype(np.float64) * scale
            s = kh[:seen] @ qt
            w = np.exp(s - s.max())
            w /= w.sum()
            out[t, h] = w @ vh[:seen]
            B = float((np.abs(kh[:seen]) @ np.abs(qt)).max()) * LOG2E
            rel = EPS * (np.log(2) * ((2 * terms + 18 if terms else 2) * B + 2 * (2 * B + 32)) + 16 + (6 if qtype == E.Q8_0 else 0))
            tiles = -(-seen // TILE)
            rel = 2 * rel + EPS * (64 + 4 * tiles + 8 * tiles + 32 + 3)
            tol[t, h] = rel * (w @ np.abs(vh[:seen])) + 1e-30
            if qtype != E.F32:
                pad = np.zeros(tiles * TILE)
                pad[:seen] = w
                top = pad.reshape(tiles, TILE).max(1)
                step = np.where(top >= np.maximum.accumulate(top), 2.0 ** -34, 2.0 ** -22) * top
                tol[t, h] += np.repeat(step, TILE)[:seen] @ np.abs(vh[:seen])
            if scales is not None:  # a code's part of what weight times scale is off by
                x = np.zeros((tiles * TILE, dim // 32))
                x[:seen] = w[:, None] * scales[h // (H // kv), :seen]
                top = x.reshape(tiles, TILE, -1).max(1)
                step = np.where(top >= np.maximum.accumulate(top, 0), 2.0 ** -34, 2.0 ** -22) * top
                codes = np.abs(vh[:seen]) / np.repeat(np.maximum(scales[h // (H // kv), :seen], 1e-30), 32, -1)
                tol[t, h] += (np.repeat(np.repeat(step, TILE, 0)[:seen], 32, -1) * codes).sum(0)
            if qtype == E.Q8_0:
                block = np.abs(vh[:seen]).reshape(seen, -1, 32).max(-1)
                tol[t, h] += 2.0 ** -22 * np.repeat(w @ block, 32)
            weights.append(w)
    return out, tol, weights


# (dim, kv, group, new, n): rows of a workgroup 1, 8, 17 to 32, 33 to 64, 65 to 128; all keys in a tile or a few
ROWS = [(64, 1, 1, 1, 5), (128, 2, 4, 2, 9), (96, 1, 5, 5, 12), (128, 1, 4, 8, 11), (64, 1, 6, 5, 7), (256, 1, 3, 2, 6), (64, 2, 8, 6, 9),
        (128, 1, 6, 9, 13), (96, 1, 10, 6, 8), (256, 1, 8, 6, 10), (64, 1, 16, 7, 10), (128, 2, 16, 8, 12), (96, 1, 16, 8, 11), (256, 1, 16, 7, 9),
        (128, 1, 12, 10, 45), (64, 1, 13, 8, 70)]
PARTS = [E.F16, E.Q8_0]


@pytest.mark.parametrize("qtype", PARTS)
@pytest.mark.parametrize("case", ROWS)
def test_both_parts_of_queries_and_weights(hipdev, qtype, case):
    dim, kv, group, new, n = case
    rng = np.random.default_rng(abs(hash(case)) % 2**31 + qtype)
    heads, page = kv * group, 64
    q = queries(rng, new, heads, dim)
    if qtype == E.Q8_0:
        x = rng.integers(-127, 128, (2, kv, n, dim))
        pool, (k, v) = encode(x, qtype, page, rng.uniform(0.5, 2, (2, kv, n, dim // 32)) / 90)
    else:
        pool, (k, v) = encode(rng.standard_normal((2, kv, n, dim)), qtype, page)
    got = run(pool, qtype, kv, dim, page, n, q, 1.0)
    want, tol, weights = expect(q, k, v, 1.0, qtype)
    err = np.abs(got - want)
    assert np.all(err <= tol), np.max(err / tol)
    # what one f16 part would give is outside: of the query, and of the weights
    top = 2.0 ** np.ceil(np.log2(np.abs(q).max(-1, keepdims=True)))
    once = expect((q / top).astype(np.float16).astype(np.float32) * top, k, v, 1.0, qtype)[0]
    assert (np.abs(once - want) > tol).any()
    if n > 1:
        once = np.array([w.astype(np.float16).astype(np.float64) @ v[i % heads // group][: len(w)] for i, w in enumerate_rows(weights, new, heads)])
        assert (np.abs(once.reshape(heads, new, dim).transpose(1, 0, 2) - want) > tol).any()


def enumerate_rows(weights, new, heads):
    """(head, weights of a row) in the order of expect: by head, then token; weights scaled to a largest of 1."""
    for i, w in enumerate(weights):
        yield i // new, w


@pytest.mark.parametrize("qtype", PARTS)
@pytest.mark.parametrize("dim,group,new,n,nats,at", [
    (128, 1, 1, 64, 16.0, 0), (128, 4, 1, 150, 16.0, 100), (64, 2, 1, 80, 12.0, 0), (256, 1, 1, 100, 16.0, 40),
    (96, 4, 8, 150, 16.0, 0), (128, 8, 16, 120, 16.0, 0), (64, 8, 16, 200, 9.0, 70), (96, 8, 10, 100, 30.0, 0),
    (256, 8, 8, 100, 16.0, 0), (128, 8, 7, 130, 16.0, 64), (128, 2, 1, 300, 16.0, 0), (128, 8, 16, 150, 5.0, 0),
    (128, 4, 1, 5000, 20.0, 4000), (64, 8, 16, 3000, 14.0, 0),
])
def test_a_heavy_key_of_no_value(hipdev, qtype, dim, group, new, n, nats, at):
    """One key far above the rest, its value zero: the rest keep their bits."""
    rng = np.random.default_rng(n + dim + int(nats))
    page = 64
    q = np.zeros((new, group, dim), np.float32)
    q[..., 0] = 1.0
    x = rng.standard_normal((2, 1, n, dim)) * 0.4
    if qtype == E.Q8_0:
        x = np.clip(np.rint(x * 60), -127, 127).astype(np.int64)
        scales = np.full((2, 1, n, dim // 32), 1 / 64)
        x[0, 0, at, 0], scales[0, 0, at, 0] = 64, nats / 64
        x[1, 0, at] = 0
        pool, (k, v) = encode(x, qtype, page, scales)
    else:
        x[0, 0, at, 0] = nats
        x[1, 0, at] = 0.0
        pool, (k, v) = encode(x, qtype, page)
    got = run(pool, qtype, 1, dim, page, n, q, 1.0)
    want, tol, _ = expect(q, k, v, 1.0, qtype, 0)
    err = np.abs(got - want)
    assert np.all(err <= tol), np.max(err / tol)


def q8_cache(rng, n, dim, typical):
    """Codes [K, V][1][n][dim] and scales, V's around `typical`."""
    codes = rng.integers(-127, 128, (2, 1, n, dim))
    scales = rng.uniform(0.5, 2, (2, 1, n, dim // 32))
    scales[0] /= 90
    scales[1] *= typical
    return codes, scales


# rows of a workgroup: 1 to 10, 16, 20, 40, 128; 128 and more
FORMS = [(128, 1, 6), (96, 2, 5), (256, 2, 4), (64, 1, 1), (96, 4, 1), (128, 4, 1), (256, 4, 2), (64, 4, 5), (128, 4, 5), (96, 8, 4),
         (128, 8, 5), (64, 8, 16), (96, 16, 8), (128, 16, 17), (256, 8, 5)]


@pytest.mark.parametrize("dim,group,new", FORMS)
@pytest.mark.parametrize("typical,large", [(0.02, 512.0), (2e-4, 512.0), (2e-4, 8192.0), (2e-4, 65504.0), (6e-8, 1.0)])
def test_a_large_value_scale_is_its_blocks_own(hipdev, dim, group, new, typical, large):
    """One block of one key has a scale far above all others: the other blocks keep their bits."""
    rng = np.random.default_rng(dim * new + int(large))
    n, page = new + 60, 32
    codes, scales = q8_cache(rng, n, dim, typical)
    scales[1, 0, 5, 1] = large
    pool, (k, v) = encode(codes, E.Q8_0, page, scales)
    q = queries(rng, new, group, dim)
    got = run(pool, E.Q8_0, 1, dim, page, n, q, 1.0)
    want, tol, _ = expect(q, k, v, 1.0, E.Q8_0, scales=scales[1].astype(np.float16).astype(np.float64))
    err = np.abs(got - want)
    assert np.all(err <= tol), np.max(err / tol)


@pytest.mark.parametrize("dim,group,new", [f for f in FORMS if f[2] > 3])
@pytest.mark.parametrize("bad", [100.0, 65504.0, np.inf, np.nan])
def test_value_scales_of_later_tokens_have_no_influence(hipdev, dim, group, new, bad):
    """A scale of one of the step's later tokens, in one block or in all of them, leaves the rows before it as they are."""
    rng = np.random.default_rng(dim + new)
    n, page, at = new + 21, 16, new + 21 - 2
    codes, scales = q8_cache(rng, n, dim, 1e-4)
    q = queries(rng, new, group, dim)
    pool, (k, v) = encode(codes, E.Q8_0, page, scales)
    plain = run(pool, E.Q8_0, 1, dim, page, n, q, 1.0)
    want, tol, _ = expect(q, k, v, 1.0, E.Q8_0, scales=scales[1].astype(np.float16).astype(np.float64))
    assert np.all(np.abs(plain - want) <= tol)
    rows = new - 2
    for blocks in (slice(0, 1), slice(None)):
        other = scales.copy()
        other[1, 0, at, blocks] = bad
        got = run(encode(codes, E.Q8_0, page, other)[0], E.Q8_0, 1, dim, page, n, q, 1.0)
        err = np.abs(got - want)
        assert np.all(err[:rows] <= tol[:rows]), np.max(err[:rows] / tol[:rows])
        if bad == 100.0:  # (units are powers of two: not a bit of difference)
            assert np.array_equal(got[:rows], plain[:rows])


@pytest.mark.parametrize("qtype", [E.F16, E.Q8_0, E.F32])
@pytest.mark.parametrize("dim,group,new", FORMS)
@pytest.mark.parametrize("at", [3, 40, -1])
def test_keys_and_values_that_are_not_finite(hipdev, qtype, dim, group, new, at):
    """Wherever they lie and whatever the signs, a value makes itself (its block with Q8_0) NaN in the rows that see it; a
    key makes them NaN, or with a score of minus infinity has no weight."""
    rng = np.random.default_rng(dim + new + at)
    n, page = new + 70, 32
    at %= n
    if qtype == E.Q8_0:
        x, scales = q8_cache(rng, n, dim, 0.02)
        x[x == 0] = 1
    else:
        x, scales = rng.standard_normal((2, 1, n, dim)), None
    q = rng.standard_normal((new, group, dim)).astype(np.float32)
    first = max(0, at - (n - new))  # the first row that sees it
    pool, (k, v) = encode(x, qtype, page, scales)
    plain = run(pool, qtype, 1, dim, page, n, q, dim ** -0.5)
    assert np.isfinite(plain).all()
    w = np.exp(np.einsum("thd,nd->thn", q.astype(np.float64), k[0]) * dim ** -0.5)
    w[np.broadcast_to(np.arange(n) > np.arange(new)[:, None, None] + n - new, w.shape)] = 0.0
    w[..., at] = 0.0
    without = (w @ v[0]) / w.sum(-1, keepdims=True)
    for bad in (np.inf, -np.inf, np.nan):
        for which in (1, 0):
            y, d = x.copy(), None if scales is None else scales.copy()
            if qtype == E.Q8_0:
                d[which, 0, at, 1] = bad
            else:
                y[which, 0, at, 37] = bad
            got = run(encode(y, qtype, page, d)[0], qtype, 1, dim, page, n, q, dim ** -0.5)
            assert np.array_equal(got[:first], plain[:first]), (bad, which)
            if which == 1:
                spoilt = slice(32, 64) if qtype == E.Q8_0 else slice(37, 38)
                assert np.isnan(got[first:, :, spoilt]).all(), bad
                rest = [e for e in range(dim) if not spoilt.start <= e < spoilt.stop]
                assert np.array_equal(got[..., rest], plain[..., rest]), bad
            else:
                nan = np.isnan(got[first:]).any(-1)
                assert np.isnan(got[first:][nan]).all() and (nan.all() or np.isinf(bad)), bad
                assert np.allclose(got[first:][~nan], without[first:][~nan], rtol=0, atol=1e-4 * np.abs(v).max()), bad
