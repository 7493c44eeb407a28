"""Rotation with the cache write, attention over the paged cache, and the cache's pages, against plain forms in 64 bits."""
import numpy as np
import pytest
import torch

import edgexpu_amd as E
import kv_plain as P

pytestmark = pytest.mark.gpu

TYPES = [E.F16, E.Q8_0, E.F32]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def make(rng, qtype, kv, dim, page, n_pages, max_seqs, layers=1, std=1.0):
    pool = P.random_pool(rng, qtype, layers, n_pages, kv, page, dim, std).cuda()
    return E.KvCache(qtype, layers, kv, dim, page, n_pages, max_seqs, pool=pool)


def pool_values(cache, qtype, layers, n_pages, page):
    return P.decode(cache.pool, qtype, layers, n_pages, cache.n_kv_heads, page, cache.head_dim)


def poison(cache, qtype, layers, n_pages, page, seqs):
    """NaN (codes of 127 with a NaN scale) in every slot that no sequence of `seqs` holds a token in."""
    kv, dim = cache.n_kv_heads, cache.head_dim
    held = np.zeros((n_pages, page), bool)
    for s in seqs:
        n, row = cache.length(s), cache.tables([s])[0]
        for i in range(-(-n // page)):
            held[row[i], : min(page, n - i * page)] = True
    b = cache.pool.cpu().numpy().reshape(layers, n_pages, 2, kv, -1).copy()
    for p, o in zip(*np.nonzero(~held)):
        if qtype == E.Q8_0:
            b[:, p, :, :, o * dim: (o + 1) * dim] = 127
            at = page * dim + o * dim // 16
            b[:, p, :, :, at: at + dim // 16] = np.full(dim // 32, np.nan, np.float16).view(np.uint8)
        else:
            v = b.view(np.float32 if qtype == E.F32 else np.float16).reshape(layers, n_pages, 2, kv, page, dim)
            v[:, p, :, :, o] = np.nan if o % 2 else np.inf
    cache.pool.copy_(torch.from_numpy(b.reshape(-1)))


def check_attention(cache, qtype, layers, n_pages, page, seqs, n_new, heads, rng, layer=0, scale=None, q=None, slack=3):
    dim = cache.head_dim
    batch = E.KvBatch(cache, heads, len(seqs) + 1, sum(n_new) + slack)
    batch.set(seqs, n_new)
    T = sum(n_new)
    assert batch.tokens() == T
    if q is None:
        q = rng.standard_normal((T + slack, heads * dim)).astype(np.float32) * 1.5
    out = torch.full((T + slack, heads * dim), 7.5, device="cuda:0")
    E.attention(batch, layer, dev(q), scale, out=out)
    got = out.cpu().numpy()
    assert np.all(got[T:] == 7.5), "rows behind the last token were written"
    vals, at, worst = pool_values(cache, qtype, layers, n_pages, page), 0, 0.0
    for s, m in zip(seqs, n_new):
        n = cache.length(s)
        k, v = P.values(vals, layer, [p for p in cache.tables([s])[0] if p >= 0], n)
        want, tol = P.attend(q[at: at + m].reshape(m, heads, dim), k, v, n - m, dim ** -0.5 if scale is None else scale, qtype)
        err = np.abs(got[at: at + m].reshape(m, heads, dim) - want)
        assert np.all(err <= tol), f"sequence of {n}, {m} new: {np.max(err / tol):.3g} times the tolerance"
        if m:
            worst = max(worst, float(np.max(err / tol)))
        at += m
    return worst


# one token and more, lengths around pages and tiles, groups that fill a tile or do not, every head size and page
SINGLE = [  # (dim, kv, group, page, length, new)
    (64, 1, 1, 16, 1, 1), (64, 3, 3, 16, 2, 2), (64, 2, 7, 32, 33, 1), (128, 2, 4, 64, 64, 1), (128, 1, 4, 64, 65, 3),
    (96, 2, 2, 16, 47, 5), (256, 1, 8, 128, 127, 1), (128, 8, 4, 32, 1000, 1), (64, 1, 1, 64, 300, 300),
    (128, 1, 3, 16, 200, 77), (256, 2, 2, 64, 150, 33), (96, 1, 16, 256, 511, 2), (128, 1, 20, 64, 90, 2),
    (64, 3, 3, 64, 4099, 1), (128, 2, 1, 128, 2500, 17),
    (64, 1, 1, 256, 140001, 1), (256, 1, 2, 16, 847, 315), (128, 1, 40, 32, 300, 1),
]


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("case", SINGLE)
def test_one_sequence(hipdev, qtype, case):
    dim, kv, group, page, n, new = case
    rng = np.random.default_rng(abs(hash(case)) % 2**31 + qtype)
    pages = -(-n // page) + 2
    c = make(rng, qtype, kv, dim, page, pages, 2)
    first, s = c.new(), c.new()
    c.extend([first], [1])
    c.extend([s], [n])
    poison(c, qtype, 1, pages, page, [first, s])
    check_attention(c, qtype, 1, pages, page, [s], [new], kv * group, rng)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("dim,kv,group,page,prefix,own,new", [
    (128, 2, 4, 64, 64 * 30, [1, 2, 64, 65, 300, 5, 6, 7, 8, 9, 10, 11], 1),
    (64, 3, 3, 16, 1000, [1, 1, 17, 40, 3, 90, 90, 2, 16, 15], 1),
    (256, 1, 8, 32, 700, [30, 31, 32, 33], 3),
    (96, 2, 2, 64, 3000, [5, 700, 1400], 2),
    (128, 1, 1, 128, 640, [40] * 40, 1),
    (128, 1, 16, 64, 2048, [20] * 9, 1),
    (128, 2, 4, 64, 5000, [70, 80], 64),
])
def test_shared_prefix(hipdev, qtype, dim, kv, group, page, prefix, own, new):
    rng = np.random.default_rng(prefix + dim + qtype)
    pages = -(-prefix // page) + sum(-(-n // page) + 2 for n in own) + 3
    c = make(rng, qtype, kv, dim, page, pages, len(own) + 2, layers=2)
    root = c.new()
    c.extend([root], [prefix])
    kids = c.fork([root] * len(own))
    half = [n // 2 for n in own]
    c.extend(kids, half)
    c.extend(kids, [n - h for n, h in zip(own, half)])
    poison(c, qtype, 2, pages, page, [root] + kids)
    order = list(rng.permutation(len(kids)))
    check_attention(c, qtype, 2, pages, page, [kids[i] for i in order], [min(new, own[i]) for i in order], kv * group,
                    rng, layer=1)


def test_a_tree_of_forks(hipdev):
    rng = np.random.default_rng(5)
    c = make(rng, E.F16, 2, 128, 32, 400, 40)
    a = c.new()
    c.extend([a], [900])
    level = [a]
    for grow in (400, 700, 130):
        level = c.fork([p for p in level for _ in range(2)])
        c.extend(level, [grow + i for i in range(len(level))])
    lone = c.new()
    c.extend([lone], [333])
    seqs = level[::2] + [a, lone] + level[1::2]
    check_attention(c, E.F16, 1, 400, 32, seqs, [1] * len(seqs), 8, rng)
    # sequences with no new token are part of no row
    check_attention(c, E.F16, 1, 400, 32, seqs, [i % 3 for i in range(len(seqs))], 8, rng)


@pytest.mark.parametrize("qtype", TYPES)
def test_extreme_scores_and_values(hipdev, qtype):
    """One key far above the rest, equal keys, very small and large magnitudes, a zero query, a negative scale."""
    rng = np.random.default_rng(11)
    dim, page, n = 128, 64, 700
    for std, qstd, scale in ((1.0, 60.0, 0.1), (2.0 ** -12, 1.0, 1.0), (200.0, 1e-3, 0.05), (1.0, 1e-30, 1e28), (1.0, 1e30, 1e-31),
                             (1.0, 2.0, -0.3), (1.0, 0.0, 0.1), (1.0, 1.0, 0.0), (1.0, 1.0, 1e-44)):
        c = make(rng, qtype, 1, dim, page, 12, 2, std=std)
        s = c.new()
        c.extend([s], [n])
        q = (rng.standard_normal((2, 4 * dim)) * qstd).astype(np.float32)
        check_attention(c, qtype, 1, 12, page, [s], [2], 4, rng, scale=scale, q=q, slack=0)


@pytest.mark.parametrize("qtype", [E.F16, E.F32])
def test_values_of_later_tokens_have_no_influence(hipdev, qtype):
    """NaN and infinities in a step's later tokens leave its earlier rows as they are, and reach those that see them."""
    rng = np.random.default_rng(3)
    dim, page, n, new = 64, 32, 70, 20
    c = make(rng, qtype, 1, dim, page, 4, 1)
    s = c.new()
    c.extend([s], [n])
    q = dev(rng.standard_normal((new, 2 * dim)).astype(np.float32))
    batch = E.KvBatch(c, 2, 1, new)
    batch.set([s], [new])
    t = torch.float16 if qtype == E.F16 else torch.float32
    view = c.pool.view(t).view(4, 2, 1, page, dim)
    k, v = P.values(pool_values(c, qtype, 1, 4, page), 0, [p for p in c.tables([s])[0] if p >= 0], n)
    want, tol = P.attend(q.cpu().numpy().reshape(new, 2, dim), k, v, n - new, dim ** -0.5, qtype)
    for bad, which in ((float("inf"), 1), (float("nan"), 1), (float("nan"), 0), (float("-inf"), 0)):
        keep = view.clone()
        at = n - 7
        view[at // page, which, 0, at % page, 5] = bad
        err = np.abs(E.attention(batch, 0, q).cpu().numpy().reshape(new, 2, dim) - want)
        rows = new - 7
        assert np.all(err[:rows] <= tol[:rows]), (bad, which)
        if which == 1:
            assert not np.isfinite(err[rows:, :, 5]).any()
            others = [e for e in range(dim) if e != 5]
            assert np.all(err[rows:][..., others] <= tol[rows:][..., others]), bad
        view.copy_(keep)


def test_long_cache_offsets_beyond_32_bits(hipdev):
    """A layer whose pages start beyond 4 GiB of the pool."""
    rng = np.random.default_rng(9)
    kv, dim, page, pages, layers = 8, 128, 256, 2200, 3
    size = E.hip().kv_pool_bytes(E.F16, layers, kv, dim, page, pages)
    assert size > 3 * 2**32 // 2
    pool = torch.zeros(size, dtype=torch.uint8, device="cuda:0")
    c = E.KvCache(E.F16, layers, kv, dim, page, pages, 3, pool=pool)
    filler, s = c.new(), c.new()
    at = pages - 5
    c.extend([filler], [page * at])
    c.extend([s], [600])
    assert c.tables([s])[0][0] == at
    v = pool.view(torch.float16).view(layers, pages, 2, kv, page, dim)
    v[:, at:] = torch.randn(v[:, at:].shape, device="cuda:0").half()
    b = E.KvBatch(c, 8, 1, 1)
    b.set([s], [1])
    q = rng.standard_normal((1, 8 * dim)).astype(np.float32)
    for layer in (0, layers - 1):
        got = E.attention(b, layer, dev(q)).cpu().numpy().reshape(1, 8, dim)
        x = v[layer, at: at + 3].double().cpu().numpy()
        k, w = (np.concatenate(list(x[:, j].transpose(0, 2, 1, 3)), 0)[:600].transpose(1, 0, 2) for j in (0, 1))
        want, tol = P.attend(q.reshape(1, 8, dim), k, w, 599, dim ** -0.5, E.F16)
        assert np.all(np.abs(got - want) <= tol)
    # a copy there too
    want = v[:, at:].clone()
    (d,) = c.fork([s])
    c.extend([d], [1])
    assert c.tables([s])[0][2] == at + 2 and c.tables([d])[0][2] == at + 3
    want[:, 3, :, :, :88] = want[:, 2, :, :, :88]
    assert torch.equal(v[:, at:], want)


# ------------------------------------------------------------------ rotation and the cache write


@pytest.mark.parametrize("dim,n_rot,inter,norm,heads,kv,m", [
    (64, 64, True, False, 9, 3, 1), (128, 128, False, True, 32, 8, 5), (256, 64, False, True, 4, 2, 3), (96, 32, True, True, 6, 2, 7),
    (10, 10, False, True, 3, 1, 4), (2, 2, True, False, 1, 1, 2), (128, 0, False, True, 4, 4, 3), (254, 100, True, True, 2, 1, 9),
    (128, 128, False, True, 32, 8, 700), (64, 48, False, False, 7, 3, 1), (256, 256, True, True, 5, 0, 2), (128, 12, False, True, 3, 2, 5),
    (96, 96, False, True, 5, 3, 40), (128, 68, True, False, 1, 1, 3),
])
def test_qk_norm_rope(hipdev, dim, n_rot, inter, norm, heads, kv, m):
    rng = np.random.default_rng(dim * 7 + n_rot)
    x = rng.standard_normal((m, (heads + 2 * kv) * dim)).astype(np.float32) * rng.choice([1e-3, 1.0, 50.0], (m, 1)).astype(np.float32)
    pos = rng.integers(0, 200000, m).astype(np.int32)
    pos[0] = 0
    pos[-1] = 1_000_003
    wq, wk = (rng.standard_normal(dim).astype(np.float32) if norm else None for _ in range(2))
    factors = rng.uniform(1, 8, n_rot // 2).astype(np.float32) if n_rot == 64 else None
    rope = E.Rope(n_rot, 500000.0, 0.5, factors, inter) if n_rot else None
    d = dev(x)
    q, k, _ = d.split([heads * dim, kv * dim, kv * dim], 1)
    w = [None if v is None else dev(v) for v in (wq, wk)]
    qo, ko = E.qk_norm_rope(q, k, heads, kv, dev(pos), rope, w[0], w[1], 1e-5)
    assert torch.equal(d, dev(x))
    eps = float(np.float32(1e-5))
    for got, h, at, wt in ((qo, heads, 0, wq), (ko, kv, heads * dim, wk)):
        y = x[:, at: at + h * dim].reshape(m, h, dim)
        want = P.rotated(y, wt, eps, pos, n_rot, 500000.0, 0.5, factors, inter)
        err = np.abs(got.cpu().numpy().reshape(m, h, dim) - want)
        assert np.all(err <= P.rotated_tol(y, wt, eps)), np.max(err / P.rotated_tol(y, wt, eps))
    # in place
    q2, k2 = q.contiguous(), k.contiguous()
    E.qk_norm_rope(q2, k2, heads, kv, dev(pos), rope, w[0], w[1], 1e-5, q_out=q2, k_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("qtype", TYPES)
@pytest.mark.parametrize("dim,n_rot,inter,norm,heads,kv,page", [
    (128, 128, False, True, 8, 2, 64), (64, 64, True, False, 9, 3, 16), (256, 64, False, True, 4, 1, 32), (96, 96, False, False, 4, 4, 128),
])
def test_append(hipdev, qtype, dim, n_rot, inter, norm, heads, kv, page):
    rng = np.random.default_rng(dim + qtype)
    pages = 24
    c = make(rng, qtype, kv, dim, page, pages, 5, layers=2)
    a, b, e = c.new(), c.new(), c.new()
    c.extend([a, b, e], [page + 3, 5, 1])
    c.extend([b, a], [page, 2])
    (f,) = c.fork([a])
    c.extend([f], [3])
    before = c.pool.clone()
    seqs, n_new = [b, f, e, a], [page, 3, 1, 0]
    T = sum(n_new)
    batch = E.KvBatch(c, heads, 4, T + 9)
    batch.set(seqs, n_new)
    x = rng.standard_normal((T + 2, (heads + 2 * kv) * dim)).astype(np.float32) * 3
    x[0] = 0.0
    x[1, heads * dim:] *= 1e-8
    wq, wk = (rng.standard_normal(dim).astype(np.float32) if norm else None for _ in range(2))
    q, k, v = dev(x).split([heads * dim, kv * dim, kv * dim], 1)
    rope = E.Rope(n_rot, 10000.0, interleaved=inter)
    q_out = torch.full((T + 2, heads * dim), -3.0, device="cuda:0")
    E.kv_append(batch, 1, q, k, v, rope, None if wq is None else dev(wq), None if wk is None else dev(wk), 1e-6, q_out=q_out)
    pos = np.concatenate([np.arange(c.length(s) - n, c.length(s)) for s, n in zip(seqs, n_new)])
    eps = float(np.float32(1e-6))
    y = x[:T, : heads * dim].reshape(T, heads, dim)
    got = q_out.cpu().numpy()
    assert np.all(got[T:] == -3.0)
    err = np.abs(got[:T].reshape(T, heads, dim) - P.rotated(y, wq, eps, pos, n_rot, interleaved=inter))
    assert np.all(err <= P.rotated_tol(y, wq, eps))
    vals = pool_values(c, qtype, 2, pages, page)
    touched = np.zeros((2, pages, 2, kv, page, dim), bool)
    at = 0
    for s, n in zip(seqs, n_new):
        row = c.tables([s])[0]
        for p in range(c.length(s) - n, c.length(s)):
            for which, lo, wt in ((0, heads * dim, wk), (1, (heads + kv) * dim, None)):
                z = x[at: at + 1, lo: lo + kv * dim].reshape(1, kv, dim)
                want = P.rotated(z, wt, eps, [p], 0 if which else n_rot, interleaved=inter)[0]
                tol = np.broadcast_to(P.rotated_tol(z, wt, eps)[0] * (which == 0), want.shape)
                g = vals[1, row[p // page], which, :, p % page]
                touched[1, row[p // page], which, :, p % page] = True
                if qtype == E.F32:
                    lim = tol
                elif qtype == E.F16:  # half a step of the value, or of the smallest normal
                    lim = tol * 1.01 + np.maximum(np.abs(want), 2.0 ** -14) * P.EPS16 * 1.01
                else:  # half a code of the block, its scale rounded to f16 (to half the smallest step at least)
                    top = np.abs(want).reshape(kv, -1, 32).max(-1, keepdims=True)
                    d = top / 127
                    lim = 0.5 * d + 127 * np.maximum(d * P.EPS16, 2.0 ** -25)
                    lim = np.broadcast_to(lim, (kv, dim // 32, 32)).reshape(kv, dim) * (1 + 1e-6) + 3 * tol
                assert np.all(np.abs(g - want) <= lim), (which, p)
            at += 1
    # nothing but the step's slots of that layer has changed
    old = P.decode(before, qtype, 2, pages, kv, page, dim)
    assert np.array_equal(vals[~touched], old[~touched])


def test_append_q8_0_codes_are_the_quantizers(hipdev):
    """Values without norm and rotation become the blocks of quantize_q8_0."""
    rng = np.random.default_rng(2)
    c = make(rng, E.Q8_0, 2, 128, 16, 4, 1)
    s = c.new()
    c.extend([s], [20])
    b = E.KvBatch(c, 2, 1, 20)
    b.set([s], [20])
    x = dev(rng.standard_normal((20, 6 * 128)).astype(np.float32) * np.exp(rng.uniform(-12, 8, (20, 1))).astype(np.float32))
    q, k, v = x.split([256, 256, 256], 1)
    E.kv_append(b, 0, q, k, v)
    raw = c.pool.cpu().numpy().reshape(4, 2, 2, -1)
    for which, y in ((0, k), (1, v)):
        blocks = E.quantize_q8_0(y.contiguous()).cpu().numpy().reshape(20, 2, 4, 34)
        for p in range(20):
            page = raw[c.tables([s])[0][p // 16], which]
            codes = page[:, : 16 * 128].reshape(2, 16, 4, 32)[:, p % 16]
            d = page[:, 16 * 128:].reshape(2, 16, 4, 2)[:, p % 16]
            assert np.array_equal(codes, blocks[p][..., 2:]) and np.array_equal(d, blocks[p][..., :2])


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("norm", [False, True])
def test_append_q8_0_of_values_at_the_limits(hipdev, offset, norm):
    """Subnormal, infinite and huge values become the quantizer's blocks; a NaN's block has a NaN scale (not a finite
    one, with which attention would not see it).  offset 1: rows that are not 16-byte aligned."""
    rng = np.random.default_rng(21)
    c = make(rng, E.Q8_0, 1, 128, 16, 2, 1)
    s = c.new()
    c.extend([s], [8])
    b = E.KvBatch(c, 1, 1, 8)
    b.set([s], [8])
    x = rng.standard_normal((8, 128)).astype(np.float32)
    x[0, :32] = 0.0
    x[1, 5:32] = np.float32(1e-44)
    x[1, :5] = np.float32(3e-37)
    x[2] *= np.float32(1e-38)
    x[3, 40], x[4, 41], x[5, 3] = np.inf, -np.inf, 3e38
    x[6, 70], x[7, 0], x[7, 127] = np.nan, -np.nan, np.inf
    wide = torch.zeros((8, 128 + offset), device="cuda:0")
    v = wide[:, offset:]
    v.copy_(dev(x))
    E.kv_append(b, 0, v, v, v, k_weight=torch.ones(128, device="cuda:0") if norm else None)
    raw = c.pool.cpu().numpy().reshape(2, 2, -1)[0]
    blocks = E.quantize_q8_0(dev(x)).cpu().numpy().reshape(8, 4, 34)
    for which in (0, 1):
        codes = raw[which, : 16 * 128].reshape(16, 4, 32)[:8]
        d = raw[which, 16 * 128:].copy().view(np.float16).reshape(16, 4)[:8]
        if which == 0 and norm:  # one that is not finite reaches all of its head
            assert np.isnan(d[[6, 7]]).all() and not np.isnan(d[:3]).any()
            continue
        nan = np.isnan(x).reshape(8, 4, 32).any(-1)
        assert np.array_equal(np.isnan(d), nan)
        assert np.array_equal(d[~nan].view(np.uint16), blocks[..., :2].copy().view(np.uint16).reshape(8, 4)[~nan])
        assert np.array_equal(codes[~nan], blocks[..., 2:][~nan])


# ------------------------------------------------------------------ pages


@pytest.mark.parametrize("qtype", TYPES)
def test_page_copies(hipdev, qtype):
    """Copy on write, copies at once and compaction move the tokens' bytes and nothing else."""
    rng = np.random.default_rng(qtype + 40)
    layers, kv, dim, page, pages = 3, 2, 96, 16, 700
    c = make(rng, qtype, kv, dim, page, pages, 400, layers=layers)
    model = P.decode(c.pool, qtype, layers, pages, kv, page, dim)
    a, b = c.new(), c.new()
    c.extend([a, b], [40, 7])
    kids = c.fork([a, b, a])
    before = c.tables(kids)
    c.extend(kids, [1, 1, 30])
    for i, s in enumerate(kids):
        used = (40, 7, 40)[i]
        src, dst = before[i][used // page], c.tables([s])[0][used // page]
        assert src != dst
        model[:, dst, :, :, : used % page] = model[:, src, :, :, : used % page]
    assert np.array_equal(P.decode(c.pool, qtype, layers, pages, kv, page, dim), model)
    # more copies than one launch takes
    many = c.fork([kids[2]] * 60, copy=True)
    n = c.length(kids[2])
    src = c.tables([kids[2]])[0]
    for s in many:
        for i, dst in enumerate(c.tables([s])[0]):
            used = min(page, n - i * page)
            model[:, dst, :, :, :used] = model[:, src[i], :, :, :used]
    assert len(set(c.tables(many).reshape(-1))) == 60 * len(src) > 256
    assert np.array_equal(P.decode(c.pool, qtype, layers, pages, kv, page, dim), model)
    c.release([a, kids[0]] + many[: 30])
    live = [b, kids[1], kids[2]] + many[30:]
    old = c.tables(live)
    n_used = c.compact()
    new = c.tables(live)
    for o, m in zip(old, new):
        for p, r in zip(o, m):
            assert (p < 0) == (r < 0)
            if p >= 0 and p != r:
                assert p >= n_used > r
                model[:, r] = model[:, p]
    assert sorted(set(new[new >= 0])) == list(range(n_used)) and c.free_pages() == pages - n_used
    assert np.array_equal(P.decode(c.pool, qtype, layers, pages, kv, page, dim), model)


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("qtype", TYPES)
def test_a_prompt_then_forked_answers(hipdev, qtype):
    """A prompt in two chunks, then steps of several answers that share it, two layers, as a serving loop makes them."""
    rng = np.random.default_rng(60 + qtype)
    layers, kv, heads, dim, page, pages = 2, 2, 8, 64, 32, 120
    c = make(rng, qtype, kv, dim, page, pages, 12, layers=layers)
    wq, wk = (rng.standard_normal(dim).astype(np.float32) for _ in range(2))
    rope = E.Rope(dim, 10000.0)
    batch = E.KvBatch(c, heads, 12, 400)

    def step(seqs, n_new):
        c.extend(seqs, n_new)
        batch.set(seqs, n_new)
        T = sum(n_new)
        for layer in range(layers):
            x = rng.standard_normal((T, (heads + 2 * kv) * dim)).astype(np.float32)
            q, k, v = dev(x).split([heads * dim, kv * dim, kv * dim], 1)
            qr = E.kv_append(batch, layer, q, k, v, rope, dev(wq), dev(wk))
            got = E.attention(batch, layer, qr).cpu().numpy()
            vals, at = pool_values(c, qtype, layers, pages, page), 0
            eps = float(np.float32(1e-6))
            for s, m in zip(seqs, n_new):
                if m == 0:
                    continue
                n = c.length(s)
                k64, v64 = P.values(vals, layer, [p for p in c.tables([s])[0] if p >= 0], n)
                pos = np.arange(n - m, n)
                y = x[at: at + m].reshape(m, heads + 2 * kv, dim)
                # the cache holds what was given: 32 bits, half a step of f16, half a code and half a step of the scale
                for g, w in ((k64, P.rotated(y[:, heads: heads + kv], wk, eps, pos, dim)), (v64, y[:, heads + kv:])):
                    step_of = {E.F32: 0.0, E.F16: P.EPS16, E.Q8_0: 1 / 254 + P.EPS16}[qtype]
                    err = np.abs(g[:, n - m:].transpose(1, 0, 2) - w)
                    assert np.all(err <= np.abs(w).max() * (step_of + 30 * P.EPS32) * 1.01)
                qs = qr[at: at + m].cpu().numpy().reshape(m, heads, dim)
                want, tol = P.attend(qs, k64, v64, n - m, dim ** -0.5, qtype)
                assert np.all(np.abs(got[at: at + m].reshape(m, heads, dim) - want) <= tol)
                at += m

    a = c.new()
    step([a], [200])
    step([a], [77])
    kids = c.fork([a] * 5)
    for i in range(3):
        step(kids, [1, 1, 1 + i, 1, 0])
    more = c.fork(kids[:2])
    c.release(kids[2:4])
    c.compact()
    step(more + kids[:2] + [a], [1, 2, 1, 1, 4])
    c.truncate(kids[0], 100)
    step([kids[0], kids[4]], [3, 1])


def test_captured_step_replays_later_plans(hipdev):
    """One graph of a layer's write and attention, replayed after other sets, with eager work between."""
    rng = np.random.default_rng(8)
    kv, heads, dim, page, pages = 2, 8, 128, 64, 200
    c = make(rng, E.F16, kv, dim, page, pages, 9)
    root = c.new()
    c.extend([root], [3000])
    kids = c.fork([root] * 6)
    c.extend(kids, [50 * i + 1 for i in range(6)])
    batch = E.KvBatch(c, heads, 8, 12)
    eager = E.KvBatch(c, heads, 8, 12)
    x = dev(rng.standard_normal((12, (heads + 2 * kv) * dim)).astype(np.float32))
    q, k, v = x.split([heads * dim, kv * dim, kv * dim], 1)
    rope = E.Rope(dim)
    qr, out = torch.zeros((12, heads * dim), device="cuda:0"), torch.zeros((12, heads * dim), device="cuda:0")
    batch.set(kids, [2] * 6)  # the largest plan first
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.kv_append(batch, 0, q, k, v, rope, q_out=qr)
        E.attention(batch, 0, qr, out=out)
    for n_new in ([2] * 6, [1, 0, 1, 2, 1, 1], [0] * 6, [1] * 6, [0, 0, 0, 0, 0, 12 - 6], [2] * 6):
        ids = kids
        c.extend(ids, [1, 0, 1, 0, 2, 0])
        n_new = [min(n, c.length(s)) for s, n in zip(ids, n_new)]
        T = sum(n_new)
        batch.set(ids, n_new)
        eager.set(ids, n_new)
        for _ in range(3):
            out.fill_(-1.0)
            graph.replay()
            junk = torch.randn(1 << 20, device="cuda:0").sum()
            torch.cuda.synchronize()
            if T:
                want_q = E.kv_append(eager, 0, q, k, v, rope)
                want = E.attention(eager, 0, want_q)
                assert torch.equal(qr[:T], want_q) and torch.equal(out[:T], want)
            assert bool((out[T:] == -1.0).all()) and torch.isfinite(junk)
    # a plan that outgrows the captured buffers, and a set inside a capture, are refused
    big = E.KvBatch(c, heads, 8, 12)
    lone = c.new()
    c.extend([lone], [10])
    big.set([lone], [1])
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        E.attention(big, 0, qr, out=out)
        with pytest.raises(E.HipError, match="captured"):
            big.set([lone], [1])
        with pytest.raises(E.HipError, match="captured"):
            c.extend([lone], [1])
    with pytest.raises(E.HipError, match="outgrows"):
        big.set(kids, [1] * 6)
    big.set([lone], [1])
    E.attention(big, 0, qr)


def test_a_captured_step_bounds_later_plans(hipdev):
    """More tokens than the captured call's buffers hold, and slots that a captured append may not write, are refused."""
    rng = np.random.default_rng(20)
    c = make(rng, E.F16, 1, 64, 16, 120, 6)
    a, e = c.new(), c.new()
    c.extend([a, e], [40, 50])
    b = E.KvBatch(c, 1, 4, 64)
    k = dev(rng.standard_normal((2, 64)).astype(np.float32))
    q, qr, out = dev(rng.standard_normal((2, 64)).astype(np.float32)), torch.zeros((2, 64), device="cuda:0"), torch.zeros((2, 64), device="cuda:0")
    b.set([a, e], [1, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.kv_append(b, 0, q, k, k, q_out=qr)
        E.attention(b, 0, qr, out=out)
    with pytest.raises(E.HipError, match="3 tokens outgrows"):
        b.set([a, e], [2, 1])
    assert b.tokens() == 2
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, E.attention(b, 0, q))
    (f,) = c.fork([e])
    with pytest.raises(E.HipError, match="appends"):
        b.set([a, e], [1, 1])
    c.extend([f], [1])
    b.set([a, f], [1, 1])
    before = c.pool.clone()
    graph.replay()
    torch.cuda.synchronize()
    x = (c.pool != before).view(120, -1).any(1).nonzero().flatten().tolist()
    assert set(x) <= {int(c.tables([a])[0].max()), int(c.tables([f])[0, 50 // 16])}
    # read only: shared slots are no matter
    r = E.KvBatch(c, 1, 4, 64)
    r.set([a, f], [1, 1])
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        E.attention(r, 0, q, out=out)
    c.fork([f])
    r.set([a, f], [1, 1])
    # as many tokens, but in pieces that need a workspace
    g = c.new()
    c.extend([g], [1000])
    with pytest.raises(E.HipError, match="outgrows the workspace"):
        r.set([g], [1])


def test_no_tokens(hipdev):
    rng = np.random.default_rng(4)
    c = make(rng, E.F16, 2, 64, 16, 8, 3)
    s = c.new()
    c.extend([s], [20])
    b = E.KvBatch(c, 4, 2, 8)
    none = torch.empty((0, 256), device="cuda:0")
    for ids, n_new in (([], []), ([s], [0])):
        b.set(ids, n_new)
        assert E.attention(b, 0, none).shape == (0, 256)
        assert E.kv_append(b, 0, none, none[:, :128], none[:, :128]).shape == (0, 256)
    e = c.new()
    assert c.fork([e]) and c.length(e) == 0 and c.tables([e]).shape == (1, 0)
    b.set([e, s], [0, 1])
    check_attention(c, E.F16, 1, 8, 16, [e, s], [0, 1], 4, rng)


def test_nan_reaches_its_rows_only(hipdev):
    """A NaN key or query makes its own rows NaN through every split of the keys, and no others."""
    rng = np.random.default_rng(14)
    for qtype in (E.F16, E.F32, E.Q8_0):
        c = make(rng, qtype, 1, 128, 64, 300, 3)
        a, e = c.new(), c.new()
        c.extend([a, e], [9000, 9000])
        b = E.KvBatch(c, 2, 2, 2)
        b.set([a, e], [1, 1])
        q = dev(rng.standard_normal((2, 256)).astype(np.float32))
        before = E.attention(b, 0, q).clone()
        q2 = q.clone()
        q2[1, 130] = float("nan")
        got = E.attention(b, 0, q2)
        assert torch.equal(got[0], before[0]) and torch.equal(got[1, :128], before[1, :128]) and got[1, 128:].isnan().all()
        page = c.tables([a])[0][3]
        raw = c.pool.view(300, 2, -1)
        if qtype == E.Q8_0:
            raw[page, 0, 64 * 128 + 10 * 8: 64 * 128 + 10 * 8 + 2] = dev(np.full(1, np.nan, np.float16).view(np.uint8))
        else:
            raw[page, 0].view(torch.float16 if qtype == E.F16 else torch.float32)[10 * 128 + 5] = float("nan")
        got = E.attention(b, 0, q)
        assert got[0].isnan().all() and torch.equal(got[1], before[1])


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("bits", [0x7C00, 0xFC00, 0x7E00])
def test_a_scale_that_is_not_finite_spoils_its_block_only(hipdev, dim, new, bits):
    rng = np.random.default_rng(bits + dim + new)
    kv, group, page, n = 1, 4, 64, 400
    c = make(rng, E.Q8_0, kv, dim, page, 8, 2)
    s = c.new()
    c.extend([s], [n])
    pages = c.tables([s])[0]
    raw = c.pool.cpu().numpy().reshape(8, 2, -1)
    scales = raw[..., page * dim:].view(np.uint16).reshape(8, 2, page, dim // 32)
    scales[pages[0], 1, 5, 1] = bits
    # the largest scale of all, next to it: the sums of its block are in range, and those of the others exact
    scales[pages[0], 1, 4, 0] = np.float16(30.0).view(np.uint16)
    c.pool.copy_(torch.from_numpy(raw.reshape(-1)))
    scales[pages[0], 1, 5, 1] = 0
    vals = P.decode(torch.from_numpy(raw.reshape(-1)), E.Q8_0, 1, 8, kv, page, dim)
    q = rng.standard_normal((new, group * kv * dim)).astype(np.float32)
    b = E.KvBatch(c, group * kv, 1, new)
    b.set([s], [new])
    got = E.attention(b, 0, dev(q)).cpu().numpy().reshape(new, group * kv, dim)
    k, v = P.values(vals, 0, [p for p in pages if p >= 0], n)
    want, tol = P.attend(q.reshape(new, group * kv, dim), k, v, n - new, dim ** -0.5, E.Q8_0)
    assert not np.isfinite(got[..., 32:64]).any()
    got[..., 32:64] = want[..., 32:64]
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


def test_two_batches_on_two_streams(hipdev):
    rng = np.random.default_rng(21)
    c = make(rng, E.Q8_0, 4, 128, 64, 300, 8)
    a, b = c.new(), c.new()
    c.extend([a, b], [9000, 4000])
    q = dev(rng.standard_normal((2, 16 * 128)).astype(np.float32))
    batches = [E.KvBatch(c, 16, 2, 2) for _ in range(2)]
    for x, s in zip(batches, (a, b)):
        x.set([s], [2])
    want = [E.attention(x, 0, q).clone() for x in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, x in zip(streams, batches):
            with torch.cuda.stream(st):
                got.append(E.attention(x, 0, q))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_results_repeat_bit_for_bit_and_in_place(hipdev):
    rng = np.random.default_rng(33)
    c = make(rng, E.F16, 2, 128, 32, 500, 20)
    root = c.new()
    c.extend([root], [5000])
    kids = c.fork([root] * 16)
    c.extend(kids, [10 * i + 1 for i in range(16)])
    b = E.KvBatch(c, 8, 16, 16)
    b.set(kids, [1] * 16)
    q = dev(rng.standard_normal((16, 8 * 128)).astype(np.float32))
    want = E.attention(b, 0, q).clone()
    for _ in range(4):
        assert torch.equal(E.attention(b, 0, q), want)
    assert torch.equal(E.attention(b, 0, q, out=q), want)


def test_refusals(hipdev):
    rng = np.random.default_rng(1)
    c = make(rng, E.F16, 2, 64, 16, 10, 3, layers=2)
    L, s = hipdev, c.new()
    c.extend([s], [20])
    b = E.KvBatch(c, 4, 2, 8)
    q = torch.zeros((8, 256), device="cuda:0")
    k = torch.zeros((8, 128), device="cuda:0")
    with pytest.raises(E.HipError, match="not set"):
        E.attention(b, 0, q)
    b.set([s], [2])
    out = E.attention(b, 0, q)
    assert out.shape == (2, 256)
    for call, what in [
        (lambda: E.attention(b, 2, q), "layer 2"), (lambda: E.attention(b, -1, q), "layer -1"),
        (lambda: b.set([s], [21]), "21 new tokens"), (lambda: b.set([s], [9]), "9 tokens"), (lambda: b.set([s, s], [1, 1]), "twice"),
        (lambda: b.set([5], [1]), "not in use"), (lambda: b.set([s, s, s], [0, 0, 0]), "3 sequences"),
        (lambda: c.extend([s], [16 * 10]), "free pages"), (lambda: c.fork([s, 2]), "not in use"),
        (lambda: c.release([s, s]), "twice"), (lambda: c.truncate(s, 21), "count"), (lambda: E.KvBatch(c, 5, 1, 1), "5 heads"),
        (lambda: E.KvCache(E.Q4_K, 1, 1, 64, 16, 4, 1, pool=q.view(torch.uint8).view(-1)[:0]), "supported"),
        (lambda: E.kv_append(b, 0, q, k, k, E.Rope(128)), "128 values"),
    ]:
        with pytest.raises(E.HipError, match=what):
            call()
    for call in (lambda: E.attention(b, 0, q[:1]), lambda: E.attention(b, 0, q.half()), lambda: E.attention(b, 0, q.cpu()),
                 lambda: E.attention(b, 0, q, out=q[:, :200]), lambda: E.kv_append(b, 0, q, k[:1], k),
                 lambda: E.kv_append(b, 0, q, k, k, q_weight=k[0, :32]), lambda: E.kv_append(b, 0, q, k.double(), k),
                 lambda: c.extend([s], [1, 2]), lambda: b.set([s], []), lambda: c.length(2),
                 lambda: E.KvCache(E.F16, 1, 1, 64, 16, 4, 1, pool=q.view(torch.uint8).view(-1)),
                 lambda: E.Rope(64, factors=[1.0] * 31), lambda: E.qk_norm_rope(q, k, 3, 2, None),
                 lambda: E.qk_norm_rope(q, k, 4, 2, torch.zeros(7, dtype=torch.int32, device="cuda:0"))):
        with pytest.raises(ValueError):
            call()
    # a batch set refused leaves the batch unset; a change of the cache makes it stale
    b.set([s], [2])
    E.kv_append(b, 1, q, k, k)
    c.extend([s], [1])
    with pytest.raises(E.HipError, match="stale"):
        E.attention(b, 0, q)
    b.set([s], [1])
    (f,) = c.fork([s])
    b.set([s], [1])
    E.attention(b, 0, q)
    with pytest.raises(E.HipError, match="another sequence"):
        E.kv_append(b, 0, q, k, k)
    assert not L.attention_dev(None, q.data_ptr(), b._h, 0, 1.0, None)
    L.clear_error()
    assert not L.attention_dev(q.data_ptr(), q.data_ptr() + 4, b._h, 0, 1.0, None)
    L.clear_error()
    for scale in (float("nan"), float("inf")):
        with pytest.raises(E.HipError, match="finite"):
            E.attention(b, 0, q, scale)
    assert not L.kv_append_dev(q.data_ptr(), q.data_ptr(), 255, k.data_ptr(), 128, k.data_ptr(), 128, b._h, 0, None, None,
                               0.0, None, None)
    L.clear_error()
    assert not L.kv_destroy(c._h)
    assert "batches" in L.last_error()[1]
    L.clear_error()
