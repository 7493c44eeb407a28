"""Routing to experts and the experts' products, against plain forms in 64 bits."""
import numpy as np
import pytest
import torch

import edgexpu_amd as E
import moe_plain as P
from edgexpu_amd import synth

pytestmark = pytest.mark.gpu

TYPES = [E.Q4_K, E.Q6_K, E.Q8_0, E.Q5_K, E.Q4_0, E.Q5_0]


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def host(t):
    return t.cpu().numpy()


def experts(qtype, n, rows, k, rng):
    return synth.np_weights(qtype, n * rows, k, rng).reshape(n, rows, -1)


# ------------------------------------------------------------------ routing


def check_route(scores, k, **kw):
    m, n = scores.shape
    plan = E.MoePlan(n, k, m + 2, 32, 32)
    bias = kw.get("bias")
    ids = torch.full((m, k), 77, dtype=torch.int32, device="cuda:0")
    names = dict(n_groups="n_groups", top_groups="top_groups", best="group_best", normalise="normalise", scale="scale",
                 score="score")
    got, w = E.moe_route(plan, dev(scores), bias=None if bias is None else dev(bias), ids=ids,
                         **{names[a]: v for a, v in kw.items() if a in names})
    assert got is ids and plan.tokens() == m
    want, ww = P.route(scores, k, **kw)
    assert np.array_equal(host(ids), want)
    # a handful of roundings in 64 bits, then half a step of f32
    assert np.all(np.abs(host(w) - ww) <= P.U * 1.0001 * np.abs(ww) + 2.0 ** -149)
    return plan, want, host(w)


@pytest.mark.parametrize("n,k,m", [(1, 1, 1), (2, 1, 3), (4, 4, 5), (8, 2, 1), (60, 4, 77), (64, 6, 64), (65, 8, 9),
                                   (128, 8, 1), (128, 8, 300), (256, 32, 5), (511, 10, 33), (512, 32, 4)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route(hipdev, n, k, m, score):
    rng = np.random.default_rng(n * 1000 + m)
    s = (rng.standard_normal((m, n)) * 2).astype(np.float32)
    check_route(s, k, score=score)
    check_route(s, k, score=score, bias=(rng.standard_normal(n) * 0.3).astype(np.float32), normalise=False, scale=2.5)


@pytest.mark.parametrize("n,groups,top,best,k", [(8, 2, 1, 1, 3), (64, 8, 4, 2, 6), (256, 8, 4, 2, 8), (64, 64, 7, 1, 7),
                                                 (60, 4, 3, 2, 10), (512, 16, 1, 2, 32), (6, 6, 2, 2, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_in_groups(hipdev, n, groups, top, best, k, score):
    rng = np.random.default_rng(n + groups)
    s = rng.standard_normal((21, n)).astype(np.float32)
    s[3, rng.random(n) < 0.6] = -np.inf
    s[4] = -np.inf
    s[5, : n // groups] = np.nan
    b = (rng.standard_normal(n) * 0.2).astype(np.float32)
    for bias in (None, b):
        check_route(s, k, score=score, bias=bias, n_groups=groups, top_groups=top, best=best)


def test_route_values_apart_from_the_ordinary(hipdev):
    rng = np.random.default_rng(5)
    n = 70
    s = rng.standard_normal((14, n)).astype(np.float32)
    s[0] = -np.inf
    s[1] = np.nan
    s[2] = np.inf
    s[3, ::2] = np.nan
    s[4, 1:] = -np.inf
    s[5] = 1.25  # equal: the lowest numbers
    s[6, 40:50] = 3.0
    s[7] *= 1e4  # most shares vanish
    s[8] = np.finfo(np.float32).max * np.sign(s[8])
    s[9] = np.finfo(np.float32).tiny * s[9]
    s[10, 3] = np.inf
    s[11] = np.finfo(np.float32).min  # the type's lowest value is a score like any other
    s[12] = -60.0  # sigmoids far below 2^-53
    s[13] = 60.0
    b = np.zeros(n, np.float32)
    b[[2, 9]] = np.nan, np.inf
    b[11] = -np.inf
    for score in ("softmax", "sigmoid"):
        for bias in (None, b):
            for normalise in (True, False):
                check_route(s, 9, score=score, bias=bias, normalise=normalise)


def test_route_without_copies_and_tokens(hipdev):
    plan = E.MoePlan(8, 2, 4, 256, 256)
    with pytest.raises(E.HipError, match="no routing yet"):
        E.moe_down(plan, dev(np.zeros((8, 256, 144), np.uint8)), E.Q4_K, torch.zeros((0, 2, 256), device="cuda:0"))
    ids, w = E.moe_route(plan, torch.zeros((0, 8), device="cuda:0"))
    assert ids.shape == (0, 2) and plan.tokens() == 0
    wz = dev(np.zeros((8, 256, 144), np.uint8))
    assert E.moe_gate_up(plan, wz, wz, E.Q4_K, torch.zeros((0, 256), device="cuda:0")).shape == (0, 2, 256)
    assert E.moe_down(plan, wz, E.Q4_K, torch.zeros((0, 2, 256), device="cuda:0")).shape == (0, 256)
    s = torch.randn((4, 8), device="cuda:0")
    L = hipdev
    assert L.moe_route_dev(plan._h, None, None, s.data_ptr(), 4, 0, None, 1, 1, 1, 1, 1.0, torch.cuda.current_stream().cuda_stream)
    assert plan.tokens() == 4


# ------------------------------------------------------------------ products


def random_ids(rng, m, n, k, none=0.0):
    ids = np.stack([rng.permutation(n)[:k] for _ in range(m)]).astype(np.int32)
    ids[rng.random((m, k)) < none] = -1
    return ids


def check_gate_up(qtype, n, k, m, n_embd, n_ff, seed=1, bias=True, act="silu", ids=None, x=None, none=0.1):
    rng = np.random.default_rng(seed)
    wg, wu = experts(qtype, n, n_ff, n_embd, rng), experts(qtype, n, n_ff, n_embd, rng)
    if x is None:
        x = rng.standard_normal((m, n_embd)).astype(np.float32)
    bg = rng.standard_normal((n, n_ff)).astype(np.float32) if bias else None
    bu = rng.standard_normal((n, n_ff)).astype(np.float32) if bias else None
    if ids is None:
        ids = random_ids(rng, m, n, k, none)
    plan = E.MoePlan(n, k, m + 3, n_embd, n_ff)
    plan.assign(dev(ids), dev(rng.random((m, k)).astype(np.float32)))
    out = torch.full((m + 3, k, n_ff), 7.5, device="cuda:0")
    E.moe_gate_up(plan, dev(wg), dev(wu), qtype, dev(x), b_gate=None if bg is None else dev(bg),
                  b_up=None if bu is None else dev(bu), activation=act, act=out)
    got = host(out)
    assert np.all(got[m:] == 7.5), "rows behind the last token were written"
    want, tol = P.gate_up(qtype, x, wg, wu, ids, bg, bu, act)
    err = np.abs(got[:m] - want)
    assert np.all(err <= tol), (float((err / (tol + 1e-300)).max()), np.argwhere(err > tol)[:4])
    assert np.all(got[:m][(ids < 0) | (ids >= n)] == 0)


def check_down(qtype, n, k, m, n_embd, n_ff, seed=1, bias=True, residual=True, ids=None, act=None, none=0.1, inplace=False):
    rng = np.random.default_rng(seed)
    w = experts(qtype, n, n_embd, n_ff, rng)
    if act is None:
        act = (rng.standard_normal((m, k, n_ff)) * rng.random((m, k, 1))).astype(np.float32)
    b = rng.standard_normal((n, n_embd)).astype(np.float32) if bias else None
    r = rng.standard_normal((m, n_embd)).astype(np.float32) if residual else None
    if ids is None:
        ids = random_ids(rng, m, n, k, none)
    g = rng.standard_normal((m, k)).astype(np.float32)
    plan = E.MoePlan(n, k, m + 2, n_embd, n_ff)
    plan.assign(dev(ids), dev(g))
    out = torch.full((m + 2, n_embd), 7.5, device="cuda:0")
    res = None if r is None else dev(r)
    if inplace:
        out[:m] = res
        res = out
    E.moe_down(plan, dev(w), qtype, dev(act), bias=None if b is None else dev(b), residual=res, out=out)
    got = host(out)
    assert np.all(got[m:] == 7.5), "rows behind the last token were written"
    want, tol = P.down(qtype, act, w, ids, g, b, r)
    err = np.abs(got[:m] - want)
    assert np.all(err <= tol), (float((err / (tol + 1e-300)).max()), np.argwhere(err > tol)[:4])


# (experts, top_k, tokens, n_embd, n_ff): one token, few, ragged, many; rows that fill no tile
SIZES = [(4, 2, 1, 256, 256), (8, 2, 1, 1024, 512), (16, 4, 1, 512, 300), (5, 1, 2, 256, 17), (8, 3, 3, 768, 256),
         (3, 3, 5, 512, 40), (16, 4, 7, 512, 272), (8, 2, 16, 256, 256), (7, 2, 33, 512, 257), (4, 2, 64, 256, 130),
         (6, 3, 100, 256, 96), (2, 1, 150, 512, 64), (40, 5, 77, 256, 33), (3, 2, 300, 256, 48)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("qtype", TYPES, ids=lambda t: E.TYPE_NAMES[t])
def test_gate_up(hipdev, qtype, size):
    n, k, m, n_embd, n_ff = size
    check_gate_up(qtype, n, k, m, n_embd, n_ff, seed=m)
    check_gate_up(qtype, n, k, m, n_embd, n_ff, seed=m + 1, bias=False, act="gelu", none=0.0)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("qtype", TYPES, ids=lambda t: E.TYPE_NAMES[t])
def test_down(hipdev, qtype, size):
    n, k, m, a, b = size
    check_down(qtype, n, k, m, b, a, seed=m)
    check_down(qtype, n, k, m, b, a, seed=m + 1, bias=False, residual=False, none=0.0)


@pytest.mark.parametrize("m", [1, 4, 20, 70])
@pytest.mark.parametrize("qtype,n_in", [(E.Q8_0, 32), (E.Q8_0, 96), (E.Q8_0, 608), (E.Q4_0, 32), (E.Q4_0, 160), (E.Q5_0, 224),
                                        (E.Q5_0, 32), (E.Q4_K, 1792), (E.Q6_K, 2816), (E.Q5_K, 4352), (E.Q8_0, 4128)])
def test_odd_row_lengths(hipdev, qtype, n_in, m):
    check_gate_up(qtype, 6, 2, m, n_in, 50, seed=n_in)
    check_down(qtype, 6, 2, m, 50, n_in, seed=n_in)


@pytest.mark.parametrize("m", [1, 3, 9, 40, 130])
@pytest.mark.parametrize("qtype", [E.Q4_K, E.Q8_0], ids=lambda t: E.TYPE_NAMES[t])
def test_crowded_and_empty_experts(hipdev, qtype, m):
    """All tokens at one expert; a token that names an expert twice; tokens and steps without any expert."""
    one = np.full((m, 2), 3, np.int32)
    one[:, 1] = 5
    twice = np.full((m, 2), 4, np.int32)
    none = np.full((m, 2), -1, np.int32)
    some = none.copy()
    some[-1] = [0, 7]
    wild = np.where(np.arange(2 * m).reshape(m, 2) % 3 == 0, 8, np.where(np.arange(2 * m).reshape(m, 2) % 3 == 1, 2 ** 31 - 1, 1)).astype(np.int32)
    wild[0, 0] = -(2 ** 31)
    for ids in (one, twice, none, some, wild):
        check_gate_up(qtype, 8, 2, m, 512, 48, ids=ids)
        check_down(qtype, 8, 2, m, 48, 512, ids=ids, inplace=True)


# where the work is shared out otherwise: (experts, choices, tokens, n_embd, n_ff)
SHARES = [(2, 2, 200, 768, 50), (3, 3, 150, 1280, 33),  # more than 128 pairs an expert
          (8, 2, 100, 768, 70), (6, 2, 66, 512, 129),  # more than 16
          (4, 2, 12, 1280, 96), (4, 2, 12, 256, 34), (8, 2, 9, 768, 47),  # few tiles
          (64, 4, 8, 512, 40), (64, 4, 9, 512, 40), (8, 2, 4, 256, 31), (8, 2, 5, 256, 31)]  # from single tokens to tiles


@pytest.mark.parametrize("size", SHARES, ids=str)
@pytest.mark.parametrize("qtype", TYPES, ids=lambda t: E.TYPE_NAMES[t])
def test_every_share_of_the_work(hipdev, qtype, size):
    n, k, m, wide, narrow = size
    check_gate_up(qtype, n, k, m, wide, narrow, seed=5)
    check_down(qtype, n, k, m, narrow, wide, seed=6)  # (the products run over the same lengths)


@pytest.mark.parametrize("m", [1, 3, 40, 200])
def test_an_expert_named_twice(hipdev, m):
    """A token's places are summed one by one, whichever experts they name."""
    rng = np.random.default_rng(m)
    ids = rng.integers(-1, 3, (m, 4)).astype(np.int32)
    ids[0] = 1
    check_gate_up(E.Q5_K, 6, 4, m, 512, 40, seed=8, ids=ids)
    check_down(E.Q6_K, 6, 4, m, 40, 512, seed=9, ids=ids)


def test_more_pairs_than_one_round_of_the_sort(hipdev):
    m, rng = 12000, np.random.default_rng(3)
    ids = random_ids(rng, m, 5, 3, 0.2)
    ids[:9000] = np.where(ids[:9000] == 4, -1, ids[:9000])  # (an expert whose pairs all come late)
    ids[100:5000] = np.where(ids[100:5000] == 0, -1, ids[100:5000])
    check_gate_up(E.Q8_0, 5, 3, m, 64, 8, seed=10, ids=ids)
    check_down(E.Q4_0, 5, 3, m, 8, 64, seed=11, ids=ids)


@pytest.mark.parametrize("n_ff", [12800, 14336])
@pytest.mark.parametrize("qtype", [E.Q4_K, E.Q6_K, E.Q8_0], ids=lambda t: E.TYPE_NAMES[t])
def test_one_token_of_long_rows(hipdev, qtype, n_ff):
    """Four rows of 50 groups are quantized by one workgroup, of 56 are not."""
    for none in (0.0, 0.5):
        check_down(qtype, 5, 4, 1, 35, n_ff, seed=7, none=none)


@pytest.mark.parametrize("qtype", TYPES, ids=lambda t: E.TYPE_NAMES[t])
@pytest.mark.parametrize("m", [1, 6, 50])
def test_zero_and_wide_activations(hipdev, qtype, m):
    """Blocks of zeros, and values of many magnitudes."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((m, 768)).astype(np.float32) * np.exp(rng.uniform(-12, 3, (m, 768))).astype(np.float32)
    x[:, 256:512] = 0
    x[m // 2] = 0
    check_gate_up(qtype, 4, 2, m, 768, 33, x=x)
    act = np.repeat(x[:, None], 2, 1)
    check_down(qtype, 4, 2, m, 33, 768, act=act)


@pytest.mark.parametrize("m", [1, 5, 40])
def test_activations_that_are_no_numbers_stay_in_their_rows(hipdev, m):
    """Another token's NaN, or its row behind the last token, changes no word."""
    rng = np.random.default_rng(3)
    n, k = 4, 2
    for qtype in (E.Q4_K, E.Q8_0):
        w = dev(experts(qtype, n, 64, 256, rng))
        x = dev(rng.standard_normal((m + 1, 256)).astype(np.float32))
        ids, g = dev(random_ids(rng, m + 1, n, k)), dev(rng.random((m + 1, k)).astype(np.float32))
        plan = E.MoePlan(n, k, m + 1, 256, 64)
        down = E.MoePlan(n, k, m + 1, 64, 256)
        plan.assign(ids, g)
        down.assign(ids, g)
        a = dev(rng.standard_normal((m + 1, k, 256)).astype(np.float32))
        want, wd = E.moe_gate_up(plan, w, w, qtype, x).clone(), E.moe_down(down, w, qtype, a).clone()
        x[m] = float("nan")
        a[m] = float("inf")
        assert torch.equal(E.moe_gate_up(plan, w, w, qtype, x)[:m], want[:m])
        assert torch.equal(E.moe_down(down, w, qtype, a)[:m], wd[:m])


def test_the_products_are_the_dense_ones(hipdev):
    """One expert that every token takes: the words of the dense projections are those of this product within f32 sums."""
    rng = np.random.default_rng(8)
    for qtype, m in ((E.Q4_K, 1), (E.Q6_K, 5), (E.Q8_0, 40)):
        w = experts(qtype, 1, 96, 512, rng)
        x = rng.standard_normal((m, 512)).astype(np.float32)
        plan = E.MoePlan(1, 1, m, 512, 96)
        plan.assign(torch.zeros((m, 1), dtype=torch.int32, device="cuda:0"), torch.ones((m, 1), device="cuda:0"))
        got = host(E.moe_gate_up(plan, dev(w), dev(w), qtype, dev(x)))[:, 0]
        y = E.linear_quant_batch(dev(w[0]), qtype, dev(x), 96, 512)
        dense = host(E.silu_mul(y, y))
        _, tol = P.gate_up(qtype, x, w, w, np.zeros((m, 1), np.int32))
        assert np.all(np.abs(got - dense) <= 2 * tol[:, 0])


# ------------------------------------------------------------------ as a step uses them


class Layer:
    def __init__(self, qtype, down_type, n, k, n_embd, n_ff, seed=4):
        rng = np.random.default_rng(seed)
        self.q, self.dq, self.n, self.k, self.n_embd, self.n_ff = qtype, down_type, n, k, n_embd, n_ff
        self.router = (rng.standard_normal((n, n_embd)) / np.sqrt(n_embd)).astype(np.float32)
        self.gate, self.up = experts(qtype, n, n_ff, n_embd, rng), experts(qtype, n, n_ff, n_embd, rng)
        self.down = experts(down_type, n, n_embd, n_ff, rng)
        self.dev = {a: dev(getattr(self, a)) for a in ("gate", "up", "down")}
        self.dev["router"] = dev(self.router.view(np.uint8))
        self.norm = dev(np.ones(n_embd, np.float32))

    def step(self, plan, h, keep=None):
        x = E.rmsnorm(h, self.norm, 1e-5)
        s = E.linear_quant_batch(self.dev["router"], E.F32, x, self.n, self.n_embd)
        ids, w = E.moe_route(plan, s)
        act = E.moe_gate_up(plan, self.dev["gate"], self.dev["up"], self.q, x)
        out = E.moe_down(plan, self.dev["down"], self.dq, act, residual=h)
        if keep is not None:
            keep.update(x=x, s=s, ids=ids, w=w, act=act, out=out)
        return out


def check_step(layer, k):
    """Each call of a step on what the call before it gave."""
    ids, w = P.route(host(k["s"]), layer.k)
    assert np.array_equal(host(k["ids"]), ids) and np.allclose(host(k["w"]), w, rtol=1e-7, atol=0)
    want, tol = P.gate_up(layer.q, host(k["x"]), layer.gate, layer.up, ids)
    assert np.all(np.abs(host(k["act"]) - want) <= tol)
    want, tol = P.down(layer.dq, host(k["act"]), layer.down, ids, host(k["w"]), residual=host(k["h"]))
    assert np.all(np.abs(host(k["out"]) - want) <= tol)


@pytest.mark.parametrize("m", [1, 2, 6, 31, 90])
@pytest.mark.parametrize("qtype,down", [(E.Q4_K, E.Q6_K), (E.Q8_0, E.Q8_0), (E.Q5_K, E.Q5_0)], ids=str)
def test_a_step(hipdev, qtype, down, m):
    layer = Layer(qtype, down, 16, 4, 512, 256)
    plan = E.MoePlan(16, 4, m, 512, 256)
    h = torch.randn((m, 512), device="cuda:0", generator=torch.Generator(device="cuda:0").manual_seed(m))
    kept = dict(h=h.clone())
    layer.step(plan, h, kept)
    check_step(layer, kept)


@pytest.mark.parametrize("m", [1, 4, 50])
def test_a_captured_step(hipdev, m):
    """Replays against the eager step, with other work of the same plan between them and new activations each time."""
    layer = Layer(E.Q4_K, E.Q6_K, 16, 4, 512, 256)
    plan, other = E.MoePlan(16, 4, 64, 512, 256), E.MoePlan(16, 4, 64, 512, 256)
    g = torch.Generator(device="cuda:0").manual_seed(m)
    h = torch.randn((m, 512), device="cuda:0", generator=g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(plan, h)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for p in (plan, other):
        graph, kept = torch.cuda.CUDAGraph(), {}
        with torch.cuda.graph(graph):
            layer.step(p, h, kept)
        graphs.append((graph, kept))
    fresh = E.MoePlan(16, 4, 64, 512, 256)
    for i in range(4):
        h.copy_(torch.randn((m, 512), device="cuda:0", generator=g))
        want = {}
        layer.step(fresh, h, want)
        layer.step(plan, torch.randn((37, 512), device="cuda:0", generator=g))  # eager work of the same plan
        for graph, kept in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a in ("ids", "w", "act", "out"):
                assert torch.equal(kept[a], want[a]), (i, a)


def test_streams_and_repeats(hipdev):
    """The same call gives the same words, on any stream."""
    layer = Layer(E.Q8_0, E.Q4_K, 16, 4, 512, 256)
    for m in (1, 3, 20, 200):
        h = torch.randn((m, 512), device="cuda:0")
        plan = E.MoePlan(16, 4, m, 512, 256)
        want = layer.step(plan, h).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [layer.step(plan, h) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, want) for a in again)


def test_more_tokens_of_one_plan(hipdev):
    """A plan's routings of many sizes, one after the other, leave nothing behind."""
    layer = Layer(E.Q4_K, E.Q6_K, 16, 4, 512, 256)
    plan = E.MoePlan(16, 4, 130, 512, 256)
    for m in (130, 1, 64, 2, 5, 129, 16, 3):
        h = torch.randn((m, 512), device="cuda:0")
        assert torch.equal(layer.step(plan, h), layer.step(E.MoePlan(16, 4, m, 512, 256), h))


def test_refusals(hipdev):
    L = hipdev
    plan = E.MoePlan(8, 2, 4, 512, 256)
    s = torch.randn((4, 8), device="cuda:0")
    for kw, what in ((dict(n_groups=3), "groups"), (dict(n_groups=0), "groups"), (dict(top_groups=2), "groups"),
                     (dict(n_groups=4, top_groups=0), "groups"), (dict(group_best=3), "best 3"), (dict(group_best=0), "best 0"),
                     (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")):
        with pytest.raises(E.HipError, match=what):
            E.moe_route(plan, s, **kw)
    with pytest.raises(E.HipError, match="5 tokens"):
        E.moe_route(plan, torch.randn((5, 8), device="cuda:0"))
    E.moe_route(plan, s)
    p = torch.zeros(1 << 16, device="cuda:0").data_ptr()
    st = torch.cuda.current_stream().cuda_stream

    def no(got, code, word):
        assert not got
        c, msg = L.last_error()
        L.clear_error()
        assert c == code and word in msg, (c, msg)

    for t in (E.F16, E.F32, 3, 15, 99):
        no(L.moe_gate_up_dev(p, p, plan._h, p, p, t, None, None, 0, st), -3, "not supported")
        no(L.moe_down_dev(p, p, plan._h, p, t, None, None, st), -3, "not supported")
    odd = E.MoePlan(8, 2, 4, 520, 264)
    E.moe_route(odd, s)
    for t in (E.Q4_K, E.Q8_0):
        no(L.moe_gate_up_dev(p, p, odd._h, p, p, t, None, None, 0, st), -2, "whole blocks")
        no(L.moe_down_dev(p, p, odd._h, p, t, None, None, st), -2, "whole blocks")
    for at in range(4):
        a = [p] * 4
        a[at] = None
        no(L.moe_gate_up_dev(a[0], a[1], plan._h, a[2], a[3], E.Q4_K, None, None, 0, st), -2, "null")
        a[at] = p + 4
        no(L.moe_gate_up_dev(a[0], a[1], plan._h, a[2], a[3], E.Q4_K, None, None, 0, st), -2, "aligned")
    for at in range(3):
        a = [p] * 3
        a[at] = None
        no(L.moe_down_dev(a[0], a[1], plan._h, a[2], E.Q4_K, None, None, st), -2, "null")
        a[at] = p + 8
        no(L.moe_down_dev(a[0], a[1], plan._h, a[2], E.Q4_K, None, None, st), -2, "aligned")
    no(L.moe_assign_dev(plan._h, None, p, 1, st), -2, "null")
    no(L.moe_assign_dev(plan._h, p, p, 5, st), -2, "5 tokens")
    no(L.moe_route_dev(plan._h, p, p, None, 1, 0, None, 1, 1, 1, 1, 1.0, st), -2, "null")
    no(L.moe_route_dev(plan._h, p, p, p, 1, 2, None, 1, 1, 1, 1, 1.0, st), -2, "score 2")
    no(L.moe_route_dev(plan._h, p, p, p, -1, 0, None, 1, 1, 1, 1, 1.0, st), -2, "-1 tokens")
    assert plan.tokens() == 4  # (a refused call leaves the routing as it was)


def test_the_python_front_refuses(hipdev):
    plan = E.MoePlan(8, 2, 4, 512, 256)
    s = torch.randn((4, 8), device="cuda:0")
    E.moe_route(plan, s)
    w = torch.zeros(8 * 256 * 288, dtype=torch.uint8, device="cuda:0")
    x = torch.zeros((4, 512), device="cuda:0")
    for call in (lambda: E.moe_route(plan, s.double()), lambda: E.moe_route(plan, s.t()), lambda: E.moe_route(plan, s[:, :7]),
                 lambda: E.moe_route(plan, s, score="tanh"), lambda: E.moe_route(plan, s, bias=s[0, :7]),
                 lambda: E.moe_route(plan, s, ids=torch.zeros((4, 2), device="cuda:0")),
                 lambda: E.moe_route(plan, s, weights=torch.zeros((4, 3), device="cuda:0")),
                 lambda: plan.assign(torch.zeros((4, 2), dtype=torch.int64, device="cuda:0"), s[:, :2].contiguous()),
                 lambda: plan.assign(torch.zeros((4, 2), dtype=torch.int32, device="cuda:0"), s[:, :2]),
                 lambda: E.moe_gate_up(plan, w, w[:-1], E.Q4_K, x), lambda: E.moe_gate_up(plan, w, w, E.Q4_K, x[:3]),
                 lambda: E.moe_gate_up(plan, w, w, E.Q4_K, x, activation="relu"),
                 lambda: E.moe_gate_up(plan, w, w, E.Q4_K, x, b_up=torch.zeros(2047, device="cuda:0")),
                 lambda: E.moe_gate_up(plan, w, w, E.Q4_K, x, act=torch.zeros(2047, device="cuda:0")),
                 lambda: E.moe_down(plan, w, E.Q4_K, x[:3]), lambda: E.moe_down(plan, w, E.Q4_K, x.cpu()),
                 lambda: E.moe_down(plan, w.cpu(), E.Q4_K, torch.zeros((4, 2, 256), device="cuda:0"))):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ routings that are captured and replayed


def capture(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


def products_of(plan, layer, m):
    """The plan's products as a caller makes them, into memory with something of its own before and behind it."""
    k, n, f = layer.k, layer.n_embd, layer.n_ff
    act, out = torch.full((m + 2, k, f), 7.5, device="cuda:0"), torch.full((m + 2, n), 7.5, device="cuda:0")
    x, a, h = torch.ones((m, n), device="cuda:0"), torch.ones((m, k, f), device="cuda:0"), torch.ones((m, n), device="cuda:0")
    E.moe_gate_up(plan, layer.dev["gate"], layer.dev["up"], layer.q, x, act=act[1:])
    E.moe_down(plan, layer.dev["down"], layer.dq, a, residual=h, out=out[1:])
    for t in (act, out):
        assert bool((t[0] == 7.5).all()) and bool((t[m + 1:] == 7.5).all()), "memory beside the tokens was written"
    return act[1:m + 1], out[1:m + 1]


# (tokens of the routing that ran, tokens of the products): single tokens, sorted pairs, and between the two
@pytest.mark.parametrize("ran,m", [(50, 20), (20, 50), (3, 50), (50, 2), (1, 2), (2, 1), (60, 40), (0, 20), (0, 1)])
def test_a_replayed_routing_of_other_tokens(hipdev, ran, m):
    """A product whose tokens are not those of the routing that ran last gives NaN and touches nothing else; with a routing
    of its own it is right again."""
    layer = Layer(E.Q4_K, E.Q6_K, 16, 4, 512, 256)
    plan = E.MoePlan(16, 4, 64, 512, 256)
    s, t = torch.randn((ran, 16), device="cuda:0"), torch.randn((m, 16), device="cuda:0")
    E.moe_route(plan, t)
    want = [v.clone() for v in products_of(plan, layer, m)]
    assert all(bool(torch.isfinite(v).all()) for v in want)
    graph = capture(lambda: E.moe_route(plan, s))
    assert plan.tokens() == ran
    E.moe_route(plan, t)
    graph.replay()
    for _ in range(2):
        assert all(bool(torch.isnan(v).all()) for v in products_of(plan, layer, m))
        E.moe_route(plan, t)
        assert all(torch.equal(a, b) for a, b in zip(products_of(plan, layer, m), want))
        graph.replay()


@pytest.mark.parametrize("m", [1, 30])
def test_a_captured_routing_that_never_ran(hipdev, m):
    layer = Layer(E.Q4_K, E.Q6_K, 16, 4, 512, 256)
    plan = E.MoePlan(16, 4, 64, 512, 256)
    s = torch.randn((m, 16), device="cuda:0")
    graph = capture(lambda: E.moe_route(plan, s))
    assert all(bool(torch.isnan(v).all()) for v in products_of(plan, layer, m))
    graph.replay()
    got = [v.clone() for v in products_of(plan, layer, m)]
    E.moe_route(plan, s)
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(got, products_of(plan, layer, m)))


def test_captured_products_after_a_routing_of_other_tokens(hipdev):
    layer = Layer(E.Q8_0, E.Q8_0, 16, 4, 512, 256)
    plan = E.MoePlan(16, 4, 64, 512, 256)
    for m in (2, 30):
        s, kept = torch.randn((m, 16), device="cuda:0"), []
        E.moe_route(plan, s)
        want = [v.clone() for v in products_of(plan, layer, m)]
        x, a = torch.ones((m, 512), device="cuda:0"), torch.ones((m, 4, 256), device="cuda:0")
        graph = capture(lambda: kept.extend([E.moe_gate_up(plan, layer.dev["gate"], layer.dev["up"], layer.q, x),
                                             E.moe_down(plan, layer.dev["down"], layer.dq, a, residual=x)]))
        for other in (31, 1, 0):
            E.moe_route(plan, torch.randn((other, 16), device="cuda:0"))
            graph.replay()
            assert all(bool(torch.isnan(v).all()) for v in kept)
            E.moe_route(plan, s)
            graph.replay()
            assert all(torch.equal(v, w) for v, w in zip(kept, want))


# ------------------------------------------------------------------ products of one routing that share the work out differently


def q4_k_of(shape, seed):
    """Q4_K rows made on the device: random codes and scales, d and dmin of a trained projection's size."""
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    w = torch.randint(0, 256, (*shape, 144), dtype=torch.uint8, device="cuda:0", generator=g)
    w[..., :4] = (torch.rand((*shape, 2), device="cuda:0", generator=g) * 1e-4 + 1e-5).half().view(torch.uint8)
    return w.view(*shape[:-1], -1)


# (experts, choices, tokens, n_embd, n_ff): a token's rows too long for its workgroup in down alone, in gate and up alone;
# matrices so large that tiles take gate and up from 8 pairs on, and down not yet; both; neither
@pytest.mark.parametrize("size", [(5, 4, 1, 256, 14336), (5, 2, 1, 131072, 256), (8, 2, 4, 8192, 4096), (4, 2, 4, 8192, 4096),
                                  (8, 2, 3, 8192, 4096), (4, 2, 3, 4096, 8192), (3, 1, 5, 4096, 14336)], ids=str)
def test_products_that_share_the_work_out_differently(hipdev, size):
    n, k, m, h, f = size
    gate, up, down = (q4_k_of((n, r, c // 256), s) for r, c, s in ((f, h, 1), (f, h, 2), (h, f, 3)))
    rng = np.random.default_rng(m)
    ids, g = random_ids(rng, m, n, k, 0.1), rng.random((m, k)).astype(np.float32)
    x, act, res = (rng.standard_normal(s).astype(np.float32) for s in ((m, h), (m, k, f), (m, h)))
    plan = E.MoePlan(n, k, m, h, f)
    for _ in range(2):
        plan.assign(dev(ids), dev(g))
        a = host(E.moe_gate_up(plan, gate, up, E.Q4_K, dev(x)))
        o = host(E.moe_down(plan, down, E.Q4_K, dev(act), residual=dev(res)))
    rows = sorted(rng.permutation(f)[:40].tolist() + [0, f - 1])
    want, tol = P.gate_up(E.Q4_K, x, host(gate[:, rows]), host(up[:, rows]), ids)
    assert np.all(np.abs(a[:, :, rows] - want) <= tol)
    rows = sorted(rng.permutation(h)[:40].tolist() + [0, h - 1])
    want, tol = P.down(E.Q4_K, act, host(down[:, rows]), ids, g, residual=res[:, rows])
    assert np.all(np.abs(o[:, rows] - want) <= tol)


def test_more_rows_than_one_launch_has_threads(hipdev):
    """Down of 2^22 tokens to rows of 1025: a row's part each makes more than 2^32."""
    m, n, f, period = 1 << 22, 1025, 32, 64
    rng = np.random.default_rng(1)
    w = experts(E.Q8_0, 2, n, f, rng)
    a = rng.standard_normal((period, 1, f)).astype(np.float32)
    ids, g = (np.arange(period) % 3 - 1).astype(np.int32)[:, None], rng.random((period, 1)).astype(np.float32)
    plan = E.MoePlan(2, 1, m, n, f)
    plan.assign(dev(ids).repeat(m // period, 1), dev(g).repeat(m // period, 1))
    out = E.moe_down(plan, dev(w), E.Q8_0, dev(a).repeat(m // period, 1, 1)).view(-1, period, n)
    want, tol = P.down(E.Q8_0, a, w, ids, g)
    assert np.all(np.abs(host(out[0]) - want) <= tol)
    for i in range(0, m // period, 4096):
        assert bool((out[i:i + 4096] == out[0]).all()), i
    del plan, out
    torch.cuda.empty_cache()
