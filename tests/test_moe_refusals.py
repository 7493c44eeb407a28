"""Arguments that the experts' entry points refuse before they touch a device."""
import numpy as np
import pytest

import edgexpu_amd as E
import moe_plain as P


@pytest.fixture
def lib():
    L = E.HipLib()
    L.clear_error()
    yield L
    L.clear_error()


def refused(L, got, code, word):
    assert not got
    c, msg = L.last_error()
    L.clear_error()
    assert c == code and word in msg, (c, msg)


@pytest.mark.parametrize("args", [
    (0, 1, 1, 256, 256), (513, 1, 1, 256, 256), (8, 0, 1, 256, 256), (8, 9, 1, 256, 256), (64, 33, 1, 256, 256),
    (8, 2, 0, 256, 256), (8, 2, 2**21 + 1, 256, 256), (8, 2, -1, 256, 256), (8, 2, 1, 0, 256), (8, 2, 1, 256, 0),
    (8, 2, 1, 2**20 + 32, 256), (8, 2, 1, 256, 2**20 + 32), (2**31 - 1, 2, 1, 256, 256), (8, 2, 2**31 - 1, 256, 256)])
def test_create(lib, args):
    refused(lib, lib.moe_create(*args), -2, "moe_create")


@pytest.mark.parametrize("args", [(8, 2, 2**21, 256, 2**14), (8, 1, 2**22, 2**14, 256), (512, 32, 2**17, 256, 8449)])
def test_create_beyond_the_counted_groups(lib, args):
    refused(lib, lib.moe_create(*args), -2, "groups of 256")


def test_null_plan(lib):
    p = 0x1000  # (refused before anything reads it)
    refused(lib, lib.moe_route_dev(None, p, p, p, 1, 0, None, 1, 1, 1, 1, 1.0, None), -2, "moe_route")
    refused(lib, lib.moe_assign_dev(None, p, p, 1, None), -2, "moe_assign")
    refused(lib, lib.moe_gate_up_dev(p, p, None, p, p, E.Q4_K, None, None, 0, None), -2, "moe_gate_up")
    refused(lib, lib.moe_gate_up_dev(p, p, None, p, p, E.Q4_K, None, None, 2, None), -2, "activation 2")
    refused(lib, lib.moe_down_dev(p, p, None, p, E.Q4_K, None, None, None), -2, "moe_down")
    assert lib.moe_tokens(None) == 0
    lib.moe_destroy(None)
    assert lib.last_error()[0] == 0


def test_the_plain_route():
    """The plain form against counts by hand."""
    s = np.array([[0.0, 1.0, 1.0, -np.inf], [np.nan, 2.0, np.inf, 2.0], [-np.inf] * 4, [5.0, 5.0, 5.0, 5.0]], np.float32)
    ids, w = P.route(s, 3, normalise=False)
    z = 1 + 2 * np.e
    assert ids.tolist() == [[1, 2, 0], [1, 3, -1], [-1, -1, -1], [0, 1, 2]]
    assert np.allclose(w, [[np.e / z, np.e / z, 1 / z], [0.5, 0.5, 0], [0, 0, 0], [0.25] * 3])
    ids, w = P.route(s[:1], 2, score="sigmoid", bias=np.array([0, 0, -5, 9], np.float32), scale=2.0)
    assert ids.tolist() == [[1, 0]] and abs(w.sum() - 2) < 1e-12
    # the second run's two best sum to more than the first run's single best
    s = np.array([[4.0, -9.0, 3.0, 2.9]], np.float32)
    assert P.route(s, 1, "sigmoid", n_groups=2, top_groups=1, best=1)[0].tolist() == [[0]]
    assert P.route(s, 1, "sigmoid", n_groups=2, top_groups=1, best=2)[0].tolist() == [[2]]


@pytest.mark.parametrize("args", [(512, 1, 2**15, 32, 2**20), (512, 8, 2**12, 32, 2**20)])
def test_create_beyond_the_workgroups_of_a_launch(lib, args):
    """2^24 workgroups of 256 threads are 2^32 threads, of which a launch would run none."""
    refused(lib, lib.moe_create(*args), -2, "workgroups")


@pytest.mark.parametrize("n,groups,top,best,k", [(9, 1, 1, 1, 4), (12, 4, 2, 1, 5), (12, 4, 2, 2, 7), (30, 6, 5, 2, 8), (8, 8, 3, 2, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_the_plain_route_by_counting(n, groups, top, best, k, score):
    """The plain form against another: an expert is chosen where fewer than k stand before it, of the runs that fewer
    than `top` stand before, and its place is how many do."""
    rng = np.random.default_rng(n + k)
    m, per = 40, n // groups
    s = rng.integers(-3, 4, (m, n)).astype(np.float32)  # (many equal scores)
    s[rng.random((m, n)) < 0.2] = -np.inf
    s[:3] = [[-np.inf], [1.0], [np.nan]]
    bias = (rng.integers(-2, 3, n) / 4).astype(np.float32)
    bias[n - 1] = np.inf
    ids, w = P.route(s, k, score, bias, groups, top, best, normalise=False)
    live = np.isfinite(s)
    x = np.where(live, s, -1e30).astype(np.float64)
    e = np.where(live, np.exp(np.minimum(x, 700)), 0)
    p = e / (1 + e) if score == "sigmoid" else e / np.maximum(e.sum(1, keepdims=True), 1e-300)
    c = np.where(live & np.isfinite(bias), p + np.where(np.isfinite(bias), bias, 0), -np.inf)
    runs = np.sort(c.reshape(m, groups, per), 2)[:, :, ::-1][:, :, :best]
    rank = np.where(np.isfinite(runs), runs, 0).sum(2) + np.where(np.isfinite(runs[:, :, 0]), 0, -np.inf)

    def before(v):  # how many stand before each, by value and then by number
        # (values that 64 bits hold apart by their last bits are equal here: the two forms round differently)
        v = np.where(np.isfinite(v), np.round(v, 12), -np.inf)
        i = np.arange(v.shape[1])
        return ((v[:, None, :] > v[:, :, None]) | ((v[:, None, :] == v[:, :, None]) & (i[None, None, :] < i[None, :, None]))).sum(2)

    stay = np.repeat(before(rank) < top, per, axis=1) if groups > 1 else np.ones((m, n), bool)
    kept = np.where(stay, c, -np.inf)
    place = np.where(np.isfinite(kept), before(kept), n)
    for t in range(m):
        want = np.full(k, -1)
        for expert in range(n):
            if place[t, expert] < k:
                want[place[t, expert]] = expert
        assert ids[t].tolist() == want.tolist(), t
        assert np.allclose(w[t], np.where(want >= 0, p[t, want], 0), rtol=1e-12, atol=0)
