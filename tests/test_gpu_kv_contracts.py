"""What the paged cache's and the batch's calls leave behind: refused ones, captured ones, handles that end."""
import numpy as np
import pytest
import torch

import edgexpu_amd as E

pytestmark = pytest.mark.gpu


def cache(lengths, page=16, pages=200, dim=64, kv=1, qtype=E.F16, seed=1):
    """A cache of random values and sequences of these lengths."""
    g = torch.Generator(device="cuda:0").manual_seed(seed)
    size = E.hip().kv_pool_bytes(qtype, 1, kv, dim, page, pages)
    c = E.KvCache(qtype, 1, kv, dim, page, pages, 12, pool=torch.zeros(size, dtype=torch.uint8, device="cuda:0"))
    c.pool.view(torch.float16).normal_(generator=g)
    seqs = [c.new() for _ in lengths]
    c.extend(seqs, lengths)
    return c, seqs


def rows(n, width, seed=2):
    return torch.randn((n, width), device="cuda:0", generator=torch.Generator(device="cuda:0").manual_seed(seed))


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_a_refused_call_in_a_capture_holds_nothing(hipdev):
    """Calls that record nothing leave the batch free: refused ones, and those of a plan without tokens."""
    L = hipdev
    c, (a, e) = cache([40, 3000])
    (f,) = c.fork([a])
    q, k, out = rows(4, 64), rows(4, 64, 3), torch.zeros((4, 64), device="cuda:0")
    st = lambda: torch.cuda.current_stream().cuda_stream

    def refused():
        assert not L.attention_dev(None, q.data_ptr(), b._h, 0, 1.0, st())
        assert not L.attention_dev(out.data_ptr(), q.data_ptr() + 4, b._h, 0, 1.0, st())
        assert not L.attention_dev(out.data_ptr(), q.data_ptr(), b._h, 0, float("nan"), st())
        assert not L.kv_append_dev(out.data_ptr(), None, 64, k.data_ptr(), 64, k.data_ptr(), 64, b._h, 0, None, None, 0.0, None, st())
        assert not L.kv_append_dev(out.data_ptr(), q.data_ptr(), 63, k.data_ptr(), 64, k.data_ptr(), 64, b._h, 0, None, None, 0.0, None, st())
        # (a's last page is shared)
        assert not L.kv_append_dev(out.data_ptr(), q.data_ptr(), 64, k.data_ptr(), 64, k.data_ptr(), 64, b._h, 0, None, None, 0.0, None, st())
        L.clear_error()

    def nothing():
        E.attention(b, 0, q, out=out)
        E.kv_append(b, 0, q, k, k, q_out=out)

    for first, calls in ((([a], [1]), refused), (([a], [0]), nothing)):
        b = E.KvBatch(c, 1, 4, 8)
        b.set(*first)
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            calls()
        b.set([e], [4])  # more tokens, pieces that need a workspace
        assert b.tokens() == 4 and torch.isfinite(E.attention(b, 0, q)).all()


def test_a_refused_set_leaves_the_batch_as_it_was(hipdev):
    """Whatever refuses it: arguments, a captured call's tokens, plan buffer, workspace or slots."""
    c, (a, e, g, h) = cache([40, 50, 2500, 6])
    (f,) = c.fork([e])
    q, k = rows(8, 64), rows(8, 64, 3)
    qr, out = torch.zeros((8, 64), device="cuda:0"), torch.zeros((8, 64), device="cuda:0")
    b = E.KvBatch(c, 1, 4, 8)
    b.set([a, h], [2, 1])
    want = E.attention(b, 0, q)[:3].clone()

    def same():
        assert b.tokens() == 3 and torch.equal(E.attention(b, 0, q)[:3], want)

    for ids, n_new, what in (([a], [41], "41 new"), ([a], [9], "9 tokens"), ([a], [-1], "-1 new"), ([a, a], [1, 1], "twice"), ([9], [1], "not in use"),
                             ([a, e, f, g, h], [1] * 5, "5 sequences")):
        with pytest.raises(E.HipError, match=what):
            b.set(ids, n_new)
        same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.kv_append(b, 0, q, k, k, q_out=qr)
        E.attention(b, 0, qr, out=out)
        with pytest.raises(E.HipError, match="captured"):
            b.set([a], [1])
    same()
    for ids, n_new, what in (([a], [4], "4 tokens outgrows"), ([e], [1], "appends"), ([g], [1], "outgrows the workspace")):
        with pytest.raises(E.HipError, match=what):
            b.set(ids, n_new)
        same()
        for _ in range(2):  # and the graph replays the plan that is set
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[:3], E.attention(b, 0, qr)[:3])
        want = E.attention(b, 0, q)[:3].clone()  # (the replays have written its tokens' slots)
    b.set([a], [1])
    assert b.tokens() == 1


def test_objects_that_go_during_a_capture(hipdev):
    """A batch, a rotation and a cache collected while a step is captured: the capture stands, their handles end later."""
    c, (a,) = cache([300])
    old, (x,) = cache([10])
    b, gone, rope = E.KvBatch(c, 1, 1, 1), E.KvBatch(old, 1, 1, 1), E.Rope(64)
    b.set([a], [1])
    gone.set([x], [1])
    q, out = rows(1, 64), torch.zeros((1, 64), device="cuda:0")
    want = E.attention(b, 0, q).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.attention(b, 0, q, out=out)
        del gone, rope, old
    assert len(E._ENDED) == 3
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    E.Rope(64)
    assert not E._ENDED
