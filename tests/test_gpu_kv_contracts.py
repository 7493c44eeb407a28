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
