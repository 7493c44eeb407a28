"""The Python front of the rotation and the paged cache: what it hands to the library, and what it refuses before.  The
tensors say they are on a device, the library is one that notes its calls; nothing is computed."""
import pytest
import torch

import edgexpu_amd as E


class OnDevice(torch.Tensor):
    is_cuda = True


def on(t):
    return t.as_subclass(OnDevice)


class Notes:
    """Stands in for the library; every entry point succeeds."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            if name != "check":
                self.calls.append((name, args))
            return 1

        return call


@pytest.fixture
def lib(monkeypatch):
    L = Notes()
    monkeypatch.setattr(E, "hip", lambda: L)
    monkeypatch.setattr(E, "_HIP", L)
    monkeypatch.setattr(E, "_stream", lambda: None)
    return L


def test_positions_are_dense(lib):
    """The kernel reads pos[t] side by side: a column of a table or an expanded number is not that."""
    q, k = on(torch.zeros(6, 256)), on(torch.zeros(6, 128))
    pos = on(torch.arange(6, dtype=torch.int32))
    E.qk_norm_rope(q, k, 4, 2, pos)
    E.qk_norm_rope(q, k, 4, 2, pos.view(2, 3))
    E.qk_norm_rope(q, k, 4, 2, on(torch.arange(12, dtype=torch.int32))[6:])
    E.qk_norm_rope(q[:1], k[:1], 4, 2, on(torch.arange(12, dtype=torch.int32))[::2][:1])
    n = len(lib.calls)
    assert n == 4
    for bad in (on(torch.arange(12, dtype=torch.int32))[::2], on(torch.zeros(6, 2, dtype=torch.int32))[:, 1],
                on(torch.zeros(1, dtype=torch.int32)).expand(6), on(torch.zeros(3, 2, dtype=torch.int32)).t()):
        with pytest.raises(ValueError):
            E.qk_norm_rope(q, k, 4, 2, bad)
    assert len(lib.calls) == n


def test_rotation_of_no_tokens(lib):
    """As kv_append and attention do; the library's entry points that take a token count have no call for none."""
    q, k = on(torch.zeros(0, 256)), on(torch.zeros(0, 128))
    qo, ko = E.qk_norm_rope(q, k, 4, 2, on(torch.zeros(0, dtype=torch.int32)))
    assert qo.shape == (0, 256) and ko.shape == (0, 128) and not lib.calls
    wide = on(torch.zeros(3, 1024))[:0]
    qo, ko = E.qk_norm_rope(wide[:, :256], wide[:, 256:384], 4, 2, None, q_out=on(torch.zeros(0, 256)))
    assert qo.shape == (0, 256) and ko.shape == (0, 128) and not lib.calls


class Ends(Notes):
    """A cache with a live batch does not end."""

    batches = 0
    made = 0

    def kv_pool_bytes(self, *args):
        return 1024

    def kv_create(self, *args):
        self.made += 1
        return self.made

    def batch_create(self, *args):
        self.batches += 1
        self.made += 1
        return self.made

    def batch_destroy(self, h):
        self.batches -= 1
        self.calls.append(("batch_destroy", h))

    def kv_destroy(self, h):
        if self.batches:
            return 0
        self.calls.append(("kv_destroy", h))
        return 1

    def rope_create(self, *args):
        self.made += 1
        return self.made

    def rope_destroy(self, h):
        self.calls.append(("rope_destroy", h))


def test_handles_end_outside_a_capture(monkeypatch):
    """An object that goes while the stream is captured keeps its handle until an object is made or goes after it; a
    cache that goes before its batch (in a cycle) ends after it."""
    L = Ends()
    monkeypatch.setattr(E, "hip", lambda: L)
    monkeypatch.setattr(E, "_HIP", L)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    pool = on(torch.zeros(1024, dtype=torch.uint8))

    def ended():
        return [c for c in L.calls if c[0].endswith("destroy")]

    def cache():
        return E.KvCache(E.F16, 1, 1, 64, 16, 4, 1, pool=pool)

    c = cache()
    b, r = E.KvBatch(c, 1, 1, 1), E.Rope(64)
    capturing = True
    del b, c, r
    assert not ended()
    capturing = False
    c = cache()
    assert ended() == [("batch_destroy", 2), ("kv_destroy", 1), ("rope_destroy", 3)]
    del L.calls[:]
    b = E.KvBatch(c, 1, 1, 1)
    c.__del__()
    c._h = None
    assert not ended()
    del b
    assert ended() == [("batch_destroy", 5)]
    E._end()
    assert ended() == [("batch_destroy", 5), ("kv_destroy", 4)] and not E._ENDED
