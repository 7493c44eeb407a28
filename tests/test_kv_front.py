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
