"""Arguments that the paged cache's and the rotation's entry points refuse before they touch a device."""
import ctypes as C

import pytest

import edgexpu_amd as E


@pytest.fixture
def lib():
    L = E.HipLib()
    L.clear_error()
    yield L
    L.clear_error()


def refused(L, got, code, word):
    assert not got or got == -1
    c, msg = L.last_error()
    L.clear_error()
    assert c == code and word in msg, (c, msg)


def test_pool_bytes(lib):
    n = lib.kv_pool_bytes
    assert n(E.F16, 2, 8, 128, 64, 10) == 2 * 10 * 2 * 8 * 64 * 128 * 2
    assert n(E.F32, 1, 1, 96, 16, 1) == 2 * 16 * 96 * 4
    assert n(E.Q8_0, 3, 2, 64, 32, 5) == 3 * 5 * 2 * 2 * 32 * (64 + 4)
    assert n(E.F16, 1, 1, 64, 16, (2**31 - 1) // 16) == 2 * ((2**31 - 1) // 16) * 16 * 64 * 2
    for bad in [(E.Q4_K, 1, 1, 64, 16, 1), (30, 1, 1, 64, 16, 1), (E.F16, 0, 1, 64, 16, 1), (E.F16, 1, 0, 64, 16, 1),
                (E.F16, 1, 1, 80, 16, 1), (E.F16, 1, 1, 512, 16, 1), (E.F16, 1, 1, 64, 8, 1), (E.F16, 1, 1, 64, 48, 1),
                (E.F16, 1, 1, 64, 512, 1), (E.F16, 1, 1, 64, 16, 0), (E.F16, 1, 1, 64, 16, 2**27), (E.F16, -1, 1, 64, 16, 1),
                (E.F32, 4096, 4096, 256, 256, 2**31 // 256 - 1)]:
        assert n(*bad) == 0
    assert lib.last_error()[0] == 0


def test_create(lib):
    refused(lib, lib.kv_create(None, E.F16, 1, 1, 72, 16, 4, 1), -2, "supported")
    refused(lib, lib.kv_create(None, E.F16, 1, 1, 64, 16, 4, 0), -2, "0 sequences")
    refused(lib, lib.kv_create(0x1008, E.F16, 1, 1, 64, 16, 4, 1), -2, "aligned")
    refused(lib, lib.batch_create(None, 4, 1, 1), -2, "null cache")
    for n_rot, base, scale in ((0, 1e4, 1.0), (7, 1e4, 1.0), (258, 1e4, 1.0), (64, 0.0, 1.0), (64, float("nan"), 1.0),
                               (64, float("inf"), 1.0), (64, 1e4, float("nan"))):
        refused(lib, lib.rope_create(n_rot, base, scale, None, 0), -2, "rope_create")


def test_null_handles(lib):
    one = (C.c_int * 1)(0)
    refused(lib, lib.kv_new(None), -2, "null")
    refused(lib, lib.kv_fork(None, 1, one, 0, one, None), -2, "null")
    refused(lib, lib.kv_extend(None, 1, one, one, None), -2, "null")
    refused(lib, lib.kv_truncate(None, 0, 0), -2, "null")
    refused(lib, lib.kv_release(None, 1, one), -2, "null")
    refused(lib, lib.kv_compact(None, None, None), -2, "null")
    refused(lib, lib.kv_tables(None, 1, one, None, 0), -2, "null")
    refused(lib, lib.batch_set(None, 1, one, one, None), -2, "null")
    assert lib.kv_length(None, 0) == -1 and lib.kv_free_pages(None) == 0 and lib.kv_pool(None) is None
    assert lib.batch_tokens(None) == 0 and lib.kv_destroy(None) == 1
    lib.batch_destroy(None)
    lib.rope_destroy(None)
    assert lib.last_error()[0] == 0


def test_rotation(lib):
    f = lib.qk_norm_rope_dev
    p = 0x1000  # (refused before anything reads it)
    for args in [(None, p, p, 256, p, 128, 1, 4, 2, 64), (p, None, p, 256, p, 128, 1, 4, 2, 64), (p, p, None, 256, p, 128, 1, 4, 2, 64),
                 (p, p, p, 255, p, 128, 1, 4, 2, 64), (p, p, p, 256, p, 127, 1, 4, 2, 64), (p, p, p, 256, p, 128, 0, 4, 2, 64),
                 (p, p, p, 256, p, 128, 1, -1, 2, 64), (p, p, p, 256, p, 128, 1, 0, 0, 64), (p, p, p, 256, p, 128, 1, 4, 2, 63),
                 (p, p, p, 256, p, 128, 1, 4, 2, 0), (p, p, p, 2000, p, 1000, 1, 4, 2, 258)]:
        refused(lib, f(*args, None, None, 1e-6, None, p, None), -2, "qk_norm_rope")
