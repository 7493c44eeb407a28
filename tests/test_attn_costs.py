"""The plan's measured costs and the kernel's forms: no form is compiled that no plan asks for, none asked for that is not
there.  The forms of csrc/attn.hip: at most 16 rows, 32 (f16: as 64), 64 (Q8_0: at 128 only), 128 (not at 256)."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("attn_costs") / "attn_costs.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-shared", "-fPIC", "-I",
                    os.path.join(HERE, "..", "edgexpu-llm_amd", "csrc"), os.path.join(HERE, "attn_costs.cpp"), "-o", so], check=True)
    return C.CDLL(so)


def forms(qtype, dim):
    """Indices of the costs that a form stands behind, and which one a number of rows goes to."""
    q8, f16 = qtype == 8, qtype == 1
    few = {0} | ({1} if dim != 256 and not f16 else set())
    many = ({2} if not q8 or dim == 128 else set()) | ({3} if dim != 256 else set())

    def of(rows):
        for k in sorted(few | many):
            if rows <= 16 << k:
                return k
        return None

    return few | many, of


@pytest.mark.parametrize("qtype", [0, 1, 8])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_every_form_is_reached_and_every_item_has_one(lib, qtype, dim):
    cost = (C.c_int * 4)()
    lib.costs(qtype, dim, cost)
    there, of = forms(qtype, dim)
    used = set()
    for tokens in range(1, 300):
        rows = (C.c_int * 4096)()
        n = lib.item_rows(qtype, dim, 1, 700, tokens, rows, 4096)
        assert 0 < n <= 4096
        for r in rows[:n]:
            k = of(r)
            assert k is not None and cost[0 if r <= 16 else 1 if r <= 32 else 2 if r <= 64 else 3] > 0, r
            used.add(k)
    assert used == there
