"""The library's code leaves every matrix result the wait states that it needs."""
import glob
import os
import shutil
import subprocess

import pytest

import mfma_waits as W

HERE = os.path.dirname(os.path.abspath(__file__))
LIB = os.path.join(HERE, "..", "edgexpu-llm_amd", "lib", "libedgexpu_hip.so")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"

PRODUCT = "v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], 0"


@pytest.mark.parametrize("code,short", [
    ([PRODUCT, "s_nop 7", "v_add_u32_e32 v4, v0, v4", "s_endpgm"], 0),
    ([PRODUCT, "s_nop 6", "v_add_u32_e32 v4, v0, v4", "s_endpgm"], 1),
    ([PRODUCT, "s_nop 6", "v_add_u32_e32 v4, v5, v6", "v_add_u32_e32 v4, v0, v4", "s_endpgm"], 0),
    ([PRODUCT, "v_mov_b32_e32 v3, 0", "s_endpgm"], 8),  # overwritten
    ([PRODUCT, "v_mfma_i32_16x16x64_i8 v[0:3], v[8:11], v[12:15], v[0:3]", "s_endpgm"], 0),  # its addend
    ([PRODUCT, "v_mfma_i32_16x16x64_i8 v[4:7], v[0:3], v[12:15], 0", "s_endpgm"], 8),  # its operand
    (["v_mfma_f32_32x32x16_f16 a[0:15], v[8:11], v[12:15], 0", "s_nop 10", "v_accvgpr_read_b32 v0, a3", "s_endpgm"], 1),
    (["v_mfma_f32_16x16x4_f32 v[0:3], v8, v9, 0", "s_nop 9", "global_store_dwordx4 v[20:21], v[0:3], off", "s_endpgm"], 0),
    # a short block on one path, the reader where the two meet
    ([PRODUCT, "s_cbranch_scc1 L0", "s_nop 7", "L0:", "v_add_u32_e32 v4, v0, v4", "s_endpgm"], 7),
    ([PRODUCT, "s_cbranch_scc1 L0", "s_nop 7", "L0:", "s_nop 6", "v_add_u32_e32 v4, v0, v4", "s_endpgm"], 0),
    # the reader at the head of the loop whose end has the product
    (["L0:", "v_add_u32_e32 v4, v0, v4", PRODUCT, "s_nop 3", "s_cbranch_scc0 L0", "s_endpgm"], 3),
    (["s_branch L1", "L0:", "v_add_u32_e32 v4, v0, v4", "s_endpgm", "L1:", PRODUCT, "s_branch L0"], 7),
])
def test_the_search(code, short):
    found = W.early_reads(code)
    assert ([s for _, _, s in found] or [0]) == [short], found


def test_the_search_knows_its_products():
    with pytest.raises(ValueError):
        W.early_reads(["v_mfma_f64_16x16x4_f64 v[0:7], v[8:9], v[10:11], 0", "s_endpgm"])


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="needs the ROCm tools")
def test_no_result_is_read_early(tmp_path):
    shutil.copy(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    bad, kernels = [], 0
    for f in sorted(glob.glob(str(tmp_path / "lib.so.*gfx950"))):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--symbolize-operands", f], check=True,
                                 capture_output=True, text=True).stdout
        if "v_mfma" not in listing and "v_smfma" not in listing:
            continue
        for name, code in W.functions(listing):
            if any(t.startswith(("v_mfma", "v_smfma")) for t in code):
                kernels += 1
                bad += [(name, *b) for b in W.early_reads(code)]
    assert not bad, bad[:5]
    assert kernels >= 40  # (the listings were there)
