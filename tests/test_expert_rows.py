"""The kernels' loads of expert weights stay inside the tensor, whatever its size."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.mark.skipif(not os.path.exists(CLANG), reason="needs the ROCm compiler")
def test_loads_stay_inside_the_tensor(tmp_path):
    exe = str(tmp_path / "expert_rows")
    # host code only
    subprocess.run([CLANG, "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-std=c++17", "-O1", "-g",
                    "-Wno-everything", "-Xarch_host", "-fsanitize=address", "-I",
                    os.path.join(HERE, "..", "edgexpu-llm_amd", "csrc"), "-I", os.path.join(HERE, "..", "include"), "-I",
                    "/opt/rocm/include", os.path.join(HERE, "expert_rows_host.cpp"), "-o", exe, "-L/opt/rocm/lib",
                    "-Wl,-rpath,/opt/rocm/lib"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and "all in bounds" in r.stdout, r.stdout[-300:] + r.stderr[:2000]
