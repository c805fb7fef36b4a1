"""The workspace of the accumulated weights against what the kernels write to it, without a GPU
(tests/native/paged_weights_check.cpp)."""
import shutil
import subprocess
from pathlib import Path

import pytest

from longvideosparseattention_amd import _capi, build_lib

ROOT = Path(__file__).resolve().parent.parent
HIPCC = shutil.which("hipcc") or ("/opt/rocm/bin/hipcc" if Path("/opt/rocm/bin/hipcc").exists() else None)


@pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
def test_sums_of_shared_rows_lie_within_the_workspace(tmp_path):
    _capi.lib()
    exe = tmp_path / "check"
    build = subprocess.run([HIPCC, "-O1", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", f"-I{ROOT / 'include'}", f"-I{ROOT / 'longvideosparseattention_amd' / 'csrc'}",
                            "-x", "hip", str(ROOT / "tests" / "native" / "paged_weights_check.cpp"), "-ldl", "-o", str(exe)],
                           capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe), str(build_lib.LIB)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "paged weights ok" in run.stdout, run.stdout + run.stderr
