"""Lookups and work shares of the paged cache's kernels, checked on the host.

tests/native/paged_map_check.cpp includes the kernels' header and runs it over
random batches, half of them with garbage for lengths, row ranges and page
numbers: nothing outside the caller's memory is named, every work unit is done
once, and the merge finds the partial sums where the attention kernel puts
them.  No GPU is used; the program is compiled with hipcc for its host code.
"""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def _hipcc():
    for c in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and Path(c).exists():
            return c
    return None


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
def test_lookups_stay_inside_and_shares_cover_the_work(tmp_path):
    exe = tmp_path / "paged_map_check"
    build = subprocess.run(
        [_hipcc(), "-O1", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", f"-I{ROOT / 'include'}", f"-I{ROOT / 'longvideosparseattention_amd' / 'csrc'}", "-x", "hip",
         str(ROOT / "tests" / "native" / "paged_map_check.cpp"), "-o", str(exe)],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "paged map ok" in run.stdout, run.stdout + run.stderr
