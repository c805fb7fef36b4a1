"""Row tiles and work shares of the paged cache's prefill launches, checked on the host.

tests/native/paged_plan_check.cpp includes the kernels' header and runs it over
random batches: tiles stay within the launch's bound, every key block of a tile
is done once, and the joining finds the partial sums where the attention kernels
put them.  No GPU is used; the program is compiled with hipcc for its host code.
"""
import subprocess

import pytest

from test_paged_map import ROOT, _hipcc


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
def test_shares_of_the_plan_cover_the_work(tmp_path):
    exe = tmp_path / "paged_plan_check"
    build = subprocess.run(
        [_hipcc(), "-O1", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
         "-packed-fp32-ops", f"-I{ROOT / 'include'}", f"-I{ROOT / 'longvideosparseattention_amd' / 'csrc'}", "-x", "hip",
         str(ROOT / "tests" / "native" / "paged_plan_check.cpp"), "-o", str(exe)],
        capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "paged plan ok" in run.stdout, run.stdout + run.stderr
