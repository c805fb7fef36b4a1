"""Which sources name the build that bench.py's committed counters belong to."""
import shutil
from pathlib import Path

import bench

ROOT = Path(__file__).resolve().parent.parent


def _copy(tmp_path, monkeypatch):
    pkg = tmp_path / "longvideosparseattention_amd"
    shutil.copytree(ROOT / "longvideosparseattention_amd" / "csrc", pkg / "csrc", ignore=shutil.ignore_patterns("__pycache__"))
    shutil.copy(ROOT / "longvideosparseattention_amd" / "build_lib.py", pkg)
    shutil.copytree(ROOT / "include", tmp_path / "include")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    return pkg


def _edit(path, old, new):
    text = path.read_text()
    assert old in text
    path.write_text(text.replace(old, new, 1))


def test_the_paged_caches_sources_do_not_rename_the_build(tmp_path, monkeypatch):
    here = bench.source_hash()
    pkg = _copy(tmp_path, monkeypatch)
    assert bench.source_hash() == here
    for f in pkg.glob("csrc/lvsa_paged*"):
        f.write_text(f.read_text() + "\n// more\n")
    (pkg / "csrc" / "lvsa_paged_more.hip").write_text("// another unit\n")
    _edit(pkg / "build_lib.py", '    "lvsa_paged.hip": [],\n', '    "lvsa_paged.hip": ["-O2"],\n    "lvsa_paged_more.hip": [],\n')
    _edit(tmp_path / "include" / "lvsa_amd.h", "typedef struct lvsa_paged_cache {", "/* more */\ntypedef struct lvsa_paged_cache {")
    assert bench.source_hash() == here


def test_the_benchmarked_kernels_sources_do(tmp_path, monkeypatch):
    pkg = _copy(tmp_path, monkeypatch)
    seen = {bench.source_hash()}
    for path, old in ((pkg / "csrc" / "lvsa_attn_d128.hip", "\n"), (pkg / "csrc" / "lvsa_common.h", "\n"),
                      (pkg / "csrc" / "lvsa_attn_stream_body.inc", "\n"), (pkg / "build_lib.py", '"-O3",'),
                      (tmp_path / "include" / "lvsa_amd.h", "typedef struct lvsa_attn_args {"),
                      (tmp_path / "include" / "lvsa_amd.h", "/* Library identification")):
        _edit(path, old, old + " ")
        seen.add(bench.source_hash())
    assert len(seen) == 7
