"""What works on parts of the paged cache, without a GPU: refusals of the C ABI with pointers that are never read, CPU
tensors, struct layouts, workspace sizes, and the places of lists and shares (tests/native/paged_lists_check.cpp)."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import longvideosparseattention_amd as lv
from longvideosparseattention_amd import _capi

ROOT = Path(__file__).resolve().parent.parent
S2, S3 = _capi._Str2, _capi._Str3


def _cache_and_batch(a):
    c, b = a.cache, a.batch
    c.k = c.v = c.k_scale = c.v_scale = 4096
    c.k_str = c.v_str = S3(4096, 128, 2048)
    c.n_pages, c.page_size, c.Hkv, c.D, c.bits, c.dtype = 10, 16, 2, 128, 16, _capi.LVSA_BF16
    b.cu_seqlens = b.kv_lens = b.page_table = 4096
    b.table_stride, b.B, b.max_pages, b.N = 8, 2, 8, 2


def _args(fn, **kw):
    """Arguments that pass every check (fake, aligned pointers: nothing is launched by these tests)."""
    cls = {"lvsa_paged_block_means": _capi.PagedMeansArgs, "lvsa_paged_select": _capi.PagedSelectArgs,
           "lvsa_paged_block_attn_fwd": _capi.PagedBlockAttnArgs, "lvsa_paged_weights": _capi.PagedWeightsArgs,
           "lvsa_paged_evict": _capi.PagedEvictArgs}[fn]
    a = cls()
    inner = a.attn if fn == "lvsa_paged_block_attn_fwd" else a
    _cache_and_batch(inner)
    if fn in ("lvsa_paged_select", "lvsa_paged_block_attn_fwd", "lvsa_paged_weights"):
        inner.q, inner.H, inner.q_str = 4096, 4, S2(512, 128)
    if fn == "lvsa_paged_block_means":
        a.means, a.m_str, a.block = 4096, S3(256, 128, 128), 16
    if fn == "lvsa_paged_select":
        a.means, a.m_str, a.blocks = 4096, S3(256, 128, 128), 4096
        a.block, a.top, a.tile, a.first, a.last, a.causal = 16, 4, 1, 1, 1, 1
    if fn == "lvsa_paged_block_attn_fwd":
        inner.o, inner.o_str, inner.scale = 1 << 20, S2(512, 128), 1.0
        a.blocks, a.block, a.top, a.tile = 4096, 16, 4, 1
    if fn == "lvsa_paged_weights":
        a.lse, a.weights, a.w_str, a.scale = 4096, 4096, S3(32, 1, 16), 1.0
    if fn == "lvsa_paged_evict":
        a.weights, a.w_str, a.kept, a.new_lens, a.keep = 4096, S3(32, 1, 16), 4096, 4096, 8
    for name, value in kw.items():
        at, _, field = name.rpartition("__")
        setattr(getattr(inner, at) if at else inner if hasattr(inner, field) else a, field, value)
    return a


FNS = ["lvsa_paged_block_means", "lvsa_paged_select", "lvsa_paged_block_attn_fwd", "lvsa_paged_weights", "lvsa_paged_evict"]
EVERY = [({"cache__D": 80}, -2, "head_dim 80"), ({"cache__bits": 8}, -2, "16 or 4 bits"), ({"cache__n_pages": 0}, -1, "0 pages"),
         ({"cache__k": None}, -1, "null cache"), ({"cache__k_str": S3(4096, 4, 2048)}, -1, "16 bytes"), ({"batch__B": -1}, -1, "batch"),
         ({"batch__kv_lens": None}, -1, "null batch"), ({"batch__max_pages": 2 ** 27, "batch__table_stride": 2 ** 27}, -2, "2^31")]
LONG = {"batch__max_pages": 64, "batch__table_stride": 64, "top": 64}       # a table of 8 steps
SOME = [
    ("lvsa_paged_block_means", {"means": None}, -1, "means"), ("lvsa_paged_block_means", {"means": 4100}, -1, "means"),
    ("lvsa_paged_block_means", {"m_str": S3(256, 3, 128)}, -1, "means"), ("lvsa_paged_block_means", {"block": 5}, -1, "blocks of 5"),
    ("lvsa_paged_block_means", {"block": 0}, -1, "blocks of 0"),
    ("lvsa_paged_block_means", {"cache__n_pages": 2 ** 28, "block": 1}, -2, "pages of 16 blocks"),
    ("lvsa_paged_select", {"batch__cu_seqlens": None}, -1, "null batch"), ("lvsa_paged_select", {"H": 3}, -1, "3 heads"),
    ("lvsa_paged_select", {"q": 4104}, -1, "16 bytes"), ("lvsa_paged_select", {"q": None}, -1, "null q"),
    ("lvsa_paged_select", {"top": 0}, -1, "lists of 0"), ("lvsa_paged_select", {"top": 1025}, -1, "lists of 1025"),
    ("lvsa_paged_select", {"tile": 0}, -1, "tiles of 0"), ("lvsa_paged_select", {"blocks": None}, -1, "null blocks"),
    ("lvsa_paged_select", {"first": 4}, -1, "do not fit"), ("lvsa_paged_select", {"last": 5}, -1, "do not fit"),
    ("lvsa_paged_select", {"first": -1}, -1, "do not fit"), ("lvsa_paged_select", {"tile": 50, "first": 0}, -1, "do not fit"),
    ("lvsa_paged_select", {"block": 3}, -1, "blocks of 3"), ("lvsa_paged_select", {"means": None}, -1, "means"),
    ("lvsa_paged_block_attn_fwd", {"H": 5}, -1, "5 heads"), ("lvsa_paged_block_attn_fwd", {"scale": 0.0}, -1, "scale"),
    ("lvsa_paged_block_attn_fwd", {"scale": float("nan")}, -1, "scale"), ("lvsa_paged_block_attn_fwd", {"o": None}, -1, "null o"),
    ("lvsa_paged_block_attn_fwd", {"o": 4096}, -1, "share memory"), ("lvsa_paged_block_attn_fwd", {"blocks": None}, -1, "blocks"),
    ("lvsa_paged_block_attn_fwd", {"block": 6}, -1, "blocks of 6"), ("lvsa_paged_block_attn_fwd", {"top": 2000}, -1, "lists of 2000"),
    ("lvsa_paged_block_attn_fwd", {"tile": -1}, -1, "tiles of -1"), ("lvsa_paged_block_attn_fwd", {"batch__B": 0}, -1, "no sequence"),
    ("lvsa_paged_block_attn_fwd", {"batch__N": 2 ** 30}, -2, "rows of"), ("lvsa_paged_block_attn_fwd", LONG, -1, "workspace needed"),
    ("lvsa_paged_block_attn_fwd", {"workspace": 4096, "workspace_bytes": 64, **LONG}, -3, "workspace of 64"),
    ("lvsa_paged_weights", {"weights": None}, -1, "weights"), ("lvsa_paged_weights", {"weights": 4098}, -1, "weights"),
    ("lvsa_paged_weights", {"lse": None}, -1, "lse"), ("lvsa_paged_weights", {"scale": -1.0}, -1, "scale"),
    ("lvsa_paged_weights", {"H": 0}, -1, "0 heads"), ("lvsa_paged_weights", {"q": None}, -1, "null q"),
    ("lvsa_paged_weights", {"batch__N": 640, "max_q_len": 320}, -1, "workspace needed"),
    ("lvsa_paged_evict", {"keep": 0}, -1, "0 tokens"), ("lvsa_paged_evict", {"first": 5, "last": 4}, -1, "first 5"),
    ("lvsa_paged_evict", {"first": -1}, -1, "first -1"), ("lvsa_paged_evict", {"weights": None}, -1, "weights"),
    ("lvsa_paged_evict", {"new_table": 4096, "new_pages": 4, "new_stride": 3}, -1, "rows 3 apart"),
    ("lvsa_paged_evict", {"new_table": 4096, "new_pages": 0, "new_stride": 3}, -1, "do not hold"),
    ("lvsa_paged_evict", {"kept": None}, -1, "null kept"), ("lvsa_paged_evict", {"new_lens": None}, -1, "null kept"),
    ("lvsa_paged_evict", {"keep": 2 ** 31 - 1}, -2, "2^31 - 4096"),
]


def _refused(fn, kw, code, text):
    lib = _capi.lib()
    assert getattr(lib, fn)(C.byref(_args(fn, **kw)), None) == code, lib.lvsa_last_error()
    assert text.encode() in lib.lvsa_last_error(), lib.lvsa_last_error()


@pytest.mark.parametrize("fn", FNS)
@pytest.mark.parametrize("i", range(len(EVERY)))
def test_cache_and_batch_are_checked(fn, i):
    _refused(fn, *EVERY[i])


@pytest.mark.parametrize("i", range(len(SOME)))
def test_arguments_are_checked(i):
    _refused(*SOME[i])


@pytest.mark.parametrize("fn", FNS)
def test_null_arguments_and_nothing_to_do(fn):
    lib = _capi.lib()
    assert getattr(lib, fn)(None, None) == -1
    if fn not in ("lvsa_paged_block_attn_fwd", "lvsa_paged_select"):
        assert getattr(lib, fn)(C.byref(_args(fn, batch__B=0)), None) == 0
    if fn != "lvsa_paged_evict":
        assert getattr(lib, fn)(C.byref(_args(fn, batch__N=0)), None) == 0


def test_workspace_sizes():
    lib, n = _capi.lib(), C.c_int64(-1)
    # 2 lists of 2 key heads over 64 keys: one step each, a share each, nothing to join
    assert lib.lvsa_paged_block_attn_workspace_query(C.byref(_args(FNS[2], batch__N=2)), C.byref(n)) == 0 and n.value == 0
    # over 8 pages of 16 blocks: 128 keys, still one step; a table of 64 pages: 8 steps, every one a share of its own
    a = _args(FNS[2], batch__max_pages=64, batch__table_stride=64, top=64)
    assert lib.lvsa_paged_block_attn_workspace_query(C.byref(a), C.byref(n)) == 0
    assert n.value == 4 * 2 * (2 * 2 * 8) * 16 * (128 + 2)
    assert lib.lvsa_paged_block_attn_workspace_query(C.byref(a), None) == -1
    assert lib.lvsa_paged_weights_workspace_query(C.byref(_args(FNS[3])), C.byref(n)) == 0 and n.value == 0
    a = _args(FNS[3], batch__N=640, max_q_len=320)
    assert lib.lvsa_paged_weights_workspace_query(C.byref(a), C.byref(n)) == 0 and n.value > 0 and n.value % 512 == 0
    assert lib.lvsa_paged_weights_workspace_query(C.byref(_args(FNS[3], H=3)), C.byref(n)) == -1


def test_cpu_tensors_are_refused():
    t = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    for call in (lambda c: lv.paged_kv_select(t, c, t, t, t, t, 4), lambda c: lv.paged_block_attention(t, c, t, 16, t, t, t),
                 lambda c: lv.paged_kv_weights(t, t, c, t, t, t, t)):
        cache = lv.PagedKVCache.__new__(lv.PagedKVCache)
        cache._packed, cache.bits, cache.dtype, cache.head_dim, cache.num_kv_heads = {torch.bfloat16: b""}, 16, torch.bfloat16, 128, 2
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(cache)


def test_structs_match_c(tmp_path):
    structs = {"lvsa_paged_means_args": _capi.PagedMeansArgs, "lvsa_paged_select_args": _capi.PagedSelectArgs,
               "lvsa_paged_block_attn_args": _capi.PagedBlockAttnArgs, "lvsa_paged_weights_args": _capi.PagedWeightsArgs,
               "lvsa_paged_evict_args": _capi.PagedEvictArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "lvsa_amd.h"', "int main(void) {"]
    for c, py in structs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    lines.append('printf("bit bad_block %d\\n", LVSA_PAGED_BAD_BLOCK);')
    lines.append("return 0; }")
    (tmp_path / "l.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", f"-I{ROOT / 'include'}", "-I/opt/rocm/include", str(tmp_path / "l.c"),
                    "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split("\n")
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out if x}
    assert got[("bit", "bad_block")] == _capi.PAGED_BAD_BLOCK
    for c, py in structs.items():
        assert got[(c, "size")] == C.sizeof(py), c
        for f, _ in py._fields_:
            assert got[(c, f)] == getattr(py, f).offset, (c, f)


def _hipcc():
    return shutil.which("hipcc") or ("/opt/rocm/bin/hipcc" if Path("/opt/rocm/bin/hipcc").exists() else None)


@pytest.mark.skipif(_hipcc() is None, reason="hipcc not available")
def test_lists_have_places_of_their_own_and_shares_cover_the_work(tmp_path):
    exe = tmp_path / "check"
    build = subprocess.run([_hipcc(), "-O1", "-std=c++17", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang",
                            "-packed-fp32-ops", f"-I{ROOT / 'include'}", f"-I{ROOT / 'longvideosparseattention_amd' / 'csrc'}",
                            "-x", "hip", str(ROOT / "tests" / "native" / "paged_lists_check.cpp"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "paged lists ok" in run.stdout, run.stdout + run.stderr
