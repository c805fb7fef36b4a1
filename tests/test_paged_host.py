"""Refusals of the paged cache that need no GPU: the C ABI with pointers that are never read, CPU tensors, sizes."""
import ctypes as C

import pytest
import torch

import longvideosparseattention_amd as lv
from longvideosparseattention_amd import _capi


def _args(cls=_capi.PagedAttnArgs, **kw):
    """Arguments that pass every check (fake, aligned pointers: nothing is launched by these tests)."""
    a = cls()
    c, b = a.cache, a.batch
    c.k = c.v = c.k_scale = c.v_scale = 4096
    c.k_str = c.v_str = _capi._Str3(4096, 128, 2048)
    c.n_pages, c.page_size, c.Hkv, c.D, c.bits, c.dtype = 10, 16, 2, 128, 16, _capi.LVSA_BF16
    b.cu_seqlens = b.kv_lens = b.page_table = 4096
    b.table_stride, b.B, b.max_pages, b.N = 8, 2, 8, 2
    a.q, a.H, a.q_str = 4096, 4, _capi._Str2(512, 128)
    if cls is _capi.PagedAttnArgs:
        a.o, a.o_str, a.scale = 4096, _capi._Str2(512, 128), 1.0
    else:
        a.k = a.v = a.q_out = 4096
        a.k_str = a.v_str = _capi._Str2(256, 128)
        a.qo_str = _capi._Str2(512, 128)
    for name, value in kw.items():
        at, _, field = name.rpartition("__")
        setattr(getattr(a, at) if at else a, field, value)
    return a


def _fails(fn, a, code, text, *more):
    lib = _capi.lib()
    assert getattr(lib, fn)(C.byref(a), *more) == code, lib.lvsa_last_error()
    assert text.encode() in lib.lvsa_last_error(), lib.lvsa_last_error()


BAD = [
    ({"cache__D": 80}, -2, "head_dim 80"), ({"cache__bits": 8}, -2, "16 or 4 bits"),
    ({"cache__dtype": _capi.LVSA_FP32}, -2, "bf16 or fp16"), ({"cache__n_pages": 0}, -1, "0 pages"),
    ({"cache__page_size": 0}, -1, "0 slots"), ({"cache__Hkv": 0}, -1, "0 heads"), ({"cache__k": None}, -1, "null cache"),
    ({"cache__bits": 4, "cache__v_scale": None}, -1, "null cache"), ({"cache__k": 4104}, -1, "16 bytes"),
    ({"cache__k_str": _capi._Str3(4096, 4, 2048)}, -1, "16 bytes"), ({"batch__B": -1}, -1, "batch"),
    ({"batch__table_stride": 7}, -1, "batch"), ({"batch__kv_lens": None}, -1, "null batch"),
    ({"batch__cu_seqlens": None}, -1, "null batch"), ({"batch__max_pages": 2 ** 27, "batch__table_stride": 2 ** 27}, -2, "2^31"),
]


@pytest.mark.parametrize("i", range(len(BAD)))
@pytest.mark.parametrize("fn,cls", [("lvsa_paged_attn_fwd", _capi.PagedAttnArgs), ("lvsa_paged_append", _capi.PagedAppendArgs)])
def test_cache_and_batch_are_checked(fn, cls, i):
    kw, code, text = BAD[i]
    _fails(fn, _args(cls, **kw), code, text, None)


def test_attention_arguments():
    fn = "lvsa_paged_attn_fwd"
    _fails(fn, _args(H=3), -1, "3 heads", None)
    _fails(fn, _args(H=0), -1, "0 heads", None)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _fails(fn, _args(scale=scale), -1, "scale", None)
    _fails(fn, _args(q=None), -1, "null q", None)
    _fails(fn, _args(q=4104), -1, "16 bytes", None)
    _fails(fn, _args(o_str=_capi._Str2(516, 128)), -1, "16 bytes", None)
    _fails(fn, _args(batch__N=2 ** 30), -2, "rows of", None)
    _fails(fn, _args(), -1, "workspace needed", None)
    _fails(fn, _args(workspace=4104, workspace_bytes=1 << 30), -1, "workspace needed", None)
    _fails(fn, _args(workspace=4096, workspace_bytes=64), -3, "workspace of 64", None)
    assert _capi.lib().lvsa_paged_attn_fwd(None, None) == -1


def test_append_and_gather_arguments():
    fn, A = "lvsa_paged_append", _capi.PagedAppendArgs
    _fails(fn, _args(A, k=None), -1, "null keys", None)
    _fails(fn, _args(A, q_out=None), -1, "go together", None)
    _fails(fn, _args(A, cos=4096), -1, "go together", None)
    for rot in (0, 8, 24, 144):
        _fails(fn, _args(A, cos=4096, sin=4096, rot=rot), -1, "rotated dimensions", None)
    _fails(fn, _args(A, k=4098), -1, "16 bytes", None)
    _fails(fn, _args(A, v_str=_capi._Str2(4, 128)), -1, "16 bytes", None)
    lib = _capi.lib()
    assert lib.lvsa_paged_append(None, None) == -1
    a = _args()
    assert lib.lvsa_paged_gather(C.byref(a.cache), C.byref(a.batch), 4096, 4096, -1, None) == -1
    assert lib.lvsa_paged_gather(C.byref(a.cache), C.byref(a.batch), 4100, 4096, 5, None) == -1
    assert b"16-byte" in lib.lvsa_last_error()
    assert lib.lvsa_paged_gather(C.byref(a.cache), C.byref(a.batch), 4096, 4096, 0, None) == 0    # nothing to do
    a.batch.N = 0
    assert lib.lvsa_paged_attn_fwd(C.byref(a), None) == 0


def test_workspace_sizes():
    lib, n = _capi.lib(), C.c_int64(-1)
    a = _args()
    assert lib.lvsa_paged_attn_workspace_query(C.byref(a), C.byref(n)) == 0
    # 2 rows a key head: tiles of 16 rows; one 128-key step of 128 positions x 2 heads x 2 sequences = 4 work-groups
    assert n.value == 4 * (2 * 4 * 16 * 128 + 2 * 2 * 4 * 16)
    a = _args(batch__N=0)
    assert lib.lvsa_paged_attn_workspace_query(C.byref(a), C.byref(n)) == 0 and n.value == 0
    a = _args(H=3)
    assert lib.lvsa_paged_attn_workspace_query(C.byref(a), C.byref(n)) == -1


def test_cpu_tensors_are_refused():
    t = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        lv.PagedKVCache(t, t)
    with pytest.raises(RuntimeError, match="lives on the GPU"):
        lv.PagedKVCache.allocate(2, 16, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        lv.PagedKVCache.allocate(2, 16, 2, 100)
    with pytest.raises(ValueError, match="pages"):
        lv.PagedKVCache.allocate(0, 16, 2, 128)


def test_structs_match_c(tmp_path):
    import subprocess
    from pathlib import Path

    root = Path(__file__).resolve().parent.parent
    structs = {"lvsa_paged_cache": _capi.PagedCache, "lvsa_paged_batch": _capi.PagedBatch,
               "lvsa_paged_append_args": _capi.PagedAppendArgs, "lvsa_paged_attn_args": _capi.PagedAttnArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "lvsa_amd.h"', "int main(void) {"]
    for c, py in structs.items():
        lines.append(f'printf("{c} size %zu\\n", sizeof({c}));')
        lines += [f'printf("{c} {f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    lines.append(f'printf("bits {" ".join(["%d"] * 5)}\\n", LVSA_PAGED_BAD_PAGE, LVSA_PAGED_BAD_LENGTH, LVSA_PAGED_BAD_CU, '
                 'LVSA_PAGED_BAD_APPEND, LVSA_PAGED_BAD_POSITION);')
    lines.append("return 0; }")
    (tmp_path / "l.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-D__HIP_PLATFORM_AMD__", f"-I{root / 'include'}", "-I/opt/rocm/include", str(tmp_path / "l.c"),
                    "-o", str(tmp_path / "l")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split("\n")
    got = {tuple(x.split()[:2]): int(x.split()[2]) for x in out if x and not x.startswith("bits")}
    for c, py in structs.items():
        assert got[(c, "size")] == C.sizeof(py), c
        for f, _ in py._fields_:
            assert got[(c, f)] == getattr(py, f).offset, (c, f)
    bits = [int(x) for line in out if line.startswith("bits") for x in line.split()[1:]]
    assert bits == [_capi.PAGED_BAD_PAGE, _capi.PAGED_BAD_LENGTH, _capi.PAGED_BAD_CU, _capi.PAGED_BAD_APPEND,
                    _capi.PAGED_BAD_POSITION]
