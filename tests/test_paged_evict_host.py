"""Eviction's arrays that share memory are refused by the C ABI, without a GPU (pointers that are never read)."""
import ctypes as C

import pytest

from longvideosparseattention_amd import _capi

S3 = _capi._Str3
LENS, TABLE, TO, KEPT, OUT = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000


def _args(**kw):
    """Three sequences of 2 heads, a table of 8 columns in rows of 12, 8 tokens to keep."""
    a = _capi.PagedEvictArgs()
    a.cache.k = a.cache.v = a.weights = 4096
    a.cache.k_str = a.cache.v_str = S3(4096, 128, 2048)
    a.cache.n_pages, a.cache.page_size, a.cache.Hkv, a.cache.D, a.cache.bits, a.cache.dtype = 10, 16, 2, 128, 16, _capi.LVSA_BF16
    a.batch.kv_lens, a.batch.page_table, a.batch.table_stride, a.batch.B, a.batch.max_pages = LENS, TABLE, 12, 3, 8
    a.w_str, a.new_table, a.new_pages, a.new_stride, a.kept, a.new_lens, a.keep = S3(32, 1, 16), TO, 2, 5, KEPT, OUT, 8
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw", [
    {"new_lens": LENS}, {"new_lens": LENS + 8}, {"new_lens": LENS - 8},              # kv_lens itself, and parts of it
    {"new_lens": TABLE + 4 * (2 * 12 + 7)}, {"new_lens": TO + 4 * (2 * 5 + 1)},      # the tables' last entries
    {"new_lens": KEPT + 4 * 47}, {"new_lens": KEPT - 8},
    {"kept": LENS - 4 * 47}, {"kept": TABLE}, {"kept": TO - 4}, {"kept": LENS + 8},
])
def test_arrays_that_share_memory_are_refused(kw):
    lib = _capi.lib()
    assert lib.lvsa_paged_evict(C.byref(_args(**kw)), None) == -1, lib.lvsa_last_error()
    assert b"share memory" in lib.lvsa_last_error(), lib.lvsa_last_error()
