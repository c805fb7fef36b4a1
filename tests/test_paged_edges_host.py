"""Refusals of the paged cache's C ABI that its other host test leaves out; pointers are never read, no kernel runs."""
import ctypes as C

import pytest

from longvideosparseattention_amd import _capi

# Sizes of every call here: two rows of two key heads and four query heads of 128, two sequences.
AT = 1 << 30


def _fill(a):
    c, b = a.cache, a.batch
    c.k, c.v = 1 << 40, 1 << 41
    c.k_str = c.v_str = _capi._Str3(4096, 128, 2048)
    c.n_pages, c.page_size, c.Hkv, c.D, c.bits, c.dtype = 10, 16, 2, 128, 16, _capi.LVSA_BF16
    b.cu_seqlens = b.kv_lens = b.page_table = 4096
    b.table_stride, b.B, b.max_pages, b.N = 8, 2, 8, 2
    a.H = 4
    return a


def _refused(fn, a, text):
    lib = _capi.lib()
    assert getattr(lib, fn)(C.byref(a), None) == -1, lib.lvsa_last_error()
    assert text in lib.lvsa_last_error(), lib.lvsa_last_error()


def test_take_status_needs_both_places():
    lib = _capi.lib()
    assert lib.lvsa_paged_take_status(None, 4096, None) == -1 and lib.lvsa_paged_take_status(4096, None, None) == -1
    assert b"null pointer" in lib.lvsa_last_error()


ROW = 4 * 128 * 2          # bytes of one token's query heads


@pytest.mark.parametrize("shift", [0, ROW, 2 * ROW - 256, -ROW, 16 - 2 * ROW])
def test_results_that_share_their_inputs_memory(shift):
    a = _fill(_capi.PagedAttnArgs())
    a.q, a.o, a.scale = AT, AT + shift, 1.0
    a.q_str = a.o_str = _capi._Str2(512, 128)
    a.workspace, a.workspace_bytes = 1 << 42, 1 << 40
    _refused("lvsa_paged_attn_fwd", a, b"o must not share memory with q")
    a.o_str = _capi._Str2(-512, 128)
    a.o = AT + shift + ROW                            # the same two rows, from the last one on
    _refused("lvsa_paged_attn_fwd", a, b"o must not share memory with q")
    for other in "qkv":
        a = _fill(_capi.PagedAppendArgs())
        a.k, a.v, a.q = 1 << 31, 1 << 32, 1 << 33
        setattr(a, other, AT)
        a.q_out = AT + (shift if other == "q" else shift // 2 // 16 * 16)
        a.k_str = a.v_str = _capi._Str2(256, 128)
        a.q_str = a.qo_str = _capi._Str2(512, 128)
        _refused("lvsa_paged_append", a, b"q_out must not share memory with k, v and q")
