"""Refusals of the paged cache's C ABI that its other host test leaves out; pointers are never read, no kernel runs."""

from longvideosparseattention_amd import _capi

def test_take_status_needs_both_places():
    lib = _capi.lib()
    assert lib.lvsa_paged_take_status(None, 4096, None) == -1 and lib.lvsa_paged_take_status(4096, None, None) == -1
    assert b"null pointer" in lib.lvsa_last_error()
