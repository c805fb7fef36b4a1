"""The paged cache where calls leave the usual path: padded batches with the caller's result, arguments that the
device finds wrong, values that a type cannot hold, far larger and smaller weights, many sequences, other streams."""
import pytest
import torch

import longvideosparseattention_amd as lv

import paged_ref as ref
from paged_ref import Batch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
ROOM = 700000        # keys a page table may have room for: chunks then run on the kernels of long caches


# ── rows of no sequence ──────────────────────────────────────────────────────


@pytest.mark.parametrize("n,room", [(1, 0), (20, 0), (60, ROOM), (150, ROOM)])
def test_lse_of_rows_of_no_sequence_beside_out(gpu, n, room):
    """A padded batch with the caller's result: its rows of no sequence stay as they were, their lse is -inf."""
    b = Batch(gpu, [(n, 200), (n, 170)], 128, 4, 2, 16, BF, tail=5, extra_columns=room // 16)
    q = b.randn(b.N, 4, 128)
    want = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, return_lse=True)
    out = torch.full_like(q, 9.0)
    held = [torch.full((b.N, 4), 5.0, device=gpu) for _ in range(8)]      # what a new tensor finds in its memory
    del held
    o, lse = lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, out=out, return_lse=True)
    assert o is out and (o[b.n_rows:] == 9.0).all() and (lse[b.n_rows:] == float("-inf")).all()
    assert torch.equal(o[:b.n_rows], want[0][:b.n_rows]) and torch.equal(lse, want[1])
    lv.paged_attention(q, b.cache, *b.call(), max_q_len=n, out=out.fill_(3.0))
    assert (out[b.n_rows:] == 3.0).all() and torch.equal(out[:b.n_rows], want[0][:b.n_rows])
    b.cache.check()
