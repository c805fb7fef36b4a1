"""Calls of the paged cache's parts that once went wrong (see test_gpu_paged_parts_edges.py)."""
import ctypes as C
import math

import pytest
import torch

import longvideosparseattention_amd as lv
from longvideosparseattention_amd import _capi, hip_ops

from paged_ref import Batch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


# ── row ranges that do not ascend, each of them fine by itself ───────────────


def _weights_args(b, q, lse, weights, cu, max_q_len):
    a = _capi.PagedWeightsArgs()
    C.memmove(C.addressof(a), b.cache._pack(b.dtype), C.sizeof(_capi.PagedCache))
    a.batch.cu_seqlens, a.batch.kv_lens, a.batch.page_table = cu.data_ptr(), b.lens.data_ptr(), b.table_dev.data_ptr()
    a.batch.table_stride, a.batch.B, a.batch.max_pages = b.table_dev.stride(0), b.table_dev.shape[0], b.table_dev.shape[1]
    a.batch.N, a.H, a.scale, a.causal, a.accumulate, a.max_q_len = q.shape[0], q.shape[1], 1 / math.sqrt(b.D), 1, 1, max_q_len
    a.q, a.lse, a.weights = q.data_ptr(), lse.data_ptr(), weights.data_ptr()
    a.q_str, a.w_str = _capi._Str2(*q.stride()[:2]), _capi._Str3(*weights.stride())
    return a


@pytest.mark.parametrize("B,N,H,L", [(200, 64, 4, 128), (64, 16, 32, 500)])
def test_weights_stay_within_their_workspace(gpu, B, N, H, L):
    """Every second sequence has all the rows: more sequences with rows than there are rows."""
    b = Batch(gpu, [(0, L)] * B, 64, H, 1, 64, BF, seed=40)
    q, lse = b.randn(N, H, 64), torch.zeros(N, H, device=gpu)
    weights = b.cache.allocate_weights().fill_(2.0)
    cu = torch.tensor([N * (i % 2) for i in range(B + 1)], dtype=torch.int32, device=gpu)
    a, need = _weights_args(b, q, lse, weights, cu, N), C.c_int64()
    assert _capi.lib().lvsa_paged_weights_workspace_query(C.byref(a), C.byref(need)) == 0 and need.value > 0
    room = torch.full((4 * need.value // 4,), 77.0, device=gpu)
    a.workspace, a.workspace_bytes = room.data_ptr(), need.value
    hip_ops._call(b.cache.device, "lvsa_paged_weights", C.byref(a))
    with pytest.raises(ValueError, match="cu_seqlens"):
        b.cache.check()
    assert (room[need.value // 4:] == 77.0).all()
    assert (weights == 2.0).all()


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("hint", [None, 1, 1000])
@pytest.mark.parametrize("B", [4, 150])
def test_weights_of_a_batch_whose_rows_do_not_ascend_are_left_alone(gpu, B, hint, n):
    b = Batch(gpu, [(n, 100)] * B, 64, 4, 2, 16, BF, seed=41)
    q, lse = b.randn(b.N, 4, 64), torch.zeros(b.N, 4, device=gpu)
    weights = b.cache.allocate_weights().fill_(2.0)
    fine = b.cu.tolist()
    for at, value in ((B - 1, fine[-1] + 1), (1, fine[0] - 1), (B, fine[-1] + 1), (2, 0 if n > 1 else -1), (B - 1, 0)):
        cu = list(fine)
        cu[at] = value
        lv.paged_kv_weights(q, lse, b.cache, weights, torch.tensor(cu, dtype=torch.int32, device=gpu), b.lens, b.table_dev, max_q_len=hint)
        with pytest.raises(ValueError, match="cu_seqlens"):
            b.cache.check()
        assert (weights == 2.0).all(), (at, value)
    lv.paged_kv_weights(q, lse, b.cache, weights, *b.call(), max_q_len=hint)
    b.cache.check()
    got = torch.stack([weights[p, 0, 0] for x in b.pages for p in x[:1]])
    assert (got != 2.0).all()


# ── eviction to new pages of long sequences ──────────────────────────────────


def _one_long(gpu, page, L, keep, seed=42):
    """One sequence over a shuffled pool, random weights, and pages for what is kept of it."""
    g = torch.Generator().manual_seed(seed)
    old, new = -(-L // page), -(-keep // page)
    cache = lv.PagedKVCache.allocate(old + new + 3, page, 1, 64, device=gpu)
    order = torch.randperm(old + new + 3, generator=g).to(torch.int32)
    rows = torch.arange(L, dtype=torch.int32)
    table, to = order[:old], order[old:old + new]
    at = table.long()[torch.arange(L) // page], torch.arange(L) % page
    k = torch.zeros(cache.num_pages, page, 1, 2, dtype=torch.int32)
    k[at[0], at[1], 0, 0] = rows                         # a token's position, in its first four bytes
    cache.k[..., :4].copy_(k.view(BF).to(gpu))
    weights, w = cache.allocate_weights(), torch.rand(L, generator=g)
    like = torch.zeros(cache.num_pages, page, 1)
    like[at[0], at[1], 0] = w
    weights.copy_(like)
    lens = torch.tensor([L], dtype=torch.int32, device=gpu)
    return cache, weights, w, lens, table[None].to(gpu), to[None].clone()


@pytest.mark.parametrize("page,L,keep", [(1, 3000, 2500), (1, 2100, 1025), (2, 9000, 8001), (3, 5000, 3100), (16, 40000, 20001), (1, 40, 30)])
def test_new_pages_of_a_long_sequence(gpu, page, L, keep):
    """More new pages than a set in LDS holds: kept ones move, and one old page among them is found wherever it is."""
    cache, weights, w, lens, table, to = _one_long(gpu, page, L, keep)
    before = weights.clone()
    n = to.shape[1]
    for at, which in ((0, 0), (n - 1, table.shape[1] - 1), (n // 2, 1), (n // 2 - 1, table.shape[1] // 2)):
        bad = to.clone()
        bad[0, at] = table[0, which].cpu()
        got, kept = lv.paged_kv_evict(cache, weights, lens, table, keep, new_table=bad.to(gpu), return_kept=True)
        with pytest.raises(ValueError, match="page number"):
            cache.check()
        assert got.tolist() == [0] and (kept == -1).all() and torch.equal(weights, before)
    got, kept = lv.paged_kv_evict(cache, weights, lens, table, keep, new_table=to.to(gpu), return_kept=True)
    cache.check()
    want = w.sort(descending=True, stable=True)[1][:keep].sort()[0]
    assert got.tolist() == [keep] and torch.equal(kept[0, 0].cpu().long(), want)
    i = torch.arange(keep)
    rows = cache.k[..., :4].cpu()[to[0].long()[i // page], i % page, 0].view(torch.int32)[:, 0]
    assert torch.equal(rows.long(), want)


def test_the_check_of_new_pages_is_linear(gpu):
    """A million tokens to half a million new pages of one slot: page by page against page that is 5e11 comparisons, about
    seven seconds by one work-group; the rest of the call is some tens of milliseconds."""
    cache, weights, w, lens, table, to = _one_long(gpu, 1, 1 << 20, 1 << 19)
    to = to.to(gpu)
    lv.paged_kv_evict(cache, weights.clone(), lens[:0], table[:0], 1)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    got, kept = lv.paged_kv_evict(cache, weights, lens, table, 1 << 19, new_table=to, return_kept=True)
    end.record()
    torch.cuda.synchronize()
    cache.check()
    assert torch.equal(kept[0, 0].cpu().long(), w.sort(descending=True, stable=True)[1][:1 << 19].sort()[0])
    assert start.elapsed_time(end) < 1500.0, start.elapsed_time(end)
    print(f"{start.elapsed_time(end):.1f} ms")


@pytest.mark.parametrize("page,L,keep", [(16, 90, 40), (16, 30, 40), (1, 3000, 2500), (2, 9000, 8001), (16, 40000, 20001)])
def test_a_new_page_that_comes_twice(gpu, page, L, keep):
    """Two places of the kept tokens in one page: the sequence is not moved.  Behind the pages that it needs anything goes."""
    cache, weights, w, lens, table, to = _one_long(gpu, page, L, keep, seed=43)
    before, k = weights.clone(), cache.k.clone()
    need = -(-min(L, keep) // page)
    for a, z in {(0, need - 1), (need // 2, need - 1), (0, need // 2), (need - 2, need - 1)} - {(i, i) for i in range(need)}:
        bad = to.clone()
        bad[0, z] = bad[0, a]
        got, kept = lv.paged_kv_evict(cache, weights, lens, table, keep, new_table=bad.to(gpu), return_kept=True)
        with pytest.raises(ValueError, match="page number"):
            cache.check()
        assert got.tolist() == [0] and (kept == -1).all() and torch.equal(weights, before)
        assert torch.equal(cache.k.view(torch.int16), k.view(torch.int16))          # bits: positions are no numbers
    more = torch.cat((to[:, :need], to[:, :1].expand(1, to.shape[1] - need + 2)), 1).contiguous()
    got, kept = lv.paged_kv_evict(cache, weights, lens, table, keep, new_table=more.to(gpu), return_kept=True)
    cache.check()
    assert got.tolist() == [min(L, keep)]
    assert torch.equal(kept[0, 0, :min(L, keep)].cpu().long(), w.sort(descending=True, stable=True)[1][:keep].sort()[0])


@pytest.mark.parametrize("first,last", [(0, 0), (1 << 30, 1 << 29)])
@pytest.mark.parametrize("in_place", [True, False])
def test_a_budget_beyond_the_table_costs_no_memory(gpu, in_place, first, last):
    """As many tokens as there may be, for "all": the list of those that stay would be 343 GB, and nobody asks for it."""
    b = Batch(gpu, [(0, 20 + i) for i in range(10)], 64, 4, 4, 16, BF, seed=44, spare=40)
    weights = b.cache.allocate_weights().copy_(torch.rand(b.cache.num_pages, 16, 4, generator=b.gen))
    free = sorted(set(range(b.cache.num_pages)) - {p for x in b.pages for p in x})
    to = torch.tensor(free[:20], dtype=torch.int32).view(10, 2)
    k, w = b.cache.k.cpu(), weights.cpu()
    got = lv.paged_kv_evict(b.cache, weights, b.lens, b.table_dev, (1 << 31) - 5000, first=first, last=last,
                            new_table=None if in_place else to.to(gpu))
    b.cache.check()
    assert torch.equal(got, b.lens)
    for s, (_, L) in enumerate(b.seqs):
        at = b.pages[s] if in_place else to[s].tolist()
        i = torch.arange(L)
        now, was = torch.tensor(at)[i // 16], torch.tensor(b.pages[s])[i // 16]
        assert torch.equal(b.cache.k.cpu()[now, i % 16], k[was, i % 16]) and torch.equal(weights.cpu()[now, i % 16], w[was, i % 16])


def test_tables_without_pages(gpu):
    """Sequences that have never had a page, to new pages and in place; a length that says otherwise is a bad one."""
    cache = lv.PagedKVCache.allocate(3, 16, 2, 64, device=gpu)
    weights = cache.allocate_weights()
    none = torch.zeros(2, 0, dtype=torch.int32, device=gpu)
    some = torch.tensor([[0], [1]], dtype=torch.int32, device=gpu)
    for lens, fine in (([0, 0], True), ([5, 0], False)):
        lens = torch.tensor(lens, dtype=torch.int32, device=gpu)
        for to in (none.clone(), some[:, :0], some, None):
            for keep in (1, 7):
                got, kept = lv.paged_kv_evict(cache, weights, lens, none, keep, new_table=to, return_kept=True)
                assert got.tolist() == ([0, 0] if fine or to is not None else lens.tolist()) and (kept == -1).all()
        if fine:
            cache.check()
        else:
            with pytest.raises(ValueError, match="kv_lens"):
                cache.check()
