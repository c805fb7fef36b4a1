"""Parts of a paged cache instead of all of it.

:func:`paged_attention` reads every cached key and value, and a cache only grows.
For caches that are long for either:

* :func:`paged_kv_block_means` — the mean key of every block of tokens, kept
  beside the pages and renewed behind an append;
* :func:`paged_kv_select` — for each tile of newest tokens and key head, the
  blocks whose mean scores highest with its queries;
* :func:`paged_block_attention` — attention over those blocks alone;
* :func:`paged_kv_weights` — the attention weight that the newest tokens give to
  each cached one, summed up from call to call;
* :func:`paged_kv_evict` — of every sequence the tokens with the most of it, moved
  together.

Batches, positions, streams and what the device checks are those of
:mod:`paged_kv`.  A page holds ``page_size / block_size`` blocks; block ``j`` of a
sequence is its positions ``j * block_size .. (j + 1) * block_size - 1``.

Rows of a sequence are taken in tiles of ``tile`` (1: every token for itself), which
share a list of blocks.  The lists of a batch are ``[T, H_kv, top]``: with ``tile``
1 list ``t`` is row ``t``'s (``T = N``), else tile ``i`` of sequence ``b`` has list
``cu_seqlens[b] // tile + b + i`` (``T = N // tile + B``, some of no tile), so that
their places follow from device data without a sum over the sequences.

Like the cache, none of this has a counterpart in the reference, whose sparsity is
a pattern of frames fixed beforehand (``lvsa/sparse_attention.py:643-706``).
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Tuple, Union

import torch
from torch.compiler import is_compiling

from . import _capi as capi
from . import hip_ops
from .paged_kv import (_ATTN, _ATTN_AT, _WORKSPACE, PagedKVCache, _batch, _int32, _no_gradient, _result, _span, _tokens)

__all__ = ["paged_kv_block_means", "paged_kv_select", "paged_block_attention", "paged_kv_weights", "paged_kv_evict"]

MAX_BLOCKS = 1024                              # of a list (lvsa_paged.h)

# The C structs behind cache and batch (see include/lvsa_amd.h).
_MEANS = struct.Struct("@P3qi4x")
_SELECT = struct.Struct("@3P5q7i4x")
_LISTS = struct.Struct("@P3i4x")
_WEIGHTS = struct.Struct("@3P5qf4i4xPq")
_EVICT = struct.Struct("@4P4q4i")
assert _ATTN_AT + _MEANS.size == C.sizeof(capi.PagedMeansArgs)
assert _ATTN_AT + _SELECT.size == C.sizeof(capi.PagedSelectArgs)
assert _ATTN_AT + _ATTN.size + _LISTS.size == C.sizeof(capi.PagedBlockAttnArgs)
assert _ATTN_AT + _WEIGHTS.size == C.sizeof(capi.PagedWeightsArgs)
assert _ATTN_AT + _EVICT.size == C.sizeof(capi.PagedEvictArgs)


def _beside(t: torch.Tensor, name: str, cache: PagedKVCache, shape, rows: bool) -> Tuple[int, ...]:
    """Strides of an fp32 tensor kept beside a cache's pages; ``rows``: its last dimension is contiguous, rows aligned."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        hip_ops._require_device(t, name)
    if t.dtype is not torch.float32 or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)} of torch.float32, got {list(t.shape)} of {t.dtype}")
    if t.get_device() != cache.device.index:
        raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    if t.requires_grad:
        _no_gradient(t, name)
    s = t.stride()
    P, S, H = shape[:3]
    W = shape[3] if rows else 1
    if s == ((H * S * W, W, S * W, 1) if rows else (H * S, 1, S)) and not t.data_ptr() & 15:
        lo = t.data_ptr()                    # as allocate_means and allocate_weights lay them out
        if lo >= cache._high or lo + 4 * P * S * H * W <= cache._low:
            return s
    if rows and (s[3] != 1 or (t.data_ptr() | (s[0] | s[1] | s[2]) * 4) & 15):
        raise ValueError(f"{name} needs a contiguous last dimension and rows at multiples of 16 bytes")
    at = 1
    for size, stride in sorted(((n, x) for n, x in zip(shape, s) if n > 1), key=lambda x: x[1]):
        if stride < at:
            raise ValueError(f"{name} has overlapping entries (shape {list(shape)}, strides {list(s)})")
        at = stride * (size - 1) + at
    if cache._holds(t):
        raise ValueError(f"{name} must not share memory with the cache")
    return s


def _apart(t: torch.Tensor, name: str, *others: torch.Tensor) -> None:
    lo, hi = _span(t)
    for o in others:
        a, e = _span(o) if o.numel() else (0, 0)
        if lo < e and a < hi:
            raise ValueError(f"{name} must not share memory with the other tensors of the call")


def _blocks_of(cache: PagedKVCache, means: torch.Tensor) -> int:
    """The block size that ``means`` are of."""
    parts = means.shape[1] if isinstance(means, torch.Tensor) and means.dim() == 4 else 0
    if parts < 1 or cache.page_size % parts:
        raise ValueError(f"means must be [{cache.num_pages}, parts, {cache.num_kv_heads}, {cache.head_dim}] with parts dividing the "
                         f"page size {cache.page_size}, got {list(getattr(means, 'shape', []))}")
    return cache.page_size // parts


def _queries(q: torch.Tensor, cache: PagedKVCache):
    dtype = q.dtype if isinstance(q, torch.Tensor) else None
    packed = cache._pack(dtype)
    q, ptr, *strides = _tokens(q, "q", None, cache, dtype)
    H = q.shape[1]
    if H < 1 or H % cache.num_kv_heads:
        raise ValueError(f"num heads {H} must be a multiple of kv heads {cache.num_kv_heads}")
    return packed, q, ptr, strides, H


def _scale(scale: Optional[float], D: int) -> float:
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale <= 2e38:              # times log2(e) within fp32
        raise ValueError(f"scale {scale} must be positive and at most 2e38")
    return scale


def _lists(N: int, B: int, top: int, tile: int) -> int:
    if not 1 <= top <= MAX_BLOCKS:
        raise ValueError(f"lists of {top} blocks: 1 to {MAX_BLOCKS}")
    if not 1 <= tile < 1 << 31:
        raise ValueError(f"tiles of {tile} rows")
    return N if tile == 1 else N // tile + B


def _needed(query: str, a, cache: PagedKVCache, N: int, H: int, page_table: torch.Tensor, *more: int) -> int:
    """Bytes of workspace of a call, asked once for its sizes."""
    key = (query, cache.device.index, cache.bits, cache.head_dim, cache.num_kv_heads, cache.page_size, N, H, *page_table.shape, *more)
    need = _WORKSPACE.get(key)
    if need is None:
        n = C.c_int64(0)
        with torch.cuda.device(cache.device):            # the size follows its compute units
            capi.check(query, getattr(capi.lib(), query)(C.byref(a), C.byref(n)))
        if len(_WORKSPACE) > 1024:
            _WORKSPACE.clear()
        need = _WORKSPACE[key] = n.value
    return need


def paged_kv_block_means(cache: PagedKVCache, means: torch.Tensor, kv_lens: torch.Tensor, page_table: torch.Tensor, *,
                         cu_seqlens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Write the mean cached key of blocks to ``means`` (fp32, ``[pages, parts, H_kv,
    D]`` with ``page_size / parts`` slots a block, see
    :meth:`PagedKVCache.allocate_means`), and return it.

    With the ``cu_seqlens`` of an append, behind it: the blocks that hold one of the
    newest tokens, each summed anew over the tokens that it holds.  Without: every
    block of every sequence, e.g. after an eviction.  Sums are fp32 and 64 bits,
    rounded once.  Blocks on a bad page and of a sequence with a bad length or row
    range are left alone, as are all others.  Where sequences share a page and count
    different numbers of tokens in a block of it, its mean is either's."""
    if is_compiling():
        return _outside["means"](cache, means, kv_lens, page_table, cu_seqlens=cu_seqlens)
    block = _blocks_of(cache, means)
    strides = _beside(means, "means", cache, (cache.num_pages, cache.page_size // block, cache.num_kv_heads, cache.head_dim), True)
    # how many rows there are is not known here: cu_seqlens counts them
    batch = _batch(cache, cu_seqlens, kv_lens, page_table, 0 if cu_seqlens is None else 0x7fffffff)
    if page_table.shape[0] == 0:
        return means
    a = capi.PagedMeansArgs.from_buffer_copy(cache._pack(cache.dtype or torch.bfloat16) + batch +
                                             _MEANS.pack(means.data_ptr(), *strides[:3], block))
    hip_ops._call(cache.device, "lvsa_paged_block_means", C.byref(a))
    return means


def paged_kv_select(q: torch.Tensor, cache: PagedKVCache, means: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                    page_table: torch.Tensor, top: int, *, tile: int = 1, first: int = 1, last: int = 1,
                    causal: bool = True) -> torch.Tensor:
    """Lists of blocks ``int32 [T, H_kv, top]`` for the newest tokens ``q [N, H, D]``.

    A tile's list holds up to ``top`` (at most 1024) of the blocks that its rows may
    attend (with ``causal`` up to its last row's): the sequence's ``first`` ones, those
    that its rows lie in with the ``last - 1`` before them (``last`` 0: none of these),
    and of the others those whose ``means`` have the highest product with the sum of
    the tile's queries over its rows and the query heads of the key head, equal ones
    by their number, NaN last; ascending, ``-1`` behind.  What is always in a list has
    to fit into it.  Sums are 64 bits: which blocks are taken depends on nothing but
    the values.  Lists of no tile and of sequences with a bad length are ``-1``, and all
    where ``cu_seqlens`` does not ascend; a block on a bad page counts as NaN.

    Many lists of few rows are ranked sixteen at a time where ``page_table`` has room for
    1024 blocks or fewer; where it has more they take up to four times as long."""
    if is_compiling():
        return _outside["select"](q, cache, means, cu_seqlens, kv_lens, page_table, top, tile=tile, first=first, last=last,
                                  causal=causal)
    packed, q, q_ptr, q_str, H = _queries(q, cache)
    block = _blocks_of(cache, means)
    strides = _beside(means, "means", cache, (cache.num_pages, cache.page_size // block, cache.num_kv_heads, cache.head_dim), True)
    N = q.shape[0]
    batch = _batch(cache, cu_seqlens, kv_lens, page_table, N)
    T = _lists(N, page_table.shape[0], top, tile)
    if first < 0 or last < 0 or first + (last - 1 + (1 if tile == 1 else (tile - 2) // block + 2) if last else 0) > top:
        raise ValueError(f"the first {first} blocks and the last {last} of tiles of {tile} rows do not fit into {top}")
    blocks = torch.empty(T, cache.num_kv_heads, top, dtype=torch.int32, device=cache.device)
    if page_table.shape[0] == 0:
        return blocks.fill_(-1)
    if T:
        a = capi.PagedSelectArgs.from_buffer_copy(packed + batch + _SELECT.pack(
            q_ptr, means.data_ptr(), blocks.data_ptr(), *q_str, *strides[:3], H, block, top, tile, first, last, int(bool(causal))))
        hip_ops._call(cache.device, "lvsa_paged_select", C.byref(a))
    return blocks


def paged_block_attention(q: torch.Tensor, cache: PagedKVCache, blocks: torch.Tensor, block_size: int, cu_seqlens: torch.Tensor,
                          kv_lens: torch.Tensor, page_table: torch.Tensor, *, tile: int = 1, causal: bool = True,
                          scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None):
    """:func:`paged_attention` over lists of blocks: a row of ``q [N, H, D]`` attends, of
    the keys that it would attend there, those in blocks of its tile's list in ``blocks
    [T, H_kv, top]`` (:func:`paged_kv_select`'s, or any others).

    A list ends at its first negative number; before it the numbers ascend and name
    blocks that start within the sequence.  Rows whose list does not, or names a block
    on a bad page, and rows of a sequence with a bad length are NaN; a row that attends
    nothing gives 0 and ``-inf``.  Shapes, types, ``out``, ``lse``, rows of no sequence
    and precision are as for :func:`paged_attention`; the split of a list's keys follows
    from the shapes alone, so that a row's result does not depend on its batch's
    lengths."""
    if is_compiling():
        return _outside["attention"](q, cache, blocks, block_size, cu_seqlens, kv_lens, page_table, tile=tile, causal=causal,
                                     scale=scale, return_lse=return_lse, out=out)
    packed, q, q_ptr, q_str, H = _queries(q, cache)
    N, _, D = q.shape
    scale = _scale(scale, D)
    if block_size < 1 or cache.page_size % block_size:
        raise ValueError(f"blocks of {block_size} slots do not divide pages of {cache.page_size}")
    batch = _batch(cache, cu_seqlens, kv_lens, page_table, N)
    _int32(blocks, "blocks", 3, cache.device)
    top = blocks.shape[2]
    T = _lists(N, page_table.shape[0], top, tile)
    if tuple(blocks.shape) != (T, cache.num_kv_heads, top):
        raise ValueError(f"blocks must be [{T}, {cache.num_kv_heads}, top] for {N} rows in tiles of {tile}, got {list(blocks.shape)}")
    blocks = blocks.contiguous()
    fresh = out is None
    out, o_ptr, *o_str = _result(out, q, "out", cache, blocks)
    lse = torch.empty(N, H, dtype=torch.float32, device=q.device) if return_lse else None
    if N and page_table.shape[0] == 0:
        if fresh:
            out.zero_()
        if return_lse:
            lse.fill_(-math.inf)
    elif N:
        a = capi.PagedBlockAttnArgs.from_buffer_copy(packed + batch + _ATTN.pack(
            q_ptr, o_ptr, 0 if lse is None else lse.data_ptr(), *q_str, *o_str, scale, H, int(bool(causal)), 1 if fresh else 2, 0, 0,
            0, 0) + _LISTS.pack(blocks.data_ptr(), block_size, top, tile))
        need = _needed("lvsa_paged_block_attn_workspace_query", a, cache, N, H, page_table, block_size, top, tile)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.attn.workspace, a.attn.workspace_bytes = ws.data_ptr(), need
        hip_ops._call(cache.device, "lvsa_paged_block_attn_fwd", C.byref(a))
    return (out, lse) if return_lse else out


def paged_kv_weights(q: torch.Tensor, lse: torch.Tensor, cache: PagedKVCache, weights: torch.Tensor, cu_seqlens: torch.Tensor,
                     kv_lens: torch.Tensor, page_table: torch.Tensor, *, causal: bool = True, scale: Optional[float] = None,
                     accumulate: bool = True, max_q_len: Optional[int] = None) -> torch.Tensor:
    """Add to ``weights [pages, page_size, H_kv]`` (fp32, see
    :meth:`PagedKVCache.allocate_weights`) what the newest tokens ``q [N, H, D]`` give to
    every cached token of their sequence, and return it: the sum of ``exp(scale q.k -
    lse)`` over the sequence's rows that attend the token and the query heads of the
    key head, with ``lse [N, H]`` as :func:`paged_attention` returns it for the same
    ``causal`` and ``scale``.

    The newest tokens' own weights start from 0, so slots need no clearing before; with
    ``accumulate=False`` all of the sequence's do (the weights of one chunk alone).
    Rows whose ``lse`` is not finite give nothing.  Sequences without new rows or with a
    bad length, tokens on bad pages and slots of no sequence are left alone, and all
    where ``cu_seqlens`` does not ascend.  Sequences that share pages must not be in one
    call (each would add to the same weights).  Scores and sums are fp32, in an order that
    follows from the shapes alone.  ``max_q_len`` (the most rows of a sequence) only
    chooses a kernel: without it more rows than sequences are taken for one long sequence,
    which runs slower for a few rows of each (8 sequences of 2 rows over 8000 keys 52
    instead of 30 us)."""
    if is_compiling():
        return _outside["weights"](q, lse, cache, weights, cu_seqlens, kv_lens, page_table, causal=causal, scale=scale,
                                   accumulate=accumulate, max_q_len=max_q_len)
    packed, q, q_ptr, q_str, H = _queries(q, cache)
    N, _, D = q.shape
    scale = _scale(scale, D)
    strides = _beside(weights, "weights", cache, (cache.num_pages, cache.page_size, cache.num_kv_heads), False)
    hip_ops._require_device(lse, "lse")
    if lse.dtype is not torch.float32 or tuple(lse.shape) != (N, H):
        raise ValueError(f"lse must be [{N}, {H}] of torch.float32, got {list(lse.shape)} of {lse.dtype}")
    if lse.device != cache.device:
        raise ValueError(f"lse is on {lse.device}, the cache on {cache.device}")
    if lse.requires_grad:
        _no_gradient(lse, "lse")
    lse = lse.contiguous()
    _apart(weights, "weights", q, lse)
    batch = _batch(cache, cu_seqlens, kv_lens, page_table, N)
    mq = int(max_q_len or 0)
    if mq < 0:
        raise ValueError(f"max_q_len {max_q_len} must not be negative")
    if N and page_table.shape[0]:
        a = capi.PagedWeightsArgs.from_buffer_copy(packed + batch + _WEIGHTS.pack(
            q_ptr, lse.data_ptr(), weights.data_ptr(), *q_str, *strides, scale, H, int(bool(causal)), int(bool(accumulate)),
            min(mq, 0x7fffffff), 0, 0))
        need = _needed("lvsa_paged_weights_workspace_query", a, cache, N, H, page_table, mq)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        hip_ops._call(cache.device, "lvsa_paged_weights", C.byref(a))
    return weights


def paged_kv_evict(cache: PagedKVCache, weights: torch.Tensor, kv_lens: torch.Tensor, page_table: torch.Tensor, keep: int, *,
                   first: int = 0, last: int = 0, new_table: Optional[torch.Tensor] = None,
                   return_kept: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Cut every sequence to ``keep`` tokens a key head; returns the new ``kv_lens``
    (and with ``return_kept`` the kept ones' old positions, ``int32 [B, H_kv, keep]``, -1
    behind).

    Kept are the ``first`` tokens, the newest ``last`` and, of the others, those of the
    largest ``weights`` (:func:`paged_kv_weights`; equal ones by their position, NaN
    last); a sequence of no more than ``keep`` keeps all.  Their keys, values, scales
    and weights move, in their order, to positions ``0 .. keep - 1``, every head's for
    itself: on the pages of ``new_table [B, new_pages]``, or without it on the
    sequence's own first pages.  Slots behind them stay as they are.  Keys that were
    turned by their positions keep their angles: new tokens' positions go on in
    :func:`paged_kv_append`'s ``positions``.  Means of blocks are the caller's to renew.
    The room of ``page_table`` chooses the kernel: with more than 32768 slots sequences of a
    few thousand tokens take up to three times as long.

    Pages of ``new_table`` belong to nothing else in the call: a sequence that finds,
    among those that its kept tokens need, one of its old pages, a page twice or a
    number outside the cache, or has a bad length, is not moved (all ``-1``, its new
    length 0, in place its old one) and noted in the status; pages of other sequences
    are not looked for.  Pages that sequences share are not to be cut in place."""
    if is_compiling():
        return _outside["evict"](cache, weights, kv_lens, page_table, keep, first=first, last=last, new_table=new_table,
                                 return_kept=return_kept)
    strides = _beside(weights, "weights", cache, (cache.num_pages, cache.page_size, cache.num_kv_heads), False)
    batch = _batch(cache, None, kv_lens, page_table, 0)
    B, pages = page_table.shape
    if not 1 <= keep < (1 << 31) - 4097 or first < 0 or last < 0 or first + last > keep:
        raise ValueError(f"{keep} tokens to keep, the first {first} and the last {last} among them")
    if keep > pages * cache.page_size and not return_kept:      # all, whatever they are: no list of more than there can be
        keep, first, last = max(pages * cache.page_size, 1), 0, 0
    to = row = new_pages = 0
    if new_table is not None:
        _int32(new_table, "new_table", 2, cache.device)
        new_pages = new_table.shape[1]
        if new_table.shape[0] != B:
            raise ValueError(f"new_table has {new_table.shape[0]} sequences, page_table {B}")
        if B and new_pages and new_table.data_ptr() == page_table.data_ptr():
            raise ValueError("new_table is page_table: leave it out to cut sequences where they lie")
        if new_pages * cache.page_size < min(keep, pages * cache.page_size):
            raise ValueError(f"{new_pages} new pages of {cache.page_size} slots do not hold {keep} tokens")
        row = new_table.stride(0) if B > 1 else new_pages
        if row < new_pages:
            raise ValueError("new_table rows overlap")
        to = new_table.data_ptr() or kv_lens.data_ptr()          # no page of an empty table is read; null would be "in place"
    lens = torch.empty(B, dtype=torch.int32, device=cache.device)
    kept = torch.empty(B, cache.num_kv_heads, keep, dtype=torch.int32, device=cache.device)
    if B:
        packed = cache._pack(cache.dtype or torch.bfloat16)
        a = capi.PagedEvictArgs.from_buffer_copy(packed + batch + _EVICT.pack(
            weights.data_ptr(), to, kept.data_ptr(), lens.data_ptr(), *strides, row, new_pages, keep, first, last))
        hip_ops._call(cache.device, "lvsa_paged_evict", C.byref(a))
    return (lens, kept) if return_kept else lens


# See paged_kv: within torch.compile the calls break the graph and run as they are.
_outside = {name: torch.compiler.disable(fn) for name, fn in
            (("means", paged_kv_block_means), ("select", paged_kv_select), ("attention", paged_block_attention),
             ("weights", paged_kv_weights), ("evict", paged_kv_evict))}
