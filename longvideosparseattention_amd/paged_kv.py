"""Keys and values kept between calls: a paged cache, and attention over it.

A chunk-by-chunk video generator keeps the frames it has finished as keys and
values, and the understanding (text) half of a model keeps its tokens'.  Here
they live in pages of ``page_size`` token slots (one latent frame, or a few
tokens), and a page table names the pages of every sequence in order, so that
sequences grow, end and share pages without moving anything:

* :class:`PagedKVCache` — the pages, in 16 bits or in 4 (E2M1 codes with a
  power-of-two scale for every 32 values of a row: 4.25 bits a value);
* :func:`paged_kv_append` — new tokens' keys and values written behind the
  cached ones, keys (and queries) turned by their positions on the way;
* :func:`paged_kv_gather` — every sequence read back as padded
  ``[B, S, H_kv, D]`` tensors, e.g. for :func:`lvsa_attention`;
* :func:`paged_attention` — attention of the newest tokens of every sequence
  over all its cached ones, causal or not, from a single token to whole chunks.

A batch is three int32 device tensors, so one captured graph serves every step:
``cu_seqlens [B + 1]`` (rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` of the
packed ``[N, H, D]`` tensors are sequence ``b``'s newest tokens), ``kv_lens [B]``
(its cached tokens, the newest included) and ``page_table [B, max_pages]``.
Row ``cu_seqlens[b] + i`` has position ``kv_lens[b] - n_b + i`` with ``n_b`` the
sequence's rows.  Rows behind ``cu_seqlens[B]`` belong to no sequence (a padded
batch).  Every call only enqueues work on the current stream.

What the host cannot see is checked on the device: page numbers outside the
cache, lengths beyond the table, row ranges outside the batch and positions
outside the angle table never leave the caller's memory.  They spoil what they
concern — attention's rows of that sequence, gathered tokens (NaN), an append's
tokens (left out) — and set the cache's status, which
:meth:`PagedKVCache.check` turns into an error.  Where ``cu_seqlens`` does
not ascend within the packed rows, nobody knows whose rows are whose: attention
returns NaN in every row, an append takes a row for the first sequence whose
range holds it.

What works on parts of a cache (blocks selected by a score, tokens that are worth
keeping) is in :mod:`paged_parts`.

Inside ``torch.compile`` the calls break the graph and run as they are.

The reference has no cache: it attends over whole tensors
(``lvsa/sparse_attention.py:643-706``) that its adapters have rotated before
(``lvsa/rope.py:10-27``).
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional, Tuple

import torch
from torch.compiler import is_compiling

from . import _capi as capi
from . import hip_ops

__all__ = ["PagedKVCache", "paged_kv_append", "paged_kv_gather", "paged_attention"]

_INT32 = torch.int32
_DTYPES = {torch.bfloat16: capi.LVSA_BF16, torch.float16: capi.LVSA_FP16}
_STATUS = {
    capi.PAGED_BAD_PAGE: "a page number outside the cache",
    capi.PAGED_BAD_LENGTH: "a length in kv_lens that is negative or beyond the page table",
    capi.PAGED_BAD_CU: "cu_seqlens that do not ascend within the packed rows",
    capi.PAGED_BAD_APPEND: "more new tokens than kv_lens counts",
    capi.PAGED_BAD_POSITION: "a position outside the rows of cos and sin",
    capi.PAGED_BAD_BLOCK: "a list of blocks that does not ascend or names one behind its sequence's end",
}

# The C structs as they are packed (see include/lvsa_amd.h): one copy per
# call instead of a ctypes assignment per field.
_CACHE = struct.Struct("@4P12q4i2iP")
_BATCH = struct.Struct("@3Pq3i4x")
_ATTN = struct.Struct("@3P4qf5iPq")
_APPEND = struct.Struct("@4P8q3P4i")
_ATTN_AT = _CACHE.size + _BATCH.size
assert _CACHE.size == C.sizeof(capi.PagedCache) and _BATCH.size == C.sizeof(capi.PagedBatch)
assert _ATTN_AT + _ATTN.size == C.sizeof(capi.PagedAttnArgs)
assert _ATTN_AT + _APPEND.size == C.sizeof(capi.PagedAppendArgs)


def _cache_rows(t: torch.Tensor, name: str, dtype: torch.dtype, width: int, align: int) -> Tuple[int, int, int]:
    hip_ops._require_device(t, name)
    _no_gradient(t, name)
    if t.dim() != 4 or t.shape[3] != width or t.dtype != dtype:
        raise ValueError(f"{name} must be [pages, page_size, H_kv, {width}] of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    es = t.element_size()
    if t.stride(3) != 1 or (t.data_ptr() | (t.stride(0) | t.stride(1) | t.stride(2)) * es) % align:
        raise ValueError(f"{name} needs a contiguous last dimension and rows at multiples of {align} bytes")
    # rows that share memory would make an append overwrite its own tokens
    at = 1
    for size, stride in sorted(((t.shape[i], t.stride(i)) for i in range(4) if t.shape[i] > 1), key=lambda x: x[1]):
        if stride < at:
            raise ValueError(f"{name} has overlapping rows (shape {tuple(t.shape)}, strides {t.stride()})")
        at = stride * (size - 1) + at
    return t.stride(0), t.stride(1), t.stride(2)


def _no_gradient(t: torch.Tensor, name: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient: the paged cache has no backward pass (detach it or use no_grad)")


class PagedKVCache:
    """Pages of keys and values.

    16 bits: ``k`` and ``v`` are ``[pages, page_size, H_kv, D]`` in bf16 or fp16.
    4 bits: ``uint8 [pages, page_size, H_kv, D / 2]`` codes (element ``d`` in byte
    ``d // 2``, the low four bits for even ``d``) and ``k_scale`` / ``v_scale``,
    ``uint8 [pages, page_size, H_kv, D / 32]``: a value is its E2M1 number times
    ``2^(scale - 127)`` (scale 255: NaN) as the caller's 16-bit type holds it, which
    is exactly, for every scale that an append writes, and as an infinity beyond
    its range.  Strides are free as long as rows start at multiples of
    16 bytes; :meth:`allocate` lays the rows of a head within a page next to each
    other, which reads fastest.  Two caches may share pages of one allocation.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        hip_ops._require_device(k, "cache keys")
        if k.dim() != 4:
            raise ValueError(f"cache keys must be [pages, page_size, H_kv, D], got shape {tuple(k.shape)}")
        if (k_scale is None) != (v_scale is None):
            raise ValueError("k_scale and v_scale go together")
        self.bits = 16 if k_scale is None else 4
        self.num_pages, self.page_size, self.num_kv_heads = (int(x) for x in k.shape[:3])
        self.head_dim = hip_ops.kernel_head_dim(int(k.shape[3]) * (1 if self.bits == 16 else 2))
        if min(self.num_pages, self.page_size, self.num_kv_heads) < 1:
            raise ValueError(f"a cache needs pages, slots and heads, got shape {tuple(k.shape)}")
        if self.bits == 16 and k.dtype not in _DTYPES:
            raise TypeError(f"unsupported cache dtype {k.dtype}: bf16 or fp16, or uint8 codes with scales")
        self.dtype = k.dtype if self.bits == 16 else None
        if v.shape != k.shape:
            raise ValueError(f"cache keys {tuple(k.shape)} and values {tuple(v.shape)} differ in shape")
        strides = []
        stored = k.dtype if self.bits == 16 else torch.uint8
        for t, name in ((k, "cache keys"), (v, "cache values")):
            strides += _cache_rows(t, name, stored, k.shape[3], 16)
        for t, name in ((k_scale, "key scales"), (v_scale, "value scales")):
            if t is None:
                strides += (0, 0, 0)
                continue
            strides += _cache_rows(t, name, torch.uint8, self.head_dim // 32, 1)
            if t.shape[:3] != k.shape[:3]:
                raise ValueError(f"{name} {tuple(t.shape)} do not match the codes {tuple(k.shape)}")
        self.device = k.device
        for t in (v, k_scale, v_scale):
            if t is not None and t.device != self.device:
                raise ValueError(f"cache tensors on {self.device} and {t.device}")
        if k.data_ptr() == v.data_ptr() or (k_scale is not None and k_scale.data_ptr() == v_scale.data_ptr()):
            raise ValueError("cache keys and values must not share memory")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._spans = [_span(t) for t in (k, v, k_scale, v_scale) if t is not None]
        self._low, self._high = min(a for a, _ in self._spans), max(e for _, e in self._spans)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        ptrs = [0 if t is None else t.data_ptr() for t in (k, v, k_scale, v_scale)]
        self._packed = {
            dt: _CACHE.pack(*ptrs, *strides, self.num_pages, self.page_size, self.num_kv_heads, self.head_dim, self.bits,
                            code, self.status.data_ptr())
            for dt, code in _DTYPES.items() if self.bits == 4 or dt == self.dtype}

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
                 bits: int = 16, device: Optional[torch.device] = None) -> "PagedKVCache":
        """A cache of its own memory (zeroed), ``dtype`` for 16 bits."""
        hip_ops.kernel_head_dim(head_dim)
        if bits not in (16, 4):
            raise ValueError(f"caches hold 16 or 4 bits, not {bits}")
        if bits == 16 and dtype not in _DTYPES:
            raise TypeError(f"unsupported cache dtype {dtype}: bf16 or fp16")
        if min(num_pages, page_size, num_kv_heads) < 1:
            raise ValueError(f"a cache needs pages, slots and heads, got {num_pages}, {page_size}, {num_kv_heads}")
        device = torch.device("cuda") if device is None else torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"a cache lives on the GPU, not on {device}")

        def rows(width, dt):
            return torch.zeros(num_pages, num_kv_heads, page_size, width, dtype=dt, device=device).transpose(1, 2)

        if bits == 16:
            return cls(rows(head_dim, dtype), rows(head_dim, dtype))
        return cls(rows(head_dim // 2, torch.uint8), rows(head_dim // 2, torch.uint8),
                   rows(head_dim // 32, torch.uint8), rows(head_dim // 32, torch.uint8))

    def allocate_means(self, block_size: int) -> torch.Tensor:
        """Zeroed means of all blocks of ``block_size`` slots, a divisor of the page
        size: fp32 ``[pages, page_size / block_size, H_kv, D]`` (see
        :func:`paged_kv_block_means`)."""
        if block_size < 1 or self.page_size % block_size:
            raise ValueError(f"blocks of {block_size} slots do not divide pages of {self.page_size}")
        return torch.zeros(self.num_pages, self.num_kv_heads, self.page_size // block_size, self.head_dim, dtype=torch.float32,
                           device=self.device).transpose(1, 2)

    def allocate_weights(self) -> torch.Tensor:
        """Zeroed weights of all slots: fp32 ``[pages, page_size, H_kv]`` (see :func:`paged_kv_weights`)."""
        return torch.zeros(self.num_pages, self.num_kv_heads, self.page_size, dtype=torch.float32, device=self.device).transpose(1, 2)

    def _holds(self, t: torch.Tensor) -> bool:
        """Whether ``t`` lies within the bounds of the cache's tensors."""
        lo, hi = _span(t)
        return t.numel() > 0 and any(lo < e and a < hi for a, e in self._spans)

    @torch.compiler.disable
    def check(self) -> None:
        """Raise ``ValueError`` for what earlier calls found wrong on the device,
        on whatever stream, and forget it.  Waits for the device; what calls
        enqueued meanwhile find is the next check's."""
        torch.cuda.synchronize(self.device)
        taken = torch.empty_like(self.status)
        hip_ops._call(self.device, "lvsa_paged_take_status", self.status.data_ptr(), taken.data_ptr())
        found = int(taken.item())
        if found:
            raise ValueError("paged cache: " + "; ".join(text for bit, text in _STATUS.items() if found & bit))

    def _pack(self, dtype: torch.dtype) -> bytes:
        packed = self._packed.get(dtype)
        if packed is None:
            raise TypeError(f"unsupported dtype {dtype} over a {self.bits}-bit cache" +
                            (f" of {self.dtype}" if self.bits == 16 else "") + ": " +
                            ("the cache's" if self.bits == 16 else "bf16 or fp16"))
        return packed


def _int32(t: torch.Tensor, name: str, dims: int, device: torch.device) -> None:
    if isinstance(t, torch.Tensor) and t.dtype is _INT32 and t.dim() == dims and t.get_device() == device.index and t.stride(-1) == 1:
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        hip_ops._require_device(t, name)
    if t.dtype != torch.int32 or t.dim() != dims:
        raise TypeError(f"{name} must be a {dims}-D int32 tensor, got {t.dim()}-D {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    if t.shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def _batch(cache: PagedKVCache, cu_seqlens: Optional[torch.Tensor], kv_lens: torch.Tensor, page_table: torch.Tensor,
           N: int) -> bytes:
    device = cache.device
    _int32(kv_lens, "kv_lens", 1, device)
    _int32(page_table, "page_table", 2, device)
    B, max_pages = page_table.shape
    if kv_lens.shape[0] != B:
        raise ValueError(f"kv_lens has {kv_lens.shape[0]} sequences, page_table {B}")
    cu = 0
    if cu_seqlens is not None:
        _int32(cu_seqlens, "cu_seqlens", 1, device)
        if cu_seqlens.shape[0] != B + 1:
            raise ValueError(f"cu_seqlens has {cu_seqlens.shape[0]} entries, {B} sequences need {B + 1}")
        cu = cu_seqlens.data_ptr()
    row = page_table.stride(0) if B > 1 else max_pages
    if row < max_pages:
        raise ValueError("page_table rows overlap")
    return _BATCH.pack(cu, kv_lens.data_ptr(), page_table.data_ptr(), row, B, max_pages, N)


def _tokens(t: torch.Tensor, name: str, heads: Optional[int], cache: PagedKVCache, dtype: torch.dtype):
    """A ``[N, heads, D]`` tensor the kernels can read (other layouts are
    repacked on the device), its address and its first two strides."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        hip_ops._require_device(t, name)
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [N, {'H' if heads is None else heads}, {cache.head_dim}], got {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {dtype}")
    if t.get_device() != cache.device.index:
        raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
    if t.requires_grad:
        _no_gradient(t, name)
    s0, s1, s2 = t.stride()
    ptr = t.data_ptr()
    if s2 != 1 or (ptr | ((s0 | s1) * 2)) & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        s0, s1, _ = t.stride()
        ptr = t.data_ptr()
    return t, ptr, s0, s1


def _result(out: Optional[torch.Tensor], like: torch.Tensor, name: str, cache: PagedKVCache, *inputs: torch.Tensor):
    """The tensor a call writes (``out``, or a new one) with its address and strides; ``inputs``: what else it reads."""
    if out is None:
        out = torch.empty_like(like, memory_format=torch.contiguous_format)
        _, H, D = like.shape
        return out, out.data_ptr(), H * D, D
    if not isinstance(out, torch.Tensor) or out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must be {tuple(like.shape)} of {like.dtype} on {like.device}")
    if out.stride(2) != 1 or (out.data_ptr() | ((out.stride(0) | out.stride(1)) * 2)) & 15:
        raise ValueError(f"{name} needs a contiguous last dimension and rows at multiples of 16 bytes")
    for t in (like, *inputs):
        if t.numel() and _span(out)[0] < _span(t)[1] and _span(t)[0] < _span(out)[1]:
            raise ValueError(f"{name} must not share memory with the input")
    if cache._holds(out):
        raise ValueError(f"{name} must not share memory with the cache")
    N, H, D = out.shape
    a, b = sorted(((N, out.stride(0)), (H, out.stride(1))), key=lambda x: x[1])
    if (a[0] > 1 and a[1] < D) or (b[0] > 1 and b[1] < (a[1] * (a[0] - 1) if a[0] > 1 else 0) + D):
        raise ValueError(f"{name} has overlapping rows")
    return out, out.data_ptr(), out.stride(0), out.stride(1)


def _span(t: torch.Tensor) -> Tuple[int, int]:
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def paged_kv_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                    kv_lens: torch.Tensor, page_table: torch.Tensor, *, q: Optional[torch.Tensor] = None,
                    cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                    positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                    q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Write new tokens' ``k`` / ``v [N, H_kv, D]`` to the cache; returns ``q
    [N, H, D]`` turned likewise (``q_out`` or a new tensor), or ``None`` without
    ``q``.

    ``kv_lens`` counts the new tokens already; their pages must be in the table.
    ``cos`` / ``sin [P, rot / 2]`` (fp32) turn the first ``rot`` dimensions of keys
    and queries, ``rot`` a multiple of 16: token at position ``p`` takes row ``p``,
    or row ``positions[t]`` with an int32 ``positions [N]`` (a video token's place
    in its grid).  Pairs are ``(2i, 2i + 1)`` if ``interleaved``, else ``(i, i +
    rot / 2)``; ``(a, b)`` becomes ``(a cos - b sin, b cos + a sin)`` in fp32 (for a
    4-bit cache in 64 bits, so that the nearest code is the exact value's).

    4-bit caches keep, for every 32 values of a row, the smallest power of two
    ``2^e`` with ``6 * 2^e`` at least their largest magnitude (``-23 <= e <= 13``:
    beyond 49152 values are clamped) and the nearest E2M1 number of each quotient,
    ties to even; 32 values with an infinity or a NaN among them become NaN.

    Rows of no sequence are left alone, in the cache and in ``q_out`` (undefined
    in a new tensor).  No two tokens of a call may have the same slot.  ``k`` and
    ``v`` may be views of the cache itself (they are copied first); ``q_out`` must
    not share memory with the inputs or the cache.  A token
    with a bad page, length, row range or position is left out, its row of
    ``q_out`` NaN."""
    if is_compiling():
        return _outside["append"](cache, k, v, cu_seqlens, kv_lens, page_table, q=q, cos=cos, sin=sin, positions=positions,
                                  interleaved=interleaved, q_out=q_out)
    dtype = k.dtype if isinstance(k, torch.Tensor) else None
    packed = cache._pack(dtype)
    Hkv = cache.num_kv_heads
    k, k_ptr, *k_str = _tokens(k, "k", Hkv, cache, dtype)
    v, v_ptr, *v_str = _tokens(v, "v", Hkv, cache, dtype)
    N = k.shape[0]
    if v.shape[0] != N:
        raise ValueError(f"k has {N} tokens, v {v.shape[0]}")
    # tokens that are the cache's own, whose slots the call may write: read before it
    if k_ptr < cache._high and k_ptr + 2 * (N * k_str[0] + Hkv * k_str[1]) > cache._low and cache._holds(k):
        k, k_ptr, *k_str = _tokens(k.clone(memory_format=torch.contiguous_format), "k", Hkv, cache, dtype)
    if v_ptr < cache._high and v_ptr + 2 * (N * v_str[0] + Hkv * v_str[1]) > cache._low and cache._holds(v):
        v, v_ptr, *v_str = _tokens(v.clone(memory_format=torch.contiguous_format), "v", Hkv, cache, dtype)
    batch = _batch(cache, cu_seqlens, kv_lens, page_table, N)
    H = q_ptr = qo_ptr = 0
    q_str = qo_str = (0, 0)
    if q is not None:
        q, q_ptr, *q_str = _tokens(q, "q", None, cache, dtype)
        H = q.shape[1]
        if q.shape[0] != N or H < 1:
            raise ValueError(f"k has {N} tokens, q {tuple(q.shape)}")
        q_out, qo_ptr, *qo_str = _result(q_out, q, "q_out", cache, k, v)
    elif q_out is not None:
        raise ValueError("q_out without q")
    rot = angles = cos_ptr = sin_ptr = pos_ptr = 0
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin go together")
    if cos is not None:
        for t, name in ((cos, "cos"), (sin, "sin")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda:
                hip_ops._require_device(t, name)
            if t.dtype is not torch.float32 or t.dim() != 2 or not t.is_contiguous() or (t is not cos and t.shape != cos.shape):
                raise TypeError(f"{name} must be a contiguous fp32 [positions, rot / 2] tensor like its partner")
            if t.get_device() != cache.device.index:
                raise ValueError(f"{name} is on {t.device}, the cache on {cache.device}")
            if t.requires_grad:
                _no_gradient(t, name)
        angles, rot = cos.shape
        rot *= 2
        if rot % 16 or not 0 < rot <= cache.head_dim:
            raise ValueError(f"cos and sin turn {rot} dimensions: a multiple of 16 up to {cache.head_dim}")
        cos_ptr, sin_ptr = cos.data_ptr(), sin.data_ptr()
    if positions is not None:
        if cos is None:
            raise ValueError("positions without cos and sin")
        _int32(positions, "positions", 1, cache.device)
        if positions.shape[0] != N:
            raise ValueError(f"k has {N} tokens, positions {positions.shape[0]}")
        pos_ptr = positions.data_ptr()
    if N == 0:
        return q_out
    a = capi.PagedAppendArgs.from_buffer_copy(packed + batch + _APPEND.pack(
        k_ptr, v_ptr, q_ptr, qo_ptr, *k_str, *v_str, *q_str, *qo_str, cos_ptr, sin_ptr, pos_ptr, H, rot,
        int(bool(interleaved)), angles))
    hip_ops._call(cache.device, "lvsa_paged_append", C.byref(a))
    return q_out


def paged_kv_gather(cache: PagedKVCache, kv_lens: torch.Tensor, page_table: torch.Tensor, max_len: int, *,
                    dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached keys and values of every sequence, ``[B, max_len, H_kv, D]``
    each: its first ``max_len`` tokens, zeros behind its end.

    ``dtype``: the cache's for 16 bits; bf16 (the default) or fp16 for 4, both of
    which hold every 4-bit value exactly.  A bad page gives NaN for its tokens, a
    bad length for the whole sequence."""
    if is_compiling():
        return _outside["gather"](cache, kv_lens, page_table, max_len, dtype=dtype)
    if dtype is None:
        dtype = cache.dtype or torch.bfloat16
    packed = cache._pack(dtype)
    if max_len < 0:
        raise ValueError(f"max_len {max_len} is negative")
    batch = _batch(cache, None, kv_lens, page_table, 0)
    shape = (page_table.shape[0], int(max_len), cache.num_kv_heads, cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache.device)
    v = torch.empty(shape, dtype=dtype, device=cache.device)
    if k.numel():
        a = capi.PagedAttnArgs()               # its first two members are what the call takes
        C.memmove(C.addressof(a), packed + batch, _ATTN_AT)
        hip_ops._call(cache.device, "lvsa_paged_gather", C.byref(a.cache), C.byref(a.batch), k.data_ptr(), v.data_ptr(),
                      int(max_len))
    return k, v


_WORKSPACE = {}


def _workspace_bytes(a: "capi.PagedAttnArgs", key, device: torch.device) -> int:
    need = _WORKSPACE.get(key)
    if need is None:
        n = C.c_int64(0)
        with torch.cuda.device(device):        # the size follows its compute units
            capi.check("lvsa_paged_attn_workspace_query",
                       capi.lib().lvsa_paged_attn_workspace_query(C.byref(a), C.byref(n)))
        if len(_WORKSPACE) > 1024:
            _WORKSPACE.clear()
        need = _WORKSPACE[key] = n.value
    return need


def paged_attention(q: torch.Tensor, cache: PagedKVCache, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                    page_table: torch.Tensor, *, causal: bool = True, scale: Optional[float] = None,
                    return_lse: bool = False, max_q_len: Optional[int] = None, max_kv_len: Optional[int] = None,
                    out: Optional[torch.Tensor] = None):
    """Attention of the newest tokens ``q [N, H, D]`` over the cache: ``o [N, H,
    D]``, and with ``return_lse`` the natural-log ``lse [N, H]`` (fp32).

    ``H`` is a multiple of the cache's heads (grouped heads).  A row attends its
    sequence's cached keys, with ``causal`` those up to its own position; keys it
    does not attend have no effect on it, NaN and infinities included.  A row
    without keys gives 0 and ``-inf``.  ``scale`` defaults to ``1 / sqrt(D)``.

    ``max_q_len`` (the most rows of a sequence) and ``max_kv_len`` (the longest
    cache) only choose a kernel and its split: results are right whatever they say.
    Without ``max_q_len`` more rows than sequences are taken for one long sequence,
    which runs slower for a few rows of each; without ``max_kv_len`` the table's
    width counts, and where that has room for long caches a short chunk takes up to
    twice the time (20 tokens over 2000 keys 33 instead of 17 us). ``out`` must not
    share memory with ``q`` or the cache; rows of no sequence are left as they were
    in ``out`` and are 0 in a new tensor (``lse``: ``-inf`` in both cases).

    Scores, softmax and sums are fp32; weights enter the second product in ``q``'s
    type (in fp16 with fewer bits below 2^-23 of their row's largest).  A run
    repeated gives the same bits, but the order of a row's sums follows from the
    lengths of the whole batch: beside other sequences a result may differ within
    rounding.  A row whose scores are all ``-inf`` counts as one without keys;
    scaled scores from 9e7 (fp16) or 1.4e9 (bf16) on may give NaN."""
    if is_compiling():
        return _outside["attention"](q, cache, cu_seqlens, kv_lens, page_table, causal=causal, scale=scale,
                                     return_lse=return_lse, max_q_len=max_q_len, max_kv_len=max_kv_len, out=out)
    dtype = q.dtype if isinstance(q, torch.Tensor) else None
    packed = cache._pack(dtype)
    q, q_ptr, *q_str = _tokens(q, "q", None, cache, dtype)
    N, H, D = q.shape
    if H < 1 or H % cache.num_kv_heads:
        raise ValueError(f"num heads {H} must be a multiple of kv heads {cache.num_kv_heads}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale <= 2e38:              # times log2(e) within fp32
        raise ValueError(f"scale {scale} must be positive and at most 2e38")
    batch = _batch(cache, cu_seqlens, kv_lens, page_table, N)
    fresh = out is None
    out, o_ptr, *o_str = _result(out, q, "out", cache)
    lse = torch.empty(N, H, dtype=torch.float32, device=q.device) if return_lse else None
    if N:
        mq, mk = int(max_q_len or 0), int(max_kv_len or 0)
        if mq < 0 or mk < 0:
            raise ValueError(f"max_q_len {max_q_len} and max_kv_len {max_kv_len} must not be negative")
        head = (q_ptr, o_ptr, 0 if lse is None else lse.data_ptr(), *q_str, *o_str, scale, H, int(bool(causal)),
                1 if fresh else 2, min(mq, 0x7fffffff), min(mk, 0x7fffffff))
        a = capi.PagedAttnArgs.from_buffer_copy(packed + batch + _ATTN.pack(*head, 0, 0))
        need = _workspace_bytes(a, (cache.device.index, cache.bits, D, cache.num_kv_heads, cache.page_size, N, H, *page_table.shape,
                                    mq, mk), cache.device)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        hip_ops._call(cache.device, "lvsa_paged_attn_fwd", C.byref(a))
    return (out, lse) if return_lse else out


# Within torch.compile the calls break the graph and run as they are: they take
# addresses and call C.  (Called through these only there: a wrapper on every call
# costs half a microsecond.)
_outside = {name: torch.compiler.disable(fn) for name, fn in
            (("append", paged_kv_append), ("gather", paged_kv_gather), ("attention", paged_attention))}
