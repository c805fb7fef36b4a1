// Attention over lists of blocks of the paged cache (gfx950).  A list's keys are
// numbered one after the other, key i at slot i % block of the list's block i /
// block.  Blocks ascend, so that what a row attends (its positions below a limit) is
// the keys below a limit in that numbering, and the dense kernels' work on a row tile
// (decode_part, prefill_part) serves lists as it is, with the keys looked up here.
#pragma once
#include "lvsa_paged_attn.h"

namespace lvsa {
namespace {

// A list in LDS: block numbers, and the page and first slot of each.
struct KeyList {
  int id[kListMax];
  int2 at[kListMax];
  int n, bad;
};

// The sequence of list `list` (the same for every lane; every lane reads one
// sequence), or -1, and its tile's first row in it.
__device__ __forceinline__ int paged_seq_of_list(const PagedView& c, const ListView& v, int64_t list, int lane, PagedSeq* q,
                                                 int* i0) {
  for (int s0 = 0; s0 < c.B; s0 += 64) {
    const int s = s0 + lane;
    PagedSeq mine = {};
    int64_t at = -1;
    if (s < c.B) {
      mine = paged_seq(c, s);
      at = list - first_list(v, s, mine);
      if (at >= list_count(v, mine)) at = -1;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(at >= 0);
    if (m) {
      const int i = __builtin_ctzll(m);
      *q = from_lane(mine, i);
      *i0 = __builtin_amdgcn_readlane((int)at, i) * v.tile.by;
      return s0 + i;
    }
  }
  return -1;
}

// A thread's part of a list, on its way from memory: blocks tid, tid + 256, ...
struct ListIds {
  int id[kListMax / 256];
  __device__ __forceinline__ void load(const ListView& v, const int32_t* blocks) {
#pragma unroll
    for (int k = 0; k < kListMax / 256; ++k) {
      const int i = threadIdx.x + 256 * k;
      id[k] = 256 * k < v.top ? blocks[i < v.top ? i : v.top - 1] : 0;
    }
  }
};

// Brings a list into LDS, for a work-group of 256; returns the number of its keys
// below L.  list.bad: what is wrong with it.
__device__ __forceinline__ int stage_list(const PagedView& c, const ListView& v, const ListIds& ids, const int32_t* table,
                                          int L, KeyList& list) {
  if (threadIdx.x == 0) {
    list.n = v.top;
    list.bad = 0;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kListMax / 256; ++k) {
    const int i = threadIdx.x + 256 * k;
    if (i >= v.top) continue;
    list.id[i] = ids.id[k];
    if (ids.id[k] < 0) atomicMin(&list.n, i);
  }
  __syncthreads();
  const int n = list.n;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int id = list.id[i];
    int flags = 0, page = 0, slot = 0;
    if ((int64_t)id * v.block.by >= L || (i > 0 && list.id[i - 1] >= id)) {
      flags = LVSA_PAGED_BAD_BLOCK;
    } else {
      const int e = id / v.parts;
      page = table[e];
      slot = (id - e * v.parts.by) * v.block.by;
      if ((uint32_t)page >= (uint32_t)c.n_pages) {
        page = 0;
        flags = LVSA_PAGED_BAD_PAGE;
      }
    }
    list.at[i] = int2{page, slot};
    if (flags) atomicOr(&list.bad, flags);
  }
  __syncthreads();
  if (list.bad || n == 0) return 0;
  const int last = list.id[n - 1] * v.block.by, left = L - last;
  return (n - 1) * v.block.by + (left < v.block.by ? left : v.block.by);
}

// Keys of a staged list at positions below `lim`.
__device__ __forceinline__ int list_limit(const KeyList& list, const Divisor& block, int lim) {
  const int b = lim / block;
  int lo = 0, hi = list.n;               // first entry that is not below block b
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list.id[mid] < b) lo = mid + 1;
    else hi = mid;
  }
  return lo * block.by + (lo < list.n && list.id[lo] == b ? lim - b * block.by : 0);
}

// See PagedKeys.
struct ListKeys {
  static constexpr bool kStaged = true;
  const KeyList& list;
  Divisor block;
  int L;
  __device__ __forceinline__ int page(int k) const { return list.at[k / block].x; }
  __device__ __forceinline__ PagedRow row(int k, int page) const {
    const int e = k / block;
    return PagedRow{page, list.at[e].y + k - e * block.by, true};
  }
  __device__ __forceinline__ bool together(int k, int n, int* slot) const {
    const int e = k / block, off = k - e * block.by;
    if (k + n > L || off + n > block.by) return false;
    *slot = list.at[e].y + off;
    return true;
  }
  __device__ __forceinline__ int limit(int lim) const {
    const int k = list_limit(list, block, lim);
    return k < L ? k : L;
  }
};

// The work-group's share: a row tile of a list and some of its key steps after the
// other, `ROWS` rows a tile, `KEYS` keys a step; `work` does a part.
template <int D, typename E, int ROWS, int KEYS, typename Work>
__device__ __forceinline__ void walk_lists(const PagedAttnParams& p, const BlockAttnParams& l, KeyList& list, Work work) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  int flags = 0;
  for (int s = lane; s < p.c.B; s += 64) flags |= paged_seq(p.c, s).flags;
  if (blockIdx.x == 0 && wave == 0 && flags) paged_flag(p.c, flags);
  if (__builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) {
    spoil_rows<E>(p, D, lane, wave, 4);
    return;
  }
  if (p.fill_tail) fill_tail_rows(p, D, lane, wave, 4);
  const int share = share_of(blockIdx.x, p.grid);
  if (share < 0) return;
  const int64_t first = unit_start(l.work, p.grid, share), end = unit_start(l.work, p.grid, share + 1);
  for (int64_t w = first; w < end;) {
    const int64_t unit = quotient(w, l.steps), w0 = unit * l.steps;
    const int s0 = (int)(w - w0), s1 = end - w0 < l.steps ? (int)(end - w0) : l.steps;
    w = w0 + s1;
    const int64_t hl = quotient(unit, l.subs);
    const int sub = (int)(unit - hl * l.subs);
    const int h = (int)quotient(hl, l.v.lists);
    const int64_t li = hl - (int64_t)h * l.v.lists;
    ListIds ids;
    ids.load(l.v, l.blocks + (li * p.c.Hkv + h) * l.v.top);
    PagedSeq sq;
    int i0;
    const int seq = paged_seq_of_list(p.c, l.v, li, lane, &sq, &i0);
    if (seq < 0) continue;
    const int r0 = i0 * p.group + sub * ROWS;
    const int i1 = tile_end(l.v, sq, i0);
    const int nrows = i1 * p.group;
    if (r0 >= nrows) continue;
    const int32_t* table = p.c.table + seq * p.c.table_str;
    __syncthreads();                     // the list before has been read
    const int keys = stage_list(p.c, l.v, ids, table, sq.L, list);
    const int r1 = r0 + ROWS < nrows ? r0 + ROWS - 1 : nrows - 1;
    ListKeys k{list, l.v.block, keys};
    k.L = uniform(list.bad ? 0 : k.limit(key_limit(p, sq, r1)));      // keys that the tile's last row attends
    if (list.bad && threadIdx.x == 0) paged_flag(p.c, list.bad);
    const int nb = (k.L + KEYS - 1) / KEYS;
    const DecodePart part = {sq, h, r0, nrows, (int)quotient((int64_t)s0 * nb, l.steps), (int)quotient((int64_t)s1 * nb, l.steps),
                             2 * (int64_t)share + (first < w0 ? 1 : 0),          // see decode_slots
                             s0 == 0 && s1 == l.steps, list.bad != 0 || (sq.flags & LVSA_PAGED_BAD_LENGTH) != 0};
    work(part, k);
  }
}

// Few rows: bound by the bytes of the lists' keys and values, and for one list by trips
// to memory one after the other (batch and list, page table, keys).  45 lists of 8 heads,
// 32 blocks of 64 of 128, 78 to 85 us, 4.6 TB/s; 4 bits, 40 of 64 blocks, 51 + 5 us, 3.4
// TB/s; one of 512 keys 11 + 4 us.
template <int D, typename E, int BITS, int NT>
__global__ __launch_bounds__(256, D == 256 || (D == 192 && NT == 2) ? 1 : paged_decode_groups(D, BITS, 16 * NT)) void paged_block_decode_kernel(PagedAttnParams p, BlockAttnParams l) {
  __shared__ KeyList list;
  walk_lists<D, E, 16 * NT, paged_decode_keys(D)>(p, l, list, [&](const DecodePart& part, const ListKeys& keys) __attribute__((always_inline)) {
    decode_part<D, E, BITS, NT>(p, part, keys);
  });
}

// Tiles of many rows: bound as the dense kernel (MFMA busy 33%, VALU issuing 37%), with
// fewer work-groups than fill it evenly: 4680 tokens of 12 heads of 128, tiles of 128, 48
// blocks of 104 of 28080 keys 186 to 198 us, 740 TFLOP/s (dense attention over as many
// keys, in tiles of 256 rows, 183 us).  Copies of 16 keys that cross blocks take the slow
// way: blocks of 104 cost a tenth more than of 64, 128 or 512.
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256, D >= 192 ? 1 : 2) void paged_block_prefill_kernel(PagedAttnParams p, BlockAttnParams l) {
  __shared__ KeyList list;
  walk_lists<D, E, kPagedTile, kPagedBlock>(p, l, list, [&](const DecodePart& part, const ListKeys& keys) __attribute__((always_inline)) {
    prefill_part<D, E, BITS>(p, part, keys);
  });
}

// Joins the partials of row tiles that shares divide, 32 rows a work-group: a lane has
// four elements of a row and a wave R rows at a time, of every partial on their way at
// once.  Bound by the partials' bytes.
template <int D, typename E>
__global__ __launch_bounds__(256) void paged_block_merge_kernel(PagedAttnParams p, BlockAttnParams l, int rows) {
  typedef E e4 __attribute__((ext_vector_type(4)));
  constexpr int LR = D / 4, R = 64 / LR;               // lanes per row, rows per wave
  constexpr int STEPS = 8 / R;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int sub = lane / LR, d = 4 * (lane % LR);
  int bad = 0;
  for (int s = lane; s < p.c.B; s += 64)
    bad |= paged_seq(p.c, s).flags & LVSA_PAGED_BAD_CU;
  if (__builtin_amdgcn_ballot_w64(bad != 0)) return;   // spoiled already
  const int64_t units = quotient(l.work, l.steps);
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const DecodeSlots parts = decode_slots(l.work, p.grid, unit * l.steps, l.steps);
    if (parts.count == 0) continue;                    // written by the attention kernel
    const int64_t hl = quotient(unit, l.subs);
    const int part = (int)(unit - hl * l.subs), h = (int)quotient(hl, l.v.lists);
    PagedSeq sq;
    int i0;
    if (paged_seq_of_list(p.c, l.v, hl - (int64_t)h * l.v.lists, lane, &sq, &i0) < 0) continue;
    const int r0 = i0 * p.group + part * rows, i1 = tile_end(l.v, sq, i0);
    const int end = i1 * p.group - r0 < rows ? i1 * p.group - r0 : rows;       // rows of the tile
    if (32 * (int)blockIdx.y >= end || sub >= R) continue;
    float M[STEPS], sum[STEPS];
    floatx4 o[STEPS];
    int r[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      r[k] = 32 * blockIdx.y + 8 * wave + R * k + sub;
      M[k] = kNoKeys;
      sum[k] = 0.f;
      o[k] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    if (32 * (int)blockIdx.y + 8 * wave >= end) continue;
    for (int i = 0; i < parts.count; ++i) {
      const int64_t slot = (i == 0 ? parts.first : parts.rest + 2 * i) * rows;
      float m[STEPS], s[STEPS];
      floatx4 x[STEPS];
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {                // rows past the end: the last one
        const int64_t at = slot + (r[k] < end ? r[k] : end - 1);
        m[k] = p.ws_ml[2 * at];
        s[k] = p.ws_ml[2 * at + 1];
        x[k] = *reinterpret_cast<const floatx4*>(p.ws_o + at * D + d);
      }
#pragma unroll
      for (int k = 0; k < STEPS; ++k) {
        const float top = __builtin_fmaxf(M[k], m[k]);
        const float a = __builtin_amdgcn_exp2f(M[k] - top), b = __builtin_amdgcn_exp2f(m[k] - top);
        sum[k] = sum[k] * a + s[k] * b;
        o[k] = o[k] * a + x[k] * b;
        M[k] = top;
      }
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (r[k] >= end) continue;
      const int i = (r0 + r[k]) / p.group, hq = h * p.group + (r0 + r[k]) - i * p.group;
      const int64_t t = (int64_t)sq.t0 + i;
      const float inv = sum[k] == 0.f ? 0.f : 1.0f / sum[k];
      *reinterpret_cast<e4*>(p.o + t * p.o_str[0] + hq * p.o_str[1] + 2 * d) =
          e4{(E)(o[k][0] * inv), (E)(o[k][1] * inv), (E)(o[k][2] * inv), (E)(o[k][3] * inv)};
      if (p.lse && d == 0)
        p.lse[t * p.H + hq] = sum[k] == 0.f ? -__builtin_inff() : (M[k] + __log2f(sum[k])) * 0.69314718055994530942f;
    }
  }
}

template <int D, typename E, int BITS>
int paged_block_launch(const PagedAttnParams& p, const BlockAttnParams& l, int rows, hipStream_t stream) {
  const dim3 grid((unsigned)(8 * ceil_div(p.grid, 8)));           // see share_of
  if (rows == kPagedTile)
    hipLaunchKernelGGL((paged_block_prefill_kernel<D, E, BITS>), grid, dim3(256), 0, stream, p, l);
  else if (rows == 16)
    hipLaunchKernelGGL((paged_block_decode_kernel<D, E, BITS, 1>), grid, dim3(256), 0, stream, p, l);
  else
    hipLaunchKernelGGL((paged_block_decode_kernel<D, E, BITS, 2>), grid, dim3(256), 0, stream, p, l);
  const int rc = launch_status("lvsa_paged_block_attn_fwd");
  if (rc || l.work == p.grid * (int64_t)l.steps) return rc;      // every share is one unit
  const int64_t units = l.work / l.steps, most = 1 << 16;
  hipLaunchKernelGGL((paged_block_merge_kernel<D, E>), dim3((unsigned)(units < most ? units : most), (unsigned)ceil_div(rows, 32)), dim3(256),
                     0, stream, p, l, rows);
  return launch_status("lvsa_paged_block_attn_fwd");
}

template <int D>
int paged_block_launch(const PagedAttnParams& p, const BlockAttnParams& l, int bits, int rows, bool bf16, hipStream_t stream) {
  if (bf16)
    return bits == 16 ? paged_block_launch<D, __bf16, 16>(p, l, rows, stream) : paged_block_launch<D, __bf16, 4>(p, l, rows, stream);
  return bits == 16 ? paged_block_launch<D, _Float16, 16>(p, l, rows, stream) : paged_block_launch<D, _Float16, 4>(p, l, rows, stream);
}

}  // namespace
}  // namespace lvsa
