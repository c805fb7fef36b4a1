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

// Brings a list into LDS, for a work-group of 256; returns the number of its keys
// below L.  list.bad: what is wrong with it.
__device__ __forceinline__ int stage_list(const PagedView& c, const ListView& v, const int32_t* blocks, const int32_t* table,
                                          int L, KeyList& list) {
  if (threadIdx.x == 0) {
    list.n = v.top;
    list.bad = 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < v.top; i += 256) {
    const int id = blocks[i];
    list.id[i] = id;
    if (id < 0) atomicMin(&list.n, i);
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

// One row tile of a list and one of the parts of its keys after the other, `ROWS`
// rows a tile, `KEYS` keys a step; `work` does a part.
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
  const int64_t total = l.units * l.splits;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t unit = quotient(w, l.splits);
    const int split = (int)(w - unit * l.splits);
    const int64_t ls = quotient(unit, p.c.Hkv);
    const int h = (int)(unit - ls * p.c.Hkv);
    const int64_t li = quotient(ls, l.subs);
    const int sub = (int)(ls - li * l.subs);
    PagedSeq sq;
    int i0;
    const int seq = paged_seq_of_list(p.c, l.v, li, lane, &sq, &i0);
    if (seq < 0) continue;
    const int r0 = i0 * p.group + sub * ROWS;
    const int i1 = i0 + l.v.tile.by < sq.n ? i0 + l.v.tile.by : sq.n;
    const int nrows = i1 * p.group;
    if (r0 >= nrows) continue;
    const int32_t* table = p.c.table + seq * p.c.table_str;
    __syncthreads();                     // the list before has been read
    const int keys = stage_list(p.c, l.v, l.blocks + (li * p.c.Hkv + h) * l.v.top, table, sq.L, list);
    const int r1 = r0 + ROWS < nrows ? r0 + ROWS - 1 : nrows - 1;
    ListKeys k{list, l.v.block, keys};
    k.L = uniform(list.bad ? 0 : k.limit(key_limit(p, sq, r1)));      // keys that the tile's last row attends
    if (list.bad && threadIdx.x == 0) paged_flag(p.c, list.bad);
    const int nb = (k.L + KEYS - 1) / KEYS;
    const DecodePart part = {sq, h, r0, nrows, (int)quotient((int64_t)split * nb, l.splits), (int)quotient((int64_t)(split + 1) * nb, l.splits),
                             w, l.splits == 1, list.bad != 0 || (sq.flags & LVSA_PAGED_BAD_LENGTH) != 0};
    work(part, k);
  }
}

template <int D, typename E, int BITS, int NT>
__global__ __launch_bounds__(256, D == 256 || (D == 192 && NT == 2) ? 1 : paged_decode_groups(D, BITS, 16 * NT)) void paged_block_decode_kernel(PagedAttnParams p, BlockAttnParams l) {
  __shared__ KeyList list;
  walk_lists<D, E, 16 * NT, paged_decode_keys(D)>(p, l, list, [&](const DecodePart& part, const ListKeys& keys) __attribute__((always_inline)) {
    decode_part<D, E, BITS, NT>(p, part, keys);
  });
}

template <int D, typename E, int BITS>
__global__ __launch_bounds__(256, D >= 192 ? 1 : 2) void paged_block_prefill_kernel(PagedAttnParams p, BlockAttnParams l) {
  __shared__ KeyList list;
  walk_lists<D, E, kPagedTile, kPagedBlock>(p, l, list, [&](const DecodePart& part, const ListKeys& keys) __attribute__((always_inline)) {
    prefill_part<D, E, BITS>(p, part, keys);
  });
}

// Joins the parts of a row: a wave per row, a lane four elements of it.
template <int D, typename E>
__global__ __launch_bounds__(256) void paged_block_merge_kernel(PagedAttnParams p, BlockAttnParams l, int rows) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < (int64_t)p.c.N * p.H; row += 4 * (int64_t)gridDim.x) {
    const int t = (uint32_t)row / (uint32_t)p.H, hq = (int)(row - (int64_t)t * p.H);
    int flags = 0, seq = -1;
    PagedSeq sq = {};
    for (int s0 = 0; s0 < p.c.B; s0 += 64) {
      PagedSeq q = {};
      bool in = false;
      if (s0 + lane < p.c.B) {
        q = paged_seq(p.c, s0 + lane);
        in = q.t0 <= t && t < q.t0 + q.n;
        flags |= q.flags;
      }
      const uint64_t m = __builtin_amdgcn_ballot_w64(in);
      if (m && seq < 0) {
        seq = s0 + __builtin_ctzll(m);
        sq = from_lane(q, __builtin_ctzll(m));
      }
    }
    if (seq < 0 || __builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) continue;    // the attention kernel's
    const int h = (uint32_t)hq / (uint32_t)p.group, i = t - sq.t0, tile = i / l.v.tile;
    const int r = (i - tile * l.v.tile.by) * p.group + (hq - h * p.group);
    const int64_t unit = ((first_list(l.v, seq, sq) + tile) * l.subs + r / rows) * p.c.Hkv + h;
    const int64_t at = unit * l.splits * rows + r % rows;
    // maxima and sums of the parts, one a lane
    float M = kNoKeys, sum = 0.f;
    for (int k = lane; k < l.splits; k += 64) M = __builtin_fmaxf(M, p.ws_ml[2 * (at + (int64_t)k * rows)]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) M = __builtin_fmaxf(M, __shfl_xor(M, d));
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < l.splits; ++k) {
      const int64_t a = at + (int64_t)k * rows;
      const float w = __builtin_amdgcn_exp2f(p.ws_ml[2 * a] - M);
      sum += w * p.ws_ml[2 * a + 1];
      if (4 * lane < D) {
        const floatx4 o = *reinterpret_cast<const floatx4*>(p.ws_o + a * D + 4 * lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += w * o[j];
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    if (4 * lane < D)
      *reinterpret_cast<u32x2*>(p.o + t * p.o_str[0] + hq * p.o_str[1] + 8 * lane) =
          u32x2{pack2<E>(acc[0] * inv, acc[1] * inv), pack2<E>(acc[2] * inv, acc[3] * inv)};
    if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? -__builtin_inff() : (M + __log2f(sum)) * 0.69314718055994530942f;
  }
}

template <int D, typename E, int BITS>
int paged_block_launch(const PagedAttnParams& p, const BlockAttnParams& l, int rows, hipStream_t stream) {
  constexpr int64_t most = 1 << 20;
  const int64_t total = l.units * l.splits;
  const dim3 grid((unsigned)(total < most ? total : most));
  if (rows == kPagedTile)
    hipLaunchKernelGGL((paged_block_prefill_kernel<D, E, BITS>), grid, dim3(256), 0, stream, p, l);
  else if (rows == 16)
    hipLaunchKernelGGL((paged_block_decode_kernel<D, E, BITS, 1>), grid, dim3(256), 0, stream, p, l);
  else
    hipLaunchKernelGGL((paged_block_decode_kernel<D, E, BITS, 2>), grid, dim3(256), 0, stream, p, l);
  const int rc = launch_status("lvsa_paged_block_attn_fwd");
  if (rc || l.splits == 1) return rc;
  const int64_t out = ceil_div((int64_t)p.c.N * p.H, 4);
  hipLaunchKernelGGL((paged_block_merge_kernel<D, E>), dim3((unsigned)(out < most ? out : most)), dim3(256), 0, stream, p, l, rows);
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
