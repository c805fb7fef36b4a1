// Eviction from the paged key/value cache on gfx950: which tokens of a sequence and
// head stay, and their way to the front.
#include "lvsa_paged_host.h"
#include "lvsa_paged_rows.h"

using namespace lvsa;

namespace lvsa {
namespace {

struct EvictParams {
  PagedView c;
  char* w;
  int64_t w_str[3];                      // bytes
  const int32_t* to;                     // new_table, or null: in place
  int64_t to_str;
  int32_t* kept; int32_t* new_lens;
  int32_t keep, first, last;
};

// A weight as a number that sorts like it: NaN below -inf, 0 and -0 alike.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, w + 0.f);
  return b >> 31 ? ~b : b | 1u << 31;
}

constexpr int kEvictHeld = 32;             // ranks that a thread of the selection holds
constexpr int kEvictSet = 1024;            // new pages that are few: their set is in LDS

// Page numbers in memory that has twice as many places: each at the first free place
// from a hash of it on, so that a search ends.  For a work-group of 1024.
struct PageSet {
  int* at;
  uint32_t places;
  __device__ __forceinline__ uint32_t first(int page) const { return (uint32_t)((uint64_t)((uint32_t)page * 0x9e3779b1u) * places >> 32); }
  __device__ __forceinline__ uint32_t next(uint32_t i) const { return i + 1 < places ? i + 1 : 0; }
  __device__ __forceinline__ void clear() const {
    for (uint32_t i = threadIdx.x; i < places; i += 1024) __hip_atomic_store(&at[i], -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // Whether the page was there already.
  __device__ __forceinline__ bool add(int page) const {
    for (uint32_t i = first(page);; i = next(i)) {
      const int was = atomicCAS(&at[i], -1, page);
      if (was == -1 || was == page) return was == page;
    }
  }
  __device__ __forceinline__ bool holds(int page) const {
    for (uint32_t i = first(page);; i = next(i)) {
      const int here = __hip_atomic_load(&at[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (here == -1 || here == page) return here == page;
    }
  }
};

// Whether one of many new pages lies outside the cache, is an old one of the sequence
// or comes twice, as far as this thread sees, in the time of reading both tables: with a set
// in `row`, the head's part of `kept`, which has a place for every kept token and is
// written behind this (half of them at a time where pages are single tokens).
__device__ __forceinline__ bool many_pages_meet(const PagedView& c, const int32_t* table, int pages, const int32_t* to, int news,
                                                int32_t* row, int keep) {
  const PageSet set = {row, (uint32_t)keep};
  const int some = keep / 2;
  bool odd = false;
  auto meet = [&]() __attribute__((always_inline)) {
    __threadfence();
    __syncthreads();
  };
  for (int i0 = 0, i1 = 0; i1 < news; i0 = i1) {
    i1 = news - i0 < some ? news : i0 + some;
    set.clear();
    meet();
    for (int i = i0 + (int)threadIdx.x; i < i1; i += 1024) {
      const int page = to[i];
      odd |= (uint32_t)page >= (uint32_t)c.n_pages || set.add(page);
    }
    meet();
    for (int i = i1 + (int)threadIdx.x; i < news; i += 1024) {
      const int page = to[i];
      if ((uint32_t)page < (uint32_t)c.n_pages) odd |= set.holds(page);
    }
    for (int e = threadIdx.x; e < pages; e += 1024) {
      const int page = table[e];
      if ((uint32_t)page < (uint32_t)c.n_pages) odd |= set.holds(page);
    }
    meet();
  }
  return odd;
}

// One work-group per sequence and head: finds the keep-th highest weight by halving the
// range of the ranks, which its threads hold (R each, or read again in every step where
// a sequence is longer), and lists the tokens from it on.  A wave has consecutive
// tokens, so that one exchange of counts gives all their places.  Latency: the page
// table, the weights, 15 to 32 counts; 64 heads of up to 16000 tokens 31 us (on 64 of 256
// units: half of it waits, the rest is addresses and counts), 256 of 2112 15 to 19.
// (Counting the values of 11 bits at a time in LDS: 53 us.)  R by the room of the table,
// whatever its sequences fill of it: 16 ranks a thread 31 us, 32 43, and read again in
// every step beyond 32768 tokens.  With the moves, in a table for 131072: the 64 heads 175
// us instead of 57, 256 heads of 2112 tokens 167 instead of 142, and 12 heads of 131040
// tokens 1.4 ms, of which 1.25 are the selection.
template <int R>
__global__ __launch_bounds__(1024) void paged_evict_select_kernel(EvictParams p) {
  __shared__ int count_s[2][16];
  __shared__ int gt_s[16], eq_s[16];
  __shared__ uint32_t lo_s[16], hi_s[16];
  __shared__ int bad_s, set_s[2 * kEvictSet];
  const int Hkv = p.c.Hkv, tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  for (int64_t u = blockIdx.x; u < (int64_t)p.c.B * Hkv; u += gridDim.x) {
    const int b = (int)quotient(u, Hkv), h = (int)(u - (int64_t)b * Hkv);
    const PagedSeq sq = paged_seq(p.c, 0, 0, p.c.lens[b]);
    const int L = sq.L, left = L < p.keep ? L : p.keep;
    const int32_t* table = p.c.table + b * p.c.table_str;
    const int32_t* to = p.to ? p.to + b * p.to_str : nullptr;
    int32_t* kept = p.kept + u * p.keep;
    // A wave's tokens: `per` times 64 from wave * 64 * per on.
    const int per = (L + 1023) / 1024, first = wave * 64 * per + lane;
    auto rank_at = [&](int pos) __attribute__((always_inline)) {
      if (pos < p.first || pos >= L - p.last) return ~0u;
      const PagedRow at = paged_row(p.c, pos, table[page_of(p.c, pos)]);
      return rank_of(*reinterpret_cast<const float*>(p.w + at.page * p.w_str[0] + at.slot * p.w_str[1] + h * p.w_str[2]));
    };
    uint32_t held[R ? R : 1];
    if constexpr (R > 0) {
      if (L > p.keep) {                    // pages, then weights, all on their way at once
        int64_t at[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const int pos = key_within(first + 64 * (k < per ? k : 0), L);
          at[k] = table[page_of(p.c, pos)];
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
          const int pos = key_within(first + 64 * (k < per ? k : 0), L);
          const PagedRow row = paged_row(p.c, pos, (int)at[k]);
          at[k] = row.page * p.w_str[0] + row.slot * p.w_str[1] + h * p.w_str[2];
        }
#pragma unroll
        for (int k = 0; k < R; ++k) held[k] = __builtin_bit_cast(uint32_t, *reinterpret_cast<const float*>(p.w + at[k]));
      }
    }
    const int pages = L > 0 ? page_of(p.c, L - 1) + 1 : 0, news = left > 0 ? page_of(p.c, left - 1) + 1 : 0;
    const bool few = to && news <= kEvictSet;
    const PageSet set = {set_s, 2 * kEvictSet};
    const int fresh = few && tid < news ? to[tid] : 0;
    __syncthreads();                       // LDS of the head before has been read
    if (tid == 0) bad_s = sq.flags;
    if (few) set.clear();
    __syncthreads();
    bool odd = (uint32_t)fresh >= (uint32_t)p.c.n_pages;       // a page outside the cache, or a new one that is an old one or comes twice
    if (few) {
      if (tid < news && !odd) odd = set.add(fresh);
      __syncthreads();
    } else if (to) {
      odd |= many_pages_meet(p.c, table, pages, to, news, kept, p.keep);
    }
    for (int e = tid; e < pages; e += 1024) {
      const int page = table[e];
      const bool in = (uint32_t)page < (uint32_t)p.c.n_pages;
      odd |= !in || (few && set.holds(page));
    }
    if (odd) atomicOr(&bad_s, LVSA_PAGED_BAD_PAGE);
    __syncthreads();
    const int bad = bad_s;
    if (bad) {
      if (h == 0 && tid == 0) {
        paged_flag(p.c, bad);
        p.new_lens[b] = to ? 0 : p.c.lens[b];
      }
      for (int i = tid; i < p.keep; i += 1024) kept[i] = -1;
      continue;
    }
    if (h == 0 && tid == 0) p.new_lens[b] = left;
    for (int i = left + tid; i < p.keep; i += 1024) kept[i] = -1;
    if (L <= p.keep) {
      for (int i = tid; i < L; i += 1024) kept[i] = i;
      continue;
    }
    if constexpr (R > 0) {
#pragma unroll
      for (int k = 0; k < R; ++k) {        // past the end 0, which no bound keeps
        const int pos = first + 64 * k;
        held[k] = k >= per || pos >= L ? 0 : pos < p.first || pos >= L - p.last ? ~0u : rank_of(__builtin_bit_cast(float, held[k]));
      }
    }
    // `test` of a wave's tokens, 64 at a time
    auto each = [&](auto test) __attribute__((always_inline)) {
      if constexpr (R > 0) {
#pragma unroll
        for (int k = 0; k < R; ++k)
          if (k < per) test(first + 64 * k, held[k]);
      } else {
#pragma unroll 1
        for (int k = 0; k < per; ++k) test(first + 64 * k, first + 64 * k < L ? rank_at(first + 64 * k) : 0);
      }
    };
    uint32_t lo = ~0u, hi = 0;
    each([&](int pos, uint32_t r) __attribute__((always_inline)) {
      if (pos < L && r < lo) lo = r;
      if (r != ~0u && r > hi) hi = r;
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t a = __shfl_xor((int)lo, d), z = __shfl_xor((int)hi, d);
      lo = a < lo ? a : lo;
      hi = z > hi ? z : hi;
    }
    if (lane == 0) {
      lo_s[wave] = lo;
      hi_s[wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      lo = lo_s[w] < lo ? lo_s[w] : lo;
      hi = hi_s[w] > hi ? hi_s[w] : hi;
    }
    // at least `keep` ranks are >= lo, and fewer are > hi
    int parity = 0;
    for (bool found = false; lo < hi && !found; parity ^= 1) {
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      int c = 0;
      each([&](int pos, uint32_t r) __attribute__((always_inline)) { c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(r >= mid)); });
      if (lane == 0) count_s[parity][wave] = c;
      __syncthreads();
      c = 0;
#pragma unroll
      for (int w = 0; w < 16; ++w) c += count_s[parity][w];
      if (c >= p.keep) lo = mid;
      else hi = mid - 1;
      found = c == p.keep;
    }
    // all above the bound, and the first of those equal to it
    int gt = 0, eq = 0;
    each([&](int pos, uint32_t r) __attribute__((always_inline)) {
      gt += __builtin_popcountll(__builtin_amdgcn_ballot_w64(r > lo));
      eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(pos < L && r == lo));
    });
    if (lane == 0) {
      gt_s[wave] = gt;
      eq_s[wave] = eq;
    }
    __syncthreads();
    int put = 0, equal = p.keep;           // places before this wave's, equal ones that still find room
#pragma unroll
    for (int w = 0; w < 16; ++w) equal -= gt_s[w];
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w >= wave) continue;
      const int e = eq_s[w] < equal ? eq_s[w] : equal;
      put += gt_s[w] + e;
      equal -= e;
    }
    const uint64_t before = (1ull << lane) - 1;
    each([&](int pos, uint32_t r) __attribute__((always_inline)) {
      const uint64_t g = __builtin_amdgcn_ballot_w64(r > lo), e = __builtin_amdgcn_ballot_w64(pos < L && r == lo);
      const int mine = __builtin_popcountll(e & before), es = __builtin_popcountll(e), taken = es < equal ? es : equal;
      const int at = put + __builtin_popcountll(g & before) + (mine < equal ? mine : equal);
      // (weights that another stream changes between two readings may give other counts)
      if (((g >> lane & 1) || ((e >> lane & 1) && mine < equal)) && (uint32_t)at < (uint32_t)p.keep) kept[at] = pos;
      put += __builtin_popcountll(g) + taken;
      equal -= taken;
    });
    if constexpr (R == 0) {
      if (wave == 15)
        for (int i = put + lane; i < p.keep; i += 64) kept[i] = i;
    }
  }
}

// Old place of kept token i of a sequence, and its new one.
struct Move {
  PagedRow from, at;
};
__device__ __forceinline__ Move move_of(const EvictParams& p, int b, int old, int i) {
  const int32_t* table = p.c.table + b * p.c.table_str;
  const int32_t* to = p.to ? p.to + b * p.to_str : table;
  return Move{paged_row(p.c, old, table[page_of(p.c, old)]), paged_row(p.c, i, to[page_of(p.c, i)])};
}

// To pages of their own: nothing is read that is written, all rows at once.  A thread
// has a 16-byte piece of a key and of its value; the first ones of a row bring its
// scales and weight.  Bound by the bytes; rows pass the L2 by on their way out, which the
// next call would find full of them: 64 heads' 2048 tokens of 128 and their selection 60.5
// us, 65 without.  Four pieces a thread on their way (two: 65, eight: 79; one behind its
// page numbers: 68).
template <int D, int BITS>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(EvictParams p, int per) {
  constexpr int CH = D * BITS / 128;       // 16-byte pieces of a row
  for (int64_t u = blockIdx.x; u < (int64_t)p.c.B * p.c.Hkv * per; u += gridDim.x) {
    const int64_t bh = quotient(u, per);
    const int part = (int)(u - bh * per), b = (int)quotient(bh, p.c.Hkv), h = (int)(bh - (int64_t)b * p.c.Hkv);
    const int left = p.new_lens[b];
    const int32_t* kept = p.kept + bh * p.keep;
    constexpr int U = 4;                   // pieces on their way
    const int64_t n = (int64_t)left * CH;
    for (int64_t k0 = (int64_t)part * 256 * U + threadIdx.x; k0 < n; k0 += (int64_t)per * 256 * U) {
      u32x4 x[U], y[U];
      Move m[U];
      int c[U], i[U], old[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int64_t k = k0 + 256 * j < n ? k0 + 256 * j : n - 1;
        i[j] = (int)quotient(k, CH);
        c[j] = (int)(k - (int64_t)i[j] * CH);
        old[j] = kept[i[j]];
      }
#pragma unroll
      for (int j = 0; j < U; ++j) m[j] = move_of(p, b, old[j], i[j]);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        x[j] = *reinterpret_cast<const u32x4*>(p.c.k + m[j].from.page * p.c.k_str[0] + m[j].from.slot * p.c.k_str[1] + h * p.c.k_str[2] + 16 * c[j]);
        y[j] = *reinterpret_cast<const u32x4*>(p.c.v + m[j].from.page * p.c.v_str[0] + m[j].from.slot * p.c.v_str[1] + h * p.c.v_str[2] + 16 * c[j]);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (k0 + 256 * j >= n) continue;
        __builtin_nontemporal_store(x[j], reinterpret_cast<u32x4*>(p.c.k + m[j].at.page * p.c.k_str[0] + m[j].at.slot * p.c.k_str[1] + h * p.c.k_str[2] + 16 * c[j]));
        __builtin_nontemporal_store(y[j], reinterpret_cast<u32x4*>(p.c.v + m[j].at.page * p.c.v_str[0] + m[j].at.slot * p.c.v_str[1] + h * p.c.v_str[2] + 16 * c[j]));
        if constexpr (BITS == 4) {         // 16 bytes are 32 elements: their scale
          p.c.ks[m[j].at.page * p.c.ks_str[0] + m[j].at.slot * p.c.ks_str[1] + h * p.c.ks_str[2] + c[j]] =
              p.c.ks[m[j].from.page * p.c.ks_str[0] + m[j].from.slot * p.c.ks_str[1] + h * p.c.ks_str[2] + c[j]];
          p.c.vs[m[j].at.page * p.c.vs_str[0] + m[j].at.slot * p.c.vs_str[1] + h * p.c.vs_str[2] + c[j]] =
              p.c.vs[m[j].from.page * p.c.vs_str[0] + m[j].from.slot * p.c.vs_str[1] + h * p.c.vs_str[2] + c[j]];
        }
        if (c[j] == 0)
          *reinterpret_cast<float*>(p.w + m[j].at.page * p.w_str[0] + m[j].at.slot * p.w_str[1] + h * p.w_str[2]) =
              *reinterpret_cast<const float*>(p.w + m[j].from.page * p.w_str[0] + m[j].from.slot * p.w_str[1] + h * p.w_str[2]);
      }
    }
  }
}

// Where they lie: kept token i comes from position i or behind it, so a work-group
// that goes through them in order, reads a batch of rows, waits for all of them and
// then writes them, never overwrites what it still has to read.  Work-groups share a
// row by columns: of keys, of values, and the weight with the scales.  Bound by the bytes:
// 256 heads' 2048 tokens of 128 107 to 123 us, 4.4 to 5.0 TB/s (153 with one batch at a
// time; 214 with the rows' loads behind their own branches, one after the other).
constexpr int kMoveDepth = 8;              // rows of a thread on their way
template <int D, int BITS>
__global__ __launch_bounds__(256) void paged_evict_slide_kernel(EvictParams p, int slices) {
  constexpr int CH = D * BITS / 128, CS = CH < 8 ? CH : 8;   // 16-byte pieces of a row, of a slice
  constexpr int RPP = 256 / CS, STEP = RPP * kMoveDepth;
  for (int64_t u = blockIdx.x; u < (int64_t)p.c.B * p.c.Hkv * slices; u += gridDim.x) {
    const int64_t bh = quotient(u, slices);
    const int slice = (int)(u - bh * slices), b = (int)quotient(bh, p.c.Hkv), h = (int)(bh - (int64_t)b * p.c.Hkv);
    const int32_t* kept = p.kept + bh * p.keep;
    if (p.new_lens[b] != p.keep || p.c.lens[b] <= p.keep || kept[0] < 0) continue;     // nothing moves
    if (slice == slices - 1) {             // weights and scales
      for (int i0 = 0; i0 < p.keep; i0 += 256) {
        const int i = i0 + (int)threadIdx.x < p.keep ? i0 + (int)threadIdx.x : p.keep - 1;
        const Move m = move_of(p, b, kept[i], i);
        const char* wf = p.w + m.from.page * p.w_str[0] + m.from.slot * p.w_str[1] + h * p.w_str[2];
        float w = *reinterpret_cast<const float*>(wf);
        uint8_t ks[D / 32], vs[D / 32];
        if constexpr (BITS == 4) {
          const uint8_t* kf = p.c.ks + m.from.page * p.c.ks_str[0] + m.from.slot * p.c.ks_str[1] + h * p.c.ks_str[2];
          const uint8_t* vf = p.c.vs + m.from.page * p.c.vs_str[0] + m.from.slot * p.c.vs_str[1] + h * p.c.vs_str[2];
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            ks[j] = kf[j];
            vs[j] = vf[j];
          }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (i0 + (int)threadIdx.x < p.keep) {
          *reinterpret_cast<float*>(p.w + m.at.page * p.w_str[0] + m.at.slot * p.w_str[1] + h * p.w_str[2]) = w;
          if constexpr (BITS == 4) {
            uint8_t* kt = p.c.ks + m.at.page * p.c.ks_str[0] + m.at.slot * p.c.ks_str[1] + h * p.c.ks_str[2];
            uint8_t* vt = p.c.vs + m.at.page * p.c.vs_str[0] + m.at.slot * p.c.vs_str[1] + h * p.c.vs_str[2];
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
              kt[j] = ks[j];
              vt[j] = vs[j];
            }
          }
        }
      }
      continue;
    }
    constexpr int SL = (CH + CS - 1) / CS;
    const bool is_v = slice >= SL;
    const int c0 = (is_v ? slice - SL : slice) * CS + threadIdx.x % CS, r0 = threadIdx.x / CS;
    const bool on = r0 < RPP && c0 < CH;   // some threads have no piece: they read the row's last one
    const int c = c0 < CH ? c0 : CH - 1;
    char* base = (is_v ? p.c.v + h * p.c.v_str[2] : p.c.k + h * p.c.k_str[2]) + 16 * c;
    const int64_t s0 = is_v ? p.c.v_str[0] : p.c.k_str[0], s1 = is_v ? p.c.v_str[1] : p.c.k_str[1];
    // the next batch's rows are on their way while this one's are written: they lie
    // behind all that is written
    struct Batch {
      u32x4 x[kMoveDepth];
      char* to[kMoveDepth];
    };
    auto place = [&](int i0, int j) __attribute__((always_inline)) {
      const int i = i0 + j * RPP + r0;
      return i < p.keep ? i : p.keep - 1;
    };
    auto load = [&](int i0, Batch& t) __attribute__((always_inline)) {
      int old[kMoveDepth];                 // past the end: the last row, which is not written
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j) old[j] = kept[place(i0, j)];
      Move m[kMoveDepth];
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j) m[j] = move_of(p, b, old[j], place(i0, j));
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j) {
        t.to[j] = base + m[j].at.page * s0 + m[j].at.slot * s1;
        t.x[j] = *reinterpret_cast<const u32x4*>(base + m[j].from.page * s0 + m[j].from.slot * s1);
      }
    };
    auto store = [&](int i0, Batch& t) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j) asm volatile("" : "+v"(t.x[j]));   // all rows of the batch are here
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j)
        if (on && i0 + j * RPP + r0 < p.keep) *reinterpret_cast<u32x4*>(t.to[j]) = t.x[j];
    };
    Batch a, z;
    load(0, a);
    for (int i0 = 0; i0 < p.keep; i0 += 2 * STEP) {
      load(i0 + STEP, z);
      store(i0, a);
      if (i0 + STEP >= p.keep) break;
      load(i0 + 2 * STEP, a);
      store(i0 + STEP, z);
    }
  }
}

constexpr int64_t kMostGroups = 1 << 20;

// An array of a call.
struct Ints {
  const int32_t* at;
  int64_t n;
  bool meets(const Ints& o) const { return at && o.at && n > 0 && o.n > 0 && at < o.at + o.n && o.at < at + n; }
};

template <int D, typename E, int BITS> struct Evict {
  static int go(const EvictParams& p, hipStream_t stream) {
    const int64_t bh = (int64_t)p.c.B * p.c.Hkv;
    auto grid = [](int64_t n) { return dim3((unsigned)(n < kMostGroups ? n : kMostGroups)); };
    // the longest sequence that the table has room for
    const int64_t cap = (int64_t)p.c.max_pages * p.c.page_size;
    if (cap <= 4 * 1024) hipLaunchKernelGGL((paged_evict_select_kernel<4>), grid(bh), dim3(1024), 0, stream, p);
    else if (cap <= 16 * 1024) hipLaunchKernelGGL((paged_evict_select_kernel<16>), grid(bh), dim3(1024), 0, stream, p);
    else if (cap <= kEvictHeld * 1024) hipLaunchKernelGGL((paged_evict_select_kernel<kEvictHeld>), grid(bh), dim3(1024), 0, stream, p);
    else hipLaunchKernelGGL((paged_evict_select_kernel<0>), grid(bh), dim3(1024), 0, stream, p);
    int rc = launch_status("lvsa_paged_evict");
    if (rc) return rc;
    constexpr int CH = D * BITS / 128;
    if (p.to) {
      const int64_t want = ceil_div((int64_t)p.keep * CH, 256 * 4);
      const int per = (int)(want < 64 ? want : 64);
      hipLaunchKernelGGL((paged_evict_move_kernel<D, BITS>), grid(bh * per), dim3(256), 0, stream, p, per);
    } else {
      const int slices = 2 * (CH < 8 ? 1 : (CH + 7) / 8) + 1;
      hipLaunchKernelGGL((paged_evict_slide_kernel<D, BITS>), grid(bh * slices), dim3(256), 0, stream, p, slices);
    }
    return launch_status("lvsa_paged_evict");
  }
};

}  // namespace
}  // namespace lvsa

extern "C" {

int lvsa_paged_evict(const lvsa_paged_evict_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_evict";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  EvictParams p{};
  const int rc = paged_view(what, &a->cache, &a->batch, false, &p.c);
  if (rc) return rc;
  LVSA_REQUIRE(a->keep < INT32_MAX - 4096, LVSA_ERR_UNSUPPORTED, "%s: %d tokens to keep: below 2^31 - 4096", what, a->keep);
  LVSA_REQUIRE(a->keep >= 1 && a->first >= 0 && a->last >= 0 && (int64_t)a->first + a->last <= a->keep, LVSA_ERR_INVALID_ARG,
               "%s: %d tokens, the first %d and last %d among them", what, a->keep, a->first, a->last);
  LVSA_REQUIRE(a->weights && ((uintptr_t)a->weights & 3) == 0, LVSA_ERR_INVALID_ARG, "%s: weights must be non-null, fp32", what);
  LVSA_REQUIRE(!a->new_table || (a->new_pages >= 0 && a->new_stride >= a->new_pages), LVSA_ERR_INVALID_ARG,
               "%s: new table of %d pages, rows %lld apart", what, a->new_pages, (long long)a->new_stride);
  const int64_t cap = (int64_t)a->batch.max_pages * a->cache.page_size;
  LVSA_REQUIRE(!a->new_table || (int64_t)a->new_pages * a->cache.page_size >= (a->keep < cap ? a->keep : cap), LVSA_ERR_INVALID_ARG,
               "%s: %d new pages of %d slots do not hold %d tokens", what, a->new_pages, a->cache.page_size, a->keep);
  if (a->batch.B == 0) return LVSA_OK;
  LVSA_REQUIRE(a->kept && a->new_lens, LVSA_ERR_INVALID_ARG, "%s: null kept or new_lens", what);
  // Other heads' work-groups, and the moves, read what the first one would have written over.
  const int64_t B = a->batch.B;
  const Ints lens = {a->batch.kv_lens, B}, table = {a->batch.page_table, (B - 1) * a->batch.table_stride + a->batch.max_pages};
  const Ints to = {a->new_table, (B - 1) * a->new_stride + a->new_pages};
  const Ints kept = {a->kept, B * a->cache.Hkv * a->keep}, out = {a->new_lens, B};
  LVSA_REQUIRE(!out.meets(lens) && !out.meets(table) && !out.meets(to) && !out.meets(kept) && !kept.meets(lens) && !kept.meets(table) &&
                   !kept.meets(to), LVSA_ERR_INVALID_ARG, "%s: kept and new_lens must not share memory with each other, kv_lens and the tables", what);
  p.c.cu = nullptr;
  p.w = (char*)a->weights;
  for (int i = 0; i < 3; ++i) p.w_str[i] = 4 * a->w_str[i];
  p.to = a->new_table;
  p.to_str = a->new_stride;
  p.kept = a->kept;
  p.new_lens = a->new_lens;
  p.keep = a->keep;
  p.first = a->first;
  p.last = a->last;
  return by_type<Evict>(a->cache.D, LVSA_BF16, a->cache.bits, p, stream);
}

}  // extern "C"
