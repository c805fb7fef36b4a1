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
  int32_t to_pages, keep, first, last, D;
};

// A weight as a number that sorts like it: NaN below -inf, 0 and -0 alike.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, w + 0.f);
  return b >> 31 ? ~b : b | 1u << 31;
}

// Sums over the work-group's 1024 threads before this one, and the total.
__device__ __forceinline__ int group_scan(int x, int* lds, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(incl, d);
    if (lane >= d) incl += y;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wave ? lds[w] : 0;
    all += lds[w];
  }
  *total = all;
  return before + incl - x;
}

// One work-group per sequence and head: finds the keep-th highest weight, 11 bits of
// it at a time by counting how often each value of them occurs, and lists the tokens
// from it on.  The counts are whole numbers, so the order of the atomics in LDS does
// not matter.
__global__ __launch_bounds__(1024) void paged_evict_select_kernel(EvictParams p) {
  __shared__ int hist[2048];
  __shared__ int lds[16];
  __shared__ int bad_s, bin_s, above_s;
  const int Hkv = p.c.Hkv, tid = threadIdx.x;
  for (int64_t u = blockIdx.x; u < (int64_t)p.c.B * Hkv; u += gridDim.x) {
    const int b = (int)quotient(u, Hkv), h = (int)(u - (int64_t)b * Hkv);
    const PagedSeq sq = paged_seq(p.c, 0, 0, p.c.lens[b]);
    const int L = sq.L, left = L < p.keep ? L : p.keep;
    const int32_t* table = p.c.table + b * p.c.table_str;
    const int32_t* to = p.to ? p.to + b * p.to_str : nullptr;
    int32_t* kept = p.kept + u * p.keep;
    __syncthreads();
    if (tid == 0) bad_s = sq.flags;
    __syncthreads();
    const int pages = L > 0 ? page_of(p.c, L - 1) + 1 : 0, news = left > 0 ? page_of(p.c, left - 1) + 1 : 0;
    for (int e = tid; e < pages; e += 1024) {
      const int page = table[e];
      bool bad = (uint32_t)page >= (uint32_t)p.c.n_pages;
      for (int i = 0; to && i < news; ++i) bad |= to[i] == page;
      if (bad) atomicOr(&bad_s, LVSA_PAGED_BAD_PAGE);
    }
    for (int i = tid; to && i < news; i += 1024)
      if ((uint32_t)to[i] >= (uint32_t)p.c.n_pages) atomicOr(&bad_s, LVSA_PAGED_BAD_PAGE);
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
    auto rank = [&](int pos) __attribute__((always_inline)) {
      if (pos < p.first || pos >= L - p.last) return ~0u;
      const PagedRow at = paged_row(p.c, pos, table[page_of(p.c, pos)]);
      return rank_of(*reinterpret_cast<const float*>(p.w + at.page * p.w_str[0] + at.slot * p.w_str[1] + h * p.w_str[2]));
    };
    uint32_t bound = 0;                    // the bits found so far
    int want = p.keep;                     // of the ranks with these bits
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {
      const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bits = step == 2 ? 10 : 11;
      hist[tid] = hist[tid + 1024] = 0;
      __syncthreads();
      for (int pos = tid; pos < L; pos += 1024) {
        const uint32_t r = rank(pos);
        if (step == 0 || r >> (shift + bits) == bound) atomicAdd(&hist[r >> shift & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      // bins from the highest down, two a thread: the one that reaches `want`
      const int hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
      int all;
      const int before = group_scan(hi + lo, lds, &all);
      if (before < want && before + hi >= want) {
        bin_s = 2047 - 2 * tid;
        above_s = before;
      } else if (before + hi < want && before + hi + lo >= want) {
        bin_s = 2046 - 2 * tid;
        above_s = before + hi;
      }
      __syncthreads();
      bound = bound << bits | (uint32_t)bin_s;
      want -= above_s;
      __syncthreads();
    }
    // all above the bound, and the first `want` equal to it
    int put = 0, seen = 0;
    for (int p0 = 0; p0 < L; p0 += 1024) {
      const int pos = p0 + tid;
      const uint32_t r = pos < L ? rank(pos) : 0;
      const bool gt = pos < L && r > bound, eq = pos < L && r == bound;
      int all;
      const int both = group_scan((gt ? 1 : 0) | (eq ? 1 << 16 : 0), lds, &all);
      const int room = want - seen, e = both >> 16;
      const int at = put + (both & 0xffff) + (e < room ? e : room);
      if ((gt || (eq && e < room)) && at < p.keep) kept[at] = pos;
      const int es = all >> 16;
      put += (all & 0xffff) + (es < room ? es : room);
      seen += es < room ? es : room;
    }
    // weights that another stream changes meanwhile: still positions
    for (int i = put + tid; i < p.keep; i += 1024) kept[i] = i;
  }
}

// Old place of kept token i of a sequence, and its new one.
struct Move {
  PagedRow from, at;
};
__device__ __forceinline__ Move move_of(const EvictParams& p, int b, const int32_t* kept, int i) {
  const int32_t* table = p.c.table + b * p.c.table_str;
  const int32_t* to = p.to ? p.to + b * p.to_str : table;
  const int old = kept[i];
  return Move{paged_row(p.c, old, table[page_of(p.c, old)]), paged_row(p.c, i, to[page_of(p.c, i)])};
}

// To pages of their own: nothing is read that is written, all rows at once.  A thread
// has a 16-byte piece of a key and of its value; the first ones of a row bring its
// scales and weight.  Bound by the bytes.
template <int D, int BITS>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(EvictParams p, int per) {
  constexpr int CH = D * BITS / 128;       // 16-byte pieces of a row
  for (int64_t u = blockIdx.x; u < (int64_t)p.c.B * p.c.Hkv * per; u += gridDim.x) {
    const int64_t bh = quotient(u, per);
    const int part = (int)(u - bh * per), b = (int)quotient(bh, p.c.Hkv), h = (int)(bh - (int64_t)b * p.c.Hkv);
    const int left = p.new_lens[b];
    const int32_t* kept = p.kept + bh * p.keep;
    for (int64_t k = (int64_t)part * 256 + threadIdx.x; k < (int64_t)left * CH; k += (int64_t)per * 256) {
      const int i = (int)(k / CH), c = (int)(k % CH);
      const Move m = move_of(p, b, kept, i);
      const int64_t kf = m.from.page * p.c.k_str[0] + m.from.slot * p.c.k_str[1], kt = m.at.page * p.c.k_str[0] + m.at.slot * p.c.k_str[1];
      const int64_t vf = m.from.page * p.c.v_str[0] + m.from.slot * p.c.v_str[1], vt = m.at.page * p.c.v_str[0] + m.at.slot * p.c.v_str[1];
      const u32x4 x = *reinterpret_cast<const u32x4*>(p.c.k + kf + h * p.c.k_str[2] + 16 * c);
      const u32x4 y = *reinterpret_cast<const u32x4*>(p.c.v + vf + h * p.c.v_str[2] + 16 * c);
      *reinterpret_cast<u32x4*>(p.c.k + kt + h * p.c.k_str[2] + 16 * c) = x;
      *reinterpret_cast<u32x4*>(p.c.v + vt + h * p.c.v_str[2] + 16 * c) = y;
      if constexpr (BITS == 4) {           // 16 bytes are 32 elements: their scale
        const int64_t ksf = m.from.page * p.c.ks_str[0] + m.from.slot * p.c.ks_str[1], kst = m.at.page * p.c.ks_str[0] + m.at.slot * p.c.ks_str[1];
        const int64_t vsf = m.from.page * p.c.vs_str[0] + m.from.slot * p.c.vs_str[1], vst = m.at.page * p.c.vs_str[0] + m.at.slot * p.c.vs_str[1];
        p.c.ks[kst + h * p.c.ks_str[2] + c] = p.c.ks[ksf + h * p.c.ks_str[2] + c];
        p.c.vs[vst + h * p.c.vs_str[2] + c] = p.c.vs[vsf + h * p.c.vs_str[2] + c];
      }
      if (c == 0) {
        const int64_t wf = m.from.page * p.w_str[0] + m.from.slot * p.w_str[1], wt = m.at.page * p.w_str[0] + m.at.slot * p.w_str[1];
        *reinterpret_cast<float*>(p.w + wt + h * p.w_str[2]) = *reinterpret_cast<const float*>(p.w + wf + h * p.w_str[2]);
      }
    }
  }
}

// Where they lie: kept token i comes from position i or behind it, so a work-group
// that goes through them in order, reads a batch of rows, waits for all of them and
// then writes them, never overwrites what it still has to read.  Work-groups share a
// row by columns: of keys, of values, and the weight with the scales.
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
        const Move m = move_of(p, b, kept, i);
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
    const int c = (is_v ? slice - SL : slice) * CS + threadIdx.x % CS, r0 = threadIdx.x / CS;
    const bool on = r0 < RPP && c < CH;
    char* base = (is_v ? p.c.v + h * p.c.v_str[2] : p.c.k + h * p.c.k_str[2]) + 16 * c;
    const int64_t s0 = is_v ? p.c.v_str[0] : p.c.k_str[0], s1 = is_v ? p.c.v_str[1] : p.c.k_str[1];
    for (int i0 = 0; i0 < p.keep; i0 += STEP) {
      u32x4 x[kMoveDepth];
      char* to[kMoveDepth];
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j) {
        const int i = i0 + j * RPP + r0;
        to[j] = nullptr;
        if (on && i < p.keep) {
          const Move m = move_of(p, b, kept, i);
          to[j] = base + m.at.page * s0 + m.at.slot * s1;
          x[j] = *reinterpret_cast<const u32x4*>(base + m.from.page * s0 + m.from.slot * s1);
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // all rows of the batch are here
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMoveDepth; ++j)
        if (to[j]) *reinterpret_cast<u32x4*>(to[j]) = x[j];
    }
  }
}

constexpr int64_t kMostGroups = 1 << 20;

template <int D, typename E, int BITS> struct Evict {
  static int go(const EvictParams& p, hipStream_t stream) {
    const int64_t bh = (int64_t)p.c.B * p.c.Hkv;
    auto grid = [](int64_t n) { return dim3((unsigned)(n < kMostGroups ? n : kMostGroups)); };
    hipLaunchKernelGGL(paged_evict_select_kernel, grid(bh), dim3(1024), 0, stream, p);
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
  p.c.cu = nullptr;
  p.w = (char*)a->weights;
  for (int i = 0; i < 3; ++i) p.w_str[i] = 4 * a->w_str[i];
  p.to = a->new_table;
  p.to_str = a->new_stride;
  p.to_pages = a->new_pages;
  p.kept = a->kept;
  p.new_lens = a->new_lens;
  p.keep = a->keep;
  p.first = a->first;
  p.last = a->last;
  return by_type<Evict>(a->cache.D, LVSA_BF16, a->cache.bits, p, stream);
}

}  // extern "C"
