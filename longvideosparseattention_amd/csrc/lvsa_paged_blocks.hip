// Blocks of the paged key/value cache on gfx950: their mean keys, the selection of
// blocks by them, and the C ABI of what works on parts of a cache.  The attention
// over selected blocks is in lvsa_paged_list.h, the accumulated weights in
// lvsa_paged_weights.h, eviction in lvsa_paged_evict.hip.
#include "lvsa_paged_host.h"
#include "lvsa_paged_list.h"
#include "lvsa_paged_rows.h"

using namespace lvsa;

namespace lvsa {
namespace {

struct MeansParams {
  PagedView c;
  char* means;
  int64_t m_str[3];                      // bytes
  Divisor block, parts;
};

// ────────────────────────────── mean keys ──────────────────────────────────

// One work-group per block and head: a thread sums 8 elements of every RPP-th key,
// the sums are joined in LDS.  fp32 within a thread (at most block / RPP keys), 64
// bits across them, one rounding at the end.  Latency where an append touched a few
// blocks (32 sequences, one token: 4.3 us), else the keys' bytes: 4680 tokens of 12
// heads of 128 7.3 us, 2.0 TB/s, of which 3 are the launch and the batch.  (Sixteen
// work-groups a unit instead of four, most without a block: 5.5 us for the former.)
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256) void paged_means_kernel(MeansParams p) {
  constexpr int CH = D / 8, RPP = 256 / CH;
  __shared__ float sum_s[RPP][D];
  const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
  // the blocks that hold new tokens, or all
  auto first_block = [&](const PagedSeq& s) __attribute__((always_inline)) { return p.c.cu && s.first > 0 ? s.first / p.block : 0; };
  auto count = [&](const PagedSeq& s) __attribute__((always_inline)) {
    if (s.L == 0 || (p.c.cu && s.n == 0)) return (int64_t)0;
    return ((int64_t)((s.L - 1) / p.block) + 1 - first_block(s)) * p.c.Hkv;
  };
  walk_units<false>(p.c, count, [&](int seq, const PagedSeq& sq, int64_t u, int64_t) __attribute__((always_inline)) {
    const int i = (int)quotient(u, p.c.Hkv), h = (int)(u - (int64_t)i * p.c.Hkv);
    const int b = first_block(sq) + i, entry = b / p.parts, part = b - entry * p.parts.by;
    const int page = p.c.table[seq * p.c.table_str + entry];
    if ((uint32_t)page >= (uint32_t)p.c.n_pages) {
      if (threadIdx.x == 0) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
      return;
    }
    const int left = sq.L - b * p.block.by, keys = left < p.block.by ? left : p.block.by;
    const int64_t slot0 = (int64_t)part * p.block.by;
    const char* kb = p.c.k + page * p.c.k_str[0] + slot0 * p.c.k_str[1] + h * p.c.k_str[2];
    const uint8_t* sb = BITS == 4 ? p.c.ks + page * p.c.ks_str[0] + slot0 * p.c.ks_str[1] + h * p.c.ks_str[2] : nullptr;
    float acc[8] = {};
    if (r0 < RPP)
      for (int r = r0; r < keys; r += RPP) {
        float x[8];
        if constexpr (BITS == 16) {
          Half<E>::unpack(*reinterpret_cast<const u32x4*>(kb + r * p.c.k_str[1] + 16 * c), x);
        } else {
          const uint32_t codes = *reinterpret_cast<const uint32_t*>(kb + r * p.c.k_str[1] + 4 * c);
          Half<__bf16>::unpack(unpack_e2m1<__bf16>(codes, sb[r * p.c.ks_str[1] + (c >> 2)]), x);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += x[j];
      }
    if (r0 < RPP)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum_s[r0][8 * c + j] = acc[j];
    __syncthreads();
    if (threadIdx.x < D) {
      double s = 0.0;
      const int n = keys < RPP ? keys : RPP;
      for (int r = 0; r < n; ++r) s += (double)sum_s[r][threadIdx.x];
      float* m = reinterpret_cast<float*>(p.means + page * p.m_str[0] + part * p.m_str[1] + h * p.m_str[2]);
      m[threadIdx.x] = (float)(s / (double)keys);
    }
    __syncthreads();
  });
}

// ────────────────────────────── selection ──────────────────────────────────

struct SelectParams {
  PagedView c;
  ListView v;
  const char* q;
  const char* means;
  int32_t* blocks;
  int64_t q_str[2], m_str[3];            // bytes
  int32_t group, first, last, causal;
};

constexpr int kSelectKeys = 4096;        // blocks ranked at a time
constexpr int kWaveKeys = 1024;          // by one wave
constexpr int kGroup = 16;               // lists of a work-group that scores on the matrix cores
constexpr int kGroupWaves = 4;
constexpr uint64_t kAlways = ~0ull;      // the rank of what is always selected

// A score as a number that sorts like it: NaN below -inf, 0 and -0 alike.
__device__ __forceinline__ uint64_t rank_of(double s) {
  if (s != s) return 0;
  const uint64_t b = __builtin_bit_cast(uint64_t, s + 0.0);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double score_of(uint64_t r) {
  return __builtin_bit_cast(double, r >> 63 ? r & ~(1ull << 63) : ~r);
}

// A bound between lo and hi (lo < bound <= hi): half way between the scores, which
// finds the border of scores that are spread in a dozen steps (half way between the
// ranks, the exponents' halves, takes 20), or between the ranks where scores do not
// say (infinities, NaN, neighbours) or have not led there in 24 steps.
__device__ __forceinline__ uint64_t bound_between(uint64_t lo, uint64_t hi, int step) {
  const uint64_t mid = step < 24 ? rank_of(0.5 * score_of(lo) + 0.5 * score_of(hi)) : 0;
  return mid > lo && mid <= hi ? mid : lo + (hi - lo) / 2 + 1;
}

// The same for fp32: half way between the numbers for 16 steps, then, where these close
// in on 0 or stand far apart, half way between their bit patterns.
__device__ __forceinline__ float float_between(float lo, float hi, int step) {
  if (step < 16) return 0.5f * lo + 0.5f * hi;
  auto flip = [](int b) { return b < 0 ? b ^ 0x7fffffff : b; };
  const int64_t a = flip(__builtin_bit_cast(int, lo)), b = flip(__builtin_bit_cast(int, hi));
  return __builtin_bit_cast(float, flip((int)((a + b + 1) >> 1)));
}

struct Span {
  uint64_t lo, hi;
};
__device__ __forceinline__ Span wave_span(Span s) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t a = __shfl_xor((unsigned long long)s.lo, d), b = __shfl_xor((unsigned long long)s.hi, d);
    s.lo = a < s.lo ? a : s.lo;
    s.hi = b > s.hi ? b : s.hi;
  }
  return s;
}

// One wave writes the `top` highest of n <= 64 K ranks (top < n), equal ones from the
// front, to `out` in their order.  It holds the ranks, and the scores rounded to fp32,
// which keeps their order, and halves the range between the lowest and the highest of
// those that are not always selected until a bound cuts off exactly `top`: an fp32
// comparison and a count per 64 of them, a dozen steps.  Where that does not come out
// (the border runs between scores that fp32 does not tell apart, infinities, NaN), the
// ranks between the two are halved: no step where they are all alike.
template <int K>
__device__ __forceinline__ void wave_select(const uint64_t* ranks, int n, int top, int lane, int32_t* out) {
  uint32_t up[K], low[K];
  float x[K];
  float lof = __builtin_inff(), hif = -__builtin_inff();
  bool nan = false;                        // or -inf
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool in = 64 * k + lane < n;
    const uint64_t r = ranks[in ? 64 * k + lane : n - 1];
    x[k] = r == kAlways ? __builtin_inff() : r == 0 ? -__builtin_inff() : (float)score_of(r);
    nan |= x[k] == -__builtin_inff();
    lof = x[k] > -__builtin_inff() ? __builtin_fminf(lof, x[k]) : lof;
    hif = r != kAlways ? __builtin_fmaxf(hif, x[k]) : hif;
    if (!in) x[k] = -__builtin_inff();     // below what any bound keeps
    up[k] = in ? (uint32_t)(r >> 32) : 0;
    low[k] = in ? (uint32_t)r : 0;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    lof = __builtin_fminf(lof, __shfl_xor(lof, d));
    hif = __builtin_fmaxf(hif, __shfl_xor(hif, d));
  }
  int count = n;
  uint64_t bound = 0;                      // at least `top` ranks from it on
  {
    if (__builtin_amdgcn_ballot_w64(nan)) {      // are the others enough?
      int fine = 0;
#pragma unroll
      for (int k = 0; k < K; ++k) fine += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[k] >= lof));
      if (fine < top) lof = -__builtin_inff();
    }
    float cut = 0.f;
    for (int step = 0; step < 48; ++step) {      // 16 and 32 close any range
      const float mid = float_between(lof, hif, step);
      if (!(mid > lof && mid <= hif)) break;
      int c = 0;
#pragma unroll
      for (int k = 0; k < K; ++k) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[k] >= mid));
      if (c >= top) lof = mid;
      else hif = mid;
      if (c == top) {
        count = c;
        cut = mid;
        break;
      }
    }
    if (count == top) {
#pragma unroll
      for (int k = 0; k < K; ++k) {        // those below the cut drop out
        if (!(x[k] >= cut)) up[k] = low[k] = 0;
      }
      bound = 1;
    }
  }
  if (count != top) {                      // the border lies among the ranks of [lof, hif]
    Span s = {kAlways, 0};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint64_t r = (uint64_t)up[k] << 32 | low[k];
      const bool in = 64 * k + lane < n && r != kAlways;
      if (in && x[k] >= lof && r < s.lo) s.lo = r;
      if (in && x[k] <= hif && r > s.hi) s.hi = r;
    }
    s = wave_span(s);
    bound = s.lo;
    uint64_t high = s.hi;
    while (bound < high && count != top) {
      const uint64_t mid = bound + (high - bound) / 2 + 1;
      int c = 0;
#pragma unroll
      for (int k = 0; k < K; ++k) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(((uint64_t)up[k] << 32 | low[k]) >= mid));
      if (c >= top) {
        bound = mid;
        count = c;
      } else {
        high = mid - 1;
      }
    }
  }
  // all above the bound, and of those equal to it the first
  int equal = n;
  if (count != top) {
    int above = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(((uint64_t)up[k] << 32 | low[k]) > bound));
    equal = top - above;
  }
  const uint64_t before = (1ull << lane) - 1;
  int put = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool in = 64 * k + lane < n;
    const uint64_t r = (uint64_t)up[k] << 32 | low[k];
    uint64_t take = __builtin_amdgcn_ballot_w64(in && r >= bound);
    if (count != top) {
      const uint64_t eq = __builtin_amdgcn_ballot_w64(in && r == bound);
      const int e = __builtin_popcountll(eq & before);
      take = __builtin_amdgcn_ballot_w64((take >> lane & 1) && (!(eq >> lane & 1) || e < equal));
      equal -= __builtin_popcountll(eq & take);
    }
    if (take >> lane & 1) out[put + __builtin_popcountll(take & before)] = 64 * k + lane;
    put += __builtin_popcountll(take);
  }
}
__device__ __forceinline__ void wave_select(const uint64_t* ranks, int n, int top, int lane, int32_t* out) {
  if (n <= 256) wave_select<4>(ranks, n, top, lane, out);
  else if (n <= 384) wave_select<6>(ranks, n, top, lane, out);
  else if (n <= 512) wave_select<8>(ranks, n, top, lane, out);
  else wave_select<kWaveKeys / 64>(ranks, n, top, lane, out);
}

// What a list may name, and always does.
struct ListRange {
  int n, near0, near1;                     // blocks [0, n), of them [near0, near1] and below `first` always
  __device__ __forceinline__ uint64_t rank(const SelectParams& p, int b, bool ok, double s) const {
    return b < p.first || (b >= near0 && b <= near1) ? kAlways : ok ? rank_of(s) : 0;
  }
};
__device__ __forceinline__ ListRange list_range(const SelectParams& p, const PagedSeq& sq, int i0, int i1) {
  ListRange r = {0, 0, -1};
  const int p0 = sq.first + i0 > 0 ? sq.first + i0 : 0, end = sq.first + i1;    // the tile's positions [p0, end)
  const int lim = !p.causal ? sq.L : end < 0 ? 0 : end;
  r.n = lim > 0 ? (lim - 1) / p.v.block + 1 : 0;
  if (p.last > 0 && end > 0) {
    r.near0 = p0 / p.v.block - (p.last - 1);
    r.near1 = (end - 1) / p.v.block;
  }
  return r;
}
// Reports what is wrong with a batch; whether its row ranges are, and then every list
// is empty.
__device__ __forceinline__ bool refuse_batch(const SelectParams& p) {
  const int lane = threadIdx.x & 63;
  int flags = 0;
  for (int s = lane; s < p.c.B; s += 64) flags |= paged_seq(p.c, s).flags;
  if (blockIdx.x == 0 && threadIdx.x < 64 && flags) paged_flag(p.c, flags);
  if (!__builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) return false;
  const int64_t n = (int64_t)p.v.lists * p.c.Hkv * p.v.top;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)blockDim.x * gridDim.x) p.blocks[i] = -1;
  return true;
}

// LDS of a selection: ranks and numbers of candidate blocks, in ascending order.
struct Ranks {
  uint64_t key[kSelectKeys];
  int id[kSelectKeys];
  int sum[2][4];
  uint64_t bound[2][4];
};

// Leaves the `top` highest of n ranks in their order, like wave_select, with the whole
// work-group of 256.
__device__ __forceinline__ void keep_highest(Ranks& r, int n, int top) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  Span s = {kAlways, 0};
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t k = r.key[i];
    s.lo = k < s.lo ? k : s.lo;
    s.hi = k != kAlways && k > s.hi ? k : s.hi;
  }
  s = wave_span(s);
  if (lane == 0) {
    r.bound[0][wave] = s.lo;
    r.bound[1][wave] = s.hi;
  }
  __syncthreads();
  uint64_t lo = s.lo, hi = s.hi;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    lo = r.bound[0][w] < lo ? r.bound[0][w] : lo;
    hi = r.bound[1][w] > hi ? r.bound[1][w] : hi;
  }
  int parity = 0;
  auto total = [&](auto test) __attribute__((always_inline)) {
    int count = 0;
    for (int i = (int)threadIdx.x - lane; i < n; i += 256)
      count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i + lane < n && test(r.key[i + lane < n ? i + lane : 0])));
    if (lane == 0) r.sum[parity][wave] = count;
    __syncthreads();
    count = r.sum[parity][0] + r.sum[parity][1] + r.sum[parity][2] + r.sum[parity][3];
    parity ^= 1;
    return count;
  };
  // at least `top` ranks are >= lo, and fewer are > hi
  for (int step = 0; lo < hi; ++step) {
    const uint64_t mid = bound_between(lo, hi, step);
    const int count = total([&](uint64_t k) __attribute__((always_inline)) { return k >= mid; });
    if (count >= top) lo = mid;
    else hi = mid - 1;
    if (count == top) break;
  }
  int equal = top - total([&](uint64_t k) __attribute__((always_inline)) { return k > lo; });
  __syncthreads();                       // r.sum has been read
  int put = 0;
  const uint64_t before = (1ull << lane) - 1;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + (int)threadIdx.x;
    const uint64_t k = i < n ? r.key[i] : 0;
    const int id = i < n ? r.id[i] : 0;
    const uint64_t gt = __builtin_amdgcn_ballot_w64(i < n && k > lo), eq = __builtin_amdgcn_ballot_w64(i < n && k == lo);
    if (lane == 0) {
      r.sum[0][wave] = __builtin_popcountll(gt);
      r.sum[1][wave] = __builtin_popcountll(eq);
    }
    __syncthreads();                     // the ranks of these 256 have been read, too
    int g = 0, e = 0, gs = 0, es = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      g += w < wave ? r.sum[0][w] : 0;
      e += w < wave ? r.sum[1][w] : 0;
      gs += r.sum[0][w];
      es += r.sum[1][w];
    }
    g += __builtin_popcountll(gt & before);
    e += __builtin_popcountll(eq & before);
    if ((gt >> lane & 1) || ((eq >> lane & 1) && e < equal)) {
      const int at = put + g + (e < equal ? e : equal);
      r.key[at] = k;
      r.id[at] = id;
    }
    const int taken = es < equal ? es : equal;
    put += gs + taken;
    equal -= taken;
    __syncthreads();
  }
}

// One work-group per list and key head: sums the tile's queries, scores every block
// with it, eight lanes a block, and keeps the highest.  64-bit sums, so that which of
// two blocks is the higher does not depend on the order they were summed in (short of
// differences of 1e-15): a list is the same on every device and beside every batch.
// Bound by trips to memory one after the other (batch, queries, page table, means) and
// one wave's search: 45 lists of 8 heads over up to 250 blocks 12 to 14 us for 27 MB.
// (The first means loaded before the queries: 15.5 us; eight of them at once: 22.)
template <int D, typename E>
__global__ __launch_bounds__(256) void paged_select_kernel(SelectParams p) {
  constexpr int CH = D / 8, RPP = 256 / CH, U = D <= 128 ? 4 : 2;    // U: blocks of eight lanes on their way
  __shared__ Ranks ranks;
  __shared__ double q_s[D];
  double* part_s = reinterpret_cast<double*>(ranks.key);     // [RPP][D]: before any rank is there
  static_assert(RPP * D <= kSelectKeys, "sums of the queries");
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  if (refuse_batch(p)) return;
  const int64_t total = (int64_t)p.v.lists * p.c.Hkv;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t li = quotient(w, p.c.Hkv);
    const int h = (int)(w - li * p.c.Hkv);
    int32_t* out = p.blocks + w * p.v.top;
    PagedSeq sq;
    int i0, seq = paged_seq_of_list(p.c, p.v, li, lane, &sq, &i0);
    if (seq >= 0 && sq.flags) seq = -1;
    ListRange range = {0, 0, -1};
    int i1 = 0;
    if (seq >= 0) {
      i1 = tile_end(p.v, sq, i0);
      range = list_range(p, sq, i0, i1);
    }
    const int n = range.n, top = p.v.top;
    if (n <= top) {                        // all of them
      for (int i = threadIdx.x; i < top; i += 256) out[i] = i < n ? i : -1;
      continue;
    }
    __syncthreads();                       // the ranks of the list before have been read
    {
      const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
      double acc[8] = {};
      const int rows = (i1 - i0) * p.group, used = rows < RPP ? rows : RPP;
      if (r0 < used) {
        for (int r = r0; r < rows; r += RPP) {
          const int i = (uint32_t)r / (uint32_t)p.group;
          const char* src = p.q + (int64_t)(sq.t0 + i0 + i) * p.q_str[0] + (h * p.group + r - i * p.group) * p.q_str[1];
          float x[8];
          Half<E>::unpack(*reinterpret_cast<const u32x4*>(src + 16 * c), x);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] += (double)x[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) part_s[r0 * D + 8 * c + j] = acc[j];
      }
      __syncthreads();
      if (threadIdx.x < D) {
        double s = 0.0;
        for (int r = 0; r < used; ++r) s += part_s[r * D + threadIdx.x];
        q_s[threadIdx.x] = s;
      }
      __syncthreads();
    }
    // lane l of eight: elements 4 l + 32 i .. + 3
    const int l8 = lane & 7;
    double q[D / 8];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[4 * i + j] = q_s[32 * i + 4 * l8 + j];
    const int32_t* table = p.c.table + seq * p.c.table_str;
    int kept = 0;
    bool bad = false;
    for (int b0 = 0; b0 < n;) {
      const int room = kSelectKeys - kept, here = n - b0 < room ? n - b0 : room;
      for (int i0 = threadIdx.x >> 3; i0 < here; i0 += 32 * U) {
        floatx4 x[U][D / 32];
        bool ok[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {      // past the end: the last one again
          const int i = i0 + 32 * k < here ? i0 + 32 * k : here - 1, e = (b0 + i) / p.v.parts;
          const int page = table[e];
          ok[k] = (uint32_t)page < (uint32_t)p.c.n_pages;
          const char* m = p.means + (int64_t)(ok[k] ? page : 0) * p.m_str[0] + (int64_t)(b0 + i - e * p.v.parts.by) * p.m_str[1] + h * p.m_str[2];
#pragma unroll
          for (int j = 0; j < D / 32; ++j) x[k][j] = *reinterpret_cast<const floatx4*>(m + 128 * j + 16 * l8);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int i = i0 + 32 * k;
          double s = 0.0;
#pragma unroll
          for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int d = 0; d < 4; ++d) s = __builtin_fma((double)x[k][j][d], q[4 * j + d], s);
          s += __shfl_xor(s, 1);
          s += __shfl_xor(s, 2);
          s += __shfl_xor(s, 4);
          bad |= !ok[k];
          if (l8 == 0 && i < here) {
            ranks.key[kept + i] = range.rank(p, b0 + i, ok[k], s);
            ranks.id[kept + i] = b0 + i;
          }
        }
      }
      b0 += here;
      kept += here;
      __syncthreads();
      if (n <= kWaveKeys) {
        if (wave == 0) wave_select(ranks.key, n, top, lane, out);
      } else if (kept > top) {
        keep_highest(ranks, kept, top);
        kept = top;
      }
    }
    if (n > kWaveKeys)
      for (int i = threadIdx.x; i < top; i += 256) out[i] = ranks.id[i];
    if (bad) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
  }
}

// One work-group per 16 lists of a sequence and key head, for lists of few rows: the
// scores of 16 blocks for 16 lists on the matrix cores, in 64 bits; a wave then selects
// for four lists.  A lane of group g = lane / 16 holds elements 16 i + 4 g .. + 3 of
// block (of list) lane % 16.
//
// 6500 tokens of prompts, 4 heads of 64, up to 325 blocks: 78 us (484 with a work-group a
// list), of which the selection is 35 (a timing variant without it takes 43) and the
// 64-bit products are 10: MFMA busy 11%, VALU issuing 33%, the rest is waiting on the
// searches' counts.  (Eight waves, two lists each: 116 us, the queries' sums twice; fp32
// scores in LDS and the ranks anew where they tie: 95, with 3 to 6 groups a unit 93 to 107.)
template <int D, typename E>
__global__ __launch_bounds__(64 * kGroupWaves) void paged_select_group_kernel(SelectParams p, ListView groups, int pitch) {
  extern __shared__ uint64_t group_ranks[];    // [16][pitch]
  typedef double doublex4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int g = lane >> 4, x = lane & 15, top = p.v.top;
  if (refuse_batch(p)) return;
  {                                        // lists of no tile: before, between and behind the sequences'
    const int64_t per = (int64_t)p.c.Hkv * top;
    for (int64_t s = (int64_t)blockIdx.x * kGroupWaves + wave; s < p.c.B; s += kGroupWaves * (int64_t)gridDim.x) {
      const PagedSeq q = paged_seq(p.c, (int)s);
      const int64_t from = first_list(p.v, (int)s, q) + list_count(p.v, q);
      const int64_t to = s + 1 < p.c.B ? first_list(p.v, (int)s + 1, paged_seq(p.c, (int)s + 1)) : p.v.lists;
      for (int64_t i = from * per + lane; i < to * per; i += 64) p.blocks[i] = -1;
      if (s == 0)
        for (int64_t i = lane; i < first_list(p.v, 0, q) * per; i += 64) p.blocks[i] = -1;
    }
  }
  const int64_t total = (int64_t)groups.lists * p.c.Hkv;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int64_t gi = quotient(w, p.c.Hkv);
    const int h = (int)(w - gi * p.c.Hkv);
    PagedSeq sq;
    int r0;
    const int seq = paged_seq_of_list(p.c, groups, gi, lane, &sq, &r0);
    if (seq < 0) continue;
    const int tile = p.v.tile.by, lists = list_count(p.v, sq), l0 = r0 / p.v.tile;
    const int64_t list0 = first_list(p.v, seq, sq) + l0;
    auto range_of = [&](int l) __attribute__((always_inline)) {
      const int i0 = (l0 + l) * tile;
      return list_range(p, sq, i0, tile_end(p.v, sq, i0));
    };
    const int here = lists - l0 < kGroup ? lists - l0 : kGroup;
    const int n = sq.flags ? 0 : range_of(here - 1).n;       // of the last list, which sees the most
    bool bad = false;
    __syncthreads();                       // the ranks before have been read
    if (n > top) {
      double q[D / 4] = {};
      {
        const int l = x < here ? x : here - 1, i0 = (l0 + l) * tile, i1 = tile_end(p.v, sq, i0);
        for (int i = i0; i < i1; ++i)
          for (int j = 0; j < p.group; ++j) {
            const char* src = p.q + (int64_t)(sq.t0 + i) * p.q_str[0] + (h * p.group + j) * p.q_str[1] + 8 * g;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              typedef E e4 __attribute__((ext_vector_type(4)));
              const e4 v = *reinterpret_cast<const e4*>(src + 32 * k);
#pragma unroll
              for (int d = 0; d < 4; ++d) q[4 * k + d] += (double)(float)v[d];
            }
          }
      }
      const ListRange mine = range_of(x < here ? x : here - 1);
      const int32_t* table = p.c.table + seq * p.c.table_str;
      // the next 16 blocks' means are on their way while these are multiplied, and the
      // page numbers of those after them
      auto block_at = [&](int b0) __attribute__((always_inline)) { return b0 + x < n ? b0 + x : n - 1; };
      floatx4 next[D / 16];
      bool ok_next = false;
      auto load = [&](int b0, int page) __attribute__((always_inline)) {
        const int b = block_at(b0), e = b / p.v.parts;
        ok_next = (uint32_t)page < (uint32_t)p.c.n_pages;
        bad |= !ok_next;
        const char* m = p.means + (int64_t)(ok_next ? page : 0) * p.m_str[0] + (int64_t)(b - e * p.v.parts.by) * p.m_str[1] + h * p.m_str[2] + 16 * g;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) next[k] = *reinterpret_cast<const floatx4*>(m + 64 * k);
      };
      load(16 * wave, table[block_at(16 * wave) / p.v.parts]);
      int page = table[block_at(16 * (wave + kGroupWaves)) / p.v.parts];
      for (int b0 = 16 * wave; b0 < n; b0 += 16 * kGroupWaves) {
        floatx4 a[D / 16];
#pragma unroll
        for (int k = 0; k < D / 16; ++k) a[k] = next[k];
        const uint64_t fine = __builtin_amdgcn_ballot_w64(ok_next);
        load(b0 + 16 * kGroupWaves, page);
        page = table[block_at(b0 + 32 * kGroupWaves) / p.v.parts];
        __builtin_amdgcn_sched_barrier(0);
        doublex4 s[2] = {};
#pragma unroll
        for (int k = 0; k < D / 4; ++k)
          s[k & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)a[k >> 2][k & 3], q[k], s[k & 1], 0, 0, 0);
        s[0] += s[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {      // block 4 k + g, list x
          const int r = 4 * k + g;
          if (b0 + r < n) group_ranks[x * pitch + b0 + r] = mine.rank(p, b0 + r, fine >> r & 1, s[0][k]);
        }
      }
      if (bad) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
    }
    __syncthreads();
    for (int l = wave; l < here; l += kGroupWaves) {
      const int nl = sq.flags ? 0 : range_of(l).n;
      int32_t* out = p.blocks + ((list0 + l) * p.c.Hkv + h) * top;
      if (nl > top) {
        wave_select(group_ranks + l * pitch, nl, top, lane, out);
      } else {
        for (int i = lane; i < top; i += 64) out[i] = i < nl ? i : -1;
      }
    }
  }
}

// ─────────────────────────────── host side ─────────────────────────────────

constexpr int64_t kMostGroups = 1 << 20;

template <int D, typename E, int BITS> struct Means {
  static int go(const MeansParams& p, unsigned grid, hipStream_t stream) {
    hipLaunchKernelGGL((paged_means_kernel<D, E, BITS>), dim3(grid), dim3(256), 0, stream, p);
    return launch_status("lvsa_paged_block_means");
  }
};
template <int D, typename E, int BITS> struct Select {
  static int go(const SelectParams& p, bool grouped, hipStream_t stream) {
    if (grouped) {
      ListView groups = p.v;
      groups.tile = divisor(p.v.tile.by * kGroup);
      groups.lists = p.c.N / groups.tile.by + p.c.B;
      const int pitch = (int)((int64_t)p.c.max_pages * p.v.parts.by) | 1;
      const int64_t want = (int64_t)groups.lists * p.c.Hkv;
      hipLaunchKernelGGL((paged_select_group_kernel<D, E>), dim3((unsigned)(want < kMostGroups ? want : kMostGroups)), dim3(64 * kGroupWaves),
                         (unsigned)(8 * kGroup * pitch), stream, p, groups, pitch);
    } else {
      const int64_t want = (int64_t)p.v.lists * p.c.Hkv;
      hipLaunchKernelGGL((paged_select_kernel<D, E>), dim3((unsigned)(want < kMostGroups ? want : kMostGroups)), dim3(256), 0, stream, p);
    }
    return launch_status("lvsa_paged_select");
  }
};

// Means beside a cache: their strides in bytes.
int means_view(const char* what, const lvsa_paged_cache* c, const void* means, const int64_t* str, int block, int64_t* out,
               Divisor* by_block, Divisor* by_parts) {
  LVSA_REQUIRE(block >= 1 && c->page_size % block == 0, LVSA_ERR_INVALID_ARG, "%s: blocks of %d slots do not divide pages of %d",
               what, block, c->page_size);
  LVSA_REQUIRE((int64_t)c->n_pages * (c->page_size / block) < (1LL << 31), LVSA_ERR_UNSUPPORTED,
               "%s: %d pages of %d blocks", what, c->n_pages, c->page_size / block);
  bool ok = means && aligned16((int64_t)(uintptr_t)means);
  for (int i = 0; i < 3 && str; ++i) {
    out[i] = 4 * str[i];
    ok = ok && aligned16(out[i]);
  }
  LVSA_REQUIRE(ok && str, LVSA_ERR_INVALID_ARG, "%s: means must be non-null and their rows start at multiples of 16 bytes", what);
  *by_block = divisor(block);
  *by_parts = divisor(c->page_size / block);
  return LVSA_OK;
}

// Tiles of rows and lists of blocks.
int list_view(const char* what, const lvsa_paged_cache* c, const lvsa_paged_batch* b, int block, int top, int tile, ListView* v) {
  LVSA_REQUIRE(block >= 1 && c->page_size % block == 0, LVSA_ERR_INVALID_ARG, "%s: blocks of %d slots do not divide pages of %d",
               what, block, c->page_size);
  LVSA_REQUIRE(top >= 1 && top <= kListMax, LVSA_ERR_INVALID_ARG, "%s: lists of %d blocks (1 to %d)", what, top, kListMax);
  LVSA_REQUIRE(tile >= 1, LVSA_ERR_INVALID_ARG, "%s: tiles of %d rows", what, tile);
  const int64_t lists = tile == 1 ? b->N : (int64_t)(b->N / tile) + b->B;
  LVSA_REQUIRE(lists < (1LL << 31), LVSA_ERR_UNSUPPORTED, "%s: %lld lists", what, (long long)lists);
  v->block = divisor(block);
  v->parts = divisor(c->page_size / block);
  v->tile = divisor(tile);
  v->lists = (int32_t)lists;
  v->top = top;
  return LVSA_OK;
}

// Queries: their strides in bytes.
int query_view(const char* what, const lvsa_paged_cache* c, const lvsa_paged_batch* b, const void* q, const int64_t* str, int H,
               int64_t* out) {
  LVSA_REQUIRE(H >= 1 && H % c->Hkv == 0, LVSA_ERR_INVALID_ARG, "%s: %d heads over %d key heads", what, H, c->Hkv);
  LVSA_REQUIRE((int64_t)b->N * H < (1LL << 31) - 4096, LVSA_ERR_UNSUPPORTED, "%s: %d rows of %d heads", what, b->N, H);
  LVSA_REQUIRE(b->N == 0 || q, LVSA_ERR_INVALID_ARG, "%s: null q", what);
  out[0] = 2 * str[0];
  out[1] = 2 * str[1];
  LVSA_REQUIRE(aligned16((int64_t)(uintptr_t)q) && aligned16(out[0]) && aligned16(out[1]), LVSA_ERR_INVALID_ARG,
               "%s: rows must start at multiples of 16 bytes", what);
  return LVSA_OK;
}

int scale_check(const char* what, float scale) {
  LVSA_REQUIRE(scale > 0.f && scale <= 2.0e38f, LVSA_ERR_INVALID_ARG, "%s: scale %g must be positive and at most 2e38", what,
               (double)scale);
  return LVSA_OK;
}

// How an attention over lists runs: rows of a tile, row tiles of a list, the steps of
// each, and the work-groups that share them.
struct BlockShape {
  int rows, subs, steps, grid;
  int64_t work, o_elems;
  int64_t bytes(int D) const { return 4 * (o_elems + o_elems / D * 2); }
};
BlockShape block_shape(const lvsa_paged_block_attn_args* a, const ListView& v) {
  BlockShape s{};
  const lvsa_paged_attn_args& t = a->attn;
  const int64_t group = t.H / t.cache.Hkv, D = t.cache.D, N = t.batch.N, cus = cu_count();
  const int64_t rows = (v.tile.by < N ? v.tile.by : N) * group;
  s.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : kPagedTile;
  s.subs = (int)ceil_div(rows, s.rows);
  const int64_t units = (int64_t)v.lists * s.subs * t.cache.Hkv;
  const int64_t cap = (int64_t)t.batch.max_pages * t.cache.page_size;
  int64_t keys = (int64_t)v.top * v.block.by < cap ? (int64_t)v.top * v.block.by : cap;
  if (keys < 1) keys = 1;
  s.steps = (int)ceil_div(keys, s.rows == kPagedTile ? kPagedBlock : paged_decode_keys((int)D));
  s.work = units * s.steps;
  // Shares: one per row tile where these are enough to keep the card busy, which is one
  // for every compute unit (of 4-bit pages, which need waves to decode, one for every
  // work-group that runs at once): nothing is to be joined, and each reads one list.
  // Otherwise as many whole parts of a tile as come near to what runs at once, else
  // equal shares.  us, with one share a tile and with equal shares:
  //   16 bits, 128: 444 tiles of 128 rows 195, 214; 384 of 16 rows 86, 86; 800 92, 94;
  //                 26000 (prompts, each token its own list, of 64) 705, 844
  //   16 bits, 64:  256 of 16 rows 27, 33; 16 bits, 256: 120 68, 56 and 132 of 128 rows 96, 90
  //   16 bits, 128: 160 of 16 rows 70, 69; 64 67, 40; 4 37, 22
  //    4 bits, 128: 800 41, 43; 320 68, 56 (54 in two parts each)
  const int64_t slots = cus * (s.rows == kPagedTile ? (D >= 192 ? 1 : 2) : paged_decode_groups((int)D, t.cache.bits, s.rows));
  const int64_t enough = t.cache.bits == 16 ? cus : slots, parts = units > 0 ? slots / units : 0;
  int64_t shares = s.work < slots ? s.work : slots;
  if (units >= enough && units <= kMostGroups) shares = units;
  else if (parts >= 2 && parts <= s.steps && 5 * parts * units >= 4 * slots) shares = parts * units;
  s.grid = (int)shares;
  s.o_elems = s.work == s.grid * (int64_t)s.steps ? 0 : 2LL * s.grid * s.rows * D;
  return s;
}

int block_attn_check(const lvsa_paged_block_attn_args* a, PagedAttnParams* p, ListView* v) {
  const char* what = "lvsa_paged_block_attn_fwd";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  const lvsa_paged_attn_args& t = a->attn;
  int rc = paged_view(what, &t.cache, &t.batch, true, &p->c);
  if (!rc) rc = query_view(what, &t.cache, &t.batch, t.q, t.q_str, t.H, p->q_str);
  if (!rc) rc = scale_check(what, t.scale);
  if (!rc) rc = list_view(what, &t.cache, &t.batch, a->block, a->top, a->tile, v);
  return rc;
}

int weights_check(const lvsa_paged_weights_args* a, PagedAttnParams* p) {
  const char* what = "lvsa_paged_weights";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  int rc = paged_view(what, &a->cache, &a->batch, true, &p->c);
  if (!rc) rc = query_view(what, &a->cache, &a->batch, a->q, a->q_str, a->H, p->q_str);
  if (!rc) rc = scale_check(what, a->scale);
  return rc;
}

// How an accumulation runs.
struct WeightsShape {
  int many, grid, splits;
  int64_t bytes;
};
WeightsShape weights_shape(const lvsa_paged_weights_args* a) {
  WeightsShape s{};
  // rows of a sequence, if unknown: one each where there are no more than sequences, else all of one
  // (8 sequences of 2, 4 and 9 rows, 4 query heads a key head, over 8000 keys: 52 to 53 us
  // without max_q_len, 30, 31 and 47 with it)
  const int64_t N = a->batch.N, q = a->max_q_len > 0 ? (a->max_q_len < N ? a->max_q_len : N) : N <= a->batch.B ? 1 : N;
  // sequences that have work: see weight_units
  const int64_t rows = q * (a->H / a->cache.Hkv), B = a->batch.B < N ? a->batch.B : N, cus = cu_count();
  // The rows' kernel from 48 rows a sequence and key head on: us, few rows' and rows'
  // kernel, 8 sequences of 8000 keys, 8 heads of 128: 16 rows 31, 51; 32 42, 51; 48 50,
  // 51; 64 58, 50; 128 90, 61 (32 sequences of 4000: 32 rows 72, 100; 64 100, 100).
  s.many = rows > 48;
  s.splits = 1;
  const int64_t cap = (int64_t)a->batch.max_pages * a->cache.page_size;
  int64_t units = B * ceil_div(cap, s.many ? kWeightKeys : paged_decode_keys(a->cache.D)) * a->cache.Hkv;
  if (units < 1) units = 1;
  if (s.many) {
    // 12 work-groups a compute unit, if the table is full: 92, 87, 82, 85 us with 4, 8, 12
    // and 16 for 6500 tokens of prompts over up to 5200 keys, 4 heads of 64 (no other shape
    // was tried).  A wider table counts as full, too: 113 instead of 85 us in one of 32768
    // slots and more; one stream's 500 tokens over 5000 keys 66 us, 47, 59 and 88 in tables
    // of 32768, 65536 and 131072.
    const int64_t want = ceil_div(12 * cus, units), tiles = ceil_div(rows, 128);
    s.splits = (int)(want < tiles ? want : tiles);
    s.bytes = s.splits == 1 ? 0 : 4 * units * s.splits * kWeightKeys;
    units *= s.splits;
  }
  const int64_t most = s.many ? 64 * cus : cus * kWeightGroups;
  s.grid = (int)(units < most ? units : most);
  return s;
}

}  // namespace
}  // namespace lvsa

extern "C" {

int lvsa_paged_block_means(const lvsa_paged_means_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_block_means";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  MeansParams p{};
  int rc = paged_view(what, &a->cache, &a->batch, false, &p.c);
  if (!rc) rc = means_view(what, &a->cache, a->means, a->m_str, a->block, p.m_str, &p.block, &p.parts);
  if (rc) return rc;
  const lvsa_paged_batch& b = a->batch;
  if (b.B == 0 || (b.cu_seqlens && b.N == 0)) return LVSA_OK;
  p.means = (char*)a->means;
  const int64_t all = (int64_t)b.B * b.max_pages * p.parts.by, touched = (int64_t)b.N / a->block + 2LL * b.B;
  const int64_t want = (b.cu_seqlens && touched < all ? touched : all) * a->cache.Hkv, most = 4LL * cu_count();
  return by_type<Means>(a->cache.D, a->cache.dtype, a->cache.bits, p, (unsigned)(want < 1 ? 1 : want < most ? want : most), stream);
}

int lvsa_paged_select(const lvsa_paged_select_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_select";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  SelectParams p{};
  Divisor block, parts;
  int rc = paged_view(what, &a->cache, &a->batch, true, &p.c);
  if (!rc) rc = query_view(what, &a->cache, &a->batch, a->q, a->q_str, a->H, p.q_str);
  if (!rc) rc = means_view(what, &a->cache, a->means, a->m_str, a->block, p.m_str, &block, &parts);
  if (!rc) rc = list_view(what, &a->cache, &a->batch, a->block, a->top, a->tile, &p.v);
  if (rc) return rc;
  const int64_t span = a->tile == 1 ? 1 : (int64_t)(a->tile - 2) / a->block + 2;
  LVSA_REQUIRE(a->first >= 0 && a->last >= 0 && a->first + (a->last ? a->last - 1 + span : 0) <= a->top, LVSA_ERR_INVALID_ARG,
               "%s: the first %d blocks, and the last %d of tiles of %d rows, do not fit into %d", what, a->first, a->last,
               a->tile, a->top);
  if (p.v.lists == 0 || a->batch.B == 0) return LVSA_OK;
  LVSA_REQUIRE(a->blocks, LVSA_ERR_INVALID_ARG, "%s: null blocks", what);
  p.q = (const char*)a->q;
  p.means = (const char*)a->means;
  p.blocks = a->blocks;
  p.group = a->H / a->cache.Hkv;
  p.first = a->first;
  p.last = a->last;
  p.causal = a->causal;
  // Sixteen lists of a sequence together where sequences have many, of few rows, and
  // there are more of them than one round of single work-groups takes.  us, sixteen
  // together and one by one, lists of 32 blocks of 64 over 8000 keys, 8 heads of 128:
  //   lists x heads 256: 17, 12; 512: 18, 12 (of one sequence 25, 11); 1024 (4 and 16 a
  //   sequence): 20, 19 and 25, 18; 2048 (8 and 256): 24, 33 and 25, 33; 16384: 59, 227
  //   rows of a list, its tokens x query heads, 16384 lists x heads: 4: 59, 227; 16: 100,
  //   248; 4096 of 16: 52, 65; 2080 of 32: 50, 36
  // LDS has room for 1024 ranks a list: a wider table goes the other way, whatever its
  // sequences fill of it (6500 tokens of prompts over up to 325 blocks 312 us, 79 in a table
  // of 325).
  const int64_t cap = (int64_t)a->batch.max_pages * p.v.parts.by;
  const bool grouped = (int64_t)a->tile * p.group <= 16 && p.v.lists >= 8LL * a->batch.B &&
                       (int64_t)p.v.lists * a->cache.Hkv >= 6LL * cu_count() && cap <= kWaveKeys;
  return by_type<Select>(a->cache.D, a->cache.dtype, 16, p, grouped, stream);
}

int lvsa_paged_block_attn_workspace_query(const lvsa_paged_block_attn_args* a, int64_t* bytes) {
  clear_error();
  LVSA_REQUIRE(bytes != nullptr, LVSA_ERR_INVALID_ARG, "lvsa_paged_block_attn_workspace_query: null output");
  PagedAttnParams p{};
  ListView v{};
  const int rc = block_attn_check(a, &p, &v);
  if (rc) return rc;
  *bytes = a->attn.batch.N == 0 || a->attn.batch.B == 0 ? 0 : block_shape(a, v).bytes(a->attn.cache.D);
  return LVSA_OK;
}

int lvsa_paged_block_attn_fwd(const lvsa_paged_block_attn_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_block_attn_fwd";
  PagedAttnParams p{};
  BlockAttnParams l{};
  int rc = block_attn_check(a, &p, &l.v);
  if (rc) return rc;
  const lvsa_paged_attn_args& t = a->attn;
  if (t.batch.N == 0) return LVSA_OK;
  LVSA_REQUIRE(t.o && a->blocks, LVSA_ERR_INVALID_ARG, "%s: null o or blocks", what);
  p.o_str[0] = 2 * t.o_str[0];
  p.o_str[1] = 2 * t.o_str[1];
  LVSA_REQUIRE(aligned16((int64_t)(uintptr_t)t.o) && aligned16(p.o_str[0]) && aligned16(p.o_str[1]), LVSA_ERR_INVALID_ARG,
               "%s: rows must start at multiples of 16 bytes", what);
  LVSA_REQUIRE(!share_memory(t.o, p.o_str, t.H, t.q, p.q_str, t.H, t.batch.N, t.cache.D), LVSA_ERR_INVALID_ARG,
               "%s: o must not share memory with q", what);
  LVSA_REQUIRE(t.batch.B > 0, LVSA_ERR_INVALID_ARG, "%s: rows of no sequence", what);
  const BlockShape s = block_shape(a, l.v);
  const int64_t need = s.bytes(t.cache.D);
  LVSA_REQUIRE(need == 0 || (t.workspace && aligned16((int64_t)(uintptr_t)t.workspace)), LVSA_ERR_INVALID_ARG,
               "%s: %lld bytes of 16-byte aligned workspace needed", what, (long long)need);
  LVSA_REQUIRE(need == 0 || t.workspace_bytes >= need, LVSA_ERR_CAPACITY, "%s: workspace of %lld bytes < %lld", what,
               (long long)t.workspace_bytes, (long long)need);
  p.q = (const char*)t.q;
  p.o = (char*)t.o;
  p.lse = t.lse;
  p.scale_log2 = t.scale * 1.4426950408889634f;
  p.H = t.H;
  p.group = t.H / t.cache.Hkv;
  p.causal = t.causal;
  p.fill_tail = t.fill_tail;
  p.short_rows = p.c.k_str[1] >= 0 && p.c.k_str[1] < (1 << 26) && p.c.v_str[1] >= 0 && p.c.v_str[1] < (1 << 26);
  p.ws_o = (float*)t.workspace;
  p.ws_ml = p.ws_o + s.o_elems;
  p.grid = s.grid;
  l.blocks = a->blocks;
  l.subs = s.subs;
  l.steps = s.steps;
  l.work = s.work;
  const bool bf16 = t.cache.dtype == LVSA_BF16;
  switch (t.cache.D) {
    case 64: return paged_block_attn_d64(p, l, t.cache.bits, s.rows, bf16, stream);
    case 96: return paged_block_attn_d96(p, l, t.cache.bits, s.rows, bf16, stream);
    case 128: return paged_block_attn_d128(p, l, t.cache.bits, s.rows, bf16, stream);
    case 192: return paged_block_attn_d192(p, l, t.cache.bits, s.rows, bf16, stream);
    default: return paged_block_attn_d256(p, l, t.cache.bits, s.rows, bf16, stream);
  }
}

int lvsa_paged_weights_workspace_query(const lvsa_paged_weights_args* a, int64_t* bytes) {
  clear_error();
  LVSA_REQUIRE(bytes != nullptr, LVSA_ERR_INVALID_ARG, "lvsa_paged_weights_workspace_query: null output");
  PagedAttnParams p{};
  const int rc = weights_check(a, &p);
  if (rc) return rc;
  *bytes = a->batch.N == 0 || a->batch.B == 0 ? 0 : weights_shape(a).bytes;
  return LVSA_OK;
}

int lvsa_paged_weights(const lvsa_paged_weights_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_weights";
  PagedAttnParams p{};
  WeightsParams w{};
  const int rc = weights_check(a, &p);
  if (rc) return rc;
  LVSA_REQUIRE(a->weights && ((uintptr_t)a->weights & 3) == 0 && (a->lse || a->batch.N == 0), LVSA_ERR_INVALID_ARG,
               "%s: weights and lse must be non-null, fp32", what);
  if (a->batch.N == 0 || a->batch.B == 0) return LVSA_OK;
  const WeightsShape s = weights_shape(a);
  LVSA_REQUIRE(s.bytes == 0 || (a->workspace && aligned16((int64_t)(uintptr_t)a->workspace)), LVSA_ERR_INVALID_ARG,
               "%s: %lld bytes of 16-byte aligned workspace needed", what, (long long)s.bytes);
  LVSA_REQUIRE(s.bytes == 0 || a->workspace_bytes >= s.bytes, LVSA_ERR_CAPACITY, "%s: workspace of %lld bytes < %lld", what,
               (long long)a->workspace_bytes, (long long)s.bytes);
  p.q = (const char*)a->q;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.H = a->H;
  p.group = a->H / a->cache.Hkv;
  p.causal = a->causal;
  p.grid = s.grid;
  w.lse = a->lse;
  w.w = (char*)a->weights;
  for (int i = 0; i < 3; ++i) w.w_str[i] = 4 * a->w_str[i];
  w.accumulate = a->accumulate;
  w.many = s.many;
  w.splits = s.splits;
  w.ws = (float*)a->workspace;
  const bool bf16 = a->cache.dtype == LVSA_BF16;
  switch (a->cache.D) {
    case 64: return paged_weights_d64(p, w, a->cache.bits, bf16, stream);
    case 96: return paged_weights_d96(p, w, a->cache.bits, bf16, stream);
    case 128: return paged_weights_d128(p, w, a->cache.bits, bf16, stream);
    case 192: return paged_weights_d192(p, w, a->cache.bits, bf16, stream);
    default: return paged_weights_d256(p, w, a->cache.bits, bf16, stream);
  }
}

}  // extern "C"
