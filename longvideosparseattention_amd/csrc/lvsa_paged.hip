// Paged key/value cache on gfx950: appending new tokens (rotation by position
// and 4-bit quantisation on the way), reading a cache back, the merge of
// attention partials, and the C ABI.  The attention kernels are in
// lvsa_paged_attn.h.
#include "lvsa_paged_host.h"
#include "lvsa_paged_rows.h"

using namespace lvsa;

namespace lvsa {
namespace {

constexpr int kMaxGrid = 1 << 20;      // work-groups of a launch that walks its rows
constexpr int kMaxGridY = 1 << 15;     // sequences of a gather's launch
constexpr int kFewTokens = 10;         // of an append, per compute unit

// x in 32 bits, rounded to odd: the two neighbours' sticky bit is kept, so that
// a later rounding to few bits (and a comparison with a number of few bits)
// comes out as if it had been made from the 64-bit value.
__device__ __forceinline__ float to_odd(double x) {
  float f = (float)x;
  if (__builtin_isinf(f) && !__builtin_isinf(x)) return __builtin_copysignf(3.0e38f, f);
  const double back = (double)f;
  if (back != x) {       // false for NaN with NaN's payload only: handled by the caller's non-finite test
    uint32_t b = __builtin_bit_cast(uint32_t, f);
    if (__builtin_fabs(back) > __builtin_fabs(x)) b -= 1;   // |f| rounded up: back to the neighbour below
    f = __builtin_bit_cast(float, b | 1u);
  }
  return f;
}

// ──────────────────────────────── append ───────────────────────────────────

struct AppendParams {
  PagedView c;
  const char* k; const char* v; const char* q; char* qo;
  int64_t k_str[2], v_str[2], q_str[2], qo_str[2];   // bytes
  const float* cos; const float* sin;
  const int32_t* positions;
  int H, rot, interleaved, n_angles;
};

// One work-group per token; a thread holds chunk `c` (8 elements) of every
// RPP-th row, where the rows are the token's keys, values and queries.  The
// chunk's angles are read once and serve all of them.  A rotated element
// needs its partner: in the same chunk with interleaved pairs, else rot / 2
// elements away, which is a second 16-byte load of a line that the neighbours
// fetch anyway.  Bound by memory, and for small calls by the trips to it one
// after the other: the batch, the page with the angles, the row.  (Rows read
// ahead of their slot cost more in registers than they save: 93 instead of 80 us
// for 7868 tokens of 32 + 8 + 8 rows of 128 into a 4-bit cache and their reading
// back.)
//
// 16-bit caches: turned in fp32, one rounding at the end.  4-bit caches: the
// turned key is formed in 64 bits, where both products are exact and the sum
// rounds once, and goes to odd-rounded fp32 for the converter: a key next to
// the border of two codes or of two scales comes out as the exact value's
// would, on every device and in every order of evaluation.
//
// 256 threads for few tokens, where the row after row of one wave would be waited
// for, 64 where there are many: each wave looks the token up for itself (the same
// 7868 tokens 72 us with 256, 64 with 128, 61 with 64; on 256 units, 256 and 64
// threads: 32 tokens 5.8, 10.3 us, 2048 16.0, 16.6, 4096 27.7, 22.1; into 16 bits
// 4.5, 7.6, 13.0, 14.7, 26.8, 26.7).
template <int D, typename E, int BITS, int THREADS>
__device__ __forceinline__ void append_token(const AppendParams& p, int t) {
  constexpr int CH = D / 8, RPP = THREADS / CH;
  const int lane = threadIdx.x & 63;
  const int c = threadIdx.x % CH, r0 = threadIdx.x / CH;
  const int half = p.rot / 2;
  const bool turn = 8 * c < p.rot;
  const bool second = !p.interleaved && 8 * c >= half;   // this chunk holds the second elements of its pairs
  const int partner = p.interleaved ? 0 : second ? -half : half;
  const int Hkv = p.c.Hkv, rows = r0 < RPP ? 2 * Hkv + (p.q ? p.H : 0) : 0;   // D = 96 and 192 leave a few threads over
  u32x4 raw = {}, other = {};
  auto load = [&](int r) __attribute__((always_inline)) {
    const char* src = r < Hkv ? p.k + t * p.k_str[0] + r * p.k_str[1]
                    : r >= 2 * Hkv ? p.q + t * p.q_str[0] + (r - 2 * Hkv) * p.q_str[1]
                                   : p.v + t * p.v_str[0] + (r - Hkv) * p.v_str[1];
    raw = *reinterpret_cast<const u32x4*>(src + 16 * c);
    if (turn && partner && (r < Hkv || r >= 2 * Hkv)) other = *reinterpret_cast<const u32x4*>(src + 16 * c + 2 * partner);
  };

  PagedSeq sq;
  const int s = paged_seq_of_row(p.c, t, lane, &sq);
  if (s < 0) return;                        // a row of no sequence: left alone
  const int64_t pos = (int64_t)sq.first + (t - sq.t0);
  int flags = sq.flags;
  int64_t page = 0, slot = 0;
  if (pos < 0) flags |= LVSA_PAGED_BAD_APPEND;
  if (!(flags & (LVSA_PAGED_BAD_LENGTH | LVSA_PAGED_BAD_APPEND | LVSA_PAGED_BAD_CU))) {
    const PagedRow row = paged_row(p.c, (int)pos, p.c.table[s * p.c.table_str + page_of(p.c, (int)pos)]);
    page = row.page;
    slot = row.slot;
    if (!row.ok) flags |= LVSA_PAGED_BAD_PAGE;
  }
  int64_t angle = pos;
  if (p.rot) {
    if (p.positions) angle = p.positions[t];
    if (angle < 0 || angle >= p.n_angles) flags |= LVSA_PAGED_BAD_POSITION;
  }
  const bool bad = flags != 0;
  if (bad && threadIdx.x == 0) paged_flag(p.c, flags);

  float cs[8], sn[8];
  if (turn && !bad) {
    const int64_t base = angle * half;
    if (p.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[i] = p.cos[base + 4 * c + i];
        sn[i] = p.sin[base + 4 * c + i];
      }
    } else {
      const int i0 = second ? 8 * c - half : 8 * c;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        cs[i] = p.cos[base + i0 + i];
        sn[i] = second ? p.sin[base + i0 + i] : -p.sin[base + i0 + i];
      }
    }
  }

  for (int r = r0; r < rows; r += RPP) {
    const bool is_k = r < Hkv, is_q = r >= 2 * Hkv;
    const int h = is_k ? r : is_q ? r - 2 * Hkv : r - Hkv;
    if (bad) {
      if (is_q) {
        const uint32_t n2 = Half<E>::kNaN * 0x10001u;
        *reinterpret_cast<u32x4*>(p.qo + t * p.qo_str[0] + h * p.qo_str[1] + 16 * c) = u32x4{n2, n2, n2, n2};
      }
      continue;
    }
    load(r);
    const bool turned = turn && (is_k || is_q);
    float x[8], y[8];
    u32x4 w = raw;
    Half<E>::unpack(raw, x);
    Half<E>::unpack(other, y);
    if (BITS == 16 || is_q) {
      if (turned) {
        float z[8];
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z[2 * i] = __builtin_fmaf(x[2 * i], cs[i], -(x[2 * i + 1] * sn[i]));
            z[2 * i + 1] = __builtin_fmaf(x[2 * i + 1], cs[i], x[2 * i] * sn[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) z[i] = __builtin_fmaf(x[i], cs[i], y[i] * sn[i]);
        }
        w = pack8<E>(z);
      }
      char* dst = is_q ? p.qo + t * p.qo_str[0] + h * p.qo_str[1]
                       : (is_k ? p.c.k + page * p.c.k_str[0] + slot * p.c.k_str[1] + h * p.c.k_str[2]
                               : p.c.v + page * p.c.v_str[0] + slot * p.c.v_str[1] + h * p.c.v_str[2]);
      // turned queries pass the L2 by (another kernel reads them): 74.7 -> 72.5 us as above
      if (is_q) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(dst + 16 * c));
      else *reinterpret_cast<u32x4*>(dst + 16 * c) = w;
    } else {
      if (turned) {
        // The angles are widened here, row by row, and two elements are formed at
        // a time: fewer registers, more waves, 73 instead of 80 us as above.
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(cs[i]), "+v"(sn[i]));
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const double a = x[2 * i], b = x[2 * i + 1], cc = cs[i], ss = sn[i];
            x[2 * i] = to_odd(__builtin_fma(a, cc, -(b * ss)));
            x[2 * i + 1] = to_odd(__builtin_fma(b, cc, a * ss));
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = to_odd(__builtin_fma((double)x[i], (double)cs[i], (double)y[i] * (double)sn[i]));
            if (i & 1) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      // the largest of the 32 values that four neighbouring threads hold; a
      // NaN or an infinity among them as infinity
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = __builtin_fabsf(x[i]);
        m = a <= 3.4028235e38f ? (a > m ? a : m) : __builtin_inff();
      }
      m = __builtin_fmaxf(m, __shfl_xor(m, 1));
      m = __builtin_fmaxf(m, __shfl_xor(m, 2));
      // smallest e with 6 * 2^e >= m: of m = f * 2^k, 1 <= f < 2, that is k - 2
      // for f <= 1.5 and k - 1 above
      const uint32_t mb = __builtin_bit_cast(uint32_t, m);
      int e = (int)(mb >> 23) - 127 - 2 + ((mb & 0x7fffffu) > 0x400000u ? 1 : 0);
      e = e < -23 ? -23 : e > 13 ? 13 : e;
      const float scale = __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
      uint32_t codes = 0;
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
      const bool finite = m <= 3.4028235e38f;
      char* dst = is_k ? p.c.k + page * p.c.k_str[0] + slot * p.c.k_str[1] + h * p.c.k_str[2]
                       : p.c.v + page * p.c.v_str[0] + slot * p.c.v_str[1] + h * p.c.v_str[2];
      uint8_t* sd = is_k ? p.c.ks + page * p.c.ks_str[0] + slot * p.c.ks_str[1] + h * p.c.ks_str[2]
                         : p.c.vs + page * p.c.vs_str[0] + slot * p.c.vs_str[1] + h * p.c.vs_str[2];
      *reinterpret_cast<uint32_t*>(dst + 4 * c) = finite ? codes : 0u;
      if ((c & 3) == 0) sd[c >> 2] = finite ? (uint8_t)(e + 127) : (uint8_t)255;
    }
  }
}

// Reports row ranges that do not ascend within the rows, whether or not a row is
// in them (a work-group beside the tokens', so that none of those waits for it).
__device__ __forceinline__ void flag_row_ranges(const PagedView& c) {
  for (int s = threadIdx.x; s < c.B; s += blockDim.x)
    if (const int bad = paged_seq(c, s).flags & LVSA_PAGED_BAD_CU) paged_flag(c, bad);
}

template <int D, typename E, int BITS, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_append_kernel(AppendParams p) {
  if (blockIdx.x == gridDim.x - 1) flag_row_ranges(p.c);
  for (int64_t t = blockIdx.x; t < p.c.N; t += gridDim.x) append_token<D, E, BITS, THREADS>(p, (int)t);
}

// ──────────────────────────────── gather ───────────────────────────────────

// Work-groups of grid.x walk (position, head, chunk) of sequence b0 + blockIdx.y
// in the order of the output, so that the writes, two thirds or more of the
// traffic, are contiguous; blockIdx.z: keys, values.  Bound by memory.  The
// output passes the L2 by, which is too small for it and serves the table and the
// cache's lines: 12 sequences of up to 2500 tokens, 16 heads of 64 in 4 bits, 38.5
// -> 24.9 us; 15600 tokens of 12 heads of 128 in 16 bits 36.5 -> 33.2 us.
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256) void paged_gather_kernel(PagedView c, char* ko, char* vo, int max_len, int b0) {
  constexpr int CH = D / 8;
  const int b = b0 + blockIdx.y;
  const bool is_v = blockIdx.z;
  int L = c.lens[b];
  const int64_t cap = (int64_t)c.max_pages * c.page_size;
  const bool bad_len = L < 0 || L > cap;
  if (bad_len && blockIdx.x == 0 && threadIdx.x == 0) paged_flag(c, LVSA_PAGED_BAD_LENGTH);
  if (L > max_len) L = max_len;
  const char* src = is_v ? c.v : c.k;
  const uint8_t* sc = is_v ? c.vs : c.ks;
  const int64_t s0 = is_v ? c.v_str[0] : c.k_str[0], s1 = is_v ? c.v_str[1] : c.k_str[1],
                s2 = is_v ? c.v_str[2] : c.k_str[2];
  const int64_t c0 = is_v ? c.vs_str[0] : c.ks_str[0], c1 = is_v ? c.vs_str[1] : c.ks_str[1],
                c2 = is_v ? c.vs_str[2] : c.ks_str[2];
  u32x4* out = reinterpret_cast<u32x4*>((is_v ? vo : ko) + (int64_t)b * max_len * c.Hkv * (2 * D));
  const uint32_t per = (uint32_t)c.Hkv * CH;                 // chunks of one position
  const int64_t total = (int64_t)max_len * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int pos = (int)(i / per);
    const uint32_t rest = (uint32_t)(i - (int64_t)pos * per), h = rest / CH, ch = rest % CH;
    u32x4 w = {0, 0, 0, 0};
    if (bad_len) {
      const uint32_t n2 = Half<E>::kNaN * 0x10001u;
      w = u32x4{n2, n2, n2, n2};
    } else if (pos < L) {
      const PagedRow at = paged_row(c, pos, c.table[b * c.table_str + page_of(c, pos)]);
      if (!at.ok) {
        paged_flag(c, LVSA_PAGED_BAD_PAGE);
        const uint32_t n2 = Half<E>::kNaN * 0x10001u;
        w = u32x4{n2, n2, n2, n2};
      } else {
        const char* row = src + at.page * s0 + at.slot * s1 + h * s2;
        if constexpr (BITS == 16) {
          w = *reinterpret_cast<const u32x4*>(row + 16 * ch);
        } else {
          const uint32_t codes = *reinterpret_cast<const uint32_t*>(row + 4 * ch);
          w = unpack_e2m1<E>(codes, sc[at.page * c0 + at.slot * c1 + h * c2 + (ch >> 2)]);
        }
      }
    }
    __builtin_nontemporal_store(w, out + i);
  }
}

// ───────────────────────── merge of the partials ───────────────────────────

// One work-group per output row: finds the row's sequence, tile and the slots
// that hold partials of it, and merges them: o = sum_i 2^(m_i - M) o_i / sum_i
// 2^(m_i - M) l_i.  The four waves take the slots in turn, each with a running
// maximum as in the attention itself, and are joined in their order, so results
// do not depend on timing.  Rows whose tile one work-group of the decode kernel
// did whole are written already.  Rows without keys, rows of no sequence and, as
// NaN, all rows of a batch whose row ranges are bad are this kernel's too.  Latency: the batch, the partials (two slots of a wave at a
// time, maxima and sums beside them), one exchange.  Every row goes through the
// batch again, 64 sequences a trip.
template <typename E>
__device__ __forceinline__ void merge_row(const PagedAttnParams& p, int row, int D, int rows, int keys,
                                          float (*acc_s)[256], float (*ml_s)[2]) {
  const int t = (uint32_t)row / (uint32_t)p.H, hq = row - t * p.H;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), B = p.c.B;
  E* out = reinterpret_cast<E*>(p.o + t * p.o_str[0] + hq * p.o_str[1]);
  float* lse = p.lse ? p.lse + (int64_t)t * p.H + hq : nullptr;
  PagedSeq sq = {};
  int s = -1;
  int64_t U = 0, base = 0;
  int flags = 0;
  for (int s0 = 0; s0 < B; s0 += 64) {
    PagedSeq q = {};
    int64_t n = 0;
    bool in = false;
    if (s0 + lane < B) {
      const int a = p.c.cu[s0 + lane], e = p.c.cu[s0 + lane + 1];
      q = paged_seq(p.c, a, e, p.c.lens[s0 + lane]);
      n = decode_units(p, q, rows, keys);
      in = a <= t && t < e;
      flags |= q.flags;
    }
    const int64_t incl = wave_scan(n, lane, B - s0);
    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
    if (m && s < 0) {
      const int at = __builtin_ctzll(m);
      s = s0 + at;
      sq = from_lane(q, at);
      base = U + from_lane(incl - n, at);
    }
    U += from_lane(incl, B - s0 < 64 ? B - s0 - 1 : 63);
  }
  if (__builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) {
    for (int d = threadIdx.x; d < D; d += 256) out[d] = (E)__builtin_nanf("");
    if (lse && threadIdx.x == 0) *lse = __builtin_nanf("");
    return;
  }
  if (s < 0) {
    if (p.fill_tail) {
      if (p.fill_tail == 1)
        for (int d = threadIdx.x; d < D; d += 256) out[d] = (E)0.f;
      if (lse && threadIdx.x == 0) *lse = -__builtin_inff();
    }
    return;
  }
  const int h = (uint32_t)hq / (uint32_t)p.group;
  const int r = (t - sq.t0) * p.group + (hq - h * p.group);
  DecodeSlots parts = {0, 0, 0};
  const int nb = (int)(((int64_t)sq.L + keys - 1) / keys);
  if (nb > 0) {
    parts = decode_slots(U, unit_shares(U, p.grid), base + ((int64_t)(r / rows) * p.c.Hkv + h) * nb, nb);
    if (parts.count == 0) return;          // written by the attention kernel
  }
  const int count = parts.count;
  const int rr = r % rows;
  auto slot_of = [&](int i) { return i == 0 ? parts.first : parts.rest + 2 * i; };

  float M = kNoKeys, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = wave; i < count; i += 8) {
    float m[2], ls[2], x[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {          // past the last one: the first again, with no weight
      const bool real = i + 4 * j < count;
      const int64_t at = slot_of(real ? i + 4 * j : i) * rows + rr;
      m[j] = real ? p.ws_ml[2 * at] : kNoKeys;
      ls[j] = real ? p.ws_ml[2 * at + 1] : 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[j][k] = real && 64 * k < D && lane + 64 * k < D ? p.ws_o[at * D + lane + 64 * k] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float top = __builtin_fmaxf(M, m[j]);
      const float a = __builtin_amdgcn_exp2f(M - top), b = __builtin_amdgcn_exp2f(m[j] - top);
      l = l * a + ls[j] * b;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = acc[k] * a + x[j][k] * b;
      M = top;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) acc_s[wave][lane + 64 * k] = acc[k];
  if (lane == 0) {
    ml_s[wave][0] = M;
    ml_s[wave][1] = l;
  }
  __syncthreads();
  M = __builtin_fmaxf(__builtin_fmaxf(ml_s[0][0], ml_s[1][0]), __builtin_fmaxf(ml_s[2][0], ml_s[3][0]));
  float w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = __builtin_amdgcn_exp2f(ml_s[k][0] - M);
  l = (ml_s[0][1] * w[0] + ml_s[1][1] * w[1]) + (ml_s[2][1] * w[2] + ml_s[3][1] * w[3]);
  if (sq.flags & LVSA_PAGED_BAD_LENGTH) l = __builtin_nanf("");
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  for (int d = threadIdx.x; d < D; d += 256)
    out[d] = (E)(((acc_s[0][d] * w[0] + acc_s[1][d] * w[1]) + (acc_s[2][d] * w[2] + acc_s[3][d] * w[3])) * inv);
  if (lse && threadIdx.x == 0) *lse = l == 0.f ? -__builtin_inff() : (M + __log2f(l)) * 0.69314718055994530942f;
}

template <typename E>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnParams p, int D, int rows, int keys) {
  __shared__ float acc_s[4][256];
  __shared__ float ml_s[4][2];
  for (int64_t row = blockIdx.x; row < (int64_t)p.c.N * p.H; row += gridDim.x) {
    merge_row<E>(p, (int)row, D, rows, keys, acc_s, ml_s);
    __syncthreads();             // the next row writes the same LDS
  }
}

// ───────────────────────── plan of a prefill launch ────────────────────────

// Sum over the work-group's 1024 threads before this one, and the total.
// `count`: threads that may hold anything but 0.
__device__ __forceinline__ int64_t block_scan(int64_t x, int count, int64_t* lds, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t incl = wave_scan(x, lane, count);
  __syncthreads();
  if (lane == (count < 64 ? count - 1 : 63)) lds[wave] = incl;
  __syncthreads();
  if (count <= 64) {                       // the first wave's
    *total = lds[0];
    return incl - x;
  }
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wave ? lds[w] : 0;
    all += lds[w];
  }
  *total = all;
  return before + incl - x;
}

// One work-group: lists the row tiles with their key blocks, where the shares
// end and what is to be joined there.  Latency only: two dependent reads of
// memory, scans and searches in LDS (searches in memory past kPlanLds tiles); 6 to
// 8 us beside launches of 25 us and more.  With it every work-group of those
// gets the same number of key blocks, whatever the lengths, where tiles as units
// leave the last round to a few (516 tiles on 256 CUs: three rounds for two
// rounds' work).
//
// A bad page spoils its whole sequence, but a causal tile does not look behind its
// last row's key: the plan looks through the pages of the rows of every tile but a
// sequence's first (8 threads each) and marks the tiles before one with a bad page.
constexpr int kPlanLds = 4096;
__global__ __launch_bounds__(1024) void paged_plan_kernel(PagedAttnParams p, int rows) {
  __shared__ int64_t lds[16];
  __shared__ int64_t before_s[kPlanLds];
  __shared__ PagedSeq seq_s[1024];
  __shared__ int64_t first_s[1024];                    // tiles before a sequence of the chunk
  __shared__ PlanTile tile_s[1024];                    // the first tiles
  __shared__ int bad_cu;
  if (threadIdx.x == 0) bad_cu = 0;
  __syncthreads();
  int64_t done = 0, units = 0;                          // tiles and units before this chunk of sequences
  for (int s0 = 0; s0 < p.c.B; s0 += 1024) {
    const int s = s0 + threadIdx.x, ns = p.c.B - s0 < 1024 ? p.c.B - s0 : 1024;
    int64_t nt = 0;
    PagedSeq q = {};
    if (s < p.c.B) {
      q = paged_seq(p.c, s);
      if (q.flags) paged_flag(p.c, q.flags);
      if (q.flags & LVSA_PAGED_BAD_CU) bad_cu = 1;
      nt = ((int64_t)q.n * p.group + rows - 1) / rows;
    }
    int64_t all;
    const int64_t at = block_scan(nt, ns, lds, &all);
    first_s[threadIdx.x] = at;
    seq_s[threadIdx.x] = q;
    __syncthreads();
    // row ranges that overlap (bad ones) give more tiles than the bound: the rest is dropped
    if (done + all > p.tiles) all = p.tiles - done;
    for (int64_t t0 = 0; t0 < all; t0 += 1024) {
      const int64_t t = t0 + threadIdx.x;
      PlanTile w = {};
      if (t < all) {
        int lo = 0, hi = ns - 1;                        // last sequence with first <= t
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (first_s[mid] <= t) lo = mid;
          else hi = mid - 1;
        }
        w.seq = s0 + lo;
        w.sq = seq_s[lo];
        w.r0 = (int)((t - first_s[lo]) * rows);
        w.blocks = tile_blocks(p, w.sq, w.r0, rows);
        w.units = w.blocks > 0 ? w.blocks : 1;
      }
      int64_t sum;
      const int64_t u = units + block_scan(w.units, all - t0 < 1024 ? (int)(all - t0) : 1024, lds, &sum);
      if (t < all) {
        p.plan_tiles[done + t] = w;
        p.before[done + t] = u;
        if (done + t < kPlanLds) before_s[done + t] = u;
        if (done + t < 1024) tile_s[done + t] = w;
      }
      units += sum;
    }
    done += all;
    __syncthreads();
  }
  const int tiles = (int)done;
  const int64_t U = units * p.c.Hkv;
  // none where the row ranges are bad: the launch then only spoils the result
  const int shares = bad_cu ? 0 : plan_shares(U, (int64_t)tiles * p.c.Hkv, p.grid);
  if (threadIdx.x == 0) *p.head = PlanHead{units, tiles, shares, bad_cu, 0};
  const bool in_lds = tiles <= kPlanLds;
  for (int w = threadIdx.x; w < shares; w += 1024) {
    const int64_t u = unit_start(U, shares, w + 1) - 1;
    const int64_t h = quotient(u, units), rest = u - h * units;
    int lo = 0, hi = tiles - 1;  // last tile with before <= rest
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((in_lds ? before_s[mid] : p.before[mid]) <= rest) lo = mid;
      else hi = mid - 1;
    }
    const int64_t b = in_lds ? before_s[lo] : p.before[lo];
    const PlanTile tile = lo < 1024 ? tile_s[lo] : p.plan_tiles[lo];
    const int blk = (int)(rest - b) + 1;
    p.ends[w] = PlanEnd{(int)h, lo, blk, 0};
    // a tile that shares divide is joined by the one it starts in
    PlanJoin j = {};
    const int64_t u0 = h * units + b;
    if (blk < tile.units && wg_of_unit(U, shares, u0) == w) {
      const DecodeSlots d = decode_slots(U, shares, u0, tile.units);
      const int left = tile.sq.n * p.group - tile.r0;
      j = PlanJoin{d.first, d.rest, d.count, (int)h, tile.r0, left < rows ? left : rows, tile.sq.t0, {0, 0, 0}};
    }
    p.joins[w] = j;
  }
  for (int i = (1023 - threadIdx.x) >> 3; p.causal && i < tiles; i += 128) {   // from the threads without shares on
    const PlanTile w = i < 1024 ? tile_s[i] : p.plan_tiles[i];
    const int left = w.sq.n * p.group - w.r0, r1 = w.r0 + (left < rows ? left : rows) - 1;
    const int k0 = key_limit(p, w.sq, w.r0), k1 = key_limit(p, w.sq, r1);
    if (w.r0 == 0 || k1 == 0) continue;
    const int32_t* table = p.c.table + w.seq * p.c.table_str;
    bool bad = false;
    for (int e = page_of(p.c, k0 > 0 ? k0 - 1 : 0) + (threadIdx.x & 7); e <= page_of(p.c, k1 - 1); e += 8)
      bad |= (uint32_t)table[e] >= (uint32_t)p.c.n_pages;
    for (int k = i - 1; bad && k >= 0 && p.plan_tiles[k].seq == w.seq; --k)
      p.plan_tiles[k].sq.flags = w.sq.flags | LVSA_PAGED_BAD_PAGE;
  }
}

// Joins the partials of the row tile that share blockIdx.x ends in, where the
// plan says so.  blockIdx.y: 32 rows of the tile.  A lane has four elements of
// a row and a wave R rows at a time, so that every partial is one 16-byte load
// per lane with the next ones in flight behind it: what bounds it is the bytes,
// 67 MB for a launch whose 256 shares all end inside a tile of 256 rows of 128 (16
// us; 9 us of head size 64).
template <int D, typename E>
__global__ __launch_bounds__(256) void paged_merge_tiles_kernel(PagedAttnParams p, int rows) {
  typedef float f4 __attribute__((ext_vector_type(4)));
  typedef E e4 __attribute__((ext_vector_type(4)));
  constexpr int LR = D / 4, R = 64 / LR;               // lanes per row, rows per wave
  if ((int)blockIdx.x >= p.head->shares) return;
  const PlanJoin j = p.joins[blockIdx.x];
  if (j.count == 0) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int sub = lane / LR, d = 4 * (lane % LR);
  if (sub >= R) return;
  constexpr int STEPS = 8 / R;
  float M[STEPS], l[STEPS];
  f4 o[STEPS];
  int r[STEPS];
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    r[k] = 32 * blockIdx.y + 8 * wave + R * k + sub;
    M[k] = kNoKeys;
    l[k] = 0.f;
    o[k] = f4{0.f, 0.f, 0.f, 0.f};
  }
  for (int i = 0; i < j.count; ++i) {
    const int64_t slot = (i == 0 ? j.first : j.rest + 2 * i) * rows;
    float m[STEPS], s[STEPS];
    f4 x[STEPS];
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      m[k] = p.ws_ml[2 * (slot + r[k])];
      s[k] = p.ws_ml[2 * (slot + r[k]) + 1];
      x[k] = *reinterpret_cast<const f4*>(p.ws_o + (slot + r[k]) * D + d);
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      const float top = __builtin_fmaxf(M[k], m[k]);
      const float a = __builtin_amdgcn_exp2f(M[k] - top), b = __builtin_amdgcn_exp2f(m[k] - top);
      l[k] = l[k] * a + s[k] * b;
      o[k] = o[k] * a + x[k] * b;
      M[k] = top;
    }
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    if (r[k] >= j.rows) continue;          // rows past the sequence's end: their slots hold nothing
    const int i = (j.r0 + r[k]) / p.group, hq = j.h * p.group + (j.r0 + r[k]) - i * p.group;
    const int64_t t = (int64_t)j.t0 + i;
    const float inv = l[k] == 0.f ? 0.f : 1.0f / l[k];
    *reinterpret_cast<e4*>(p.o + t * p.o_str[0] + hq * p.o_str[1] + 2 * d) =
        e4{(E)(o[k][0] * inv), (E)(o[k][1] * inv), (E)(o[k][2] * inv), (E)(o[k][3] * inv)};
    if (p.lse && d == 0)
      p.lse[t * p.H + hq] = l[k] == 0.f ? -__builtin_inff() : (M[k] + __log2f(l[k])) * 0.69314718055994530942f;
  }
}

// The status word, and 0 in its place: in one step, so that what a call of another
// stream finds meanwhile stays for the next taker.
__global__ void paged_take_status_kernel(int32_t* status, int32_t* found) { *found = atomicExch(status, 0); }

// ─────────────────────────────── host side ─────────────────────────────────

template <int D, typename E, int BITS> struct Append {
  static int go(const AppendParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)(p.c.N < kMaxGrid ? p.c.N : kMaxGrid) + 1);
    if (p.c.N <= kFewTokens * cu_count())
      hipLaunchKernelGGL((paged_append_kernel<D, E, BITS, 256>), grid, dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL((paged_append_kernel<D, E, BITS, 64>), grid, dim3(64), 0, stream, p);
    return launch_status("lvsa_paged_append");
  }
};
template <int D, typename E, int BITS> struct Gather {
  static int go(const PagedView& c, void* ko, void* vo, int max_len, hipStream_t stream) {
    const int64_t chunks = (int64_t)max_len * c.Hkv * (D / 8);
    const int64_t want = ceil_div(chunks, 256);
    const unsigned gx = (unsigned)(want < 4096 ? want : 4096);
    for (int64_t b0 = 0; b0 < c.B; b0 += kMaxGridY)
      hipLaunchKernelGGL((paged_gather_kernel<D, E, BITS>), dim3(gx, (unsigned)(c.B - b0 < kMaxGridY ? c.B - b0 : kMaxGridY), 2),
                         dim3(256), 0, stream, c, (char*)ko, (char*)vo, max_len, (int)b0);
    return launch_status("lvsa_paged_gather");
  }
};

// How an attention call runs: row tiles of 16 or 32 rows on the decode kernel
// or 128 or 256 on the prefill kernels, the work-groups that share its key
// blocks, and its workspace.
struct AttnShape {
  int rows, grid, tiles;
  int64_t o_elems, ml_elems, plan_bytes;
  int64_t bytes() const { return 4 * (o_elems + ml_elems) + plan_bytes; }
};
int64_t plan_offset(const AttnShape& s, int part) {
  const int64_t head = 64, tiles = head + (int64_t)s.tiles * sizeof(PlanTile),
                before = tiles + ((int64_t)s.tiles + 2) * 8, ends = before + (int64_t)s.grid * sizeof(PlanEnd),
                joins = ends + (int64_t)s.grid * sizeof(PlanJoin);
  const int64_t at[] = {0, head, tiles, before, ends, joins};
  return ceil_div(at[part], 16) * 16;
}

AttnShape attn_shape(const lvsa_paged_attn_args* a) {
  AttnShape s{};
  const int group = a->H / a->cache.Hkv, D = a->cache.D;
  const int64_t N = a->batch.N, cus = cu_count(), B = a->batch.B < N ? a->batch.B : N;
  const int64_t cap = (int64_t)a->batch.max_pages * a->cache.page_size;
  // unknown: single tokens where there are no more rows than sequences, else one sequence of all rows
  const int64_t q = a->max_q_len > 0 ? (a->max_q_len < N ? a->max_q_len : N) : N <= a->batch.B ? 1 : N;
  const int64_t tile_rows = q * group;
  // Rows of the tiles, from sequences of n rows over 8000 keys, 16 heads of 128
  // (us):                16 bits: n = 16   24   32   40     4 bits: 16   24   32   40
  //   decode, 16 rows           107  140  143                      43   62   66
  //   decode, 32 rows           106  110  114  143                 51   55   60   90
  //   prefill, 128 rows         124  124  124  127                 96   97   97   98
  // (head sizes 64 and 256 cross at the same places).  Above 128 rows, where a
  // tall tile's rows share twice the keys' copies: 160 rows 110 -> 98, 256 rows
  // 124 -> 106, 400 rows 180 -> 158 us; 96 rows 94 -> 94, of 64 56 -> 61 us.
  const int64_t kv = a->max_kv_len > 0 && a->max_kv_len < cap ? a->max_kv_len : cap;
  const int64_t steps = ceil_div(kv, paged_decode_keys(D)) * a->cache.Hkv;     // of a row tile
  const int64_t short_units = steps * (ceil_div(N * group, 32) + B);
  if (tile_rows <= 32 || N * a->H + 2 * short_units <= kPagedShort * cus) {
    s.rows = tile_rows <= 16 ? 16 : 32;
    const int64_t units = tile_rows <= 32 ? steps * B : short_units;
    const int64_t slots = cus * paged_decode_groups(D, a->cache.bits, s.rows);
    s.grid = (int)(units < slots ? (units > 0 ? units : 1) : slots);
  } else {
    s.rows = D <= 128 && tile_rows > kPagedTile ? kPagedTall : kPagedTile;
    s.tiles = (int)(ceil_div(N * group, s.rows) + B);
    const int64_t units = s.tiles * ceil_div(cap > 0 ? cap : 1, kPagedBlock) * a->cache.Hkv;
    // Two work-groups of 128 rows on a unit hide each other's waits, but where
    // there are fewer tiles than units most of a share's work is its partial: 4
    // sequences of 128 rows, 16 heads of 128, 8000 keys 98 -> 81 us with one, 16
    // of them 219 -> 241 (of 64: 58 -> 52 and 133 -> 161).
    const bool two = D <= 128 && s.rows == kPagedTile && (int64_t)s.tiles * a->cache.Hkv > cus;
    const int64_t slots = two ? 2 * cus : cus;
    // a multiple of the XCDs: see share_of
    s.grid = (int)(8 * ceil_div(units < slots ? units : slots, 8));
    s.plan_bytes = plan_offset(s, 5);
  }
  s.o_elems = 2LL * s.grid * s.rows * D;
  s.ml_elems = 2LL * 2 * s.grid * s.rows;
  return s;
}

template <int D, typename E, int BITS> struct MergeTiles {
  static int go(const PagedAttnParams& p, const AttnShape& s, hipStream_t stream) {
    hipLaunchKernelGGL((paged_merge_tiles_kernel<D, E>), dim3((unsigned)s.grid, (unsigned)(s.rows / 32)), dim3(256), 0, stream,
                       p, s.rows);
    return launch_status("lvsa_paged_attn_fwd");
  }
};

int attn_check(const lvsa_paged_attn_args* a, PagedView* v) {
  const char* what = "lvsa_paged_attn_fwd";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  const int rc = paged_view(what, &a->cache, &a->batch, true, v);
  if (rc) return rc;
  LVSA_REQUIRE(a->H >= 1 && a->H % a->cache.Hkv == 0, LVSA_ERR_INVALID_ARG, "%s: %d heads over %d key heads", what, a->H,
               a->cache.Hkv);
  LVSA_REQUIRE((int64_t)a->batch.N * a->H < (1LL << 31) - 4096, LVSA_ERR_UNSUPPORTED, "%s: %d rows of %d heads", what,
               a->batch.N, a->H);
  LVSA_REQUIRE(a->scale > 0.f && a->scale <= 2.0e38f, LVSA_ERR_INVALID_ARG, "%s: scale %g must be positive and at most 2e38",
               what, (double)a->scale);
  return LVSA_OK;
}

}  // namespace
}  // namespace lvsa

extern "C" {

int lvsa_paged_append(const lvsa_paged_append_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_append";
  LVSA_REQUIRE(a != nullptr, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  AppendParams p{};
  const int rc = paged_view(what, &a->cache, &a->batch, true, &p.c);
  if (rc) return rc;
  LVSA_REQUIRE(a->batch.N == 0 || (a->k && a->v), LVSA_ERR_INVALID_ARG, "%s: null keys or values", what);
  LVSA_REQUIRE((a->q == nullptr) == (a->q_out == nullptr), LVSA_ERR_INVALID_ARG, "%s: q and q_out go together", what);
  LVSA_REQUIRE(!a->q || a->H >= 1, LVSA_ERR_INVALID_ARG, "%s: %d query heads", what, a->H);
  LVSA_REQUIRE((a->cos == nullptr) == (a->sin == nullptr), LVSA_ERR_INVALID_ARG, "%s: cos and sin go together", what);
  LVSA_REQUIRE(!a->cos || (a->rot >= 16 && a->rot % 16 == 0 && a->rot <= a->cache.D && a->n_angles >= 0), LVSA_ERR_INVALID_ARG,
               "%s: %d rotated dimensions of %d (a multiple of 16), %d angle rows", what, a->rot, a->cache.D, a->n_angles);
  const void* ptrs[4] = {a->k, a->v, a->q, a->q_out};
  const int64_t* strs[4] = {a->k_str, a->v_str, a->q_str, a->qo_str};
  int64_t* outs[4] = {p.k_str, p.v_str, p.q_str, p.qo_str};
  for (int i = 0; i < 4; ++i) {
    if (!ptrs[i]) continue;
    outs[i][0] = 2 * strs[i][0];
    outs[i][1] = 2 * strs[i][1];
    LVSA_REQUIRE(aligned16((int64_t)(uintptr_t)ptrs[i]) && aligned16(outs[i][0]) && aligned16(outs[i][1]),
                 LVSA_ERR_INVALID_ARG, "%s: rows must start at multiples of 16 bytes", what);
  }
  if (a->batch.N == 0 || a->batch.B == 0) return LVSA_OK;
  // a half-split row's partners are read after other threads have written theirs
  const int heads[3] = {a->cache.Hkv, a->cache.Hkv, a->H};
  for (int i = 0; i < 3; ++i)
    LVSA_REQUIRE(!a->q || !share_memory(a->q_out, p.qo_str, a->H, ptrs[i], outs[i], heads[i], a->batch.N, a->cache.D),
                 LVSA_ERR_INVALID_ARG, "%s: q_out must not share memory with k, v and q", what);
  p.k = (const char*)a->k;
  p.v = (const char*)a->v;
  p.q = (const char*)a->q;
  p.qo = (char*)a->q_out;
  p.cos = a->cos;
  p.sin = a->sin;
  p.positions = a->positions;
  p.H = a->H;
  p.rot = a->cos ? a->rot : 0;
  p.interleaved = a->interleaved;
  p.n_angles = a->n_angles;
  return by_type<Append>(a->cache.D, a->cache.dtype, a->cache.bits, p, stream);
}

int lvsa_paged_take_status(int32_t* status, int32_t* found, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_take_status";
  LVSA_REQUIRE(status && found, LVSA_ERR_INVALID_ARG, "%s: null pointer", what);
  hipLaunchKernelGGL(paged_take_status_kernel, dim3(1), dim3(1), 0, stream, status, found);
  return launch_status(what);
}

int lvsa_paged_gather(const lvsa_paged_cache* cache, const lvsa_paged_batch* batch, void* k_out, void* v_out,
                      int32_t max_len, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_gather";
  LVSA_REQUIRE(cache && batch, LVSA_ERR_INVALID_ARG, "%s: null args", what);
  PagedView c{};
  const int rc = paged_view(what, cache, batch, false, &c);
  if (rc) return rc;
  LVSA_REQUIRE(max_len >= 0, LVSA_ERR_INVALID_ARG, "%s: %d tokens", what, max_len);
  if (batch->B == 0 || max_len == 0) return LVSA_OK;
  LVSA_REQUIRE(k_out && v_out && aligned16((int64_t)(uintptr_t)k_out) && aligned16((int64_t)(uintptr_t)v_out),
               LVSA_ERR_INVALID_ARG, "%s: outputs must be non-null and 16-byte aligned", what);
  return by_type<Gather>(cache->D, cache->dtype, cache->bits, c, k_out, v_out, max_len, stream);
}

int lvsa_paged_attn_workspace_query(const lvsa_paged_attn_args* a, int64_t* bytes) {
  clear_error();
  LVSA_REQUIRE(bytes != nullptr, LVSA_ERR_INVALID_ARG, "lvsa_paged_attn_workspace_query: null output");
  PagedView v{};
  const int rc = attn_check(a, &v);
  if (rc) return rc;
  const AttnShape s = attn_shape(a);
  *bytes = a->batch.N == 0 ? 0 : s.bytes();
  return LVSA_OK;
}

int lvsa_paged_attn_fwd(const lvsa_paged_attn_args* a, hipStream_t stream) {
  clear_error();
  const char* what = "lvsa_paged_attn_fwd";
  PagedAttnParams p{};
  int rc = attn_check(a, &p.c);
  if (rc) return rc;
  if (a->batch.N == 0) return LVSA_OK;
  LVSA_REQUIRE(a->q && a->o, LVSA_ERR_INVALID_ARG, "%s: null q or o", what);
  bool ok = aligned16((int64_t)(uintptr_t)a->q) && aligned16((int64_t)(uintptr_t)a->o);
  for (int i = 0; i < 2; ++i) {
    p.q_str[i] = 2 * a->q_str[i];
    p.o_str[i] = 2 * a->o_str[i];
    ok = ok && aligned16(p.q_str[i]) && aligned16(p.o_str[i]);
  }
  LVSA_REQUIRE(ok, LVSA_ERR_INVALID_ARG, "%s: rows must start at multiples of 16 bytes", what);
  const AttnShape s = attn_shape(a);
  const int64_t need = s.bytes();
  LVSA_REQUIRE(need == 0 || (a->workspace && aligned16((int64_t)(uintptr_t)a->workspace)), LVSA_ERR_INVALID_ARG,
               "%s: %lld bytes of 16-byte aligned workspace needed", what, (long long)need);
  LVSA_REQUIRE(need == 0 || a->workspace_bytes >= need, LVSA_ERR_CAPACITY, "%s: workspace of %lld bytes < %lld", what,
               (long long)a->workspace_bytes, (long long)need);
  LVSA_REQUIRE(!share_memory(a->o, p.o_str, a->H, a->q, p.q_str, a->H, a->batch.N, a->cache.D), LVSA_ERR_INVALID_ARG,
               "%s: o must not share memory with q", what);
  p.q = (const char*)a->q;
  p.o = (char*)a->o;
  p.lse = a->lse;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.H = a->H;
  p.group = a->H / a->cache.Hkv;
  p.causal = a->causal;
  p.short_rows = p.c.k_str[1] >= 0 && p.c.k_str[1] < (1 << 26) && p.c.v_str[1] >= 0 && p.c.v_str[1] < (1 << 26);
  p.fill_tail = a->fill_tail;
  p.grid = s.grid;
  p.tiles = s.tiles;
  char* ws = (char*)a->workspace;
  p.head = (PlanHead*)(ws + plan_offset(s, 0));
  p.plan_tiles = (PlanTile*)(ws + plan_offset(s, 1));
  p.before = (int64_t*)(ws + plan_offset(s, 2));
  p.ends = (PlanEnd*)(ws + plan_offset(s, 3));
  p.joins = (PlanJoin*)(ws + plan_offset(s, 4));
  p.ws_o = (float*)(ws + s.plan_bytes);
  p.ws_ml = p.ws_o + s.o_elems;
  const bool bf16 = a->cache.dtype == LVSA_BF16;
  if (a->batch.B > 0) {
    if (s.tiles > 0) {
      hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(1024), 0, stream, p, s.rows);
      rc = launch_status(what);
      if (rc) return rc;
    }
    switch (a->cache.D) {
      case 64: rc = paged_attn_d64(p, a->cache.bits, s.rows, bf16, stream); break;
      case 96: rc = paged_attn_d96(p, a->cache.bits, s.rows, bf16, stream); break;
      case 128: rc = paged_attn_d128(p, a->cache.bits, s.rows, bf16, stream); break;
      case 192: rc = paged_attn_d192(p, a->cache.bits, s.rows, bf16, stream); break;
      default: rc = paged_attn_d256(p, a->cache.bits, s.rows, bf16, stream); break;
    }
    if (rc) return rc;
  }
  if (s.tiles > 0 && a->batch.B > 0) {
    return by_type<MergeTiles>(a->cache.D, a->cache.dtype, 16, p, s, stream);
  }
  const int out_rows = a->batch.N * a->H;
  const dim3 grid((unsigned)(out_rows < kMaxGrid ? out_rows : kMaxGrid));
  const int keys = paged_decode_keys(a->cache.D);
  if (bf16) {
    hipLaunchKernelGGL((paged_merge_kernel<__bf16>), grid, dim3(256), 0, stream, p, a->cache.D, s.rows, keys);
  } else {
    hipLaunchKernelGGL((paged_merge_kernel<_Float16>), grid, dim3(256), 0, stream, p, a->cache.D, s.rows, keys);
  }
  return launch_status(what);
}

}  // extern "C"
