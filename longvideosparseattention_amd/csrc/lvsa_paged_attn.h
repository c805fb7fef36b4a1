// Attention over the paged key/value cache (gfx950): o = softmax(scale q K^T) V
// for the newest tokens of every sequence, 16-bit pages or 4-bit ones.  One
// unit per head size instantiates the kernels (lvsa_paged_d*.hip).
//
// The query heads of a key head are packed: row r of a (sequence, key head)
// pair is token r / group, head r % group of the group, so that a tile of rows
// reads each key and value once for all of them.
//
//   paged_decode_kernel   few rows (tiles of 16 or 32) and short chunks: bound by
//                         the bytes of the cache, or by latency.  Matrix
//                         instructions of 16 rows, each wave on keys of its own.
//   paged_prefill_kernel  tiles of 128 rows: bound by the matrix cores and the
//                         softmax.  Four waves of 32 rows share key blocks of
//                         64 in LDS.
//   paged_tall_kernel     tiles of 256 rows (head sizes up to 128): the same
//                         bound, eight waves on the same blocks.
// Which one runs follows from the sizes (attn_shape, lvsa_paged.hip).
//
// All form S^T = K Q^T, so that a lane owns one row's scores, and O^T += V^T
// P^T with P straight from S^T's registers: the order of the keys within a
// step is permuted alike on both operands.  V^T comes out of LDS by
// transposing reads.  P is rounded to the rows' 16-bit type, the nearest, since the
// matrix instructions take both operands alike; a row's sum is of the unrounded
// weights, in fp32.  In bf16 results are then off by 0.0018 to 0.0024 of their size
// (root mean square, against 64 bits) instead of the 0.0017 of their own rounding; what
// the rounding leaves off as a second operand would double the second product.
//
// LDS tiles of K and V, in 16-byte chunks (chunk c: elements 8c .. 8c + 7):
//   decode    16 keys: key r of chunk c at 256 c + 16 (r ^ 8 (c & 1)).  A lane
//             loads whole pieces of one key, so it looks one page up per tile.
//   prefill   8 keys (tile t of the matrix): 128 (c ^ (t & 1)) + 16 (r ^ 4 ((c >>
//             1) & 1)).  One copy instruction brings 128 bytes of each of 8
//             keys (16 keys x 64 bytes, as in decode, cost the L1 twice the
//             lookups and 100 of 800 us for 4680 tokens over 32760 keys).  Head
//             size 96, whose 12 chunks do not divide by 8, keeps 16 keys x 64
//             bytes with 4 (c & 3) in the place of 8 (c & 1).
// In each, what 16 lanes of a 16-byte read, or 32 of a transposing read (8 keys
// of two chunks in decode, 4 keys of four in prefill), take in one cycle covers
// the 64 banks once.
#pragma once
#include "lvsa_paged.h"

#include <type_traits>

namespace lvsa {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

// A row's weights are 2^(score - m), m its reference: the running maximum less a
// lift, and moved only when a score exceeds it by lift and rise, so that the usual
// step rescales nothing.  bf16 has fp32's range: no lift, weights up to 2^8.
// fp16's normal numbers reach from 2^-14 to 2^16: lifted by 9 with a rise of 6, a
// row's largest weight is 2^9 to 2^15, and weights down to 2^-23 of it keep all
// their bits (unlifted they were subnormal from 2^-14 of it on and 0 below 2^-25:
// the rest of a row beside keys with nearly all its weight, but values of 0, came
// out up to 20% off).  The rise costs rescaled steps: causal prompts of head size
// 64 in fp16 185.6 us with 8 (and a lift of 7), 187.3 with 6, 188.7 with 5, 190.9
// with 4.  Scores from 2^20 on, which fp32 holds to an eighth and worse, have no
// lift: half a step of theirs more would overflow from 2^24 on (2^27 without).
template <typename E>
struct Mat;
template <>
struct Mat<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExp = 0x7f80u;
  static constexpr bool kLifted = false;
  static constexpr uint32_t kFinite = 252;    // largest scale byte that leaves every 4-bit value finite: 6 * 2^125
  __device__ static floatx4 mfma16(shortx8 a, shortx8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static floatx4 mfma16(shortx4 a, shortx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  }
  __device__ static floatx16 mfma32(shortx8 a, shortx8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  template <int SEL>
  __device__ static uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
  }
};
template <>
struct Mat<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExp = 0x7c00u;
  static constexpr bool kLifted = true;
  static constexpr uint32_t kFinite = 140;    // 6 * 2^13
  __device__ static floatx4 mfma16(shortx8 a, shortx8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  __device__ static floatx4 mfma16(shortx4 a, shortx4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4, a), __builtin_bit_cast(v4, b), c, 0, 0, 0);
  }
  __device__ static floatx16 mfma32(shortx8 a, shortx8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  template <int SEL>
  __device__ static uint32_t decode(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
  }
};

constexpr float kFarScore = 1048576.f;
// A row's reference: m, and the score above which it moves.
template <typename E>
struct Reference {
  float m = kNoKeys;
  float above = kNoKeys;                  // kept in a register where the rise depends on the row
  __device__ __forceinline__ bool exceeded(float top) const { return Mat<E>::kLifted ? top > above : top > m + 8.0f; }
  // Moves to a block's largest score; returns the factor of what was summed so far.
  __device__ __forceinline__ float move(float top) {
    if constexpr (Mat<E>::kLifted) top -= __builtin_fabsf(top) < kFarScore ? 9.0f : 0.0f;
    const float next = __builtin_fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - next);
    m = next;
    if constexpr (Mat<E>::kLifted) above = m + (__builtin_fabsf(m) < kFarScore ? 15.0f : 8.0f);
    return alpha;
  }
};

// IEEE maximum: unlike fmaxf it needs no canonicalisation of matrix results first
// (764 instead of 770 us for 4680 tokens of 12 heads of 128 over 32760 keys, 184 instead of
// 187 us for causal prompts of head size 64).  A NaN score is NaN in the row's weights either way.
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

template <typename E>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, typename Mat<E>::v2{(E)a, (E)b});
}
template <typename E>
__device__ __forceinline__ shortx8 decode8(uint32_t codes, uint32_t scale_byte) {
  const float s = __builtin_bit_cast(float, scale_byte << 23);   // byte 255: an infinite scale, which decodes to NaN
  return __builtin_bit_cast(shortx8, u32x4{Mat<E>::template decode<0>(codes, s), Mat<E>::template decode<1>(codes, s),
                                           Mat<E>::template decode<2>(codes, s), Mat<E>::template decode<3>(codes, s)});
}

__device__ __forceinline__ int decode_chunk(int D, int r, int c) {
  return (r >> 4) * 32 * D + 256 * c + 16 * ((r & 15) ^ (8 * (c & 1)));
}
template <int D>
__device__ __forceinline__ int prefill_chunk(int r, int c) {
  if constexpr (D == 96) return (r >> 4) * 32 * D + 256 * c + 16 * ((r & 15) ^ (4 * (c & 3)));
  const int t = r >> 3;
  return t * 16 * D + 128 * (c ^ (t & 1)) + 16 * ((r & 7) ^ (4 * ((c >> 1) & 1)));
}

// Four keys (rows of the tile) x 16 elements of V, transposed: the lane's
// element of four consecutive keys.  `at`: byte offset of the lane's own 8
// bytes of the 4 x 16 patch its group of 16 lanes reads.
__device__ __forceinline__ shortx4 read_tr(const lds_char* at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)at);
}

// Whether any of eight 16-bit values is an infinity or NaN.
template <typename E>
__device__ __forceinline__ bool any_nonfinite(shortx8 x) {
  const u32x4 u = __builtin_bit_cast(u32x4, x);
  bool r = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r |= (u[i] & Mat<E>::kExp) == Mat<E>::kExp || ((u[i] >> 16) & Mat<E>::kExp) == Mat<E>::kExp;
  return r;
}

// Infinities and NaN among the values of keys that only some rows attend: the
// zero weight of a row that does not attend the key would carry them into it
// (0 * inf is NaN).  Blocks with masked keys are searched for such values on
// their way into LDS, and the matrix product runs on zeros in their place
// (finite8).  Where any were found, they are added at the end, from memory, to
// the rows that attend them (add_nonfinite): no sum of finite terms changes an
// infinity or a NaN, so the order does not matter.  4-bit values count as the
// 16-bit numbers they are decoded to: infinities too where a caller's scale
// takes them past the type's range.
template <typename E>
__device__ __forceinline__ shortx8 finite8(shortx8 x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = ((uint16_t)x[i] & Mat<E>::kExp) == Mat<E>::kExp ? (short)0 : x[i];
  return x;
}
template <typename E>
__device__ __forceinline__ float add_nonfinite(float o, uint32_t bits, bool seen) {
  const float v = (float)__builtin_bit_cast(E, (uint16_t)bits);
  return seen && (bits & Mat<E>::kExp) == Mat<E>::kExp ? o + v : o;
}

// Adds what keys [k0, k1) hold besides finite numbers to a row that attends
// keys below `lim`: quad q of the row's elements, d0 + q * step .. + 3, in
// o(q).  Rare, and slow: a key at a time.
template <typename E, int BITS, int NQ, typename Keys, typename O>
__device__ __forceinline__ void add_nonfinite_keys(const PagedView& c, const Keys& keys, int h, int k0, int k1,
                                                   int lim, int d0, int step, O o) {
#pragma unroll 1
  for (int k = k0; k < k1; ++k) {
    const PagedRow at = keys.row(k, keys.page(k));
    const char* row = c.v + at.page * c.v_str[0] + at.slot * c.v_str[1] + h * c.v_str[2];
    const bool seen = k < lim;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int d = d0 + q * step;
      u32x2 v;
      if constexpr (BITS == 16) {
        v = *reinterpret_cast<const u32x2*>(row + 2 * d);
      } else {
        const uint32_t codes = *reinterpret_cast<const uint16_t*>(row + d / 2);
        const uint32_t sb = c.vs[at.page * c.vs_str[0] + at.slot * c.vs_str[1] + h * c.vs_str[2] + d / 32];
        const float s = __builtin_bit_cast(float, sb << 23);
        v = u32x2{Mat<E>::template decode<0>(codes, s), Mat<E>::template decode<1>(codes, s)};
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) o(q, r, (v[r >> 1] >> (16 * (r & 1))) & 0xffffu, seen);
    }
  }
}

// The keys that a tile of rows walks, numbered from 0 to L - 1: all of a
// sequence's by position, each looked up in the page table ...
struct PagedKeys {
  static constexpr bool kStaged = false;      // looked up and checked before; there may be none
  const PagedView& c;
  const int32_t* table;
  int L;
  __device__ __forceinline__ int page(int k) const { return table[page_of(c, k)]; }
  __device__ __forceinline__ PagedRow row(int k, int page) const { return paged_row(c, k, page); }
  // Whether `n` keys from k on lie in slots one after the other, from `slot`.
  __device__ __forceinline__ bool together(int k, int n, int* slot) const {
    *slot = k - page_of(c, k) * c.page_size;
    return k + n <= L && *slot + n <= c.page_size;
  }
  __device__ __forceinline__ int limit(int lim) const { return lim; }       // keys below position `lim`
};

// Row r of a (sequence, key head) pair: its token and query head.
struct RowRef {
  int64_t tok;
  int head;
};
__device__ __forceinline__ RowRef row_ref(const PagedAttnParams& p, const PagedSeq& s, int h, int r) {
  const int i = r / p.group;
  return RowRef{(int64_t)s.t0 + i, h * p.group + (r - i * p.group)};
}
// ─────────────────────────────── decode ────────────────────────────────────

// Keys and values of one step of a wave, on their way from memory: T tiles of
// 16 keys.  16 bits: lane (g = lane / 16, x = lane % 16) holds chunks 4 i + g
// of key x, which is also the K operand of its matrix instruction.  4 bits:
// elements [g D / 4, (g + 1) D / 4) of key x and the scales of the first and
// the last of them; step i of the matrix products then takes elements g D / 4
// + 8 i .. + 7, and Q is held in the same order.
template <int D, int BITS, int T>
struct Step {
  u32x4 k[T][D / 32], v[T][D / 32];
};
template <int D, int T>
struct Step<D, 4, T> {
  uint32_t k[T][D / 32], v[T][D / 32];
  uint32_t ks[T][2], vs[T][2];
};

// What a work-group does next: key steps [blk0, blk1) of the rows [r0, r0 + ROWS)
// before row nrows of sequence sq and key head h; into the result where that is the
// rows' whole work, else to partial `slot`.  bad: the rows come out as NaN.
struct DecodePart {
  PagedSeq sq;
  int h, r0, nrows, blk0, blk1;
  int64_t slot;
  bool whole, bad;
};

// A part, with the keys that `keys` names; behind it the work-group may go on to another one.
template <int D, typename E, int BITS, int NT, typename Keys>
__device__ __forceinline__ void decode_part(const PagedAttnParams& p, const DecodePart& part, const Keys& keys) {
  constexpr int T = D >= 192 ? 1 : 2;          // 16-key tiles per wave and step
  constexpr int KW = 16 * T, KEYS = 4 * KW;    // keys per wave, per work-group
  static_assert(KEYS == paged_decode_keys(D), "merge and kernel count key steps alike");
  constexpr int ND = D / 32, NO = D / 16, ROWS = 16 * NT;
  constexpr int TB = 32 * D;                   // bytes of a 16-key tile
  constexpr int OP = D + 4;                    // row pitch of the exchanged O
  constexpr bool kTwoScales = D == 96 || D >= 192;
  constexpr int kVBytes = 4 * T * TB, kOBytes = 4 * 16 * OP * 4;
  __shared__ __attribute__((aligned(1024))) char smem_raw[kVBytes > kOBytes ? kVBytes : kOBytes];
  __shared__ float m_s[4][16], l_s[4][16];
  __shared__ int bad_s;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, x = lane & 15;
  lds_char* vbuf = (lds_char*)smem_raw + wave * (T * TB);
  float* obuf = reinterpret_cast<float*>(smem_raw);
  const PagedSeq& sq = part.sq;
  const int h = part.h, r0 = part.r0, nrows = part.nrows, blk0 = part.blk0, blk1 = part.blk1;
  const int64_t slot = part.slot;
  const bool whole = part.whole;

  // Q of the tile, in the order of the keys' elements; rows past the end
  // repeat the last one.
  shortx8 qf[NT][ND];
  int lim[NT];
  int lim_min = keys.L;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 16 * n + x < nrows ? r0 + 16 * n + x : nrows - 1;
    const RowRef ref = row_ref(p, sq, h, r);
    const char* qp = p.q + ref.tok * p.q_str[0] + ref.head * p.q_str[1];
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const int d = BITS == 16 ? 32 * i + 8 * g : (D / 4) * g + 8 * i;
      qf[n][i] = *reinterpret_cast<const shortx8*>(qp + 2 * d);
    }
    lim[n] = keys.limit(key_limit(p, sq, r));
  }
  {
    const int first = keys.limit(key_limit(p, sq, r0));
    lim_min = first < lim_min ? first : lim_min;
  }

  floatx4 o[NT][NO];
  Reference<E> ref_run[NT];
  float l_run[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l_run[n] = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i) o[n][i] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  bool bad = part.bad, odd_keys = false;

  const char* kbase = p.c.k + h * p.c.k_str[2];
  const char* vbase = p.c.v + h * p.c.v_str[2];
  const uint8_t* ksbase = BITS == 4 ? p.c.ks + h * p.c.ks_str[2] : nullptr;
  const uint8_t* vsbase = BITS == 4 ? p.c.vs + h * p.c.vs_str[2] : nullptr;

  // Key x of tile j of step b (past the end: the last key).
  auto key_pos = [&](int b, int j) __attribute__((always_inline)) {
    return key_within(b * KEYS + wave * KW + 16 * j + x, keys.L);
  };
  auto load_pages = [&](int b, int* page) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < T; ++j) page[j] = keys.page(key_pos(b, j));
  };
  auto load = [&](int b, const int* page, Step<D, BITS, T>& st) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const PagedRow at = keys.row(key_pos(b, j), page[j]);
      bad |= !at.ok;
      const char* kr = kbase + at.page * p.c.k_str[0] + at.slot * p.c.k_str[1];
      const char* vr = vbase + at.page * p.c.v_str[0] + at.slot * p.c.v_str[1];
      if constexpr (BITS == 16) {
#pragma unroll
        for (int i = 0; i < ND; ++i) st.k[j][i] = *reinterpret_cast<const u32x4*>(kr + 64 * i + 16 * g);
#pragma unroll
        for (int i = 0; i < ND; ++i) st.v[j][i] = *reinterpret_cast<const u32x4*>(vr + 64 * i + 16 * g);
      } else {
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(kr + (D / 8) * g);
        const uint32_t* vw = reinterpret_cast<const uint32_t*>(vr + (D / 8) * g);
#pragma unroll
        for (int i = 0; i < ND; ++i) st.k[j][i] = kw[i];
#pragma unroll
        for (int i = 0; i < ND; ++i) st.v[j][i] = vw[i];
        const uint8_t* ksr = ksbase + at.page * p.c.ks_str[0] + at.slot * p.c.ks_str[1];
        const uint8_t* vsr = vsbase + at.page * p.c.vs_str[0] + at.slot * p.c.vs_str[1];
        const int lo = (D / 4) * g / 32, hi = ((D / 4) * g + D / 4 - 1) / 32;
        st.ks[j][0] = ksr[lo];
        st.vs[j][0] = vsr[lo];
        st.ks[j][1] = kTwoScales ? ksr[hi] : 0;
        st.vs[j][1] = kTwoScales ? vsr[hi] : 0;
      }
    }
  };
  // Elements of step i of a lane's piece, in the scale that covers them.
  auto scale_of = [&](const uint32_t* s, int i) __attribute__((always_inline)) {
    if constexpr (!kTwoScales) return s[0];
    return ((D / 4) * g + 8 * i) / 32 == (D / 4) * g / 32 ? s[0] : s[1];
  };

  auto compute = [&](int b, Step<D, BITS, T>& st) __attribute__((always_inline)) {
    const int key0 = b * KEYS + wave * KW;
    if (key0 >= keys.L) return;                // the last step's waves past the end
    // V to LDS, chunk by chunk
    const bool masked = key0 + KW > lim_min;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        shortx8 w;
        int c;
        if constexpr (BITS == 16) {
          w = __builtin_bit_cast(shortx8, st.v[j][i]);
          c = 4 * i + g;
        } else {
          w = decode8<E>(st.v[j][i], scale_of(st.vs[j], i));
          c = ND * g + i;
        }
        if (masked) {
          odd |= any_nonfinite<E>(w);
          w = finite8<E>(w);
        }
        *reinterpret_cast<__attribute__((address_space(3))) shortx8*>(vbuf + decode_chunk(D, 16 * j + x, c)) = w;
      }
    if (masked) odd_keys |= odd;
    // S^T: row 4 g + r of tile j, column x
    floatx4 s[NT][T];
#pragma unroll
    for (int j = 0; j < T; ++j) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        shortx8 kf;
        if constexpr (BITS == 16) kf = __builtin_bit_cast(shortx8, st.k[j][i]);
        else kf = decode8<E>(st.k[j][i], scale_of(st.ks[j], i));
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][j] = Mat<E>::mfma16(kf, qf[n][i], s[n][j]);
      }
    }
    typedef short vp __attribute__((ext_vector_type(4 * T)));
    vp pb[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (masked) {
#pragma unroll
        for (int j = 0; j < T; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool seen = key0 + 16 * j + 4 * g + r < lim[n];
            s[n][j][r] = seen ? s[n][j][r] : -__builtin_inff();
          }
      }
      float top = __builtin_fmaxf(__builtin_fmaxf(s[n][0][0], s[n][0][1]), __builtin_fmaxf(s[n][0][2], s[n][0][3]));
      if constexpr (T == 2)
        top = __builtin_fmaxf(top, __builtin_fmaxf(__builtin_fmaxf(s[n][1][0], s[n][1][1]),
                                                   __builtin_fmaxf(s[n][1][2], s[n][1][3])));
      top *= p.scale_log2;
      if (__builtin_amdgcn_ballot_w64(ref_run[n].exceeded(top))) {
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float alpha = ref_run[n].move(top);
        l_run[n] *= alpha;
#pragma unroll
        for (int i = 0; i < NO; ++i) o[n][i] *= alpha;
      }
      uint32_t w[2 * T];
#pragma unroll
      for (int j = 0; j < T; ++j) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j][r], p.scale_log2, -ref_run[n].m));
          l_run[n] += e[r];
        }
        w[2 * j] = pack2<E>(e[0], e[1]);
        w[2 * j + 1] = pack2<E>(e[2], e[3]);
      }
      if constexpr (T == 2) pb[n] = __builtin_bit_cast(vp, u32x4{w[0], w[1], w[2], w[3]});
      else pb[n] = __builtin_bit_cast(vp, u32x2{w[0], w[1]});
    }
    // O^T: row (element) 16 i + 4 g + r, column (query row) x
    const int half = x & 3, row = 4 * g + (x >> 2);
    auto vfrag = [&](int i) __attribute__((always_inline)) {
      const int c = 2 * i + (half >> 1);
      vp a;
      const shortx4 a0 = read_tr(vbuf + decode_chunk(D, row, c) + 8 * (half & 1));
      if constexpr (T == 2) {
        const shortx4 a1 = read_tr(vbuf + decode_chunk(D, 16 + row, c) + 8 * (half & 1));
        a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        a = a0;
      }
      return a;
    };
#pragma unroll
    for (int i = 0; i < NO; ++i) {
      const vp a = vfrag(i);
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n][i] = Mat<E>::mfma16(a, pb[n], o[n][i]);
    }
  };

  // Two steps in flight: while one is computed the next one's rows are on
  // their way, and the page numbers of the one after that.
  if (!Keys::kStaged || blk0 < blk1) {
    Step<D, BITS, T> sa, sb;
    int page[T];
    load_pages(blk0, page);
    load(blk0, page, sa);
    load_pages(blk0 + 1, page);
    for (int b = blk0; b < blk1; b += 2) {
      if (b + 1 < blk1) {
        load(b + 1, page, sb);
        load_pages(b + 2, page);
      }
      __builtin_amdgcn_sched_barrier(0);
      compute(b, sa);
      if (b + 1 < blk1) {
        if (b + 2 < blk1) {
          load(b + 2, page, sa);
          load_pages(b + 3, page);
        }
        __builtin_amdgcn_sched_barrier(0);
        compute(b + 1, sb);
      }
    }
  }

  if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd_keys) != 0, 0)) {
    const int from = lim_min / KEYS > blk0 ? lim_min / KEYS : blk0;
    for (int b = from; b < blk1; ++b) {
      const int k0 = b * KEYS + wave * KW, k1 = k0 + KW < keys.L ? k0 + KW : keys.L;
      if (k0 + KW <= lim_min) continue;             // not masked: its values are in the sums already
#pragma unroll
      for (int n = 0; n < NT; ++n)
        add_nonfinite_keys<E, BITS, NO>(p.c, keys, h, k0, k1, lim[n], 4 * g, 16,
                                        [&](int q, int r, uint32_t v, bool seen) __attribute__((always_inline)) {
                                          o[n][q][r] = add_nonfinite<E>(o[n][q][r], v, seen);
                                        });
    }
  }

  // Join the four waves: rows' sums over the lanes, then maxima, sums and O
  // through LDS, in the order of the waves.
  if (threadIdx.x == 0) bad_s = 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float l = l_run[n];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();                         // V tiles (and the last tile's exchange) have been read
    if (g == 0) m_s[wave][x] = ref_run[n].m;
    if (n == 0 && __builtin_amdgcn_ballot_w64(bad) && lane == 0) bad_s = 1;
    __syncthreads();
    const float M = __builtin_fmaxf(__builtin_fmaxf(m_s[0][x], m_s[1][x]), __builtin_fmaxf(m_s[2][x], m_s[3][x]));
    const float w = __builtin_amdgcn_exp2f(ref_run[n].m - M);
    if (g == 0) l_s[wave][x] = l * w;
#pragma unroll
    for (int i = 0; i < NO; ++i)
      *reinterpret_cast<floatx4*>(obuf + (wave * 16 + x) * OP + 16 * i + 4 * g) = o[n][i] * w;
    __syncthreads();
    // thread: row tr, elements of every 16th quad
    const int tr = threadIdx.x >> 4, td = threadIdx.x & 15;
    const int r = r0 + 16 * n + tr;
    const float Mr = __builtin_fmaxf(__builtin_fmaxf(m_s[0][tr], m_s[1][tr]), __builtin_fmaxf(m_s[2][tr], m_s[3][tr]));
    float lr = (l_s[0][tr] + l_s[1][tr]) + (l_s[2][tr] + l_s[3][tr]);
    if (bad_s) lr = __builtin_nanf("");
    if (r < nrows) {
      const float inv = lr == 0.f ? 0.f : 1.0f / lr;
      const RowRef ref = row_ref(p, sq, h, r);
      char* op = p.o + ref.tok * p.o_str[0] + ref.head * p.o_str[1];
      float* wo = whole ? nullptr : p.ws_o + (slot * ROWS + 16 * n + tr) * D;
      for (int d = 4 * td; d < D; d += 64) {
        floatx4 a = *reinterpret_cast<const floatx4*>(obuf + tr * OP + d);
#pragma unroll
        for (int k = 1; k < 4; ++k) a += *reinterpret_cast<const floatx4*>(obuf + (k * 16 + tr) * OP + d);
        if (whole) {
          *reinterpret_cast<u32x2*>(op + 2 * d) = u32x2{pack2<E>(a[0] * inv, a[1] * inv), pack2<E>(a[2] * inv, a[3] * inv)};
        } else {
          *reinterpret_cast<floatx4*>(wo + d) = a;
        }
      }
      if (td == 0) {
        if (!whole) {
          float* ml = p.ws_ml + 2 * (slot * ROWS + 16 * n + tr);
          ml[0] = Mr;
          ml[1] = lr;
        } else if (p.lse) {
          p.lse[ref.tok * p.H + ref.head] =
              lr == 0.f ? -__builtin_inff() : (Mr + __log2f(lr)) * 0.69314718055994530942f;
        }
      }
    }
  }
  if (!Keys::kStaged && bad_s && threadIdx.x == 0 && !(sq.flags & LVSA_PAGED_BAD_LENGTH)) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
  __syncthreads();                           // the exchange has been read: V tiles and bad_s may be written
}

// Bound by the bytes: 45 sequences of up to 16000 keys, 32 heads over 8 of 128, in
// 16 bits at 5.7 TB/s (329 us), 40 of up to 32000 in 4 bits at 4.9 TB/s (154 us;
// there the decoding of codes on the vector units takes as long as the bytes).  A
// single sequence of 1001 keys takes 8 us, all of it trips to memory one after
// the other, and its merge 5 us.
//
// The launch's work, sum over sequences of row tiles x key heads x key steps,
// is cut into `grid` equal shares, so that ragged batches keep every
// work-group busy to the end and a single long sequence is spread over all of
// them.  A share may end inside a (row tile, head): its partial sums go to one
// of two slots of the work-group and paged_merge_kernel joins them.  The
// share's bounds follow from the lengths alone, so the merge finds the slots
// without a word from this kernel.
//
// Launch bounds: the registers of the work-groups that are to be on a unit at
// once; of the large heads those fit without being asked for, and asking spoils
// the schedule (D = 256, 4 bits: 275 instead of 215 us for 40 sequences of 12000).
template <int D, typename E, int BITS, int NT>
__global__ __launch_bounds__(256, D == 256 || (D == 192 && NT == 2) ? 1 : paged_decode_groups(D, BITS, 16 * NT)) void paged_decode_kernel(PagedAttnParams p) {
  constexpr int ROWS = 16 * NT, KEYS = paged_decode_keys(D);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);

  // The share [u, u_end) and the sequence it starts in.  A lane holds one
  // sequence, so that a batch of up to 64 is read once.
  const int B = p.c.B;
  PagedSeq mine = {};
  int64_t n_mine = 0, upto = 0;                // units of the lane's sequence; with those before it
  int64_t U = 0;
  int flags = 0;
  auto read_batch = [&](int s0) __attribute__((always_inline)) {
    n_mine = 0;
    if (s0 + lane < B) {
      mine = paged_seq(p.c, s0 + lane);
      n_mine = decode_units(p, mine, ROWS, KEYS);
      flags |= mine.flags;
    }
    upto = wave_scan(n_mine, lane, B - s0);
  };
  for (int s0 = 0; s0 < B; s0 += 64) {
    read_batch(s0);
    U += from_lane(upto, B - s0 < 64 ? B - s0 - 1 : 63);
  }
  if (blockIdx.x == 0 && wave == 0 && flags) paged_flag(p.c, flags);
  if (U == 0 || __builtin_amdgcn_ballot_w64(flags & LVSA_PAGED_BAD_CU)) return;   // bad row ranges: the merge spoils all rows
  const int shares = unit_shares(U, p.grid);
  if ((int)blockIdx.x >= shares) return;
  int64_t u = unit_start(U, shares, blockIdx.x);
  const int64_t u_end = unit_start(U, shares, blockIdx.x + 1);
  int seq = 0, held = 0;                       // lanes hold sequences [held, held + 64)
  int64_t base = 0;                            // units before sequence `seq`
  for (int s0 = 0; s0 < B; s0 += 64) {
    if (B > 64) read_batch(s0);
    held = s0;
    const uint64_t above = __builtin_amdgcn_ballot_w64(s0 + lane < B && base + upto > u);
    if (above) {
      const int at = __builtin_ctzll(above);
      seq = s0 + at;
      base += from_lane(upto - n_mine, at);
      break;
    }
    base += from_lane(upto, 63);
  }

  const int64_t u_first = u;
  while (u < u_end && seq < B) {
    if (seq >= held + 64) read_batch(held += 64);
    const PagedSeq sq = from_lane(mine, seq - held);
    const int64_t units = decode_units(p, sq, ROWS, KEYS);
    if (u >= base + units) {
      base += units;
      ++seq;
      continue;
    }
    const int nb = (int)(((int64_t)sq.L + KEYS - 1) / KEYS);
    const int64_t run = quotient(u - base, nb);
    const int blk0 = (int)((u - base) - run * nb);
    const int64_t left = u_end - u;
    const int blk1 = left < nb - blk0 ? blk0 + (int)left : nb;
    const int rt = (int)quotient(run, p.c.Hkv), h = (int)(run - (int64_t)rt * p.c.Hkv);
    const DecodePart part = {sq, h, rt * ROWS, sq.n * p.group, blk0, blk1,
                             2 * (int64_t)blockIdx.x + (u_first < u - blk0 ? 1 : 0),   // see decode_slots
                             blk0 == 0 && blk1 == nb, (sq.flags & LVSA_PAGED_BAD_LENGTH) != 0};
    decode_part<D, E, BITS, NT>(p, part, PagedKeys{p.c, p.c.table + seq * p.c.table_str, sq.L});
    u += blk1 - blk0;
  }
}

// ─────────────────────────────── prefill ───────────────────────────────────

// Rows before the first and behind the last sequence: 0 (fill_tail 1) and -inf.
__device__ __forceinline__ void fill_tail_rows(const PagedAttnParams& p, int D, int lane, int wave, int waves) {
  const int head = p.c.cu[0] < 0 ? 0 : p.c.cu[0] > p.c.N ? p.c.N : p.c.cu[0];
  const int tail = p.c.cu[p.c.B] < head ? head : p.c.cu[p.c.B] > p.c.N ? p.c.N : p.c.cu[p.c.B];
  const int64_t n = (int64_t)(head + p.c.N - tail) * p.H;
  const int64_t wg = blockIdx.x, wgs = gridDim.x;
  for (int64_t i = wg * waves + wave; i < n; i += waves * wgs) {
    const int64_t r = i / p.H, hq = i - r * p.H, t = r < head ? r : tail + (r - head);
    if (p.fill_tail == 1)
      for (int d = lane; d < D; d += 64) reinterpret_cast<uint16_t*>(p.o + t * p.o_str[0] + hq * p.o_str[1])[d] = 0;
    if (p.lse && lane == 0) p.lse[t * p.H + hq] = -__builtin_inff();
  }
}

// All rows of a batch whose row ranges are bad: NaN.
template <typename E>
__device__ __forceinline__ void spoil_rows(const PagedAttnParams& p, int D, int lane, int wave, int waves) {
  const int64_t n = (int64_t)p.c.N * p.H;
  for (int64_t i = (int64_t)blockIdx.x * waves + wave; i < n; i += (int64_t)waves * gridDim.x) {
    const int64_t t = i / p.H, hq = i - t * p.H;
    for (int d = lane; d < D; d += 64) reinterpret_cast<E*>(p.o + t * p.o_str[0] + hq * p.o_str[1])[d] = (E)__builtin_nanf("");
    if (p.lse && lane == 0) p.lse[i] = __builtin_nanf("");
  }
}

// A row's result, or its partial sums where shares divide its tile: O of
// element 32 dt + 8 q + 4 half + i in o[dt][4 q + i].
template <int D, typename E>
__device__ __forceinline__ void store_rows(const PagedAttnParams& p, bool whole, int64_t slot, int rows, int r, int half,
                                           const RowRef& ref, const floatx16* o, float m_run, float l) {
  if (!whole) {
    const int64_t at = slot * rows + r;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<floatx4*>(p.ws_o + at * D + 32 * dt + 8 * q + 4 * half) =
            floatx4{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
    if (half == 0) {
      p.ws_ml[2 * at] = m_run;
      p.ws_ml[2 * at + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  char* op = p.o + ref.tok * p.o_str[0] + ref.head * p.o_str[1];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<u32x2*>(op + 2 * (32 * dt + 8 * q + 4 * half)) =
          u32x2{pack2<E>(o[dt][4 * q] * inv, o[dt][4 * q + 1] * inv), pack2<E>(o[dt][4 * q + 2] * inv, o[dt][4 * q + 3] * inv)};
  if (p.lse && half == 0)
    p.lse[ref.tok * p.H + ref.head] = l == 0.f ? -__builtin_inff() : (m_run + __log2f(l)) * 0.69314718055994530942f;
}

// 16 bytes per lane, global -> LDS at `l` + 16 * lane, past the registers.  In
// asm, so that the compiler does not wait for it before LDS reads it cannot
// tell apart; the kernel orders the copies by its own wait and barrier.
__device__ __forceinline__ void copy16(const char* from, const lds_char* l) {
  const uint32_t la = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)l);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(la) : "m0", "memory");
#pragma clang diagnostic pop
}

// The same from a uniform base and a 32-bit offset per lane.
__device__ __forceinline__ void copy16(const char* base, uint32_t off, const lds_char* l) {
  const uint32_t la = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)l);
  const uint64_t b = (uint64_t)base;
  const uint64_t sb = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32)) << 32) |
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(sb), "s"(la) : "m0", "memory");
#pragma clang diagnostic pop
}

// How a wave copies its 16 keys of a 64-key matrix: instruction i of lane l
// brings chunk(i) of key key(i), counted in the tile, to 16 l behind 1024 i.
template <int D>
struct CopyMap {
  static constexpr int N = D / 32;                  // instructions
  int lane;
  __device__ __forceinline__ int key(int i) const {
    if constexpr (D == 96) return (lane & 15) ^ (4 * (lane >> 4));
    return ((lane & 7) ^ (4 * ((lane >> 4) & 1))) + 8 * (i / (D / 64));
  }
  __device__ __forceinline__ int chunk(int i) const {
    if constexpr (D == 96) return 4 * i + (lane >> 4);
    return 8 * (i % (D / 64)) + ((lane >> 3) ^ (i / (D / 64)));
  }
};

// Puts zeros in the place of what a wave's own tile of V holds besides finite
// numbers; whether there was any.
template <typename E>
__device__ __forceinline__ bool search_tile(lds_char* tile, int bytes, int lane) {
  typedef __attribute__((address_space(3))) shortx8 lds8;
  bool odd = false;
#pragma unroll 1
  for (int at = 16 * lane; at < bytes; at += 1024) odd |= any_nonfinite<E>(*reinterpret_cast<const lds8*>(tile + at));
  if (!__builtin_amdgcn_ballot_w64(odd)) return false;
#pragma unroll 1
  for (int at = 16 * lane; at < bytes; at += 1024)
    *reinterpret_cast<lds8*>(tile + at) = finite8<E>(*reinterpret_cast<const lds8*>(tile + at));
  return true;
}

// Workgroup barrier that nothing crosses: the memory clobber orders LDS and
// global accesses, the scheduling barriers keep a phase's arithmetic in it.
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// Materialise x here, so that the compiler does not sink its computation into
// the phase that uses it.
template <typename T>
__device__ __forceinline__ void keep(T& x) {
  asm volatile("" : "+v"(x));
}
template <int N>
__device__ __forceinline__ void wait_copies() {
  static_assert(N >= 0 && N < 16, "vmcnt immediate");
  __builtin_amdgcn_s_waitcnt(0x0F70 | N);
}
// Rows [r0, r0 + 128) before row nrows of sequence sq and key head h over key blocks
// [blk0, blk1), with the keys that `keys` names; see DecodePart.
template <int D, typename E, int BITS, typename Keys>
__device__ __forceinline__ void prefill_part(const PagedAttnParams& p, const DecodePart& part, const Keys& keys) {
  constexpr int ND = D / 32, NK = D / 16, NO = D / 32;
  constexpr int TB = 32 * D, MAT = 4 * TB;           // 16-key tile, 64-key matrix
  constexpr bool kTwoScales = D == 96 || D >= 192;
  __shared__ __attribute__((aligned(1024))) char smem_raw[4 * MAT];   // K of even and odd blocks, V of them
  __shared__ int bad_s, odd_s;
  lds_char* smem = (lds_char*)smem_raw;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, i32 = lane & 31;       // S^T: column (row of the tile) i32
  const int g = lane >> 4, x = lane & 15;

  const PagedSeq& sq = part.sq;
  const int h = part.h, r0 = part.r0, nrows = part.nrows, blk0 = part.blk0, blk1 = part.blk1;
  const int64_t slot = part.slot;
  const bool whole = part.whole;
  const int r_last = r0 + kPagedTile < nrows ? r0 + kPagedTile - 1 : nrows - 1;
  const int lim_min = keys.limit(key_limit(p, sq, r0)), lim_max = keys.limit(key_limit(p, sq, r_last));

  const int row = r0 + 32 * wave + i32;             // this lane's row of the pair
  const int rc = row < nrows ? row : nrows - 1;
  const RowRef ref = row_ref(p, sq, h, rc);
  const int lim = keys.limit(key_limit(p, sq, rc));
  shortx8 qf[NK];
  {
    const char* qp = p.q + ref.tok * p.q_str[0] + ref.head * p.q_str[1] + 16 * half;
#pragma unroll
    for (int c = 0; c < NK; ++c) qf[c] = *reinterpret_cast<const shortx8*>(qp + 32 * c);
  }

  const char* kbase = p.c.k + h * p.c.k_str[2];
  const char* vbase = p.c.v + h * p.c.v_str[2];
  // Wave w brings keys 16 w .. 16 w + 15 of a block (past the end: the last key).
  auto key_pos = [&](int b, int key) __attribute__((always_inline)) {
    return key_within(b * kPagedBlock + 16 * wave + key, keys.L);
  };
  bool bad = part.bad;
  auto row_of = [&](int b, int key, int page, int64_t& pg, int64_t& slot) __attribute__((always_inline)) {
    const PagedRow at = keys.row(key_pos(b, key), page);
    bad |= !at.ok;
    pg = at.page;
    slot = at.slot;
  };
  const CopyMap<D> map{lane};
  uint32_t koffs[ND], voffs[ND];                    // of a lane's copies within keys of one page
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    koffs[i] = (uint32_t)map.key(i) * (uint32_t)p.c.k_str[1] + 16 * map.chunk(i);
    voffs[i] = (uint32_t)map.key(i) * (uint32_t)p.c.v_str[1] + 16 * map.chunk(i);
  }
  // Copies keys 16 w .. + 15 of block b of one matrix; `page`: key x's, per lane.
  auto bring16 = [&](int b, int page, const char* base, const int64_t* str, const uint32_t* offs, lds_char* to)
      __attribute__((always_inline)) {
    const int key0 = b * kPagedBlock + 16 * wave;
    int slot0;
    if (p.short_rows && keys.together(key0, 16, &slot0)) {   // the 16 keys lie in one page
      const int pg0 = uniform(page);
      const bool ok = (uint32_t)pg0 < (uint32_t)p.c.n_pages;
      bad |= !ok;
      const char* r = base + (int64_t)(ok ? pg0 : 0) * str[0] + slot0 * str[1];
#pragma unroll
      for (int i = 0; i < ND; ++i) copy16(r, offs[i], to + 1024 * i);
      return;
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      int64_t pg, slot;
      row_of(b, map.key(i), __shfl(page, map.key(i)), pg, slot);
      copy16(base + pg * str[0] + slot * str[1] + 16 * map.chunk(i), to + 1024 * i);
    }
  };
  struct Codes {
    uint32_t w[ND], s[2];
  };
  auto load4 = [&](int b, int page, const char* base, const int64_t* str, const uint8_t* sbase, const int64_t* sstr, Codes& c)
      __attribute__((always_inline)) {
    int64_t pg, slot;
    row_of(b, x, page, pg, slot);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(base + pg * str[0] + slot * str[1] + (D / 8) * g);
#pragma unroll
    for (int i = 0; i < ND; ++i) c.w[i] = w[i];
    const uint8_t* s = sbase + h * sstr[2] + pg * sstr[0] + slot * sstr[1];
    c.s[0] = s[(D / 4) * g / 32];
    c.s[1] = kTwoScales ? s[((D / 4) * g + D / 4 - 1) / 32] : 0;
  };
  typedef __attribute__((address_space(3))) shortx8 lds8;
  auto store4 = [&](const Codes& c, bool masked, lds_char* to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const bool up = kTwoScales && ((D / 4) * g + 8 * i) / 32 != (D / 4) * g / 32;
      const uint32_t sb = up ? c.s[1] : c.s[0];
      shortx8 w = decode8<E>(c.w[i], sb);
      if (masked && sb > Mat<E>::kFinite && any_nonfinite<E>(w)) {
        w = finite8<E>(w);
        odd_s = 1;
      }
      *reinterpret_cast<lds8*>(to + prefill_chunk<D>(x, ND * g + i)) = w;
    }
  };

  // LDS reads.  K: key i32 (+ 32), elements 16 c + 8 half .. + 7.  V: keys 4
  // half + (x >> 2) (+ 8) of tile st, elements 32 dt + 16 ((lane >> 4) & 1) +
  // 4 (x & 3) .. + 3; the transposing read hands lane x element x of them.
  constexpr int KS = D == 96 ? 512 : 256, VS = 2 * KS;   // bytes from chunk to chunk + 2, to chunk + 4
  const int koff[2] = {prefill_chunk<D>(i32, half), prefill_chunk<D>(i32, 2 + half) - KS};   // even and odd c
  const int vrow = 4 * half + (x >> 2), vc = 2 * (g & 1) + ((x & 3) >> 1);
  const int voff0 = prefill_chunk<D>(vrow, vc) + 8 * (x & 1), voff1 = prefill_chunk<D>(vrow + 8, vc) + 8 * (x & 1);

  floatx16 o[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i] = floatx16{0};
  Reference<E> ref_run;
  float l4[4] = {0.f, 0.f, 0.f, 0.f};
  struct Scores {
    floatx16 a, b;                                      // keys 0 .. 31 and 32 .. 63 of a block
  };
  struct Weights {
    shortx8 w[4];
  };
  auto kread = [&](const lds_char* m, int k) __attribute__((always_inline)) {   // operand k of the 2 NK of a block
    return *reinterpret_cast<const lds8*>(m + koff[(k >> 1) & 1] + KS * (k >> 1) + (k & 1) * 2 * TB);
  };
  auto vread = [&](const lds_char* m, int k) __attribute__((always_inline)) {   // operand k of the 4 NO
    const int st = k / NO, dt = k % NO;
    const shortx4 a = read_tr(m + voff0 + st * TB + VS * dt), c = read_tr(m + voff1 + st * TB + VS * dt);
    return __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto is_masked = [&](int j) __attribute__((always_inline)) { return (blk0 + j + 1) * kPagedBlock > lim_min; };

  constexpr int NPV = 4 * NO, NQK = 2 * NK, NM = NPV + NQK, LA = 6, NE = 16;
  Codes kc, vc4;                                        // 4 bits: of blocks j + 2 and j on their way
  int page[4];                                          // key x's page of blocks j .. j + 3
  // Block j: O += V(j - 1) P(j - 1) and S(j + 1) on the matrix core while P(j) is
  // formed from S(j); K(j + 2) and V(j) are brought meanwhile, to where K(j) and
  // V(j - 2) were.  S: parity of j, a constant.
  auto step = [&](auto par, int j, Scores& s, Weights& pv, Scores& sn, Weights& pn) __attribute__((always_inline)) {
    constexpr int S = decltype(par)::value;
    lds_char* kto = smem + S * MAT + wave * TB;
    lds_char* vto = smem + (2 + S) * MAT + wave * TB;
    const lds_char* kfrom = smem + (1 - S) * MAT;
    const lds_char* vfrom = smem + (3 - S) * MAT;
    if constexpr (BITS == 16) {
      bring16(blk0 + j + 2, page[2], kbase, p.c.k_str, koffs, kto);
      bring16(blk0 + j, page[0], vbase, p.c.v_str, voffs, vto);
    } else {
      store4(kc, false, kto);
      store4(vc4, is_masked(j), vto);
      load4(blk0 + j + 3, page[3], kbase, p.c.k_str, p.c.ks, p.c.ks_str, kc);
      load4(blk0 + j + 1, page[1], vbase, p.c.v_str, p.c.vs, p.c.vs_str, vc4);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) page[i] = page[i + 1];
    page[3] = keys.page(key_pos(blk0 + j + 4, x));

    if (is_masked(j)) {
      const int here = lim - (blk0 + j) * kPagedBlock - 4 * half;   // keys of this block that the row attends, from 4 half on
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int k = 8 * (r >> 2) + (r & 3);
        s.a[r] = k < here ? s.a[r] : -__builtin_inff();
        s.b[r] = k + 32 < here ? s.b[r] : -__builtin_inff();
      }
    }
    float t[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float m = vmax(s.a[4 * c], s.a[4 * c + 1]);
      m = vmax(vmax(m, s.a[4 * c + 2]), s.a[4 * c + 3]);
      m = vmax(vmax(m, s.b[4 * c]), s.b[4 * c + 1]);
      t[c] = vmax(vmax(m, s.b[4 * c + 2]), s.b[4 * c + 3]);
    }
    float top = vmax(vmax(t[0], t[1]), vmax(t[2], t[3])) * p.scale_log2;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(ref_run.exceeded(top)) != 0, 0)) {
      // The reference is kept a whole number, so that this factor is a power of two
      // and the weights of block j - 1, rounded already, scale exactly.
      top = __builtin_floorf(__builtin_fmaxf(top, __shfl_xor(top, 32)));
      const float alpha = ref_run.move(top);
#pragma unroll
      for (int i = 0; i < 4; ++i) l4[i] *= alpha;
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= alpha;
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        typedef E v8e __attribute__((ext_vector_type(8)));
        v8e w = __builtin_bit_cast(v8e, pv.w[st]);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (E)((float)w[i] * alpha);
        pv.w[st] = __builtin_bit_cast(shortx8, w);
      }
    }
    __builtin_amdgcn_sched_barrier(0);

    shortx8 opa[NM];
    sn.a = floatx16{0};
    sn.b = floatx16{0};
    int done = 0;
#pragma unroll
    for (int i = 0; i < LA; ++i) opa[i] = vread(vfrom, i);
    // Nothing moves from one matrix instruction's slot to another: left to itself
    // the scheduler puts every LDS read right before its use.
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      if (i < NPV) {
        o[i % NO] = Mat<E>::mfma32(opa[i], pv.w[i / NO], o[i % NO]);
      } else {
        const int k = i - NPV;
        if (k & 1) sn.b = Mat<E>::mfma32(opa[i], qf[k >> 1], sn.b);
        else sn.a = Mat<E>::mfma32(opa[i], qf[k >> 1], sn.a);
      }
      const int li = i + LA;
      if (li < NPV) opa[li] = vread(vfrom, li);
      else if (li < NM) opa[li] = kread(kfrom, li - NPV);
      // the weights of two keys, and their share of the row sum, in every few slots
#pragma unroll
      for (; done < (i + 1) * NE / NM; ++done) {
        const int st = done / 4, q = done % 4;
        const floatx16& y = st < 2 ? s.a : s.b;
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(y[8 * (st & 1) + 2 * q], p.scale_log2, -ref_run.m));
        const float c = __builtin_amdgcn_exp2f(__builtin_fmaf(y[8 * (st & 1) + 2 * q + 1], p.scale_log2, -ref_run.m));
        l4[q] += a + c;
        u32x4 w = __builtin_bit_cast(u32x4, pn.w[st]);
        w[q] = pack2<E>(a, c);
        pn.w[st] = __builtin_bit_cast(shortx8, w);
      }
    }
#pragma unroll
    for (int st = 0; st < 4; ++st) keep(pn.w[st]);      // formed here, not where they are used
#pragma unroll
    for (int q = 0; q < 4; ++q) keep(l4[q]);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (BITS == 16) {
      wait_copies<0>();
      if (is_masked(j) && search_tile<E>(vto, TB, lane)) odd_s = 1;
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);                 // LDS writes are in place for the others' reads
    phase_barrier();
  };

  if (threadIdx.x == 0) bad_s = odd_s = 0;
  __syncthreads();
  const int n = blk1 - blk0;
  if (n > 0) {
    // K of blocks 0 and 1; V of the block before the first: zeros, with P = 0
    for (int at = 16 * (int)threadIdx.x; at < MAT; at += 4096) *reinterpret_cast<lds8*>(smem + 3 * MAT + at) = shortx8{0};
#pragma unroll
    for (int i = 0; i < 4; ++i) page[i] = keys.page(key_pos(blk0 + i, x));
    if constexpr (BITS == 16) {
      bring16(blk0, page[0], kbase, p.c.k_str, koffs, smem + wave * TB);
      bring16(blk0 + 1, page[1], kbase, p.c.k_str, koffs, smem + MAT + wave * TB);
      wait_copies<0>();
    } else {
      load4(blk0, page[0], kbase, p.c.k_str, p.c.ks, p.c.ks_str, kc);
      load4(blk0 + 1, page[1], kbase, p.c.k_str, p.c.ks, p.c.ks_str, vc4);
      store4(kc, false, smem + wave * TB);
      store4(vc4, false, smem + MAT + wave * TB);
      load4(blk0 + 2, page[2], kbase, p.c.k_str, p.c.ks, p.c.ks_str, kc);
      load4(blk0, page[0], vbase, p.c.v_str, p.c.vs, p.c.vs_str, vc4);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);
    phase_barrier();
    Scores sa, sb;
    Weights wa, wb;
    sa.a = sa.b = floatx16{0};
#pragma unroll
    for (int k = 0; k < NQK; ++k) {
      if (k & 1) sa.b = Mat<E>::mfma32(kread(smem, k), qf[k >> 1], sa.b);
      else sa.a = Mat<E>::mfma32(kread(smem, k), qf[k >> 1], sa.a);
    }
#pragma unroll
    for (int st = 0; st < 4; ++st) wa.w[st] = wb.w[st] = shortx8{0};
    phase_barrier();                                    // K(0) has been read
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    int j = 0;
    for (; j + 1 < n; j += 2) {
      step(Even{}, j, sa, wa, sb, wb);
      step(Odd{}, j + 1, sb, wb, sa, wa);
    }
    if (j < n) {
      step(Even{}, j, sa, wa, sb, wb);
      wa = wb;
    }
    const lds_char* vlast = smem + (2 + ((n - 1) & 1)) * MAT;
#pragma unroll
    for (int k = 0; k < NPV; ++k) o[k % NO] = Mat<E>::mfma32(vread(vlast, k), wa.w[k / NO], o[k % NO]);
  }

  // A bad page seen by any wave spoils the tile.
  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) bad_s = 1;
  __syncthreads();
  if (!Keys::kStaged && bad_s && threadIdx.x == 0 && !(sq.flags & LVSA_PAGED_BAD_LENGTH)) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);

  if (__builtin_expect(odd_s != 0, 0)) {
    const int from = lim_min / kPagedBlock > blk0 ? lim_min / kPagedBlock : blk0;
    const int k1 = blk1 * kPagedBlock < lim_max ? blk1 * kPagedBlock : lim_max;
    add_nonfinite_keys<E, BITS, 4 * NO>(p.c, keys, h, from * kPagedBlock, k1, lim, 4 * half, 8,
                                        [&](int q, int r, uint32_t v, bool seen) __attribute__((always_inline)) {
                                          o[q >> 2][4 * (q & 3) + r] = add_nonfinite<E>(o[q >> 2][4 * (q & 3) + r], v, seen);
                                        });
  }
  const float l_run = (l4[0] + l4[1]) + (l4[2] + l4[3]);
  float l = l_run + __shfl_xor(l_run, 32);
  if (bad_s) l = __builtin_nanf("");
  if (row < nrows) store_rows<D, E>(p, whole, slot, kPagedTile, row - r0, half, ref, o, ref_run.m, l);
}

// Four waves of 32 rows, the matrix core of each SIMD with one or two of them:
// a wave feeds it by itself, with the products of the blocks before and after
// while it forms the weights of its own block between them.  Two LDS places
// each for K and V of a block of 64 keys; wave w brings tile w (16 keys).
// 16-bit pages are copied without passing registers; of 4-bit pages the codes
// are loaded a step ahead and written to LDS as 16-bit values, so every row is
// decoded once for 128 query rows.
//
// 780 tokens of 12 heads over 4 of 256, over 31980 keys in 4 bits: 378 us with
// plan and joining, 790 TFLOP/s (500 us with a phase of products after a phase of
// softmax).  The decoding of K and V, their addresses, the mask and the maximum
// stand before a step's first product, on the only wave of a SIMD: MFMA busy a
// third of the time, vector instructions another.  4 sequences of 128 tokens, 16 heads of 128, over 16384 keys: 141 us.
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256, D >= 192 ? 1 : 2) void paged_prefill_kernel(PagedAttnParams p) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const PlanHead hd = *p.head;
  if (uniform(hd.bad_cu)) {
    spoil_rows<E>(p, D, lane, wave, 4);
    return;
  }
  if (p.fill_tail) fill_tail_rows(p, D, lane, wave, 4);
  const int shares = uniform(hd.shares), share = share_of(blockIdx.x, shares);
  if (share < 0) return;
  // The share's tiles from the last to the first: the part that it ends with
  // starts at its tile's first key block and the one it starts with ends at the
  // last, so that the work-groups of an XCD walk a head's keys at about the
  // same place at the same time, and its L2 serves them.
  const int64_t U = hd.per_head * p.c.Hkv;
  int left = uniform((int)(unit_start(U, shares, share + 1) - unit_start(U, shares, share)));
  int h = uniform(p.ends[share].h), ti = uniform(p.ends[share].tile), blk_end = uniform(p.ends[share].blk);
  for (;;) {
  const PlanTile tile = p.plan_tiles[ti];
  const int seq = uniform(tile.seq), r0 = uniform(tile.r0), units = uniform(tile.units), nb = uniform(tile.blocks);
  const PagedSeq sq = uniform(tile.sq);
  const int blk0 = left < blk_end ? blk_end - left : 0;
  const bool whole = blk0 == 0 && blk_end == units;
  const int64_t slot = 2 * (int64_t)share + (left > blk_end ? 1 : 0);   // the share comes from another tile: see decode_slots
  const int blk1 = blk_end < nb ? blk_end : nb;
  const DecodePart part = {sq, h, r0, sq.n * p.group, blk0, blk1, slot, whole,
                           (sq.flags & (LVSA_PAGED_BAD_LENGTH | LVSA_PAGED_BAD_PAGE)) != 0};
  prefill_part<D, E, BITS>(p, part, PagedKeys{p.c, p.c.table + seq * p.c.table_str, sq.L});
  left -= blk_end - blk0;
  if (left <= 0) break;
  if (--ti < 0) {
    ti = hd.tiles - 1;
    --h;
  }
  blk_end = uniform(p.plan_tiles[ti].units);
  __syncthreads();                                      // LDS of this tile has been read
  }
}

// ──────────────────────────── prefill, tall tiles ──────────────────────────

// 4 bytes per lane, global -> LDS at `l` + 4 * lane (see copy16).
__device__ __forceinline__ void copy4(const void* from, const lds_char* l) {
  const uint32_t la = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)l);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(from), "s"(la) : "m0", "memory");
#pragma clang diagnostic pop
}

// Eight waves of 32 rows in two groups of four that alternate between a phase
// of matrix products and a phase of softmax, one barrier after each: on every
// SIMD one wave keeps the matrix core busy while the other one's
// exponentials run, which two independent work-groups do only by chance.
//
//   M(j)  S(j) = K(j) Q^T and O += V(j-1) P(j-1) as one stream of matrix
//         instructions whose LDS operands are read LA instructions ahead
//   S(j)  masks, maximum, P(j), row sums
//
// The products get the higher priority of the two waves on a SIMD (3%).  4680
// tokens of 12 heads of 128 over 32760 keys: 750 to 780 us with plan and joining,
// by the card's clock, 1.03 to 1.07 PFLOP/s (950 us with tiles of 128 rows and two independent work-groups; 840 us
// with products and exponentials of one wave interleaved, which the issue of the
// vector instructions beside the matrix ones holds up; 660 us without the copies,
// which is what the data's way costs).  Causal prompts of head size 64: 189 us,
// 660 TFLOP/s: half the products per weight, so the softmax is the longer phase, and
// only one of a SIMD's two waves is in it at a time, which issues a vector
// instruction every 8 cycles where two would every 4 (VALU issuing 50%, MFMA 32%).
//
// Group 0 runs M(j) in phase 2 j and S(j) in phase 2 j + 1, group 1 one phase
// later.  LDS holds four blocks of 64 keys of K and of V; group 0 brings K,
// group 1 V, wave w of each the block's tile w, two blocks ahead: block j + 2
// goes where block j - 2 was, whose last readers (group 1's M(j - 1) in phase
// 2 j - 1) are done before M(j).
//   16 bits: copies past the registers, issued in the middle of M(j) and waited
//   for at the end of M(j + 1), with the page numbers of block j + 4 behind them
//   on the same way, so that no wait of the compiler's own for an ordinary load
//   ever drains the copies.
//   4 bits: codes of block j + 3 are loaded in M(j), decoded and written to LDS
//   in S(j + 1).
template <int D, typename E, int BITS>
__global__ __launch_bounds__(512, 1) void paged_tall_kernel(PagedAttnParams p) {
  constexpr int ND = D / 32, NK = D / 16, NO = D / 32;
  constexpr int TB = 32 * D, MAT = 4 * TB;
  constexpr int VB = 4 * MAT, PB = 8 * MAT;
  constexpr bool kTwoScales = D == 96;
  // K and V rings, page numbers [wave][4][64]
  __shared__ __attribute__((aligned(1024))) char smem_raw[PB + (BITS == 16 ? 8 * 4 * 256 : 0)];
  __shared__ int bad_s, odd_s;
  lds_char* smem = (lds_char*)smem_raw;
  typedef __attribute__((address_space(3))) shortx8 lds8;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = wave >> 2, dw = wave & 3;
  const int half = lane >> 5, i32 = lane & 31;
  const int g = lane >> 4, x = lane & 15;

  const PlanHead hd = *p.head;
  if (uniform(hd.bad_cu)) {
    spoil_rows<E>(p, D, lane, wave, 8);
    return;
  }
  if (p.fill_tail) fill_tail_rows(p, D, lane, wave, 8);
  const int shares = uniform(hd.shares), share = share_of(blockIdx.x, shares);
  if (share < 0) return;
  // The share's tiles from the last to the first: the part that it ends with
  // starts at its tile's first key block and the one it starts with ends at the
  // last, so that the work-groups of an XCD walk a head's keys at about the
  // same place at the same time, and its L2 serves them.
  const int64_t U = hd.per_head * p.c.Hkv;
  int left = uniform((int)(unit_start(U, shares, share + 1) - unit_start(U, shares, share)));
  int h = uniform(p.ends[share].h), ti = uniform(p.ends[share].tile), blk_end = uniform(p.ends[share].blk);
  for (;;) {
  const PlanTile tile = p.plan_tiles[ti];
  const int seq = uniform(tile.seq), r0 = uniform(tile.r0), units = uniform(tile.units), nb = uniform(tile.blocks);
  const PagedSeq sq = uniform(tile.sq);
  const int blk0 = left < blk_end ? blk_end - left : 0;
  const bool whole = blk0 == 0 && blk_end == units;
  const int64_t slot = 2 * (int64_t)share + (left > blk_end ? 1 : 0);   // the share comes from another tile: see decode_slots
  const int blk1 = blk_end < nb ? blk_end : nb;
  const int nrows = sq.n * p.group;
  const int r_last = r0 + kPagedTall < nrows ? r0 + kPagedTall - 1 : nrows - 1;
  const int lim_min = key_limit(p, sq, r0), lim_max = key_limit(p, sq, r_last);
  const int n = blk1 - blk0;

  const int row = r0 + 32 * wave + i32;
  const int rc = row < nrows ? row : nrows - 1;
  const RowRef ref = row_ref(p, sq, h, rc);
  const int lim = key_limit(p, sq, rc);

  const char* src = grp == 0 ? p.c.k + h * p.c.k_str[2] : p.c.v + h * p.c.v_str[2];
  const int64_t str0 = grp == 0 ? p.c.k_str[0] : p.c.v_str[0], str1 = grp == 0 ? p.c.k_str[1] : p.c.v_str[1];
  const uint8_t* scl = BITS == 16 ? nullptr : grp == 0 ? p.c.ks + h * p.c.ks_str[2] : p.c.vs + h * p.c.vs_str[2];
  const int64_t sst0 = grp == 0 ? p.c.ks_str[0] : p.c.vs_str[0], sst1 = grp == 0 ? p.c.ks_str[1] : p.c.vs_str[1];
  const int32_t* table = p.c.table + seq * p.c.table_str;
  lds_char* ring = smem + grp * VB + dw * TB;           // this wave's tile of stage 0
  lds_char* pids = smem + PB + wave * 1024;
  auto key_pos = [&](int j, int key) __attribute__((always_inline)) {
    return key_within((blk0 + j) * kPagedBlock + 16 * dw + key, sq.L);
  };
  bool bad = (sq.flags & (LVSA_PAGED_BAD_LENGTH | LVSA_PAGED_BAD_PAGE)) != 0;
  auto row_at = [&](int j, int key, int page, int64_t& sc) __attribute__((always_inline)) {
    const PagedRow at = paged_row(p.c, key_pos(j, key), page);
    bad |= !at.ok;
    if constexpr (BITS == 4) sc = at.page * sst0 + at.slot * sst1;
    return src + at.page * str0 + at.slot * str1;
  };
  // 16 bits: brings keys 16 dw .. + 15 of block j.  Keys of one page, the usual
  // case: one uniform address, made on the scalar unit.
  const CopyMap<D> map{lane};
  uint32_t offs[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) offs[i] = (uint32_t)map.key(i) * (uint32_t)str1 + 16 * map.chunk(i);
  typedef const __attribute__((address_space(3))) int lds_int;
  auto bring16 = [&](int j) __attribute__((always_inline)) {
    const lds_char* at = pids + 256 * (j & 3);
    lds_char* to = ring + (j & 3) * MAT;
    const int key0 = (blk0 + j) * kPagedBlock + 16 * dw, slot0 = key0 - page_of(p.c, key0) * p.c.page_size;
    if (p.short_rows && key0 + 16 <= sq.L && slot0 + 16 <= p.c.page_size) {
      const int pg0 = uniform(*reinterpret_cast<lds_int*>(at));
      const bool ok = (uint32_t)pg0 < (uint32_t)p.c.n_pages;
      bad |= !ok;
      const char* base = src + (int64_t)(ok ? pg0 : 0) * str0 + slot0 * str1;
#pragma unroll
      for (int i = 0; i < ND; ++i) copy16(base, offs[i], to + 1024 * i);
      return;
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      int64_t none;
      const int key = map.key(i);
      copy16(row_at(j, key, *reinterpret_cast<lds_int*>(at + 4 * key), none) + 16 * map.chunk(i), to + 1024 * i);
    }
  };
  auto bring_pages = [&](int j) __attribute__((always_inline)) {
    copy4(table + page_of(p.c, key_pos(j, x)), pids + 256 * (j & 3));
  };

  if (threadIdx.x == 0) bad_s = odd_s = 0;
  __syncthreads();
  // V of the block before the first (stage 3): read by M(0) with P = 0
  for (int at = 16 * (int)threadIdx.x; at < MAT; at += 8192) *reinterpret_cast<lds8*>(smem + VB + 3 * MAT + at) = shortx8{0};

  shortx8 qf[NK];
  {
    const char* qp = p.q + ref.tok * p.q_str[0] + ref.head * p.q_str[1] + 16 * half;
#pragma unroll
    for (int c = 0; c < NK; ++c) qf[c] = *reinterpret_cast<const shortx8*>(qp + 32 * c);
    wait_copies<0>();                                   // no load of the compiler's own is left for the loop to wait for
#pragma unroll
    for (int c = 0; c < NK; ++c) keep(qf[c]);
  }

  // 4 bits: codes and scales of the next block to decode, and of the one after it.
  struct Codes {
    uint32_t w[ND], s[2];
  } here4, coming;
  int page_next = 0;                                    // 4 bits: page number of the next block to load
  auto load4 = [&](int j, int page, Codes& c) __attribute__((always_inline)) {
    int64_t sc = 0;
    const char* r = row_at(j, x, page, sc) + (D / 8) * g;
#pragma unroll
    for (int i = 0; i < ND; ++i) c.w[i] = reinterpret_cast<const uint32_t*>(r)[i];
    c.s[0] = scl[sc + (D / 4) * g / 32];
    c.s[1] = kTwoScales ? scl[sc + ((D / 4) * g + D / 4 - 1) / 32] : 0;
  };
  auto is_masked = [&](int j) __attribute__((always_inline)) { return (blk0 + j + 1) * kPagedBlock > lim_min; };
  auto store4 = [&](int j, int stage, const Codes& c) __attribute__((always_inline)) {
    const bool masked = grp == 1 && is_masked(j);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const bool up = kTwoScales && ((D / 4) * g + 8 * i) / 32 != (D / 4) * g / 32;
      const uint32_t sb = up ? c.s[1] : c.s[0];
      shortx8 w = decode8<E>(c.w[i], sb);
      if (masked && sb > Mat<E>::kFinite && any_nonfinite<E>(w)) {
        w = finite8<E>(w);
        odd_s = 1;
      }
      *reinterpret_cast<lds8*>(ring + stage * MAT + prefill_chunk<D>(x, ND * g + i)) = w;
    }
  };

  // LDS reads (see paged_prefill_kernel).
  constexpr int KS = D == 96 ? 512 : 256, VS = 2 * KS;   // bytes from chunk to chunk + 2, to chunk + 4
  const int koff[2] = {prefill_chunk<D>(i32, half), prefill_chunk<D>(i32, 2 + half) - KS};   // even and odd c
  const int vrow = 4 * half + (x >> 2), vc = 2 * (g & 1) + ((x & 3) >> 1);
  const int voff0 = VB + prefill_chunk<D>(vrow, vc) + 8 * (x & 1), voff1 = VB + prefill_chunk<D>(vrow + 8, vc) + 8 * (x & 1);

  floatx16 o[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i] = floatx16{0};
  floatx16 s0 = floatx16{0}, s1 = floatx16{0};
  shortx8 pb[4];
#pragma unroll
  for (int st = 0; st < 4; ++st) pb[st] = shortx8{0};
  Reference<E> ref_run;
  float l4[4] = {0.f, 0.f, 0.f, 0.f};

  constexpr int LA = D == 128 ? 6 : 4;
  constexpr bool kEarly = D == 128;
  constexpr int NQK = 2 * NK, NM = NQK + 4 * NO;
  // D = 128: the first operands of M(j + 1), K's, are read in S(j), so that its
  // first products need not wait (788 -> 779 us for 4680 tokens of 12 heads over
  // 32760 keys; of head size 64 187 -> 190 us for the causal prompts, whose S is
  // the longer phase).
  shortx8 first[LA];
  auto read_first = [&](int j) __attribute__((always_inline)) {
    const int kst = (j & 3) * MAT;
#pragma unroll
    for (int i = 0; i < LA; ++i) first[i] = *reinterpret_cast<const lds8*>(smem + koff[(i >> 1) & 1] + kst + KS * (i >> 1) + (i & 1) * 2 * TB);
  };
  auto mphase = [&](int j) __attribute__((always_inline)) {
    const int kst = (j & 3) * MAT, kat[2] = {koff[0] + kst, koff[1] + kst}, vst = ((j + 3) & 3) * MAT, v0 = voff0 + vst, v1 = voff1 + vst;
    if constexpr (BITS == 4) {
      const int page = page_next;
      page_next = table[page_of(p.c, key_pos(j + 4, x))];
      load4(j + 3, page, coming);
    }
    shortx8 opa[NM];
    s0 = floatx16{0};
    s1 = floatx16{0};
    if constexpr (!kEarly) read_first(j);
#pragma unroll
    for (int i = 0; i < LA; ++i) opa[i] = first[i];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const int li = i + LA;
      if (li < NM) {
        if (li < NQK) {
          opa[li] = *reinterpret_cast<const lds8*>(smem + kat[(li >> 1) & 1] + KS * (li >> 1) + (li & 1) * 2 * TB);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        } else {
          const int k = li - NQK, st = k / NO, dt = k % NO;
          const shortx4 a = read_tr(smem + v0 + st * TB + VS * dt), c = read_tr(smem + v1 + st * TB + VS * dt);
          opa[li] = __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
      }
      {
        if (i < NQK) {
          if (i & 1) s1 = Mat<E>::mfma32(opa[i], qf[i >> 1], s1);
          else s0 = Mat<E>::mfma32(opa[i], qf[i >> 1], s0);
        } else {
          const int k = i - NQK;
          o[k % NO] = Mat<E>::mfma32(opa[i], pb[k / NO], o[k % NO]);
        }
        if (BITS == 16 && i == NQK - 1) {
          bring16(j + 2);
          bring_pages(j + 4);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      }
    }
    keep(s0);
    keep(s1);
#pragma unroll
    for (int dt = 0; dt < NO; ++dt) keep(o[dt]);
    if constexpr (BITS == 16) wait_copies<ND + 1>();      // block j + 1 and the page numbers of block j + 3 have landed
  };

  auto sphase = [&](int j) __attribute__((always_inline)) {
    if constexpr (kEarly) read_first(j + 1);
    if (is_masked(j)) {
      const int here = lim - (blk0 + j) * kPagedBlock - 4 * half;   // keys of this block that the row attends, from 4 half on
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int k = 8 * (r >> 2) + (r & 3);
        s0[r] = k < here ? s0[r] : -__builtin_inff();
        s1[r] = k + 32 < here ? s1[r] : -__builtin_inff();
      }
    }
    float t[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float m = vmax(s0[4 * c], s0[4 * c + 1]);
      m = vmax(vmax(m, s0[4 * c + 2]), s0[4 * c + 3]);
      m = vmax(vmax(m, s1[4 * c]), s1[4 * c + 1]);
      t[c] = vmax(vmax(m, s1[4 * c + 2]), s1[4 * c + 3]);
    }
    float top = vmax(vmax(t[0], t[1]), vmax(t[2], t[3])) * p.scale_log2;
    if (__builtin_amdgcn_ballot_w64(ref_run.exceeded(top))) {
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float alpha = ref_run.move(top);
#pragma unroll
      for (int i = 0; i < 4; ++i) l4[i] *= alpha;
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= alpha;
    }
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const floatx16& s = st < 2 ? s0 : s1;
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * (st & 1) + 2 * i], p.scale_log2, -ref_run.m));
        const float c = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * (st & 1) + 2 * i + 1], p.scale_log2, -ref_run.m));
        l4[i] += a + c;
        w[i] = pack2<E>(a, c);
      }
      pb[st] = __builtin_bit_cast(shortx8, w);
    }
    if constexpr (BITS == 4) {
      store4(j + 2, (j + 2) & 3, here4);
      here4 = coming;
    } else {
      if (grp == 1 && is_masked(j + 1) && search_tile<E>(ring + ((j + 1) & 3) * MAT, TB, lane)) odd_s = 1;
    }
#pragma unroll
    for (int st = 0; st < 4; ++st) keep(pb[st]);
#pragma unroll
    for (int i = 0; i < 4; ++i) keep(l4[i]);
    keep(ref_run.m);
#pragma unroll
    for (int dt = 0; dt < NO; ++dt) keep(o[dt]);
#pragma unroll
    for (int i = 0; i < (kEarly ? LA : 0); ++i) keep(first[i]);
    // LDS writes of this phase are in place for the others' reads after the barrier
    if (BITS == 4 || grp == 1) __builtin_amdgcn_s_waitcnt(0xC07F);
  };

  if (n > 0) {
    if constexpr (BITS == 16) {
      for (int j = 0; j < 4; ++j) bring_pages(j);
      wait_copies<0>();
      bring16(0);
      bring16(1);
      wait_copies<ND>();                                // block 0
      if (grp == 1 && is_masked(0) && search_tile<E>(ring, TB, lane)) odd_s = 1;
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        load4(j, table[page_of(p.c, key_pos(j, x))], here4);
        store4(j, j, here4);
      }
      load4(2, table[page_of(p.c, key_pos(2, x))], here4);
      page_next = table[page_of(p.c, key_pos(3, x))];
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);                 // LDS writes: V of stage 3, tiles, notes
    phase_barrier();
    if (grp == 1) phase_barrier();
    if constexpr (kEarly) read_first(0);
    // Each group passes n matrix and n softmax phases, and the last block's
    // second product; the barriers (2 n + 1 for both after the first) pair phase
    // with phase.  One copy of each phase and one exit, at the bottom: with the
    // ring's stages as constants (four copies) the compiler spilled hundreds of
    // registers, and with the exit after M(n) it moved O to and fro in every
    // step (64 moves).
    for (int j = 0; j < n; ++j) {
      __builtin_amdgcn_s_setprio(1);                    // the matrix instructions before the other group's exponentials: 3%
      mphase(j);
      __builtin_amdgcn_s_setprio(0);
      phase_barrier();
      sphase(j);
      phase_barrier();
    }
    {
      const int vst = ((n + 3) & 3) * MAT, v0 = voff0 + vst, v1 = voff1 + vst;
#pragma unroll
      for (int st = 0; st < 4; ++st)
#pragma unroll
        for (int dt = 0; dt < NO; ++dt) {
          const shortx4 a = read_tr(smem + v0 + st * TB + VS * dt), c = read_tr(smem + v1 + st * TB + VS * dt);
          o[dt] = Mat<E>::mfma32(__builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7), pb[st], o[dt]);
        }
    }
    if (grp == 0) phase_barrier();
    wait_copies<0>();                                   // copies past the last block land before the work-group ends
  }

  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) bad_s = 1;
  __syncthreads();
  if (bad_s && threadIdx.x == 0 && !(sq.flags & LVSA_PAGED_BAD_LENGTH)) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
  if (__builtin_expect(odd_s != 0, 0)) {
    const int from = lim_min / kPagedBlock > blk0 ? lim_min / kPagedBlock : blk0;
    const int k1 = blk1 * kPagedBlock < lim_max ? blk1 * kPagedBlock : lim_max;
    add_nonfinite_keys<E, BITS, 4 * NO>(p.c, PagedKeys{p.c, table, sq.L}, h, from * kPagedBlock, k1, lim, 4 * half, 8,
                                        [&](int q, int r, uint32_t v, bool seen) __attribute__((always_inline)) {
                                          o[q >> 2][4 * (q & 3) + r] = add_nonfinite<E>(o[q >> 2][4 * (q & 3) + r], v, seen);
                                        });
  }
  const float l_run = (l4[0] + l4[1]) + (l4[2] + l4[3]);
  float l = l_run + __shfl_xor(l_run, 32);
  if (bad_s) l = __builtin_nanf("");
  if (row < nrows) store_rows<D, E>(p, whole, slot, kPagedTall, row - r0, half, ref, o, ref_run.m, l);
  left -= blk_end - blk0;
  if (left <= 0) break;
  if (--ti < 0) {
    ti = hd.tiles - 1;
    --h;
  }
  blk_end = uniform(p.plan_tiles[ti].units);
  __syncthreads();                                      // LDS of this tile has been read
  }
}

template <int D, typename E, int BITS>
int paged_launch(const PagedAttnParams& p, int rows, hipStream_t stream) {
  if (rows == kPagedTall) {
    if constexpr (D <= 128)
      hipLaunchKernelGGL((paged_tall_kernel<D, E, BITS>), dim3((unsigned)p.grid), dim3(512), 0, stream, p);
  } else if (rows == kPagedTile) {
    hipLaunchKernelGGL((paged_prefill_kernel<D, E, BITS>), dim3((unsigned)p.grid), dim3(256), 0, stream, p);
  } else if (rows == 16) {
    hipLaunchKernelGGL((paged_decode_kernel<D, E, BITS, 1>), dim3((unsigned)p.grid), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((paged_decode_kernel<D, E, BITS, 2>), dim3((unsigned)p.grid), dim3(256), 0, stream, p);
  }
  return launch_status("lvsa_paged_attn_fwd");
}

template <int D>
int paged_launch(const PagedAttnParams& p, int bits, int rows, bool bf16, hipStream_t stream) {
  if (bf16) return bits == 16 ? paged_launch<D, __bf16, 16>(p, rows, stream) : paged_launch<D, __bf16, 4>(p, rows, stream);
  return bits == 16 ? paged_launch<D, _Float16, 16>(p, rows, stream) : paged_launch<D, _Float16, 4>(p, rows, stream);
}

}  // namespace
}  // namespace lvsa
