// Attention over the paged key/value cache (gfx950): o = softmax(scale q K^T) V
// for the newest tokens of every sequence, 16-bit pages or 4-bit ones.  One
// unit per head size instantiates the kernels (lvsa_paged_d*.hip).
//
// The query heads of a key head are packed: row r of a (sequence, key head)
// pair is token r / group, head r % group of the group, so that a tile of rows
// reads each key and value once for all of them.
//
//   paged_decode_kernel   few rows (tiles of 16 or 32): bound by the bytes of
//                         the cache.  Matrix instructions of 16 rows, each
//                         wave on keys of its own.
//   paged_prefill_kernel  tiles of 128 rows: bound by the matrix cores and the
//                         softmax.  Four waves of 32 rows share key blocks of
//                         64 in LDS.
//
// Both form S^T = K Q^T, so that a lane owns one row's scores, and O^T += V^T
// P^T with P straight from S^T's registers: the order of the keys within a
// step is permuted alike on both operands.  V^T comes out of LDS by
// transposing reads.
//
// LDS tile of 16 keys (K or V): 16-byte chunk c (elements 8c .. 8c + 7) of key
// r at 256 c + 16 (r ^ 8 (c & 1)).  A lane that copies key r always holds that
// one key, so it looks its page up once per tile; reading 16 keys of a chunk
// covers all 64 banks, and so does a transposing read of 4 or 8 keys over two
// chunks (with 16 r alone its two chunks would share half the banks).
#pragma once
#include "lvsa_paged.h"

namespace lvsa {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

template <typename E>
struct Mat;
template <>
struct Mat<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static constexpr uint32_t kExp = 0x7f80u, kOne = 0x3f80u;
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
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u;
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

__device__ __forceinline__ int lds_chunk(int tile_bytes, int r, int c) {
  return (r >> 4) * tile_bytes + 256 * c + 16 * ((r & 15) ^ (8 * (c & 1)));
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
// (0 * inf is NaN).  Blocks with masked keys are searched for such values; if
// there are any, they are added to the rows that attend them by themselves
// (add_nonfinite) and the matrix product runs on the tile with zeros in their
// place (finite8).
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

// Row r of a (sequence, key head) pair: its q and o / lse, and the end of the
// keys it attends.
struct RowRef {
  int64_t tok;
  int head;
};
__device__ __forceinline__ RowRef row_ref(const PagedAttnParams& p, const PagedSeq& s, int h, int r) {
  const int i = r / p.group;
  return RowRef{(int64_t)s.t0 + i, h * p.group + (r - i * p.group)};
}
__device__ __forceinline__ int key_limit(const PagedAttnParams& p, const PagedSeq& s, int r) {
  if (!p.causal) return s.L;
  const int64_t e = (int64_t)s.first + r / p.group + 1;
  return e < 0 ? 0 : e > s.L ? s.L : (int)e;
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

// Two work-groups per CU (up to 256 registers) where the operands allow it.
//
// The launch's work, sum over sequences of row tiles x key heads x key steps,
// is cut into `grid` equal shares, so that ragged batches keep every
// work-group busy to the end and a single long sequence is spread over all of
// them.  A share may end inside a (row tile, head): its partial sums go to one
// of two slots of the work-group and paged_merge_kernel joins them.  The
// share's bounds follow from the lengths alone, so the merge finds the slots
// without a word from this kernel.
template <int D, typename E, int BITS, int NT>
__global__ __launch_bounds__(256, (D == 256 || (D == 192 && NT == 2)) ? 1 : 2) void paged_decode_kernel(PagedAttnParams p) {
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

  // The share [u, u_end) and the sequence it starts in.
  int64_t U = 0;
  int flags = 0;
  for (int s0 = 0; s0 < p.c.B; s0 += 64) {
    int64_t n = 0;
    if (s0 + lane < p.c.B) {
      const PagedSeq q = paged_seq(p.c, s0 + lane);
      n = decode_units(p, q, ROWS, KEYS);
      flags |= q.flags;
    }
    U += __shfl(wave_scan(n, lane), 63);
  }
  if (blockIdx.x == 0 && wave == 0 && flags) paged_flag(p.c, flags);
  if (U == 0) return;
  const int shares = unit_shares(U, p.grid);
  if ((int)blockIdx.x >= shares) return;
  int64_t u = unit_start(U, shares, blockIdx.x);
  const int64_t u_end = unit_start(U, shares, blockIdx.x + 1);
  int seq = 0;
  int64_t base = 0;                            // units before sequence `seq`
  for (int s0 = 0; s0 < p.c.B; s0 += 64) {
    int64_t n = 0;
    if (s0 + lane < p.c.B) n = decode_units(p, paged_seq(p.c, s0 + lane), ROWS, KEYS);
    const int64_t incl = wave_scan(n, lane);
    const uint64_t above = __builtin_amdgcn_ballot_w64(base + incl > u);
    if (above) {
      const int at = __builtin_ctzll(above);
      seq = s0 + at;
      base += __shfl(incl - n, at);
      break;
    }
    base += __shfl(incl, 63);
  }

  const int64_t u_first = u;
  while (u < u_end && seq < p.c.B) {
    const PagedSeq sq = paged_seq(p.c, seq);
    const int64_t units = decode_units(p, sq, ROWS, KEYS);
    if (u >= base + units) {
      base += units;
      ++seq;
      continue;
    }
    const int nb = (int)(((int64_t)sq.L + KEYS - 1) / KEYS);
    const int64_t run = (u - base) / nb;
    const int blk0 = (int)((u - base) - run * nb);
    const int64_t left = u_end - u;
    const int blk1 = left < nb - blk0 ? blk0 + (int)left : nb;
    const int rt = (int)(run / p.c.Hkv), h = (int)(run - (int64_t)rt * p.c.Hkv);
    const int nrows = sq.n * p.group;
    const int r0 = rt * ROWS;

    // Q of the tile, in the order of the keys' elements; rows past the end
    // repeat the last one.
    shortx8 qf[NT][ND];
    int lim[NT];
    int lim_min = sq.L;
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
      lim[n] = key_limit(p, sq, r);
    }
    {
      const int first = key_limit(p, sq, r0);
      lim_min = first < lim_min ? first : lim_min;
    }

    floatx4 o[NT][NO];
    float m_run[NT], l_run[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m_run[n] = kNoKeys;
      l_run[n] = 0.f;
#pragma unroll
      for (int i = 0; i < NO; ++i) o[n][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    bool bad = (sq.flags & LVSA_PAGED_BAD_LENGTH) != 0;

    const char* kbase = p.c.k + h * p.c.k_str[2];
    const char* vbase = p.c.v + h * p.c.v_str[2];
    const uint8_t* ksbase = BITS == 4 ? p.c.ks + h * p.c.ks_str[2] : nullptr;
    const uint8_t* vsbase = BITS == 4 ? p.c.vs + h * p.c.vs_str[2] : nullptr;
    const int32_t* table = p.c.table + seq * p.c.table_str;

    // Key x of tile j of step b (past the end: the last key).
    auto key_pos = [&](int b, int j) __attribute__((always_inline)) {
      return key_within(b * KEYS + wave * KW + 16 * j + x, sq.L);
    };
    auto load_pages = [&](int b, int* page) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < T; ++j) page[j] = table[page_of(p.c, key_pos(b, j))];
    };
    auto load = [&](int b, const int* page, Step<D, BITS, T>& st) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < T; ++j) {
        const PagedRow at = paged_row(p.c, key_pos(b, j), page[j]);
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
      if (key0 >= sq.L) return;                // the last step's waves past the end
      // V to LDS, chunk by chunk
      bool odd_v = false;
      const bool masked = key0 + KW > lim_min;
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
          if (masked) odd_v |= any_nonfinite<E>(w);
          *reinterpret_cast<__attribute__((address_space(3))) shortx8*>(vbuf + lds_chunk(TB, 16 * j + x, c)) = w;
        }
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
        // The running maximum moves only when some score exceeds it by 2^8:
        // weights up to 256 are as exact, and the usual step rescales nothing.
        if (__builtin_amdgcn_ballot_w64(top > m_run[n] + 8.0f)) {
          top = __builtin_fmaxf(top, __shfl_xor(top, 16));
          top = __builtin_fmaxf(top, __shfl_xor(top, 32));
          const float m_new = __builtin_fmaxf(m_run[n], top);
          const float alpha = __builtin_amdgcn_exp2f(m_run[n] - m_new);
          l_run[n] *= alpha;
#pragma unroll
          for (int i = 0; i < NO; ++i) o[n][i] *= alpha;
          m_run[n] = m_new;
        }
        uint32_t w[2 * T];
#pragma unroll
        for (int j = 0; j < T; ++j) {
          float e[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][j][r], p.scale_log2, -m_run[n]));
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
        const shortx4 a0 = read_tr(vbuf + lds_chunk(TB, row, c) + 8 * (half & 1));
        if constexpr (T == 2) {
          const shortx4 a1 = read_tr(vbuf + lds_chunk(TB, 16 + row, c) + 8 * (half & 1));
          a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          a = a0;
        }
        return a;
      };
      if (__builtin_expect(masked && __builtin_amdgcn_ballot_w64(odd_v) != 0, 0)) {
        typedef __attribute__((address_space(3))) u32x2 lds4;
        typedef __attribute__((address_space(3))) shortx8 lds8;
#pragma unroll 1
        for (int k = 0; k < KW; ++k) {
#pragma unroll
          for (int i = 0; i < NO; ++i) {
            const u32x2 v = *reinterpret_cast<const lds4*>(vbuf + lds_chunk(TB, k, 2 * i + (g >> 1)) + 8 * (g & 1));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                o[n][i][r] = add_nonfinite<E>(o[n][i][r], (v[r >> 1] >> (16 * (r & 1))) & 0xffffu, key0 + k < lim[n]);
          }
        }
#pragma unroll 1
        for (int at = 16 * lane; at < T * TB; at += 1024)
          *reinterpret_cast<lds8*>(vbuf + at) = finite8<E>(*reinterpret_cast<const lds8*>(vbuf + at));
      }
#pragma unroll
      for (int i = 0; i < NO; ++i) {
        const vp a = vfrag(i);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][i] = Mat<E>::mfma16(a, pb[n], o[n][i]);
      }
    };

    // Two steps in flight: while one is computed the next one's rows are on
    // their way, and the page numbers of the one after that.
    {
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

    // Join the four waves: rows' sums over the lanes, then maxima, sums and O
    // through LDS, in the order of the waves.
    const bool whole = blk0 == 0 && blk1 == nb;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (u_first < u - blk0 ? 1 : 0);   // see decode_slots
    if (threadIdx.x == 0) bad_s = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float l = l_run[n];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      __syncthreads();                         // V tiles (and the last tile's exchange) have been read
      if (g == 0) m_s[wave][x] = m_run[n];
      if (n == 0 && __builtin_amdgcn_ballot_w64(bad) && lane == 0) bad_s = 1;
      __syncthreads();
      const float M = __builtin_fmaxf(__builtin_fmaxf(m_s[0][x], m_s[1][x]), __builtin_fmaxf(m_s[2][x], m_s[3][x]));
      const float w = __builtin_amdgcn_exp2f(m_run[n] - M);
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
    if (bad_s && threadIdx.x == 0 && !(sq.flags & LVSA_PAGED_BAD_LENGTH)) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
    __syncthreads();                           // the exchange has been read: V tiles and bad_s may be written
    u += blk1 - blk0;
  }
}

// ─────────────────────────────── prefill ───────────────────────────────────

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

// Four waves of 32 rows.  Key blocks of 64 keys in two LDS stages: wave w
// brings tile w (16 keys) of the next block while all four work on the current
// one.  16-bit pages are copied without passing registers; of 4-bit pages the
// codes are loaded at the start of a step and written to LDS as 16-bit values
// at its end, so every row is decoded once for 128 query rows.
template <int D, typename E, int BITS>
__global__ __launch_bounds__(256, D >= 192 ? 1 : 2) void paged_prefill_kernel(PagedAttnParams p) {
  constexpr int ND = D / 32, NK = D / 16, NO = D / 32;
  constexpr int TB = 32 * D, MAT = 4 * TB, STAGE = 2 * MAT;   // 16-key tile, 64-key matrix, K and V
  constexpr bool kTwoScales = D == 96 || D >= 192;
  __shared__ __attribute__((aligned(1024))) char smem_raw[2 * STAGE];
  lds_char* smem = (lds_char*)smem_raw;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, i32 = lane & 31;       // S^T: column (row of the tile) i32
  const int g = lane >> 4, x = lane & 15;

  // rows before the first and behind the last sequence
  if (p.fill_tail) {
    const int head = p.c.cu[0] < 0 ? 0 : p.c.cu[0] > p.c.N ? p.c.N : p.c.cu[0];
    const int tail = p.c.cu[p.c.B] < head ? head : p.c.cu[p.c.B] > p.c.N ? p.c.N : p.c.cu[p.c.B];
    const int64_t n = (int64_t)(head + p.c.N - tail) * p.H;
    const int64_t wg = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, wgs = (int64_t)gridDim.x * gridDim.y;
    for (int64_t i = wg * 4 + wave; i < n; i += 4 * wgs) {
      const int64_t r = i / p.H, hq = i - r * p.H, t = r < head ? r : tail + (r - head);
      for (int d = lane; d < D; d += 64) reinterpret_cast<uint16_t*>(p.o + t * p.o_str[0] + hq * p.o_str[1])[d] = 0;
      if (p.lse && lane == 0) p.lse[t * p.H + hq] = -__builtin_inff();
    }
  }

  // Tile and key head of this work-group.  Tiles run from the last to the
  // first: with a causal order the later ones are the longer ones, and a
  // launch that ends on short tiles ends evenly.  Consecutive work-groups,
  // which go to different XCDs, are the key heads of one tile, so an XCD keeps
  // to a few heads and their keys stay in its L2.
  const int h = (int)(blockIdx.x % (uint32_t)p.c.Hkv);
  const int64_t want = p.tiles - 1 - (int64_t)(blockIdx.x / (uint32_t)p.c.Hkv);
  int seq = -1;
  int64_t base = 0;
  int flags = 0;
  for (int s0 = 0; s0 < p.c.B; s0 += 64) {
    int64_t n = 0;
    if (s0 + lane < p.c.B) {
      const PagedSeq q = paged_seq(p.c, s0 + lane);
      n = ((int64_t)q.n * p.group + kPagedTile - 1) / kPagedTile;
      flags |= q.flags;
    }
    const int64_t incl = wave_scan(n, lane);
    const uint64_t above = __builtin_amdgcn_ballot_w64(base + incl > want);
    if (above) {
      const int at = __builtin_ctzll(above);
      seq = s0 + at;
      base += __shfl(incl - n, at);
      break;
    }
    base += __shfl(incl, 63);
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && wave == 0 && flags) paged_flag(p.c, flags);
  if (seq < 0) return;                              // the launch's bound, past the last tile
  const PagedSeq sq = paged_seq(p.c, seq);
  const int nrows = sq.n * p.group;
  const int r0 = (int)(want - base) * kPagedTile;
  const int r_last = r0 + kPagedTile < nrows ? r0 + kPagedTile - 1 : nrows - 1;
  const int lim_min = key_limit(p, sq, r0), lim_max = key_limit(p, sq, r_last);
  const int nb = (lim_max + kPagedBlock - 1) / kPagedBlock;
  const int blk0 = (int)((int64_t)nb * blockIdx.y / p.splits), blk1 = (int)((int64_t)nb * (blockIdx.y + 1) / p.splits);

  const int row = r0 + 32 * wave + i32;             // this lane's row of the pair
  const int rc = row < nrows ? row : nrows - 1;
  const RowRef ref = row_ref(p, sq, h, rc);
  const int lim = key_limit(p, sq, rc);
  shortx8 qf[NK];
  {
    const char* qp = p.q + ref.tok * p.q_str[0] + ref.head * p.q_str[1] + 16 * half;
#pragma unroll
    for (int c = 0; c < NK; ++c) qf[c] = *reinterpret_cast<const shortx8*>(qp + 32 * c);
  }

  const char* kbase = p.c.k + h * p.c.k_str[2];
  const char* vbase = p.c.v + h * p.c.v_str[2];
  const int32_t* table = p.c.table + seq * p.c.table_str;
  // The key of tile `wave` that this lane brings (past the end: the last key).
  // 16 bits: chunks 4 i + g of key x ^ 8 (g & 1), so that a copy's fixed order
  // in LDS is the tile's layout.
  const int my_key = 16 * wave + (BITS == 16 ? x ^ (8 * (g & 1)) : x);
  auto key_pos = [&](int b) __attribute__((always_inline)) {
    return key_within(b * kPagedBlock + my_key, sq.L);
  };
  bool bad = (sq.flags & LVSA_PAGED_BAD_LENGTH) != 0;
  auto row_of = [&](int b, int page, int64_t& pg, int64_t& slot) __attribute__((always_inline)) {
    const PagedRow at = paged_row(p.c, key_pos(b), page);
    bad |= !at.ok;
    pg = at.page;
    slot = at.slot;
  };
  auto bring16 = [&](int b, int page, lds_char* st) __attribute__((always_inline)) {
    int64_t pg, slot;
    row_of(b, page, pg, slot);
    const char* kr = kbase + pg * p.c.k_str[0] + slot * p.c.k_str[1] + 16 * g;
    const char* vr = vbase + pg * p.c.v_str[0] + slot * p.c.v_str[1] + 16 * g;
#pragma unroll
    for (int i = 0; i < ND; ++i) copy16(kr + 64 * i, st + wave * TB + 1024 * i);
#pragma unroll
    for (int i = 0; i < ND; ++i) copy16(vr + 64 * i, st + MAT + wave * TB + 1024 * i);
  };
  struct Codes {
    uint32_t k[ND], v[ND], ks[2], vs[2];
  } codes;
  auto load4 = [&](int b, int page) __attribute__((always_inline)) {
    int64_t pg, slot;
    row_of(b, page, pg, slot);
    const uint32_t* kw = reinterpret_cast<const uint32_t*>(kbase + pg * p.c.k_str[0] + slot * p.c.k_str[1] + (D / 8) * g);
    const uint32_t* vw = reinterpret_cast<const uint32_t*>(vbase + pg * p.c.v_str[0] + slot * p.c.v_str[1] + (D / 8) * g);
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      codes.k[i] = kw[i];
      codes.v[i] = vw[i];
    }
    const uint8_t* ks = p.c.ks + h * p.c.ks_str[2] + pg * p.c.ks_str[0] + slot * p.c.ks_str[1];
    const uint8_t* vs = p.c.vs + h * p.c.vs_str[2] + pg * p.c.vs_str[0] + slot * p.c.vs_str[1];
    const int lo = (D / 4) * g / 32, hi = ((D / 4) * g + D / 4 - 1) / 32;
    codes.ks[0] = ks[lo];
    codes.vs[0] = vs[lo];
    codes.ks[1] = kTwoScales ? ks[hi] : 0;
    codes.vs[1] = kTwoScales ? vs[hi] : 0;
  };
  auto store4 = [&](lds_char* st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < ND; ++i) {
      const bool up = kTwoScales && ((D / 4) * g + 8 * i) / 32 != (D / 4) * g / 32;
      const int at = lds_chunk(TB, 16 * wave + x, ND * g + i);
      typedef __attribute__((address_space(3))) shortx8 lds8;
      *reinterpret_cast<lds8*>(st + at) = decode8<E>(codes.k[i], up ? codes.ks[1] : codes.ks[0]);
      *reinterpret_cast<lds8*>(st + MAT + at) = decode8<E>(codes.v[i], up ? codes.vs[1] : codes.vs[0]);
    }
  };

  // LDS reads.  K: key i32 (+ 32), elements 16 c + 8 half .. + 7.  V: keys 4
  // half + (x >> 2) (+ 8) of tile st, elements 32 dt + 16 ((lane >> 4) & 1) +
  // 4 (x & 3) .. + 3; the transposing read hands lane x element x of them.
  const int koff = lds_chunk(TB, i32, half);
  const int vrow = 4 * half + (x >> 2), vc = 2 * (g & 1) + ((x & 3) >> 1);
  const int voff0 = lds_chunk(TB, vrow, vc) + 8 * (x & 1), voff1 = lds_chunk(TB, vrow + 8, vc) + 8 * (x & 1);

  floatx16 o[NO];
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i] = floatx16{0};
  float m_run = kNoKeys, l_run = 0.f;

  auto compute = [&](int b, lds_char* ks) __attribute__((always_inline)) {
    lds_char* vs = ks + MAT;
    typedef const __attribute__((address_space(3))) shortx8 lds8;
    floatx16 s0 = floatx16{0}, s1 = floatx16{0};
#pragma unroll
    for (int c = 0; c < NK; ++c) {
      const shortx8 a0 = *reinterpret_cast<lds8*>(ks + koff + 512 * c);
      const shortx8 a1 = *reinterpret_cast<lds8*>(ks + koff + 512 * c + 2 * TB);
      s0 = Mat<E>::mfma32(a0, qf[c], s0);
      s1 = Mat<E>::mfma32(a1, qf[c], s1);
    }
    const bool masked = (b + 1) * kPagedBlock > lim_min;
    const int here = lim - b * kPagedBlock - 4 * half;   // keys of this block that the row attends, from 4 half on
    if (masked) {
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
      float m = __builtin_fmaxf(s0[4 * c], s0[4 * c + 1]);
      m = __builtin_fmaxf(__builtin_fmaxf(m, s0[4 * c + 2]), s0[4 * c + 3]);
      m = __builtin_fmaxf(__builtin_fmaxf(m, s1[4 * c]), s1[4 * c + 1]);
      t[c] = __builtin_fmaxf(__builtin_fmaxf(m, s1[4 * c + 2]), s1[4 * c + 3]);
    }
    float top = __builtin_fmaxf(__builtin_fmaxf(t[0], t[1]), __builtin_fmaxf(t[2], t[3])) * p.scale_log2;
    // the running maximum moves only when some score exceeds it by 2^8
    if (__builtin_amdgcn_ballot_w64(top > m_run + 8.0f)) {
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float m_new = __builtin_fmaxf(m_run, top);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] *= alpha;
      m_run = m_new;
    }
    shortx8 pb[4];
    float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const floatx16& s = st < 2 ? s0 : s1;
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * (st & 1) + 2 * j], p.scale_log2, -m_run));
        const float c = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * (st & 1) + 2 * j + 1], p.scale_log2, -m_run));
        ls[j] += a + c;
        w[j] = pack2<E>(a, c);
      }
      pb[st] = __builtin_bit_cast(shortx8, w);
    }
    l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);

    auto vfrag = [&](int st, int dt) __attribute__((always_inline)) {
      const shortx4 a = read_tr(vs + voff0 + st * TB + 1024 * dt), c = read_tr(vs + voff1 + st * TB + 1024 * dt);
      return __builtin_shufflevector(a, c, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    bool odd = false;
    if (masked) {
      #pragma unroll 1
      for (int i = lane; i < MAT / 16; i += 64) odd |= any_nonfinite<E>(*reinterpret_cast<lds8*>(vs + 16 * i));
    }
    if (__builtin_expect(masked && __builtin_amdgcn_ballot_w64(odd) != 0, 0)) {   // alike in all four waves
      typedef __attribute__((address_space(3))) u32x2 lds4;
#pragma unroll 1
      for (int k = 0; k < kPagedBlock; ++k) {
        const bool seen = b * kPagedBlock + k < lim;
#pragma unroll
        for (int q = 0; q < 4 * NO; ++q) {
          const u32x2 v = *reinterpret_cast<const lds4*>(vs + lds_chunk(TB, k, q) + 8 * half);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            o[q >> 2][4 * (q & 3) + r] =
                add_nonfinite<E>(o[q >> 2][4 * (q & 3) + r], (v[r >> 1] >> (16 * (r & 1))) & 0xffffu, seen);
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int at = 16 * (int)threadIdx.x; at < MAT; at += 4096)
        *reinterpret_cast<__attribute__((address_space(3))) shortx8*>(vs + at) = finite8<E>(*reinterpret_cast<lds8*>(vs + at));
      __syncthreads();
    }
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int dt = 0; dt < NO; ++dt) o[dt] = Mat<E>::mfma32(vfrag(st, dt), pb[st], o[dt]);
  };

  if (blk0 < blk1) {
    int page = table[page_of(p.c, key_pos(blk0))];
    if constexpr (BITS == 16) {
      bring16(blk0, page, smem);
    } else {
      load4(blk0, page);
      store4(smem);
    }
    page = table[page_of(p.c, key_pos(blk0 + 1))];
    auto step = [&](int b, lds_char* cur, lds_char* nxt) __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0F70);           // vmcnt(0): this wave's copies of block b have landed
      __syncthreads();                              // everyone's; and the other stage has been read
      if (b + 1 < blk1) {
        if constexpr (BITS == 16) bring16(b + 1, page, nxt);
        else load4(b + 1, page);
        page = table[page_of(p.c, key_pos(b + 2))];
      }
      compute(b, cur);
      if constexpr (BITS == 4) {
        if (b + 1 < blk1) store4(nxt);
      }
    };
    for (int b = blk0; b < blk1; b += 2) {
      step(b, smem, smem + STAGE);
      if (b + 1 < blk1) step(b + 1, smem + STAGE, smem);
    }
  }

  // A bad page seen by any wave spoils the tile.
  __shared__ int bad_s;
  if (threadIdx.x == 0) bad_s = 0;
  __syncthreads();
  if (__builtin_amdgcn_ballot_w64(bad) && lane == 0) bad_s = 1;
  __syncthreads();
  if (bad_s && threadIdx.x == 0 && !(sq.flags & LVSA_PAGED_BAD_LENGTH)) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);

  float l = l_run + __shfl_xor(l_run, 32);
  if (bad_s) l = __builtin_nanf("");
  if (row >= nrows) return;
  if (p.splits > 1) {
    const int64_t slot = (want * p.c.Hkv + h) * p.splits + blockIdx.y;
    const int64_t at = slot * kPagedTile + (row - r0);
#pragma unroll
    for (int dt = 0; dt < NO; ++dt)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq)
        *reinterpret_cast<floatx4*>(p.ws_o + at * D + 32 * dt + 8 * rq + 4 * half) =
            floatx4{o[dt][4 * rq], o[dt][4 * rq + 1], o[dt][4 * rq + 2], o[dt][4 * rq + 3]};
    if (half == 0) {
      p.ws_ml[2 * at] = m_run;
      p.ws_ml[2 * at + 1] = l;
    }
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  char* op = p.o + ref.tok * p.o_str[0] + ref.head * p.o_str[1];
#pragma unroll
  for (int dt = 0; dt < NO; ++dt)
#pragma unroll
    for (int rq = 0; rq < 4; ++rq)
      *reinterpret_cast<u32x2*>(op + 2 * (32 * dt + 8 * rq + 4 * half)) =
          u32x2{pack2<E>(o[dt][4 * rq] * inv, o[dt][4 * rq + 1] * inv),
                pack2<E>(o[dt][4 * rq + 2] * inv, o[dt][4 * rq + 3] * inv)};
  if (p.lse && half == 0)
    p.lse[ref.tok * p.H + ref.head] = l == 0.f ? -__builtin_inff() : (m_run + __log2f(l)) * 0.69314718055994530942f;
}

template <int D, typename E, int BITS>
int paged_launch(const PagedAttnParams& p, int rows, hipStream_t stream) {
  if (rows == kPagedTile) {
    hipLaunchKernelGGL((paged_prefill_kernel<D, E, BITS>), dim3((unsigned)(p.tiles * p.c.Hkv), (unsigned)p.splits),
                       dim3(256), 0, stream, p);
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
