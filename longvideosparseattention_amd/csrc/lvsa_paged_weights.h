// Weights that the newest rows give to the cached tokens (gfx950): w_j (+)= sum_i
// exp(scale q_i.k_j - lse_i) over the rows of a sequence and the query heads of a key
// head.
#pragma once
#include "lvsa_paged_attn.h"

namespace lvsa {
namespace {

constexpr int kWeightTiles = 2;            // 16-key tiles of a wave

// Writes a lane group's sums: lane x < 4 of group g has key 4 g + x of a 16-key tile.
__device__ __forceinline__ void store_weight(const PagedAttnParams& p, const WeightsParams& wp, const PagedSeq& sq, int h, int key,
                                             const PagedRow& at, float sum) {
  float* w = reinterpret_cast<float*>(wp.w + at.page * wp.w_str[0] + at.slot * wp.w_str[1] + h * wp.w_str[2]);
  *w = (wp.accumulate && key < sq.first ? *w : 0.f) + sum;
}

template <int D, typename E, int BITS>
__global__ __launch_bounds__(256) void paged_weights_kernel(PagedAttnParams p, WeightsParams wp) {
  constexpr int T = kWeightTiles, ND = D / 32, KW = 16 * T, KEYS = 4 * KW;
  constexpr bool kTwoScales = D == 96 || D >= 192;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int g = lane >> 4, x = lane & 15;
  auto count = [&](const PagedSeq& s) __attribute__((always_inline)) {
    return s.n ? ((int64_t)s.L + KEYS - 1) / KEYS * p.c.Hkv : (int64_t)0;
  };
  walk_units(p.c, count, [&](int seq, const PagedSeq& sq, int64_t u) __attribute__((always_inline)) {
    const int chunk = (int)quotient(u, p.c.Hkv), h = (int)(u - (int64_t)chunk * p.c.Hkv);
    const int key0 = chunk * KEYS + wave * KW;
    if (key0 >= sq.L) return;
    const int32_t* table = p.c.table + seq * p.c.table_str;
    shortx8 kf[T][ND];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int pos = key_within(key0 + 16 * j + x, sq.L);
      const PagedRow at = paged_row(p.c, pos, table[page_of(p.c, pos)]);
      bad |= !at.ok;
      const char* kr = p.c.k + h * p.c.k_str[2] + at.page * p.c.k_str[0] + at.slot * p.c.k_str[1];
      if constexpr (BITS == 16) {
#pragma unroll
        for (int i = 0; i < ND; ++i) kf[j][i] = *reinterpret_cast<const shortx8*>(kr + 64 * i + 16 * g);
      } else {
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(kr + (D / 8) * g);
        const uint8_t* ks = p.c.ks + h * p.c.ks_str[2] + at.page * p.c.ks_str[0] + at.slot * p.c.ks_str[1];
        const uint32_t lo = ks[(D / 4) * g / 32], hi = kTwoScales ? ks[((D / 4) * g + D / 4 - 1) / 32] : lo;
#pragma unroll
        for (int i = 0; i < ND; ++i)
          kf[j][i] = decode8<E>(kw[i], kTwoScales && ((D / 4) * g + 8 * i) / 32 != (D / 4) * g / 32 ? hi : lo);
      }
    }
    if (bad) paged_flag(p.c, LVSA_PAGED_BAD_PAGE);
    float acc[T][4] = {};
    const int nrows = sq.n * p.group;
    int from = 0;                          // the first row that attends key0
    if (p.causal && key0 > sq.first) from = (key0 - sq.first) * p.group / 16 * 16;
    for (int r0 = from; r0 < nrows; r0 += 16) {
      const int r = r0 + x < nrows ? r0 + x : nrows - 1;
      const RowRef ref = row_ref(p, sq, h, r);
      const char* qp = p.q + ref.tok * p.q_str[0] + ref.head * p.q_str[1];
      shortx8 qf[ND];
#pragma unroll
      for (int i = 0; i < ND; ++i) qf[i] = *reinterpret_cast<const shortx8*>(qp + 2 * (BITS == 16 ? 32 * i + 8 * g : (D / 4) * g + 8 * i));
      const float lse = wp.lse[ref.tok * p.H + ref.head] * 1.4426950408889634f;
      const int lim = r0 + x < nrows && __builtin_fabsf(lse) < __builtin_inff() ? key_limit(p, sq, r) - key0 : 0;
#pragma unroll
      for (int j = 0; j < T; ++j) {
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < ND; ++i) s = Mat<E>::mfma16(kf[j][i], qf[i], s);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], p.scale_log2, -lse));
          acc[j][k] += 16 * j + 4 * g + k < lim ? w : 0.f;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < T; ++j) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a = acc[j][k];
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) a += __shfl_xor(a, d);
        const int key = key0 + 16 * j + 4 * g + k;
        if (x == k && key < sq.L) {
          const PagedRow at = paged_row(p.c, key, table[page_of(p.c, key)]);
          if (at.ok) store_weight(p, wp, sq, h, key, at, a);
        }
      }
    }
  });
}

template <int D, typename E, int BITS>
int paged_weights_launch(const PagedAttnParams& p, const WeightsParams& w, hipStream_t stream) {
  hipLaunchKernelGGL((paged_weights_kernel<D, E, BITS>), dim3((unsigned)p.grid), dim3(256), 0, stream, p, w);
  return launch_status("lvsa_paged_weights");
}

template <int D>
int paged_weights_launch(const PagedAttnParams& p, const WeightsParams& w, int bits, bool bf16, hipStream_t stream) {
  if (bf16) return bits == 16 ? paged_weights_launch<D, __bf16, 16>(p, w, stream) : paged_weights_launch<D, __bf16, 4>(p, w, stream);
  return bits == 16 ? paged_weights_launch<D, _Float16, 16>(p, w, stream) : paged_weights_launch<D, _Float16, 4>(p, w, stream);
}

}  // namespace
}  // namespace lvsa
