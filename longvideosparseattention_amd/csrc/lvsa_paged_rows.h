// Rows of the paged cache in registers: 16-bit elements and 4-bit codes, eight at
// a time, from and to what is stored.
#pragma once
#include "lvsa_paged.h"

namespace lvsa {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename E> struct Half;
template <> struct Half<__bf16> {
  static constexpr uint32_t kNaN = 0x7fc0u;
  __device__ static void unpack(u32x4 u, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __builtin_bit_cast(float, u[i] << 16);
      x[2 * i + 1] = __builtin_bit_cast(float, u[i] & 0xffff0000u);
    }
  }
};
template <> struct Half<_Float16> {
  static constexpr uint32_t kNaN = 0x7e00u;
  __device__ static void unpack(u32x4 u, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)u[i]);
      x[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u[i] >> 16));
    }
  }
};
template <typename E>
__device__ __forceinline__ u32x4 pack8(const float* x) {
  u32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    typedef E v2 __attribute__((ext_vector_type(2)));
    u[i] = __builtin_bit_cast(uint32_t, v2{(E)x[2 * i], (E)x[2 * i + 1]});
  }
  return u;
}

// Eight 4-bit values at byte scale `s` (2^(s - 127), 255: NaN).  Exact in both
// types for the scales that the append writes.
template <typename E>
__device__ __forceinline__ u32x4 unpack_e2m1(uint32_t codes, uint32_t s) {
  const float f = __builtin_bit_cast(float, s << 23);
  u32x4 u;
  if constexpr (__is_same(E, __bf16)) {
    u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 0));
    u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 1));
    u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 2));
    u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, f, 3));
  } else {
    u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, f, 0));
    u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, f, 1));
    u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, f, 2));
    u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, f, 3));
  }
  return u;
}

}  // namespace
}  // namespace lvsa
