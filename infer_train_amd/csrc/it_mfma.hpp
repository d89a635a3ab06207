// it_mfma.hpp -- what the attention kernels on the matrix cores share: 32x32x16
// products of 16-bit operands, loads from global memory straight into LDS, and
// sums over the two halves of a wave.
#pragma once
#include <hip/hip_runtime.h>

#include "it_device.hpp"

namespace itkv {

typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint32_t lds_off(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)p));
}
__device__ __forceinline__ void dma_b128(const void* g, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(m0), "v"(g) : "memory", "m0");
}
template <bool kBf16>
__device__ __forceinline__ v16f mfma(const uint4& a, const uint4& b, const v16f& c) {
  if constexpr (kBf16) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
}
// Two fp32 -> packed 16-bit pair (lo first), round to nearest even.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBf16) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    bf2 p;
    p[0] = (__bf16)lo;  // v_cvt_pk_bf16_f32
    p[1] = (__bf16)hi;
    return __builtin_bit_cast(uint32_t, p);
  } else {
    return f32_to_f16_bits(lo) | (f32_to_f16_bits(hi) << 16);
  }
}
// acc + lo + hi of a packed bf16 / f16 pair (v_dot2c_f32_*).
template <bool kBf16>
__device__ __forceinline__ float dot2_ones(uint32_t w, float acc, uint32_t ones) {
  if constexpr (kBf16) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2, w), __builtin_bit_cast(bf2, ones), acc, false);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), __builtin_bit_cast(h2, ones), acc, false);
  }
}
// max / sum of x over this lane and lane ^ 32 (v_permlane32_swap, no LDS).
__device__ __forceinline__ float max_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

}  // namespace itkv
