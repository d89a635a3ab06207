// it_rows.hpp -- rows of F32, F16 or BF16 elements as float vectors, and their
// single elements.
#pragma once
#include <hip/hip_runtime.h>

#include "it_device.hpp"
#include "it_kv.h"
#include "it_quant.hpp"

namespace itkv {

// Two floats as bf16, each rounded to nearest even (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair p = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
  return __builtin_bit_cast(uint32_t, p);
}

// V elements of dtype DT at an address aligned to their size, 16 bytes at most <-> floats.
template <int DT, int V>
struct RowVec {
  static constexpr int kWords = DT == IT_F32 ? V : V / 2;
  static constexpr int kAlign = kWords * 4 < 16 ? kWords * 4 : 16;
  typedef uint32_t vec __attribute__((ext_vector_type(DT == IT_F32 ? V : V / 2)));
  typedef vec raw __attribute__((aligned(kAlign)));
  static __device__ __forceinline__ void widen(const raw& w, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (DT == IT_F32) {
        x[i] = __uint_as_float(w[i]);
      } else if constexpr (DT == IT_BF16) {
        x[2 * i] = bf16_lo(w[i]);
        x[2 * i + 1] = bf16_hi(w[i]);
      } else {
        x[2 * i] = f16_bits_to_f32(w[i] & 0xFFFFu);
        x[2 * i + 1] = f16_bits_to_f32(w[i] >> 16);
      }
    }
  }
  // Rounded to nearest even, once.
  static __device__ __forceinline__ raw narrow(const float (&x)[V]) {
    raw w;
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (DT == IT_F32) {
        w[i] = __float_as_uint(x[i]);
      } else if constexpr (DT == IT_BF16) {
        w[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
      } else {
        w[i] = f16_bits_rne(x[2 * i]) | (f16_bits_rne(x[2 * i + 1]) << 16);
      }
    }
    return w;
  }
};
template <int V>
__device__ __forceinline__ void store_row_vec(void* base, int64_t element, int dtype, const float (&x)[V]) {
  if (dtype == IT_F32)
    *reinterpret_cast<typename RowVec<IT_F32, V>::raw*>(static_cast<float*>(base) + element) = RowVec<IT_F32, V>::narrow(x);
  else if (dtype == IT_BF16)
    *reinterpret_cast<typename RowVec<IT_BF16, V>::raw*>(static_cast<uint16_t*>(base) + element) = RowVec<IT_BF16, V>::narrow(x);
  else
    *reinterpret_cast<typename RowVec<IT_F16, V>::raw*>(static_cast<uint16_t*>(base) + element) = RowVec<IT_F16, V>::narrow(x);
}

__device__ __forceinline__ float load_element(const void* base, int64_t element, int dtype) {
  if (dtype == IT_F32) return static_cast<const float*>(base)[element];
  const uint32_t b = static_cast<const uint16_t*>(base)[element];
  return dtype == IT_BF16 ? bf16_lo(b) : f16_bits_to_f32(b);
}
__device__ __forceinline__ void store_element(void* base, int64_t element, int dtype, float x) {
  if (dtype == IT_F32) static_cast<float*>(base)[element] = x;
  else static_cast<uint16_t*>(base)[element] = uint16_t(dtype == IT_BF16 ? bf16_pair(x, x) & 0xFFFFu : f16_bits_rne(x));
}

}  // namespace itkv
