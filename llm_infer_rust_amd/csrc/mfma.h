// The 32 x 32 x 16 matrix product of 16-bit elements and what the prefill kernels share around it.
#pragma once

#include "common.h"

namespace mi355x {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

template <int DT>
struct Mfma;

template <>
struct Mfma<0> {
  __device__ __forceinline__ static floatx16 run(const uint4& a, const uint4& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};

template <>
struct Mfma<1> {
  __device__ __forceinline__ static floatx16 run(const uint4& a, const uint4& b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16;

// q = x / d, r = x % d for 0 <= x < 2^22 and 1 <= d, via a float reciprocal and one
// correction step each way.
__device__ __forceinline__ int div_small(int x, int d, float inv, int& r) {
  int q = static_cast<int>(static_cast<float>(x) * inv);
  r = x - q * d;
  if (r >= d) {
    ++q;
    r -= d;
  }
  if (r < 0) {
    --q;
    r += d;
  }
  return q;
}

}  // namespace mi355x
