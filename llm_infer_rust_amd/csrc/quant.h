// Row quantisation, shared by the 8-bit projections (quant.hip) and the 8-bit experts (experts.hip).
#pragma once

#include "product.h"

namespace mi355x {

// 16 elements of a row as floats; `n` of them exist, the others are 0.
template <int DT>
__device__ __forceinline__ void load16(const uint8_t* row, int64_t at, int n, bool vec,
                                       float (&f)[16]) {
  constexpr int kSize = DT == kFloatOut ? 4 : 2;
  const uint8_t* p = row + at * kSize;
  if (vec && n >= 16) {
    if constexpr (DT == kFloatOut) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(p + 16 * i);
        f[4 * i] = v.x, f[4 * i + 1] = v.y, f[4 * i + 2] = v.z, f[4 * i + 3] = v.w;
      }
    } else {
      float lo[8], hi[8];
      unpack8<DT>(ld128(p), lo);
      unpack8<DT>(ld128(p + 16), hi);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = lo[i], f[8 + i] = hi[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i >= n) {
        f[i] = 0.f;
      } else if constexpr (DT == kFloatOut) {
        f[i] = reinterpret_cast<const float*>(p)[i];
      } else {
        f[i] = Elem<DT>::to_float(reinterpret_cast<const uint16_t*>(p)[i]);
      }
    }
  }
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(v, d)));
  return v;
}

// The largest magnitude of 16 elements, as its bits: inf and NaN come out on top.
__device__ __forceinline__ uint32_t magnitude16(const float (&f)[16]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  return top;
}

// The 8-bit form of a row whose largest magnitude is known. A row with an inf or a NaN gets the
// scale NaN, so its products are NaN and no other row's. The quotient 127 x / max is correctly
// rounded (q0 = p r with the correctly rounded reciprocal r, then one residual step, after
// P. Markstein, IBM J. Res. Dev. 34, 1990), which makes q the nearest integer of the exact
// quotient for 16-bit x: 127 x is exact there and no quotient of such numbers lies closer to a half
// than fp32 resolves. Rows near the ends of the fp32 range are scaled by 2^-32 or 2^64 first.
struct RowQuant {
  float scale, a, p127, r;
  bool finite;

  __device__ __forceinline__ explicit RowQuant(uint32_t top) {
    const float largest = __uint_as_float(top);
    finite = top < 0x7f800000u;
    scale = finite ? largest / 127.f : __uint_as_float(0x7fc00000u);
    const float range = largest > 1e30f ? 0x1p-32f : largest < 1e-30f ? 0x1p64f : 1.f;
    a = largest * range;
    p127 = 127.f * range;
    r = finite && top != 0 ? 1.f / a : 0.f;
  }
  __device__ __forceinline__ uint4 values(const float (&f)[16]) const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = f[4 * i + e] * p127;
        const float q0 = p * r;
        const float q = fmaf(fmaf(-q0, a, p), r, q0);
        // 1.5 * 2^23 leaves the rounded integer in the low bits (half to even)
        b[e] = __float_as_uint(q + 12582912.f) & 0xffu;
      }
      w[i] = finite ? b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24 : 0u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// values[r, :] and scales[r] of `rows` rows of `width` elements (dtype 0 bf16, 1 fp16, 2 fp32), row
// stride in bytes. Columns up to the next multiple of 16 are written as zeros.
const char* run_quantize_rows(const void* x, int64_t stride, void* values, int64_t ldv,
                              float* scales, int64_t rows, int64_t width, int dtype,
                              hipStream_t s);

}  // namespace mi355x
