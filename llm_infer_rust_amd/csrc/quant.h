// Row quantisation, shared by the 8-bit projections (quant.hip) and the 8-bit experts (experts.hip).
#pragma once

#include "product.h"

namespace mi355x {

// 16 elements of a row as floats; `n` of them exist, the others are 0.
template <int DT>
__device__ __forceinline__ void load16(const uint8_t* row, int64_t at, int n, float (&f)[16]) {
  constexpr int kSize = DT == kFloatOut ? 4 : 2;
  const uint8_t* p = row + at * kSize;
  if (n >= 16) {
    if constexpr (DT == kFloatOut) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 v = ld128_any(p + 16 * i);
        f[4 * i] = __uint_as_float(v.x), f[4 * i + 1] = __uint_as_float(v.y);
        f[4 * i + 2] = __uint_as_float(v.z), f[4 * i + 3] = __uint_as_float(v.w);
      }
    } else {
      float lo[8], hi[8];
      unpack8<DT>(ld128_any(p), lo);
      unpack8<DT>(ld128_any(p + 16), hi);
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

struct RowsToQuantize {
  const uint8_t* x;
  uint8_t* values;
  float* scales;
  int64_t stride, ldv, rows;  // stride in bytes
  int32_t width, chunks;      // chunks of 16 columns to write, zeros past the width
};

// A grid has fewer than 2^32 threads: of a larger one a part is launched, without an error.
constexpr int64_t kMaxGridThreads = (int64_t(1) << 32) - 1;
// Rows that one launch takes where up to 256 threads stand for each.
constexpr int64_t kMaxLaunchRows = int64_t(1) << 23;

inline RowsToQuantize rows_to_quantize(const void* x, int64_t stride, void* values, int64_t ldv,
                                       float* scales, int64_t rows, int64_t width,
                                       int64_t padded) {
  return {static_cast<const uint8_t*>(x), static_cast<uint8_t*>(values), scales, stride, ldv, rows,
          static_cast<int32_t>(width), static_cast<int32_t>(padded / 16)};
}

// K of an int8 product in bytes: the weight rows' elements and, where their stride `ld` holds them,
// the rest of the last 128-byte step, else of the last 16 bytes. The quantised rows are zeros
// there.
inline int64_t int8_k(int64_t k, int64_t ld) {
  const int64_t steps = (k + 127) / 128 * 128;
  return ld >= steps ? steps : (k + 15) / 16 * 16;
}

// One row per LANES threads (a wave, or four). The row's first HELD chunks of 16 a thread stay in
// registers between the two passes, the rest is read again. Bound by memory: every row is read once
// and written at half its size (8,192 rows of 4,096 bf16: 100 MB). `wave_top` is an LDS word a wave
// of the workgroup.
template <int DT, int LANES, int HELD>
__device__ __forceinline__ void quantize_row(const RowsToQuantize& q, int64_t row,
                                             uint32_t* wave_top) {
  static_assert(LANES == kWave || LANES == 4 * kWave, "a wave or four");
  const int lane = threadIdx.x % LANES;
  const bool there = row < q.rows;
  const uint8_t* src = q.x + (there ? row : 0) * q.stride;
  uint8_t* dst = q.values + row * q.ldv;
  const int chunks = there ? q.chunks : 0;
  float held[HELD][16];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = lane + h * LANES;
    if (c < chunks) {
      load16<DT>(src, c * 16, q.width - c * 16, held[h]);
      top = max(top, magnitude16(held[h]));
    }
  }
  for (int c = lane + HELD * LANES; c < chunks; c += LANES) {
    float f[16];
    load16<DT>(src, c * 16, q.width - c * 16, f);
    top = max(top, magnitude16(f));
  }
  top = wave_max(top);
  if constexpr (LANES > kWave) {
    wave_top += threadIdx.x / LANES * 4;
    if (threadIdx.x % kWave == 0) wave_top[threadIdx.x % LANES / kWave] = top;
    __syncthreads();
    top = max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3]));
  }
  const RowQuant form(top);
  if (there && lane == 0) q.scales[row] = form.scale;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = lane + h * LANES;
    if (c < chunks) st128(dst + c * 16, form.values(held[h]));
  }
  for (int c = lane + HELD * LANES; c < chunks; c += LANES) {
    float f[16];
    load16<DT>(src, c * 16, q.width - c * 16, f);
    st128(dst + c * 16, form.values(f));
  }
}

// values[r, :] and scales[r] of `rows` rows of `width` elements (dtype 0 bf16, 1 fp16, 2 fp32), row
// stride in bytes. Columns up to `padded`, a multiple of 16, are written as zeros.
const char* run_quantize_rows(const void* x, int64_t stride, void* values, int64_t ldv,
                              float* scales, int64_t rows, int64_t width, int64_t padded, int dtype,
                              hipStream_t s);

}  // namespace mi355x
