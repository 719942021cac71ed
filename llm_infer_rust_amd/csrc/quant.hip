// 8-bit projections on gfx950: rows quantised to int8 with one scale a token, int8 products with one
// scale an output channel.
//
//   sx[m] = max_k |x[m,k]| / 127,   q[m,k] = rint(127 x[m,k] / max_k |x[m,k]|)
//   out[m,n] = sx[m] sw[n] sum_k q[m,k] w[n,k]          (int32 sums, one rounding)
//
// Replaces the projections of src/layers/linear.rs:5-7 for weights held in 8 bits; the reference
// itself has none.
#include <algorithm>

#include "product_vec.h"

namespace mi355x {
namespace {

// One row per LANES threads (a wave, or the whole workgroup of 256). The row's first HELD chunks of
// 16 a thread stay in registers between the two passes, the rest is read again. Bound by memory:
// every row is read once and written at half its size (8,192 rows of 4,096 bf16: 100 MB).
template <int DT, int LANES, int HELD>
__global__ __launch_bounds__(256) void quantize_rows(const uint8_t* __restrict__ x, int64_t stride,
                                                     uint8_t* __restrict__ values, int64_t ldv,
                                                     float* __restrict__ scales, int64_t rows,
                                                     int width, bool vec) {
  constexpr int kRows = 256 / LANES;
  __shared__ uint32_t wave_top[4];
  const int64_t row = blockIdx.x * int64_t(kRows) + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  if (LANES == kWave && row >= rows) return;
  const uint8_t* src = x + row * stride;
  uint8_t* dst = values + row * ldv;
  const int chunks = (width + 15) >> 4;
  float held[HELD][16];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = lane + h * LANES;
    if (c < chunks) {
      load16<DT>(src, c * 16, width - c * 16, vec, held[h]);
      top = max(top, magnitude16(held[h]));
    }
  }
  for (int c = lane + HELD * LANES; c < chunks; c += LANES) {
    float f[16];
    load16<DT>(src, c * 16, width - c * 16, vec, f);
    top = max(top, magnitude16(f));
  }
  top = wave_max(top);
  if constexpr (LANES > kWave) {
    if (threadIdx.x % kWave == 0) wave_top[threadIdx.x / kWave] = top;
    __syncthreads();
    top = max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3]));
  }
  const RowQuant q(top);
  if (lane == 0) scales[row] = q.scale;
  auto put = [&](int c, const float (&f)[16]) { st128(dst + c * 16, q.values(f)); };
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = lane + h * LANES;
    if (c < chunks) put(c, held[h]);
  }
  for (int c = lane + HELD * LANES; c < chunks; c += LANES) {
    float f[16];
    load16<DT>(src, c * 16, width - c * 16, vec, f);
    put(c, f);
  }
}

template <int DT>
void launch_quantize(const uint8_t* x, int64_t stride, uint8_t* values, int64_t ldv, float* scales,
                     int64_t rows, int width, bool vec, hipStream_t s) {
  // A wave a row where that keeps the row in registers, a workgroup a row for longer ones.
  if (width <= 1024)
    quantize_rows<DT, kWave, 1><<<dim3(static_cast<uint32_t>((rows + 3) / 4)), 256, 0, s>>>(
        x, stride, values, ldv, scales, rows, width, vec);
  else if (width <= 4096)
    quantize_rows<DT, 256, 1><<<dim3(static_cast<uint32_t>(rows)), 256, 0, s>>>(
        x, stride, values, ldv, scales, rows, width, vec);
  else
    quantize_rows<DT, 256, 3><<<dim3(static_cast<uint32_t>(rows)), 256, 0, s>>>(
        x, stride, values, ldv, scales, rows, width, vec);
}

constexpr int64_t kMaxInt8K = 131072;  // 127 * 127 * K stays inside int32

int64_t padded16(int64_t n) { return (n + 15) / 16 * 16; }

struct Int8Workspace {
  int64_t values, scales, bytes;
};

// One or two rows are quantised inside the product (see product_vec.h) where they fit its LDS.
bool on_vector_math(int64_t M, int64_t K) { return M <= 2 && M * padded16(K) <= kVecLds; }

Int8Workspace int8_workspace(int64_t M, int64_t K) {
  Int8Workspace w{};
  if (on_vector_math(M, K)) return w;
  w.values = 0;
  w.scales = padded16(M * padded16(K));
  w.bytes = w.scales + padded16(M * 4);
  return w;
}

template <int OT, bool SILU>
void launch_int8_vec(const ProductArgs& base, int64_t M, int64_t columns, int width, bool vec,
                     hipStream_t s) {
  ProductArgs a = base;
  constexpr int kWaves = 16, kRows = 2;
  const int bn = kWaves * (SILU ? kRows / 2 : kRows);
  a.tiles_m = 1;
  a.tiles_n = static_cast<int32_t>((columns + bn - 1) / bn);
  const dim3 g(static_cast<uint32_t>((a.tiles_n + 7) / 8 * 8));
  if (M == 1)
    product_vec<kInt8, OT, OT, kDense, SILU, 1, kRows, kWaves><<<g, 64 * kWaves, 0, s>>>(a, width, vec);
  else
    product_vec<kInt8, OT, OT, kDense, SILU, 2, kRows, kWaves><<<g, 64 * kWaves, 0, s>>>(a, width, vec);
}

template <int OT, bool SILU>
void launch_int8(const ProductArgs& base, int64_t M, int64_t columns, hipStream_t s) {
  ProductArgs a = base;
  auto grid = [&](int bm, int bn) {
    a.tiles_m = static_cast<int32_t>((M + bm - 1) / bm);
    a.tiles_n = static_cast<int32_t>((columns + bn - 1) / bn);
    return dim3(static_cast<uint32_t>((int64_t(a.tiles_m) * a.tiles_n + 7) / 8 * 8));
  };
  if (M <= 16) {
    const dim3 g = grid(16, SILU ? 16 : 32);
    product_rows<kInt8, OT, kDense, SILU, 2, 4><<<g, 256, 0, s>>>(a);
  } else if (M <= 256) {
    const dim3 g = grid(64, SILU ? 32 : 64);
    product_tile<kInt8, OT, kDense, SILU, 64, 64, 2, 2, 4><<<g, 256, 0, s>>>(a);
  } else {
    const dim3 g = grid(256, SILU ? 128 : 256);
    if (a.k_bytes % kProdRow)
      product_large<kInt8, OT, kDense, SILU, 256, 8, true><<<g, 512, 0, s>>>(a);
    else
      product_large<kInt8, OT, kDense, SILU, 256, 8, false><<<g, 512, 0, s>>>(a);
  }
}

}  // namespace

const char* run_quantize_rows(const void* x, int64_t stride, void* values, int64_t ldv,
                              float* scales, int64_t rows, int64_t width, int dtype,
                              hipStream_t s) {
  const bool vec = aligned(x, 16) && stride % 16 == 0;
  const auto* xb = static_cast<const uint8_t*>(x);
  auto* vb = static_cast<uint8_t*>(values);
  if (dtype == 0)
    launch_quantize<0>(xb, stride, vb, ldv, scales, rows, static_cast<int>(width), vec, s);
  else if (dtype == 1)
    launch_quantize<1>(xb, stride, vb, ldv, scales, rows, static_cast<int>(width), vec, s);
  else
    launch_quantize<2>(xb, stride, vb, ldv, scales, rows, static_cast<int>(width), vec, s);
  return launch_status("quantize_rows");
}

}  // namespace mi355x

using namespace mi355x;

extern "C" const char* mi355x_quantize_rows(const void* x, int64_t ldx, void* values, int64_t ldv,
                                            void* scales, int64_t rows, int64_t width, int dtype,
                                            void* stream) {
  if (rows < 0 || width <= 0 || width > (int64_t(1) << 30) || rows >= (int64_t(1) << 31) ||
      ldx < width || ldv < width || ldv % 16 || dtype < 0 || dtype > 2)
    return set_error("mi355x_quantize_rows: unsupported shape (rows of values in 16-byte steps)");
  if (rows == 0) return nullptr;
  if (!x || !values || !scales) return set_error("mi355x_quantize_rows: null pointer");
  if (!aligned(values, 16) || !aligned(scales, 4) || !aligned(x, dtype == 2 ? 4 : 2))
    return set_error("mi355x_quantize_rows: misaligned operand");
  return run_quantize_rows(x, ldx * (dtype == 2 ? 4 : 2), values, ldv,
                           static_cast<float*>(scales), rows, width, dtype,
                           static_cast<hipStream_t>(stream));
}

extern "C" int64_t mi355x_linear_int8_workspace_bytes(int64_t M, int64_t K) {
  if (M < 0 || K <= 0 || K > kMaxInt8K || M > (int64_t(1) << 24)) return -1;
  return int8_workspace(M, K).bytes;
}

extern "C" const char* mi355x_linear_int8(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                          const float* w_scales, void* out, int64_t ldo, int64_t M,
                                          int64_t N, int64_t K, bool silu_mul, void* workspace,
                                          int64_t workspace_bytes, int64_t dtype, void* stream) {
  const int64_t columns = silu_mul ? N / 2 : N;
  if (M < 0 || N <= 0 || K <= 0 || K > kMaxInt8K || N > (int64_t(1) << 24) ||
      M > (int64_t(1) << 24) || (silu_mul && N % 2) || ldx < K || ldo < columns ||
      ldw < padded16(K) || ldw % 16 || ldw * N >= (int64_t(1) << 32) ||
      (dtype != 0 && dtype != 1))
    return set_error("mi355x_linear_int8: unsupported shape (K up to 131072, weight rows of whole "
                     "16-byte words, less than 4 GiB)");
  if (M == 0) return nullptr;
  const Int8Workspace ws = int8_workspace(M, K);
  if (!x || !w || !w_scales || !out || (!workspace && ws.bytes))
    return set_error("mi355x_linear_int8: null pointer");
  if (!aligned(x, 2) || !aligned(w, 16) || !aligned(w_scales, 4) || !aligned(out, 2) ||
      !aligned(workspace, 16))
    return set_error("mi355x_linear_int8: misaligned operand");
  if (workspace_bytes < ws.bytes) return set_error("mi355x_linear_int8: workspace too small");
  // More row and column tiles than a grid holds (16 x 16 is the smallest tile).
  if ((M + 15) / 16 * ((columns + 15) / 16) >= (int64_t(1) << 30))
    return set_error("mi355x_linear_int8: grid too large");
  auto s = static_cast<hipStream_t>(stream);
  ProductArgs a{};
  a.w = static_cast<const uint8_t*>(w);
  a.out = out;
  a.w_scales = w_scales;
  a.w_stride = ldw;
  a.ldo = ldo;
  a.rows = static_cast<int32_t>(M);
  a.columns = static_cast<int32_t>(columns);
  a.k_bytes = static_cast<int32_t>(padded16(K));
  a.vec_out = ldo % 4 == 0 && aligned(out, 8);
  a.vec16_out = ldo % 8 == 0 && aligned(out, 16);
  if (on_vector_math(M, K)) {
    a.x = static_cast<const uint8_t*>(x);
    a.x_stride = ldx * 2;
    const bool vec = aligned(x, 16) && ldx % 8 == 0;
    const int width = static_cast<int>(K);
    if (dtype == 0)
      silu_mul ? launch_int8_vec<0, true>(a, M, columns, width, vec, s)
               : launch_int8_vec<0, false>(a, M, columns, width, vec, s);
    else
      silu_mul ? launch_int8_vec<1, true>(a, M, columns, width, vec, s)
               : launch_int8_vec<1, false>(a, M, columns, width, vec, s);
    return launch_status("product (int8)");
  }
  auto* base = static_cast<uint8_t*>(workspace);
  auto* scales = reinterpret_cast<float*>(base + ws.scales);
  if (const char* e = run_quantize_rows(x, ldx * 2, base, padded16(K), scales, M, K,
                                        static_cast<int>(dtype), s))
    return e;
  a.x = base;
  a.x_scales = scales;
  a.x_stride = padded16(K);
  if (dtype == 0)
    silu_mul ? launch_int8<0, true>(a, M, columns, s) : launch_int8<0, false>(a, M, columns, s);
  else
    silu_mul ? launch_int8<1, true>(a, M, columns, s) : launch_int8<1, false>(a, M, columns, s);
  return launch_status("product (int8)");
}
