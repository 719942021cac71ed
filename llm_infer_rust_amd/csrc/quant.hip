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

template <int DT, int LANES, int HELD>
__global__ __launch_bounds__(256) void quantize_rows(RowsToQuantize q) {
  __shared__ uint32_t wave_top[4];
  const int64_t row = blockIdx.x * int64_t(256 / LANES) + threadIdx.x / LANES;
  quantize_row<DT, LANES, HELD>(q, row, wave_top);
}

template <int DT>
void launch_quantize(const RowsToQuantize& q, hipStream_t s) {
  const auto rows = static_cast<uint32_t>(q.rows);
  // A wave a row where that keeps the row in registers, a workgroup a row for longer ones.
  if (q.width <= 1024)
    quantize_rows<DT, kWave, 1><<<dim3((rows + 3) / 4), 256, 0, s>>>(q);
  else if (q.width <= 4096)
    quantize_rows<DT, 256, 1><<<dim3(rows), 256, 0, s>>>(q);
  else
    quantize_rows<DT, 256, 3><<<dim3(rows), 256, 0, s>>>(q);
}

constexpr int64_t kMaxInt8K = 131072;  // 127 * 127 * K stays inside int32

int64_t padded16(int64_t n) { return (n + 15) / 16 * 16; }

// How a product is computed.
struct Int8Plan {
  enum Kind { kVec, kRows, kTiles } kind;
  Tile tile;
  int splits;  // parts of K, summed by a pass of their own where there are several
};

// One or two rows go to vector math, which quantises them itself, where they fit its LDS; up to 16 to
// the rows kernel or the least estimate of the tiles. K is split where the tiles leave CUs without
// one: 4096 x 12288 at 64 rows 33 us whole. The rows kernel's step is 0.18 us a round of 32 columns a
// CU (4096 x 4096 at 16 rows 8.5 us, 4096 x 12288 22, 24576 x 4096 22).
Int8Plan int8_plan(int64_t M, int64_t N, int64_t K, int cus) {
  if (M <= 2 && M * padded16(K) <= kVecLds) return {Int8Plan::kVec, Tile::k64, 1};
  Int8Plan best{Int8Plan::kTiles, Tile::k64, 1};
  float best_us = 1e30f;
  const int64_t kb = padded16(K), steps = (kb + kProdRow - 1) / kProdRow;
  const float weights = static_cast<float>(N) * static_cast<float>(kb);
  if (M <= 16) {
    const float rounds = std::max(1.f, 1.1f * static_cast<float>(N) / (32.f * cus));
    best = {Int8Plan::kRows, Tile::k64, 1};
    best_us = 3.f + std::max(0.18f * steps * rounds, weights / 5.8e6f);
  }
  for (int i = 0; i < kTiles; ++i) {
    const TileShape& t = kTileShapes[i];
    const float tm = static_cast<float>((M + t.bm - 1) / t.bm);
    const float tn = static_cast<float>((N + t.bn - 1) / t.bn);
    for (int s = 1; s <= (i < 2 ? 8 : 1); s *= 2) {
      const int64_t per = (steps + s - 1) / s;
      if (s > 1 && (per < 4 || per * (s - 1) >= steps || tm * tn * (s / 2) >= cus)) break;
      float us = tile_estimate(static_cast<Tile>(i), tm * s, tn, per * kProdRow, weights,
                               M % 256 != 0 && M % 256 <= 128 && M < 256, cus);
      // the sums go out and come back at about 4.5 TB/s, in one more launch
      if (s > 1) us += 2.5f + 8e-6f / 4.5f * static_cast<float>(s * M * N);
      if (us < best_us) {
        best_us = us;
        best = {Int8Plan::kTiles, static_cast<Tile>(i), s};
      }
    }
  }
  return best;
}

struct Int8Workspace {
  int64_t values, scales, sums, bytes;
};

Int8Workspace int8_workspace(int64_t M, int64_t N, int64_t K, const Int8Plan& p) {
  Int8Workspace w{};
  if (p.kind == Int8Plan::kVec) return w;
  w.values = 0;
  w.scales = M * ((K + 127) / 128 * 128);
  w.sums = w.scales + padded16(M * 4);
  w.bytes = w.sums + (p.splits > 1 ? p.splits * M * (N + 3) / 4 * 4 * 4 + 64 : 0);
  return w;
}

// out from the int32 sums of the parts of K, four columns a thread.
template <int OT, bool SILU>
__global__ __launch_bounds__(256) void finish_splits(ProductArgs a, const int* __restrict__ sums,
                                                     int64_t lds) {
  const int quads = (a.columns + 3) / 4;
  const int64_t i = blockIdx.x * int64_t(256) + threadIdx.x;
  if (i >= static_cast<int64_t>(a.rows) * quads) return;
  const int row = static_cast<int>(i / quads);
  const int c = static_cast<int>(i - static_cast<int64_t>(row) * quads) * 4;
  const int64_t plane = static_cast<int64_t>(a.rows) * lds;
  const int* p = sums + row * lds + c;
  int v[4] = {}, u[4] = {};
  for (int s = 0; s < a.splits; ++s, p += plane) {
    const int4 g = *reinterpret_cast<const int4*>(p);
    v[0] += g.x, v[1] += g.y, v[2] += g.z, v[3] += g.w;
    if constexpr (SILU) {  // the up columns start anywhere; those past the end repeat the last one
#pragma unroll
      for (int e = 0; e < 4; ++e) u[e] += p[a.columns + min(e, a.columns - 1 - c)];
    }
  }
  const RowOut r{row, a.x_scales[row], 1.f};
  finish4<kInt8, OT, kDense, SILU>(a, r, c, a.w_scales, v, u);
}

template <int OT, bool SILU>
void launch_int8_vec(const ProductArgs& base, int64_t M, int64_t columns, int width,
                     hipStream_t s) {
  ProductArgs a = base;
  constexpr int kWaves = 16, kRows = 2;
  const int bn = kWaves * (SILU ? kRows / 2 : kRows);
  a.tiles_m = 1;
  a.tiles_n = static_cast<int32_t>((columns + bn - 1) / bn);
  const dim3 g(static_cast<uint32_t>((a.tiles_n + 7) / 8 * 8));
  if (M == 1)
    product_vec<kInt8, OT, OT, kDense, SILU, 1, kRows, kWaves><<<g, 64 * kWaves, 0, s>>>(a, width);
  else
    product_vec<kInt8, OT, OT, kDense, SILU, 2, kRows, kWaves><<<g, 64 * kWaves, 0, s>>>(a, width);
}

template <int OT, int MODE, bool SILU>
void launch_int8_tiles(ProductArgs& a, Tile tile, hipStream_t s) {
  const TileShape& t = kTileShapes[static_cast<int>(tile)];
  const int bn = SILU ? t.bn / 2 : t.bn;
  a.tiles_m = (a.rows + t.bm - 1) / t.bm;
  a.tiles_n = (a.columns + bn - 1) / bn;
  const dim3 g(static_cast<uint32_t>((int64_t(a.tiles_m) * a.tiles_n * a.splits + 7) / 8 * 8));
  if (tile == Tile::k64) {
    product_tile<kInt8, OT, MODE, SILU, 64, 64, 2, 2, 3><<<g, 256, 0, s>>>(a);
  } else if (tile == Tile::k128) {
    product_tile<kInt8, OT, MODE, SILU, 128, 128, 4, 2, 4><<<g, 512, 0, s>>>(a);
  } else if constexpr (MODE == kDense) {
    if (tile == Tile::k128Two)
      product_tile<kInt8, OT, MODE, SILU, 128, 128, 4, 2, 2><<<g, 512, 0, s>>>(a);
    else if (tile == Tile::k256x128)
      product_tile<kInt8, OT, MODE, SILU, 256, 128, 4, 2, 3><<<g, 512, 0, s>>>(a);
    else if (a.k_bytes % kProdRow)
      product_large<kInt8, OT, MODE, SILU, 256, 8, true><<<g, 512, 0, s>>>(a);
    else
      product_large<kInt8, OT, MODE, SILU, 256, 8, false><<<g, 512, 0, s>>>(a);
  }
}

template <int OT, bool SILU>
const char* launch_int8(const ProductArgs& base, const Int8Plan& p, int* sums, hipStream_t s) {
  ProductArgs a = base;
  a.splits = p.splits;
  if (p.kind == Int8Plan::kRows) {
    const int bn = SILU ? 16 : 32;
    a.tiles_m = 1;
    a.tiles_n = (a.columns + bn - 1) / bn;
    product_rows<OT, SILU, 2, 4>
        <<<dim3(static_cast<uint32_t>((a.tiles_n + 7) / 8 * 8)), 256, 0, s>>>(a);
  } else if (p.splits == 1) {
    launch_int8_tiles<OT, kDense, SILU>(a, p.tile, s);
  } else {
    ProductArgs parts = a;
    parts.out = sums;
    parts.columns = SILU ? 2 * a.columns : a.columns;
    parts.ldo = (parts.columns + 3) / 4 * 4;
    launch_int8_tiles<OT, kSplit, false>(parts, p.tile, s);
    if (const char* e = launch_status("product (int8)")) return e;
    const int64_t threads = static_cast<int64_t>(a.rows) * ((a.columns + 3) / 4);
    finish_splits<OT, SILU><<<dim3(static_cast<uint32_t>((threads + 255) / 256)), 256, 0, s>>>(
        a, sums, parts.ldo);
    return launch_status("finish_splits");
  }
  return launch_status("product (int8)");
}

}  // namespace

const char* run_quantize_rows(const void* x, int64_t stride, void* values, int64_t ldv,
                              float* scales, int64_t rows, int64_t width, int64_t padded, int dtype,
                              hipStream_t s) {
  for (int64_t r = 0; r < rows; r += kMaxLaunchRows) {
    const RowsToQuantize q = rows_to_quantize(
        static_cast<const uint8_t*>(x) + r * stride, stride, static_cast<uint8_t*>(values) + r * ldv,
        ldv, scales + r, std::min(kMaxLaunchRows, rows - r), width, padded);
    if (dtype == 0)
      launch_quantize<0>(q, s);
    else if (dtype == 1)
      launch_quantize<1>(q, s);
    else
      launch_quantize<2>(q, s);
    if (const char* e = launch_status("quantize_rows")) return e;
  }
  return nullptr;
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
                           static_cast<float*>(scales), rows, width, padded16(width), dtype,
                           static_cast<hipStream_t>(stream));
}

extern "C" int64_t mi355x_linear_int8_workspace_bytes(int64_t M, int64_t N, int64_t K,
                                                      int32_t cus) {
  if (M < 0 || N <= 0 || K <= 0 || K > kMaxInt8K || M > (int64_t(1) << 24) ||
      N > (int64_t(1) << 24))
    return -1;
  return M == 0 ? 0 : int8_workspace(M, N, K, int8_plan(M, N, K, cus > 0 ? cus : 256)).bytes;
}

extern "C" bool mi355x_linear_int8_plan(int64_t M, int64_t N, int64_t K, int32_t cus,
                                        int32_t* plan) {
  if (!plan || M == 0 || mi355x_linear_int8_workspace_bytes(M, N, K, cus) < 0) return false;
  const Int8Plan p = int8_plan(M, N, K, cus > 0 ? cus : 256);
  plan[0] = static_cast<int32_t>(p.kind);
  plan[1] = static_cast<int32_t>(p.tile);
  plan[2] = p.splits;
  return true;
}

extern "C" const char* mi355x_linear_int8(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                          const float* w_scales, void* out, int64_t ldo, int64_t M,
                                          int64_t N, int64_t K, bool silu_mul, void* workspace,
                                          int64_t workspace_bytes, int32_t cus, int64_t dtype,
                                          void* stream) {
  const int64_t columns = silu_mul ? N / 2 : N;
  if (M < 0 || N <= 0 || K <= 0 || K > kMaxInt8K || N > (int64_t(1) << 24) ||
      M > (int64_t(1) << 24) || (silu_mul && N % 2) || ldx < K || ldo < columns ||
      ldw < padded16(K) || ldw % 16 || ldw * N >= (int64_t(1) << 32) ||
      (dtype != 0 && dtype != 1))
    return set_error("mi355x_linear_int8: unsupported shape (K up to 131072, weight rows of whole "
                     "16-byte words, less than 4 GiB)");
  if (M == 0) return nullptr;
  const Int8Plan plan = int8_plan(M, N, K, cus > 0 ? cus : 256);
  const Int8Workspace ws = int8_workspace(M, N, K, plan);
  if (!x || !w || !w_scales || !out || (!workspace && ws.bytes))
    return set_error("mi355x_linear_int8: null pointer");
  if (!aligned(x, 2) || !aligned(w, 16) || !aligned(w_scales, 4) || !aligned(out, 2) ||
      !aligned(workspace, 16))
    return set_error("mi355x_linear_int8: misaligned operand");
  if (workspace_bytes < ws.bytes) return set_error("mi355x_linear_int8: workspace too small");
  const TileShape& tile = kTileShapes[static_cast<int>(plan.tile)];
  const int64_t bn = silu_mul && plan.splits == 1 ? tile.bn / 2 : tile.bn;
  const int64_t across = plan.splits == 1 ? columns : N;
  if (plan.kind == Int8Plan::kTiles &&
      ((M + tile.bm - 1) / tile.bm * ((across + bn - 1) / bn) * plan.splits + 8) * 512 >
          kMaxGridThreads)
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
  if (plan.kind == Int8Plan::kVec) {
    a.x = static_cast<const uint8_t*>(x);
    a.x_stride = ldx * 2;
    const int width = static_cast<int>(K);
    if (dtype == 0)
      silu_mul ? launch_int8_vec<0, true>(a, M, columns, width, s)
               : launch_int8_vec<0, false>(a, M, columns, width, s);
    else
      silu_mul ? launch_int8_vec<1, true>(a, M, columns, width, s)
               : launch_int8_vec<1, false>(a, M, columns, width, s);
    return launch_status("product (int8)");
  }
  auto* base = static_cast<uint8_t*>(workspace);
  auto* scales = reinterpret_cast<float*>(base + ws.scales);
  const int64_t k = int8_k(K, ldw);
  if (const char* e = run_quantize_rows(x, ldx * 2, base, k, scales, M, K, k,
                                        static_cast<int>(dtype), s))
    return e;
  a.k_bytes = static_cast<int32_t>(k);
  a.x = base;
  a.x_scales = scales;
  a.x_stride = k;
  int* sums = reinterpret_cast<int*>(base + ws.sums);
  if (dtype == 0)
    return silu_mul ? launch_int8<0, true>(a, plan, sums, s) : launch_int8<0, false>(a, plan, sums, s);
  return silu_mul ? launch_int8<1, true>(a, plan, sums, s) : launch_int8<1, false>(a, plan, sums, s);
}
