// Tile cores of the products whose weights are 8-bit or chosen per token: out = x . w^T for a
// dense weight [N, K] (quant.hip) and for the experts' weights [E, N, K] over rows grouped by
// expert (experts.hip).
//
// Both operands are handled as rows of bytes. An MFMA operand is 16 bytes a lane in every type
// here (8 bf16 / fp16 elements, 16 int8 ones) and a step of the K loop is 128 bytes of a row, so
// one core serves bf16, fp16 and int8; only the instruction and the accumulator differ:
//   bf16 / fp16  32x32x16, fp32 accumulators
//   int8         32x32x32 and 16x16x64, int32 accumulators (exact up to K = 131,072)
//
// Three kernels:
//   * product_tile: a BM x BN tile, x and w rows copied to an LDS ring of 128-byte rows
//     (global_load_lds_dwordx4, 16-byte chunks XOR-swizzled);
//   * product_large: the same for many rows, 256 x 256 on a written-out schedule;
//   * product_rows (int8): up to 16 rows of x, weights from global memory straight into MFMA operands,
//     the waves of a workgroup sharing K. For few rows, where the weight bytes are all that counts.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "common.h"

namespace mi355x {

// Element kinds of the operands and of the output.
constexpr int kBf16 = 0, kFp16 = 1, kInt8 = 2;  // operands
constexpr int kFloatOut = 2;                    // outputs: 0 bf16, 1 fp16, 2 fp32

// Rows of x and of the output.
//   kDense    row r of x and of out is r; one weight
//   kGateUp   row r of the grouped order reads x row order[r] / top_k and writes out row r
//   kDown     row r of the grouped order reads x row r and writes out row order[r], times that
//             slot's weight, in fp32
//   kSplit    kDense over a part of K, the int32 sums left as they are (int8 only)
constexpr int kDense = 0, kGateUp = 1, kDown = 2, kSplit = 3;

struct ProductArgs {
  const uint8_t* x;
  const uint8_t* w;
  void* out;
  const float* x_scales;      // int8: one a row of x
  const float* w_scales;      // int8: [E][w_rows]
  const int32_t* order;       // grouped: slot (token * top_k + s) of every row; null (product_vec): the row
  const int32_t* ids;         // with a null tile list (one slot a tile): expert of every slot
  const int4* tiles;          // grouped: {expert, first row, end row, 0} per row tile
  const int32_t* tile_count;  // grouped: tiles in the list
  const float* row_weights;   // kDown: weight of every row of the grouped order
  int64_t x_stride;           // bytes a row
  int64_t w_stride;           // bytes a row
  int64_t w_expert;           // bytes an expert
  int64_t ldo;                // elements a row of out
  int32_t rows;               // kDense: rows of x. Grouped without a tile list: slots
  int32_t columns;            // columns of out (SILU: half the weight rows)
  int32_t k_bytes;            // bytes of K, a multiple of 16
  int32_t top_k;
  int32_t experts;
  int32_t tiles_m, tiles_n;   // kDense, kSplit: row tiles; column tiles of every row tile
  int32_t splits;             // parts of K. kSplit: out is int32 [splits][rows][ldo]. kDown
                              // (product_tile): out has a plane of `rows` slots a part, summed later
};

// ---------------------------------------------------------------------------- MFMA by type
typedef __bf16 prod_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 prod_f16x8 __attribute__((ext_vector_type(8)));
typedef int prod_i32x4 __attribute__((ext_vector_type(4)));
typedef float prod_f32x16 __attribute__((ext_vector_type(16)));
typedef int prod_i32x16 __attribute__((ext_vector_type(16)));

template <int IN>
struct Mma {
  using Acc16 = std::conditional_t<IN == kInt8, prod_i32x16, prod_f32x16>;  // 32 x 32 block
  using Scalar = std::conditional_t<IN == kInt8, int, float>;

  __device__ __forceinline__ static Acc16 block32(const uint4& a, const uint4& b, Acc16 c) {
    if constexpr (IN == kBf16)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(prod_bf16x8, a),
                                                     __builtin_bit_cast(prod_bf16x8, b), c, 0, 0,
                                                     0);
    else if constexpr (IN == kFp16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(prod_f16x8, a),
                                                    __builtin_bit_cast(prod_f16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(prod_i32x4, a),
                                                   __builtin_bit_cast(prod_i32x4, b), c, 0, 0, 0);
  }
};

// A 16 x 16 block in 8 bits.
__device__ __forceinline__ prod_i32x4 block16_int8(const uint4& a, const uint4& b, prod_i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(prod_i32x4, a),
                                               __builtin_bit_cast(prod_i32x4, b), c, 0, 0, 0);
}

// silu(g) * u, with the hardware reciprocal (1 ulp; an IEEE quotient doubles the epilogue of a large
// gate_up tile). exp(-g) overflows to +inf for g below about -88: g * 0 = -0, the limit.
__device__ __forceinline__ float silu_mul(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.f + __expf(-g)) * u;
}

// Four consecutive output elements of a row, of which the first `n` exist.
template <int OT>
__device__ __forceinline__ void store4(void* out, int64_t at, const float (&v)[4], int n) {
  if constexpr (OT == kFloatOut) {
    float* p = static_cast<float*>(out) + at;
    if (n >= 4) {
      st128_any(p, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                              __float_as_uint(v[3])));
    } else {
      for (int e = 0; e < 4; ++e)
        if (e < n) p[e] = v[e];
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(out) + at;
    if (n >= 4) {
      st64_any(p, make_uint2(Elem<OT>::pack2(v[0], v[1]), Elem<OT>::pack2(v[2], v[3])));
    } else {
      for (int e = 0; e < 4; ++e)
        if (e < n) p[e] = Elem<OT>::from_float(v[e]);
    }
  }
}

// What a row of a tile is multiplied with and where it goes.
struct RowOut {
  int64_t at;    // row of out
  float scale;   // int8: scale of the x row
  float weight;  // kDown: weight of the slot
};

template <int IN, int MODE>
__device__ __forceinline__ RowOut row_out(const ProductArgs& a, int row) {
  RowOut r{row, 1.f, 1.f};
  if constexpr (MODE == kDense) {
    if constexpr (IN == kInt8) r.scale = a.x_scales[row];
  } else {
    const int slot = a.order[row];
    if constexpr (MODE == kGateUp) {
      if constexpr (IN == kInt8) r.scale = a.x_scales[slot / a.top_k];
    } else {
      if constexpr (IN == kInt8) r.scale = a.x_scales[row];
      r.at = slot;
      r.weight = a.row_weights[row];
    }
  }
  return r;
}

// The accumulators of four consecutive columns of a row, scaled: first with the weight row's scale,
// which is of ordinary size in any weight, so that the largest and smallest rows of x stay inside
// the range of fp32 wherever the result does. `acc` (SILU: the gate columns, with
// the matching up columns in `up`); the scales are those of the weight rows.
template <int IN, int MODE, bool SILU, typename T>
__device__ __forceinline__ void finish_values(const ProductArgs& a, const RowOut& r, int column,
                                              const float* w_scales, const T (&acc)[4],
                                              const T (&up)[4], float (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float g = static_cast<float>(acc[e]);
    if constexpr (IN == kInt8) g *= w_scales[min(column + e, a.columns - 1)];
    if constexpr (MODE == kDown)
      g *= r.scale * r.weight;
    else if constexpr (IN == kInt8)
      g *= r.scale;
    if constexpr (SILU) {
      float u = static_cast<float>(up[e]);
      if constexpr (IN == kInt8)
        u = u * w_scales[a.columns + min(column + e, a.columns - 1)] * r.scale;
      g = silu_mul(g, u);
    }
    v[e] = g;
  }
}

// The same, stored.
template <int IN, int OT, int MODE, bool SILU, typename T>
__device__ __forceinline__ void finish4(const ProductArgs& a, const RowOut& r, int column,
                                        const float* w_scales, const T (&acc)[4],
                                        const T (&up)[4]) {
  const int n = a.columns - column;
  if (n <= 0) return;
  float v[4];
  finish_values<IN, MODE, SILU>(a, r, column, w_scales, acc, up, v);
  store4<OT>(a.out, r.at * a.ldo + column, v, n);
}

// A row tile: its expert and rows. Returns false where the workgroup has none.
struct RowTile {
  int expert, begin, end;
};

template <int MODE, int BM>
__device__ __forceinline__ bool row_tile(const ProductArgs& a, int tm, RowTile* t) {
  if constexpr (MODE == kDense || MODE == kSplit) {
    *t = {0, tm * BM, min(a.rows, (tm + 1) * BM)};
    return true;
  } else if (a.tiles) {
    const int4 v = a.tiles[tm];
    *t = {__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y),
          __builtin_amdgcn_readfirstlane(v.z)};
    return true;
  } else {  // one slot a tile
    const int e = __builtin_amdgcn_readfirstlane(a.ids[tm]);
    *t = {e, tm, tm + 1};
    return e >= 0 && e < a.experts;
  }
}

// Workgroup -> (row tile, column tile). Workgroup i runs on XCD i mod 8; every XCD takes a
// contiguous eighth of the tiles, so those that share weights or rows of x meet in its L2. False
// for the workgroups past the last tile (the grid of a grouped product is sized for the most tiles
// that its rows can need). Where K is split, tm counts the row tiles of every part in turn.
template <int MODE>
__device__ __forceinline__ bool tile_of_block(const ProductArgs& a, int splits, int* tm, int* tn) {
  int count;
  if constexpr (MODE == kDense)
    count = a.tiles_m;
  else if constexpr (MODE == kSplit)
    count = a.tiles_m * splits;
  else
    count = (a.tiles ? *a.tile_count : a.rows) * splits;
  const int total = count * a.tiles_n;
  const int per = (total + 7) >> 3;
  const int i = static_cast<int>(blockIdx.x >> 3);
  const int lin = static_cast<int>(blockIdx.x & 7) * per + i;
  if (i >= per || lin >= total) return false;
  if constexpr (MODE == kDense) {
    // Column tiles in groups of eight, every row tile within a group: the 32 tiles that an XCD runs
    // at once then read 4 x 8 tiles' rows instead of 2 x 16 (int8 8192 x 24576 x 4096 834 -> 788
    // us; 8192 x 4096 x 12288 and 6144 x 4096 the same within the noise).
    constexpr int kGroup = 8;
    const int group = lin / (kGroup * count);
    const int wide = min(kGroup, a.tiles_n - group * kGroup);
    const int in = lin - group * kGroup * count;
    *tm = in / wide;
    *tn = group * kGroup + in - *tm * wide;
  } else {
    *tm = lin / a.tiles_n;
    *tn = lin - *tm * a.tiles_n;
  }
  return true;
}

__device__ __forceinline__ uint32_t source_row(const ProductArgs& a, int row, bool gathered) {
  if (!gathered) return row;
  return (a.order ? a.order[row] : row) / a.top_k;
}

// ---------------------------------------------------------------------------- product_tile
static __device__ __align__(16) const uint32_t kProductZeros[4] = {0, 0, 0, 0};

constexpr int kProdRow = 128;  // bytes of a tile row in a stage

// Swizzled position of 16-byte chunk c in tile row r: any 8 consecutive rows put a chunk in 8
// positions and over 16 rows the (row parity, position) pairs are distinct, so the 32 lanes of an
// operand read hit every bank evenly.
__device__ __forceinline__ int prod_chunk(int c, int r) { return c ^ ((r & 7) ^ ((r >> 3) & 1)); }

// 16 bytes a lane from base + offset into lds_base + 16 * lane (see copy_to_lds).
__device__ __forceinline__ void copy_offset_to_lds(const uint8_t* base, uint32_t offset,
                                                   uint32_t lds_base) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_base), "v"(offset),
               "s"(base)
               : "m0");
}

// All of this wave's LDS reads have returned; then the workgroup barrier. The memory clobbers keep
// the compiler's LDS reads on their side of it.
__device__ __forceinline__ void barrier_after_reads() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// At most `ahead` (up to MAX) steps of PER copies are still under way.
template <int PER, int MAX>
__device__ __forceinline__ void wait_steps(int ahead) {
  static_assert(PER * MAX < 64, "vmcnt range");
  if constexpr (MAX > 0) {
    if (ahead < MAX) return wait_steps<PER, MAX - 1>(ahead);
  }
  wait_vmcnt<PER * MAX>();
}

// With SILU, rows 8 q .. 8 q + 7 of each 32-row block of the weight tile are gate rows for even q
// and the matching up rows for odd q, so a lane holds gate and up of a column side by side.
// Column of a tile row, relative to the tile's first column:
__device__ __forceinline__ int silu_column(int r) {
  const int rr = r & 31;
  return (r >> 5) * 16 + (rr >> 4) * 8 + (rr & 7);
}

template <int IN, int OT, int MODE, bool SILU, int BM, int BN, int WM, int WN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, 1) void product_tile(ProductArgs a) {
  constexpr int NW = WM * WN;
  constexpr int kWaveM = BM / WM, kWaveN = BN / WN;
  constexpr int A_BLK = kWaveN / 32, B_BLK = kWaveM / 32;
  static_assert(kWaveM % 32 == 0 && kWaveN % 32 == 0, "wave tile must be 32-aligned");
  constexpr int kGroups = (BM + BN) / 8;
  static_assert(kGroups % NW == 0 && (BM / 8) % NW == 0, "copies must split evenly over the waves");
  constexpr int kCopies = kGroups / NW, kCopiesX = BM / 8 / NW;
  constexpr int kStage = (BM + BN) * kProdRow;
  static_assert(STAGES >= 2 && STAGES * kStage <= 160 * 1024, "LDS");
  constexpr int kBnOut = SILU ? BN / 2 : BN;
  using M = Mma<IN>;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * kStage];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  if (a.columns < 0) lds[tid] = 0;  // never taken; the copies' LDS writes are invisible

  int tm, tn;
  constexpr bool kParts = MODE == kSplit || MODE == kDown;
  if (!tile_of_block<MODE>(a, kParts ? a.splits : 1, &tm, &tn)) return;
  const int all_k = (a.k_bytes + kProdRow - 1) / kProdRow;
  int first_k = 0, n_k = all_k, split = 0;
  if constexpr (kParts) {
    const int row_tiles = MODE == kSplit ? a.tiles_m : *a.tile_count;
    split = tm / row_tiles;
    tm -= split * row_tiles;
    const int per = (all_k + a.splits - 1) / a.splits;
    first_k = split * per;
    n_k = min(per, all_k - first_k);
  }
  RowTile t;
  if (!row_tile<MODE, BM>(a, tm, &t)) return;
  const int n0 = tn * kBnOut;
  const bool tail = a.k_bytes % kProdRow != 0;

  // Copy side: copy j of a wave covers tile rows 8 g .. 8 g + 7, g = wave + NW j (x rows first);
  // lane -> row 8 g + lane / 8, position lane % 8. Rows past the end repeat the last one and are
  // never stored.
  const uint32_t lds_base = lds_address(lds);
  const uint8_t* x_base = a.x;
  if constexpr (MODE != kGateUp) x_base += t.begin * a.x_stride;
  const uint8_t* w_base = a.w + t.expert * a.w_expert;
  if constexpr (!SILU) w_base += static_cast<int64_t>(n0) * a.w_stride;
  uint32_t off[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int g = wave + NW * j;
    int r = 8 * g + (lane >> 3);
    uint32_t row, stride;
    if (j < kCopiesX) {
      const int m = min(t.begin + r, t.end - 1);
      row = MODE == kGateUp ? source_row(a, m, true) : m - t.begin;
      stride = static_cast<uint32_t>(a.x_stride);
    } else {
      r -= BM;
      if constexpr (SILU) {
        const int c = min(n0 + silu_column(r), a.columns - 1);
        row = ((r >> 3) & 1) ? a.columns + c : c;
      } else {
        row = min(r, a.columns - 1 - n0);
      }
      stride = static_cast<uint32_t>(a.w_stride);
    }
    off[j] = row * stride + prod_chunk(lane & 7, r) * 16;
  }
  auto issue = [&](int step, int stage) {
    const uint32_t dst = lds_base + stage * kStage + wave * 1024;
    const int64_t k = static_cast<int64_t>(first_k + step) * kProdRow;
    const uint8_t* xb = x_base + k;
    const uint8_t* wb = w_base + k;
    if (tail && first_k + step == all_k - 1) {
      // chunks past K come as zeros in both operands
#pragma unroll
      for (int j = 0; j < kCopies; ++j) {
        const int r = 8 * (wave + NW * j) + (lane >> 3);
        const int c = prod_chunk(lane & 7, j < kCopiesX ? r : r - BM);
        const uint8_t* src = (j < kCopiesX ? xb : wb) + off[j];
        if (k + c * 16 >= a.k_bytes) src = reinterpret_cast<const uint8_t*>(kProductZeros);
        copy_to_lds(src, dst + j * NW * 1024);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kCopies; ++j)
        copy_offset_to_lds(j < kCopiesX ? xb : wb, off[j], dst + j * NW * 1024);
    }
  };

  // Operand side: block rows r + 32 i share the swizzle of r; chunk 2 kk + half of a row.
  const int wm = wave % WM, wn = wave / WM;
  const int col = lane & 31, half = lane >> 5;
  const int xr = wm * kWaveM + col, wr = wn * kWaveN + col;
  uint32_t x_at[4], w_at[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    x_at[kk] = xr * kProdRow + prod_chunk(2 * kk + half, xr) * 16;
    w_at[kk] = (BM + wr) * kProdRow + prod_chunk(2 * kk + half, wr) * 16;
  }
  typename M::Acc16 acc[A_BLK][B_BLK];
#pragma unroll
  for (int i = 0; i < A_BLK; ++i)
#pragma unroll
    for (int j = 0; j < B_BLK; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  uint4 af[2][A_BLK], bf[2][B_BLK];
  auto read = [&](int stage, int kk, int to) {
    const uint8_t* sb = lds + stage * kStage;
#pragma unroll
    for (int i = 0; i < A_BLK; ++i)
      af[to][i] = *reinterpret_cast<const uint4*>(sb + w_at[kk] + i * 32 * kProdRow);
#pragma unroll
    for (int j = 0; j < B_BLK; ++j)
      bf[to][j] = *reinterpret_cast<const uint4*>(sb + x_at[kk] + j * 32 * kProdRow);
  };

  // Ring of STAGES steps. The operands of a quarter step are read while the quarter before is
  // multiplied, also across the barrier between two steps.
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < n_k) issue(s, s);
  wait_steps<kCopies, STAGES - 1>(min(STAGES - 1, n_k - 1));
  barrier_after_reads();
  read(0, 0, 0);
  int stage = 0;
  for (int step = 0; step < n_k; ++step) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk < 3) {
        read(stage, kk + 1, (kk + 1) & 1);
      } else if (step + 1 < n_k) {
        // The next step's copies are in, every wave has read this one: its buffer is free.
        wait_steps<kCopies, STAGES - 2>(min(STAGES - 2, n_k - 2 - step));
        barrier_after_reads();
        if (step + STAGES < n_k) issue(step + STAGES, stage);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        read(stage, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < A_BLK; ++i)
#pragma unroll
        for (int j = 0; j < B_BLK; ++j)
          acc[i][j] = M::block32(af[kk & 1][i], bf[kk & 1][j], acc[i][j]);
    }
  }

  // A lane holds x row `col` of each B block and weight rows 8 q + 4 half + e of each A block in
  // accumulator elements 4 q + e.
  const float* w_scales = nullptr;
  if constexpr (IN == kInt8 && MODE != kSplit)
    w_scales = a.w_scales + static_cast<int64_t>(t.expert) * (SILU ? 2 : 1) * a.columns;
#pragma unroll
  for (int j = 0; j < B_BLK; ++j) {
    const int row = t.begin + wm * kWaveM + 32 * j + col;
    if (row >= t.end) continue;
    if constexpr (MODE == kSplit) {
      int* out = static_cast<int*>(a.out) + (static_cast<int64_t>(split) * a.rows + row) * a.ldo;
#pragma unroll
      for (int i = 0; i < A_BLK; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int column = n0 + wn * kWaveN + 32 * i + 8 * q + 4 * half;
          if (column < a.columns)  // ldo is a multiple of 4
            *reinterpret_cast<int4*>(out + column) =
                make_int4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                          acc[i][j][4 * q + 3]);
        }
      continue;
    }
    RowOut r = row_out<IN, MODE>(a, row);
    if constexpr (MODE == kDown) r.at += static_cast<int64_t>(split) * a.rows;
#pragma unroll
    for (int i = 0; i < A_BLK; ++i)
#pragma unroll
      for (int q = 0; q < 4; q += SILU ? 2 : 1) {
        typename M::Scalar v[4], u[4] = {};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = acc[i][j][4 * q + e];
          if constexpr (SILU) u[e] = acc[i][j][4 * q + 4 + e];
        }
        const int wrow = wn * kWaveN + 32 * i + 8 * q + 4 * half;
        finish4<IN, OT, MODE, SILU>(a, r, n0 + (SILU ? silu_column(wrow) : wrow), w_scales, v, u);
      }
  }
}

// ---------------------------------------------------------------------------- product_large
// For many rows: a BM x 256 tile on NW = 8 waves, two a SIMD, each with a (BM / 2) x 64 block of it,
// and as many 128-byte steps in flight as LDS holds. The schedule is written out: an MFMA, then one
// of the next quarter step's operand reads or one of the copies into the buffer that the last
// barrier freed, fixed by scheduling barriers.
// Measured on the experts of an 8,192-token prefill (65,536 rows in 128 groups): the copies alone take
// 335 us of gate_up's 440 (11 TB/s into LDS, 44% of it from beyond L2), the MFMAs with operands in L1
// 320; down 247 and 184 of 333, its fp32 outputs being half a gigabyte. Four waves of 128 x 128 read LDS
// a third less but leave each SIMD idle at every wait (480 us for gate_up); 64-byte steps with 128 KiB
// in flight instead of 64 are no quicker (480), so it is not latency.
constexpr int kLargeN = 256;

template <int BM>
constexpr int large_stages() {
  return BM == 256 ? 2 : 3;
}
template <int BM>
constexpr int large_stage_bytes() {
  return (BM + kLargeN) * kProdRow;
}
constexpr int kLargeEdges = 3 * large_stage_bytes<128>();  // LDS behind the stages: the edges
static_assert(kLargeEdges >= 2 * large_stage_bytes<256>(), "the edges follow the stages");

// The tile's K loop: acc[i][j] of A block i (32 weight rows) and B block j (32 rows of x). TAIL: K
// ends inside a step. Compiled apart, as the question at every copy costs 8% of the loop.
template <int IN, int MODE, bool SILU, int BM, int NW, bool TAIL>
__device__ __forceinline__ void large_loop(const ProductArgs& a, const RowTile& t, int n0,
                                           uint8_t* lds,
                                           typename Mma<IN>::Acc16 (&acc)[16 / NW][BM / 64]) {
  constexpr int A_BLK = 16 / NW, B_BLK = BM / 64, S = large_stages<BM>();
  constexpr int kCopies = (BM + kLargeN) / 8 / NW, kCopiesX = BM / 8 / NW;
  constexpr int kStage = large_stage_bytes<BM>();
  using M = Mma<IN>;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int n_k = (a.k_bytes + kProdRow - 1) / kProdRow;

  // Copy j of a wave covers tile rows 8 g .. 8 g + 7, g = wave + NW j, x rows first.
  const uint32_t lds_base = lds_address(lds) + wave * 1024;
  const uint8_t* x_base = a.x;
  if constexpr (MODE != kGateUp) x_base += t.begin * a.x_stride;
  const uint8_t* w_base = a.w + t.expert * a.w_expert;
  if constexpr (!SILU) w_base += static_cast<int64_t>(n0) * a.w_stride;
  uint32_t off[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    int r = 8 * (wave + NW * j) + (lane >> 3);
    uint32_t row, stride;
    if (j < kCopiesX) {
      const int m = min(t.begin + r, t.end - 1);
      row = MODE == kGateUp ? source_row(a, m, true) : m - t.begin;
      stride = static_cast<uint32_t>(a.x_stride);
    } else {
      r -= BM;
      if constexpr (SILU) {
        const int c = min(n0 + silu_column(r), a.columns - 1);
        row = ((r >> 3) & 1) ? a.columns + c : c;
      } else {
        row = min(r, a.columns - 1 - n0);
      }
      stride = static_cast<uint32_t>(a.w_stride);
    }
    off[j] = row * stride + prod_chunk(lane & 7, r) * 16;
  }
  auto copy = [&](int step, uint32_t buffer, int j) {
    const int64_t k = static_cast<int64_t>(step) * kProdRow;
    const uint8_t* base = (j < kCopiesX ? x_base : w_base) + k;
    const uint32_t dst = buffer + j * NW * 1024;
    if (TAIL && step == n_k - 1) {  // chunks past K come as zeros in both operands
      int r = 8 * (wave + NW * j) + (lane >> 3);
      if (j >= kCopiesX) r -= BM;
      const uint8_t* src = base + off[j];
      if (k + prod_chunk(lane & 7, r) * 16 >= a.k_bytes)
        src = reinterpret_cast<const uint8_t*>(kProductZeros);
      copy_to_lds(src, dst);
    } else {
      copy_offset_to_lds(base, off[j], dst);
    }
  };

  const int wm = wave & 1, wn = wave >> 1;
  const int col = lane & 31, half = lane >> 5;
  const int xr = wm * (BM / 2) + col, wr = wn * (32 * A_BLK) + col;
  uint32_t x_at[4], w_at[4];
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    x_at[kk] = xr * kProdRow + prod_chunk(2 * kk + half, xr) * 16;
    w_at[kk] = (BM + wr) * kProdRow + prod_chunk(2 * kk + half, wr) * 16;
  }
#pragma unroll
  for (int i = 0; i < A_BLK; ++i)
#pragma unroll
    for (int j = 0; j < B_BLK; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  uint4 af[2][A_BLK], bf[2][B_BLK];
  constexpr int kReads = A_BLK + B_BLK, kMfma = A_BLK * B_BLK;
  constexpr int kSlots = std::max({kMfma, kReads, kCopies});
  // in the order in which the MFMAs want them: A block 0, the B blocks, the other A blocks
  auto read = [&](const uint8_t* sb, int kk, int f) {
    const int to = kk & 1;
    if (f >= 1 && f <= B_BLK) {
      bf[to][f - 1] = *reinterpret_cast<const uint4*>(sb + x_at[kk] + (f - 1) * 32 * kProdRow);
    } else {
      const int i = f == 0 ? 0 : f - B_BLK;
      af[to][i] = *reinterpret_cast<const uint4*>(sb + w_at[kk] + i * 32 * kProdRow);
    }
  };
  auto barrier = [&] {  // this wave's reads are done (its copies were waited for); then all waves'
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < n_k)
#pragma unroll
      for (int j = 0; j < kCopies; ++j) copy(s, lds_base + s * kStage, j);
  wait_steps<kCopies, S - 1>(min(S - 1, n_k - 1));
  barrier();
#pragma unroll
  for (int f = 0; f < kReads; ++f) read(lds, 0, f);
  int stage = 0;
  for (int step = 0; step < n_k; ++step) {
    const uint8_t* now = lds + stage * kStage;
    const uint32_t freed = lds_base + stage * kStage;
    stage = stage == S - 1 ? 0 : stage + 1;
    const uint8_t* next = lds + stage * kStage;
    const bool more = step + 1 < n_k, fill = step + S < n_k;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      if (kk == 3 && more) {  // the next step is in and this one is read: its buffer is free
        wait_steps<kCopies, S - 2>(min(S - 2, n_k - 2 - step));
        barrier();
      }
#pragma unroll
      for (int m = 0; m < kSlots; ++m) {
        const int i = m / B_BLK, j = m % B_BLK;
        if (m < kMfma) acc[i][j] = M::block32(af[kk & 1][i], bf[kk & 1][j], acc[i][j]);
        if (m < kReads) {
          if (kk < 3)
            read(now, kk + 1, m);
          else if (more)
            read(next, 0, m);
        }
        if (kk == 3 && fill && m < kCopies) copy(step + S, freed, m);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// What the epilogue needs of the tile's rows and columns, in LDS once the stages are free.
struct LargeEdges {
  int64_t out[256];         // byte offset of the row
  float row_scale[256];     // int8: of the x row; kDown: times the slot's weight
  float column_scale[256];  // int8: of the tile's weight rows (SILU: 128 gate, then 128 up)
};

// The epilogue: every wave turns 32 rows of its block at a time through LDS, so that rows go out in
// 16-byte stores of whole 64- to 256-byte pieces instead of 8 bytes a row and store.
template <int IN, int OT, int MODE, bool SILU, int BM, int NW>
__device__ __forceinline__ void large_store(const ProductArgs& a, const RowTile& t, int n0,
                                            uint8_t* lds, const LargeEdges& edges,
                                            typename Mma<IN>::Acc16 (&acc)[16 / NW][BM / 64]) {
  constexpr int A_BLK = 16 / NW, B_BLK = BM / 64;
  constexpr int kOutSize = OT == kFloatOut ? 4 : 2;
  constexpr int kCols = (SILU ? 16 : 32) * A_BLK;        // columns of a wave
  constexpr int kPitch = kCols * kOutSize + 16;          // bytes of a row in LDS
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int wm = wave & 1, wn = wave >> 1;
  const int col = lane & 31, half = lane >> 5;
  uint8_t* turn = lds + wave * 32 * kPitch;
  // int8: scales of the weight rows of a lane's quads
  float gs[A_BLK][4][4], us[A_BLK][4][4];
  if constexpr (IN == kInt8) {
#pragma unroll
    for (int i = 0; i < A_BLK; ++i)
#pragma unroll
      for (int q = 0; q < 4; q += SILU ? 2 : 1) {
        const int wrow = 32 * i + 8 * q + 4 * half;
        const float* at = edges.column_scale + wn * kCols + (SILU ? silu_column(wrow) : wrow);
        *reinterpret_cast<float4*>(gs[i][q]) = *reinterpret_cast<const float4*>(at);
        if constexpr (SILU)
          *reinterpret_cast<float4*>(us[i][q]) = *reinterpret_cast<const float4*>(at + 128);
      }
  }
  // A lane stores 16-byte piece lane % kChunks of rows kRows apart.
  constexpr int kChunks = kCols * kOutSize / 16;  // pieces of a row
  constexpr int kPer = 16 / kOutSize;             // elements of a piece
  constexpr int kRows = kWave / kChunks;
  const int piece = lane % kChunks, piece_row = lane / kChunks;
  const int column = n0 + wn * kCols + piece * kPer;
  const bool whole = column + kPer <= a.columns;
  uint8_t* out = static_cast<uint8_t*>(a.out) + static_cast<int64_t>(column) * kOutSize;
#pragma unroll
  for (int j = 0; j < B_BLK; ++j) {
    const int begin = wm * (BM / 2) + 32 * j;  // row of the tile
    if (t.begin + begin >= t.end) break;
    const float row_scale = edges.row_scale[begin + col];
#pragma unroll
    for (int i = 0; i < A_BLK; ++i) {
      float f[16];  // of 32 columns (SILU: the 8 of 16)
#pragma unroll
      for (int q = 0; q < 4; q += SILU ? 2 : 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float g = static_cast<float>(acc[i][j][4 * q + e]);
          if constexpr (IN == kInt8) g *= gs[i][q][e];
          if constexpr (IN == kInt8 || MODE == kDown) g *= row_scale;
          if constexpr (SILU) {
            float u = static_cast<float>(acc[i][j][(4 * q + 4 + e) & 15]);
            if constexpr (IN == kInt8) u = u * us[i][q][e] * row_scale;
            g = silu_mul(g, u);
          }
          f[4 * q + e] = g;
        }
      }
#pragma unroll
      for (int q = 0; q < 4; q += SILU ? 2 : 1) {
        const int wrow = 32 * i + 8 * q + 4 * half;
        uint8_t* p = turn + col * kPitch + (SILU ? silu_column(wrow) : wrow) * kOutSize;
        const float* v = f + 4 * q;
        if constexpr (OT == kFloatOut)
          *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
          *reinterpret_cast<uint2*>(p) =
              make_uint2(Elem<OT>::pack2(v[0], v[1]), Elem<OT>::pack2(v[2], v[3]));
      }
    }
    // A wave's LDS operations keep their order, so its reads follow its writes of all lanes; the
    // clobbers keep the compiler from exchanging them.
    asm volatile("" ::: "memory");
#pragma unroll
    for (int s = 0; s < 32 / kRows; ++s) {
      const int lr = s * kRows + piece_row;
      const uint4 v = *reinterpret_cast<const uint4*>(turn + lr * kPitch + piece * 16);
      if (t.begin + begin + lr >= t.end || column >= a.columns) continue;
      uint8_t* o = out + edges.out[begin + lr];
      if (whole) {
        st128_any(o, v);
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          if (column + e >= a.columns) continue;
          if constexpr (OT == kFloatOut)
            reinterpret_cast<uint32_t*>(o)[e] = w[e];
          else
            reinterpret_cast<uint16_t*>(o)[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
        }
      }
    }
    asm volatile("" ::: "memory");
  }
}

template <int IN, int OT, int MODE, bool SILU, int BM, int NW, bool TAIL>
__device__ __forceinline__ void large_tile(const ProductArgs& a, const RowTile& t, int n0,
                                           uint8_t* lds) {
  // Loaded now and needed after the loop: the row and column that this thread stands for.
  const int r = threadIdx.x & 255;
  const int row = min(t.begin + r, t.end - 1);
  int slot = row;
  float row_scale = 1.f, weight = 1.f, column_scale = 1.f;
  if constexpr (MODE != kDense) slot = a.order[row];
  if constexpr (MODE == kDown) weight = a.row_weights[row];
  if constexpr (IN == kInt8 && MODE != kGateUp) row_scale = a.x_scales[row];
  if constexpr (IN == kInt8) {
    const float* scales = a.w_scales + static_cast<int64_t>(t.expert) * (SILU ? 2 : 1) * a.columns;
    const int c = min(n0 + (SILU ? r & 127 : r), a.columns - 1);
    column_scale = scales[SILU && r >= 128 ? a.columns + c : c];
  }
  typename Mma<IN>::Acc16 acc[16 / NW][BM / 64];
  large_loop<IN, MODE, SILU, BM, NW, TAIL>(a, t, n0, lds, acc);
  auto& edges = *reinterpret_cast<LargeEdges*>(lds + kLargeEdges);
  if constexpr (IN == kInt8 && MODE == kGateUp) row_scale = a.x_scales[slot / a.top_k];
  if (threadIdx.x < 256) {
    edges.out[r] = (MODE == kDown ? slot : row) * a.ldo * (OT == kFloatOut ? 4 : 2);
    edges.row_scale[r] = row_scale * weight;
    edges.column_scale[r] = column_scale;
  }
  __syncthreads();  // the edges are written and every wave is done with the stages
  large_store<IN, OT, MODE, SILU, BM, NW>(a, t, n0, lds, edges, acc);
}

// A tile of up to BM rows. Of the row tiles that a group ends with, those of up to BM / 2 rows run
// as half tiles: a ragged group of rows then wastes a quarter of a tile on average, not half.
template <int IN, int OT, int MODE, bool SILU, int BM, int NW, bool TAIL>
__global__ __launch_bounds__(64 * NW, 1) void product_large(ProductArgs a) {
  static_assert(BM == 256, "the edges are those of 256 rows");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kLargeEdges + sizeof(LargeEdges)];
  if (a.columns < 0) lds[threadIdx.x] = 0;  // never taken; the copies' LDS writes are invisible
  int tm, tn;
  if (!tile_of_block<MODE>(a, 1, &tm, &tn)) return;
  RowTile t;
  if (!row_tile<MODE, BM>(a, tm, &t)) return;
  const int n0 = tn * (SILU ? kLargeN / 2 : kLargeN);
  if (t.end - t.begin > BM / 2)
    large_tile<IN, OT, MODE, SILU, BM, NW, TAIL>(a, t, n0, lds);
  else
    large_tile<IN, OT, MODE, SILU, BM / 2, NW, TAIL>(a, t, n0, lds);
}

// ---------------------------------------------------------------------------- product_rows
// Up to 16 rows of x against 16 columns a block (SILU: 16 gate and the matching 16 up rows; else
// NB blocks of 16 weight rows). The four waves take a quarter of K each and their sums are joined
// in LDS. A lane's operand rows are lane % 16; of a 128-byte step it holds bytes 32 g .. 32 g + 31,
// g = lane / 16, as two operands: K is summed in another order than it is stored, the same one in
// both operands, so whole 128-byte lines are read.
template <int OT, bool SILU, int NB, int DEPTH>
__global__ __launch_bounds__(256) void product_rows(ProductArgs a) {
  static_assert(!SILU || NB == 2, "a gate and an up block");
  constexpr int kOut = SILU ? 16 : 16 * NB;
  __shared__ prod_i32x4 sums[NB][4][64];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  int tm, tn;
  if (!tile_of_block<kDense>(a, 1, &tm, &tn)) return;
  RowTile t;
  if (!row_tile<kDense, 16>(a, tm, &t)) return;
  const int n0 = tn * kOut;
  const int r = lane & 15, g = lane >> 4;

  const int m = min(t.begin + r, t.end - 1);
  const uint8_t* x_row =
      a.x + static_cast<int64_t>(m) * a.x_stride + g * 32;
  const uint8_t* w_row[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int c = min(n0 + (SILU ? 0 : 16 * b) + r, a.columns - 1);
    w_row[b] = a.w + static_cast<int64_t>(SILU && b ? a.columns + c : c) * a.w_stride + g * 32;
  }
  const int n_k = (a.k_bytes + kProdRow - 1) / kProdRow;
  const int per = (n_k + 3) >> 2;
  const int first = min(n_k, wave * per), last = min(n_k, first + per);

  uint4 wf[DEPTH][NB][2], xf[DEPTH][2];
  auto load = [&](int step, int to) {
    const int64_t k = static_cast<int64_t>(step) * kProdRow;
    if (k + kProdRow <= a.k_bytes) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < NB; ++b) wf[to][b][h] = ld128_nt(w_row[b] + k + 16 * h);
        xf[to][h] = ld128(x_row + k + 16 * h);
      }
    } else {  // the end of K: chunks past it are zeros in both operands
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = k + g * 32 + 16 * h < a.k_bytes;
#pragma unroll
        for (int b = 0; b < NB; ++b)
          wf[to][b][h] = in ? ld128(w_row[b] + k + 16 * h) : make_uint4(0, 0, 0, 0);
        xf[to][h] = in ? ld128(x_row + k + 16 * h) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  prod_i32x4 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[b][e] = 0;

#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (first + d < last) load(first + d, d);
  for (int step = first; step < last; step += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (step + d >= last) break;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = block16_int8(wf[d][b][h], xf[d][h], acc[b]);
      if (step + d + DEPTH < last) load(step + d + DEPTH, d);
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) sums[b][wave][lane] = acc[b];
  __syncthreads();

  // Wave b finishes block b (SILU: wave 0 both). A lane holds x row lane % 16 and weight rows
  // 4 g + e.
  if (wave >= (SILU ? 1 : NB)) return;
  const int row = t.begin + r;
  if (row >= t.end) return;
  const RowOut ro = row_out<kInt8, kDense>(a, row);
  auto total = [&](int b, int(&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = (sums[b][0][lane][e] + sums[b][1][lane][e]) +
             (sums[b][2][lane][e] + sums[b][3][lane][e]);
  };
  int v[4], u[4] = {};
  total(SILU ? 0 : wave, v);
  if constexpr (SILU) total(NB - 1, u);
  finish4<kInt8, OT, kDense, SILU>(a, ro, n0 + (SILU ? 0 : 16 * wave) + 4 * g, a.w_scales, v, u);
}

// ---------------------------------------------------------------------------- the choice of tiles
// The tiles that a product can take, smallest first. k128 has four stages and a CU for itself,
// k128Two has two stages and shares the CU with another.
enum class Tile { k64, k128, k128Two, k256x128, k256 };
constexpr int kTiles = 5;

struct TileShape {
  int bm, bn;        // rows of x, weight rows
  float step, busy;  // us a 128-byte step: with few workgroups, and what a full chip adds
};
constexpr TileShape kTileShapes[] = {
    {64, 64, 0.29f, 0.f},   {128, 128, 0.5f, 0.2f},  {128, 128, 0.58f, 0.f},
    {256, 128, 0.8f, 0.3f}, {256, 256, 1.2f, 0.6f}};

// Estimated time in us of `row_tiles` x `column_tiles` tiles over K. A CU's copies into LDS come at
// about 60 GB/s where they miss L2, whatever the depth of the ring, which makes the step of a tile
// its bytes; one workgroup a CU, but three of 64 x 64 (with three stages in LDS; with four, two of
// them: the 8-bit experts of 40 tokens 57 + 33 us instead of 53 + 29). A 256 x 256 tile of up to
// 128 rows runs as half a tile. Weights come at 5.8 TB/s at most. Measured, int8: 4096 x 4096 at 64
// rows 64 x 64 tiles 13.0 us, 128 x 128 19.5, 256 x 256 25.2; 6144 x 4096 at 512 rows 33.9 / 25.2 /
// 34.4 (256 x 128) / 47.2, at 1,024 rows 62 / 54 / 37.5 / 49, at 2,048 rows 118 / 79 / 76 / 56.
// bf16 experts 128 x (1536 x 2048) at 64 rows each 202 / 182 / 221 / 187, at 128 rows 296 / 229 /
// 239 / 208.
inline float tile_estimate(Tile tile, float row_tiles, float column_tiles, int64_t k_bytes,
                           float weight_bytes, bool half, int cus) {
  const TileShape& t = kTileShapes[static_cast<int>(tile)];
  const float r = row_tiles * column_tiles / static_cast<float>(cus);
  const float busy = std::min(r, 1.f);
  float step = t.step + t.busy * busy, rounds = 1.f;
  if (tile == Tile::k256 && half) step = 0.65f + 0.8f * busy;
  if (tile == Tile::k64) {
    if (r > 1.f) rounds = std::max(1.07f * r - 0.07f, std::min(2.f, 1.f + 2.5f * (r - 1.f)));
  } else if (tile == Tile::k128Two) {
    rounds = std::max(2.f, r + 0.3f);
  } else if (r > 1.06f) {
    rounds = r <= 3.f ? std::ceil(r - 0.06f) : r + 0.3f;
  }
  const float steps = static_cast<float>((k_bytes + kProdRow - 1) / kProdRow);
  return 3.3f + std::max(steps * step * rounds, weight_bytes / 5.8e6f);
}

}  // namespace mi355x
