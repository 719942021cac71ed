// Products of one or two rows on vector math. A row of the weight is read by consecutive lanes, a
// kilobyte a load, and the lanes' partial sums are joined at the end. That is quicker than MFMA
// operands loaded from memory, whose lanes hop from row to row (gate_up of one token and 8 experts,
// 50 MB: 10.2 us against 13.6), and the rows of x are quantised on the way instead of in a launch of
// their own (6144 x 4096 int8: 6.8 us at one row and 9.7 at two, against 8.2 and a launch of 2 us;
// at four rows 12.1, no gain). Bound by latency: such a product is a few loads a lane.
#pragma once

#include "quant.h"

namespace mi355x {

// acc += the products of 16 bytes of a weight row and of x.
template <int IN>
__device__ __forceinline__ void dot_piece(const uint4& w, const uint4& x,
                                          typename Mma<IN>::Scalar& acc) {
  if constexpr (IN == kInt8) {
    acc = __builtin_amdgcn_sdot4(static_cast<int>(w.x), static_cast<int>(x.x), acc, false);
    acc = __builtin_amdgcn_sdot4(static_cast<int>(w.y), static_cast<int>(x.y), acc, false);
    acc = __builtin_amdgcn_sdot4(static_cast<int>(w.z), static_cast<int>(x.z), acc, false);
    acc = __builtin_amdgcn_sdot4(static_cast<int>(w.w), static_cast<int>(x.w), acc, false);
  } else {
    float a[8], b[8];
    unpack8<IN>(w, a);
    unpack8<IN>(x, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = fmaf(a[i], b[i], acc);
  }
}

// Sum over groups of G lanes; every lane of a group gets it.
template <int G, typename T>
__device__ __forceinline__ T group_sum(T v) {
#pragma unroll
  for (int d = 1; d < G; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// The 8-bit form of a row of `width` elements of type XT in LDS (whole 16-byte words, zeros behind the
// end) and its scale, by a workgroup of THREADS. `tops` is an LDS word a wave.
template <int XT, int THREADS>
__device__ __forceinline__ float quantize_to_lds(const uint8_t* row, int width,
                                                 uint8_t* to, uint32_t* tops) {
  const int chunks = (width + 15) >> 4;
  uint32_t top = 0;
  float f[16];
  for (int c = threadIdx.x; c < chunks; c += THREADS) {
    load16<XT>(row, c * 16, width - c * 16, f);
    top = max(top, magnitude16(f));
  }
  top = wave_max(top);
  __syncthreads();  // tops may still be read for the row before
  if (threadIdx.x % kWave == 0) tops[threadIdx.x / kWave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) top = max(top, tops[w]);
  const RowQuant q(top);
  for (int c = threadIdx.x; c < chunks; c += THREADS) {
    if (chunks > THREADS) load16<XT>(row, c * 16, width - c * 16, f);
    st128(to + c * 16, q.values(f));
  }
  return q.scale;
}

// The same by one wave. No barrier: the row is for the workgroup after its next one.
template <int XT>
__device__ __forceinline__ float quantize_by_wave(const uint8_t* row, int width,
                                                  uint8_t* to) {
  const int lane = threadIdx.x % kWave;
  const int chunks = (width + 15) >> 4;
  uint32_t top = 0;
  float f[16];
  for (int c = lane; c < chunks; c += kWave) {
    load16<XT>(row, c * 16, width - c * 16, f);
    top = max(top, magnitude16(f));
  }
  const RowQuant q(wave_max(top));
  for (int c = lane; c < chunks; c += kWave) {
    if (chunks > kWave) load16<XT>(row, c * 16, width - c * 16, f);
    st128(to + c * 16, q.values(f));
  }
  return q.scale;
}

constexpr int kVecLds = 32 * 1024;  // bytes of quantised rows that a workgroup holds

// MR rows of x (kDense: a.rows of them; kGateUp: one, of slot tm) against R weight rows a wave (SILU:
// R / 2 gate rows and the matching up rows). For int8 the rows of x, of type XT, are quantised in
// the workgroup while its first weights are on their way.
template <int IN, int XT, int OT, int MODE, bool SILU, int MR, int R, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void product_vec(ProductArgs a, int width) {
  constexpr int kOut = SILU ? R / 2 : R;  // columns of a wave
  constexpr int U = 4;                    // pieces of a row on their way at once
  constexpr bool kQuant = IN == kInt8;
  __shared__ __attribute__((aligned(16))) uint8_t rows[kQuant ? kVecLds : 16];
  __shared__ uint32_t tops[WAVES];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  int tm, tn;
  if (!tile_of_block<MODE>(a, 1, &tm, &tn)) return;
  RowTile t;
  if (!row_tile<MODE, MR>(a, tm, &t)) return;
  const int n0 = (tn * WAVES + wave) * kOut;
  const uint8_t* w_row[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int c = min(n0 + (SILU ? r / 2 : r), a.columns - 1);
    w_row[r] = a.w + t.expert * a.w_expert +
               static_cast<int64_t>(SILU && (r & 1) ? a.columns + c : c) * a.w_stride;
  }
  const uint8_t* x_row[MR];
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    const int row = min(t.begin + m, t.end - 1);
    x_row[m] = a.x + static_cast<int64_t>(source_row(a, row, MODE == kGateUp)) * a.x_stride;
  }
  struct Pieces {
    uint4 w[U][R], x[kQuant ? 1 : U][MR];
  };
  auto load = [&](int k, Pieces& p) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + (u * kWave + lane) * 16;
      const bool in = at < a.k_bytes;
#pragma unroll
      for (int r = 0; r < R; ++r) p.w[u][r] = in ? ld128_nt(w_row[r] + at) : make_uint4(0, 0, 0, 0);
      if constexpr (!kQuant) {
#pragma unroll
        for (int m = 0; m < MR; ++m) p.x[u][m] = in ? ld128(x_row[m] + at) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  typename Mma<IN>::Scalar acc[MR][R] = {};
  auto multiply = [&](int k, const Pieces& p) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + (u * kWave + lane) * 16;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        uint4 x;
        if constexpr (kQuant)
          x = *reinterpret_cast<const uint4*>(rows + m * a.k_bytes + min(at, a.k_bytes - 16));
        else
          x = p.x[u][m];
#pragma unroll
        for (int r = 0; r < R; ++r) dot_piece<IN>(p.w[u][r], x, acc[m][r]);
      }
    }
  };
  constexpr int kBatch = U * kWave * 16;
  Pieces p;
  load(0, p);
  float scale[MR];
  if constexpr (kQuant) {
#pragma unroll
    for (int m = 0; m < MR; ++m)
      scale[m] = quantize_to_lds<XT, 64 * WAVES>(x_row[m], width, rows + m * a.k_bytes, tops);
    __syncthreads();
  }
  for (int k = kBatch; k < a.k_bytes; k += kBatch) {
    Pieces next;
    load(k, next);
    multiply(k - kBatch, p);
    p = next;
  }
  multiply((a.k_bytes - 1) / kBatch * kBatch, p);
  const float* w_scales = nullptr;
  if constexpr (kQuant)
    w_scales = a.w_scales + static_cast<int64_t>(t.expert) * (SILU ? 2 : 1) * a.columns;
#pragma unroll
  for (int m = 0; m < MR; ++m) {
#pragma unroll
    for (int r = 0; r < R; ++r) acc[m][r] = group_sum<kWave>(acc[m][r]);
    const int row = t.begin + m;
    if (lane != m || row >= t.end) continue;  // lane m stores row m
#pragma unroll
    for (int r = 0; r < R; r += SILU ? 2 : 1) {
      const int c = n0 + (SILU ? r / 2 : r);
      if (c >= a.columns) continue;
      float v = static_cast<float>(acc[m][r]);
      if constexpr (kQuant) v = v * w_scales[c] * scale[m];
      if constexpr (SILU) {
        float u = static_cast<float>(acc[m][r + 1]);
        if constexpr (kQuant) u = u * w_scales[a.columns + c] * scale[m];
        v = silu_mul(v, u);
      }
      if constexpr (OT == kFloatOut)
        static_cast<float*>(a.out)[row * a.ldo + c] = v;
      else
        static_cast<uint16_t*>(a.out)[row * a.ldo + c] = Elem<OT>::from_float(v);
    }
  }
}

// out[t] of a token's slots in one pass: column c is the sum over the slots s of weight[s] times row
// c of the slot's down weight times the slot's row of act, in fp32, so neither slot outputs nor a
// pass over them are needed. G lanes take a slot's row (the fewest of 16, 32 and 64 that hold it in
// three pieces), 64 / G slots at a time. A wave takes a column, a workgroup WAVES of them. For int8 the
// token's rows of act (fp32) are quantised in the workgroup.
struct DownArgs {
  const uint8_t* act;   // fp32, a row a slot
  const uint8_t* w;
  uint16_t* out;
  const float* w_scales;
  const int32_t* ids;
  const float* weights;
  int64_t act_stride, w_stride, w_expert;  // bytes
  int64_t ldo;
  int32_t top_k, experts, columns, k_bytes, width;
};

constexpr int kVecDownSlots = 16;  // top_k that product_vec_down takes

template <int IN, int OT, int G, int N, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void product_vec_down(DownArgs a) {
  constexpr bool kQuant = IN == kInt8;
  constexpr int kAtOnce = kWave / G, U = 3;
  constexpr int kXWords = kQuant ? 1 : 2;  // 16-byte words of act to one of the weight
  __shared__ __attribute__((aligned(16))) uint8_t rows[kQuant ? kVecLds : 16];
  __shared__ float scales[kVecDownSlots];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t token = blockIdx.y;
  const int64_t first = token * a.top_k;
  if constexpr (kQuant) {
    for (int s = wave; s < a.top_k; s += WAVES) {
      const int e = a.ids[first + s];
      if (e < 0 || e >= a.experts) continue;
      const float scale = quantize_by_wave<kFloatOut>(a.act + (first + s) * a.act_stride, a.width,
                                                      rows + s * a.k_bytes);
      if (lane == 0) scales[s] = scale;
    }
    __syncthreads();
  }
  const int c = blockIdx.x * WAVES + wave;
  if (c >= a.columns) return;
  const int g = lane / G, l = lane % G;
  float sum = 0.f;
  for (int s0 = 0; s0 < a.top_k; s0 += N * kAtOnce) {  // N slots a group of lanes at once
    int e[N], slot[N];
    float weight[N];
    bool in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int s = s0 + i * kAtOnce + g;
      slot[i] = min(s, a.top_k - 1);
      e[i] = a.ids[first + slot[i]];
      weight[i] = a.weights[first + slot[i]];
      in[i] = s < a.top_k && e[i] >= 0 && e[i] < a.experts;
    }
    typename Mma<IN>::Scalar acc[N] = {};
    for (int k = l * 16; k < a.k_bytes; k += U * G * 16) {
      uint4 w[N][U], x[N][U][kXWords];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = k + u * G * 16;
          const bool there = in[i] && at < a.k_bytes;
          w[i][u] = there ? ld128_nt(a.w + e[i] * a.w_expert + c * a.w_stride + at)
                          : make_uint4(0, 0, 0, 0);
          const uint8_t* from = kQuant ? rows + slot[i] * a.k_bytes + at
                                       : a.act + (first + slot[i]) * a.act_stride + 2 * at;
#pragma unroll
          for (int h = 0; h < kXWords; ++h)
            x[i][u][h] = there ? ld128(from + 16 * h) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if constexpr (kQuant) {
            dot_piece<IN>(w[i][u], x[i][u][0], acc[i]);
          } else {
            float f[8];
            unpack8<IN>(w[i][u], f);
            const float* v = reinterpret_cast<const float*>(x[i][u]);
#pragma unroll
            for (int q = 0; q < 8; ++q) acc[i] = fmaf(f[q], v[q], acc[i]);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const auto total = group_sum<G>(acc[i]);
      if (!in[i]) continue;
      float v = static_cast<float>(total);
      if constexpr (kQuant)
        v = v * a.w_scales[static_cast<int64_t>(e[i]) * a.columns + c] * scales[slot[i]];
      sum += v * weight[i];
    }
  }
#pragma unroll
  for (int d = G; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) a.out[token * a.ldo + c] = Elem<OT>::from_float(sum);
}

}  // namespace mi355x
