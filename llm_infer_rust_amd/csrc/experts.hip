// Expert layers on gfx950: routing, and the gate_up -> SiLU x mul -> down products of the experts
// that each token was routed to.
//
//   p = softmax(logits[t]);  ids[t, :] = the top_k largest, ties to the lowest index
//   weights[t, s] = p[ids[t, s]]  (normalised: divided by their sum)
//   out[t] = sum_s weights[t, s] down[e] . (silu(g) * u),  (g; u) = gate_up[e] . x[t],  e = ids[t, s]
//
// The slots (token, s) are grouped by expert on the device, so nothing is read back to the host:
// the products run over a list of row tiles (expert, first row, end row) and a grid sized for the
// most tiles that so many slots can need. Replaces, for layers of experts, the MLP of
// src/models/qwen3/model.rs:478-534; the reference itself has dense layers only.
#include <algorithm>

#include "product_vec.h"

namespace mi355x {
namespace {

// ---------------------------------------------------------------------------- routing
constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 64;

template <int DT>
__device__ __forceinline__ float logit(const void* p, int64_t at) {
  if constexpr (DT == kFloatOut)
    return static_cast<const float*>(p)[at];
  else
    return Elem<DT>::to_float(static_cast<const uint16_t*>(p)[at]);
}

// Floats in order as unsigned integers (-0 as 0, NaN above +inf); 0 is below every float.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <int Ctrl>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), Ctrl, 0xf,
                                                                  0xf, false)));
}

// Maximum over the wave as a scalar: within rows of 16 lanes by DPP, then over the four rows.
__device__ __forceinline__ uint32_t wave_max_uniform(uint32_t x) {
  x = dpp_max<kDppQuadSwap1>(x);
  x = dpp_max<kDppQuadSwap2>(x);
  x = dpp_max<kDppRowHalfMirror>(x);
  x = dpp_max<kDppRowMirror>(x);
  const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16);
  const uint32_t c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
  return max(max(a, b), max(c, d));
}

// One wave a token, expert v * 64 + lane in register v. Selection is on the logits (the softmax
// keeps their order), so ids are exact; top_k rounds of a wave maximum over (value, lowest index).
// Latency-bound: a row is E logits.
template <int DT, int V>
__global__ __launch_bounds__(256) void route_kernel(const void* __restrict__ logits, int64_t stride,
                                                    float* __restrict__ weights,
                                                    int32_t* __restrict__ ids, int64_t tokens,
                                                    int experts, int top_k, bool normalize) {
  const int64_t t = blockIdx.x * int64_t(4) + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  if (t >= tokens) return;
  uint32_t key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * kWave + lane;
    key[v] = e < experts ? order_key(logit<DT>(logits, t * stride + e)) : 0u;
  }
  uint32_t all[V];
#pragma unroll
  for (int v = 0; v < V; ++v) all[v] = key[v];
  float top = 0.f, mine = 0.f;
  int my_id = 0;
  for (int s = 0; s < top_k; ++s) {
    uint32_t best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = max(best, key[v]);
    best = wave_max_uniform(best);
    int id = 0;
#pragma unroll
    for (int v = V - 1; v >= 0; --v) {
      const uint64_t holders = __ballot(key[v] == best);
      if (holders) id = v * kWave + __builtin_ctzll(holders);
    }
    const float value = key_value(best);
    if (s == 0) top = value;
    if (lane == s) mine = value, my_id = id;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * kWave + lane == id) key[v] = 0;
  }
  // A row of only -inf has no expert to weigh: weights 0. NaN and +inf make the row's weights NaN.
  const bool none = top == -INFINITY;
  float e = lane < top_k && !none ? expf(mine - top) : 0.f;
  float sum = 0.f;
  if (normalize) {
    sum = wave_sum(e);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (all[v] != 0 && !none) sum += expf(key_value(all[v]) - top);
    sum = wave_sum(sum);
  }
  if (lane < top_k) {
    weights[t * top_k + lane] = none ? 0.f : e / sum;
    ids[t * top_k + lane] = my_id;
  }
}

template <int DT>
void launch_route(const void* logits, int64_t stride, float* weights, int32_t* ids, int64_t tokens,
                  int experts, int top_k, bool normalize, hipStream_t s) {
  const dim3 grid(static_cast<uint32_t>((tokens + 3) / 4));
#define MI355X_ROUTE(V)                                                                     \
  route_kernel<DT, V><<<grid, 256, 0, s>>>(logits, stride, weights, ids, tokens, experts, top_k, \
                                           normalize)
  if (experts <= 64)
    MI355X_ROUTE(1);
  else if (experts <= 128)
    MI355X_ROUTE(2);
  else if (experts <= 256)
    MI355X_ROUTE(4);
  else if (experts <= 512)
    MI355X_ROUTE(8);
  else
    MI355X_ROUTE(16);
#undef MI355X_ROUTE
}

// ---------------------------------------------------------------------------- grouping
constexpr int kGroupThreads = 1024;
constexpr int kGroupChunk = 2048;  // slots a workgroup of the grouping passes takes

__device__ __forceinline__ bool takes_part(int e, int experts) { return e >= 0 && e < experts; }

// counts[chunk][e]: slots of a chunk that go to expert e.
__global__ __launch_bounds__(kGroupThreads) void count_slots(const int32_t* __restrict__ ids,
                                                             int slots, int experts,
                                                             int32_t* __restrict__ counts) {
  __shared__ int hist[kMaxExperts];
  for (int e = threadIdx.x; e < experts; e += kGroupThreads) hist[e] = 0;
  __syncthreads();
  const int begin = blockIdx.x * kGroupChunk, end = min(slots, begin + kGroupChunk);
  for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
    const int e = ids[i];
    if (takes_part(e, experts)) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kGroupThreads)
    counts[blockIdx.x * experts + e] = hist[e];
}

// Exclusive prefix sum of one value a thread over the workgroup.
__device__ __forceinline__ int block_exclusive(int v, int4 (&wave_totals)[4]) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int s = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == kWave - 1) reinterpret_cast<int*>(wave_totals)[wave] = s;
  __syncthreads();
  int before = s - v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int4 t = wave_totals[i];
    before += (4 * i < wave ? t.x : 0) + (4 * i + 1 < wave ? t.y : 0) + (4 * i + 2 < wave ? t.z : 0) +
              (4 * i + 3 < wave ? t.w : 0);
  }
  return before;
}

// order[row]: the slots in the order of their experts; row_weights[row]: their weights. `counts`
// may be null with one chunk. The first workgroup writes the list of row tiles for the gate_up
// product, the second (or the first, if alone) that for the down product. The order of the slots
// within an expert is that of the LDS atomics; a row's products do not depend on the row it stands
// in.
struct SlotsToPlace {
  const int32_t* ids;
  const float* weights;
  const int32_t* counts;
  int32_t* order;
  float* row_weights;
  int4* gate_up_tiles;
  int4* down_tiles;
  int32_t* tile_counts;
  int32_t slots, experts, gate_up_bm, down_bm, chunks;
};

__device__ __forceinline__ void place_chunk(const SlotsToPlace& p) {
  static_assert(kMaxExperts == kGroupThreads, "an expert a thread");
  __shared__ int cursor[kMaxExperts], totals[kMaxExperts];
  __shared__ int4 wave_totals[4];
  const int e = threadIdx.x;
  const int begin = blockIdx.x * kGroupChunk, end = min(p.slots, begin + kGroupChunk);
  cursor[e] = totals[e] = 0;  // slots of the chunks before this one, and of all
  __syncthreads();
  if (p.counts) {
    const int before = static_cast<int>(blockIdx.x) * p.experts;
    for (int i = threadIdx.x; i < p.chunks * p.experts; i += kGroupThreads) {
      const int n = p.counts[i];
      if (n == 0) continue;
      atomicAdd(&totals[i % p.experts], n);
      if (i < before) atomicAdd(&cursor[i % p.experts], n);
    }
  } else {
    for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
      const int x = p.ids[i];
      if (takes_part(x, p.experts)) atomicAdd(&totals[x], 1);
    }
  }
  __syncthreads();
  const int total = totals[e];
  const int first = block_exclusive(total, wave_totals);
  cursor[e] += first;
  for (int product = 0; product < 2; ++product) {
    if (static_cast<int>(blockIdx.x) != min(product, p.chunks - 1)) continue;
    const int bm = product ? p.down_bm : p.gate_up_bm;
    int4* tiles = product ? p.down_tiles : p.gate_up_tiles;
    const int n = (total + bm - 1) / bm;
    const int at = block_exclusive(n, wave_totals);
    for (int i = 0; i < n; ++i)
      tiles[at + i] = make_int4(e, first + i * bm, min(first + (i + 1) * bm, first + total), 0);
    if (e == kGroupThreads - 1) p.tile_counts[product] = at + n;
  }
  __syncthreads();
  for (int i = begin + threadIdx.x; i < end; i += kGroupThreads) {
    const int x = p.ids[i];
    if (takes_part(x, p.experts)) {
      const int row = atomicAdd(&cursor[x], 1);
      p.order[row] = i;
      p.row_weights[row] = p.weights[i];
    }
  }
}

__global__ __launch_bounds__(kGroupThreads) void place_slots(SlotsToPlace p) { place_chunk(p); }

// The same with the rows of x quantised by the workgroups behind the chunks': one launch less
// before the products (8-bit experts of 40 tokens 110 -> 108 us). A wave a row of up to 2,048
// columns (6,208 rows of 1,497 in 12.8 us, 19.8 with four waves each).
template <int DT, int LANES, int HELD>
__global__ __launch_bounds__(kGroupThreads) void place_and_quantize(SlotsToPlace p,
                                                                    RowsToQuantize q) {
  __shared__ uint32_t wave_top[kGroupThreads / kWave];
  if (static_cast<int>(blockIdx.x) < p.chunks)
    place_chunk(p);
  else
    quantize_row<DT, LANES, HELD>(
        q, (int64_t(blockIdx.x) - p.chunks) * (kGroupThreads / LANES) + threadIdx.x / LANES,
        wave_top);
}

// ---------------------------------------------------------------------------- the sum over slots
// out[t] = sum of y[t * top_k + s] (fp32) over the slots that take part and the parts of K, in
// fp32 and in this order. A thread takes 4 H columns. Bound by memory where there are many tokens
// (8,192 of 8 slots and 2,048 columns: 570 MB in 111 us, 5.1 TB/s), else by latency: H 1 and
// workgroups of a wave spread over the chip (40 tokens 4.0 to 4.8 us).
template <int DT, int H, int THREADS, bool PARTS>
__global__ __launch_bounds__(THREADS) void sum_slots(const float* __restrict__ y, int64_t ldy,
                                                 const int32_t* __restrict__ ids,
                                                 uint16_t* __restrict__ out, int64_t ldo,
                                                 int64_t tokens, int top_k, int splits, int experts,
                                                 int width) {
  const int chunks = (width + 4 * H - 1) / (4 * H);
  // at most 2^17 tokens of 2^14 chunks a pass (H 1: fewer than kManyValues values)
  const uint32_t i = blockIdx.x * uint32_t(THREADS) + threadIdx.x;
  const uint32_t t = i / static_cast<uint32_t>(chunks);
  if (t >= tokens) return;
  const int c = static_cast<int>(i - t * chunks) * (4 * H);
  float sum[4 * H] = {};
  constexpr int kAtOnce = 8;  // slots whose loads are on their way together
  const int first = static_cast<int>(t) * top_k, plane = static_cast<int>(tokens) * top_k;
  for (int s0 = 0; s0 < top_k * splits; s0 += kAtOnce) {
    bool in[kAtOnce];
    int32_t slots[kAtOnce];
    uint4 v[kAtOnce][H];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int n = min(s0 + i, top_k * splits - 1);
      int slot = first + n;
      slots[i] = slot;
      if constexpr (PARTS) {  // plane n / top_k of the slots
        const int part = n / top_k;
        slot -= part * top_k;
        slots[i] = part * plane + slot;
      }
      in[i] = s0 + i < top_k * splits && takes_part(ids[slot], experts);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (in[i]) {
        // rows of y are padded to 8 columns
#pragma unroll
        for (int h = 0; h < H; ++h)
          v[i][h] = ld128(y + static_cast<int64_t>(slots[i]) * ldy + c + 4 * h);
      }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        sum[4 * h] += __uint_as_float(v[i][h].x);
        sum[4 * h + 1] += __uint_as_float(v[i][h].y);
        sum[4 * h + 2] += __uint_as_float(v[i][h].z);
        sum[4 * h + 3] += __uint_as_float(v[i][h].w);
      }
    }
  }
  uint16_t* o = out + static_cast<int64_t>(t) * ldo + c;
  if (c + 4 * H <= width) {
    if constexpr (H == 2)
      st128_any(o, pack8<DT>(sum));
    else
      st64_any(o, make_uint2(Elem<DT>::pack2(sum[0], sum[1]), Elem<DT>::pack2(sum[2], sum[3])));
  } else {
#pragma unroll
    for (int e = 0; e < 4 * H; ++e)
      if (c + e < width) o[e] = Elem<DT>::from_float(sum[e]);
  }
}

// ---------------------------------------------------------------------------- the products
int64_t pad(int64_t n, int64_t a) { return (n + a - 1) / a * a; }

// A few slots run one by one on vector math, without grouping (see product_vec.h), a token's slots
// summed in the down product. That reads an expert's weights once a slot in two launches; the
// grouped products read them once in four and more. Estimated in us: a slot costs 0.2 and its
// weights (b MB) at 7.1 TB/s, in 8 bits, where each workgroup quantises the rows it takes, at 4;
// grouping costs 12 and the weights of the experts that so many tokens reach on average, at 7.1.
// Measured one by one / grouped: 128 experts of 9.4 MB, 8 a token, bf16, 1 to 8 tokens 18 / 31, 28
// / 39, 39 / 49, 49 / 60, 70 / 84 (6), 91 / 91 us; 8 of 17 MB, 2 a token 30 / 29 at 4 tokens, 52 /
// 32 at 8; in 8 bits 34 / 26 and 59 / 28. Over 96 such batches the rule costs 1.3% more than the
// better of the two every time (a limit of 16 slots 13%).
constexpr int64_t kMaxOneByOne = 64;
bool one_by_one(int64_t tokens, int64_t top_k, int64_t experts, int64_t hidden, int64_t inter,
                bool int8) {
  const int64_t slots = tokens * top_k;
  if (slots > kMaxOneByOne || top_k > kVecDownSlots ||
      (int8 && (pad(hidden, 16) > kVecLds || top_k * pad(inter, 16) > kVecLds)))
    return false;
  const float b = static_cast<float>(3 * hidden * inter) * (int8 ? 1e-6f : 2e-6f);
  const float e = static_cast<float>(experts);
  const float share = std::min(1.f, static_cast<float>(top_k) / e);
  const float reached = e * (1.f - std::pow(1.f - share, static_cast<float>(tokens)));
  return static_cast<float>(slots) * (0.2f + (int8 ? 0.25f : 0.14f) * b) < 12.f + reached * 0.14f * b;
}

// How a grouped product is computed: the tiles and, for the down product, the parts of K.
struct GroupedPlan {
  Tile tile;
  int splits;
};

// Estimated time in us of `count` tiles over `steps` 128-byte steps of K, as tile_estimate does for
// dense rows but with what gathered rows and ragged groups cost: a step of 128 rows two a CU 0.66
// instead of 0.58, and a second round of 256-row tiles from 0.95 of a round on, as the groups are
// never even.
float grouped_estimate(Tile tile, float count, float steps, float weight_bytes, bool half, int cus) {
  const float r = count / static_cast<float>(cus), busy = std::min(r, 1.f);
  float step, rounds = 1.f;
  if (tile == Tile::k64) {
    step = 0.27f;
    if (r > 1.f) rounds = std::max(1.07f * r - 0.07f, std::min(2.f, 1.f + 2.5f * (r - 1.f)));
  } else if (tile == Tile::k128Two) {
    step = 0.66f;
    rounds = std::max(2.f, r + 0.3f);
  } else {
    step = half ? 0.65f + 0.7f * busy : 1.2f + 0.6f * busy;
    if (r > 0.95f) rounds = r <= 3.f ? std::ceil(r + 0.05f) : r + 0.3f;
  }
  return 3.3f + std::max(steps * step * rounds, weight_bytes / 5.8e6f);
}

// The least estimate. How many rows an expert gets is not known on the host; it is taken to be the
// same for all, with 0.4 of a tile more each for the ragged ends. Tiles of 64, of 128 two a CU and
// of 256 rows: over 114 products of 4 to 132 experts and 8 to 1,637 rows each, int8 and bf16, the
// choice costs 2.4% more than the best of the three every time. A product whose slot outputs are
// summed afterwards may be cut along K as well, where its tiles leave CUs without one: the parts
// are summed with the slots (down of 8 experts 1024 x 2816 at 77 tokens 17.0 us whole, 11.9 in two
// parts).
constexpr int64_t kManyValues = int64_t(1) << 22;  // slot outputs that fill the chip by themselves
GroupedPlan choose_grouped(int64_t slots, int64_t experts, int64_t weight_rows, int64_t k_bytes,
                           bool summed, int cus) {
  const float active = static_cast<float>(std::min(slots, experts));
  const float per = static_cast<float>(slots) / active;
  const float weights = active * static_cast<float>(weight_rows) * static_cast<float>(k_bytes);
  const int64_t steps = (k_bytes + kProdRow - 1) / kProdRow;
  GroupedPlan best{Tile::k64, 1};
  float best_us = 1e30f;
  for (const Tile tile : {Tile::k64, Tile::k128Two, Tile::k256}) {
    const TileShape& t = kTileShapes[static_cast<int>(tile)];
    const float count = active * std::max(1.f, per / static_cast<float>(t.bm) + 0.4f) *
                        std::ceil(static_cast<float>(weight_rows) / static_cast<float>(t.bn));
    for (int s = 1; s <= (summed && tile == Tile::k64 ? 4 : 1); s *= 2) {
      const int64_t part = (steps + s - 1) / s;
      if (s > 1 && (part < 8 || part * (s - 1) >= steps ||
                    count * static_cast<float>(s / 2) >= static_cast<float>(cus) ||
                    slots * weight_rows >= kManyValues))
        break;
      float us = grouped_estimate(tile, count * static_cast<float>(s), static_cast<float>(part),
                                  weights, per <= 128.f, cus);
      // four bytes a value more, out and back
      us += static_cast<float>(s - 1) * (0.3f + static_cast<float>(slots * weight_rows) * 8 / 4.5e6f);
      if (us < best_us) {
        best_us = us;
        best = {tile, s};
      }
    }
  }
  return best;
}

constexpr int64_t kMaxSlots = 131072;  // slots a pass takes; more tokens run in several passes

struct ExpertWorkspace {
  int64_t order, row_weights, gate_up_tiles, down_tiles, tile_counts, counts, xq, xs, act, actq, acts,
      y, bytes;
  int64_t tokens;  // a pass
  GroupedPlan gate_up, down;
};

ExpertWorkspace expert_workspace(int64_t tokens, int64_t top_k, int64_t experts, int64_t hidden,
                                 int64_t inter, bool int8, int64_t x_stride, int cus) {
  ExpertWorkspace w{};
  // Row offsets into x are 32-bit within a pass.
  const int64_t most = std::max<int64_t>(
      1, std::min<int64_t>(kMaxSlots / top_k, ((int64_t(1) << 32) - 1) / x_stride));
  const int64_t t = std::min(tokens, most);
  const int64_t slots = t * top_k;
  w.tokens = t;
  w.gate_up =
      choose_grouped(slots, experts, 2 * inter, int8 ? pad(hidden, 16) : hidden * 2, false, cus);
  w.down = choose_grouped(slots, experts, hidden, int8 ? pad(inter, 16) : inter * 2, true, cus);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at = pad(at + bytes, 256);
    return o;
  };
  w.order = take(slots * 4);
  w.row_weights = take(slots * 4);
  const int64_t tiles = std::min(experts, slots) + slots / kTileShapes[0].bm + 1;
  w.gate_up_tiles = take(tiles * 16);
  w.down_tiles = take(tiles * 16);
  w.tile_counts = take(8);
  w.counts = take(pad(slots, kGroupChunk) / kGroupChunk * experts * 4);
  // fp32 for int8 and where slots run one by one
  w.act = take(std::max(slots * (int8 ? pad(inter, 4) * 4 : inter * 2),
                        std::min(slots, kMaxOneByOne) * inter * 4));
  if (int8) {
    w.xq = take(t * pad(hidden, 128));
    w.xs = take(t * 4);
    w.actq = take(slots * pad(inter, 128));
    w.acts = take(slots * 4);
  }
  w.y = take(slots * w.down.splits * pad(hidden, 8) * 4);
  w.bytes = at;
  return w;
}

// Workgroups of a grouped product over `columns` columns in tiles of `bn` of them: the row tiles that
// so many slots need at most (every full one and one more an expert) by the column tiles.
int64_t grouped_grid(Tile tile, int64_t bn, int64_t slots, int64_t experts, int64_t columns,
                     int64_t splits) {
  const int64_t most =
      slots / kTileShapes[static_cast<int>(tile)].bm + std::min(experts, slots);
  return pad(most * ((columns + bn - 1) / bn) * splits, 8);
}

template <int IN, int OT, int MODE, bool SILU>
void launch_product(const ProductArgs& base, Tile tile, int64_t slots, int64_t experts,
                    hipStream_t s) {
  ProductArgs a = base;
  const TileShape& t = kTileShapes[static_cast<int>(tile)];
  const int bn = SILU ? t.bn / 2 : t.bn;
  a.tiles_n = (a.columns + bn - 1) / bn;
  const dim3 g(
      static_cast<uint32_t>(grouped_grid(tile, bn, slots, experts, a.columns, a.splits)));
  switch (tile) {
    case Tile::k64: product_tile<IN, OT, MODE, SILU, 64, 64, 2, 2, 3><<<g, 256, 0, s>>>(a); break;
    case Tile::k128Two:
      product_tile<IN, OT, MODE, SILU, 128, 128, 4, 2, 2><<<g, 512, 0, s>>>(a);
      break;
    default:  // k256
      if (a.k_bytes % kProdRow)
        product_large<IN, OT, MODE, SILU, 256, 8, true><<<g, 512, 0, s>>>(a);
      else
        product_large<IN, OT, MODE, SILU, 256, 8, false><<<g, 512, 0, s>>>(a);
      break;
  }
}

struct ExpertCall {
  const uint8_t* x;
  int64_t x_stride;  // bytes
  const int32_t* ids;
  const float* weights;
  const uint8_t* gate_up;
  const float* gate_up_scales;
  const uint8_t* down;
  const float* down_scales;
  int64_t ld_gate_up, ld_down;  // bytes a row
  uint16_t* out;
  int64_t ldo;
  int64_t tokens, top_k, experts, hidden, inter;
};

// The slots one by one.
template <int IN, int OT>
const char* expert_slots(const ExpertCall& c, const ExpertWorkspace& w, uint8_t* ws,
                         hipStream_t s) {
  constexpr bool kQuant = IN == kInt8;
  constexpr int kWaves = kQuant ? 16 : 4;
  const int64_t slots = c.tokens * c.top_k;
  ProductArgs a{};
  a.x = c.x;
  a.x_stride = c.x_stride;
  a.k_bytes = static_cast<int32_t>(kQuant ? pad(c.hidden, 16) : c.hidden * 2);
  a.w = c.gate_up;
  a.w_stride = c.ld_gate_up;
  a.w_expert = 2 * c.inter * c.ld_gate_up;
  a.w_scales = c.gate_up_scales;
  a.ids = c.ids;
  a.rows = static_cast<int32_t>(slots);
  a.top_k = static_cast<int32_t>(c.top_k);
  a.experts = static_cast<int32_t>(c.experts);
  a.out = ws + w.act;
  a.ldo = kQuant ? pad(c.inter, 4) : c.inter;
  a.columns = static_cast<int32_t>(c.inter);
  a.tiles_n = static_cast<int32_t>((c.inter + kWaves - 1) / kWaves);
  product_vec<IN, OT, kFloatOut, kGateUp, true, 1, 2, kWaves>
      <<<dim3(static_cast<uint32_t>(pad(slots * a.tiles_n, 8))), 64 * kWaves, 0, s>>>(
          a, static_cast<int>(c.hidden));
  if (const char* e = launch_status("product (gate_up)")) return e;
  DownArgs d{};
  d.act = ws + w.act;
  d.act_stride = a.ldo * 4;
  d.w = c.down;
  d.w_stride = c.ld_down;
  d.w_expert = c.hidden * c.ld_down;
  d.w_scales = c.down_scales;
  d.out = c.out;
  d.ldo = c.ldo;
  d.ids = c.ids;
  d.weights = c.weights;
  d.top_k = a.top_k;
  d.experts = a.experts;
  d.columns = static_cast<int32_t>(c.hidden);
  d.k_bytes = static_cast<int32_t>(kQuant ? pad(c.inter, 16) : c.inter * 2);
  d.width = static_cast<int32_t>(c.inter);
  constexpr int kDownWaves = kQuant ? 8 : 4;
  const dim3 grid(static_cast<uint32_t>((c.hidden + kDownWaves - 1) / kDownWaves),
                  static_cast<uint32_t>(c.tokens));
  if (d.k_bytes <= 16 * 48)
    product_vec_down<IN, OT, 16, 2, kDownWaves><<<grid, 64 * kDownWaves, 0, s>>>(d);
  else if (d.k_bytes <= 32 * 48)
    product_vec_down<IN, OT, 32, 4, kDownWaves><<<grid, 64 * kDownWaves, 0, s>>>(d);
  else
    product_vec_down<IN, OT, 64, 4, kDownWaves><<<grid, 64 * kDownWaves, 0, s>>>(d);
  return launch_status("product (down)");
}

// One pass over c.tokens tokens. IN: the operands' kind, OT: x's and out's type.
template <int IN, int OT>
const char* expert_pass(const ExpertCall& c, const ExpertWorkspace& w, uint8_t* ws, hipStream_t s) {
  constexpr bool kQuant = IN == kInt8;
  const int64_t slots = c.tokens * c.top_k;
  if (one_by_one(c.tokens, c.top_k, c.experts, c.hidden, c.inter, kQuant))
    return expert_slots<IN, OT>(c, w, ws, s);
  const int64_t gate_up_k = kQuant ? int8_k(c.hidden, c.ld_gate_up) : c.hidden * 2;
  const int64_t down_k = kQuant ? int8_k(c.inter, c.ld_down) : c.inter * 2;
  auto* order = reinterpret_cast<int32_t*>(ws + w.order);
  auto* row_weights = reinterpret_cast<float*>(ws + w.row_weights);
  auto* gate_up_tiles = reinterpret_cast<int4*>(ws + w.gate_up_tiles);
  auto* down_tiles = reinterpret_cast<int4*>(ws + w.down_tiles);
  auto* tile_counts = reinterpret_cast<int32_t*>(ws + w.tile_counts);
  auto* counts = reinterpret_cast<int32_t*>(ws + w.counts);
  const int chunks = static_cast<int>(pad(slots, kGroupChunk) / kGroupChunk);
  if (chunks > 1) {
    count_slots<<<dim3(chunks), kGroupThreads, 0, s>>>(c.ids, static_cast<int>(slots),
                                                       static_cast<int>(c.experts), counts);
    if (const char* e = launch_status("count_slots")) return e;
  }
  const SlotsToPlace place{c.ids,
                           c.weights,
                           chunks > 1 ? counts : nullptr,
                           order,
                           row_weights,
                           gate_up_tiles,
                           down_tiles,
                           tile_counts,
                           static_cast<int32_t>(slots),
                           static_cast<int32_t>(c.experts),
                           kTileShapes[static_cast<int>(w.gate_up.tile)].bm,
                           kTileShapes[static_cast<int>(w.down.tile)].bm,
                           chunks};
  auto* xs = reinterpret_cast<float*>(ws + w.xs);
  if constexpr (kQuant) {
    const RowsToQuantize rows = rows_to_quantize(c.x, c.x_stride, ws + w.xq, gate_up_k, xs,
                                                 c.tokens, c.hidden, gate_up_k);
    auto launch = [&](auto kernel, int lanes) {
      const int64_t groups = (c.tokens * lanes + kGroupThreads - 1) / kGroupThreads;
      kernel<<<dim3(static_cast<uint32_t>(chunks + groups)), kGroupThreads, 0, s>>>(place, rows);
    };
    if (c.hidden <= 2048)
      launch(place_and_quantize<OT, kWave, 2>, kWave);
    else
      launch(place_and_quantize<OT, 256, 1>, 256);
  } else {
    place_slots<<<dim3(chunks), kGroupThreads, 0, s>>>(place);
  }
  if (const char* e = launch_status("place_slots")) return e;
  ProductArgs a{};
  a.order = order;
  a.tiles = gate_up_tiles;
  a.tile_count = tile_counts;
  a.row_weights = row_weights;
  a.rows = static_cast<int32_t>(slots);
  a.top_k = static_cast<int32_t>(c.top_k);
  a.experts = static_cast<int32_t>(c.experts);
  a.splits = 1;
  // gate_up with SiLU x mul into act, one row a slot. In 16 bits act is rounded to x's type, as it is
  // the operand of the next product's matrix instructions: one more independent rounding beside the
  // output's (rms error against 64 bits 0.0023 for 0.0017 in bf16, 0.00029 for 0.00021 in fp16). Two
  // operands for its high and low half would double that product's instructions, which already take
  // a third of an 8,192-token layer. Past fp16's range act is inf, as in the dense MLP. In 8 bits it
  // stays fp32 for the row pass behind it.
  if (kQuant) {
    a.x = ws + w.xq;
    a.x_stride = gate_up_k;
    a.x_scales = xs;
    a.k_bytes = static_cast<int32_t>(gate_up_k);
  } else {
    a.x = c.x;
    a.x_stride = c.x_stride;
    a.k_bytes = static_cast<int32_t>(gate_up_k);
  }
  a.w = c.gate_up;
  a.w_stride = c.ld_gate_up;
  a.w_expert = 2 * c.inter * c.ld_gate_up;
  a.w_scales = c.gate_up_scales;
  a.out = ws + w.act;
  a.ldo = kQuant ? pad(c.inter, 4) : c.inter;
  a.columns = static_cast<int32_t>(c.inter);
  launch_product<IN, kQuant ? kFloatOut : OT, kGateUp, true>(a, w.gate_up.tile, slots, c.experts, s);
  if (const char* e = launch_status("product (gate_up)")) return e;
  // down into y, one weighted row a slot
  if (kQuant) {
    // Every row of act is quantised; rows that no slot wrote (ids that take no part) are never read.
    auto* acts = reinterpret_cast<float*>(ws + w.acts);
    if (const char* e = run_quantize_rows(ws + w.act, a.ldo * 4, ws + w.actq, down_k, acts, slots,
                                          c.inter, down_k, kFloatOut, s))
      return e;
    a.x = ws + w.actq;
    a.x_stride = down_k;
    a.x_scales = acts;
    a.k_bytes = static_cast<int32_t>(down_k);
  } else {
    a.x = ws + w.act;
    a.x_stride = c.inter * 2;
    a.k_bytes = static_cast<int32_t>(down_k);
  }
  a.tiles = down_tiles;
  a.tile_count = tile_counts + 1;
  a.w = c.down;
  a.w_stride = c.ld_down;
  a.w_expert = c.hidden * c.ld_down;
  a.w_scales = c.down_scales;
  a.out = ws + w.y;
  a.splits = w.down.splits;
  a.ldo = pad(c.hidden, 8);
  a.columns = static_cast<int32_t>(c.hidden);
  launch_product<IN, kFloatOut, kDown, false>(a, w.down.tile, slots, c.experts, s);
  if (const char* e = launch_status("product (down)")) return e;
  const auto* y = reinterpret_cast<const float*>(ws + w.y);
  auto sum = [&](auto kernel, int columns, int threads) {
    const int64_t n = c.tokens * ((c.hidden + columns - 1) / columns);
    kernel<<<dim3(static_cast<uint32_t>((n + threads - 1) / threads)), threads, 0, s>>>(
        y, a.ldo, c.ids, c.out, c.ldo, c.tokens,
        static_cast<int>(c.top_k), w.down.splits, static_cast<int>(c.experts),
        static_cast<int>(c.hidden));
  };
  if (w.down.splits > 1)
    sum(sum_slots<OT, 1, kWave, true>, 4, kWave);
  else if (c.tokens * c.hidden >= kManyValues)
    sum(sum_slots<OT, 2, 256, false>, 8, 256);
  else
    sum(sum_slots<OT, 1, kWave, false>, 4, kWave);
  return launch_status("sum_slots");
}

bool expert_shape_ok(int64_t tokens, int64_t top_k, int64_t experts, int64_t hidden,
                     int64_t inter, bool int8) {
  return tokens >= 0 && tokens < (int64_t(1) << 31) && top_k > 0 && top_k <= kMaxTopK &&
         experts > 0 && experts <= kMaxExperts && hidden > 0 && inter > 0 &&
         hidden <= 131072 && inter <= 131072 && (int8 || (hidden % 8 == 0 && inter % 8 == 0));
}

}  // namespace
}  // namespace mi355x

using namespace mi355x;

extern "C" const char* mi355x_route_experts(const void* logits, int64_t ld, void* weights,
                                            int32_t* ids, int64_t tokens, int64_t experts,
                                            int64_t top_k, bool normalize, int dtype,
                                            void* stream) {
  if (tokens < 0 || tokens >= (int64_t(1) << 31) || experts <= 0 || experts > kMaxExperts ||
      top_k <= 0 || top_k > std::min<int64_t>(experts, kMaxTopK) || ld < experts || dtype < 0 ||
      dtype > 2)
    return set_error("mi355x_route_experts: unsupported shape (up to 1024 experts, top_k up to 64)");
  if (tokens == 0) return nullptr;
  if (!logits || !weights || !ids) return set_error("mi355x_route_experts: null pointer");
  if (!aligned(logits, dtype == 2 ? 4 : 2) || !aligned(weights, 4) || !aligned(ids, 4))
    return set_error("mi355x_route_experts: misaligned operand");
  auto s = static_cast<hipStream_t>(stream);
  const int e = static_cast<int>(experts), k = static_cast<int>(top_k);
  auto* p = static_cast<float*>(weights);
  for (int64_t t = 0; t < tokens; t += kMaxLaunchRows) {
    const int64_t n = std::min(kMaxLaunchRows, tokens - t);
    const auto* rows = static_cast<const uint8_t*>(logits) + t * ld * (dtype == 2 ? 4 : 2);
    float* w = p + t * top_k;
    int32_t* chosen = ids + t * top_k;
    if (dtype == 0)
      launch_route<0>(rows, ld, w, chosen, n, e, k, normalize, s);
    else if (dtype == 1)
      launch_route<1>(rows, ld, w, chosen, n, e, k, normalize, s);
    else
      launch_route<2>(rows, ld, w, chosen, n, e, k, normalize, s);
    if (const char* err = launch_status("route_kernel")) return err;
  }
  return nullptr;
}

extern "C" int64_t mi355x_expert_mlp_workspace_bytes(int64_t tokens, int64_t top_k, int64_t experts,
                                                     int64_t hidden, int64_t inter, int64_t ldx,
                                                     bool int8, int32_t cus) {
  if (!expert_shape_ok(tokens, top_k, experts, hidden, inter, int8) || ldx < hidden ||
      ldx >= (int64_t(1) << 31))
    return -1;
  return expert_workspace(tokens, top_k, experts, hidden, inter, int8, ldx * 2,
                          cus > 0 ? cus : 256)
      .bytes;
}

extern "C" bool mi355x_expert_mlp_plan(int64_t tokens, int64_t top_k, int64_t experts,
                                       int64_t hidden, int64_t inter, int64_t ldx, bool int8,
                                       int32_t cus, int32_t* plan) {
  if (!plan || tokens == 0 ||
      mi355x_expert_mlp_workspace_bytes(tokens, top_k, experts, hidden, inter, ldx, int8, cus) < 0)
    return false;
  const ExpertWorkspace w =
      expert_workspace(tokens, top_k, experts, hidden, inter, int8, ldx * 2, cus > 0 ? cus : 256);
  plan[0] = one_by_one(w.tokens, top_k, experts, hidden, inter, int8);
  plan[1] = static_cast<int32_t>(w.gate_up.tile);
  plan[2] = static_cast<int32_t>(w.down.tile);
  plan[3] = w.down.splits;
  return true;
}

extern "C" const char* mi355x_expert_mlp(const void* x, int64_t ldx, const int32_t* ids,
                                         const float* weights, const void* gate_up,
                                         int64_t ld_gate_up, const float* gate_up_scales,
                                         const void* down, int64_t ld_down,
                                         const float* down_scales, void* out, int64_t ldo,
                                         int64_t tokens, int64_t top_k, int64_t experts,
                                         int64_t hidden, int64_t inter, void* workspace,
                                         int64_t workspace_bytes, int32_t cus, int64_t dtype,
                                         void* stream) {
  const bool int8 = gate_up_scales != nullptr;
  if (int8 != (down_scales != nullptr))
    return set_error("mi355x_expert_mlp: gate_up and down weights must be of one kind");
  const int64_t size = int8 ? 1 : 2;
  if (!expert_shape_ok(tokens, top_k, experts, hidden, inter, int8) || ldx < hidden ||
      ldx >= (int64_t(1) << 31) || ldo < hidden || ld_gate_up < (int8 ? pad(hidden, 16) : hidden) ||
      ld_down < (int8 ? pad(inter, 16) : inter) || ld_gate_up * size % 16 || ld_down * size % 16 ||
      (!int8 && ldx % 8) || (dtype != 0 && dtype != 1))
    return set_error("mi355x_expert_mlp: unsupported shape (up to 1024 experts, top_k up to 64, "
                     "weight and 16-bit x rows of whole 16-byte words)");
  if (2 * inter * ld_gate_up * size >= (int64_t(1) << 32) ||
      hidden * ld_down * size >= (int64_t(1) << 32))
    return set_error("mi355x_expert_mlp: an expert's weight must be less than 4 GiB");
  if (tokens == 0) return nullptr;
  if (!x || !ids || !weights || !gate_up || !down || !out || !workspace)
    return set_error("mi355x_expert_mlp: null pointer");
  if (!aligned(x, int8 ? 2 : 16) || !aligned(gate_up, 16) || !aligned(down, 16) ||
      !aligned(out, 2) || !aligned(workspace, 16) || !aligned(ids, 4) || !aligned(weights, 4))
    return set_error("mi355x_expert_mlp: misaligned operand");
  const ExpertWorkspace w =
      expert_workspace(tokens, top_k, experts, hidden, inter, int8, ldx * 2, cus > 0 ? cus : 256);
  if (workspace_bytes < w.bytes) return set_error("mi355x_expert_mlp: workspace too small");
  const auto threads = [&](Tile tile, bool silu, int64_t columns, int64_t splits) {
    const int bn = kTileShapes[static_cast<int>(tile)].bn / (silu ? 2 : 1);
    return grouped_grid(tile, bn, w.tokens * top_k, experts, columns, splits) *
           (tile == Tile::k64 ? 256 : 512);
  };
  if (threads(w.gate_up.tile, true, inter, 1) > kMaxGridThreads ||
      threads(w.down.tile, false, hidden, w.down.splits) > kMaxGridThreads)
    return set_error("mi355x_expert_mlp: grid too large");
  auto s = static_cast<hipStream_t>(stream);
  for (int64_t t = 0; t < tokens; t += w.tokens) {
    ExpertCall c{};
    c.x = static_cast<const uint8_t*>(x) + t * ldx * 2;
    c.x_stride = ldx * 2;
    c.ids = ids + t * top_k;
    c.weights = weights + t * top_k;
    c.gate_up = static_cast<const uint8_t*>(gate_up);
    c.gate_up_scales = gate_up_scales;
    c.down = static_cast<const uint8_t*>(down);
    c.down_scales = down_scales;
    c.ld_gate_up = ld_gate_up * size;
    c.ld_down = ld_down * size;
    c.out = static_cast<uint16_t*>(out) + t * ldo;
    c.ldo = ldo;
    c.tokens = std::min(w.tokens, tokens - t);
    c.top_k = top_k;
    c.experts = experts;
    c.hidden = hidden;
    c.inter = inter;
    auto* ws = static_cast<uint8_t*>(workspace);
    const char* e = int8 ? (dtype == 0 ? expert_pass<kInt8, 0>(c, w, ws, s)
                                       : expert_pass<kInt8, 1>(c, w, ws, s))
                         : (dtype == 0 ? expert_pass<kBf16, 0>(c, w, ws, s)
                                       : expert_pass<kFp16, 1>(c, w, ws, s));
    if (e) return e;
  }
  return nullptr;
}
