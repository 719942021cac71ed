// Attention over prefixes that requests of a batch share, computed once for all of them and joined
// with what each has of its own. No counterpart in the reference, whose backends read every
// request's whole cache (src/models/attention/backend.rs:316-804).
//
//   o = sum_i 2^(a_i) o_i / sum_i 2^(a_i),  (o_i, a_i) the normalised output and the log2 of the sum
//   of 2^score over part i of a request's keys: parts of the prefix and parts of its own.
//
// A group's queries (every token's G heads under a kv head, heads fastest: tokens x G columns) meet
// the prefix's keys as one matrix product, where plain decode reads the prefix once a request. Two
// loops, by the number of columns:
//
// stream_items, up to 32 columns: the decode kernel's copy pipeline (tiles of 16 whole K and V rows
// through an LDS ring, one wave a kv head) with up to two sets of 16 columns on the tile a wave has
// in LDS. Streaming a tile takes a CU longer than two sets of products on it, so it is bound by
// memory, as decode is. The own keys of requests with few new tokens are items too, under the same
// balanced schedule.
//
// gemm_items, more: 32 columns a wave against a range of 64-key tiles, as the prefill kernel
// (S^T = K Q^T, P^T = 2^(S^T - m), O^T += V^T P^T on 32 x 32 x 16 products), K and V read once for
// 256 columns. Own keys of requests with many new tokens go there too, under a horizon a column.
//
// One is bound by memory and the other by the matrix cores, so one launch holds both where the number
// of kv heads lets it: shared_wide_kernel on whole CUs for either, shared_kernel on halves of a CU.
// shared_gemm_kernel and shared_stream_kernel follow each other elsewhere.
//
// Every part that is joined writes fp32 outputs and their log2-sum-exp; shared_merge_kernel joins
// them. A request that shares nothing and whose keys one item holds is written directly.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <limits>

#include "buffer.h"
#include "mfma.h"
#include "shared.h"

namespace mi355x {
namespace {

constexpr int kD = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int32_t kNoHorizon = 1 << 30;  // queries that see every key of their range
constexpr int64_t kMaxKeys = int64_t(1) << 22;  // of the products: div_small is exact below this

// --- device workspace, int32
constexpr int kHeaderInts = 4;
constexpr int kHeaderGemmItems = 0, kHeaderStreamWgs = 1, kHeaderOnce = 2, kHeaderGemmWgs = 3;
constexpr int kInfoInts = 8;    // a request: {first slot, splits, tokens, token0} of the prefix's
                                // parts, then of its own (splits 0: none)
constexpr int kStreamInts = 8;  // {token0, tokens, first page entry, key begin | key end, slot or -1
                                // (written directly), position of token0, 0}
constexpr int kGemmInts = 12;   // {token0, columns, first column, kv head | first page entry, tile
                                // begin, tile end, slot | position of token0, keys, 0, 0}
// A slot is a token's q heads of partial outputs: row slot * Hq + qh of part_o [rows][128].

// The products' references (gemm_items) follow every row's maximum where each row has one new token, as
// plain decode's do: the largest probability is exactly 1 when it is rounded to 16 bits, and a row that
// shares a prefix is as exact as one that does not. With more tokens they follow maxima more than 8 above
// them, as the prefill kernel's: fewer tiles are rescaled, p stays below 2^8, and the largest p is rounded
// like the others. Relative error of outputs, 2,432 bf16 keys whose scores have a deviation of 2, exact
// ones rounded once 0.0017: 0.0020, with slack 0.0024; us a layer, 256 rows sharing 8,192 tokens 125 and
// 116, 48 rows of up to 40 new tokens behind 4,096 100 and 96.5, the smaller cases as before.
constexpr float kDecodeSlack = 0.f, kExtendSlack = 8.f;

struct SharedArgs {
  const uint16_t* q;
  int64_t q_sn, q_sh;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  int64_t o_sn, o_sh;
  const int32_t* header;
  const int4* info;
  const int32_t* row_of;  // request of a token; NULL: its own number
  const int4* stream_work;
  const int32_t* stream_wg;
  const int4* gemm_work;
  const int32_t* indices;
  float* part_o;
  float* part_lse;
  int64_t rows;           // tokens * q heads
  int32_t num_q_heads, num_kv_heads, group_log2, page_size, gemm_grid;
  float scale_log2;
  float slack;            // gemm_items: how far a maximum may pass its reference, in log2 units
};

// ---------------------------------------------------------------------------
// Few columns: streamed.
// ---------------------------------------------------------------------------
constexpr int kStreamTile = 16;
constexpr int kStreamStages = 2;
constexpr int kStreamEntries = 2048;  // page entries of an item in LDS
constexpr int kStreamColumns = 32;  // two sets: a third does not fit the registers

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ floatx4 mma_16x16x32(const uint4& a, const uint4& b, floatx4 c) {
  if constexpr (DT == 0)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ floatx4 mma_16x16x16(const uint2& a, const uint2& b, floatx4 c) {
  if constexpr (DT == 0)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4i16_t, a),
                                                     __builtin_bit_cast(v4i16_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a),
                                                 __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
}

// W waves, one a kv head of the slice; SETS: sets of 16 columns an item may have. Tiles
// lie in LDS as decode_mma_kernel's: 16-byte chunk c of a head's 256 bytes at c ^ (token & 15).
template <int DT, int W, int SETS, bool ONCE>
__device__ __forceinline__ void stream_items(const SharedArgs& a, uint8_t* lds, int32_t* entries,
                                             int wg, int slice) {
  constexpr int T = kStreamTile;
  constexpr int kRow = W * 256;              // bytes of one token's slice (K or V)
  constexpr int kHalf = T * kRow;            // K (or V) bytes of a tile
  constexpr int kStage = 2 * kHalf;
  constexpr int kCopies = 2 * kHalf / 1024;  // 1 KiB copies of a tile
  constexpr int kPerWave = kCopies / W;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 15;   // column of a set / operand row
  const int quad = lane >> 4;  // 16-lane group
  const int h = slice * W + wave;
  const int G = 1 << a.group_log2;
  const uint32_t lds_base = lds_address(lds);
  const uint32_t entries_lds = lds_address(entries);
  const uint32_t row_elems = static_cast<uint32_t>(a.num_kv_heads) * kD;
  const uint16_t* kslice = a.k + slice * W * kD;
  const uint16_t* vslice = a.v + slice * W * kD;
  const int item_begin = a.stream_wg[wg], item_end = a.stream_wg[wg + 1];

  for (int item = item_begin; item < item_end; ++item) {
    const bool first_item = item == item_begin;
    const int4 w0 = a.stream_work[2 * item], w1 = a.stream_work[2 * item + 1];
    const int token0 = w0.x, tokens = w0.y, beg = w0.w, end = w1.x, slot = w1.y, pos0 = w1.z;
    const int first_page = beg / a.page_size;
    const int n_entries = (end - 1) / a.page_size - first_page + 1;
    const int32_t* pages = a.indices + w0.z;
    const int n_tiles = (end - beg + T - 1) / T;
    const int sets = (tokens * G + 15) >> 4;
    // Copy c of a tile: half c / (kCopies / 2), bytes from (c % (kCopies / 2)) * 1024 of its token
    // rows. An item's first tile takes its pages from memory, the others from the entries in LDS.
    auto issue = [&](int t, int stage, bool from_memory) {
#pragma unroll
      for (int j = 0; j < kPerWave; ++j) {
        const int c = wave * kPerWave + j;
        const int half = c / (kCopies / 2);
        const int r = c % (kCopies / 2);
        const int byte = r * 1024 + (W < 4 ? lane * 16 : 0);  // whole rows a copy: uniform token
        const int tile_tok = byte / kRow;
        const int tok = min(beg + t * T + tile_tok, end - 1);
        const int page = tok / a.page_size;
        int e;
        if (!from_memory) {
          e = entries[page - first_page];
        } else if constexpr (W < 4) {
          e = pages[page - first_page];
        } else {
          e = *((const __attribute__((address_space(4))) int32_t*)(pages) +
                __builtin_amdgcn_readfirstlane(page - first_page));
        }
        const uint32_t at = static_cast<uint32_t>(e) * static_cast<uint32_t>(a.page_size) +
                            static_cast<uint32_t>(tok - page * a.page_size);
        const int chunk = W < 4 ? (byte % kRow) / 16 : ((r * 1024) % kRow) / 16 + lane;
        const int src_chunk = (chunk & ~15) | ((chunk & 15) ^ (tile_tok & 15));
        const uint16_t* src =
            (half ? vslice : kslice) + static_cast<uint64_t>(at) * row_elems + src_chunk * 8;
        if constexpr (ONCE)
          copy_to_lds_nt(src, lds_base + stage * kStage + half * kHalf + r * 1024);
        else
          copy_to_lds(src, lds_base + stage * kStage + half * kHalf + r * 1024);
      }
    };
    if (!first_item) __syncthreads();  // the ring and the entries are free
    issue(0, 0, true);
    for (int base = wave * 64; base < n_entries; base += W * 64)
      copy_dword_to_lds(pages + min(base + lane, n_entries - 1), entries_lds + base * 4);
    // Q^T as the B operand: the lane's column 16 c + col is head column % G of token column / G;
    // columns past the tokens are zero.
    uint4 qb[SETS][4];
    int limit[SETS];  // last key the column sees
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
      const int column = 16 * c + col;
      const int token = column >> a.group_log2;
      limit[c] = min(end - 1, pos0 + token);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        qb[c][kk] = token < tokens ? ld128(a.q + static_cast<int64_t>(token0 + token) * a.q_sn +
                                           (h * G + (column & (G - 1))) * a.q_sh + 32 * kk +
                                           8 * quad)
                                   : make_uint4(0, 0, 0, 0);
    }
    wait_vmem_loads();  // queries, entries and the first tile

    floatx4 o[SETS][8];
    float m[SETS], l[SETS];
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
      m[c] = -1e30f;
      l[c] = 0.f;
#pragma unroll
      for (int b = 0; b < 8; ++b) o[c][b] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    for (int t = 0; t < n_tiles; ++t) {
      wait_vmcnt<0>();
      __syncthreads();
      if (t + 1 < n_tiles) issue(t + 1, (t + 1) % kStreamStages, false);
      const uint8_t* kb = lds + (t % kStreamStages) * kStage + wave * 256;
      const uint8_t* vb = kb + kHalf;
      uint4 kf[4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        kf[kk] = *reinterpret_cast<const uint4*>(kb + col * kRow + (((4 * kk + quad) ^ col) * 16));
      uint2 vf[8];
      const int vt = 4 * quad + (col >> 2);
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const int chunk = 2 * b + ((col & 3) >> 1);
        lds_u8* vp = (lds_u8*)vb + vt * kRow + ((chunk ^ vt) * 16) + 8 * (col & 1);
        vf[b] =
            __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)vp));
      }
      const int key0 = beg + t * T + 4 * quad;
      // The steps of the sets side by side.
      floatx4 sc[SETS];
#pragma unroll
      for (int c = 0; c < SETS; ++c) sc[c] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int c = 0; c < SETS; ++c) sc[c] = mma_16x16x32<DT>(kf[kk], qb[c][kk], sc[c]);
      // The lane holds S[key0 + i][column].
      float s[SETS][4], mx[SETS], corr[SETS];
#pragma unroll
      for (int c = 0; c < SETS; ++c) {
        mx[c] = m[c];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[c][i] = key0 + i <= limit[c] ? sc[c][i] * a.scale_log2 : -INFINITY;
          mx[c] = fmaxf(mx[c], s[c][i]);
        }
      }
#pragma unroll
      for (int c = 0; c < SETS; ++c) mx[c] = fmaxf(mx[c], __shfl_xor(mx[c], 16));
#pragma unroll
      for (int c = 0; c < SETS; ++c) mx[c] = fmaxf(mx[c], __shfl_xor(mx[c], 32));
      uint2 pb[SETS];
#pragma unroll
      for (int c = 0; c < SETS; ++c) {
        corr[c] = __builtin_amdgcn_exp2f(m[c] - mx[c]);
        m[c] = mx[c];
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[c][i] - mx[c]);
        l[c] = l[c] * corr[c] + ((p[0] + p[1]) + (p[2] + p[3]));
        // rounded to the type of V for the product; the sum takes the fp32 values
        pb[c] = make_uint2(Elem<DT>::pack2(p[0], p[1]), Elem<DT>::pack2(p[2], p[3]));
      }
#pragma unroll
      for (int b = 0; b < 8; ++b)
#pragma unroll
        for (int c = 0; c < SETS; ++c) {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[c][b][i] *= corr[c];
          o[c][b] = mma_16x16x16<DT>(vf[b], pb[c], o[c][b]);
        }
    }
#pragma unroll
    for (int c = 0; c < SETS; ++c) {
      if (c >= sets) break;
      float sum = l[c];
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      const int column = 16 * c + col;
      const int token = column >> a.group_log2;
      if (token >= tokens) continue;
      const int qh = h * G + (column & (G - 1));
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // 0: no key of the part is seen
      if (slot < 0) {
        uint16_t* dst =
            a.out + static_cast<int64_t>(token0 + token) * a.o_sn + qh * a.o_sh + 4 * quad;
#pragma unroll
        for (int b = 0; b < 8; ++b)
          *reinterpret_cast<uint2*>(dst + 16 * b) =
              make_uint2(Elem<DT>::pack2(o[c][b][0] * inv, o[c][b][1] * inv),
                         Elem<DT>::pack2(o[c][b][2] * inv, o[c][b][3] * inv));
      } else {
        const int64_t row = static_cast<int64_t>(slot + token) * a.num_q_heads + qh;
        float* dst = a.part_o + row * kD + 4 * quad;
#pragma unroll
        for (int b = 0; b < 8; ++b)
          *reinterpret_cast<float4*>(dst + 16 * b) = make_float4(
              o[c][b][0] * inv, o[c][b][1] * inv, o[c][b][2] * inv, o[c][b][3] * inv);
        if (quad == 0)
          a.part_lse[row] = sum == 0.f ? -INFINITY : m[c] + __builtin_amdgcn_logf(sum);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Many columns: matrix products of 32 columns a wave.
// ---------------------------------------------------------------------------
constexpr int kTileK = 64;
constexpr int kTileBytes = kTileK * kD * 2;
constexpr int kStageBytes = 2 * kTileBytes;  // K + V

// K and V tiles lie in LDS as the prefill kernel's do: [key][d], 16-byte chunk c of key r at
// c ^ (r & 15) (K) and c ^ 4 (r & 3) (V), which keeps the operand reads free of bank conflicts.
// NW waves: 8 read K and V once for 256 columns through a ring of four tiles; 4 leave half of the CU
// to another workgroup.
template <int DT, int NW>
__device__ __forceinline__ void gemm_items(const SharedArgs& a, uint8_t* lds, int first_item,
                                           int step) {
  constexpr int kStages = NW / 2;
  constexpr int kAhead = kStages - 1;
  constexpr int kGroupsPerWave = 16 / NW;  // 4-row groups of each tile this wave copies
  constexpr int kCopiesPerTile = 2 * kGroupsPerWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 31;
  const int half = lane >> 5;
  const uint32_t lds_base = lds_address(lds);
  const int64_t slot_stride = static_cast<int64_t>(a.num_kv_heads) * kD;
  const float inv_page = 1.0f / static_cast<float>(a.page_size);
  const bool fast_pages =
      a.page_size >= 4 && a.page_size <= kTileK && kTileK % a.page_size == 0;
  const int pages_per_tile = fast_pages ? kTileK / a.page_size : 0;
  const float c = a.scale_log2;

  // Operand read offsets, as in the prefill kernel.
  const int gq = lane >> 4;
  const int p16 = lane & 15;
  const int v_key = 4 * (gq >> 1) + (p16 >> 2);
  const int v_chunk_lo = 2 * (gq & 1) + ((p16 >> 1) & 1);
  int v_off[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
    v_off[db] = kTileBytes + v_key * 256 + ((4 * db + v_chunk_lo) ^ (4 * (p16 >> 2))) * 16 +
                8 * (p16 & 1);
  const int row_in_group = lane >> 4;
  const int pos = lane & 15;
  const int heads = 1 << a.group_log2;

  const int items = a.header[kHeaderGemmItems];
  for (int item = first_item; item < items; item += step) {
    const int4* work = a.gemm_work + kGemmInts / 4 * item;
    const int4 w0 = work[0], w1 = work[1], w2 = work[2];
    const int token0 = w0.x, rows = w0.y, row0 = w0.z, kvh = w0.w;
    const int page_base = w1.x, t_begin = w1.y, nt = w1.z - w1.y, slot = w1.w;
    const int pos0 = w2.x, kv_len = w2.y;
    const int my_row0 = row0 + wave * 32;
    const bool wave_active = my_row0 < rows;
    const int first_horizon = pos0 + (my_row0 >> a.group_log2);
    const int last_horizon = pos0 + (min(my_row0 + 31, rows - 1) >> a.group_log2);
    const int row = min(my_row0 + col, rows - 1);
    const int token = row >> a.group_log2;
    const int horizon = min(pos0 + token, kv_len - 1);  // the last key the column sees

    uint4 qreg[8];
    {
      const int qh = (kvh << a.group_log2) + (row & (heads - 1));
      const uint16_t* qp = a.q + static_cast<int64_t>(token0 + token) * a.q_sn + qh * a.q_sh;
#pragma unroll
      for (int s = 0; s < 8; ++s) qreg[s] = ld128(qp + 16 * s + 8 * half);
      wait_vmem_loads();
#pragma unroll
      for (int s = 0; s < 8; ++s)  // kept in registers, never reloaded inside the loop
        asm volatile("" : "+v"(qreg[s].x), "+v"(qreg[s].y), "+v"(qreg[s].z), "+v"(qreg[s].w));
    }

    const uint16_t* k_head = a.k + kvh * kD;
    const uint16_t* v_head = a.v + kvh * kD;
    const __attribute__((address_space(4))) int32_t* pages =
        (const __attribute__((address_space(4))) int32_t*)(a.indices) + page_base;
    // A tile that ends past the keys, or pages of another size: every key's own address. Keys past
    // the end repeat the last one (finite data, masked later).
    auto issue_general = [&](int t, int stage) {
      const uint32_t sbase = lds_base + stage * kStageBytes;
#pragma unroll
      for (int j = 0; j < kGroupsPerWave; ++j) {
        const int g = wave * kGroupsPerWave + j;
        const int row = 4 * g + row_in_group;
        const int key = min(t * kTileK + row, kv_len - 1);
        const int key0 =
            __builtin_amdgcn_readfirstlane(min(t * kTileK + 4 * g, (kv_len - 1) & ~3));
        int r0;
        const int p0 = __builtin_amdgcn_readfirstlane(div_small(key0, a.page_size, inv_page, r0));
        const int i0 = pages[p0], i1 = pages[p0 + 1], i2 = pages[p0 + 2], i3 = pages[p0 + 3];
        int off;
        const int sel = div_small(key, a.page_size, inv_page, off) - p0;
        const int page = sel == 0 ? i0 : sel == 1 ? i1 : sel == 2 ? i2 : i3;
        const int64_t at = static_cast<int64_t>(page) * a.page_size + off;
        copy_to_lds(k_head + at * slot_stride + (pos ^ (row & 15)) * 8, sbase + g * 1024);
        copy_to_lds(v_head + at * slot_stride + (pos ^ (4 * (row & 3))) * 8,
                    sbase + kTileBytes + g * 1024);
      }
    };
    // Whole tiles of pages of 4 to 64 tokens: a group of 4 keys lies in one page, whose id is loaded
    // a tile ahead.
    const int last_page = (kv_len - 1) / a.page_size;
    int ids[kGroupsPerWave];
    auto load_ids = [&](int t) {
#pragma unroll
      for (int j = 0; j < kGroupsPerWave; ++j) {
        const int g = wave * kGroupsPerWave + j;
        ids[j] = pages[min(t * pages_per_tile + (4 * g) / a.page_size, last_page)];
      }
    };
    auto issue_fast = [&](int t, int stage) {
      const uint32_t sbase = lds_base + stage * kStageBytes;
#pragma unroll
      for (int j = 0; j < kGroupsPerWave; ++j) {
        const int g = wave * kGroupsPerWave + j;
        const int row = 4 * g + row_in_group;
        const int64_t first = static_cast<int64_t>(ids[j]) * a.page_size + (4 * g) % a.page_size;
        const int64_t at = (first + row_in_group) * slot_stride;
        copy_to_lds(k_head + at + (pos ^ (row & 15)) * 8, sbase + g * 1024);
        copy_to_lds(v_head + at + (pos ^ (4 * (row & 3))) * 8, sbase + kTileBytes + g * 1024);
      }
    };
    auto issue = [&](int t, int stage) {
      if (fast_pages && (t + 1) * kTileK <= kv_len)
        issue_fast(t, stage);
      else
        issue_general(t, stage);
      if (fast_pages) load_ids(t + 1);
    };

    floatx16 o[4];
    // ref: the lane's reference, in log2 units; p = 2^(c s - ref), one fma a score. Its rounding
    // scales p and the sums alike.
    float ref = 0.f, l = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;

    auto compute = [&](int t, int stage, bool first) {
      const int k0 = t * kTileK;
      if (!(wave_active && k0 <= last_horizon)) return;
      const uint8_t* sb = lds + stage * kStageBytes;
      uint4 kf[2][8];
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          kf[T][kk] = *reinterpret_cast<const uint4*>(
              sb + (32 * T + col) * 256 + (((2 * kk + half) ^ (col & 15)) * 16));
      floatx16 s[2];
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[T][r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
#pragma unroll
        for (int T = 0; T < 2; ++T) s[T] = Mfma<DT>::run(kf[T][kk], qreg[kk], s[T]);
      auto load_v = [&](int kk, int db) {
        lds_u8* vp = (lds_u8*)sb + v_off[db] + 16 * kk * 256;
        const uint2 l2 =
            __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)vp));
        const uint2 h2 = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vp + 8 * 256)));
        return make_uint4(l2.x, l2.y, h2.x, h2.y);
      };
      // Half of V's operands are loaded behind the scores' products, the others where they are used:
      // all of them early do not fit the registers (us a layer, 256 rows sharing 8,192 tokens: none
      // early 125.5, half 124.8, all, with spills, 135).
      constexpr int kEarly = NW == 8 ? 2 : 0;
      uint4 vf[2][4];
#pragma unroll
      for (int kk = 0; kk < kEarly; ++kk)
#pragma unroll
        for (int db = 0; db < 4; ++db) vf[kk][db] = load_v(kk, db);
      if (k0 + kTileK - 1 > first_horizon || k0 + kTileK > kv_len) {
        const int limit = horizon - (k0 + 4 * half);
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 32 * T + (r >> 2) * 8 + (r & 3);
            s[T][r] = key <= limit ? s[T][r] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[T][r]);
      {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                          false, false);
        mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * c;
      }
      // The reference moves on the first tile and then when a row's maximum passes it by more than
      // the slack. A first tile without a finite score (past a row's horizon, or all -inf) leaves it
      // below every other, so that later scores count however far below 0 they are.
      if (first || __any(mx > ref + a.slack)) {
        const float to = fmaxf(first ? -1e30f : ref, mx);
        // nothing is accumulated before the first tile
        const float alpha = first ? 1.f : __builtin_amdgcn_exp2f(ref - to);
        ref = to;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      }
      uint4 pb[4];
      float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[T][8 * hh + i], c, -ref));
            ls[i & 3] += p[i];
          }
          // rounded to the type of V for the product; the row sums take the fp32 values
          pb[2 * T + hh] =
              make_uint4(Elem<DT>::pack2(p[0], p[1]), Elem<DT>::pack2(p[2], p[3]),
                         Elem<DT>::pack2(p[4], p[5]), Elem<DT>::pack2(p[6], p[7]));
        }
      l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int db = 0; db < 4; ++db)
          o[db] = Mfma<DT>::run(kk < kEarly ? vf[kk & 1][db] : load_v(kk, db), pb[kk], o[db]);
    };

    if (fast_pages) load_ids(t_begin);
#pragma unroll
    for (int st = 0; st < kAhead; ++st)
      if (st < nt) issue(t_begin + st, st);
    for (int u = 0; u < nt; ++u) {
      wait_tiles_ahead<kCopiesPerTile, kAhead - 1>(min(kAhead - 1, nt - 1 - u));
      __syncthreads();
      if (u + kAhead < nt) issue(t_begin + u + kAhead, (u + kAhead) % kStages);
      compute(t_begin + u, u % kStages, u == 0);
    }

    // The wave's 32 x 128 outputs go out as whole rows, through its share of the ring (16-byte chunk c
    // of row r at c ^ r): 512 bytes a row instead of 32 at a time.
    __syncthreads();
    if (wave_active) {
      const float row_sum = l + __shfl_xor(l, 32);
      const float inv = row_sum == 0.f ? 0.f : 1.f / row_sum;
      uint8_t* tile = lds + wave * (32 * kD * 4);
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
          *reinterpret_cast<float4*>(tile + col * 512 + ((8 * db + 2 * g4 + half) ^ col) * 16) =
              make_float4(o[db][4 * g4] * inv, o[db][4 * g4 + 1] * inv, o[db][4 * g4 + 2] * inv,
                          o[db][4 * g4 + 3] * inv);
      auto part_row = [&](int r) {  // partial row of the wave's row r
        const int t = (my_row0 + r) >> a.group_log2;
        return static_cast<int64_t>(slot + t) * a.num_q_heads + (kvh << a.group_log2) +
               ((my_row0 + r) & (heads - 1));
      };
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int r = 2 * j + half;
        const float4 val =
            *reinterpret_cast<const float4*>(tile + r * 512 + ((lane & 31) ^ r) * 16);
        if (my_row0 + r < rows)
          *reinterpret_cast<float4*>(a.part_o + part_row(r) * kD + (lane & 31) * 4) = val;
      }
      if (half == 0 && my_row0 + col < rows)
        a.part_lse[part_row(col)] =
            row_sum == 0.f ? -INFINITY : ref + __builtin_amdgcn_logf(row_sum);
    }
    __syncthreads();  // the next item's copies overwrite the ring
  }
}

// Both in one launch, where a slice of four kv heads lets a workgroup of either kind have half of a
// CU: the products of one hide behind the copies of the other. The first gemm_grid workgroups take
// the products, one a CU; the others stream, and have the CUs to themselves afterwards.
template <int DT, int SETS>
__global__ __launch_bounds__(256, 2) void shared_kernel(SharedArgs a) {
  constexpr int kRing = kStreamStages * 2 * kStreamTile * 4 * 256;
  static_assert(kRing == 2 * kStageBytes, "either ring");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kRing];
  __shared__ int32_t entries[kStreamEntries];
  if (a.num_kv_heads < 0) {  // the copies are invisible to the compiler: stores it sees, never taken
    lds[threadIdx.x] = 0;
    entries[threadIdx.x] = 0;
  }
  const int block = blockIdx.x;
  if (block < a.gemm_grid) {
    gemm_items<DT, 4>(a, lds, block, a.gemm_grid);
    return;
  }
  const int slices = a.num_kv_heads / 4;
  const int wg = (block - a.gemm_grid) / slices, slice = (block - a.gemm_grid) - wg * slices;
  if (wg >= a.header[kHeaderStreamWgs]) return;  // graph plans' grids
  if (a.header[kHeaderOnce])                     // uniform
    stream_items<DT, 4, SETS, true>(a, lds, entries, wg, slice);
  else
    stream_items<DT, 4, SETS, false>(a, lds, entries, wg, slice);
}

// The same with whole CUs for either kind: products of 256 columns on some, copies of eight kv heads
// on the others and, when the products are done, on all.
template <int DT, int SETS>
__global__ __launch_bounds__(512, 2) void shared_wide_kernel(SharedArgs a) {
  constexpr int kRing = kStreamStages * 2 * kStreamTile * 8 * 256;
  static_assert(kRing == 4 * kStageBytes, "either ring");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kRing];
  __shared__ int32_t entries[kStreamEntries];
  if (a.num_kv_heads < 0) {
    lds[threadIdx.x] = 0;
    entries[threadIdx.x] = 0;
  }
  const int block = blockIdx.x;
  if (block < a.gemm_grid) {
    const int wgs = a.header[kHeaderGemmWgs];
    if (block < wgs) gemm_items<DT, 8>(a, lds, block, wgs);
    return;
  }
  const int slices = a.num_kv_heads / 8;
  const int wg = (block - a.gemm_grid) / slices, slice = (block - a.gemm_grid) - wg * slices;
  if (wg >= a.header[kHeaderStreamWgs]) return;
  if (a.header[kHeaderOnce])
    stream_items<DT, 8, SETS, true>(a, lds, entries, wg, slice);
  else
    stream_items<DT, 8, SETS, false>(a, lds, entries, wg, slice);
}

// One and two kv heads a slice: the launches follow each other.
template <int DT, int W, int SETS>
__global__ __launch_bounds__(64 * W, 2) void shared_stream_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t
      lds[kStreamStages * 2 * kStreamTile * W * 256];
  __shared__ int32_t entries[kStreamEntries];
  if (a.num_kv_heads < 0) {
    lds[threadIdx.x] = 0;
    entries[threadIdx.x] = 0;
  }
  const int slices = a.num_kv_heads / W;
  const int wg = blockIdx.x / slices, slice = blockIdx.x - wg * slices;
  if (wg >= a.header[kHeaderStreamWgs]) return;
  if (a.header[kHeaderOnce])
    stream_items<DT, W, SETS, true>(a, lds, entries, wg, slice);
  else
    stream_items<DT, W, SETS, false>(a, lds, entries, wg, slice);
}

template <int DT, int NW>
__global__ __launch_bounds__(64 * NW, 2) void shared_gemm_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NW / 2 * kStageBytes];
  if (a.num_kv_heads < 0) lds[threadIdx.x] = 0;
  gemm_items<DT, NW>(a, lds, blockIdx.x, gridDim.x);
}

// Running softmax join of partial outputs, four dims a thread.
struct Join {
  float mx = -INFINITY, den = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  template <int N>
  __device__ __forceinline__ void add(const float (&lse)[N], const float4 (&v)[N]) {
    float m_new = mx;
#pragma unroll
    for (int u = 0; u < N; ++u) m_new = fmaxf(m_new, lse[u]);
    const float ref = m_new == -INFINITY ? 0.f : m_new;  // nothing yet: every weight is 0
    const float corr = __builtin_amdgcn_exp2f(mx - ref);
    den *= corr;
    acc = make_float4(acc.x * corr, acc.y * corr, acc.z * corr, acc.w * corr);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float w = __builtin_amdgcn_exp2f(lse[u] - ref);
      den += w;
      acc = make_float4(fmaf(w, v[u].x, acc.x), fmaf(w, v[u].y, acc.y), fmaf(w, v[u].z, acc.z),
                        fmaf(w, v[u].w, acc.w));
    }
    mx = m_new;
  }
};

// 32 threads a row (a token's q head) and run of partials; RUNS threads groups share a row's partials
// and join through LDS. Bound by the rounds of loads, kUnroll partials each.
template <int DT, int RUNS>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs a) {
  constexpr int kUnroll = 8;
  constexpr int kRows = 8 / RUNS;  // rows of a workgroup
  const int f = threadIdx.x & 31;
  const int sub = threadIdx.x >> 5;
  const int run = sub % RUNS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub / RUNS;
  const bool in_range = row < a.rows;
  if (RUNS == 1 && !in_range) return;
  const int64_t at_row = in_range ? row : a.rows - 1;
  const int token = static_cast<int>(at_row / a.num_q_heads);
  const int qh = static_cast<int>(at_row - static_cast<int64_t>(token) * a.num_q_heads);
  const int req = a.row_of ? a.row_of[token] : token;
  Join j;
  const int4 parts[2] = {a.info[2 * req], a.info[2 * req + 1]};
  const bool joined = parts[0].y + parts[1].y > 0;  // else written directly
  if (RUNS == 1 && !joined) return;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int4 src = parts[part];  // {first slot, splits, tokens, token0}
    const int64_t first = static_cast<int64_t>(src.x + token - src.w) * a.num_q_heads + qh;
    const int64_t step = static_cast<int64_t>(src.z) * a.num_q_heads;
    for (int s0 = run * kUnroll; s0 < src.y; s0 += RUNS * kUnroll) {
      float lse[kUnroll];
      float4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t at = first + min(s0 + u, src.y - 1) * step;
        lse[u] = s0 + u < src.y ? a.part_lse[at] : -INFINITY;
        v[u] = *reinterpret_cast<const float4*>(a.part_o + at * kD + f * 4);
      }
      j.add(lse, v);
    }
  }
  if constexpr (RUNS > 1) {
    __shared__ float4 acc[8][32];
    __shared__ float2 stat[8];
    acc[sub][f] = j.acc;
    if (f == 0) stat[sub] = make_float2(j.mx, j.den);
    __syncthreads();
    if (run > 0 || !in_range || !joined) return;
    float mx = j.mx;
#pragma unroll
    for (int r = 1; r < RUNS; ++r) mx = fmaxf(mx, stat[sub + r].x);
    j.den = 0.f;
    j.acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
      const float2 st = stat[sub + r];
      const float w = st.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.x - mx);
      const float4 v = acc[sub + r][f];
      j.den = fmaf(w, st.y, j.den);
      j.acc = make_float4(fmaf(w, v.x, j.acc.x), fmaf(w, v.y, j.acc.y), fmaf(w, v.z, j.acc.z),
                          fmaf(w, v.w, j.acc.w));
    }
  }
  const float inv = 1.f / j.den;
  *reinterpret_cast<uint2*>(a.out + token * a.o_sn + qh * a.o_sh + f * 4) =
      make_uint2(Elem<DT>::pack2(j.acc.x * inv, j.acc.y * inv),
                 Elem<DT>::pack2(j.acc.z * inv, j.acc.w * inv));
}

// Up to this many rows a workgroup's threads all work on one: few rows have many parts, and leave
// most of the chip idle.
constexpr int64_t kMergeTogether = 512;

template <int DT>
void launch_merge(const SharedArgs& a, hipStream_t s) {
  if (a.rows <= kMergeTogether)
    shared_merge_kernel<DT, 8><<<dim3(static_cast<uint32_t>(a.rows)), dim3(256), 0, s>>>(a);
  else
    shared_merge_kernel<DT, 1><<<dim3(static_cast<uint32_t>((a.rows + 7) / 8)), dim3(256), 0, s>>>(
        a);
}

// ---------------------------------------------------------------------------
// Planning.
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The streaming launch for a kv-head count: the widest slice of whole rows that divides it.
struct StreamShape {
  int64_t waves, grid_y, workgroups, wg_capacity, max_item;
};
enum class Form {
  kInTurn,  // products, then copies
  kHalves,  // shared_kernel: half a CU for a workgroup of either kind (four kv heads a slice)
  kWhole,   // shared_wide_kernel: a CU for a workgroup of either kind (eight)
};

StreamShape stream_shape(int64_t cus, int64_t num_kv_heads, int64_t page_size, int64_t widest) {
  StreamShape s{};
  for (s.waves = widest; num_kv_heads % s.waves; s.waves /= 2) {
  }
  s.grid_y = num_kv_heads / s.waves;
  const int64_t lds = kStreamStages * 2 * kStreamTile * s.waves * 256 + kStreamEntries * 4;
  // eight waves of up to 256 registers on a CU
  const int64_t per_cu = std::max<int64_t>(1, std::min((160 * 1024) / lds, 8 / s.waves));
  s.workgroups = std::max<int64_t>(1, cus * per_cu / s.grid_y);
  s.wg_capacity = s.workgroups + s.workgroups / 3 + 2;  // schedule() tries more than it takes
  s.max_item = int64_t(kStreamEntries - 1) * page_size;
  return s;
}

// Query tokens against a range of keys: a group's against its prefix, or a request's own.
struct Source {
  int32_t token0, tokens, page_base, begin, end, pos0;
  int32_t slot = 0, splits = 0;
};


struct GemmCount {
  int64_t items = 0, slots = 0;
  int64_t longs = 0;    // items of at least half the longest part's tiles ...
  int64_t rest = 0;     // ... and what the others take, in tiles
};
constexpr int64_t kItemTiles = 2;  // an item besides its tiles: its queries, first tile, partial
GemmCount count_gemm(const std::vector<Source>& sources, int64_t group, int64_t num_kv_heads,
                     int64_t columns, int64_t length) {
  GemmCount n;
  for (const Source& s : sources) {
    const int64_t tiles = ceil_div(s.end, kTileK) - s.begin / kTileK;
    const int64_t splits = std::max<int64_t>(1, ceil_div(tiles, length));
    const int64_t items = ceil_div(s.tokens * group, columns) * num_kv_heads * splits;
    n.items += items;
    n.slots += s.tokens * splits;
    if (2 * tiles >= splits * length)
      n.longs += items;
    else
      n.rest += items * (ceil_div(tiles, splits) + kItemTiles);
  }
  return n;
}

// Tiles of a part's keys, such that the launch and its merge end soonest: rounds of long items over
// the chip, the short ones in what the last round leaves, and the partial outputs that are written and
// read again (`merge_tiles` a slot, in tiles of time).
struct GemmLength {
  int64_t tiles;
  double tile_times;  // until the last item has ended, in tiles
};
GemmLength gemm_length(const std::vector<Source>& sources, int64_t group, int64_t num_kv_heads,
                       int64_t columns, int64_t wgs, double merge_tiles, const GemmCount& cap) {
  int64_t longest = 1;
  for (const Source& s : sources)
    longest = std::max(longest, ceil_div(s.end, kTileK) - s.begin / kTileK);
  GemmLength best{longest, 0};
  double least = 0;
  for (int64_t parts = 1, last = 0; parts <= std::min<int64_t>(longest, 256);
       parts += 1 + parts / 8) {
    const int64_t l = ceil_div(longest, parts);
    if (l == last) continue;
    last = l;
    const GemmCount n = count_gemm(sources, group, num_kv_heads, columns, l);
    if (n.items > cap.items || n.slots > cap.slots) break;
    const int64_t rounds = ceil_div(n.longs, wgs);
    const int64_t idle = (rounds * wgs - n.longs) * (l + kItemTiles);
    const double run = static_cast<double>(rounds * (l + kItemTiles)) +
                       static_cast<double>(std::max<int64_t>(0, n.rest - idle)) / wgs;
    const double est = run + merge_tiles * n.slots;
    if (parts == 1 || est < least) {
      least = est;
      best = {l, run};
    }
  }
  return best;
}

// Appends the sources' work items, longest first; `slot`: the next free one.
void schedule_gemm(std::vector<Source>& sources, int64_t group, int64_t num_kv_heads,
                   int64_t columns, int64_t length, int64_t& slot, std::vector<int32_t>& work) {
  struct Item {
    int64_t tiles;
    int32_t source, row0, head, split, begin, end;
  };
  std::vector<Item> items;
  for (size_t i = 0; i < sources.size(); ++i) {
    Source& s = sources[i];
    const int64_t rows = s.tokens * group;
    const int64_t first = s.begin / kTileK, tiles = ceil_div(s.end, kTileK) - first;
    s.splits = static_cast<int32_t>(std::max<int64_t>(1, ceil_div(tiles, length)));
    s.slot = static_cast<int32_t>(slot);
    slot += static_cast<int64_t>(s.splits) * s.tokens;
    for (int32_t p = 0; p < s.splits; ++p)
      for (int64_t row0 = 0; row0 < rows; row0 += columns) {
        const int64_t begin = first + tiles * p / s.splits;
        int64_t end = first + tiles * (p + 1) / s.splits;
        if (s.pos0 < kNoHorizon) {  // no tile past what the item's last row sees
          const int64_t last = s.pos0 + (std::min<int64_t>(row0 + columns, rows) - 1) / group;
          end = std::max<int64_t>(begin, std::min<int64_t>(end, last / kTileK + 1));
        }
        for (int32_t h = 0; h < num_kv_heads; ++h)
          items.push_back({end - begin, static_cast<int32_t>(i), static_cast<int32_t>(row0), h, p,
                           static_cast<int32_t>(begin), static_cast<int32_t>(end)});
      }
  }
  // Heads stay fastest, so that with 8 of them a head's items, which read the same keys, meet in the
  // L2 of one XCD.
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& x, const Item& y) { return x.tiles > y.tiles; });
  work.reserve(items.size() * kGemmInts);
  for (const Item& it : items) {
    const Source& s = sources[it.source];
    work.insert(work.end(), {s.token0, static_cast<int32_t>(s.tokens * group), it.row0, it.head,
                             s.page_base, it.begin, it.end, s.slot + it.split * s.tokens, s.pos0,
                             s.end, 0, 0});
  }
}

}  // namespace

const char* check_groups(const int32_t* group_rows, const int32_t* group_lens, int64_t groups,
                         int64_t batch, const int32_t* cached, const char* too_long) {
  int64_t row = 0;
  for (int64_t g = 0; g < groups; ++g) {
    if (group_rows[g] <= 0 || group_lens[g] < 0 || group_rows[g] > batch - row)
      return "invalid shared prefix groups";
    for (const int64_t end = row + group_rows[g]; row < end; ++row)
      if (group_lens[g] > cached[row]) return too_long;
  }
  return row == batch ? nullptr : "invalid shared prefix groups";
}

namespace {
// MI355X_SHARED_FROM (bytes) overrides from when on prefixes are shared: least_saved(), the shortest
// prefix, kOneSliceOwn and the comparison with the plain kernels' time (tuning knob, read for every plan).
bool forced() { return std::getenv("MI355X_SHARED_FROM") != nullptr; }
// Bytes of K and V that sharing has to save a layer: less is lost again on the products' launch and
// the merge. us a layer, plain against shared (32 heads, 8 kv heads): 2 rows of 1,024 tokens (4 MB)
// 11.7, 13.2; 8 of 256 (7 MB) 13.5, 13.1; 4 of 1,024 (12 MB) 13.4, 13.3; 16 of 1,024 (60 MB) 16.2,
// 14.3; 256 of 1,024 117, 33. With fewer kv heads than a slice has the plain kernel is the slower one
// throughout (one kv head: 22, 13).
int64_t least_saved(int64_t num_kv_heads) {
  if (forced()) return std::strtoll(std::getenv("MI355X_SHARED_FROM"), nullptr, 10);
  return num_kv_heads % 4 ? 0 : int64_t(num_kv_heads == 4 ? 16 : 8) << 20;
}
// Four kv heads are one slice on halves of CUs, which streams rows' own keys at 5.2 TB/s where the plain
// kernel reaches 5.9: there the prefix has to save a third of what the rows read of their own, and twice the
// bytes (us, 48 rows, 32 heads: 256 shared tokens and 3,000 own 56.4, 63.7; 512 63.1, 67.4; 1,024 69.9, 67.7;
// 12 rows, 1,024 and 3,000 23.7, 27.3, 512 and 64 10.2, 11.2; 1,500 and 1,500 20.2, 18.5).
constexpr int64_t kOneSliceOwn = 3;
// Prefixes of 64 tokens are not worth it in any batch (256 rows: 24.4 us plain, 30.5 shared).
int32_t shortest_prefix() { return forced() ? kTileK : 2 * kTileK; }
// Most bytes of partial outputs of a batch: the workspace stands beside the caller's memory and is kept.
// A token takes 516 bytes a q head and part, at least two parts: 4 GiB are some 40,000 new tokens of 64
// heads, without a limit a batch could ask for more than 64 GiB. MI355X_SHARED_MOST overrides it (tuning
// knob, read for every plan).
int64_t most_partials() {
  if (const char* env = std::getenv("MI355X_SHARED_MOST")) return std::strtoll(env, nullptr, 10);
  return int64_t(4) << 30;
}
}  // namespace

struct SharedPlan::State {
  int64_t cus, num_q_heads, num_kv_heads, page_size, dtype, group;
  int group_log2 = 0;
  StreamShape shape{};
  // Current plan.
  int64_t batch = 0, tokens = 0;
  bool ready = false;
  bool by_token = false;  // requests of one token each
  int64_t stream_grid = 0, gemm_grid = 0, gemm_items = 0, gemm_wgs = 0;
  int sets = 1, nw = 4;
  Form form = Form::kInTurn;
  int64_t slices = 1;  // kv-head slices of the streaming launch
  int64_t groups_shared = 0, tokens_shared = 0, prefix_items = 0;
  int64_t o_info = 0, o_row_of = 0, o_stream = 0, o_wg = 0, o_gemm = 0;
  // What prepare() has decided, for upload() to lay out.
  struct Of {
    int32_t kind, index;  // 0 none, 1 of stream, 2 of gemm
  };
  struct Draft {
    std::vector<Source> stream, gemm;  // own and prefix sources of either kernel
    std::vector<Of> prefix_of, own_of;
    std::vector<int32_t> work, wg;     // the streaming schedule's
    int64_t items = 0, wgs = 0, slot = 0, columns = 0, tiles = 0;
    bool once = true;
  } draft;
  Buffer ints, staging, part_o, part_lse;
  hipEvent_t upload_done = nullptr;

  ~State() {
    if (upload_done) {
      (void)hipEventSynchronize(upload_done);
      (void)hipEventDestroy(upload_done);
    }
  }

  // Whole tiles of each group's prefix that leave every request its own tokens; 0 for groups of one.
  std::vector<int32_t> lengths(const SharedBatch& b) const {
    std::vector<int32_t> eff(b.groups, 0);
    int64_t row = 0;
    for (int64_t g = 0; g < b.groups; ++g) {
      int64_t len = std::min<int64_t>(b.group_lens[g], kMaxKeys - kTileK);
      for (int64_t r = row; r < row + b.group_rows[g]; ++r)
        len = std::min<int64_t>(len, b.kv_len[r] - (b.q_start[r + 1] - b.q_start[r]));
      if (b.group_rows[g] > 1 && len >= shortest_prefix())
        eff[g] = static_cast<int32_t>(len / kTileK * kTileK);
      row += b.group_rows[g];
    }
    return eff;
  }
};

SharedPlan::SharedPlan(int64_t cus, int64_t num_q_heads, int64_t num_kv_heads, int64_t page_size,
                       int64_t dtype)
    : st_(new State{cus, num_q_heads, num_kv_heads, page_size, dtype,
                    num_q_heads / num_kv_heads}) {
  while ((1 << st_->group_log2) < st_->group) ++st_->group_log2;
  st_->shape = stream_shape(cus, num_kv_heads, page_size, 4);
  st_->staging.pinned = true;
}
SharedPlan::~SharedPlan() = default;

bool SharedPlan::pays(const SharedBatch& b) const {
  const std::vector<int32_t> eff = st_->lengths(b);
  int64_t saved = 0, own = 0;
  bool any = false;
  // The merge takes 32 threads a row of a q head, and a grid of 2^32 would be cut short.
  if (int64_t(b.q_start[b.batch]) * st_->num_q_heads >= int64_t(1) << 26) return false;
  for (int64_t g = 0, row = 0; g < b.groups; ++g) {
    saved += int64_t(b.group_rows[g] - 1) * eff[g];
    any |= eff[g] > 0;
    for (const int64_t end = row + b.group_rows[g]; row < end; ++row) own += b.kv_len[row] - eff[g];
  }
  const int64_t heads = st_->num_kv_heads;
  if (!any || saved * heads * kD * 4 < least_saved(heads)) return false;
  return forced() || heads != 4 || kOneSliceOwn * saved >= own;
}

SharedFit SharedPlan::prepare(const SharedBatch& b, int64_t graph_rows, int64_t graph_tokens,
                              uint64_t& allocations) {
  State& st = *st_;
  st.ready = false;
  const int64_t group = st.group, heads = st.num_kv_heads;
  const int64_t tokens = b.q_start[b.batch];
  const std::vector<int32_t> eff = st.lengths(b);
  using Of = State::Of;
  st.draft = {};
  std::vector<Source>&stream = st.draft.stream, &gemm = st.draft.gemm;
  std::vector<Of>&prefix_of = st.draft.prefix_of, &own_of = st.draft.own_of;
  std::vector<int32_t>&work = st.draft.work, &wg = st.draft.wg;
  int64_t &items = st.draft.items, &wgs = st.draft.wgs, &slot = st.draft.slot;
  std::vector<int32_t> lens, merge;
  GemmCount cap;
  int64_t items_cap = 0;
  prefix_of.assign(b.batch, Of{0, 0});
  own_of.assign(b.batch, Of{0, 0});
  st.groups_shared = st.tokens_shared = 0;
  for (int64_t r = 0, g = 0, left = 0, before = 0; r < b.batch; ++r) {
    if (left == 0 && g < b.groups) {  // a group begins
      left = b.group_rows[g];
      before = eff[g];
      ++g;
      if (before > 0) {
        ++st.groups_shared;
        st.tokens_shared += before;
        const int64_t all = b.q_start[r + left] - b.q_start[r];
        const Source src{b.q_start[r], static_cast<int32_t>(all), b.page_base[r], 0,
                         static_cast<int32_t>(before), kNoHorizon};
        if (all * group <= kStreamColumns) {
          for (int64_t i = r; i < r + left; ++i)
            prefix_of[i] = {1, static_cast<int32_t>(stream.size())};
          stream.push_back(src);
        } else {
          for (int64_t i = r; i < r + left; ++i)
            prefix_of[i] = {2, static_cast<int32_t>(gemm.size())};
          gemm.push_back(src);
        }
      }
    }
    const int32_t t = b.q_start[r + 1] - b.q_start[r];
    const Source own{b.q_start[r], t, b.page_base[r], static_cast<int32_t>(left ? before : 0),
                     b.kv_len[r], b.kv_len[r] - t};
    if (left) --left;
    if (t * group <= kStreamColumns) {
      own_of[r] = {1, static_cast<int32_t>(stream.size())};
      stream.push_back(own);
    } else {
      own_of[r] = {2, static_cast<int32_t>(gemm.size())};
      gemm.push_back(own);
    }
  }
  int64_t bytes = 0;
  for (const Source& src : stream) bytes += int64_t(src.end - src.begin) * heads * kD * 4;
  // A CU's tile of 256 columns while others stream, and the copies' rate on the whole chip.
  constexpr double kTileUs = 1.68, kBytesPerUs = 5.86e6;
  // A tile of 128 columns while the CU does another, and what a plan costs beside its loops, more where
  // it has both.
  constexpr double kNarrowTileUs = 1.28, kLaunchesUs = 8, kBothUs = 5;
  double stream_us = static_cast<double>(bytes) / kBytesPerUs;
  // A few requests with little of their own take products too: not half a CU's worth of items and no
  // launch that would wait for the others' (48 rows of up to 40 new tokens behind 4,096, two layers 226
  // us, 213; 20 of up to 100 211, 198; 30 of up to 14, where the items are at this bound, 84.4, 85.2).
  if (!graph_rows && !gemm.empty() && stream_us <= 1 &&
      2 * static_cast<int64_t>(stream.size()) * heads <= st.cus &&
      std::none_of(stream.begin(), stream.end(),
                   [](const Source& src) { return src.end > kMaxKeys; })) {
    for (std::vector<Of>* ofs : {&prefix_of, &own_of})
      for (Of& of : *ofs)
        if (of.kind == 1) of = {2, of.index + static_cast<int32_t>(gemm.size())};
    gemm.insert(gemm.end(), stream.begin(), stream.end());
    stream.clear();
    bytes = 0;
    stream_us = 0;
  }
  // How the products and the copies share the chip. Whole CUs for either wherever there are both and
  // eight kv heads (us a layer, in turn, in halves, on whole CUs: 256 rows sharing 8,192 tokens 142,
  // 137, 125; 64 sharing 2,048 43, 36, 30; 75 rows of up to 16 new tokens in 8 groups 65, 63, 54);
  // halves with four; in turn where the copies are next to nothing (48 rows of up to 40 new tokens
  // 103, 141, 110).
  int64_t cost4 = 0, cost8 = 0;  // tiles of 128 and of 256 columns
  for (const Source& src : gemm) {
    const int64_t tiles = ceil_div(src.end, kTileK) - src.begin / kTileK;
    cost4 += ceil_div(src.tokens * group, 128) * tiles * heads;
    cost8 += ceil_div(src.tokens * group, 256) * tiles * heads;
  }
  st.form = st.shape.waves == 4 && !stream.empty() ? Form::kHalves : Form::kInTurn;
  if (heads % 8 == 0 && (graph_rows ? graph_rows * group > 128
                                    : !gemm.empty() && stream_us > 1))
    st.form = Form::kWhole;
  else if (!graph_rows && !gemm.empty() && stream_us <= 1)
    st.form = Form::kInTurn;
  // Fixed for a graph plan, whose captured launch holds one of the two.
  const bool filled = !graph_rows && st.form == Form::kInTurn && 4 * cost8 <= 3 * cost4;
  st.nw = st.form == Form::kWhole || filled ? 8 : 4;
  const int64_t columns = 32 * st.nw;
  // Bounds on the products' items and partial outputs, beside one part a source: a graph plan's
  // hold for whatever its rows will share.
  const int64_t extra = graph_rows ? st.cus : 2 * st.cus, per = columns / group;  // tokens of an item
  if (graph_rows) {
    // at most rows / 2 groups share, each with a last tile that is not full
    cap.items = (graph_rows / per + graph_rows / 2) * heads + extra;
    cap.slots = graph_rows + extra * per / heads;
  } else {
    cap = count_gemm(gemm, group, heads, columns, std::numeric_limits<int32_t>::max());
    cap.items += extra;
    cap.slots += extra * per;
  }
  // A slot's partial outputs, written and read at about 5 TB/s.
  const double merge_tiles = static_cast<double>(st.num_q_heads * 1056) / 5e6 / kTileUs;
  StreamShape shape = st.shape;
  int64_t gemm_wgs = st.form == Form::kHalves || st.nw == 8 ? st.cus : 2 * st.cus;
  if (st.form == Form::kWhole) {
    // As many CUs for the products as end the launch soonest. A CU streams no faster for others'
    // not streaming: the copies take longer by the products' share.
    double least = std::numeric_limits<double>::infinity();
    gemm_wgs = 0;
    for (int64_t wgs8 = std::max<int64_t>(1, st.cus / 16);
         wgs8 <= st.cus - st.cus / 8 && !gemm.empty();
         wgs8 += std::max<int64_t>({1, st.cus / 32, wgs8 / 8})) {
      const double run =
          kTileUs * gemm_length(gemm, group, heads, columns, wgs8, merge_tiles, cap).tile_times;
      const double est =
          std::max(run, stream_us * static_cast<double>(st.cus) / (st.cus - wgs8));
      if (est < least) {
        least = est;
        gemm_wgs = wgs8;
      }
    }
    // A share for every CU that streams: more of them end later where the last ones find no CU free
    // (64 rows sharing 8,192 tokens, 154 such CUs: 154 shares 35 us, 192 46, 224 41, 256 39).
    shape = stream_shape(st.cus, heads, st.page_size, 8);
    shape.workgroups = std::max<int64_t>(1, (st.cus - gemm_wgs) / shape.grid_y);
    shape.wg_capacity = st.cus / shape.grid_y + st.cus / 3 + 2;
  }
  // The streaming launch.
  items_cap = shape.wg_capacity;
  int widest = 1;
  for (const Source& src : stream) {
    lens.push_back(src.end - src.begin);
    items_cap += 1 + ceil_div(lens.back(), shape.max_item);
    widest = std::max<int>(widest, src.tokens * static_cast<int>(group));
  }
  st.draft.once = bytes >= int64_t(8) << 20;  // as the decode kernel's copies
  st.sets = widest <= 16 ? 1 : 2;
  work.resize(4 * items_cap);
  merge.resize(2 * stream.size());
  wg.resize(shape.wg_capacity + 1);
  int64_t share = 0;
  if (!stream.empty()) {
    items = schedule(lens.data(), static_cast<int64_t>(stream.size()), shape.workgroups,
                     shape.max_item, kStreamTile, /*graph=*/true, work.data(), items_cap,
                     merge.data(), &share, wg.data(), shape.wg_capacity, &wgs);
    if (items < 0) {
      set_error("shared prefix work list exceeds its capacity");
      return SharedFit::kError;
    }
  }
  // Items of a source are consecutive: its slots follow each other.
  std::vector<bool> joined(stream.size(), true);
  for (int64_t r = 0; r < b.batch; ++r)
    if (own_of[r].kind == 1 && prefix_of[r].kind == 0)
      joined[own_of[r].index] = merge[2 * own_of[r].index + 1] > 1;
  for (size_t i = 0; i < stream.size(); ++i) {
    Source& src = stream[i];
    src.splits = joined[i] ? merge[2 * i + 1] : 0;
    src.slot = static_cast<int32_t>(slot);
    slot += static_cast<int64_t>(src.splits) * src.tokens;
  }
  // The matrix products.
  GemmLength length{};
  GemmCount products;
  if (!gemm.empty()) {
    length = gemm_length(gemm, group, heads, columns, gemm_wgs, merge_tiles, cap);
    products = count_gemm(gemm, group, heads, columns, length.tiles);
  }
  const int64_t slots = slot + products.slots;
  if (!graph_rows && !forced()) {
    // Against the plain kernels' time: the launches, products and copies as above (they take an eighth
    // longer than their loops alone), partial outputs written and read.
    const double products_us = (st.nw == 8 ? kTileUs : kNarrowTileUs) * length.tile_times;
    if (st.form == Form::kWhole) stream_us *= static_cast<double>(st.cus) / (st.cus - gemm_wgs);
    const double both = st.form == Form::kInTurn ? products_us + stream_us
                                                 : std::max(products_us, stream_us);
    const double partials_us = static_cast<double>(slots * st.num_q_heads * 1056) / 5e6;
    const double beside_us = kLaunchesUs + (stream.empty() || gemm.empty() ? 0 : kBothUs);
    if (beside_us + 1.12 * both + partials_us >= b.plain_us) return SharedFit::kPlain;
  }
  st.draft.columns = columns;
  st.draft.tiles = length.tiles;
  st.slices = shape.grid_y;
  st.gemm_wgs = std::min(gemm_wgs, products.items);
  st.gemm_items = products.items;

  // Layout; a graph plan's does not depend on what is shared.
  st.by_token = tokens == b.batch;
  int64_t stream_cap = items, wg_cap = wgs, gemm_cap = st.gemm_items, slot_cap = slots;
  if (graph_rows) {
    // A workgroup's share, and each request's and prefix's own items and cuts; a slot an item of a
    // request, and as many as a streamed prefix has tokens an item of one.
    const int64_t cuts = 1 + ceil_div(graph_tokens, shape.max_item);
    stream_cap = shape.wg_capacity + (graph_rows + graph_rows / 2) * cuts;
    wg_cap = shape.wg_capacity;
    gemm_cap = cap.items;
    slot_cap = stream_cap + cap.slots +
               (shape.wg_capacity + graph_rows / 2 * cuts) *
                   std::min<int64_t>(kStreamColumns / group, graph_rows);
  }
  st.o_info = kHeaderInts;
  st.o_row_of = st.o_info + kInfoInts * b.batch;
  st.o_stream = st.o_row_of + (st.by_token ? 0 : ceil_div(tokens, 4) * 4);
  st.o_gemm = st.o_stream + kStreamInts * stream_cap;
  st.o_wg = st.o_gemm + kGemmInts * gemm_cap;
  const int64_t total = st.o_wg + wg_cap + 1;
  const size_t rows = static_cast<size_t>(slot_cap) * st.num_q_heads;
  if (!graph_rows && static_cast<int64_t>(rows * (kD + 1) * 4) > most_partials())
    return SharedFit::kPlain;
  hipError_t err = hipSuccess;
  if (!st.upload_done) err = hipEventCreateWithFlags(&st.upload_done, hipEventDisableTiming);
  if (err == hipSuccess) err = hipEventSynchronize(st.upload_done);  // staging is free
  const bool grows = total * 4 > static_cast<int64_t>(st.ints.capacity) ||
                     rows * kD * 4 > st.part_o.capacity || rows * 4 > st.part_lse.capacity;
  if (graph_rows && st.batch && grows) {
    set_error("graph decode metadata capacity exceeded");
    return SharedFit::kError;
  }
  if (err == hipSuccess) err = st.ints.reserve(total * 4, allocations);
  if (err == hipSuccess) err = st.staging.reserve(total * 4, allocations);
  if (err == hipSuccess) err = st.part_o.reserve(rows * kD * 4, allocations);
  if (err == hipSuccess) err = st.part_lse.reserve(rows * 4, allocations);
  if (err == hipErrorOutOfMemory && !graph_rows) return SharedFit::kPlain;
  if (err != hipSuccess) {
    hip_error(err, "shared prefix workspace");
    return SharedFit::kError;
  }
  st.tokens = tokens;
  if (graph_rows) st.sets = 2;
  st.stream_grid = graph_rows ? wg_cap : wgs;
  st.gemm_grid = graph_rows ? st.cus : st.gemm_wgs;
  return SharedFit::kRuns;
}

bool SharedPlan::upload(const SharedBatch& b, hipStream_t s) {
  State& st = *st_;
  State::Draft& d = st.draft;
  std::vector<int32_t> gemm_work;
  schedule_gemm(d.gemm, st.group, st.num_kv_heads, d.columns, d.tiles, d.slot, gemm_work);
  int32_t* host = static_cast<int32_t*>(st.staging.ptr);
  host[kHeaderGemmItems] = static_cast<int32_t>(st.gemm_items);
  host[kHeaderStreamWgs] = static_cast<int32_t>(d.wgs);
  host[kHeaderOnce] = d.once;
  host[kHeaderGemmWgs] = static_cast<int32_t>(st.gemm_wgs);
  for (int64_t r = 0; r < b.batch; ++r) {
    int32_t* info = host + st.o_info + kInfoInts * r;
    for (const State::Of& of : {d.prefix_of[r], d.own_of[r]}) {
      const Source* src = of.kind == 0 ? nullptr : of.kind == 1 ? &d.stream[of.index]
                                                                : &d.gemm[of.index];
      info[0] = src ? src->slot : 0;
      info[1] = src ? src->splits : 0;
      info[2] = src ? src->tokens : 0;
      info[3] = src ? src->token0 : 0;
      info += 4;
    }
    if (!st.by_token)
      std::fill(host + st.o_row_of + b.q_start[r], host + st.o_row_of + b.q_start[r + 1],
                static_cast<int32_t>(r));
  }
  st.prefix_items = 0;
  for (size_t i = 0; i < gemm_work.size(); i += kGemmInts)
    st.prefix_items += gemm_work[i + 8] == kNoHorizon;
  for (int64_t i = 0, part = 0; i < d.items; ++i) {
    const int32_t of = d.work[4 * i];
    part = i && d.work[4 * (i - 1)] == of ? part + 1 : 0;
    const Source& src = d.stream[of];
    const int32_t begin = src.begin + d.work[4 * i + 1], end = src.begin + d.work[4 * i + 2];
    const int32_t out[kStreamInts] = {
        src.token0, src.tokens,
        src.page_base + begin / static_cast<int32_t>(st.page_size), begin, end,
        src.splits ? src.slot + static_cast<int32_t>(part) * src.tokens : -1, src.pos0, 0};
    std::memcpy(host + st.o_stream + kStreamInts * i, out, sizeof out);
    st.prefix_items += src.pos0 == kNoHorizon;
  }
  std::copy(d.wg.begin(), d.wg.begin() + (d.stream.empty() ? 0 : d.wgs + 1), host + st.o_wg);
  std::copy(gemm_work.begin(), gemm_work.end(), host + st.o_gemm);
  // wg comes last and only its used part is written: a graph plan's unused workgroups leave early.
  hipError_t err =
      hipMemcpyAsync(st.ints.ptr, host, (st.o_wg + d.wgs + 1) * 4, hipMemcpyHostToDevice, s);
  if (err == hipSuccess) err = hipEventRecord(st.upload_done, s);
  if (err != hipSuccess) {
    hip_error(err, "shared prefix upload");
    return false;
  }
  st.ready = true;
  st.batch = b.batch;
  return true;
}

void SharedPlan::info(int64_t* out4) const {
  out4[0] = st_->groups_shared;
  out4[1] = st_->tokens_shared;
  out4[2] = st_->prefix_items;
  out4[3] = st_->gemm_items;
}

namespace {
template <int DT, int W>
void launch_stream(const SharedArgs& a, int sets, uint32_t grid, hipStream_t s) {
  if (sets == 1) shared_stream_kernel<DT, W, 1><<<dim3(grid), dim3(64 * W), 0, s>>>(a);
  else shared_stream_kernel<DT, W, 2><<<dim3(grid), dim3(64 * W), 0, s>>>(a);
}
template <int DT>
const char* launch_all(SharedArgs a, Form form, int64_t waves, int sets, int nw,
                       int64_t stream_grid, hipStream_t s) {
  const uint32_t streams = static_cast<uint32_t>(stream_grid);
  const uint32_t products = static_cast<uint32_t>(a.gemm_grid);
  if (form == Form::kInTurn) {
    if (products) {
      if (nw == 8) shared_gemm_kernel<DT, 8><<<dim3(products), dim3(512), 0, s>>>(a);
      else shared_gemm_kernel<DT, 4><<<dim3(products), dim3(256), 0, s>>>(a);
      if (const char* err = launch_status("shared_gemm_kernel")) return err;
    }
    a.gemm_grid = 0;
    if (streams) {
      if (waves == 2) launch_stream<DT, 2>(a, sets, streams, s);
      else if (waves == 1) launch_stream<DT, 1>(a, sets, streams, s);
      else if (sets == 1) shared_kernel<DT, 1><<<dim3(streams), dim3(256), 0, s>>>(a);
      else shared_kernel<DT, 2><<<dim3(streams), dim3(256), 0, s>>>(a);
      if (const char* err = launch_status("shared_stream_kernel")) return err;
    }
  } else {
    const dim3 grid(products + streams);
    if (form == Form::kWhole) {
      if (sets == 1) shared_wide_kernel<DT, 1><<<grid, dim3(512), 0, s>>>(a);
      else shared_wide_kernel<DT, 2><<<grid, dim3(512), 0, s>>>(a);
    } else {
      if (sets == 1) shared_kernel<DT, 1><<<grid, dim3(256), 0, s>>>(a);
      else shared_kernel<DT, 2><<<grid, dim3(256), 0, s>>>(a);
    }
    if (const char* err = launch_status("shared_kernel")) return err;
  }
  launch_merge<DT>(a, s);
  return launch_status("shared_merge_kernel");
}
}  // namespace

const char* SharedPlan::run(const int32_t* indices, const void* q, int64_t q_sn, int64_t q_sh,
                            const void* k, const void* v, void* out, int64_t o_sn, int64_t o_sh,
                            hipStream_t s) const {
  const State& st = *st_;
  if (!st.ready) return set_error("shared prefixes were not prepared");
  const int32_t* ints = static_cast<const int32_t*>(st.ints.ptr);
  SharedArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sn = q_sn;
  a.q_sh = q_sh;
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.o_sn = o_sn;
  a.o_sh = o_sh;
  a.header = ints;
  a.info = reinterpret_cast<const int4*>(ints + st.o_info);
  a.row_of = st.by_token ? nullptr : ints + st.o_row_of;
  a.stream_work = reinterpret_cast<const int4*>(ints + st.o_stream);
  a.stream_wg = ints + st.o_wg;
  a.gemm_work = reinterpret_cast<const int4*>(ints + st.o_gemm);
  a.indices = indices;
  a.part_o = static_cast<float*>(st.part_o.ptr);
  a.part_lse = static_cast<float*>(st.part_lse.ptr);
  a.rows = st.tokens * st.num_q_heads;
  a.num_q_heads = static_cast<int32_t>(st.num_q_heads);
  a.num_kv_heads = static_cast<int32_t>(st.num_kv_heads);
  a.group_log2 = st.group_log2;
  a.page_size = static_cast<int32_t>(st.page_size);
  a.scale_log2 = (1.0f / std::sqrt(static_cast<float>(kD))) * kLog2e;
  a.slack = st.by_token ? kDecodeSlack : kExtendSlack;
  a.gemm_grid = static_cast<int32_t>(st.gemm_grid);
  const int64_t stream_grid = st.stream_grid * st.slices;
  return st.dtype == 0
             ? launch_all<0>(a, st.form, st.shape.waves, st.sets, st.nw, stream_grid, s)
             : launch_all<1>(a, st.form, st.shape.waves, st.sets, st.nw, stream_grid, s);
}

}  // namespace mi355x
