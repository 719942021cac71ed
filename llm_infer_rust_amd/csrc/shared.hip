// Attention over a prefix that several requests share, computed once for all of them, and the merge
// with what each has of its own. No counterpart in the reference, whose backends read every
// request's whole cache (src/models/attention/backend.rs:316-804).
//
//   o = (2^a o_p + 2^b o_s) / (2^a + 2^b),  (o_p, a) and (o_s, b) the normalised outputs and log2 of
//   the sums of 2^score over the prefix and over the request's own keys.
//
// A group's queries (every token's G heads under a kv head, heads fastest: tokens x G rows) meet the
// prefix's keys as one matrix product, so K and V are read once a group (and once for every 256
// rows) where plain decode reads them once a request. One workgroup = 32 rows a wave against a
// range of 64-key tiles, as the prefill kernel: S^T = K Q^T, P^T = 2^(S^T - m), O^T += V^T P^T on
// 32 x 32 x 16 products, K and V tiles through an LDS ring by direct copies. Ranges are cut so that
// the items fill the chip; each writes an fp32 partial and its log2-sum-exp, joined by one more
// launch together with the own parts: decode's split-KV partials, or (several new tokens a request)
// items of the same kernel, with a horizon.
#include <algorithm>
#include <cmath>
#include <limits>

#include "mfma.h"
#include "shared.h"

namespace mi355x {
namespace {

constexpr int kD = 128;
constexpr int kTileK = kSharedTile;
constexpr int kTileBytes = kTileK * kD * 2;
constexpr int kStageBytes = 2 * kTileBytes;  // K + V

// K and V tiles lie in LDS as the prefill kernel's do: [key][d], 16-byte chunk c of key r at
// c ^ (r & 15) (K) and c ^ 4 (r & 3) (V), which keeps the operand reads free of bank conflicts.
template <int DT, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 1 : 2) void shared_kernel(SharedArgs a) {
  constexpr int kStages = NW == 8 ? 4 : 2;
  constexpr int kAhead = kStages - 1;
  constexpr int kGroupsPerWave = 16 / NW;  // 4-row groups of each tile this wave copies
  constexpr int kCopiesPerTile = 2 * kGroupsPerWave;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * kStageBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 31;
  const int half = lane >> 5;
  // The copies are invisible to the compiler: one store it sees, never taken.
  if (a.num_kv_heads < 0) lds[threadIdx.x] = 0;
  const uint32_t lds_base = lds_address(lds);
  const int64_t slot_stride = static_cast<int64_t>(a.num_kv_heads) * kD;
  const float inv_page = 1.0f / static_cast<float>(a.page_size);
  const bool fast_pages =
      a.page_size >= 4 && a.page_size <= kTileK && kTileK % a.page_size == 0;
  const int pages_per_tile = fast_pages ? kTileK / a.page_size : 0;
  const float c = a.scale_log2;
  const float lazy_limit = 8.f / c;  // 2^8 in p

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

  const int items = a.header[0];
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int4 w0 = a.work[3 * item], w1 = a.work[3 * item + 1], w2 = a.work[3 * item + 2];
    const int token0 = w0.x, rows = w0.y, row0 = w0.z, kvh = w0.w;
    const int page_base = w1.x, t_begin = w1.y, nt = w1.z - w1.y, record = w1.w;
    const int pos0 = w2.x, kv_len = w2.y;
    const int my_row0 = row0 + wave * 32;
    const bool wave_active = my_row0 < rows;
    const int my_row = min(my_row0 + col, rows - 1);
    const int token = my_row / a.group;
    const int qh = kvh * a.group + (my_row - token * a.group);
    const int horizon = pos0 + token;  // the last key this row sees
    const int first_horizon = pos0 + my_row0 / a.group;
    const int last_horizon = pos0 + min(my_row0 + 31, rows - 1) / a.group;

    uint4 qreg[8];
    {
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
        const int64_t slot = static_cast<int64_t>(page) * a.page_size + off;
        copy_to_lds(k_head + slot * slot_stride + (pos ^ (row & 15)) * 8, sbase + g * 1024);
        copy_to_lds(v_head + slot * slot_stride + (pos ^ (4 * (row & 3))) * 8,
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
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    // m: this lane's reference of the raw scores; the accumulators start at -m, p = 2^(c (s - m)).
    float m = 0.f, l = 0.f;
    floatx16 negm;
#pragma unroll
    for (int r = 0; r < 16; ++r) negm[r] = 0.f;

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
      for (int kk = 0; kk < 8; ++kk)
#pragma unroll
        for (int T = 0; T < 2; ++T)
          s[T] = Mfma<DT>::run(kf[T][kk], qreg[kk], kk == 0 ? negm : s[T]);
      uint4 vf[4][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          lds_u8* vp = (lds_u8*)sb + v_off[db] + 16 * kk * 256;
          const uint2 l2 =
              __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)vp));
          const uint2 h2 = __builtin_bit_cast(
              uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vp + 8 * 256)));
          vf[kk][db] = make_uint4(l2.x, l2.y, h2.x, h2.y);
        }
      if (k0 + kTileK - 1 > first_horizon || k0 + kTileK > kv_len) {
        const int limit = min(horizon, kv_len - 1) - (k0 + 4 * half);
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
        mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      }
      // m moves on the first tile and then only when a row's maximum passes it by 8 / c. A first
      // tile wholly past a row's horizon (mx = -inf) leaves m at 0.
      if (first || __any(mx > lazy_limit)) {
        const float shift = first ? (mx == -INFINITY ? 0.f : mx) : fmaxf(mx, 0.f);
        const float alpha = first ? 1.f : __builtin_amdgcn_exp2f(-shift * c);
        m += shift;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[0][r] -= shift;
          s[1][r] -= shift;
          negm[r] = -m;
        }
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
            p[i] = __builtin_amdgcn_exp2f(s[T][8 * hh + i] * c);
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
        for (int db = 0; db < 4; ++db) o[db] = Mfma<DT>::run(vf[kk][db], pb[kk], o[db]);
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

    if (wave_active && my_row0 + col < rows) {
      const float row_sum = l + __shfl_xor(l, 32);
      const float inv = row_sum > 0.f ? 1.f / row_sum : 0.f;
      const int64_t rec = record + wave;
      float* po = a.part_o + rec * kSharedRecord;
      // Lanes' own order (float4 (4 db + g4) * 64 + lane): whole lines for a wave's rows.
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
          *reinterpret_cast<float4*>(po + ((4 * db + g4) * 64 + lane) * 4) =
              make_float4(o[db][4 * g4] * inv, o[db][4 * g4 + 1] * inv, o[db][4 * g4 + 2] * inv,
                          o[db][4 * g4 + 3] * inv);
      if (half == 0)
        a.part_lse[rec * 32 + col] =
            row_sum > 0.f ? m * c + __builtin_amdgcn_logf(row_sum)
                          : row_sum == 0.f ? -INFINITY : row_sum;  // NaN stays
    }
    __syncthreads();  // the next item's copies overwrite the ring
  }
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

// 32 threads a row (a token's q head), eight rows a workgroup: dims 4 f .. 4 f + 3 of a row sit in
// float4 (f / 2) * 64 + row % 32 + 32 (f % 2) of a record. Bound by the rounds of loads, kUnroll
// partials each.
template <int DT>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedMergeArgs a) {
  constexpr int kUnroll = 8;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= a.rows) return;
  const int f = threadIdx.x & 31;
  const int token = static_cast<int>(row / a.num_q_heads);
  const int qh = static_cast<int>(row - static_cast<int64_t>(token) * a.num_q_heads);
  const int h = qh / a.group, g = qh - h * a.group;
  const int req = a.row_of ? a.row_of[token] : token;
  int own_first = 0, own_count = 0;
  if (a.own_merge) {
    own_first = a.own_merge[2 * req];
    own_count = a.own_merge[2 * req + 1];
  }
  Join j;
  bool any = false;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int4 src = a.info[2 * req + part];  // {record, splits, row_tiles, token0}
    if (src.y == 0) continue;
    any = true;
    const int i = (token - src.w) * a.group + g;
    const int64_t first = src.x + static_cast<int64_t>(h) * src.z + i / 32;
    const int64_t step = static_cast<int64_t>(a.num_kv_heads) * src.z;
    for (int s0 = 0; s0 < src.y; s0 += kUnroll) {
      float lse[kUnroll];
      float4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t rec = first + min(s0 + u, src.y - 1) * step;
        lse[u] = s0 + u < src.y ? a.part_lse[rec * 32 + i % 32] : -INFINITY;
        v[u] = *reinterpret_cast<const float4*>(
            a.part_o + rec * kSharedRecord + ((f >> 1) * 64 + i % 32 + 32 * (f & 1)) * 4);
      }
      j.add(lse, v);
    }
  }
  if (own_count > 0 && (any || own_count > 1)) {
    for (int c0 = 0; c0 < own_count; c0 += kUnroll) {
      float lse[kUnroll];
      float4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t p =
            static_cast<int64_t>(own_first + min(c0 + u, own_count - 1)) * a.num_q_heads + qh;
        lse[u] = c0 + u < own_count ? a.own_lse[p] : -INFINITY;
        v[u] = *reinterpret_cast<const float4*>(a.own_o + p * kD + f * 4);
      }
      j.add(lse, v);
    }
  } else if (!any) {
    return;  // one item held the whole request and has written it
  }
  const float inv = 1.f / j.den;
  *reinterpret_cast<uint2*>(a.out + token * a.o_sn + qh * a.o_sh + f * 4) =
      make_uint2(Elem<DT>::pack2(j.acc.x * inv, j.acc.y * inv),
                 Elem<DT>::pack2(j.acc.z * inv, j.acc.w * inv));
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t slots_of(int64_t cus, int nw) { return nw == 8 ? cus : 2 * cus; }

// Items and records when a part of a source holds at most `length` tiles.
SharedCapacity count_at(const std::vector<SharedSource>& sources, int64_t group,
                        int64_t num_kv_heads, int nw, int64_t length) {
  SharedCapacity n{0, 0};
  for (const SharedSource& s : sources) {
    const int64_t rows = s.tokens * group;
    const int64_t splits =
        std::max<int64_t>(1, ceil_div(s.tile_end - s.tile_begin, std::max<int64_t>(length, 1)));
    n.items += ceil_div(rows, 32 * nw) * num_kv_heads * splits;
    n.records += ceil_div(rows, 32) * num_kv_heads * splits;
  }
  return n;
}

}  // namespace

int shared_waves(const std::vector<SharedSource>& sources, int64_t group) {
  // 256 rows a workgroup where they are mostly filled: K and V are read half as often. Fewer rows
  // leave waves of it idle, which two workgroups of 128 rows a CU do not.
  int64_t cost8 = 0, cost4 = 0;
  for (const SharedSource& s : sources) {
    const int64_t rows = s.tokens * group, tiles = s.tile_end - s.tile_begin;
    cost8 += 2 * ceil_div(rows, 256) * tiles;
    cost4 += ceil_div(rows, 128) * tiles;
  }
  return cost8 <= cost4 ? 8 : 4;
}

SharedCapacity shared_capacity(const std::vector<SharedSource>& sources, int64_t group,
                               int64_t num_kv_heads, int64_t cus, int nw) {
  const SharedCapacity whole =
      count_at(sources, group, num_kv_heads, nw, std::numeric_limits<int32_t>::max());
  return {whole.items + slots_of(cus, nw), whole.records + slots_of(cus, nw) * nw};
}

SharedCapacity shared_decode_capacity(int64_t rows, int64_t group, int64_t num_kv_heads,
                                      int64_t cus, int nw) {
  // At most rows / 2 groups share, each with a last tile that is not full.
  const int64_t groups = rows / 2;
  return {(rows * group / (32 * nw) + groups) * num_kv_heads + slots_of(cus, nw),
          (rows * group / 32 + groups) * num_kv_heads + slots_of(cus, nw) * nw};
}

int64_t schedule_shared(std::vector<SharedSource>& sources, int64_t group, int64_t num_kv_heads,
                        int64_t cus, int nw, const SharedCapacity& cap,
                        std::vector<int32_t>& work) {
  int64_t longest = 1;
  for (const SharedSource& s : sources)
    longest = std::max<int64_t>(longest, s.tile_end - s.tile_begin);
  // The length of a part that ends the launch soonest: rounds of items over the chip, each as long
  // as its longest part and what an item costs besides its tiles (its queries, its first tile and
  // its partial: about two tiles), and the parts that the merge has to read.
  constexpr double kItemTiles = 2.0, kMergeTiles = 0.25;
  const int64_t slots = slots_of(cus, nw);
  int64_t length = longest;
  double best = 0;
  for (int64_t parts = 1; parts <= std::min<int64_t>(longest, 256); ++parts) {
    const int64_t l = ceil_div(longest, parts);
    const SharedCapacity n = count_at(sources, group, num_kv_heads, nw, l);
    if (n.items > cap.items || n.records > cap.records) break;
    const double est = static_cast<double>(ceil_div(n.items, slots)) * (l + kItemTiles) +
                       kMergeTiles * parts;
    if (parts == 1 || est < best) {
      best = est;
      length = l;
    }
  }
  struct Item {
    int64_t tiles;
    int32_t source, row0, head, split, begin, end;
  };
  std::vector<Item> items;
  int64_t records = 0;
  for (size_t i = 0; i < sources.size(); ++i) {
    SharedSource& s = sources[i];
    const int64_t rows = s.tokens * group, tiles = s.tile_end - s.tile_begin;
    s.splits = static_cast<int32_t>(std::max<int64_t>(1, ceil_div(tiles, length)));
    s.row_tiles = static_cast<int32_t>(ceil_div(rows, 32));
    s.record = static_cast<int32_t>(records);
    records += static_cast<int64_t>(s.splits) * num_kv_heads * s.row_tiles;
    for (int32_t p = 0; p < s.splits; ++p)
      for (int64_t row0 = 0; row0 < rows; row0 += 32 * nw) {
        const int32_t begin = static_cast<int32_t>(s.tile_begin + tiles * p / s.splits);
        int64_t end = s.tile_begin + tiles * (p + 1) / s.splits;
        if (s.pos0 < kNoHorizon) {  // no tile past what the item's last row sees
          const int64_t last = s.pos0 + (std::min<int64_t>(row0 + 32 * nw, rows) - 1) / group;
          end = std::max<int64_t>(begin, std::min<int64_t>(end, last / kSharedTile + 1));
        }
        for (int32_t h = 0; h < num_kv_heads; ++h)
          items.push_back({end - begin, static_cast<int32_t>(i), static_cast<int32_t>(row0), h, p,
                           begin, static_cast<int32_t>(end)});
      }
  }
  // Longest first; heads stay fastest, so that with 8 of them a head's items, which read the same
  // keys, meet in the L2 of one XCD.
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& x, const Item& y) { return x.tiles > y.tiles; });
  work.reserve(work.size() + items.size() * kSharedItemInts);
  for (const Item& it : items) {
    const SharedSource& s = sources[it.source];
    const int64_t rec = s.record +
                        (static_cast<int64_t>(it.split) * num_kv_heads + it.head) * s.row_tiles +
                        it.row0 / 32;
    work.insert(work.end(),
                {s.token0, static_cast<int32_t>(s.tokens * group), it.row0, it.head, s.page_base,
                 it.begin, it.end, static_cast<int32_t>(rec), s.pos0, s.kv_len, 0, 0});
  }
  return records;
}

bool shared_lengths(const int32_t* group_rows, const int32_t* group_lens, int64_t groups,
                    const int32_t* limit, int64_t num_kv_heads, std::vector<int32_t>& eff) {
  eff.assign(groups, 0);
  bool any = false;
  int64_t row = 0;
  for (int64_t g = 0; g < groups; ++g) {
    int64_t len = std::min<int64_t>(group_lens[g], kSharedMaxKeys - kSharedTile);
    for (int64_t r = row; r < row + group_rows[g]; ++r) len = std::min<int64_t>(len, limit[r]);
    row += group_rows[g];
    if (group_rows[g] < 2) continue;
    eff[g] = static_cast<int32_t>(len / kSharedTile * kSharedTile);
    any |= eff[g] > 0;
  }
  return any;
}

const char* launch_shared(const SharedArgs& a, int64_t dtype, int nw, int64_t grid,
                          hipStream_t s) {
  const dim3 blocks(static_cast<uint32_t>(grid));
  if (dtype == 0) {
    if (nw == 8) shared_kernel<0, 8><<<blocks, dim3(512), 0, s>>>(a);
    else shared_kernel<0, 4><<<blocks, dim3(256), 0, s>>>(a);
  } else {
    if (nw == 8) shared_kernel<1, 8><<<blocks, dim3(512), 0, s>>>(a);
    else shared_kernel<1, 4><<<blocks, dim3(256), 0, s>>>(a);
  }
  return launch_status("shared_kernel");
}

const char* launch_shared_merge(const SharedMergeArgs& a, int64_t dtype, hipStream_t s) {
  const dim3 blocks(static_cast<uint32_t>((a.rows + 7) / 8));
  if (dtype == 0) shared_merge_kernel<0><<<blocks, dim3(256), 0, s>>>(a);
  else shared_merge_kernel<1><<<blocks, dim3(256), 0, s>>>(a);
  return launch_status("shared_merge_kernel");
}

}  // namespace mi355x
