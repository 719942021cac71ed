// Log probabilities of given tokens, entropy and the most likely alternatives of logits rows.
//
//   lp[r]      = x[r, tokens[r]] - lse(x[r]),  lse(x) = log sum_j exp(x_j)
//   entropy[r] = lse(x[r]) - sum_j p_j x_j,    p = softmax(x[r])
//   ids[r, :]  = the `top` largest logits, largest first, equal ones by the lower index (a NaN
//                sorts above +inf), top_lp[r, s] = x[r, ids[r, s]] - lse(x[r])
//
// No counterpart in the reference, whose sampler (src/engine/sampling.rs:239-372) returns ids only.
//
// One pass over the row. A thread keeps a reference M (the largest logit it has seen), and, with
// t = x log2(e) - M log2(e) formed by one fma, s = sum 2^t and w = sum t 2^t; both are rescaled when
// M moves. Then lp = (t_token - log2 s) ln 2 and entropy = (log2 s - w / s) ln 2: no difference of
// large numbers anywhere (the rounding of log2(e) acts as a change of temperature by 1e-8). All sums
// are fp32, up to 1,024 terms a thread (594 at 151,936 logits) and trees above them.
//
// Alternatives, from the same pass: every thread keeps its largest logit and where it first met
// it, and the largest of every 32 logits goes to LDS. The top-th largest of the threads' bests is a
// threshold that at least `top` logits reach and few others do; only the groups of 32 whose largest
// reaches it are read again (from the caches) and compared, and one wave sorts what passes. Rows
// for which that does not hold (a NaN or an infinity, more than kCandidates logits in reach) are
// selected by repeated maxima instead, at the cost of a pass over the row an alternative (256 rows of
// 151,936 logits with 20 alternatives: 25.6 us, with 100 finite logits a row 31.5, with a NaN in every row
// 3.7 ms, and 0.35 ms without alternatives).
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "common.h"

namespace mi355x {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 64;            // one lane an alternative
constexpr int kGroup = 32;             // logits under one maximum in LDS
constexpr int kCandidates = 1024;      // (key, index) entries in LDS
constexpr int kListed = 128;           // groups that a wave lists before it reads them ...
constexpr int kLook = 4;               // maxima that a thread looks at together
constexpr int kReads = 4;              // ... two at a time in each of so many loads
// Threads of a workgroup, for long rows and short ones. us, 256 threads a long row against 512 and 128:
// 4,096 rows of 151,936 bf16 logits with 5 alternatives 230, 239, 268 (now 228 at 256, 5.45 TB/s),
// without 216 (5.8 TB/s), 219, 229; 256 rows with 20 alternatives 27.0, 30.2, 42.8 (now 23.5), without
// 16.7, 23, 27. Bound by memory and, nearly as much, by the dozen vector operations a logit. At 87
// registers five waves fit a SIMD; a cap at 80, for a sixth, spills (4,096 rows 414 us).
constexpr int kWide = 256, kNarrow = 64;
// Rows up to this go to single waves, which have no barriers to wait at (4,096 rows of 8,000 logits:
// 22 us, with four waves a row 40).
constexpr int64_t kNarrowVocab = 8192;
constexpr int kMaxSegments = 64;       // of a row: what the joining workgroup holds
// Logits under one workgroup: bounds the maxima in LDS to 32 KiB.
constexpr int64_t kMaxSegment = 262144;
// A reference from here on is left to careful_stats: the streaming loop's exponents are off by the
// rounding of M log2(e), which all of a row share, so that it only scales s and w; here it is 2^0.09.
constexpr float kFarRef = 1e6f;
constexpr float kOverflow = 2e38f;     // times log2(e) may be infinite
constexpr float kFarStep = -1e4f;      // 2^-10000 is 0 and stays finite times any s

template <int DT>
struct Row {  // logits of dtype codes 0 (bf16), 1 (fp16), 2 (fp32)
  using Word = uint16_t;
  static constexpr int kVec = 8;
  static constexpr int kKeyShift = DT == 0 ? 16 : 13;  // low bits of a widened value that are zero
  __device__ __forceinline__ static float value(Word w) { return Elem<DT>::to_float(w); }
  __device__ __forceinline__ static uint4 load(const Word* p) { return ld128_any(p); }
  __device__ __forceinline__ static void widen(const uint4& v, float (&f)[kVec]) {
    unpack8<DT>(v, f);
  }
};
typedef uint32_t Words4Float __attribute__((ext_vector_type(4), aligned(4)));
template <>
struct Row<2> {
  using Word = float;
  static constexpr int kVec = 4;
  static constexpr int kKeyShift = 0;
  __device__ __forceinline__ static float value(Word w) { return w; }
  __device__ __forceinline__ static uint4 load(const Word* p) {
    const Words4Float v = *reinterpret_cast<const Words4Float*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
  }
  __device__ __forceinline__ static void widen(const uint4& v, float (&f)[kVec]) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
};

// Orders like the value, -0 as 0, every NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xfffffffeu;  // so that every rank key lies below ~0
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// Orders alternatives: by value, equal ones by the lower index. 0 stands for none.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
  return (static_cast<uint64_t>(order_key(x)) << 32) | ~index;
}
__device__ __forceinline__ float rank_value(uint64_t key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ uint32_t rank_index(uint64_t key) {
  return ~static_cast<uint32_t>(key);
}

// The value of lane ^ MASK, by register moves (LDS shuffles take several times as long, and sorting
// is a chain of them).
template <int MASK>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  constexpr int kQuadReverse = 0x1B, kRowRotate8 = 0x128;
  auto move = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  if constexpr (MASK == 1) {
    return move(v, std::integral_constant<int, kDppQuadSwap1>{});
  } else if constexpr (MASK == 2) {
    return move(v, std::integral_constant<int, kDppQuadSwap2>{});
  } else if constexpr (MASK == 4) {  // 7 - i, then 3 - i within four
    return move(move(v, std::integral_constant<int, kDppRowHalfMirror>{}),
                std::integral_constant<int, kQuadReverse>{});
  } else if constexpr (MASK == 8) {
    return move(v, std::integral_constant<int, kRowRotate8>{});
  } else if constexpr (MASK == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? s[0] : s[1];
  } else if constexpr (MASK == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? s[0] : s[1];
  } else {
    static_assert(MASK == 63, "one bit, or all");
    return lane_xor<32>(
        lane_xor<16>(move(v, std::integral_constant<int, kDppRowMirror>{})));
  }
}
template <int MASK>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  const uint32_t lo = lane_xor<MASK>(static_cast<uint32_t>(v));
  const uint32_t hi = lane_xor<MASK>(static_cast<uint32_t>(v >> 32));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
template <int MASK>
__device__ __forceinline__ float lane_xor(float v) {
  return __uint_as_float(lane_xor<MASK>(__float_as_uint(v)));
}
// f(std::integral_constant<int, 2^i>) for the strides FROM, FROM / 2, .. 1.
template <int FROM, typename F>
__device__ __forceinline__ void strides_down(F&& f) {
  f(std::integral_constant<int, FROM>{});
  if constexpr (FROM > 1) strides_down<FROM / 2>(f);
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The wave's 64 keys in descending order, lane 0 the largest: SIZE keys at a time.
template <int SIZE = 64>
__device__ __forceinline__ uint64_t sort_desc(uint64_t v, int lane) {
  if constexpr (SIZE > 2) v = sort_desc<SIZE / 2>(v, lane);
  strides_down<SIZE / 2>([&](auto stride) {
    constexpr int kStride = decltype(stride)::value;
    const uint64_t o = lane_xor<kStride>(v);
    const bool larger = ((lane & SIZE) == 0 || SIZE == 64) == ((lane & kStride) == 0);
    v = (v > o) == larger ? v : o;
  });
  return v;
}
// The 64 largest of two descending runs, descending.
__device__ __forceinline__ uint64_t merge_desc(uint64_t a, uint64_t b, int lane) {
  uint64_t v = max64(a, lane_xor<63>(b));
  strides_down<32>([&](auto stride) {
    constexpr int kStride = decltype(stride)::value;
    const uint64_t o = lane_xor<kStride>(v);
    v = (v > o) == ((lane & kStride) == 0) ? v : o;
  });
  return v;
}

// A part's sums relative to its reference; s = 0: nothing in it yet.
struct Stats {
  float m, s, w;
};

// log2(e) times a reference as the sums are formed with it: rounded. Contracted into a difference it
// would not be, and parts whose references differ would be joined with weights that are off by its
// rounding (2^-4 at logits of a million).
__device__ __forceinline__ float in_log2(float m) {
#pragma clang fp contract(off)
  return m * kLog2e;
}
__device__ __forceinline__ bool near(float m) { return fabsf(m) < kFarRef; }
// What a's sums are relative to, less what b's are. A far reference is an exact one.
__device__ __forceinline__ float ref_step(float a, float b) {
  if (a == b) return 0.f;
  if (near(a) && near(b)) return in_log2(a) - in_log2(b);
  if (near(b)) return fmaf(a, kLog2e, -in_log2(b));
  if (near(a)) return -fmaf(b, kLog2e, -in_log2(a));
  return (a - b) * kLog2e;
}
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
  Stats r;
  r.m = fmaxf(a.m, b.m);
  r.s = r.w = 0.f;
  const Stats parts[2] = {a, b};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Stats& p = parts[i];
    if (p.s == 0.f) continue;
    const float d = fmaxf(ref_step(p.m, r.m), kFarStep);
    const float f = __builtin_amdgcn_exp2f(d);
    r.s = fmaf(p.s, f, r.s);
    r.w = fmaf(fmaf(d, p.s, p.w), f, r.w);
  }
  return r;
}
__device__ __forceinline__ Stats wave_join(Stats v) {
  strides_down<32>([&](auto stride) {
    constexpr int kStride = decltype(stride)::value;
    v = join(v, {lane_xor<kStride>(v.m), lane_xor<kStride>(v.s), lane_xor<kStride>(v.w)});
  });
  return v;
}

struct LogprobArgs {
  const void* logits;
  int64_t vocab, stride;
  const int64_t* tokens;
  float* lp;
  float* entropy;
  int64_t* ids;
  float* top_lp;
  int32_t top, segments;
  int64_t segment;       // logits of a segment, a multiple of 8
  float4* part_stats;    // [rows][segments] {m, s, w, 0}
  uint64_t* part_keys;   // [rows][segments][top]
};

// The given token's logit: NaN outside the vocabulary. Loaded at a kernel's start, as it takes two
// loads in turn.
template <int DT>
__device__ __forceinline__ float given_logit(const LogprobArgs& a, int64_t row) {
  using R = Row<DT>;
  const int64_t tok = a.tokens[row];
  return tok >= 0 && tok < a.vocab
             ? R::value(static_cast<const typename R::Word*>(a.logits)[row * a.stride + tok])
             : __builtin_nanf("");
}

// What one wave writes of a row whose sums and alternatives (descending over the lanes) it has.
__device__ __forceinline__ void write_row(const LogprobArgs& a, int64_t row, const Stats& st,
                                          uint64_t key, float given, int lane) {
  // v_log_f32 (log2); s >= 1 or 0, NaN for rows with a NaN or +inf. A row of only -inf: s = 0.
  const float bits = __builtin_amdgcn_logf(st.s);
  auto lp = [&](float v) {
    if (bits != bits) return bits;  // of joined parts only s shows a NaN: the largest m is a number
    if (!near(st.m)) return (v - st.m) - bits * kLn2;
    if (fabsf(v) >= kOverflow) return v - st.m;  // log2 s is far below its rounding
    return (fmaf(v, kLog2e, -in_log2(st.m)) - bits) * kLn2;
  };
  if (lane == 0) {
    a.lp[row] = lp(given);
    a.entropy[row] = (bits - st.w / st.s) * kLn2;
  }
  if (lane < a.top) {
    a.ids[row * a.top + lane] = rank_index(key);
    a.top_lp[row * a.top + lane] = lp(rank_value(key));
  }
}

template <int THREADS>
struct Scratch {
  static constexpr int kWaves = THREADS / kWave;
  Stats stats[kWaves];
  uint64_t best[kWaves];
  uint32_t bound_key, bound_vec, count;
  uint32_t key[THREADS];  // a thread's largest logit (0: it has none) ...
  uint32_t vec[THREADS];  // ... and the vector in which it met it first
  uint64_t cand[kCandidates];
  uint16_t groups[kWaves][kListed];
};

// Largest of the threads' keys, in every thread.
template <int THREADS>
__device__ __forceinline__ uint64_t block_max(Scratch<THREADS>& sh, uint64_t v) {
  strides_down<32>([&](auto stride) { v = max64(v, lane_xor<decltype(stride)::value>(v)); });
  if constexpr (THREADS > kWave) {
    if (threadIdx.x % kWave == 0) sh.best[threadIdx.x / kWave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Scratch<THREADS>::kWaves; ++w) v = max64(v, sh.best[w]);
    __syncthreads();
  }
  return v;
}

// The sums of n logits by their definition, for references out of the streaming loop's range and
// rows with a NaN or an infinity.
template <int DT, int THREADS>
__device__ __noinline__ Stats careful_stats(const typename Row<DT>::Word* x, int64_t n,
                                            Scratch<THREADS>& sh) {
  using R = Row<DT>;
  uint64_t top = 0;
  for (int64_t i = threadIdx.x; i < n; i += THREADS)
    top = max64(top, rank_key(R::value(x[i]), static_cast<uint32_t>(i)));
  top = block_max<THREADS>(sh, top);
  const float m = R::value(x[rank_index(top)]);
  if (m == -INFINITY) return {-FLT_MAX, 0.f, 0.f};
  Stats st{m, 0.f, 0.f};
  for (int64_t i = threadIdx.x; i < n; i += THREADS) {
    const float t = (R::value(x[i]) - m) * kLog2e;  // NaN where m is NaN or +inf
    const float e = __builtin_amdgcn_exp2f(t);
    st.s += e;
    st.w = fmaf(fmaxf(t, kFarStep), e, st.w);
  }
  // The references are equal: plain sums, which carry a NaN.
#pragma unroll
  for (int off = 1; off < kWave; off *= 2) {
    st.s += __shfl_xor(st.s, off);
    st.w += __shfl_xor(st.w, off);
  }
  if constexpr (THREADS > kWave) {
    if (threadIdx.x % kWave == 0) sh.stats[threadIdx.x / kWave] = st;
    __syncthreads();
    st.s = st.w = 0.f;
#pragma unroll
    for (int w = 0; w < Scratch<THREADS>::kWaves; ++w) {
      st.s += sh.stats[w].s;
      st.w += sh.stats[w].w;
    }
    __syncthreads();
  }
  return st;
}

// The `top` largest of n logits by repeated maxima; lane s of every wave gets the s-th.
template <int DT, int THREADS>
__device__ __noinline__ uint64_t careful_top(const typename Row<DT>::Word* x, int64_t n, int top,
                                             Scratch<THREADS>& sh) {
  using R = Row<DT>;
  uint64_t mine = 0, last = ~0ull;
  for (int s = 0; s < top; ++s) {
    uint64_t best = 0;
    for (int64_t i = threadIdx.x; i < n; i += THREADS) {
      const uint64_t k = rank_key(R::value(x[i]), static_cast<uint32_t>(i));
      if (k < last) best = max64(best, k);
    }
    last = block_max<THREADS>(sh, best);
    if (static_cast<int>(threadIdx.x % kWave) == s) mine = last;
  }
  return mine;
}

// One wave: a bound that at least `top` of the threads' bests reach, as {key, vector}: a best
// reaches it with a larger key, or with this key in a vector up to this one.
template <int DT, int THREADS>
__device__ __forceinline__ void find_bound(Scratch<THREADS>& sh, int top, int lane) {
  constexpr int kPer = THREADS / kWave;
  constexpr int kSlack = 8;  // bests beyond `top` that end the search early
  uint32_t key[kPer];
  int present = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = sh.key[i * kWave + lane];
    present += __popcll(__ballot(key[i] != 0));
  }
  uint32_t bound = 0, vec = 0xffffffffu;
  if (present >= top) {
    int reach = present;
    constexpr int kTopBit = 31 - Row<DT>::kKeyShift;
    for (int b = kTopBit; b >= 0 && reach > top + kSlack; --b) {
      const uint32_t t = bound | (1u << b);
      int c = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) c += __popcll(__ballot(key[i] >= t));
      if (c >= top) {
        bound = t;
        reach = c;
      }
    }
    if (reach > top + kSlack) {  // many equal bests: the first of them will do
      int need = top;
#pragma unroll
      for (int i = 0; i < kPer; ++i) need -= __popcll(__ballot(key[i] > bound));
      vec = 0;
      for (int b = 17; b >= 0; --b) {  // the largest v that fewer than `need` lie below
        const uint32_t t = vec | (1u << b);
        int c = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          c += __popcll(__ballot(key[i] == bound && sh.vec[i * kWave + lane] < t));
        if (c < need) vec = t;
      }
    }
  }
  if (lane == 0) {
    sh.bound_key = bound;
    sh.bound_vec = vec;
    sh.count = 0;
  }
}

// VPT vectors a thread and step, which hold kGroup logits. Dynamic LDS: the maxima of the groups,
// [step][thread].
template <int DT, int THREADS, bool TOP>
__global__ __launch_bounds__(THREADS) void logprob_kernel(LogprobArgs a) {
  using R = Row<DT>;
  using W = typename R::Word;
  constexpr int V = R::kVec;
  constexpr int VPT = kGroup / V;
  constexpr int kWaves = THREADS / kWave;
  __shared__ Scratch<THREADS> sh;
  extern __shared__ float group_max[];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t row = blockIdx.x / static_cast<uint32_t>(a.segments);
  const int seg = static_cast<int>(blockIdx.x - row * a.segments);
  const int64_t begin = seg * a.segment;
  const int n = static_cast<int>(min(a.vocab - begin, a.segment));
  const W* x = static_cast<const W*>(a.logits) + row * a.stride + begin;
  const int vecs = n / V;  // whole ones; what is left is one more
  const int all_vecs = (n + V - 1) / V;
  const int steps = (all_vecs + VPT * THREADS - 1) / (VPT * THREADS);
  const int whole_steps = vecs / (VPT * THREADS);

  float given = 0.f;
  if (wave == 0 && a.segments == 1) given = given_logit<DT>(a, row);

  float m = -kFarRef, ref = 0.f, s = 0.f, w = 0.f;
  float best = -INFINITY;
  uint32_t best_vec = 0xffffffffu;
  // Group j of 8 or 4 logits of a step, the step's first vector of this thread being v0.
  auto consume = [&](int step, const uint4 (&raw)[VPT], int have) {
    float f[VPT][V];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      R::widen(raw[j], f[j]);
      float vm = f[j][0];
#pragma unroll
      for (int i = 1; i < V; ++i) vm = fmaxf(vm, f[j][i]);
      if constexpr (TOP) {
        // The first vector counts also where all its logits are -inf.
        if (j < have && (vm > best || best_vec == 0xffffffffu)) {
          best = vm;
          best_vec = (step * VPT + j) * THREADS + tid;
        }
      }
      top = fmaxf(top, vm);
    }
    if constexpr (TOP) group_max[step * THREADS + tid] = top;
    if (top > m) {
      const float to = in_log2(top);
      const float d = fmaxf(ref - to, kFarStep);
      const float c = s == 0.f ? 0.f : __builtin_amdgcn_exp2f(d);
      w = fmaf(d, s, w) * c;
      s *= c;
      m = top;
      ref = to;
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float t = fmaf(f[j][i], kLog2e, -ref);
        const float e = __builtin_amdgcn_exp2f(t);
        s += e;
        // a logit of -inf: 2^t is 0, and so has to be its part of w; a NaN stays in s
        w = fmaf(fmaxf(t, kFarStep), e, w);
      }
  };
  if (whole_steps > 0) {
    uint4 now[VPT], next[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) now[j] = R::load(x + (j * THREADS + tid) * V);
    for (int step = 0; step < whole_steps; ++step) {
      const int ahead = min(step + 1, whole_steps - 1);
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        next[j] = R::load(x + ((ahead * VPT + j) * THREADS + tid) * V);
      consume(step, now, VPT);
#pragma unroll
      for (int j = 0; j < VPT; ++j) now[j] = next[j];
    }
  }
  uint4 raw[VPT];
  if (steps > whole_steps) {  // the last step: vectors that are there, the row's end by logits
    constexpr uint32_t kNone = DT == 0 ? 0xff80ff80u : DT == 1 ? 0xfc00fc00u : 0xff800000u;
    int have = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = (whole_steps * VPT + j) * THREADS + tid;
      raw[j] = make_uint4(kNone, kNone, kNone, kNone);
      if (v < vecs) {
        raw[j] = R::load(x + v * V);
      } else if (v < all_vecs) {
        W last[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int at = v * V + i;
          if constexpr (DT == 2) last[i] = at < n ? x[at] : -INFINITY;
          else last[i] = at < n ? x[at] : static_cast<W>(kNone);
        }
        __builtin_memcpy(&raw[j], last, sizeof(uint4));
      }
      if (v < all_vecs) have = j + 1;
    }
    consume(whole_steps, raw, have);
  }

  // The row's (or segment's) sums, in every thread.
  Stats st = wave_join({m, s, w});
  if constexpr (TOP) {
    sh.key[tid] = best_vec == 0xffffffffu ? 0 : order_key(best) >> R::kKeyShift;
    sh.vec[tid] = best_vec;
  }
  if constexpr (kWaves > 1) {
    if (lane == 0) sh.stats[wave] = st;
    __syncthreads();
    st = sh.stats[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) st = join(st, sh.stats[i]);
    __syncthreads();
  } else {
    __syncthreads();
  }
  // No NaN and no +inf: the maxima order as the keys do (all that follows is uniform).
  const bool ordered = st.s == st.s;
  if (!ordered || !near(st.m)) st = careful_stats<DT, THREADS>(x, n, sh);

  uint64_t key = 0;
  if constexpr (TOP) {
    bool selected = false;
    if (ordered) {
      if (wave == 0) find_bound<DT, THREADS>(sh, a.top, lane);
      __syncthreads();
      const uint32_t bound = sh.bound_key, bound_vec = sh.bound_vec;
      auto consider = [&](float value, int v, int at) {
        const uint32_t k = order_key(value) >> R::kKeyShift;
        if (k > bound || (k == bound && static_cast<uint32_t>(v) <= bound_vec)) {
          const uint32_t slot = atomicAdd(&sh.count, 1u);
          if (slot < kCandidates) sh.cand[slot] = rank_key(value, static_cast<uint32_t>(begin) + at);
        }
      };
      if (whole_steps == 0) {
        // All of it is still in registers: the threads whose largest is in reach compare their own.
        if (sh.key[tid] >= bound && sh.key[tid] != 0) {
#pragma unroll
          for (int j = 0; j < VPT; ++j) {
            const int v = j * THREADS + tid;
            float f[V];
            R::widen(raw[j], f);
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (v * V + i < n) consider(f[i], v, v * V + i);
          }
        }
      } else {
        // Groups in reach are listed, then read some at a time: read where they are found, each read
        // waits for the one before it (256 rows of 151,936 logits with 20 alternatives 25.9 us, listed
        // 24.0, with some maxima looked at together 23.5; 4,096 rows with 5 231, 229 and 228.3).
        uint16_t* list = sh.groups[wave];
        int listed = 0;
        auto read_listed = [&] {
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes' entries
          for (int first = 0; first < listed; first += 2 * kReads) {
            float f[kReads];
            int v[kReads];
#pragma unroll
            for (int r = 0; r < kReads; ++r) {
              const int g = list[min(first + 2 * r + lane / kGroup, listed - 1)];
              v[r] = (g / THREADS * VPT + lane % kGroup / V) * THREADS + g % THREADS;
              f[r] = R::value(x[min(v[r] * V + lane % V, n - 1)]);
            }
#pragma unroll
            for (int r = 0; r < kReads; ++r) {
              const int at = v[r] * V + lane % V;
              if (first + 2 * r + lane / kGroup < listed && at < n) consider(f[r], v[r], at);
            }
          }
          listed = 0;
        };
        for (int step = 0; step < steps; step += kLook) {
          float gm[kLook];
#pragma unroll
          for (int j = 0; j < kLook; ++j)
            gm[j] = group_max[min(step + j, steps - 1) * THREADS + tid];
#pragma unroll
          for (int j = 0; j < kLook; ++j) {
            const int at = (step + j) * THREADS + tid;
            const bool in_row = step + j < steps && (step + j) * VPT * THREADS + tid < all_vecs;
            const uint64_t hits = __ballot(in_row && order_key(gm[j]) >> R::kKeyShift >= bound);
            if (hits == 0) continue;
            if (hits >> lane & 1)
              list[listed + __popcll(hits & ((uint64_t(1) << lane) - 1))] = static_cast<uint16_t>(at);
            listed += __popcll(hits);
            if (listed > kListed - kWave) read_listed();
          }
        }
        read_listed();
      }
      __syncthreads();
      const int count = static_cast<int>(sh.count);
      selected = count <= kCandidates;  // uniform
      if (selected && wave == 0)
        for (int c = 0; c < count; c += kWave) {
          const uint64_t run = sort_desc(c + lane < count ? sh.cand[c + lane] : 0, lane);
          key = c == 0 ? run : merge_desc(key, run, lane);
        }
    }
    if (!selected) {
      key = careful_top<DT, THREADS>(x, n, min(a.top, n), sh);
      if (key) key -= static_cast<uint32_t>(begin);  // index + begin, as the key holds ~index
    }
  }
  if (wave != 0) return;
  if (a.segments == 1) {
    write_row(a, row, st, key, given, lane);
    return;
  }
  const int64_t part = row * a.segments + seg;
  if (lane == 0) a.part_stats[part] = make_float4(st.m, st.s, st.w, 0.f);
  if (lane < a.top) a.part_keys[part * a.top + lane] = key;
}

// Joins a row's segments, whose descending runs lie in LDS: 16 waves merge four each, then four waves
// four of theirs, then one the last four. The merge stands in one place, in a loop: a launch of a few
// workgroups pays for fetching its instructions, and unrolled copies cost more than they save.
template <int DT>
__global__ __launch_bounds__(1024) void logprob_join_kernel(LogprobArgs a) {
  __shared__ uint64_t runs[kMaxSegments][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = blockIdx.x;
  const int64_t part0 = row * a.segments;
  float given = 0.f;
  Stats st{-FLT_MAX, 0.f, 0.f};
  if (wave == 0) {
    given = given_logit<DT>(a, row);
    if (lane < a.segments) {
      const float4 p = a.part_stats[part0 + lane];
      st = {p.x, p.y, p.z};
    }
  }
  uint64_t key = 0;
  if (a.top) {
    uint64_t mine[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int seg = 4 * wave + r;
      mine[r] = seg < a.segments && lane < a.top ? a.part_keys[(part0 + seg) * a.top + lane] : 0;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) runs[4 * wave + r][lane] = mine[r];
#pragma unroll 1
    for (int step = 1; step < a.segments; step *= 4) {  // uniform; run 4 step w + i step, i < 4
      __syncthreads();
      const int first = wave * 4 * step;
      if (first < a.segments) {
        key = runs[first][lane];
#pragma unroll 1
        for (int i = 1; i < 4 && first + i * step < a.segments; ++i)
          key = merge_desc(key, runs[first + i * step][lane], lane);
        runs[first][lane] = key;
      }
    }
  }
  if (wave != 0) return;
  write_row(a, row, wave_join(st), key, given, lane);
}

// Segments of a row, so that few rows fill the chip: a workgroup a CU (two a CU: 256 rows of 151,936
// logits 29.5 us against 27.0, of 32,000 18.4 against 14.2).
struct Split {
  int64_t segments, length;
};
Split split_of(int64_t rows, int64_t vocab, int64_t cus) {
  const int64_t least = (vocab + kMaxSegment - 1) / kMaxSegment;
  int64_t want = rows > 0 ? (cus + rows - 1) / rows : 1;
  want = std::min(want, vocab / 2048);  // shorter ones cost more to join than they save
  const int64_t segments = std::max<int64_t>(least, std::min<int64_t>(want, kMaxSegments));
  const int64_t length = ((vocab + segments - 1) / segments + 7) / 8 * 8;
  return {(vocab + length - 1) / length, length};
}

int threads_of(const Split& sp) {
  return sp.length <= kNarrowVocab && sp.segments == 1 ? kNarrow : kWide;
}

template <int DT>
void launch(LogprobArgs a, int64_t rows, int threads, hipStream_t s) {
  const int64_t steps = (a.segment + kGroup * threads - 1) / (kGroup * threads);
  const uint32_t lds = a.top ? static_cast<uint32_t>(steps * threads * sizeof(float)) : 0;
  const dim3 grid(static_cast<uint32_t>(rows * a.segments)), block(threads);
  if (threads == kNarrow) {
    if (a.top) logprob_kernel<DT, kNarrow, true><<<grid, block, lds, s>>>(a);
    else logprob_kernel<DT, kNarrow, false><<<grid, block, lds, s>>>(a);
  } else {
    if (a.top) logprob_kernel<DT, kWide, true><<<grid, block, lds, s>>>(a);
    else logprob_kernel<DT, kWide, false><<<grid, block, lds, s>>>(a);
  }
  if (a.segments > 1)
    logprob_join_kernel<DT><<<dim3(static_cast<uint32_t>(rows)), dim3(1024), 0, s>>>(a);
}

bool valid_shape(int64_t rows, int64_t vocab, int64_t top, int32_t cus) {
  return rows >= 0 && vocab > 0 && vocab <= kMaxSegments * kMaxSegment && top >= 0 && top <= kMaxTop &&
         top <= vocab && cus > 0 && rows < (int64_t(1) << 31);
}

}  // namespace
}  // namespace mi355x

using namespace mi355x;

extern "C" int64_t mi355x_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top,
                                                         int32_t cus) {
  if (!valid_shape(rows, vocab, top, cus)) return -1;
  const Split sp = split_of(rows, vocab, cus);
  return sp.segments == 1 ? 0 : rows * sp.segments * (16 + 8 * top);
}

extern "C" const char* mi355x_token_logprobs(const void* logits, int64_t rows, int64_t vocab,
                                             int64_t row_stride, int dtype, const int64_t* tokens,
                                             int64_t top, void* logprobs, void* entropy,
                                             int64_t* top_ids, void* top_logprobs,
                                             void* workspace, int64_t workspace_bytes,
                                             int32_t cus, void* stream) {
  if (!valid_shape(rows, vocab, top, cus) || dtype < 0 || dtype > 2)
    return set_error("mi355x_token_logprobs: bad shape");
  if (rows == 0) return nullptr;
  if (!logits || !tokens || !logprobs || !entropy || (top && (!top_ids || !top_logprobs)))
    return set_error("mi355x_token_logprobs: null pointer");
  if (!aligned(logits, dtype == 2 ? 4 : 2) || (rows > 1 && row_stride < vocab))
    return set_error("mi355x_token_logprobs: rows must not overlap");
  const Split sp = split_of(rows, vocab, cus);
  // A grid of 2^32 threads or more would be cut short without an error.
  if (rows * sp.segments * threads_of(sp) >= int64_t(1) << 32)
    return set_error("mi355x_token_logprobs: too many rows for a launch");
  LogprobArgs a{};
  if (sp.segments > 1) {
    if (!workspace || !aligned(workspace, 16) ||
        workspace_bytes < rows * sp.segments * (16 + 8 * top))
      return set_error("mi355x_token_logprobs: workspace too small");
    a.part_stats = static_cast<float4*>(workspace);
    a.part_keys = reinterpret_cast<uint64_t*>(a.part_stats + rows * sp.segments);
  }
  a.logits = logits;
  a.vocab = vocab;
  a.stride = row_stride;
  a.tokens = tokens;
  a.lp = static_cast<float*>(logprobs);
  a.entropy = static_cast<float*>(entropy);
  a.ids = top_ids;
  a.top_lp = static_cast<float*>(top_logprobs);
  a.top = static_cast<int32_t>(top);
  a.segments = static_cast<int32_t>(sp.segments);
  a.segment = sp.length;
  auto s = static_cast<hipStream_t>(stream);
  const int threads = threads_of(sp);
  if (dtype == 0) launch<0>(a, rows, threads, s);
  else if (dtype == 1) launch<1>(a, rows, threads, s);
  else launch<2>(a, rows, threads, s);
  return launch_status("mi355x_token_logprobs");
}
