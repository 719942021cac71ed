// Copies of cache pages over every layer's K and V, for sequences that are forked inside a page and
// pages that move. No counterpart in the reference (src/engine/kvcache/pool.rs:81-179 hands pages
// out and takes them back).
//
// A pool is [planes][pages][page_tokens][token_bytes]; a copy moves the first tokens of a page to
// another page of every plane. The destinations are distinct and none of them is a source, so the
// copies are independent of each other. Bound by memory: every byte is read and written once.
//
// The pairs travel as kernel arguments, some hundreds a launch: no upload, no staging buffer that a
// later call would have to wait for, and a captured launch carries its own.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "common.h"

namespace mi355x {
namespace {

constexpr int kThreads = 256;

// Whole pages, and pages of which some tokens are copied: under the 4 KiB of arguments.
struct WholeBatch {
  static constexpr int kPairs = 480;
  int32_t src[kPairs], dst[kPairs];
  __device__ int64_t tokens(int, int64_t page_tokens) const { return page_tokens; }
};
struct PartialBatch {
  static constexpr int kPairs = 320;
  int32_t src[kPairs], dst[kPairs], valid[kPairs];
  __device__ int64_t tokens(int pair, int64_t) const { return valid[pair]; }
};

// Grid: {parts of a page, pairs, planes}; a thread copies a word. us, one word a thread against four
// loaded together: 255 copies of 9 tokens of few sources in 56 planes 62 and 94 (the sources come
// from the caches), 400 pages of 64 tokens in 8 planes 139 and 158 (6.0 TB/s read and written).
template <typename Word, typename Batch>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(uint8_t* pool, int64_t plane_bytes,
                                                              int64_t page_tokens,
                                                              int64_t token_bytes, Batch batch) {
  const int pair = blockIdx.y;
  const int64_t page_bytes = page_tokens * token_bytes;
  const int64_t words =
      batch.tokens(pair, page_tokens) * token_bytes / static_cast<int64_t>(sizeof(Word));
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (at >= words) return;
  uint8_t* plane = pool + blockIdx.z * plane_bytes;
  const Word* src = reinterpret_cast<const Word*>(plane + batch.src[pair] * page_bytes);
  Word* dst = reinterpret_cast<Word*>(plane + batch.dst[pair] * page_bytes);
  dst[at] = src[at];
}

struct Pool {
  uint8_t* base;
  int64_t planes, plane_pages, page_tokens, token_bytes;
};

// Workgroups that copy some tokens of a page.
int64_t parts_of(const Pool& p, int64_t tokens, int64_t word) {
  return (tokens * p.token_bytes / word + kThreads - 1) / kThreads;
}

// `most`: the longest copy's tokens.
template <typename Word, typename Batch>
const char* launch(const Pool& p, const Batch& batch, int pairs, int64_t most, hipStream_t s) {
  const int64_t parts = parts_of(p, most, sizeof(Word));
  const dim3 grid(static_cast<uint32_t>(parts), static_cast<uint32_t>(pairs),
                  static_cast<uint32_t>(p.planes));
  copy_pages_kernel<Word><<<grid, dim3(kThreads), 0, s>>>(
      p.base, p.plane_pages * p.page_tokens * p.token_bytes, p.page_tokens, p.token_bytes, batch);
  return launch_status("mi355x_copy_pages");
}

// Launches of about equal size for all pairs, each of fewer than 2^32 threads (a grid of more would be
// cut short without an error).
template <typename Batch>
const char* copy_all(const Pool& p, const int32_t* src, const int32_t* dst, const int32_t* tokens,
                     int64_t pairs, bool wide, hipStream_t s) {
  const int64_t pair_threads =
      parts_of(p, p.page_tokens, wide ? sizeof(uint4) : sizeof(uint16_t)) * kThreads * p.planes;
  const int64_t room = std::min<int64_t>(Batch::kPairs, ((int64_t(1) << 32) - 1) / pair_threads);
  if (room == 0) return set_error("mi355x_copy_pages: page too large");
  const int64_t launches = (pairs + room - 1) / room;
  Batch batch;
  for (int64_t l = 0; l < launches; ++l) {
    int n = 0;
    int64_t most = 0;
    for (int64_t i = pairs * l / launches; i < pairs * (l + 1) / launches; ++i) {
      const int32_t t = tokens ? tokens[i] : static_cast<int32_t>(p.page_tokens);
      if (t == 0) continue;
      batch.src[n] = src[i];
      batch.dst[n] = dst[i];
      if constexpr (std::is_same_v<Batch, PartialBatch>) batch.valid[n] = t;
      ++n;
      most = std::max<int64_t>(most, t);
    }
    if (n == 0) continue;
    if (const char* err = wide ? launch<uint4>(p, batch, n, most, s)
                               : launch<uint16_t>(p, batch, n, most, s))
      return err;
  }
  return nullptr;
}

// One mark a page of the pool, kept between calls of a thread and cleared after each.
enum : uint8_t { kSource = 1, kDestination = 2 };

const char* check_pairs(int64_t pages, int64_t page_tokens, const int32_t* src, const int32_t* dst,
                        const int32_t* tokens, int64_t pairs) {
  static thread_local std::vector<uint8_t> marks;
  if (marks.size() < static_cast<size_t>(pages)) marks.resize(pages);
  for (int64_t i = 0; i < pairs; ++i) {
    if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
      return set_error("mi355x_copy_pages: a page is outside the pool");
    if (tokens && (tokens[i] < 0 || tokens[i] > page_tokens))
      return set_error("mi355x_copy_pages: a token count is outside the page");
  }
  bool twice = false;
  for (int64_t i = 0; i < pairs; ++i) marks[src[i]] = kSource;
  for (int64_t i = 0; i < pairs; ++i) {
    twice |= marks[dst[i]] != 0;
    marks[dst[i]] = kDestination;
  }
  for (int64_t i = 0; i < pairs; ++i) marks[src[i]] = marks[dst[i]] = 0;
  return twice ? set_error("mi355x_copy_pages: a destination is a source or another destination")
               : nullptr;
}

}  // namespace
}  // namespace mi355x

using namespace mi355x;

extern "C" const char* mi355x_copy_pages(void* pool, int64_t planes, int64_t plane_pages,
                                         int64_t page_tokens, int64_t token_bytes,
                                         const int32_t* src, const int32_t* dst,
                                         const int32_t* tokens, int64_t pairs, void* stream) {
  try {
    if (planes <= 0 || planes > 65535 || plane_pages <= 0 || plane_pages >= int64_t(1) << 31 ||
        page_tokens <= 0 || token_bytes <= 0 || token_bytes % 2 || pairs < 0 ||
        page_tokens >= int64_t(1) << 31 || token_bytes >= int64_t(1) << 31 ||
        page_tokens * token_bytes >= int64_t(1) << 40)
      return set_error("mi355x_copy_pages: invalid geometry");
    if (pairs == 0) return nullptr;
    if (!pool || !src || !dst) return set_error("mi355x_copy_pages: null pointer");
    if (!aligned(pool, 2)) return set_error("mi355x_copy_pages: misaligned pool");
    if (const char* err = check_pairs(plane_pages, page_tokens, src, dst, tokens, pairs))
      return err;
    const bool wide = token_bytes % 16 == 0 && aligned(pool, 16);
    const Pool p{static_cast<uint8_t*>(pool), planes, plane_pages, page_tokens, token_bytes};
    auto s = static_cast<hipStream_t>(stream);
    return tokens ? copy_all<PartialBatch>(p, src, dst, tokens, pairs, wide, s)
                  : copy_all<WholeBatch>(p, src, dst, nullptr, pairs, wide, s);
  } catch (const std::exception& e) {
    return set_error(e.what());
  }
}
