// Copies of cache pages over every layer's K and V, for sequences that are forked inside a page and
// pages that move. No counterpart in the reference (src/engine/kvcache/pool.rs:81-179 hands pages
// out and takes them back).
//
// A pool is [planes][pages][page_tokens][token_bytes]; a copy moves the first tokens of a page to
// another page of every plane. The destinations are distinct and none of them is a source, so the
// copies are independent of each other. Bound by memory: every byte is read and written once.
//
// The pairs travel as kernel arguments, kBatch a launch: no upload, no staging buffer that a later
// call would have to wait for, and a captured launch carries its own.
#include <algorithm>
#include <vector>

#include "common.h"

namespace mi355x {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // 16-byte words of a thread, loaded together
constexpr int kBatch = 240; // pairs of a launch: 12 bytes each, under the 4 KiB of arguments

struct CopyBatch {
  int32_t src[kBatch], dst[kBatch], tokens[kBatch];
};

// Grid: {parts of a page, pairs, planes}; a workgroup copies kThreads * kUnroll words.
template <typename Word>
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(uint8_t* pool, int64_t plane_bytes,
                                                              int64_t page_bytes,
                                                              int64_t token_bytes,
                                                              CopyBatch batch) {
  const int pair = blockIdx.y;
  const int64_t bytes = batch.tokens[pair] * token_bytes;
  const int64_t words = bytes / static_cast<int64_t>(sizeof(Word));
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * kUnroll) + threadIdx.x;
  uint8_t* plane = pool + blockIdx.z * plane_bytes;
  const Word* src = reinterpret_cast<const Word*>(plane + batch.src[pair] * page_bytes);
  Word* dst = reinterpret_cast<Word*>(plane + batch.dst[pair] * page_bytes);
  Word w[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (first + u * kThreads < words) w[u] = src[first + u * kThreads];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (first + u * kThreads < words) dst[first + u * kThreads] = w[u];
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
    const int64_t page_bytes = page_tokens * token_bytes;
    const bool wide = token_bytes % 16 == 0 && aligned(pool, 16);
    const int64_t word = wide ? 16 : 2;
    auto s = static_cast<hipStream_t>(stream);
    CopyBatch batch;
    for (int64_t done = 0; done < pairs;) {
      int n = 0;
      int64_t most = 0;
      for (; done < pairs && n < kBatch; ++done) {
        const int32_t t = tokens ? tokens[done] : static_cast<int32_t>(page_tokens);
        if (t == 0) continue;
        batch.src[n] = src[done];
        batch.dst[n] = dst[done];
        batch.tokens[n++] = t;
        most = std::max<int64_t>(most, t);
      }
      if (n == 0) break;
      const int64_t parts = (most * token_bytes / word + kThreads * kUnroll - 1) /
                            (kThreads * kUnroll);
      if (parts > (int64_t(1) << 31) / kThreads)
        return set_error("mi355x_copy_pages: page too large");
      const dim3 grid(static_cast<uint32_t>(parts), static_cast<uint32_t>(n),
                      static_cast<uint32_t>(planes));
      auto* base = static_cast<uint8_t*>(pool);
      if (wide)
        copy_pages_kernel<uint4><<<grid, dim3(kThreads), 0, s>>>(
            base, plane_pages * page_bytes, page_bytes, token_bytes, batch);
      else
        copy_pages_kernel<uint16_t><<<grid, dim3(kThreads), 0, s>>>(
            base, plane_pages * page_bytes, page_bytes, token_bytes, batch);
      if (const char* err = launch_status("mi355x_copy_pages")) return err;
    }
    return nullptr;
  } catch (const std::exception& e) {
    return set_error(e.what());
  }
}
