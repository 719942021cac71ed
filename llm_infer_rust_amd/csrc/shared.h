// Attention over prefixes that several requests of a batch share (shared.hip): what the decode and
// prefill plans need of it.
#pragma once

#include <cstdint>
#include <limits>
#include <memory>
#include <vector>

#include "common.h"

namespace mi355x {

// Split-KV schedule of decode.hip over requests of `lengths` tokens, in tiles of `tile`. Fills work
// (4 ints an item: request, token range, partial or -1), merge (2 ints a request: first partial or
// -1, items) and wg (first item of each workgroup, one past the last); the items, or -1 when a
// capacity is too small. decode.hip has the whole comment.
int64_t schedule(const int32_t* lengths, int64_t batch, int64_t workgroups, int64_t max_item,
                 int64_t tile, bool graph, int32_t* work, int64_t capacity, int32_t* merge,
                 int64_t* share_out, int32_t* wg = nullptr, int64_t wg_capacity = 0,
                 int64_t* wgs_out = nullptr);

// A batch for the shared plan. Requests hold consecutive query tokens, whose positions are the last
// of their keys.
struct SharedBatch {
  int64_t batch;
  const int32_t* q_start;    // [batch + 1] first query token of each request
  const int32_t* kv_len;     // [batch] keys, the query tokens' own among them
  const int32_t* page_base;  // [batch] first page entry of each request in the packed indices
  const int32_t* group_rows; // [groups]
  const int32_t* group_lens; // [groups] leading keys that a group's requests share
  int64_t groups;
  // us that the plain kernels are estimated to take; a plan that is estimated no quicker does not run.
  double plain_us = std::numeric_limits<double>::infinity();
};

// nullptr, or why the groups are refused. cached[r]: keys of request r that may be shared.
const char* check_groups(const int32_t* group_rows, const int32_t* group_lens, int64_t groups,
                         int64_t batch, const int32_t* cached, const char* too_long);

enum class SharedFit { kRuns, kPlain, kError };  // kPlain: the plain kernels are to run the batch

class SharedPlan {
 public:
  SharedPlan(int64_t cus, int64_t num_q_heads, int64_t num_kv_heads, int64_t page_size,
             int64_t dtype);
  ~SharedPlan();
  // Whether computing the shared prefixes of such a batch once beats the plain kernels.
  bool pays(const SharedBatch& b) const;
  // Plans, on the host. kPlain: no quicker than plain_us, partial outputs of more than most_partials(), or
  // no memory for them. Graph plans (graph_rows > 0: as many requests of one token and up to graph_tokens
  // keys) hold room for any groups and launch the same grids whatever is shared; they are never kPlain.
  // kError, and false of upload(): mi355x_attn_error says why.
  SharedFit prepare(const SharedBatch& b, int64_t graph_rows, int64_t graph_tokens,
                    uint64_t& allocations);
  // Lays out what prepare() planned for the same batch, beside what the stream runs meanwhile, and sends
  // it. The plan runs from then on.
  bool upload(const SharedBatch& b, hipStream_t s);
  const char* run(const int32_t* indices, const void* q, int64_t q_sn, int64_t q_sh, const void* k,
                  const void* v, void* out, int64_t o_sn, int64_t o_sh, hipStream_t s) const;
  void info(int64_t* out4) const;

 private:
  struct State;
  std::unique_ptr<State> st_;
};

}  // namespace mi355x
