// Attention over prefixes that several requests of a batch share (shared.hip): what the decode and
// prefill plans need of it.
#pragma once

#include <cstdint>
#include <vector>

#include "common.h"

namespace mi355x {

constexpr int kSharedTile = 64;          // keys of a tile: shared lengths are cut to whole tiles
constexpr int kSharedItemInts = 12;      // ints of a work item
constexpr int kSharedInfoInts = 8;       // ints of a request for the merge
constexpr int kSharedHeaderInts = 4;     // {number of work items, 0, 0, 0}
constexpr int64_t kSharedRecord = 32 * 128;  // floats of a record: 32 rows' partial outputs
constexpr int32_t kNoHorizon = 1 << 30;  // queries that see every key of their range
constexpr int64_t kSharedMaxKeys = int64_t(1) << 22;

// Query rows (the tokens' heads under one kv head, heads fastest) against a range of key tiles.
struct SharedSource {
  int32_t token0, tokens;        // query tokens, consecutive
  int32_t page_base;             // index of the keys' first page entry
  int32_t tile_begin, tile_end;  // key tiles
  int32_t pos0;                  // position of token0, whose query sees keys <= pos0 (kNoHorizon)
  int32_t kv_len;                // keys there are
  int32_t splits, record, row_tiles;  // set by schedule_shared: parts along the keys, first record,
                                      // 32-row tiles of a head
};

// Waves of a workgroup for these sources: 8 (256 rows) or 4 (128 rows, two workgroups a CU).
int shared_waves(const std::vector<SharedSource>& sources, int64_t group);

// Work items and records that schedule_shared needs at most.
struct SharedCapacity {
  int64_t items, records;
};
SharedCapacity shared_capacity(const std::vector<SharedSource>& sources, int64_t group,
                               int64_t num_kv_heads, int64_t cus, int nw);
// The same for any grouping of `rows` requests of one token each.
SharedCapacity shared_decode_capacity(int64_t rows, int64_t group, int64_t num_kv_heads,
                                      int64_t cus, int nw);

// Cuts the sources into work items (kSharedItemInts each, appended to `work`); returns the records.
int64_t schedule_shared(std::vector<SharedSource>& sources, int64_t group, int64_t num_kv_heads,
                        int64_t cus, int nw, const SharedCapacity& cap,
                        std::vector<int32_t>& work);

// Tokens of every group's prefix that are worth computing once: whole tiles, 0 where not.
// limit[r]: keys of request r that may be shared. Returns whether any group shares some.
bool shared_lengths(const int32_t* group_rows, const int32_t* group_lens, int64_t groups,
                    const int32_t* limit, int64_t num_kv_heads, std::vector<int32_t>& eff);

struct SharedArgs {
  const uint16_t* q;
  int64_t q_sn, q_sh;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* header;   // kSharedHeaderInts
  const int4* work;
  const int32_t* indices;
  float* part_o;           // [record][kSharedRecord] normalised outputs, lanes' own order
  float* part_lse;         // [record][32] log2-sum-exp
  int32_t group, num_kv_heads, page_size;
  float scale_log2;
};

struct SharedMergeArgs {
  uint16_t* out;
  int64_t o_sn, o_sh;
  int64_t rows;            // tokens * q heads
  const int4* info;        // two a request: {record, splits, row_tiles, token0} of the shared part
                           // and of the request's own (splits 0: none)
  const int32_t* row_of;   // request of a token; NULL: its own number
  const float* part_o;
  const float* part_lse;
  const int32_t* own_merge;   // decode: per request {first partial, count} of its own part, whose
  const float* own_o;         // partials are [partial][q head][128] ...
  const float* own_lse;       // ... and [partial][q head]
  int32_t num_q_heads, group, num_kv_heads;
};

const char* launch_shared(const SharedArgs& a, int64_t dtype, int nw, int64_t grid,
                          hipStream_t s);
const char* launch_shared_merge(const SharedMergeArgs& a, int64_t dtype, hipStream_t s);

}  // namespace mi355x
