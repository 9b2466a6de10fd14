// Work lists of packed attention, laid out by pkv_packed_plan on the host and read by the kernels.
#pragma once

#include <stdint.h>

namespace pkv {

constexpr int kPackedRows = 128;  // query rows (token x head of the group) of a work item
// Blocks of at most so many rows, without a window, share their keys over the workgroup's four waves.
constexpr int kPackedFewRows = 16;
// Blocks of at most so many rows (one wave's) and ranges merge in the launch: the last range to end does it.
constexpr int kPackedLastRows = 32, kPackedLastRanges = 64;

// One key range of one row block of one sequence, for every KV head.  48 bytes.
struct PackedItem {
  int32_t tok0;    // the sequence's first row of q and out
  int32_t n_new;   // its new tokens
  int32_t ctx;     // its keys before them
  int32_t seq;     // its row of the block table
  int32_t row0;    // the block's first query row, new token x group size + head in the group
  int32_t stage0;  // the range's first stage (of 32 keys, head_dim 128, or 64)
  int32_t stages;
  int32_t slot;    // where its partial result goes, -1 for a block of one range
  int32_t first, count;  // the block's slots, where its ranges merge in the launch (count 0: a PackedMerge does)
  int32_t pad[2];
};

// Any other row block of several ranges: their partials are slots slot .. slot + count - 1.  32 bytes.
struct PackedMerge {
  int32_t tok0, n_new, row0, slot, count;
  int32_t pad[3];
};

}  // namespace pkv
