// Work lists of pkv_key_weights, laid out by pkv_key_weights_plan on the host and read by the kernels.
#pragma once

#include <stdint.h>

namespace pkv {

constexpr int kWeightBlock = 256;    // keys of a block that many query rows go over
// Sequences with at most so many query rows stream their keys past them.  16 sequences of 4000 keys, 28 heads on 4: 63
// rows 21 us this way and 25 by blocks of keys, 126 rows 26 and 28; 40 heads on 8: 60 rows 33 and 43, 125 rows 41 and 51.
// More rows would not fit four workgroups' LDS.
constexpr int kWeightFewRows = 128;
constexpr int kWeightFewKeys = 3968; // keys of such an item at most: a wave's page ids, one per 16 keys, fit its lanes

// Keys [key0, key0 + keys) of one sequence against query rows [row0, row0 + rows) of those that count, for every KV
// head.  48 bytes.
struct WeightItem {
  int32_t tok0;    // the first row of q and lse that counts
  int32_t n_tok;   // how many count
  int32_t pos0;    // the first one's position
  int32_t seq;     // the sequence's row of the block table
  int32_t key0, keys;
  int32_t fresh;   // keys from this one on start from nothing
  int32_t row0, rows;  // query row: new token that counts * group size + head in the group
  int32_t part;    // where its sums go, -1: to the weights.  Of a merge: its first partial
  int32_t count;   // of a merge: how many
  int32_t pad;
};

}  // namespace pkv
