// Host side of packed attention: the step's work list, cut and ordered before the kernels run.
#include <algorithm>
#include <exception>
#include <functional>
#include <vector>

#include "pkv_common.h"
#include "pkv_packed.h"

namespace pkv {
namespace {

// Costs in stages (of 16 KB of K and V).  A range's start and end take about five stages' time: loads of the item,
// then of Q and pages, then of the first tiles, one behind the other.  Below six stages a piece is not worth that: one
// decode token on 27 stages takes 9.4 us a call in four pieces, 11.5 in two, 14.0 whole.
constexpr int kRangeCost = 5;
constexpr int kPartialCost = 8;  // of 128 rows: 66 KB each way
constexpr int kMinRange = 6;
constexpr int kWorkgroupsPerCu = 2;

struct Block {
  int seq, row0, stage0, stages;
  int rows;
  bool few;  // its keys go round four waves
  // of each piece, where it is cut: its partial is written and read back
  int cut_cost() const { return (kPartialCost * rows + kPackedRows - 1) / kPackedRows; }
};

// Row blocks of kPackedRows query rows, each with the stages that its rows see: up to its last row's own key, from
// its first row's window on.
std::vector<Block> row_blocks(const int32_t* new_lens, const int32_t* ctx_lens, int batch, int g, int tok, int window) {
  std::vector<Block> blocks;
  for (int b = 0; b < batch; ++b) {
    const int rows = new_lens[b] * g, ctx = ctx_lens[b];
    for (int r0 = 0; r0 < rows; r0 += kPackedRows) {
      const int last = ctx + (std::min(r0 + kPackedRows, rows) - 1) / g;
      const int first = window > 0 ? std::max(ctx + r0 / g - window + 1, 0) : 0;
      blocks.push_back({b, r0, first / tok, last / tok + 1 - first / tok, std::min(kPackedRows, rows - r0),
                        window == 0 && rows - r0 <= kPackedFewRows});
    }
  }
  return blocks;
}

struct Piece {
  int block, stage0, stages;
};

// The launch as the card will run it: `slots` ranges at once per KV head, the next of the list where one ends.
struct Schedule {
  std::vector<int64_t> load;  // a heap: when each slot is free, the earliest in front
  std::vector<Piece> list;
  int64_t end = 0;  // of the last range
  explicit Schedule(int slots) : load(slots, 0) {}
  void add(const Block& b, int block, int stage0, int stages) {
    std::pop_heap(load.begin(), load.end(), std::greater<int64_t>());
    load.back() += stages + kRangeCost + (stages < b.stages ? b.cut_cost() : 0);
    end = std::max(end, load.back());
    std::push_heap(load.begin(), load.end(), std::greater<int64_t>());
    list.push_back({block, stage0, stages});
  }
};

int pieces(int stages, int64_t chunk) {
  return int(std::max<int64_t>(std::min<int64_t>((stages + chunk - 1) / chunk, stages / kMinRange), 1));
}

// The blocks longest first, in equal pieces of about `chunk` stages.
Schedule in_chunks(const std::vector<Block>& blocks, int slots, int64_t chunk) {
  Schedule s(slots);
  for (int i = 0; i < int(blocks.size()); ++i) {
    const int n = blocks[i].stages;
    const int count = pieces(n, chunk);
    const int len = (n + count - 1) / count;
    for (int at = 0; at < n; at += len) s.add(blocks[i], i, at, std::min(len, n - at));
  }
  return s;
}

// The blocks longest first, each whole where it ends by `target`, else in pieces that do.
Schedule filled(const std::vector<Block>& blocks, int slots, int64_t target) {
  Schedule s(slots);
  for (int i = 0; i < int(blocks.size()); ++i) {
    for (int at = 0, take; at < blocks[i].stages; at += take) {
      const int left = blocks[i].stages - at;
      const int64_t room = target - s.load[0] - kRangeCost;
      take = left;
      if (left > room + kMinRange / 2 && left >= 2 * kMinRange)
        take = int(std::min<int64_t>(std::max<int64_t>(room, kMinRange), left - kMinRange));
      s.add(blocks[i], i, at, take);
    }
  }
  return s;
}

// Pieces of one length, for two workgroups per CU, for one or for fewer, whichever ends soonest.  One per CU already
// reads as fast as the card does (5.8 TB/s: all CUs together 370 stages a us, 0.6 us each); two even out what the
// blocks' lengths leave uneven (in between some CUs would have one and some two), at the price of more partials: 0.4
// us per MB written and read, and 2.7 us and 0.2 per range of a block to merge them (half of that at 64 a head).
// Decode rows' stages take 0.3 us where few workgroups read, 0.45 at 128 of them.  us a call, two per CU always / so:
// 6 decode tokens and two chunks on 40 k keys (7B) 124 / 112; one decode token on 20 k keys 24 / 19, 4 on 3000 each
// 12.9 / 11.7, 8 on 500 each (not cut) 10.3 / 8.9; one KV head, two on 70 k each 37 / 28.
Schedule even(const std::vector<Block>& blocks, int slots, int n_kv, int head_dim) {
  int64_t total = 0;
  for (const Block& b : blocks) total += b.stages;
  int64_t best_chunk = 0;
  double best = 0;
  for (int64_t room = slots; room > 0; room /= 2) {
    if (int64_t(blocks.size()) > room) break;
    for (int64_t chunk = std::max<int64_t>((total + room - 1) / room, kMinRange);;
         chunk += std::max<int64_t>(chunk / 16, 1)) {
      int64_t ranges = 0, rows = 0, most = 0, longest_few = 0, longest = 0;
      for (const Block& b : blocks) {
        const int count = pieces(b.stages, chunk);
        ranges += count;
        int64_t& length = b.few ? longest_few : longest;
        length = std::max<int64_t>(length, (b.stages + count - 1) / count);
        if (count > 1) rows += int64_t(count) * b.rows;
        most = std::max<int64_t>(most, count);
      }
      if (ranges > room) continue;
      const double few_us = std::min(std::max(0.32, (head_dim == 128 ? 0.2 : 0.37) + ranges * n_kv / 512.0), 0.58);
      const double us = std::max({total * n_kv / 370.0, 0.58 * longest, few_us * longest_few}) +
                        (rows ? 2.7 + 0.0016 * head_dim * most + 0.4e-6 * rows * n_kv * (head_dim + 4) * 4 : 0.0);
      if (best_chunk == 0 || us < best) {
        best = us;
        best_chunk = chunk;
      }
      break;
    }
  }
  return in_chunks(blocks, slots, best_chunk);
}

// Whole blocks can need a round more than their work does (129 blocks of 34 stages on 64 slots, a window's, take
// three rounds for one block too many), and few blocks leave the card idle.  Two ways to cut them: pieces of one
// length that fit one round, and pieces that fill every slot up to an even share of the work.
// Up to one block per slot: one length, or, with more than half as many blocks as slots and where that schedule would
// end a tenth earlier, filled.  (Less than that is lost again: pieces that wait for a slot start into a card that reads
// as fast as it can.)  us a call, uncut / one length / filled: 47 decode tokens and two chunks (7B) 111 / 56 / 70; 6 and
// two on 40 k keys 1063 / 112 / 137; 208 short chats (0.5B) 28 / 22 / 19.
// More blocks than slots: filled or whole.  Filling goes on past the share by the price of its own cuts, in ever shorter
// pieces, and a cut costs the launch more than its slot, as the others read no faster meanwhile: about kCutWait stages of
// one slot each.  us a call, whole / filled, and what the schedules' ends alone would promise: six chunks of 1000 in a
// window of 512 (7B) 76 / 92 (1.31 of whole), four of 2048 in 2048 (0.5B) 85 / 106 (1.33), four of 700 in 1024 (14B)
// 80 / 104 (1.31); 300 decode tokens on 900 keys (7B) 107 / 114 (0.95), 64 on 2000 and three chunks (14B) 147 / 161
// (0.92); 140 decode tokens on 3000 (7B) 179 / 164 (0.58), three chunks of 700 on 8000 (14B) 424 / 382 (0.74), chunks and
// decode tokens in a window of 1024 (14B, three cuts) 107 / 96 (0.93), one decode token on 100 k keys among 1100 short
// chats (7B) 1290 / 218 (0.06), a chunk of 600 on 30 k among them 577 / 387 (0.43).  Whole blocks, longest first, end
// at most the longest past the share: where that is under one part in kRounds nothing is scheduled to see (9000 chats on
// 100 keys, 349 us of host time as the list's start alone, 483 with both schedules).
constexpr int kRounds = 8;
constexpr int kCutWait = 20;
std::vector<Piece> cut(std::vector<Block>& blocks, int slots, int n_kv, int head_dim) {
  std::stable_sort(blocks.begin(), blocks.end(), [](const Block& a, const Block& b) { return a.stages > b.stages; });
  const int64_t n = int64_t(blocks.size());
  if (n == 0) return {};
  int64_t total = 0;
  for (const Block& b : blocks) total += b.stages;
  const int64_t share = (total + kRangeCost * n + slots - 1) / slots;
  if (n <= slots) {
    Schedule best = filled(blocks, slots, share + kRangeCost);
    Schedule one = even(blocks, slots, n_kv, head_dim);
    if (n <= slots / 2 || 9 * one.end <= 10 * best.end) best = std::move(one);
    return std::move(best.list);
  }
  if (kRounds * (blocks[0].stages + kRangeCost) <= share) return in_chunks(blocks, 1, INT64_MAX / 2).list;
  Schedule best = in_chunks(blocks, slots, INT64_MAX / 2);
  Schedule full = filled(blocks, slots, share + kRangeCost);
  if ((best.end - full.end) * slots > kCutWait * (int64_t(full.list.size()) - n)) best = std::move(full);
  return std::move(best.list);
}

}  // namespace

static void plan(const int32_t* new_lens, const int32_t* ctx_lens, int batch, int g, int n_kv, int head_dim, int window,
                 int slots, std::vector<PackedItem>& items, std::vector<PackedMerge>& merges, int32_t* partials,
                 int32_t* merge_rows) {
  std::vector<Block> blocks = row_blocks(new_lens, ctx_lens, batch, g, head_dim == 128 ? 32 : 64, window);
  const std::vector<Piece> list = cut(blocks, slots, n_kv, head_dim);
  std::vector<int32_t> tok0(batch);
  for (int b = 1; b < batch; ++b) tok0[b] = tok0[b - 1] + new_lens[b - 1];
  *partials = *merge_rows = 0;
  for (size_t i = 0; i < list.size(); ++i) {  // the pieces of a block are next to each other
    const Piece& k = list[i];
    const Block& b = blocks[k.block];
    const int n_new = new_lens[b.seq];
    const bool whole = k.stages == b.stages;
    items.push_back({tok0[b.seq], n_new, ctx_lens[b.seq], b.seq, b.row0, b.stage0 + k.stage0, k.stages,
                     whole ? -1 : (*partials)++, 0, 0, {0, 0}});
    if (whole || k.stage0 + k.stages < b.stages) continue;
    // the block's last piece: its first is as many items back
    size_t first = i;
    while (list[first].stage0 > 0) --first;
    const int count = int(i - first) + 1, slot = *partials - count;
    if (b.rows <= kPackedLastRows && count <= kPackedLastRanges) {
      for (size_t j = first; j <= i; ++j) {
        items[j].first = slot;
        items[j].count = count;
      }
      continue;
    }
    merges.push_back({tok0[b.seq], n_new, b.row0, slot, count, {0, 0, 0}});
    *merge_rows = std::max(*merge_rows, b.rows);
  }
}

}  // namespace pkv

namespace pkv {
// Sequence lengths as every entry here takes them; the tokens in all, -1 where one does not fit (recorded).
static int64_t check_lengths(const char* fn, const int32_t* new_lens, const int32_t* ctx_lens, int batch) {
  int64_t tokens = 0;
  for (int b = 0; b < batch; ++b) {
    if (new_lens[b] < 0 || ctx_lens[b] < 0 || int64_t(new_lens[b]) + ctx_lens[b] > (int64_t(1) << 27)) {
      fail(PKV_EINVAL, "%s: sequence %d has %d new and %d cached tokens: not negative, and at most 2^27 together", fn, b,
           new_lens[b], ctx_lens[b]);
      return -1;
    }
    tokens += new_lens[b];
  }
  return tokens;
}
}  // namespace pkv

extern "C" int pkv_packed_layout(const int32_t* new_lens, const int32_t* ctx_lens, int32_t batch,
                                 const int32_t* block_table, int64_t bt_stride, int32_t max_blocks, int32_t page_size,
                                 int32_t num_pages, int32_t window, int32_t* positions, int32_t* slots) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_packed_layout";
  if (batch < 0 || max_blocks < 0 || bt_stride < max_blocks || window < 0)
    return fail(PKV_EINVAL, "%s: bad sizes batch=%d max_blocks=%d bt_stride=%lld window=%d", fn, batch, max_blocks,
                (long long)bt_stride, window);
  if (!is_pow2(page_size) || page_size < 16)
    return fail(PKV_EINVAL, "%s: page_size %d must be a power of two >= 16", fn, page_size);
  if (num_pages <= 0 || int64_t(num_pages) * page_size > 0x7fffffff)
    return fail(PKV_EINVAL, "%s: %d pages of %d tokens: the pool must have 1 to 2^31 - 1 slots", fn, num_pages, page_size);
  if (batch > 0 && (!new_lens || !ctx_lens || (max_blocks > 0 && !block_table)))
    return fail(PKV_EINVAL, "%s: null argument", fn);
  const int64_t tokens = check_lengths(fn, new_lens, ctx_lens, batch);
  if (tokens < 0) return PKV_EINVAL;
  if (tokens > 0 && (!positions || !slots)) return fail(PKV_EINVAL, "%s: null argument", fn);
  const int log2_page = ilog2(page_size);
  try {
    std::vector<bool> written(num_pages, false);
    int64_t t = 0;
    for (int b = 0; b < batch; ++b) {
      const int n = new_lens[b], c = ctx_lens[b];
      if (n == 0) continue;
      const int32_t* row = block_table + b * bt_stride;
      const int last = (c + n - 1) >> log2_page;
      if (last >= max_blocks)
        return fail(PKV_EINVAL, "%s: sequence %d needs %d pages, the block table has %d columns", fn, b, last + 1, max_blocks);
      for (int col = (window > 0 ? std::max(c - window + 1, 0) : 0) >> log2_page; col <= last; ++col)
        if (unsigned(row[col]) >= unsigned(num_pages))
          return fail(PKV_EINVAL, "%s: sequence %d needs block-table column %d, which lists page %d, outside [0, %d)", fn, b,
                      col, row[col], num_pages);
      for (int col = c >> log2_page; col <= last; ++col) {
        if (written[row[col]])
          return fail(PKV_EINVAL, "%s: two places of the batch write to one page, %d, sequence %d the second (the same "
                      "sequence twice, or a shared page that was not copied before the write)", fn, row[col], b);
        written[row[col]] = true;
      }
      for (int pos = c; pos < c + n; ++pos, ++t) {
        positions[t] = pos;
        slots[t] = row[pos >> log2_page] * page_size + (pos & (page_size - 1));
      }
    }
  } catch (const std::exception& e) {  // no memory: no C++ exception leaves a C entry
    return fail(PKV_EINVAL, "%s: %s", fn, e.what());
  }
  return PKV_OK;
}

extern "C" int pkv_packed_plan(const int32_t* new_lens, const int32_t* ctx_lens, int32_t batch, int32_t n_heads,
                               int32_t n_kv, int32_t head_dim, int32_t window, int32_t compute_units, int32_t* items,
                               int32_t max_items, int32_t* merges, int32_t max_merges, int32_t* counts) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_packed_plan";
  if (batch < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || window < 0 || compute_units <= 0)
    return fail(PKV_EINVAL, "%s: bad sizes batch=%d n_heads=%d n_kv=%d window=%d compute_units=%d", fn, batch, n_heads,
                n_kv, window, compute_units);
  if (head_dim != 64 && head_dim != 128) return fail(PKV_EINVAL, "%s: head_dim %d unsupported (64 or 128)", fn, head_dim);
  if ((batch > 0 && (!new_lens || !ctx_lens)) || !counts) return fail(PKV_EINVAL, "%s: null argument", fn);
  const int g = n_heads / n_kv;
  const int64_t tokens = check_lengths(fn, new_lens, ctx_lens, batch);
  if (tokens < 0) return PKV_EINVAL;
  if (tokens * n_heads > (int64_t(1) << 30)) return fail(PKV_EINVAL, "%s: more than 2^30 query rows", fn);
  try {
    std::vector<PackedItem> it;
    std::vector<PackedMerge> mg;
    const int slots = std::max(compute_units * kWorkgroupsPerCu / n_kv, 1);
    plan(new_lens, ctx_lens, batch, g, n_kv, head_dim, window, slots, it, mg, &counts[2], &counts[3]);
    counts[0] = int32_t(it.size());
    counts[1] = int32_t(mg.size());
    if (!items) return PKV_OK;
    if (counts[0] > max_items || counts[1] > max_merges || (counts[1] > 0 && !merges))
      return fail(PKV_ENOSPC, "%s: %d items and %d merges do not fit %d and %d", fn, counts[0], counts[1], max_items,
                  max_merges);
    std::copy(it.begin(), it.end(), reinterpret_cast<PackedItem*>(items));
    std::copy(mg.begin(), mg.end(), reinterpret_cast<PackedMerge*>(merges));
  } catch (const std::exception& e) {  // no memory: no C++ exception leaves a C entry
    return fail(PKV_EINVAL, "%s: %s", fn, e.what());
  }
  return PKV_OK;
}
