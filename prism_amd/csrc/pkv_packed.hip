// Host side of packed attention: the step's work list, cut and ordered before the kernels run.
#include <algorithm>
#include <exception>
#include <vector>

#include "pkv_common.h"
#include "pkv_packed.h"

namespace pkv {
namespace {

// A range pays about two stages' time to start and one to end, and a launch that merges: see kMinStages in
// pkv_prefill.h, whose walk this is.
constexpr int kMinRange = 8;
constexpr int kWorkgroupsPerCu = 2;

struct Block {
  int seq, row0, stage0, stages;
};

int range_count(int stages, int64_t chunk) {
  return int(std::max<int64_t>(std::min<int64_t>((stages + chunk - 1) / chunk, stages / kMinRange), 1));
}

}  // namespace

// Row blocks of kPackedRows query rows, each with the stages that its rows see: up to its last row's own key, from
// its first row's window on.  `slots` ranges run at once per KV head.  With fewer blocks than slots the longest
// are cut until the card is full in one round (a range count just past the slots would cost a second round: the
// ranges are lengthened until they fit); with more, only blocks above the average slot's share are cut, so that
// none of them is what the launch ends with.  The longest go first.
static int plan_blocks(const int32_t* new_lens, const int32_t* ctx_lens, int batch, int g, int tok, int window,
                       int slots, std::vector<PackedItem>& items, std::vector<PackedMerge>& merges, int32_t* partials,
                       int32_t* merge_rows) {
  std::vector<Block> blocks;
  int64_t total = 0;
  for (int b = 0; b < batch; ++b) {
    const int rows = new_lens[b] * g, ctx = ctx_lens[b];
    for (int r0 = 0; r0 < rows; r0 += kPackedRows) {
      const int last = ctx + (std::min(r0 + kPackedRows, rows) - 1) / g;
      const int first = window > 0 ? std::max(ctx + r0 / g - window + 1, 0) : 0;
      const int stage0 = first / tok;
      blocks.push_back({b, r0, stage0, last / tok + 1 - stage0});
      total += blocks.back().stages;
    }
  }
  int64_t chunk = std::max<int64_t>((total + slots - 1) / slots, kMinRange);
  if (int64_t(blocks.size()) <= slots) {
    for (;;) {
      int64_t ranges = 0;
      for (const Block& k : blocks) ranges += range_count(k.stages, chunk);
      if (ranges <= slots) break;
      chunk += std::max<int64_t>(chunk / 16, 1);
    }
  }
  std::vector<int32_t> tok0(batch);
  int32_t t = 0;
  for (int b = 0; b < batch; ++b) {
    tok0[b] = t;
    t += new_lens[b];
  }
  *partials = 0;
  *merge_rows = 0;
  for (const Block& k : blocks) {
    const int count = range_count(k.stages, chunk);
    const int len = (k.stages + count - 1) / count;
    PackedItem it = {tok0[k.seq], new_lens[k.seq], ctx_lens[k.seq], k.seq, k.row0, k.stage0, k.stages, -1};
    if (count == 1) {
      items.push_back(it);
      continue;
    }
    int used = 0;
    for (int s = 0; s < k.stages; s += len) {
      it.stage0 = k.stage0 + s;
      it.stages = std::min(len, k.stages - s);
      it.slot = *partials + used++;
      items.push_back(it);
    }
    merges.push_back({it.tok0, it.n_new, it.row0, *partials, used, {0, 0, 0}});
    *partials += used;
    *merge_rows = std::max(*merge_rows, std::min(kPackedRows, it.n_new * g - it.row0));
  }
  std::stable_sort(items.begin(), items.end(),
                   [](const PackedItem& a, const PackedItem& b) { return a.stages > b.stages; });
  return PKV_OK;
}

}  // namespace pkv

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
  int64_t tokens = 0;
  for (int b = 0; b < batch; ++b) {
    if (new_lens[b] < 0 || ctx_lens[b] < 0 || int64_t(new_lens[b]) + ctx_lens[b] > (int64_t(1) << 27))
      return fail(PKV_EINVAL, "%s: sequence %d has %d new and %d cached tokens (0 to 2^27 in all)", fn, b, new_lens[b],
                  ctx_lens[b]);
    tokens += new_lens[b];
  }
  if (tokens * n_heads > (int64_t(1) << 30)) return fail(PKV_EINVAL, "%s: more than 2^30 query rows", fn);
  try {
    std::vector<PackedItem> it;
    std::vector<PackedMerge> mg;
    const int slots = std::max(compute_units * kWorkgroupsPerCu / n_kv, 1);
    plan_blocks(new_lens, ctx_lens, batch, g, head_dim == 128 ? 32 : 64, window, slots, it, mg, &counts[2], &counts[3]);
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
