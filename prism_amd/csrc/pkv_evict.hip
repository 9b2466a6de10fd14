// Eviction of the keys that attention weighed least (pkv_evict): per layer, sequence and KV head, which of the cached
// tokens stay, and their way to the front of the sequence's pages.
//
// Two launches.  The first finds each head's threshold, a radix descent over the weights' bits (no sort: what stays is
// a set, and is written in the order of positions), writes the kept positions and moves the weights.  The second moves
// K and V.  In place and in order: kept position k[d] goes to d <= k[d], and a chunk of destinations [c, c + C) never
// holds a source of a later chunk (k[d] >= d >= c + C), so one workgroup that reads a whole chunk before it writes it
// needs no other care, and may have read the next chunk by then.
#include "pkv_common.h"

namespace pkv {
namespace {

struct EvictParams {
  uint16_t* k;
  uint16_t* v;
  float* w;
  const int32_t* bt;
  const int32_t* lens;
  const int32_t* keeps;
  int32_t* kept;
  int32_t* status;
  int64_t k_layer, page_stride, w_layer, w_page, bt_stride;
  int batch, n_kv, log2_page, num_pages, max_blocks, max_keep, first, recent;
};

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;

// A sequence's sizes, read by every workgroup that works for it.
struct Sizes {
  int n, keep, first, recent;  // keep < n: something goes
  bool bad;
};
__device__ __forceinline__ Sizes sizes_of(const EvictParams& p, int b) {
  Sizes s;
  s.n = p.lens[b];
  const int keep = p.keeps[b];
  s.bad = s.n < 0 || keep < 0 || s.n > (int64_t(p.max_blocks) << p.log2_page) || min(s.n, keep) > p.max_keep;
  s.keep = min(s.n, keep);
  s.first = min(p.first, s.keep);
  s.recent = min(p.recent, s.keep - s.first);
  return s;
}

// Weights in an order that unsigned integers compare: larger floats are larger, -0 is 0, a NaN is above +inf (whatever
// its sign: as torch sorts it).
__device__ __forceinline__ uint32_t ordered(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams p) {
  constexpr int BITS = 11, BINS = 1 << BITS;
  __shared__ int hist[BINS];
  __shared__ int wave_sum[kSelectWaves];
  __shared__ int found_bin, found_above;
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Sizes s = sizes_of(p, b);
  int32_t* kept = p.kept + ((int64_t(layer) * p.batch + b) * p.n_kv + h) * p.max_keep;
  const int32_t* bt = p.bt + b * p.bt_stride;
  bool bad = s.bad;
  if (!bad) {
    const int pages = (s.n + (1 << p.log2_page) - 1) >> p.log2_page;
    for (int c = tid; c < pages; c += kSelectThreads) bad |= unsigned(bt[c]) >= unsigned(p.num_pages);
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) flag_status(p.status, PKV_STATUS_BAD_PAGE);
    for (int d = tid; d < p.max_keep; d += kSelectThreads) kept[d] = -1;
    return;
  }
  for (int d = s.keep + tid; d < p.max_keep; d += kSelectThreads) kept[d] = -1;
  if (s.keep == s.n) {
    for (int d = tid; d < s.n; d += kSelectThreads) kept[d] = d;
    return;
  }
  float* const w = p.w + layer * p.w_layer + (int64_t(h) << p.log2_page);
  const int in_page = (1 << p.log2_page) - 1;
  auto place = [&](int t) -> float* { return w + bt[t >> p.log2_page] * p.w_page + (t & in_page); };
  const int lo = s.first, hi = s.n - s.recent;  // whose weights decide
  int need = s.keep - s.first - s.recent;       // how many of them stay
  // the need-th largest key, digit by digit; `need` becomes how many of those equal to it stay
  uint32_t threshold = 0xffffffffu;
  if (need > 0) {
    threshold = 0;
    for (int shift = 32; shift > 0;) {
      const int bits = min(BITS, shift);
      shift -= bits;
      for (int i = tid; i < BINS; i += kSelectThreads) hist[i] = 0;
      __syncthreads();
      const uint32_t above_mask = shift + bits == 32 ? 0 : ~0u << (shift + bits);
      for (int t = lo + tid; t < hi; t += kSelectThreads) {
        const uint32_t key = ordered(*place(t));
        if ((key & above_mask) == threshold) atomicAdd(&hist[(key >> shift) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      // counts from the top: thread i has two bins, largest digits first
      const int top = (1 << bits) - 1 - 2 * tid;
      const int c0 = top >= 0 ? hist[top] : 0, c1 = top >= 1 ? hist[top - 1] : 0;
      int run = c0 + c1;
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(run, o);
        if (lane >= o) run += up;
      }
      if (lane == 63) wave_sum[wave] = run;
      __syncthreads();
      int before = run - c0 - c1;
      for (int i = 0; i < wave; ++i) before += wave_sum[i];
      if (before < need && before + c0 >= need) {
        found_bin = top;
        found_above = before;
      } else if (before + c0 < need && before + c0 + c1 >= need) {
        found_bin = top - 1;
        found_above = before + c0;
      }
      __syncthreads();
      threshold |= uint32_t(found_bin) << shift;
      need -= found_above;
    }
  }
  // in the order of positions: what lies above the threshold, and the first `need` that equal it
  int above = 0, equal = 0;  // so far
  for (int t0 = 0; t0 < s.n; t0 += kSelectThreads) {
    const int t = t0 + tid;
    const float f = t < s.n ? *place(t) : 0.0f;
    const bool middle = t >= lo && t < hi;
    const uint32_t key = ordered(f);
    const bool is_above = t < s.n && (!middle || (s.keep > s.first + s.recent && key > threshold));
    const bool is_equal = middle && s.keep > s.first + s.recent && key == threshold;
    const uint64_t a = __ballot(is_above), e = __ballot(is_equal), below = (uint64_t(1) << lane) - 1;
    if (lane == 0) wave_sum[wave] = __popcll(a) << 16 | __popcll(e);
    __syncthreads();  // and every weight of this chunk is read
    int packed = 0, all = 0;
    for (int i = 0; i < kSelectWaves; ++i) {
      if (i == wave) packed = all;
      all += wave_sum[i];
    }
    const int my_above = above + (packed >> 16) + __popcll(a & below);
    const int my_equal = equal + (packed & 0xffff) + __popcll(e & below);
    if (is_above || (is_equal && my_equal < need)) {
      const int d = my_above + min(my_equal, need);
      kept[d] = t;
      if (d != t) *place(d) = f;
    }
    above += all >> 16;
    equal += all & 0xffff;
    __syncthreads();
  }
}

// One workgroup moves `PART` 16-byte chunks of every kept row of K or of V of one head.
template <int THREADS, int U>
__global__ __launch_bounds__(THREADS) void evict_move_kernel(const EvictParams p, int chunks, int log2_part) {
  const int parts = chunks >> log2_part;
  const int stream = blockIdx.x % (2 * parts), b = blockIdx.y, layer = blockIdx.z, h = blockIdx.x / (2 * parts);
  const Sizes s = sizes_of(p, b);
  if (s.bad || s.keep == s.n) return;
  const int32_t* kept = p.kept + ((int64_t(layer) * p.batch + b) * p.n_kv + h) * p.max_keep;
  const int32_t* bt = p.bt + b * p.bt_stride;
  const int lane_chunk = threadIdx.x & ((1 << log2_part) - 1), row = threadIdx.x >> log2_part;
  const int rows = THREADS >> log2_part;  // a pass
  uint16_t* const base = (stream < parts ? p.k : p.v) + layer * p.k_layer +
                         (h * chunks + (stream % parts << log2_part) + lane_chunk) * 8;
  const int64_t key_st = int64_t(p.n_kv) * chunks * 8;
  const int in_page = (1 << p.log2_page) - 1;
  auto place = [&](int t) { return base + bt[t >> p.log2_page] * p.page_stride + (t & in_page) * key_st; };
  // nothing before the first evicted position moves: kept[d] == d up to there
  int d0 = 0;
  for (int end = s.keep; d0 < end;) {
    const int mid = (d0 + end) >> 1;
    if (kept[mid] == mid)
      d0 = mid + 1;
    else
      end = mid;
  }
  if (d0 >= s.keep || kept[0] < 0) return;
  u32x4 now[U];
  for (int c = d0; c < s.keep; c += U * rows) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int d = c + u * rows + row;
      if (d < s.keep) now[u] = ld16(place(kept[d]));
    }
    __syncthreads();  // every source of the chunk is read
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int d = c + u * rows + row;
      if (d < s.keep) st16(place(d), now[u]);
    }
  }
}

}  // namespace
}  // namespace pkv

extern "C" int pkv_evict(void* k_pool, void* v_pool, int64_t layer_stride, int64_t cache_page_stride, float* weights,
                         int64_t weights_layer_stride, int64_t weights_page_stride, const int32_t* block_table,
                         int64_t bt_stride, const int32_t* seq_lens, const int32_t* keep_lens, int32_t* kept,
                         int32_t layers, int32_t batch, int32_t n_kv, int32_t head_dim, int32_t page_size,
                         int32_t num_pages, int32_t max_blocks, int32_t max_keep, int32_t first, int32_t recent,
                         int32_t* status, void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_evict";
  if (layers < 0 || max_keep < 0 || first < 0 || recent < 0)
    return fail(PKV_EINVAL, "%s: bad sizes layers=%d max_keep=%d first=%d recent=%d", fn, layers, max_keep, first, recent);
  int rc = validate_paged(fn, k_pool, v_pool, cache_page_stride, block_table, bt_stride, seq_lens, batch, n_kv, head_dim,
                          page_size, num_pages, max_blocks);
  if (rc) return rc;
  if (!weights || !keep_lens || (max_keep > 0 && !kept)) return fail(PKV_EINVAL, "%s: null argument", fn);
  if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(kept)) & 3u)
    return fail(PKV_EINVAL, "%s: weights/kept not 4-byte aligned", fn);
  if (layer_stride % 8 || weights_page_stride < int64_t(n_kv) * page_size)
    return fail(PKV_EINVAL, "%s: layer stride not 16-byte aligned, or the weights' pages overlap", fn);
  if (layers > 65535 || batch > 65535) return fail(PKV_EINVAL, "%s: layers/batch exceed the grid limit", fn);
  if (layers == 0 || batch == 0 || max_keep == 0) return PKV_OK;
  EvictParams p;
  p.k = static_cast<uint16_t*>(k_pool);
  p.v = static_cast<uint16_t*>(v_pool);
  p.w = weights;
  p.bt = block_table;
  p.lens = seq_lens;
  p.keeps = keep_lens;
  p.kept = kept;
  p.status = status;
  p.k_layer = layer_stride;
  p.page_stride = cache_page_stride;
  p.w_layer = weights_layer_stride;
  p.w_page = weights_page_stride;
  p.bt_stride = bt_stride;
  p.batch = batch;
  p.n_kv = n_kv;
  p.log2_page = ilog2(page_size);
  p.num_pages = num_pages;
  p.max_blocks = max_blocks;
  p.max_keep = max_keep;
  p.first = first;
  p.recent = recent;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  evict_select_kernel<<<dim3(n_kv, batch, layers), kSelectThreads, 0, s>>>(p);
  const int chunks = head_dim / 8;
  evict_move_kernel<1024, 4><<<dim3(n_kv * 2, batch, layers), 1024, 0, s>>>(p, chunks, ilog2(chunks));
  return check_launch(fn);
}
