// Eviction of the keys that attention weighed least (pkv_evict): per layer, sequence and KV head, which of the cached
// tokens stay, and their way to the front of the sequence's pages.
//
// Two launches.  The first finds each head's threshold, a radix descent over the weights' bits (no sort: what stays is
// a set, and is written in the order of positions), writes the kept positions and moves the weights.  The second moves
// K and V, in place: the token at position k[d] goes to d <= k[d].
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
  int32_t* marks;  // per layer, sequence, head and K or V: a ticket, then a flag for each workgroup of the second launch
  int32_t* status;
  int64_t k_layer, page_stride, w_layer, w_page, bt_stride;
  int batch, n_kv, log2_page, num_pages, max_blocks, max_keep, first, recent, move_chunks;
};

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

// Four at once: sums of exponentials are as they should be, not negative and no NaN.
__device__ __forceinline__ void ordered4(f32x4 x, uint32_t (&key)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(x[i]);
  const bool fine = max(max(u[0], u[1]), max(u[2], u[3])) <= 0x7f800000u;
#pragma unroll
  for (int i = 0; i < 4; ++i) key[i] = u[i] | 0x80000000u;
  if (!fine) {
#pragma unroll
    for (int i = 0; i < 4; ++i) key[i] = ordered(x[i]);
  }
}

// Sums of a wave up to each lane: within rows of 16, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_from(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_running_sum(int x) {
  x = add_from<0x111, 0xf>(x);  // the lane before, two, four, eight before
  x = add_from<0x112, 0xf>(x);
  x = add_from<0x114, 0xf>(x);
  x = add_from<0x118, 0xf>(x);
  x = add_from<0x142, 0xa>(x);         // lane 15 of the row before, into rows 1 and 3
  return add_from<0x143, 0xc>(x);      // lane 31, into rows 2 and 3
}

// The place from the top of a histogram of 2^bits counts where the running sum reaches `need`.
template <int THREADS>
struct Digit {
  int hist[2048];
  int wave_sum[THREADS / 64], chunk_sum[2][THREADS / 64];
  int bin, above, count;
};
template <int THREADS>
__device__ __forceinline__ void find_digit(Digit<THREADS>& sh, int bits, int need) {
  constexpr int PER = 2048 / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int top = (1 << bits) - 1 - PER * tid;  // this thread's bins, from the top
  int c[PER], mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    c[i] = top >= i ? sh.hist[top - i] : 0;
    mine += c[i];
  }
  const int run = wave_running_sum(mine);
  if (lane == 63) sh.wave_sum[wave] = run;
  __syncthreads();
  int before = run - mine;
  for (int i = 0; i < wave; ++i) before += sh.wave_sum[i];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < need && before + c[i] >= need) {
      sh.bin = top - i;
      sh.above = before;
      sh.count = c[i];
    }
    before += c[i];
  }
  __syncthreads();
}

// A workgroup per layer, sequence and head.  Reads the weights three times (first digit; the keys of that digit, which
// then lie in LDS where CANDIDATES hold them; the kept ones), 16 bytes a lane with the next ones on the way.  What bounds
// it is its one CU, whose vector ALU is busy 63 %, and whose waves wait half of their time: 28 layers' one head of 105 k
// tokens take 66 us on 28 of 256 CUs, 0.9 us for 4096 weights and pass; 28 layers of 6 sequences of 2800 tokens with 4
// heads, which fill the device, 19 us.  More workgroups to a head would need four launches, and the move of K and V
// behind it is the longer one already (110 and 206 us).
// COLS: a sequence's row of the block table lies in LDS (0: not), as it does up to 8192 columns.  From global memory the
// long eviction takes 14 us more, those of six sequences the same.
template <int THREADS, int COLS, int CANDIDATES>
__global__ __launch_bounds__(THREADS) void evict_select_kernel(const EvictParams p) {
  constexpr bool TABLE = COLS > 0;
  constexpr int WAVES = THREADS / 64;
  __shared__ Digit<THREADS> sh;
  __shared__ int table[TABLE ? COLS : 1];
  __shared__ __align__(16) uint32_t keys[CANDIDATES];  // later what stays of a chunk, twice
  static_assert(CANDIDATES >= 2 * 2 * 4 * THREADS, "two chunks of pairs");
  __shared__ int candidates;
  const int h = blockIdx.x, b = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Sizes s = sizes_of(p, b);
  const int64_t head = (int64_t(layer) * p.batch + b) * p.n_kv + h;
  int32_t* kept = p.kept + head * p.max_keep;
  // the second launch's tickets and flags
  for (int i = tid; i < 2 * (1 + p.move_chunks); i += THREADS) p.marks[head * 2 * (1 + p.move_chunks) + i] = 0;
  const int32_t* bt = p.bt + b * p.bt_stride;
  bool bad = s.bad;
  if (!bad) {
    const int pages = (s.n + (1 << p.log2_page) - 1) >> p.log2_page;
    for (int c = tid; c < pages; c += THREADS) {
      const int page = bt[c];
      bad |= unsigned(page) >= unsigned(p.num_pages);
      if constexpr (TABLE) table[c] = page;
    }
  }
  if (tid == 0) candidates = 0;
  if (__syncthreads_or(bad)) {
    if (tid == 0) flag_status(p.status, PKV_STATUS_BAD_PAGE);
    for (int d = tid; d < p.max_keep; d += THREADS) kept[d] = -1;
    return;
  }
  for (int d = s.keep + tid; d < p.max_keep; d += THREADS) kept[d] = -1;
  if (s.keep == s.n) {
    for (int d = tid; d < s.n; d += THREADS) kept[d] = d;
    return;
  }
  float* const w = p.w + layer * p.w_layer + (int64_t(h) << p.log2_page);
  const int in_page = (1 << p.log2_page) - 1;
  auto place = [&](int t) -> float* {
    const int col = t >> p.log2_page;
    int page;
    if constexpr (TABLE)
      page = table[col];
    else
      page = bt[col];
    return w + page * p.w_page + (t & in_page);
  };
  const int lo = s.first, hi = s.n - s.recent;  // whose weights decide
  int need = s.keep - s.first - s.recent;       // how many of them stay
  const bool choose = need > 0;
  // f(four keys, whether all of them count) for every group of four tokens some of whose weights decide, 0 for those that
  // do not; a batch of loads is on its way while the one before it is worked on
  constexpr int kUnroll = 4, kStride = THREADS * 4;
  auto each = [&](auto&& f) {
    f32x4 next[kUnroll];
    auto load = [&](int t0) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (t0 + u * kStride < s.n) next[u] = *reinterpret_cast<const f32x4*>(place(t0 + u * kStride));
    };
    load(tid * 4);
    for (int t0 = tid * 4; t0 < s.n; t0 += kUnroll * kStride) {
      f32x4 x[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) x[u] = next[u];
      load(t0 + kUnroll * kStride);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int t = t0 + u * kStride;
        if (t + 3 < lo || t >= hi) continue;
        uint32_t key[4];
        ordered4(x[u], key);
        const bool whole = t >= lo && t + 3 < hi;
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (t + i < lo || t + i >= hi) key[i] = 0;
        }
        f(key, whole);
      }
    }
  };
  // the need-th largest key, digit by digit; `need` becomes how many of those equal to it stay
  uint32_t threshold = 0xffffffffu;
  if (choose) {
    threshold = 0;
    bool listed = false;
    int n_listed = 0;
    for (int shift = 32; shift > 0;) {
      const int bits = min(11, shift);
      shift -= bits;
      for (int i = tid; i < 2048; i += THREADS) sh.hist[i] = 0;
      __syncthreads();
      const uint32_t done = shift + bits == 32 ? 0 : ~0u << (shift + bits), mask = (1u << bits) - 1;
      if (listed) {
        for (int i = tid; i < n_listed; i += THREADS)
          if ((keys[i] & done) == threshold) atomicAdd(&sh.hist[(keys[i] >> shift) & mask], 1);
      } else {
        each([&](const uint32_t (&key)[4], bool whole) {
          if (done == 0 && whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) atomicAdd(&sh.hist[key[i] >> 21], 1);
            return;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key[i] != 0 && (key[i] & done) == threshold) atomicAdd(&sh.hist[(key[i] >> shift) & mask], 1);
        });
      }
      __syncthreads();
      find_digit(sh, bits, need);
      threshold |= uint32_t(sh.bin) << shift;
      need -= sh.above;
      n_listed = sh.count;
      if (!listed && shift > 0 && n_listed <= CANDIDATES) {
        listed = true;
        const uint32_t upto = ~0u << shift;
        each([&](const uint32_t (&key)[4], bool whole) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((key[i] & upto) == threshold && (whole || key[i] != 0)) keys[atomicAdd(&candidates, 1)] = key[i];
        });
      }
      __syncthreads();
      if (listed) n_listed = candidates;
    }
  }
  // in the order of positions: what lies above the threshold, and the first `need` that equal it.  A kept weight moves to
  // d <= t: never to where a later chunk's lie, and this chunk's are in registers by then.
  constexpr int kAhead = 4;  // chunks on their way
  int above = 0, equal = 0;  // so far
  f32x4 next[kAhead];
  auto load = [&](int j, int t) {
    if (t < s.n) next[j] = *reinterpret_cast<const f32x4*>(place(t));
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j) load(j, tid * 4 + j * kStride);
  for (int base = 0; base < s.n; base += kAhead * kStride) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (base + j * kStride >= s.n) break;
      const int t = base + j * kStride + tid * 4;
      const f32x4 x = next[j];
      load(j, t + kAhead * kStride);
      // without a choice (need 0) the threshold is above every key but NaN's, and none of those equal to it stay
      uint32_t key[4], is_above = 0, is_equal = 0;
      ordered4(x, key);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        is_above |= uint32_t(key[i] > threshold) << i;
        is_equal |= uint32_t(key[i] == threshold) << i;
      }
      if (t < lo || t + 3 >= hi) {
        const uint32_t inside = t + 3 < s.n ? 15 : t < s.n ? (1u << (s.n - t)) - 1 : 0;
        uint32_t middle = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) middle |= uint32_t(t + i >= lo && t + i < hi) << i;
        is_above = (is_above & middle) | (inside & ~middle);
        is_equal &= middle;
      }
      const int mine = __popc(is_above) << 16 | __popc(is_equal), run = wave_running_sum(mine);
      int* const sums = sh.chunk_sum[j & 1];  // the other one may still be read
      if (lane == 63) sums[wave] = run;
      __syncthreads();
      const int waves = wave_running_sum(lane < WAVES ? sums[lane] : 0);  // up to each of them
      const int all = __builtin_amdgcn_readlane(waves, WAVES - 1);
      const int before = (wave > 0 ? __builtin_amdgcn_readlane(waves, wave - 1) : 0) + run - mine;
      int my_above = above + (before >> 16), my_equal = equal + (before & 0xffff);
      const int start = above + min(equal, need);
      uint2* const stage = reinterpret_cast<uint2*>(keys) + (j & 1) * kStride;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool a = is_above >> i & 1, e = is_equal >> i & 1;
        if (a || (e && my_equal < need))
          stage[my_above + min(my_equal, need) - start] = uint2{uint32_t(t + i), __float_as_uint(x[i])};
        my_above += a;
        my_equal += e;
      }
      above += all >> 16;
      equal += all & 0xffff;
      const int count = above + min(equal, need) - start;
      __syncthreads();
      for (int i = tid; i < count; i += THREADS) {
        const uint2 it = stage[i];
        const int d = start + i;
        kept[d] = int(it.x);
        if (d != int(it.x)) *place(d) = __uint_as_float(it.y);
      }
    }
  }
}

// Which of them: a workgroup of 1024 threads has its CU to itself (137 KB of LDS), of 256 a CU holds six.  So these take
// tables of up to 4096 tokens where there are more heads than CUs, and of up to 1024 always.  Evictions as a whole, by
// 1024 threads and by 256: 4608 heads of 150 tokens 238 and 126 us, of 2000 1083 and 975, 672 heads of 4000 320 and 309,
// 112 of 4000 62 and 67, 48 of 1000 21 and 20, of 2000 the same.  512 threads are between the two.
constexpr int kManyTokens = 4096, kFewTokens = 1024, kManyHeads = 256;
bool short_tables(int64_t tokens, int64_t heads) { return tokens <= (heads > kManyHeads ? kManyTokens : kFewTokens); }

// ---- K and V ----
// A workgroup takes 32 KB of destination rows of K or of V of one head: it reads their sources, and writes them once the
// sources that lie in its destinations have been read by the workgroups that they belong to.  Those have smaller
// destinations (k[d] >= d), and a workgroup's place in that order is a ticket that it draws when it starts: whoever it
// waits for has started, reads without waiting for anybody, and then raises its flag.  So every wait ends, whatever
// else runs on the device.  Bounds: HBM, by bytes read and written.  28 layers of 6 sequences of 2800 tokens cut in half
// (968 MB of K and V): 205 us, 4.7 TB/s, where a copy reaches 4.9; one of 105 k tokens cut to 14 k: 110 us, 3.7 TB/s, its
// sources are 256 bytes here and there.
template <int U>
__global__ __launch_bounds__(256) void evict_move_kernel(const EvictParams p, int log2_chunks) {
  __shared__ int ticket_lds, wait_lds[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int stream = blockIdx.x / p.move_chunks, b = blockIdx.y, layer = blockIdx.z, h = stream >> 1;
  const Sizes s = sizes_of(p, b);
  const int rows = 256 >> log2_chunks;  // a pass of the workgroup
  const int per = rows * U;
  if (s.bad || s.keep == s.n || int(blockIdx.x % p.move_chunks) * per >= s.keep) return;  // as many as the kept rows need go on
  const int64_t head = (int64_t(layer) * p.batch + b) * p.n_kv + h;
  const int32_t* kept = p.kept + head * p.max_keep;
  int32_t* const marks = p.marks + (head * 2 + (stream & 1)) * (1 + p.move_chunks);
  if (tid == 0) {
    ticket_lds = atomicAdd(&marks[0], 1);
    wait_lds[0] = wait_lds[1] = -1;
  }
  __syncthreads();
  const int mine = ticket_lds, d0 = mine * per, d1 = min(d0 + per, s.keep);
  const int last = kept[d1 - 1];
  if (last < 0 || last == d1 - 1) return;  // refused by the first launch, or all in place (nobody else reads these slots)
  const int32_t* bt = p.bt + b * p.bt_stride;
  const int chunk = tid & ((1 << log2_chunks) - 1), row = tid >> log2_chunks;
  const int64_t key_st = int64_t(p.n_kv) << (log2_chunks + 3);
  uint16_t* const base = (stream & 1 ? p.v : p.k) + layer * p.k_layer + (((h << log2_chunks) + chunk) << 3);
  const int in_page = (1 << p.log2_page) - 1;
  auto place = [&](int t) { return base + bt[t >> p.log2_page] * p.page_stride + (t & in_page) * key_st; };
  int from[U];
  u32x4 x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) from[u] = kept[min(d0 + u * rows + row, d1 - 1)];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u] = ld16(place(from[u]));
  // meanwhile: the destinations [a, b) whose sources lie in this workgroup's, 64 places tried at once.  At most `per`
  // of them, so they belong to two workgroups at most.
  if (wave < 2) {
    const int want = wave == 0 ? d0 : d1;
    int lo = 0, hi = d1;  // the first d with kept[d] >= want lies in [lo, hi] (kept[d] >= d)
    while (lo < hi) {
      const int step = (hi - lo + 63) >> 6;
      const int at = min(lo + (lane + 1) * step - 1, hi - 1);
      const int less = __popcll(__ballot(kept[at] < want && lo + (lane + 1) * step - 1 < hi));
      const int next = min(lo + less * step, hi);
      hi = min(next + step - 1, hi);
      lo = next;
      if (step == 1) {
        hi = lo;
      }
    }
    if (lane == 0) wait_lds[wave] = lo;
  }
  __syncthreads();
  const int a = wait_lds[0], e = wait_lds[1];
  // the loads have arrived
#pragma unroll
  for (int u = 0; u < U; ++u) asm volatile("" ::"v"(x[u]));
  __syncthreads();
  if (tid == 0) {
    __hip_atomic_store(&marks[1 + mine], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (e > a)
      for (int i = a / per; i <= min((e - 1) / per, mine - 1); ++i)
        while (__hip_atomic_load(&marks[1 + i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0) __builtin_amdgcn_s_sleep(1);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int d = d0 + u * rows + row;
    if (d < d1 && from[u] != d) st16(place(d), x[u]);
  }
}

// Rows of 16 bytes a thread: 32 KB a workgroup.  With 16 KB the two evictions above take 240 and 182 us in all, with 32
// 214 and 167, with 64 222 and 164; a chat's (1700 tokens, 24 layers of two heads of 64) 28, 28 and 30.
constexpr int kMoveUnroll = 8;
int move_chunks(int max_keep, int head_dim) {
  const int per = 256 / (head_dim / 8) * kMoveUnroll;
  return (max_keep + per - 1) / per;
}

}  // namespace
}  // namespace pkv

extern "C" size_t pkv_evict_workspace_bytes(int32_t layers, int32_t batch, int32_t n_kv, int32_t head_dim, int32_t max_keep) {
  if (layers <= 0 || batch <= 0 || n_kv <= 0 || max_keep <= 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return size_t(layers) * batch * n_kv * 2 * (1 + pkv::move_chunks(max_keep, head_dim)) * sizeof(int32_t);
}

extern "C" int pkv_evict(void* k_pool, void* v_pool, int64_t layer_stride, int64_t cache_page_stride, float* weights,
                         int64_t weights_layer_stride, int64_t weights_page_stride, const int32_t* block_table,
                         int64_t bt_stride, const int32_t* seq_lens, const int32_t* keep_lens, int32_t* kept,
                         int32_t layers, int32_t batch, int32_t n_kv, int32_t head_dim, int32_t page_size,
                         int32_t num_pages, int32_t max_blocks, int32_t max_keep, int32_t first, int32_t recent,
                         void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_evict";
  if (layers < 0 || max_keep < 0 || first < 0 || recent < 0)
    return fail(PKV_EINVAL, "%s: bad sizes layers=%d max_keep=%d first=%d recent=%d", fn, layers, max_keep, first, recent);
  int rc = validate_paged(fn, k_pool, v_pool, cache_page_stride, block_table, bt_stride, seq_lens, batch, n_kv, head_dim,
                          page_size, num_pages, max_blocks);
  if (rc) return rc;
  if (!weights || !keep_lens || (max_keep > 0 && !kept)) return fail(PKV_EINVAL, "%s: null argument", fn);
  if (!aligned16(weights) || weights_layer_stride % 4 || weights_page_stride % 4)
    return fail(PKV_EINVAL, "%s: weights or their strides not 16-byte aligned", fn);
  if (reinterpret_cast<uintptr_t>(kept) & 3u) return fail(PKV_EINVAL, "%s: kept not 4-byte aligned", fn);
  if (layer_stride % 8 || weights_page_stride < int64_t(n_kv) * page_size)
    return fail(PKV_EINVAL, "%s: layer stride not 16-byte aligned, or the weights' pages overlap", fn);
  if (layers > 65535 || batch > 65535) return fail(PKV_EINVAL, "%s: layers/batch exceed the grid limit", fn);
  if (layers == 0 || batch == 0 || max_keep == 0) return PKV_OK;
  const size_t need = pkv_evict_workspace_bytes(layers, batch, n_kv, head_dim, max_keep);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3u))
    return fail(PKV_EINVAL, "%s: workspace null or not 4-byte aligned", fn);
  if (workspace_bytes < need) return fail(PKV_ENOSPC, "%s: workspace %zu bytes < %zu needed", fn, workspace_bytes, need);
  const int64_t wgs = int64_t(n_kv) * 2 * move_chunks(max_keep, head_dim);
  if (wgs * 256 > 0x7fffffff) return fail(PKV_EINVAL, "%s: %d heads of %d kept tokens exceed the grid limit", fn, n_kv, max_keep);
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
  p.marks = static_cast<int32_t*>(workspace);
  p.move_chunks = move_chunks(max_keep, head_dim);
  const dim3 heads(n_kv, batch, layers);
  if (short_tables(int64_t(max_blocks) << p.log2_page, int64_t(n_kv) * batch * layers))
    evict_select_kernel<256, kManyTokens / 16, kManyTokens><<<heads, 256, 0, s>>>(p);
  else if (max_blocks <= 8192)
    evict_select_kernel<1024, 8192, 24576><<<heads, 1024, 0, s>>>(p);
  else
    evict_select_kernel<1024, 0, 24576><<<heads, 1024, 0, s>>>(p);
  evict_move_kernel<kMoveUnroll><<<dim3(unsigned(wgs), batch, layers), 256, 0, s>>>(p, ilog2(head_dim / 8));
  return check_launch(fn);
}
