// Drawing the next tokens (pkv_sample): temperature, top-k, top-p, min-p and the draw from a given uniform number.
//
// With w_i = exp((x_i - max x) / T) and the tokens in the order (x descending, token ascending): the first k stay; of
// those the shortest prefix whose weights sum to top_p of theirs; of those the ones with w_i >= min_p.  Each rule keeps
// a prefix of that order, so nothing has to be sorted: what stays is all that lies before one place in it.  The drawn token is the
// first, in the order of the vocabulary, at which the running sum of the weights that stay passes u times their sum.
//
// Two launches.  The first has a workgroup per slice of a row: its maximum, the sum of its weights (fp64, from its own
// maximum on) and, where a rule is set, a list of its largest tokens.  The second has a workgroup per row, which finds
// the place among the lists where they hold it (all above the largest token that any slice left out), else among the
// row's logits themselves, by a radix descent over sums in 64-bit integers.
//
// A decision can fall between tokens 1e-6 of the sum apart, so the weights are taken in fp64 and their sums are fp64 in
// a fixed order or integers (2^-42 of the largest weight or finer): no order of atomics changes a token.
#include <algorithm>
#include <cmath>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kSliceThreads = 256;
constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kListMax = 8192;   // tokens that a row's lists hold together
constexpr int kSlicesMax = 512;
constexpr int kBins = 2048;
constexpr int kBinBits = 11;

struct SliceHead {
  uint64_t best;   // (ordered value, ~token) of the largest, 0: no token of the slice can be drawn
  double sum;      // of the weights, relative to the slice's own maximum
  uint32_t count;  // listed tokens
  uint32_t left;   // the largest ordered value among those not listed, 0: every one is
  uint32_t valid;  // tokens that can be drawn
  uint32_t pad;
};

struct Setting {
  const void* rows;  // one value a row, or NULL: `all`
  double all;
};

struct SampleParams {
  const void* logits;
  const float* uniforms;
  int64_t* tokens;
  float* logprobs;
  SliceHead* heads;
  uint2* lists;  // (ordered value, token)
  Setting temperature, top_k, top_p, min_p;
  int64_t stride;
  int vocab, slices, cap;
};

// What a row asks for.
struct Rules {
  double scale;  // log2 e / T
  double top_p, min_p;
  int top_k;     // 0: off
  bool greedy, use_p, use_m;
  __device__ __forceinline__ bool filtered() const { return top_k > 0 || use_p || use_m; }
  // the weights of the whole row are summed: to draw from, or for top-p's share
  __device__ __forceinline__ bool summed() const { return !greedy && top_k == 0 && (use_p || !use_m); }
};

__device__ __forceinline__ double setting(const Setting& s, int row) {
  return s.rows ? double(static_cast<const float*>(s.rows)[row]) : s.all;
}
__device__ __forceinline__ Rules rules_of(const SampleParams& p, int row) {
  Rules r;
  const double t = setting(p.temperature, row);
  r.greedy = !(t > 0.0);
  r.scale = 1.4426950408889634 / t;
  const int k = p.top_k.rows ? static_cast<const int32_t*>(p.top_k.rows)[row] : int(p.top_k.all);
  r.top_k = k > 0 && k < p.vocab ? k : 0;
  if (r.top_k == 1) r.greedy = true;
  r.top_p = setting(p.top_p, row);
  r.use_p = r.top_p < 1.0;
  if (r.top_p <= 0.0) r.greedy = true;
  r.min_p = fmin(setting(p.min_p, row), 1.0);
  r.use_m = r.min_p > 0.0;
  return r;
}

// Logits in an order that unsigned integers compare; 0 for one that cannot be drawn (-inf, NaN).
__device__ __forceinline__ uint32_t ordered(float f) {
  if (!(f > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return key == 0 ? -INFINITY : __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^t, t <= 0: the series of exp(f ln 2) on |f| <= 1/2 to its 11th power (6e-15), scaled by the whole part; nothing
// below 2^-1000.
__device__ __forceinline__ double exp2_neg(double t) {
  if (t < -1000.0) return 0.0;
  const double n = rint(t), f = t - n;
  double r = 4.4455382718708114e-10;
  r = fma(r, f, 7.0549116208011233e-09);
  r = fma(r, f, 1.0178086009239699e-07);
  r = fma(r, f, 1.3215486790144309e-06);
  r = fma(r, f, 1.5252733804059841e-05);
  r = fma(r, f, 1.5403530393381608e-04);
  r = fma(r, f, 1.3333558146428443e-03);
  r = fma(r, f, 9.6181291076284771e-03);
  r = fma(r, f, 5.5504108664821580e-02);
  r = fma(r, f, 2.4022650695910072e-01);
  r = fma(r, f, 6.9314718055994531e-01);
  r = fma(r, f, 1.0);
  return ldexp(r, int(n));
}

// exp((x - top) / T); an infinite top leaves weight to its equals alone.
__device__ __forceinline__ double weight_of(float x, float top, double scale) {
  if (x == top) return 1.0;
  if (!(x > -INFINITY) || top == INFINITY) return 0.0;
  return exp2_neg((double(x) - double(top)) * scale);
}

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__bf16 v) { return float(v); }
template <>
__device__ __forceinline__ float to_float(_Float16 v) { return float(v); }

// A row as 16-byte pieces from the 16-byte boundary at or before its start on (a piece that holds any of the row lies
// in the row's own allocation, whose start and size are multiples of 16 bytes at least): element j of them is token j - skip.
template <class T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const u32x4* pieces;
  int skip, vocab;
  __device__ __forceinline__ Row(const SampleParams& p, int row) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<const T*>(p.logits) + row * p.stride);
    pieces = reinterpret_cast<const u32x4*>(at & ~uintptr_t(15));
    skip = int(at & 15) / int(sizeof(T));
    vocab = p.vocab;
  }
  // piece i's values, -inf outside the row
  __device__ __forceinline__ void get(int i, float (&x)[kVec]) const {
    const int first = i * kVec - skip;
    if (first >= vocab || first + kVec <= 0) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] = -INFINITY;
      return;
    }
    struct alignas(16) Values {
      T v[kVec];
    };
    const Values v = __builtin_bit_cast(Values, pieces[i]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float f = to_float(v.v[e]);
      x[e] = unsigned(first + e) < unsigned(vocab) && f == f ? f : -INFINITY;
    }
  }
};

__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = max(x, uint64_t(__shfl_xor((unsigned long long)x, o)));
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// ---- a slice of a row ----
// Which of 1024 classes by the distance from the slice's maximum: 32 to the octave, from 2^-12 to 2^20.
__device__ __forceinline__ int distance_bin(float x, float top) {
  if (x == top) return 0;
  const int b = int(__float_as_uint(top - x) >> 18) - (115 * 32 - 1);
  return min(max(b, 0), 1023);
}

template <class T, int E>
__global__ __launch_bounds__(kSliceThreads) void sample_slice_kernel(const SampleParams p) {
  constexpr int V = Row<T>::kVec, L = E / V, W = kSliceThreads / 64;
  __shared__ uint64_t best_lds[W];
  __shared__ double sum_lds[W];
  __shared__ int hist[1024];
  __shared__ int count_lds[W], taken, bins_lds[2];
  __shared__ uint32_t left_lds[W];
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Rules rules = rules_of(p, row);
  const Row<T> src(p, row);
  float x[L][V];
  const int piece0 = slice * (kSliceThreads * L);
#pragma unroll
  for (int l = 0; l < L; ++l) src.get(piece0 + l * kSliceThreads + tid, x[l]);
  auto token = [&](int l, int e) { return (piece0 + l * kSliceThreads + tid) * V + e - src.skip; };
  uint64_t best = 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t key = ordered(x[l][e]);
      if (key > uint32_t(best >> 32)) best = uint64_t(key) << 32 | uint32_t(~token(l, e));
    }
  // of equal values the lowest token: a thread meets its own in ascending order, other threads' are compared by ~token
  best = wave_max(best);
  if (lane == 0) best_lds[wave] = best;
  for (int i = tid; i < 1024; i += kSliceThreads) hist[i] = 0;
  if (tid == 0) taken = 0;
  if (tid < 2) bins_lds[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) best = max(best, best_lds[i]);
  const float top = value_of(uint32_t(best >> 32));
  SliceHead* const head = p.heads + int64_t(row) * p.slices + slice;
  if (rules.greedy || best == 0) {
    if (tid == 0) *head = SliceHead{best, 0.0, 0, 0, 0, 0};
    return;
  }
  double sum = 0.0;
  if (rules.summed()) {
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int e = 0; e < V; ++e) sum += weight_of(x[l][e], top, rules.scale);
    sum = wave_sum(sum);
    if (lane == 0) sum_lds[wave] = sum;
  }
  int valid = 0;
  if (rules.filtered()) {
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (x[l][e] > -INFINITY) {
          ++valid;
          atomicAdd(&hist[distance_bin(x[l][e], top)], 1);
        }
  }
  __syncthreads();
  sum = 0.0;
  if (rules.summed())
#pragma unroll
    for (int i = 0; i < W; ++i) sum += sum_lds[i];
  if (!rules.filtered()) {
    if (tid == 0) *head = SliceHead{best, sum, 0, 0, 0, 0};
    return;
  }
  // how many classes fit the list, and how many hold the first top_k
  int c[4], run = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[i] = hist[tid * 4 + i];
    run += c[i];
  }
  int upto = run;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(upto, o);
    if (lane >= o) upto += up;
  }
  if (lane == 63) count_lds[wave] = upto;
  __syncthreads();
  int before = upto - run;
  for (int i = 0; i < wave; ++i) before += count_lds[i];
  int fit = 0, less = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    before += c[i];
    fit += before <= p.cap;
    less += before < rules.top_k;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    fit += __shfl_xor(fit, o);
    less += __shfl_xor(less, o);
  }
  if (lane == 0) {
    atomicAdd(&bins_lds[0], fit);
    atomicAdd(&bins_lds[1], less);
  }
  __syncthreads();
  int bins = bins_lds[0];
  if (rules.top_k > 0) bins = min(bins, bins_lds[1] + 1);
  uint2* const list = p.lists + (int64_t(row) * p.slices + slice) * p.cap;
  uint32_t left = 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t key = ordered(x[l][e]);
      if (key == 0) continue;
      if (distance_bin(x[l][e], top) < bins)
        list[atomicAdd(&taken, 1)] = uint2{key, uint32_t(token(l, e))};
      else
        left = max(left, key);
    }
  left = uint32_t(wave_max(uint64_t(left)));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) valid += __shfl_xor(valid, o);
  __syncthreads();
  if (lane == 0) {
    left_lds[wave] = left;
    count_lds[wave] = valid;
  }
  __syncthreads();
  if (tid == 0) {
    valid = 0;
    for (int i = 0; i < W; ++i) {
      left = max(left, left_lds[i]);
      valid += count_lds[i];
    }
    *head = SliceHead{best, sum, uint32_t(taken), left, uint32_t(valid), 0};
  }
}

// ---- a row ----
struct RowShared {
  uint64_t hist[kBins];
  uint64_t wave[kRowWaves];
  double wave_d[kRowWaves];
  uint64_t found_before, found_value;
  int found_bin;
  int n;
  double total, target;
  int slice, token;
};

// The first place of a descending order at which the running sum of values reaches `target` (1 or more, and the sum
// of all is no less): digit by digit from the top, f(add) calls add(sort key, value) for every element.
struct Place {
  uint32_t key;
  uint64_t left;   // of the target, at that key
  uint64_t value;  // of all elements of that key
};
template <class F>
__device__ Place descend(RowShared& sh, int bits_total, uint64_t target, F&& f) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t key = 0;
  Place out = {0, target, 0};
  for (int shift = bits_total; shift > 0;) {
    const int bits = min(kBinBits, shift);
    shift -= bits;
    for (int i = tid; i < kBins; i += kRowThreads) sh.hist[i] = 0;
    __syncthreads();
    const uint32_t done = shift + bits >= 32 ? 0u : ~0u << (shift + bits);
    f([&](uint32_t k, uint64_t v) {
      if ((k & done) == key && v > 0)
        atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(k >> shift) & ((1u << bits) - 1)]), (unsigned long long)v);
    });
    __syncthreads();
    const int at = (1 << bits) - 1 - 2 * tid;  // this thread's two bins, from the top
    const uint64_t v0 = at >= 0 ? sh.hist[at] : 0, v1 = at >= 1 ? sh.hist[at - 1] : 0;
    uint64_t run = v0 + v1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t up = __shfl_up((unsigned long long)run, o);
      if (lane >= o) run += up;
    }
    if (lane == 63) sh.wave[wave] = run;
    __syncthreads();
    uint64_t before = run - v0 - v1;
    for (int i = 0; i < wave; ++i) before += sh.wave[i];
    if (before < out.left && before + v0 >= out.left) {
      sh.found_bin = at;
      sh.found_before = before;
      sh.found_value = v0;
    } else if (before + v0 < out.left && before + v0 + v1 >= out.left) {
      sh.found_bin = at - 1;
      sh.found_before = before + v0;
      sh.found_value = v1;
    }
    __syncthreads();
    key |= uint32_t(sh.found_bin) << shift;
    out.left -= sh.found_before;
    out.value = sh.found_value;
  }
  out.key = key;
  __syncthreads();
  return out;
}

__device__ __forceinline__ uint64_t block_sum(RowShared& sh, uint64_t x) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor((unsigned long long)x, o);
  if (lane == 0) sh.wave[wave] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) x += sh.wave[i];
  __syncthreads();
  return x;
}

// Where in the order (value descending, token ascending) the last token that stays lies.
struct Cut {
  uint32_t key, token;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t t) const { return k > key || (k == key && t <= token); }
};
constexpr int kTokenBits = 20;
constexpr uint32_t kTokenMask = (1u << kTokenBits) - 1;

// The shortest prefix, within `cut`, whose values sum to `target`.
template <class Source, class Value>
__device__ Cut cut_at(RowShared& sh, const Source& src, Cut cut, uint64_t target, Value&& value) {
  const Place at = descend(sh, 32, target, [&](auto&& add) {
    src.each([&](uint32_t k, uint32_t t, auto&& w) {
      if (cut.keeps(k, t)) add(k, value(w));
    });
  });
  // of the tokens with that very value, all of one weight, the lowest
  uint64_t one = 0;
  src.each([&](uint32_t k, uint32_t t, auto&& w) {
    if (k == at.key && cut.keeps(k, t)) one = value(w);
  });
  uint64_t m = one;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max(m, uint64_t(__shfl_xor((unsigned long long)m, o)));
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = m;
  __syncthreads();
  one = 0;
  for (int i = 0; i < kRowWaves; ++i) one = max(one, sh.wave[i]);
  __syncthreads();
  const uint64_t ties = at.value / one, stay = (at.left + one - 1) / one;
  if (stay >= ties) return {at.key, cut.key == at.key ? cut.token : kTokenMask};
  const Place last = descend(sh, kTokenBits, stay, [&](auto&& add) {
    src.each([&](uint32_t k, uint32_t t, auto&&) {
      if (k == at.key && cut.keeps(k, t)) add(kTokenMask - t, 1);
    });
  });
  return {at.key, kTokenMask - last.key};
}

struct Drawn {
  uint32_t token;
  double total;  // of the weights that stay
};

// The rules and the draw over a source of (ordered value, token, weight in units of 2^-bits of the largest).
// row_total: the whole row's weights (only where no top-k limits it).
template <class Source>
__device__ Drawn choose(RowShared& sh, const Source& src, const Rules& r, double row_total, uint64_t valid, double u, int bits) {
  const double unit = ldexp(1.0, bits);
  Cut cut = {0, kTokenMask};
  if (r.top_k > 0 && uint64_t(r.top_k) < valid) cut = cut_at(sh, src, cut, uint64_t(r.top_k), [](auto&&) { return uint64_t(1); });
  if (r.use_p) {
    uint64_t here = 0;
    src.each([&](uint32_t k, uint32_t t, auto&& w) {
      if (cut.keeps(k, t)) here += w();
    });
    here = block_sum(sh, here);
    const double share = r.top_p * (r.top_k > 0 ? double(here) : row_total * unit);
    const uint64_t target = max(uint64_t(ceil(share)), uint64_t(1));
    if (target < here) cut = cut_at(sh, src, cut, target, [](auto&& w) { return w(); });
  }
  const uint64_t least = r.use_m ? max(uint64_t(r.min_p * unit), uint64_t(1)) : 1;
  uint64_t total = 0;
  src.each([&](uint32_t k, uint32_t t, auto&& w) {
    if (cut.keeps(k, t)) {
      const uint64_t v = w();
      if (v >= least) total += v;
    }
  });
  total = block_sum(sh, total);
  const uint64_t below = min(uint64_t(fmin(fmax(u, 0.0), 1.0) * double(total)), total - 1);
  const Place at = descend(sh, kTokenBits, below + 1, [&](auto&& add) {
    src.each([&](uint32_t k, uint32_t t, auto&& w) {
      if (cut.keeps(k, t)) {
        const uint64_t v = w();
        if (v >= least) add(kTokenMask - t, v);
      }
    });
  });
  return {min(kTokenMask - at.key, uint32_t(src.vocab - 1)), double(total) / unit};
}

struct ListSource {
  const uint32_t* keys;
  const uint32_t* tokens;
  const uint64_t* weights;
  int n, vocab;
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    for (int i = threadIdx.x; i < n; i += kRowThreads) f(keys[i], tokens[i], [&] { return weights[i]; });
  }
};

template <class T>
struct RowSource {
  Row<T> row;
  float top;
  double scale, unit;
  int pieces, vocab;
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    constexpr int V = Row<T>::kVec;
    for (int i = threadIdx.x; i < pieces; i += kRowThreads) {
      float x[V];
      row.get(i, x);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t key = ordered(x[e]);
        if (key != 0)
          f(key, uint32_t(i * V + e - row.skip), [&] { return uint64_t(weight_of(x[e], top, scale) * unit + 0.5); });
      }
    }
  }
};

template <class T>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(const SampleParams p, int slice_size) {
  __shared__ RowShared sh;
  __shared__ uint32_t list_keys[kListMax], list_tokens[kListMax];
  __shared__ uint64_t list_weights[kListMax];
  __shared__ uint64_t best_lds[kRowWaves];
  __shared__ uint32_t left_lds[kRowWaves], valid_lds[kRowWaves];
  __shared__ double slice_sums[kSlicesMax];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Rules rules = rules_of(p, row);
  const Row<T> src(p, row);
  const SliceHead* heads = p.heads + int64_t(row) * p.slices;
  SliceHead head = {};
  if (tid < p.slices) head = heads[tid];
  uint64_t best = wave_max(head.best);
  uint32_t left = uint32_t(wave_max(uint64_t(head.left)));
  uint32_t valid = head.valid;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) valid += __shfl_xor(valid, o);
  if (lane == 0) {
    best_lds[wave] = best;
    left_lds[wave] = left;
    valid_lds[wave] = valid;
  }
  if (tid == 0) sh.n = 0;
  __syncthreads();
  valid = 0;
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) {
    best = max(best, best_lds[i]);
    left = max(left, left_lds[i]);
    valid += valid_lds[i];
  }
  const float top = value_of(uint32_t(best >> 32));
  const int best_token = int(~uint32_t(best));
  if (best == 0 || rules.greedy) {  // nothing to draw, or nothing to choose
    if (tid == 0) {
      p.tokens[row] = best == 0 ? -1 : best_token;
      if (p.logprobs) p.logprobs[row] = best == 0 ? -INFINITY : 0.0f;
    }
    return;
  }
  const double u = p.uniforms[row];
  double total = 0.0;
  if (rules.summed()) {
    if (tid < p.slices)
      slice_sums[tid] = head.best ? head.sum * weight_of(value_of(uint32_t(head.best >> 32)), top, rules.scale) : 0.0;
    __syncthreads();
    // in order, by every thread alike
    for (int i = 0; i < p.slices; ++i) total += slice_sums[i];
  }
  if (!rules.filtered()) {
    // the slice, then the token in it
    const double target = fmin(fmax(u, 0.0), 1.0) * total;
    if (tid == 0) {
      double run = 0.0;
      int at = -1;
      double at_before = 0.0;
      for (int i = 0; i < p.slices; ++i) {
        if (slice_sums[i] > 0.0) {
          at = i;
          at_before = run;
        }
        run += slice_sums[i];
        if (run > target) break;
      }
      sh.slice = at;
      sh.target = target - at_before;
      sh.token = -1;
    }
    __syncthreads();
    const int per = slice_size / kRowThreads;
    const int first = sh.slice * slice_size + tid * per - src.skip;
    double mine = 0.0;
    int last = -1;  // this thread's last token with any weight
    const T* values = static_cast<const T*>(p.logits) + row * p.stride;
    for (int e = 0; e < per; ++e)
      if (unsigned(first + e) < unsigned(p.vocab)) {
        const float x = to_float(values[first + e]);
        const double w = x == x ? weight_of(x, top, rules.scale) : 0.0;
        mine += w;
        if (w > 0.0) last = first + e;
      }
    double run = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(run, o);
      if (lane >= o) run += up;
    }
    if (lane == 63) sh.wave_d[wave] = run;
    // the sums of this order may fall short of the slice's own by their rounding: then it is the last token
    atomicMax(&sh.token, last);
    __syncthreads();
    const int fallback = sh.token;
    double before = 0.0;
    for (int i = 0; i < wave; ++i) before += sh.wave_d[i];
    before += run - mine;
    __syncthreads();
    if (tid == 0) sh.token = 0x7fffffff;
    __syncthreads();
    if (before + mine > sh.target) {
      double sum = before;
      for (int e = 0; e < per; ++e)
        if (unsigned(first + e) < unsigned(p.vocab)) {
          const float x = to_float(values[first + e]);
          const double w = x == x ? weight_of(x, top, rules.scale) : 0.0;
          sum += w;
          if (w > 0.0 && sum > sh.target) {
            atomicMin(&sh.token, first + e);
            break;
          }
        }
    }
    __syncthreads();
    if (tid == 0) {
      const int token = sh.token == 0x7fffffff ? fallback : sh.token;
      p.tokens[row] = token;
      if (p.logprobs) {
        const float x = to_float(values[token]);
        p.logprobs[row] = float((x == top ? 0.0 : (double(x) - double(top)) * rules.scale / 1.4426950408889634) - log(total));
      }
    }
    return;
  }
  // the lists, as far as they are whole: above the largest value that some slice left out
  constexpr int kListBits = 49;
  const double list_unit = ldexp(1.0, kListBits);
  uint64_t sum = 0;
  for (int s = wave; s < p.slices; s += kRowWaves) {
    const int count = min(int(heads[s].count), p.cap);
    const uint2* list = p.lists + (int64_t(row) * p.slices + s) * p.cap;
    for (int i0 = 0; i0 < count; i0 += 64) {
      const uint2 it = i0 + lane < count ? list[i0 + lane] : uint2{0, 0};
      const bool take = it.x > left;
      const uint64_t all = __ballot(take);
      int at = 0;
      if (lane == 0) at = atomicAdd(&sh.n, __popcll(all));
      at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((uint64_t(1) << lane) - 1));
      if (take && at < kListMax) {
        const uint64_t w = uint64_t(weight_of(value_of(it.x), top, rules.scale) * list_unit + 0.5);
        list_keys[at] = it.x;
        list_tokens[at] = it.y;
        list_weights[at] = w;
        sum += w;
      }
    }
  }
  sum = block_sum(sh, sum);
  const int n = min(sh.n, kListMax);
  const bool min_within = rules.use_m && weight_of(value_of(left), top, rules.scale) < rules.min_p;
  const bool whole = left == 0 ||
                     (rules.top_k > 0 ? uint32_t(n) >= uint32_t(rules.top_k) || (!rules.use_p && min_within)
                                      : (rules.use_p && double(sum) >= rules.top_p * total * list_unit) || min_within);
  Drawn got;
  if (whole) {
    got = choose(sh, ListSource{list_keys, list_tokens, list_weights, n, p.vocab}, rules, total, uint64_t(n), u, kListBits);
  } else {
    const int bits = 62 - kTokenBits;
    const int pieces = (src.skip + p.vocab + Row<T>::kVec - 1) / Row<T>::kVec;
    got = choose(sh, RowSource<T>{src, top, rules.scale, ldexp(1.0, bits), pieces, p.vocab}, rules, total, valid, u, bits);
  }
  if (tid == 0) {
    p.tokens[row] = got.token;
    if (p.logprobs) {
      const float x = to_float((static_cast<const T*>(p.logits) + row * p.stride)[got.token]);
      p.logprobs[row] = float((x == top ? 0.0 : (double(x) - double(top)) * rules.scale / 1.4426950408889634) - log(got.total));
    }
  }
}

// ---- the host side ----
struct Split {
  int elements;  // of a slice, a thread
  int slices, cap;
};
// Slices of 4096 tokens.
Split split_of(int64_t rows, int vocab, int dtype) {
  Split s;
  s.elements = vocab > 4096 * 256 - 16 ? 0 : 16;
  const int size = kSliceThreads * s.elements;
  s.slices = s.elements ? (vocab + 7 + size - 1) / size : 0;
  s.cap = s.slices ? std::min(512, kListMax / s.slices) : 0;
  return s;
}

template <class T>
void launch(const SampleParams& p, const Split& s, int rows, hipStream_t stream) {
  sample_slice_kernel<T, 16><<<dim3(s.slices, rows), kSliceThreads, 0, stream>>>(p);
  sample_row_kernel<T><<<rows, kRowThreads, 0, stream>>>(p, kSliceThreads * s.elements);
}

}  // namespace
}  // namespace pkv

extern "C" size_t pkv_sample_workspace_bytes(int32_t rows, int32_t vocab, int32_t dtype) {
  using namespace pkv;
  if (rows <= 0 || vocab <= 0) return 0;
  const Split s = split_of(rows, vocab, dtype);
  return size_t(rows) * s.slices * (sizeof(SliceHead) + size_t(s.cap) * sizeof(uint2));
}

extern "C" int pkv_sample(const void* logits, int64_t stride, int32_t dtype, const float* uniforms,
                          const float* temperatures, float temperature, const int32_t* top_ks, int32_t top_k,
                          const float* top_ps, float top_p, const float* min_ps, float min_p, int64_t* tokens,
                          float* logprobs, int32_t rows, int32_t vocab, void* workspace, size_t workspace_bytes,
                          void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_sample";
  if (rows < 0 || vocab <= 0 || vocab > 1000000)
    return fail(PKV_EINVAL, "%s: %d rows of %d tokens: a vocabulary of 1 to 1000000", fn, rows, vocab);
  if (rows > 65535) return fail(PKV_EINVAL, "%s: %d rows exceed the grid limit", fn, rows);
  if (dtype != PKV_BF16 && dtype != PKV_FP16 && dtype != PKV_FP32) return fail(PKV_EINVAL, "%s: bad dtype %d", fn, dtype);
  if (rows == 0) return PKV_OK;
  if (!logits || !uniforms || !tokens) return fail(PKV_EINVAL, "%s: null logits, uniforms or tokens", fn);
  if (rows > 1 && stride < vocab) return fail(PKV_EINVAL, "%s: rows of logits overlap", fn);
  const uintptr_t size = dtype == PKV_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return fail(PKV_EINVAL, "%s: logits not aligned to their type", fn);
  if ((reinterpret_cast<uintptr_t>(uniforms) | reinterpret_cast<uintptr_t>(temperatures) | reinterpret_cast<uintptr_t>(top_ks) |
       reinterpret_cast<uintptr_t>(top_ps) | reinterpret_cast<uintptr_t>(min_ps) | reinterpret_cast<uintptr_t>(logprobs)) & 3u)
    return fail(PKV_EINVAL, "%s: an array of 4-byte values is not aligned to them", fn);
  if (reinterpret_cast<uintptr_t>(tokens) & 7u) return fail(PKV_EINVAL, "%s: tokens not 8-byte aligned", fn);
  const size_t need = pkv_sample_workspace_bytes(rows, vocab, dtype);
  if (!workspace || !aligned16(workspace)) return fail(PKV_EINVAL, "%s: workspace null or not 16-byte aligned", fn);
  if (workspace_bytes < need)
    return fail(PKV_ENOSPC, "%s: workspace %zu bytes < %zu needed", fn, workspace_bytes, need);
  const Split s = split_of(rows, vocab, dtype);
  SampleParams p;
  p.logits = logits;
  p.uniforms = uniforms;
  p.tokens = tokens;
  p.logprobs = logprobs;
  p.heads = static_cast<SliceHead*>(workspace);
  p.lists = reinterpret_cast<uint2*>(p.heads + size_t(rows) * s.slices);
  p.temperature = {temperatures, temperature};
  p.top_k = {top_ks, double(top_k)};
  p.top_p = {top_ps, top_p};
  p.min_p = {min_ps, min_p};
  p.stride = stride;
  p.vocab = vocab;
  p.slices = s.slices;
  p.cap = s.cap;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == PKV_BF16)
    launch<__bf16>(p, s, rows, st);
  else if (dtype == PKV_FP16)
    launch<_Float16>(p, s, rows, st);
  else
    launch<float>(p, s, rows, st);
  return check_launch(fn);
}
