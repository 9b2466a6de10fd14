// Drawing the next tokens (pkv_sample): temperature, top-k, top-p, min-p and the draw from a given uniform number.
//
// With w_i = exp((x_i - max x) / T) and the tokens in the order (x descending, token ascending): the first k stay; of
// those the shortest prefix whose weights sum to top_p of theirs; of those the ones with w_i >= min_p.  Each rule keeps
// a prefix of that order, so nothing has to be sorted: what stays is all that lies before one place in it.  The drawn
// token is the first, in the order of the vocabulary, at which the running sum of the weights that stay passes u times
// their sum.
//
// Two launches, three where some rows have top-k and some do not.  The first has a workgroup per slice of a row: its
// maximum and what the row's rules need of it.
//   no rule:          the sum of its weights
//   top-p or min-p:   the running sums of its weights over classes of value, 1/16 octave of weight each
//   top-k:            a list of its largest tokens
// The second has a workgroup per row.  It joins the slices, finds the place where the order is cut (among the few
// tokens of one class, or on the lists), then the slice that the draw falls into, and reads that one again.  Rows whose
// cut lies in none of these (thousands of equal logits, top-k past the lists) are searched through by a radix descent
// over all their tokens.
//
// The first launch is bound by fp64, an exponential a token: 256 plain fp32 rows of 131072 take 30 us (134 MB, 4.5 TB/s),
// 32 bf16 rows of 151003 with top-p 13.  The second by the latency of its steps, one workgroup a row: plain rows 13 us,
// top-p 33 (2 to join the slices' heads, 2 their sums, 5 the classes, 10 to read the row for the cut class, 4 to sort it,
// 5 to draw), top-k 11 for one row of 32000, 24 for 60 of 128000 with settings of their own.
//
// A decision can fall between tokens 1e-6 of the sum apart, so the weights are taken in fp64 and their sums are fp64 in
// a fixed order or integers (2^-42 of the largest weight or finer): no order of atomics changes a token.
#include <algorithm>
#include <cmath>

#include "pkv_common.h"

namespace pkv {
namespace {

constexpr int kSliceThreads = 256;
// In slices of 8192, 256 plain rows of 131072 take 54 us, not 46, 32 of 151003 with top-p 52, not 49.
constexpr int kSlice = 16 * kSliceThreads;
constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kListMax = 8192;   // tokens that a row's lists hold together
constexpr int kSlicesMax = 256;
constexpr int kBins = 2048;
constexpr int kBinBits = 11;
constexpr int kClasses = 512;    // of value, kPerOctave to the octave of weight
constexpr double kPerOctave = 16.0;
constexpr int kClassBits = 50;   // the classes' sums are in units of 2^-50 of the slice's reference

struct SliceHead {
  uint64_t best;   // (ordered value, ~token) of the largest, 0: no token of the slice can be drawn.  The token for
                   // greedy rows alone
  double sum;      // no rule: of the weights, relative to the slice's own maximum.  Classes: of all, in their units
  double ref;      // classes: the octave that they count from
  uint32_t count;  // listed tokens
  uint32_t left;   // the largest ordered value among those not listed, 0: every one is
  uint32_t valid;  // tokens that can be drawn
  uint32_t pad[3];
};

struct Setting {
  const void* rows;  // one value a row, or NULL: `all`
  double all;
};
constexpr double kLog2e = 1.4426950408889634;

struct SampleParams {
  const void* logits;
  const float* uniforms;
  int64_t* tokens;
  float* logprobs;
  SliceHead* heads;
  void* lists;  // a slice's part: `cap` tokens as (ordered value, token), or kClasses running sums
  Setting temperature, top_k, top_p, min_p;
  double scale;  // log2 e / T, where T is one number
  int64_t stride;
  int vocab, slices, cap;
  int64_t part;  // bytes of a slice's part
};

// What a row asks for.
struct Rules {
  double scale;  // log2 e / T
  double top_p, min_p;
  int top_k;     // 0: off
  bool greedy, use_p, use_m;
  __device__ __forceinline__ bool lists() const { return !greedy && top_k > 0; }
  __device__ __forceinline__ bool classes() const { return !greedy && top_k == 0 && (use_p || use_m); }
};

__device__ __forceinline__ double setting(const Setting& s, int row) {
  return s.rows ? double(static_cast<const float*>(s.rows)[row]) : s.all;
}
__device__ __forceinline__ Rules rules_of(const SampleParams& p, int row) {
  Rules r;
  const double t = setting(p.temperature, row);
  r.greedy = !(t > 0.0);
  r.scale = p.temperature.rows ? kLog2e / t : p.scale;
  const int k = p.top_k.rows ? static_cast<const int32_t*>(p.top_k.rows)[row] : int(p.top_k.all);
  r.top_k = k > 0 && k < p.vocab ? k : 0;
  if (r.top_k == 1) r.greedy = true;
  r.top_p = setting(p.top_p, row);
  r.use_p = r.top_p < 1.0;
  if (r.top_p <= 0.0) r.greedy = true;
  const double m = setting(p.min_p, row);
  r.use_m = m > 0.0;  // not a NaN: a setting that is none takes nothing away
  r.min_p = fmin(m, 1.0);
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

// 2^t for -1000 <= t <= 60: on |f| <= 1/2 the polynomial of degree 9 through the Chebyshev points (3e-14), its exponent
// raised by the whole part, which t + 1.5 * 2^52 has rounded into its lowest bits.
__device__ __forceinline__ double exp2_within(double t) {
  constexpr double kWhole = 6755399441055744.0;
  const double n = t + kWhole, f = t - (n - kWhole);
  double r = 1.0209419265549968e-07;
  r = fma(r, f, 1.3259628068862384e-06);
  r = fma(r, f, 1.5252653613517797e-05);
  r = fma(r, f, 1.5403433825801269e-04);
  r = fma(r, f, 1.3333558236151045e-03);
  r = fma(r, f, 9.6181291938355444e-03);
  r = fma(r, f, 5.5504108664411090e-02);
  r = fma(r, f, 2.4022650695640746e-01);
  r = fma(r, f, 6.9314718055995062e-01);
  r = fma(r, f, 1.0);
  return __hiloint2double(__double2hiint(r) + (__double2loint(n) << 20), __double2loint(r));
}
// The same, nothing below 2^-1000.
__device__ __forceinline__ double exp2_of(double t) { return t < -1000.0 ? 0.0 : exp2_within(t); }
// A weight of at most 2^51 units as an integer, rounded by the sum's last place.
__device__ __forceinline__ uint64_t whole(double units) {
  return uint64_t(__double_as_longlong(units + 4503599627370496.0)) & 0xfffffffffffffull;
}

// exp((x - top) / T); an infinite top leaves weight to its equals alone.
__device__ __forceinline__ double weight_of(float x, float top, double scale) {
  if (x == top) return 1.0;
  if (!(x > -INFINITY) || top == INFINITY) return 0.0;
  return exp2_of((double(x) - double(top)) * scale);
}

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__bf16 v) { return float(v); }
template <>
__device__ __forceinline__ float to_float(_Float16 v) { return float(v); }

// The same where no maximum of the row is known yet: x / T in octaves, from a reference octave at or above the
// largest (with +inf, whose equals alone weigh anything, one that leaves nothing to any other).
__device__ __forceinline__ double octave_of(float top, double scale) {
  return top == INFINITY ? 1e300 : ceil(double(top) * scale);
}
__device__ __forceinline__ double octaves_below(float x, double ref, double scale) {  // 0 or less; -1e300: no weight
#pragma clang fp contract(off)  // the same bits wherever it is computed, and 0 for a product that is whole
  if (!(x > -INFINITY)) return -1e300;
  if (x == INFINITY) return 0.0;
  const double octaves = double(x) * scale;
  return fmin(octaves - ref, 0.0);
}
__device__ __forceinline__ int class_of(double t) { return int(fmin(-t * kPerOctave, 1e9)); }

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
  // piece i as it is, its values whatever they are outside the row
  __device__ __forceinline__ u32x4 raw(int i) const {
    const int first = i * kVec - skip;
    return first < vocab && first + kVec > 0 ? pieces[i] : u32x4{};
  }
  __device__ __forceinline__ static float value(const u32x4& v, int e) {
    struct alignas(16) Values {
      T v[kVec];
    };
    return to_float(__builtin_bit_cast(Values, v).v[e]);
  }
  // whether pieces [i, i + n) lie in the row with all they hold
  __device__ __forceinline__ bool inside(int i, int n) const {
    return i * kVec >= skip && (i + n) * kVec - skip <= vocab;
  }
  // piece i's values, -inf outside the row and for NaN
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

// Lane l's partner l ^ MASK, without a way through LDS.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, 0xf, 0xf, true));
}
template <int MASK>
__device__ __forceinline__ uint32_t across(uint32_t x) {
  if constexpr (MASK == 1) return moved<0xb1>(x);            // quad 1 0 3 2
  if constexpr (MASK == 2) return moved<0x4e>(x);            // quad 2 3 0 1
  if constexpr (MASK == 4) return moved<0x141>(moved<0x1b>(x));  // within eight: 7 - l of quad 3 2 1 0
  if constexpr (MASK == 8) return moved<0x128>(x);           // a row of 16 turned by 8
  if constexpr (MASK == 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return __lane_id() & 16 ? a[0] : a[1];
  }
  if constexpr (MASK == 32) {
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __lane_id() & 32 ? a[0] : a[1];
  }
}
template <int MASK>
__device__ __forceinline__ uint64_t across(uint64_t x) {
  return uint64_t(across<MASK>(uint32_t(x >> 32))) << 32 | across<MASK>(uint32_t(x));
}
template <int MASK>
__device__ __forceinline__ float across(float x) {
  return __uint_as_float(across<MASK>(__float_as_uint(x)));
}
__device__ __forceinline__ float wave_top(float x) {
  x = fmaxf(x, across<1>(x));
  x = fmaxf(x, across<2>(x));
  x = fmaxf(x, across<4>(x));
  x = fmaxf(x, across<8>(x));
  x = fmaxf(x, across<16>(x));
  return fmaxf(x, across<32>(x));
}
template <int MASK>
__device__ __forceinline__ double across(double x) {
  return __longlong_as_double(int64_t(across<MASK>(uint64_t(__double_as_longlong(x)))));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = max(x, uint64_t(__shfl_xor((unsigned long long)x, o)));
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
  x += across<32>(x);
  x += across<16>(x);
  x += across<8>(x);
  x += across<4>(x);
  x += across<2>(x);
  return x + across<1>(x);
}

// ---- a slice of a row ----
// Which of 1024 classes by the distance from the slice's maximum: 32 to the octave, from 2^-12 to 2^20.
__device__ __forceinline__ int distance_bin(float x, float top) {
  if (x == top) return 0;
  const int b = int(__float_as_uint(top - x) >> 18) - (115 * 32 - 1);
  return min(max(b, 0), 1023);
}

// PLAIN: no row has a rule (the settings are numbers, and none of them is one).
template <class T, int E, bool PLAIN>
__global__ __launch_bounds__(kSliceThreads) void sample_slice_kernel(const SampleParams p) {
  constexpr int V = Row<T>::kVec, L = E / V, W = kSliceThreads / 64;
  __shared__ uint64_t low_lds[W], classes[PLAIN ? 1 : kClasses], total_lds[W];
  __shared__ double sum_lds[W];
  __shared__ float top_lds[W];
  __shared__ int hist[PLAIN ? 1 : 1024];
  __shared__ int count_lds[W], taken, bins_lds[2];
  __shared__ uint32_t left_lds[W];
  const int slice = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row<T> src(p, row);
  float x[L][V];
  const int piece0 = slice * (kSliceThreads * L);
  if (src.inside(piece0, kSliceThreads * L)) {
    u32x4 raw[L];
#pragma unroll
    for (int l = 0; l < L; ++l) raw[l] = src.pieces[piece0 + l * kSliceThreads + tid];
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int e = 0; e < V; ++e) x[l][e] = fmaxf(Row<T>::value(raw[l], e), -INFINITY);  // NaN to -inf
  } else {
#pragma unroll
    for (int l = 0; l < L; ++l) src.get(piece0 + l * kSliceThreads + tid, x[l]);
  }
  const Rules rules = rules_of(p, row);
  auto token = [&](int l, int e) { return (piece0 + l * kSliceThreads + tid) * V + e - src.skip; };
  float top = -INFINITY;
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int e = 0; e < V; ++e) top = fmaxf(top, x[l][e]);
  top = wave_top(top);
  if (lane == 0) top_lds[wave] = top;
  if constexpr (!PLAIN) {
    if (rules.lists())
      for (int i = tid; i < 1024; i += kSliceThreads) hist[i] = 0;
    else if (rules.classes())
      for (int i = tid; i < kClasses; i += kSliceThreads) classes[i] = 0;
    if (tid == 0) taken = rules.greedy ? 0x7fffffff : 0;
    if (tid < 2) bins_lds[tid] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) top = fmaxf(top, top_lds[i]);
  SliceHead* const head = p.heads + int64_t(row) * p.slices + slice;
  char* const part = static_cast<char*>(p.lists) + (int64_t(row) * p.slices + slice) * p.part;
  if (top == -INFINITY) {
    if (tid == 0) *head = SliceHead{0, 0.0, 0.0, 0, 0, 0, {}};
    return;
  }
  uint64_t best = uint64_t(ordered(top)) << 32;
  if (!PLAIN && rules.greedy) {
    // of equal values the lowest token
    int first = 0x7fffffff;
#pragma unroll
    for (int l = L - 1; l >= 0; --l)
#pragma unroll
      for (int e = V - 1; e >= 0; --e)
        if (x[l][e] == top) first = token(l, e);
    if (first != 0x7fffffff) atomicMin(&taken, first);
    __syncthreads();
    if (tid == 0) *head = SliceHead{best | uint32_t(~taken), 0.0, 0.0, 0, 0, 0, {}};
    return;
  }
  if (PLAIN || (!rules.lists() && !rules.classes())) {
    double sum = 0.0;
    const double bias = -double(top) * rules.scale;
    if (rules.scale > 0.0 && fabs(bias) < 1e6) {  // rounded to 2^-33 of an octave at most, for all of the slice alike
      // -inf comes out as 2^-1000 of the slice's own largest: nothing
#pragma unroll
      for (int l = 0; l < L; ++l)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += exp2_within(fmax(fma(double(x[l][e]), rules.scale, bias), -1000.0));
    } else {
#pragma unroll
      for (int l = 0; l < L; ++l)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += weight_of(x[l][e], top, rules.scale);
    }
    sum = wave_sum(sum);
    if (lane == 0) sum_lds[wave] = sum;
    __syncthreads();
    if (tid == 0) {
      sum = 0.0;
      for (int i = 0; i < W; ++i) sum += sum_lds[i];
      *head = SliceHead{best, sum, 0.0, 0, 0, 0, {}};
    }
    return;
  }
  if constexpr (PLAIN) return;
  if (rules.classes()) {
    const double ref = octave_of(top, rules.scale);
    uint64_t low = 0;  // behind the last class
    int valid = 0;
#pragma unroll
    for (int l = 0; l < L; ++l)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (!(x[l][e] > -INFINITY)) continue;
        ++valid;
        const double t = fmax(octaves_below(x[l][e], ref, rules.scale), -900.0);
        const uint64_t w = whole(exp2_within(t + kClassBits));
        const int c = class_of(t);
        if (c < kClasses)
          atomicAdd(reinterpret_cast<unsigned long long*>(&classes[c]), (unsigned long long)w);
        else
          low += w;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      low += __shfl_xor((unsigned long long)low, o);
      valid += __shfl_xor(valid, o);
    }
    __syncthreads();
    // running sums, two classes a thread
    const uint64_t c0 = classes[2 * tid], c1 = classes[2 * tid + 1];
    uint64_t run = c0 + c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t up = __shfl_up((unsigned long long)run, o);
      if (lane >= o) run += up;
    }
    if (lane == 63) total_lds[wave] = run;
    if (lane == 0) {
      low_lds[wave] = low;
      count_lds[wave] = valid;
    }
    __syncthreads();
    for (int i = 0; i < wave; ++i) run += total_lds[i];
    uint64_t* const sums = reinterpret_cast<uint64_t*>(part);
    *reinterpret_cast<u32x4*>(&sums[2 * tid]) =
        u32x4{uint32_t(run - c1), uint32_t((run - c1) >> 32), uint32_t(run), uint32_t(run >> 32)};
    if (tid == 0) {
      uint64_t all = 0;
      valid = 0;
      for (int i = 0; i < W; ++i) {
        all += total_lds[i] + low_lds[i];
        valid += count_lds[i];
      }
      *head = SliceHead{best, double(all), ref, 0, 0, uint32_t(valid), {}};
    }
    return;
  }
  int valid = 0;
#pragma unroll
  for (int l = 0; l < L; ++l)
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (x[l][e] > -INFINITY) {
        ++valid;
        atomicAdd(&hist[distance_bin(x[l][e], top)], 1);
      }
  __syncthreads();
  // how many bins fit the list, and how many hold the first top_k
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
    valid += __shfl_xor(valid, o);
  }
  if (lane == 0) {
    atomicAdd(&bins_lds[0], fit);
    atomicAdd(&bins_lds[1], less);
  }
  __syncthreads();
  const int bins = min(bins_lds[0], bins_lds[1] + 1);
  uint2* const list = reinterpret_cast<uint2*>(part);
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
  if (lane == 0) {
    left_lds[wave] = left;
    total_lds[wave] = valid;
  }
  __syncthreads();
  if (tid == 0) {
    valid = 0;
    for (int i = 0; i < W; ++i) {
      left = max(left, left_lds[i]);
      valid += int(total_lds[i]);
    }
    *head = SliceHead{best, 0.0, 0.0, uint32_t(taken), left, uint32_t(valid), {}};
  }
}

// ---- a row ----
struct RowShared {
  uint64_t hist[kBins];
  uint64_t wave[kRowWaves];
  double wave_d[kRowWaves];
  uint64_t found_before, found_value;
  int found_bin;
  int n, thinned;  // tokens listed, and those of them that thinning leaves
  double target;
  int slice, token, first;
  uint32_t cut_key, cut_token;
};

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

constexpr int kTokenBits = 20;
constexpr uint32_t kTokenMask = (1u << kTokenBits) - 1;

// Where in the order (value descending, token ascending) the last token that stays lies.
struct Cut {
  uint32_t key, token;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t t) const { return k > key || (k == key && t <= token); }
};

// A search through (ordered value, token, weight in units) by radix descents, each to the place of a descending order
// where a running sum reaches a target.  Five steps use the one loop: the first top_k by value, and by token among
// those of the last value; the shortest prefix of top_p by value, and by token; the token drawn.  (One piece of code,
// not five: it is rarely run, and the registers of the kernels around it are better left to them.)
enum { kByCount, kCountTies, kByShare, kShareTies, kDraw };
struct Search {
  Cut cut;
  int top_k;          // 0: not a rule
  double top_p;       // 1 or more: not a rule
  double row_units;   // the whole row's weights, for top_p where there is no top_k; negative: the sum of what is searched
  uint64_t least;     // min_p's weight, 1 or more
  double u;
  uint64_t need;      // kByShare: where not 0, the sum that the prefix has to reach
  // results of the draw
  uint32_t token;
  uint64_t total;
};
template <class Source>
__device__ __forceinline__ void search(RowShared& sh, const Source& src, Search& st, int from, int to) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint64_t ties = 0;  // how many of the last value stay; 0: all
  for (int step = from; step <= to; ++step) {
    uint64_t target = ties, sum = 0;
    if (step == kByShare || step == kDraw) {
      const uint64_t least = step == kDraw ? st.least : 1;
      src.each([&](uint32_t k, uint32_t t, auto&& w) {
        if (!st.cut.keeps(k, t)) return;
        const uint64_t v = w();
        if (v >= least) sum += v;
      });
      sum = block_sum(sh, sum);
    }
    if (step == kByCount) target = st.top_k;
    if (step == kByShare) {
      target = st.need;
      if (target == 0) target = max(uint64_t(ceil(st.top_p * (st.row_units < 0.0 ? double(sum) : st.row_units))), uint64_t(1));
      if (st.top_p >= 1.0 || target >= sum) target = 0;
    }
    if (step == kDraw) {
      st.total = sum;
      target = min(uint64_t(st.u * double(sum)), sum - 1) + 1;
    }
    ties = 0;
    if (target == 0) continue;
    const bool by_value = step == kByCount || step == kByShare, weighted = step == kByShare || step == kDraw;
    const bool tied = step == kCountTies || step == kShareTies;
    uint32_t key = 0;
    uint64_t value = 0;  // of all that have the key
    for (int shift = by_value ? 32 : kTokenBits; shift > 0;) {
      const int bits = min(kBinBits, shift);
      shift -= bits;
      for (int i = tid; i < kBins; i += kRowThreads) sh.hist[i] = 0;
      __syncthreads();
      const uint32_t done = shift + bits >= 32 ? 0u : ~0u << (shift + bits);
      src.each([&](uint32_t k, uint32_t t, auto&& w) {
        if (!st.cut.keeps(k, t) || (tied && k != st.cut.key)) return;
        const uint32_t order = by_value ? k : kTokenMask - t;
        if ((order & done) != key) return;
        uint64_t v = weighted ? w() : 1;
        if (step == kDraw && v < st.least) v = 0;
        if (v > 0)
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(order >> shift) & ((1u << bits) - 1)]), (unsigned long long)v);
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
      const bool first = before < target && before + v0 >= target;
      if (first || (before + v0 < target && before + v0 + v1 >= target)) {
        sh.found_bin = first ? at : at - 1;
        sh.found_before = first ? before : before + v0;
        sh.found_value = first ? v0 : v1;
      }
      __syncthreads();
      key |= uint32_t(sh.found_bin) << shift;
      target -= sh.found_before;
      value = sh.found_value;
    }
    __syncthreads();
    if (step == kDraw) {
      st.token = min(kTokenMask - key, uint32_t(src.vocab - 1));
    } else if (tied) {
      st.cut.token = kTokenMask - key;
    } else {
      // of the tokens of that very value, all of one weight, the lowest
      const uint64_t one = weighted ? max(src.weight(key), uint64_t(1)) : 1;
      const uint64_t stay = (target + one - 1) / one;
      if (st.cut.key != key) st.cut = {key, kTokenMask};
      if (stay * one < value) ties = stay;
    }
  }
}

struct ListSource {
  const uint32_t* keys;
  const uint32_t* tokens;
  const uint64_t* weights;
  int n, vocab;
  float top;
  double ref, scale, unit;  // ref: the octave that units count from; NaN: they are of the largest weight
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    for (int i = threadIdx.x; i < n; i += kRowThreads) f(keys[i], tokens[i], [&] { return weights[i]; });
  }
  // the same bits as the list's
  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    const float x = value_of(key);
    return ref == ref ? whole(exp2_within(octaves_below(x, ref, scale) + kClassBits))
                      : uint64_t(weight_of(x, top, scale) * unit + 0.5);
  }
};

template <class T>
struct RowSource {
  Row<T> row;
  float top;
  double scale, unit;
  int pieces, vocab;
  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    return uint64_t(weight_of(value_of(key), top, scale) * unit + 0.5);
  }
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    constexpr int V = Row<T>::kVec;
    for (int i = threadIdx.x; i < pieces; i += kRowThreads) {
      float x[V];
      row.get(i, x);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t key = ordered(x[e]);
        if (key != 0) f(key, uint32_t(i * V + e - row.skip), [&] { return uint64_t(weight_of(x[e], top, scale) * unit + 0.5); });
      }
    }
  }
};

// All the rules: of weights in `unit`s of the largest, where `valid` tokens can be drawn.
__device__ __forceinline__ Search whole_search(const Rules& r, double u, double unit, double row_units, uint32_t valid) {
  Search st = {};
  st.cut = {0, kTokenMask};
  st.top_k = uint32_t(r.top_k) < valid ? r.top_k : 0;
  st.top_p = r.use_p ? r.top_p : 1.0;
  st.row_units = row_units;
  st.least = r.use_m ? max(uint64_t(r.min_p * unit), uint64_t(1)) : 1;
  st.u = u;
  return st;
}

// Strides STRIDE .. 1 of a bitonic merge of blocks of `size`.
template <int STRIDE>
__device__ __forceinline__ uint64_t merge_down(uint64_t key, int size) {
  const uint64_t other = across<STRIDE>(key);
  const bool larger = ((threadIdx.x & size) == 0) == ((threadIdx.x & STRIDE) == 0);  // this place takes the larger
  key = (key > other) == larger ? key : other;
  if constexpr (STRIDE > 1) return merge_down<STRIDE / 2>(key, size);
  return key;
}
// 64 keys of a wave, each block of them by `size`'s direction (64: the largest first).
__device__ __forceinline__ uint64_t sort_wave(uint64_t key) {
  key = merge_down<1>(key, 2);
  key = merge_down<2>(key, 4);
  key = merge_down<4>(key, 8);
  key = merge_down<8>(key, 16);
  key = merge_down<16>(key, 32);
  return merge_down<32>(key, 64);
}
// One key a thread, the largest first, over the first n threads (a power of two from 64 on).  Every thread calls it.
__device__ uint64_t sort_down(uint64_t* lds, uint64_t key, int n) {
  const int tid = threadIdx.x;
  key = sort_wave(key);
  for (int size = 128; size <= n; size <<= 1) {
    for (int stride = size >> 1; stride >= 64; stride >>= 1) {
      __syncthreads();
      if (tid < n) lds[tid] = key;
      __syncthreads();
      const uint64_t other = tid < n ? lds[tid ^ stride] : 0;
      const bool larger = ((tid & size) == 0) == ((tid & stride) == 0);
      key = (key > other) == larger ? key : other;
    }
    key = merge_down<32>(key, size);
  }
  return key;
}

__device__ __forceinline__ double wave_running_sum(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(x, o);
    if (int(threadIdx.x & 63) >= o) x += up;
  }
  return x;
}

// The running sum over the first n threads, in their order; `all` the sum.
__device__ __forceinline__ double running_sum(double* lds, double x, int n, double& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (n + 63) >> 6;
  double run = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(run, o);
    if (lane >= o) run += up;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = run;
  __syncthreads();
  double before = 0.0;
  all = 0.0;
  for (int i = 0; i < waves; ++i) {
    if (i < wave) before += lds[i];
    all += lds[i];
  }
  return before + run;
}

struct RowLds {
  RowShared sh;
  struct {
    uint32_t keys[kListMax], tokens[kListMax];
    uint64_t weights[kListMax];
  } list;
  uint64_t best[kRowWaves];
  uint32_t left[kRowWaves], valid[kRowWaves];
  double ref[kRowWaves];
  double slice[kSlicesMax];     // its weights that stay, in order
  double factor[kSlicesMax];    // of its sums to the row's reference
  int shift[kSlicesMax];        // of its classes
  unsigned long long extra[kSlicesMax];  // what stays of the cut class
  double class_sum[kClasses];
  int cut;
};

// The logarithm of a token's share of `total`, which is relative to the largest weight.
__device__ __forceinline__ float log_share(float x, float top, const Rules& r, double total) {
  return float((x == top ? 0.0 : (double(x) - double(top)) * r.scale * 0.69314718055994531) - log(total));
}

// The slices' weights together: every lane and wave adds in the same tree, and gets the same bits.
__device__ __forceinline__ double slices_sum(const double* slice, int n) {
  double x = 0.0;
  for (int s = threadIdx.x & 63; s < n; s += 64) x += slice[s];
  return wave_sum(x);
}

// The token in the slice that the draw fell into (sh.slice, sh.target from its start on); weight(x, token) is 0 for what
// does not stay.
template <int PER, int THREADS, class T, class Shared, class Weight>
__device__ __forceinline__ int draw_in_slice(Shared& sh, const SampleParams& p, const Row<T>& src, int row, Weight&& weight) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = (sh.slice * THREADS + tid) * PER - src.skip;
  const T* values = static_cast<const T*>(p.logits) + row * p.stride;
  float x[PER];
  double w[PER], mine = 0.0;
#pragma unroll
  for (int e = 0; e < PER; ++e) x[e] = unsigned(first + e) < unsigned(p.vocab) ? to_float(values[first + e]) : -INFINITY;
  int last = -1;  // this thread's last token with any weight
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    w[e] = x[e] > -INFINITY ? weight(x[e], first + e) : 0.0;
    mine += w[e];
    if (w[e] > 0.0) last = first + e;
  }
  const double run = wave_running_sum(mine);
  if (lane == 63) sh.wave_d[wave] = run;
  // the sums of this order may fall short of the slice's own by their rounding: then it is the last token
  if (last >= 0) atomicMax(&sh.token, last);
  __syncthreads();
  double sum = 0.0;
  for (int i = 0; i < wave; ++i) sum += sh.wave_d[i];
  sum += run - mine;
  int got = 0x7fffffff;
#pragma unroll
  for (int e = PER - 1; e >= 0; --e) {
    double upto = sum;
#pragma unroll
    for (int j = 0; j <= e; ++j) upto += w[j];
    if (w[e] > 0.0 && upto > sh.target) got = first + e;
  }
  if (got != 0x7fffffff) atomicMin(&sh.first, got);
  __syncthreads();
  return min(max(sh.first == 0x7fffffff ? sh.token : sh.first, 0), p.vocab - 1);
}

// The draw among the weights of the slices (lds.slice): the slice, then the token in it.
template <int PER, class T, class Lds, class Weight>
__device__ int draw_from_slices(Lds& lds, const SampleParams& p, const Row<T>& src, int row, double target, Weight&& weight) {
  auto& sh = lds.sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave == 0) {
    // 64 slices at a time; the sums run on in order
    double run = 0.0, before = 0.0;
    int at = -1;
    for (int s0 = 0; s0 < p.slices; s0 += 64) {
      const double mine = s0 + lane < p.slices ? lds.slice[s0 + lane] : 0.0;
      double sum = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(sum, o);
        if (lane >= o) sum += up;
      }
      sum += run;
      const uint64_t past = __ballot(mine > 0.0 && sum > target), some = __ballot(mine > 0.0);
      if (some) {
        const int i = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);  // else the last that has any, so far
        at = s0 + i;
        before = __shfl(sum, i) - __shfl(mine, i);
      }
      if (past) break;
      run = __shfl(sum, 63);
    }
    if (lane == 0) {
      sh.slice = at;
      sh.target = target - before;
      sh.token = -1;
      sh.first = 0x7fffffff;
    }
  }
  __syncthreads();
  return draw_in_slice<PER, kRowThreads>(sh, p, src, row, weight);
}

// Rows without a rule: the first wave takes all slices' sums, four a lane, and picks the slice.  256 rows of 131072 take
// 46 us with both launches, by the kernel of the other rows 50; one row 16 and 17.
struct PlainLds {
  struct {
    double wave_d[kRowWaves], target;
    int slice, token, first;
  } sh;
  double total;
  float top;
};
constexpr int kPlainThreads = 256;
template <class T>
__global__ __launch_bounds__(kPlainThreads) void sample_plain_kernel(const SampleParams p) {
  constexpr int PER = kSlice / kPlainThreads;
  static_assert(kSlicesMax == 256, "four slices a lane");
  __shared__ PlainLds lds;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Rules rules = rules_of(p, row);
  const Row<T> src(p, row);
  if (wave == 0) {
    const SliceHead* heads = p.heads + int64_t(row) * p.slices;
    float tops[4], top = -INFINITY;
    double w[4], mine = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int s = lane * 4 + j;
      const uint64_t best = s < p.slices ? heads[s].best : 0;
      w[j] = s < p.slices ? heads[s].sum : 0.0;
      tops[j] = value_of(uint32_t(best >> 32));
      top = fmaxf(top, tops[j]);
    }
    const double u = fmin(fmax(double(p.uniforms[row]), 0.0), 1.0);
    top = wave_top(top);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] *= weight_of(tops[j], top, rules.scale);
      mine += w[j];
    }
    const double run = wave_running_sum(mine), total = __shfl(run, 63), target = u * total;
    const uint64_t past = __ballot(mine > 0.0 && run > target), some = __ballot(mine > 0.0);
    if (lane == (past ? __builtin_ctzll(past) : some ? 63 - __builtin_clzll(some) : 0)) {
      // the first slice past the target, else the last that weighs anything
      int at = 0;
      double upto = run - mine, before = upto;
      bool found = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!found && w[j] > 0.0) {
          at = lane * 4 + j;
          before = upto;
          found = upto + w[j] > target;
        }
        upto += w[j];
      }
      lds.sh.slice = at;
      lds.sh.target = target - before;
      lds.sh.token = -1;
      lds.sh.first = 0x7fffffff;
      lds.total = total;
      lds.top = top;
    }
  }
  __syncthreads();
  const float top = lds.top;
  if (top == -INFINITY) {
    if (tid == 0) {
      p.tokens[row] = -1;
      if (p.logprobs) p.logprobs[row] = -INFINITY;
    }
    return;
  }
  const int token = draw_in_slice<PER, kPlainThreads>(lds.sh, p, src, row, [&](float x, int) { return weight_of(x, top, rules.scale); });
  if (tid == 0) {
    p.tokens[row] = token;
    if (p.logprobs)
      p.logprobs[row] = log_share(to_float((static_cast<const T*>(p.logits) + row * p.stride)[token]), top, rules, lds.total);
  }
}

// Rows with top-k.
template <class T>
__device__ __forceinline__ void lists_row(const SampleParams& p, const Rules& rules, int row, RowLds& lds) {
  RowShared& sh = lds.sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row<T> src(p, row);
  SliceHead head = {};
  if (tid < p.slices) head = p.heads[int64_t(row) * p.slices + tid];
  uint64_t best = wave_max(head.best);
  uint32_t left = uint32_t(wave_max(uint64_t(head.left)));
  uint32_t valid = head.valid;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) valid += __shfl_xor(valid, o);
  if (lane == 0) {
    lds.best[wave] = best;
    lds.left[wave] = left;
    lds.valid[wave] = valid;
  }
  if (tid == 0) sh.n = sh.thinned = 0;
  __syncthreads();
  valid = 0;
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) {
    best = max(best, lds.best[i]);
    left = max(left, lds.left[i]);
    valid += lds.valid[i];
  }
  const float top = value_of(uint32_t(best >> 32));
  const T* const values = static_cast<const T*>(p.logits) + row * p.stride;
  if (best == 0) {  // nothing to draw
    if (tid == 0) {
      p.tokens[row] = -1;
      if (p.logprobs) p.logprobs[row] = -INFINITY;
    }
    return;
  }
  const double u = fmin(fmax(double(p.uniforms[row]), 0.0), 1.0);
  const char* const parts = static_cast<const char*>(p.lists) + int64_t(row) * p.slices * p.part;
  auto finish = [&](int token, double total) {  // total: of the weights that stay, relative to the largest
    if (tid == 0) {
      p.tokens[row] = token;
      if (p.logprobs) p.logprobs[row] = log_share(to_float(values[token]), top, rules, total);
    }
  };
  // the lists, as far as they are whole: above the largest value that some slice left out.  All loads at once: a list
  // has `cap` places, kListMax together at most.
  if (tid < p.slices) lds.shift[tid] = min(int(head.count), p.cap);
  __syncthreads();
  uint2 it[kListMax / kRowThreads];
#pragma unroll
  for (int j = 0; j < kListMax / kRowThreads; ++j) {
    const int i = tid + j * kRowThreads, s = i / p.cap;
    it[j] = uint2{0, 0};
    if (s < p.slices && i - s * p.cap < lds.shift[s]) it[j] = reinterpret_cast<const uint2*>(parts + s * p.part)[i - s * p.cap];
  }
#pragma unroll
  for (int j = 0; j < kListMax / kRowThreads; ++j) {
    const bool take = it[j].x > left;
    const uint64_t all = __ballot(take);
    if (!all) continue;
    int at = 0;
    if (lane == 0) at = atomicAdd(&sh.n, __popcll(all));
    at = __builtin_amdgcn_readfirstlane(at) + __popcll(all & ((uint64_t(1) << lane) - 1));
    if (take) {
      lds.list.keys[at] = it[j].x;
      lds.list.tokens[at] = it[j].y;
    }
  }
  __syncthreads();
  int n = min(sh.n, kListMax);
  const bool enough = left == 0 || n >= rules.top_k;
  if (n > kRowThreads && enough && rules.top_k < kRowThreads) {
    // first down to those in the classes of distance that the first top_k reach.  They have a count of their own: a wave
    // may not have read sh.n yet, which decides whether it comes here at all.
    int* const hist = reinterpret_cast<int*>(sh.hist);
    hist[tid] = 0;
    __syncthreads();
    uint32_t keys[kListMax / kRowThreads], tokens[kListMax / kRowThreads];
    int bins[kListMax / kRowThreads];
#pragma unroll
    for (int j = 0; j < kListMax / kRowThreads; ++j) {
      const int i = tid + j * kRowThreads;
      bins[j] = 1024;
      if (i >= n) continue;
      keys[j] = lds.list.keys[i];
      tokens[j] = lds.list.tokens[i];
      bins[j] = distance_bin(value_of(keys[j]), top);
      atomicAdd(&hist[bins[j]], 1);
    }
    __syncthreads();
    // the class that the first `want` end in; `run`: how many up to this thread's
    int run;
    auto reach = [&](int want) {
      run = hist[tid];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(run, o);
        if (lane >= o) run += up;
      }
      if (lane == 63) lds.left[wave] = uint32_t(run);
      __syncthreads();
      for (int i = 0; i < wave; ++i) run += int(lds.left[i]);
      return __syncthreads_count(run < want);
    };
    const int last = reach(rules.top_k);
    if (tid == last - 1) sh.slice = run;
    if (tid == last) sh.found_bin = run;
    __syncthreads();
    if (last > 0 && last < 1023 && sh.found_bin > kRowThreads) {
      // and of that class by the next ten bits of the distance (60 rows of 128000 with settings of their own: 87 us in
      // place of 98, as fewer are searched through); classes 0 and 1023 take in what lies behind them, and are not cut
      const int want = rules.top_k - sh.slice;
      hist[tid] = 0;
      __syncthreads();
      auto finer = [&](uint32_t key) { return int(__float_as_uint(top - value_of(key)) >> 8 & 1023); };
#pragma unroll
      for (int j = 0; j < kListMax / kRowThreads; ++j)
        if (bins[j] == last) atomicAdd(&hist[finer(keys[j])], 1);
      __syncthreads();
      const int finer_last = reach(want);
#pragma unroll
      for (int j = 0; j < kListMax / kRowThreads; ++j)
        if (bins[j] == last && finer(keys[j]) > finer_last) bins[j] = 1024;
    }
#pragma unroll
    for (int j = 0; j < kListMax / kRowThreads; ++j)
      if (bins[j] <= last && bins[j] < 1024) {
        const int at = atomicAdd(&sh.thinned, 1);
        lds.list.keys[at] = keys[j];
        lds.list.tokens[at] = tokens[j];
      }
    __syncthreads();
    n = sh.thinned;
  }
  if (n <= kRowThreads && enough) {
    // sorted, a token a thread: top-k is the first so many, top-p and min-p a prefix of them
    uint64_t key = tid < n ? uint64_t(lds.list.keys[tid]) << 32 | uint32_t(~lds.list.tokens[tid]) : 0;
    __syncthreads();
    int size = 64;
    while (size < n) size <<= 1;
    key = sort_down(sh.hist, key, size);
    const int k = min(n, rules.top_k);
    if (k <= 64) {  // all in the first wave: nothing to wait for
      if (wave > 0) return;
      double w = lane < k ? weight_of(value_of(uint32_t(key >> 32)), top, rules.scale) : 0.0;
      int stay = k;
      if (rules.use_p) {
        const double run = wave_running_sum(w), all = __shfl(run, 63);
        stay = __popcll(__ballot(lane < k && (lane == 0 || run - w < rules.top_p * all)));
      }
      if (rules.use_m) stay = min(stay, int(__popcll(__ballot(lane < k && w >= rules.min_p))));
      // and by token, for the draw
      w = lane < stay ? w : 0.0;
      key = sort_wave(lane < stay ? uint64_t(uint32_t(key)) << 32 | uint32_t(lane) : 0);
      w = lane < stay ? __shfl(w, int(uint32_t(key))) : 0.0;
      const double run = wave_running_sum(w), all = __shfl(run, 63);
      // the first past the target, else (roundings aside there is one) the last with any weight
      const uint64_t past = __ballot(lane < stay && run > u * all), some = __ballot(w > 0.0);
      const int pick = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
      finish(int(~uint32_t(__shfl((unsigned long long)key, pick) >> 32)), all);
      return;
    }
    const float x = value_of(uint32_t(key >> 32));
    double w = tid < k ? weight_of(x, top, rules.scale) : 0.0, all;
    int stay = k;
    if (rules.use_p) {
      const double run = running_sum(sh.wave_d, w, k, all);
      stay = __syncthreads_count(tid < k && (tid == 0 || run - w < rules.top_p * all));
    }
    if (rules.use_m) stay = min(stay, __syncthreads_count(tid < k && w >= rules.min_p));
    // and by token, for the draw
    w = tid < stay ? w : 0.0;
    key = tid < stay ? uint64_t(uint32_t(key)) << 32 | uint32_t(tid) : 0;
    __syncthreads();
    if (tid < stay) lds.list.weights[tid] = __double_as_longlong(w);
    size = 64;
    while (size < stay) size <<= 1;
    key = sort_down(sh.hist, key, size);
    __syncthreads();
    w = tid < stay ? __longlong_as_double(lds.list.weights[uint32_t(key)]) : 0.0;
    const double run = running_sum(sh.wave_d, w, stay, all);
    // the first past the target; rounding aside there is one, else the last with any weight
    const int before = __syncthreads_count(tid < stay && !(run > u * all));
    int pick = before;
    if (before >= stay) {
      if (tid == 0) sh.token = 0;
      __syncthreads();
      if (tid < stay && w > 0.0) atomicMax(&sh.token, tid);
      __syncthreads();
      pick = sh.token;
    }
    if (tid == pick) sh.slice = int(~uint32_t(key >> 32));
    __syncthreads();
    finish(sh.slice, all);
    return;
  }
  if (enough) {
    constexpr int kListBits = 49;
    const double unit = ldexp(1.0, kListBits);
    for (int i = tid; i < n; i += kRowThreads)
      lds.list.weights[i] = uint64_t(weight_of(value_of(lds.list.keys[i]), top, rules.scale) * unit + 0.5);
    __syncthreads();
    Search st = whole_search(rules, u, unit, -1.0, uint32_t(n));
    search(sh, ListSource{lds.list.keys, lds.list.tokens, lds.list.weights, n, p.vocab, top, NAN, rules.scale, unit}, st, kByCount, kDraw);
    finish(int(st.token), double(st.total) / unit);
    return;
  }
  const double unit = ldexp(1.0, 62 - kTokenBits);
  const int pieces = (src.skip + p.vocab + Row<T>::kVec - 1) / Row<T>::kVec;
  Search st = whole_search(rules, u, unit, -1.0, valid);
  search(sh, RowSource<T>{src, top, rules.scale, unit, pieces, p.vocab}, st, kByCount, kDraw);
  finish(int(st.token), double(st.total) / unit);
}

// Every other row, where some have rules.
template <class T, int PER>
__device__ __forceinline__ void classes_row(const SampleParams& p, const Rules& rules, int row, RowLds& lds) {
  constexpr int slice_size = PER * kRowThreads;
  RowShared& sh = lds.sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Row<T> src(p, row);
  SliceHead head = {};
  if (tid < p.slices) head = p.heads[int64_t(row) * p.slices + tid];
  uint64_t best = wave_max(head.best);
  uint32_t valid = head.valid;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) valid += __shfl_xor(valid, o);
  if (lane == 0) {
    lds.best[wave] = best;
    lds.valid[wave] = valid;
  }
  if (tid == 0) sh.n = 0;
  __syncthreads();
  valid = 0;
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) {
    best = max(best, lds.best[i]);
    valid += lds.valid[i];
  }
  const float top = value_of(uint32_t(best >> 32));
  const T* const values = static_cast<const T*>(p.logits) + row * p.stride;
  if (best == 0 || rules.greedy) {  // nothing to draw, or nothing to choose
    if (tid == 0) {
      p.tokens[row] = best == 0 ? -1 : int(~uint32_t(best));
      if (p.logprobs) p.logprobs[row] = best == 0 ? -INFINITY : 0.0f;
    }
    return;
  }
  const double u = fmin(fmax(double(p.uniforms[row]), 0.0), 1.0);
  const char* const parts = static_cast<const char*>(p.lists) + int64_t(row) * p.slices * p.part;
  auto finish = [&](int token, double total) {  // total: of the weights that stay, relative to the largest
    if (tid == 0) {
      p.tokens[row] = token;
      if (p.logprobs) p.logprobs[row] = log_share(to_float(values[token]), top, rules, total);
    }
  };
  double total = 0.0;  // of the row's weights
  if (!rules.classes()) {
    if (tid < p.slices)
      lds.slice[tid] = head.best ? head.sum * weight_of(value_of(uint32_t(head.best >> 32)), top, rules.scale) : 0.0;
    __syncthreads();
    total = slices_sum(lds.slice, p.slices);
    const int token = draw_from_slices<PER>(lds, p, src, row, u * total,
                                            [&](float x, int) { return weight_of(x, top, rules.scale); });
    finish(token, total);
    return;
  }
  // the row's classes: the slices' counted from the row's reference
  const double ref = octave_of(top, rules.scale);
  if (tid < p.slices) {
    const double down = head.best ? fmin(ref - head.ref, 4096.0) : 4096.0;
    lds.shift[tid] = int(down) * int(kPerOctave);
    lds.factor[tid] = head.best ? exp2_of(-down) : 0.0;
    lds.slice[tid] = head.best ? head.sum * lds.factor[tid] : 0.0;
    lds.extra[tid] = 0;
  }
  if (tid == 0) {
    lds.cut = kClasses;
    sh.cut_key = 0;  // all of the class stays where its sum falls short
    sh.cut_token = kTokenMask;
  }
  __syncthreads();
  total = slices_sum(lds.slice, p.slices);
  auto upto = [&](int s, int c) -> double {  // slice s's weights in classes 0 .. c, in units of 2^-kClassBits
    const int at = min(c - lds.shift[s], kClasses - 1);
    if (at < 0 || lds.factor[s] == 0.0) return 0.0;
    return double(reinterpret_cast<const uint64_t*>(parts + s * p.part)[at]) * lds.factor[s];
  };
  {
    // the even and the odd slices, by the two halves of the workgroup, eight loads on their way
    const int c = tid & (kClasses - 1), odd = tid / kClasses;
    double sum = 0.0;
    for (int s0 = odd; s0 < p.slices; s0 += 16) {
      uint64_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = min(s0 + 2 * i, p.slices - 1);
        v[i] = reinterpret_cast<const uint64_t*>(parts + s * p.part)[min(max(c - lds.shift[s], 0), kClasses - 1)];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = s0 + 2 * i;
        if (s < p.slices && c >= lds.shift[s] && lds.factor[s] != 0.0) sum += double(v[i]) * lds.factor[s];
      }
    }
    if (odd) lds.class_sum[c] = sum;
    __syncthreads();
    if (!odd) lds.class_sum[c] += sum;
  }
  __syncthreads();
  // the largest weight lies below the reference by up to an octave
  const double t_top = octaves_below(top, ref, rules.scale);
  const double t_min = rules.use_m ? t_top + log2(rules.min_p) : -1e300;
  const double target = rules.top_p * total;
  if (tid < kClasses && rules.use_p && lds.class_sum[tid] >= target) atomicMin(&lds.cut, tid);
  __syncthreads();
  const int p_cut = lds.cut;
  const int cut = rules.use_m ? min(p_cut, class_of(t_min)) : p_cut;
  if (cut < kClasses) {
    const double above = cut > 0 ? lds.class_sum[cut - 1] : 0.0;
    // the cut class's tokens: those between the logits that bound it (a little more, then exactly)
    const double inv = 1.0 / rules.scale;
    const double slack = 1e-9 * (1.0 + fabs(ref));  // the octaves' own rounding, far from the reference's whole part
    double hi = (ref - cut / kPerOctave + slack) * inv, lo = (ref - (cut + 1) / kPerOctave - slack) * inv;
    hi += 1e-6 * fabs(hi);
    lo -= 1e-6 * fabs(lo);
    const bool infinite = top == INFINITY;
    const float x_hi = infinite ? INFINITY : float(hi), x_lo = infinite ? INFINITY : float(lo);
    const int pieces = (src.skip + p.vocab + Row<T>::kVec - 1) / Row<T>::kVec;
    constexpr int kAhead = 6, V = Row<T>::kVec;
    for (int i0 = tid; i0 < pieces; i0 += kAhead * kRowThreads) {
      u32x4 v[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) v[a] = src.raw(i0 + a * kRowThreads);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        float x[V], most = -INFINITY;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[e] = Row<T>::value(v[a], e);
          most = fmaxf(most, x[e]);
        }
        if (!(most >= x_lo) || i0 + a * kRowThreads >= pieces) continue;  // most pieces hold nothing so large
#pragma unroll
        for (int e = 0; e < V; ++e) {
          if (!(x[e] >= x_lo && x[e] <= x_hi)) continue;
          const int at = atomicAdd(&sh.n, 1);
          if (at < kListMax) {
            lds.list.keys[at] = __float_as_uint(x[e]);
            lds.list.tokens[at] = uint32_t((i0 + a * kRowThreads) * V + e - src.skip);
          }
        }
      }
    }
    __syncthreads();
    const int n = sh.n;
    if (n <= kListMax) {
      // now exactly: what is not of the class weighs nothing
      for (int i = tid; i < n; i += kRowThreads) {
        const float x = __uint_as_float(lds.list.keys[i]);
        const double t = octaves_below(x, ref, rules.scale);
        const bool in = lds.list.tokens[i] < uint32_t(p.vocab) && class_of(t) == cut;
        lds.list.keys[i] = in ? ordered(x) : 0;
        lds.list.weights[i] = in ? whole(exp2_within(t + kClassBits)) : 0;
        if (!in) lds.list.tokens[i] = 0;
      }
      __syncthreads();
      Cut at = {0, kTokenMask};
      if (p_cut == cut && n <= kRowThreads) {
        // sorted: the place where the running sum gets there
        const double rest = target - above;
        const uint64_t need = max(uint64_t(ceil(fmax(rest, 0.0))), uint64_t(1));
        uint64_t key = tid < n ? uint64_t(lds.list.keys[tid]) << 32 | uint64_t(kTokenMask - lds.list.tokens[tid]) << 10 | uint32_t(tid) : 0;
        int size = 64;
        while (size < n) size <<= 1;
        key = sort_down(sh.hist, key, size);
        const uint64_t mine = tid < n ? lds.list.weights[uint32_t(key) & (kRowThreads - 1)] : 0;
        uint64_t run = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint64_t up = __shfl_up((unsigned long long)run, o);
          if (lane >= o) run += up;
        }
        if (lane == 63) sh.wave[wave] = run;
        __syncthreads();
        for (int i = 0; i < wave; ++i) run += sh.wave[i];
        if (tid < n && run >= need && run - mine < need) {
          sh.cut_key = uint32_t(key >> 32);
          sh.cut_token = kTokenMask - (uint32_t(key) >> 10 & kTokenMask);
        }
        __syncthreads();
        at = {sh.cut_key, sh.cut_token};
      } else if (p_cut == cut) {
        Search st = {{0, kTokenMask}, 0, 0.0, 0.0, 1, 0.0, max(uint64_t(ceil(fmax(target - above, 0.0))), uint64_t(1)), 0, 0};
        search(sh, ListSource{lds.list.keys, lds.list.tokens, lds.list.weights, n, p.vocab, top, ref, rules.scale, 0.0}, st,
               kByShare, kShareTies);
        at = st.cut;
      }
      auto stays = [&](double t, uint32_t key, uint32_t token) {
        const int c = class_of(t);
        return c < cut || (c == cut && t >= t_min && at.keeps(key, token));
      };
      for (int i = tid; i < n; i += kRowThreads) {
        const uint32_t key = lds.list.keys[i], token = lds.list.tokens[i];
        if (stays(octaves_below(value_of(key), ref, rules.scale), key, token))
          atomicAdd(&lds.extra[(token + src.skip) / slice_size], (unsigned long long)lds.list.weights[i]);
      }
      __syncthreads();
      if (tid < p.slices) lds.slice[tid] = (cut > 0 ? upto(tid, cut - 1) : 0.0) + double(lds.extra[tid]);
      __syncthreads();
      const double kept = slices_sum(lds.slice, p.slices);
      const double unit = ldexp(1.0, kClassBits);
      const int token = draw_from_slices<PER>(lds, p, src, row, u * kept, [&](float x, int token) {
        const double t = octaves_below(x, ref, rules.scale);
        return stays(t, ordered(x), token) ? exp2_of(t) * unit : 0.0;
      });
      finish(token, kept / unit / exp2_of(t_top));
      return;
    }
  }
  total = total / ldexp(1.0, kClassBits) / exp2_of(t_top);
  const double unit = ldexp(1.0, 62 - kTokenBits);
  const int pieces = (src.skip + p.vocab + Row<T>::kVec - 1) / Row<T>::kVec;
  Search st = whole_search(rules, u, unit, total * unit, valid);
  search(sh, RowSource<T>{src, top, rules.scale, unit, pieces, p.vocab}, st, kByCount, kDraw);
  finish(int(st.token), double(st.total) / unit);
}

// The rows with top-k, or the others; where a call has both, each kernel leaves the other's.
enum { kListRows, kOtherRows };
template <class T, int PER, int ROWS>
__global__ __launch_bounds__(kRowThreads) void sample_row_kernel(const SampleParams p) {
  __shared__ RowLds lds;
  const int row = blockIdx.x;
  const Rules rules = rules_of(p, row);
  if (rules.lists() != (ROWS == kListRows)) return;
  if constexpr (ROWS == kListRows)
    lists_row<T>(p, rules, row, lds);
  else
    classes_row<T, PER>(p, rules, row, lds);
}

// ---- the host side ----
struct Split {
  int slices, cap;
  int64_t part;  // bytes of a slice's list or classes
};
Split split_of(int vocab) {
  Split s;
  const int size = kSlice;
  s.slices = (vocab + 7 + size - 1) / size;
  // a slice lists the first top_k of its own, as far as there is room (with 512 places at most, 115 rows of 6883 tokens
  // with top-k of up to 1000, more than these places hold, took 83 us, not 51, 17 rows of 1826 61, not 40)
  s.cap = std::min(kSlice, kListMax / s.slices);
  s.part = (std::max<int64_t>(s.cap * sizeof(uint2), kClasses * sizeof(uint64_t)) + 15) / 16 * 16;
  return s;
}

// Which rows there are: plain ones alone, with top-k, any others.
struct Kinds {
  bool plain, lists, others;
};
template <class T>
void launch(const SampleParams& p, const Kinds& k, int rows, hipStream_t stream) {
  constexpr int PER = kSlice / kRowThreads;
  const dim3 slices(p.slices, rows);
  if (k.plain) {
    sample_slice_kernel<T, 16, true><<<slices, kSliceThreads, 0, stream>>>(p);
    sample_plain_kernel<T><<<rows, kPlainThreads, 0, stream>>>(p);
  } else {
    sample_slice_kernel<T, 16, false><<<slices, kSliceThreads, 0, stream>>>(p);
    // two kernels, not one with both: that one would have to spill (60 rows, some of either kind: 24 and 40 us)
    if (k.lists) sample_row_kernel<T, PER, kListRows><<<rows, kRowThreads, 0, stream>>>(p);
    if (k.others) sample_row_kernel<T, PER, kOtherRows><<<rows, kRowThreads, 0, stream>>>(p);
  }
}

}  // namespace
}  // namespace pkv

extern "C" size_t pkv_sample_workspace_bytes(int32_t rows, int32_t vocab) {
  using namespace pkv;
  if (rows <= 0 || vocab <= 0 || vocab > 1000000) return 0;
  const Split s = split_of(vocab);
  return size_t(rows) * s.slices * (sizeof(SliceHead) + s.part);
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
  const size_t need = pkv_sample_workspace_bytes(rows, vocab);
  if (!workspace || !aligned16(workspace)) return fail(PKV_EINVAL, "%s: workspace null or not 16-byte aligned", fn);
  if (workspace_bytes < need)
    return fail(PKV_ENOSPC, "%s: workspace %zu bytes < %zu needed", fn, workspace_bytes, need);
  const bool warm = !temperatures && temperature > 0.f, no_k = !top_ks && (top_k <= 0 || top_k >= vocab);
  Kinds kinds;
  kinds.plain = warm && no_k && !top_ps && !(top_p < 1.f) && !min_ps && !(min_p > 0.f);
  kinds.lists = !no_k;
  kinds.others = no_k || top_ks || !warm || top_ps || top_p <= 0.f || top_k == 1;  // greedy rows among them
  const Split s = split_of(vocab);
  SampleParams p;
  p.logits = logits;
  p.uniforms = uniforms;
  p.tokens = tokens;
  p.logprobs = logprobs;
  p.heads = static_cast<SliceHead*>(workspace);
  p.lists = p.heads + size_t(rows) * s.slices;
  p.temperature = {temperatures, temperature};
  p.scale = kLog2e / double(temperature);
  p.top_k = {top_ks, double(top_k)};
  p.top_p = {top_ps, top_p};
  p.min_p = {min_ps, min_p};
  p.stride = stride;
  p.vocab = vocab;
  p.slices = s.slices;
  p.cap = s.cap;
  p.part = s.part;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == PKV_BF16)
    launch<__bf16>(p, kinds, rows, st);
  else if (dtype == PKV_FP16)
    launch<_Float16>(p, kinds, rows, st);
  else
    launch<float>(p, kinds, rows, st);
  return check_launch(fn);
}
