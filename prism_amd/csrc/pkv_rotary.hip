// Rotary positions of packed tokens in their general form, for gfx950: an optional RMSNorm of every query and
// key head, the rotation (half or interleaved layout, all or the first rotary_dim elements of the head, any
// frequencies through fp32 tables) and, for the fused QKV projection's output, the append of the rotated keys
// and of the values to a paged cache, in one pass.
//
//   y = w x / sqrt(mean(x^2) + eps)                                      (norm; else y = x)
//   (y_i, y_p(i)) -> (y_i c_i - y_p(i) s_i,  y_p(i) c_i + y_i s_i)       c_i, s_i = cos / sin[position, i]
//   p(i) = i + rotary_dim / 2 (half), or elements 2 i and 2 i + 1 (interleaved), i < rotary_dim / 2
//
// Everything is fp32 up to the one rounding of each output.  (rope_qk_kernel keeps the reference's bf16
// rounding after each operation and its full-head half layout; it stays for callers that need those bits.)
//
// Memory bounds it: every element is read and written once, the tables add 8 bytes per rotated pair and token.
#include <type_traits>

#include "pkv_common.h"

namespace pkv {

struct RotaryParams {
  const void* q;
  const void* k;
  const uint16_t* v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  void* q_out;
  void* k_out;
  int64_t qo_st, qo_sh, ko_st, ko_sh;
  const int32_t* positions;
  const float* cos_tab;
  const float* sin_tab;
  const void* q_norm_w;
  const void* k_norm_w;
  uint16_t* k_cache;
  uint16_t* v_cache;
  int64_t page_stride;
  const int32_t* slots;
  int32_t* status;
  float eps;
  int n_pos, n_heads, n_kv, head_dim, rotary, interleaved;
  int log2_page, num_pages;
  int log2_lanes;       // a head has 2^log2_lanes lanes
  uint32_t tokens;      // of the launch
  uint32_t rows;        // heads of a token: queries, keys, and values where they are appended
  uint32_t magic;       // row r of the launch is in token (r magic) >> shift
  int shift;
};

// 16 bytes of T as floats, and back (rounded to nearest even); N floats of a table.
template <typename T>
struct Chunk {
  static constexpr int V = 16 / sizeof(T);
  typedef T TV __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ void load(const T* src, float (&f)[V]) {
    const TV v = __builtin_bit_cast(TV, ld16(src));
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = static_cast<float>(v[e]);
  }
  static __device__ __forceinline__ void store(T* dst, const float (&f)[V]) {
    TV v;
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = static_cast<T>(f[e]);
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(dst));
  }
};
template <int N>
__device__ __forceinline__ void load_table(const float* src, float (&f)[N]) {
  typedef float FN __attribute__((ext_vector_type(N < 4 ? N : 4)));
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const FN v = *reinterpret_cast<const FN*>(src + e);
#pragma unroll
    for (int k = 0; k < (N < 4 ? N : 4); ++k) f[e + k] = v[k];
  }
}
// N / 2 neighbouring pairs.
template <int N>
__device__ __forceinline__ void turn_pairs(float (&x)[N], const float (&c)[N / 2], const float (&s)[N / 2]) {
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    const float a = x[2 * k], b = x[2 * k + 1];
    x[2 * k] = a * c[k] - b * s[k];
    x[2 * k + 1] = b * c[k] + a * s[k];
  }
}

// Row of the rotation tables of token t, clamped (and flagged) outside them.
__device__ __forceinline__ int table_row(const RotaryParams& p, uint32_t t) {
  const int pos = p.positions[t];
  if (unsigned(pos) < unsigned(p.n_pos)) return pos;
  flag_status(p.status, PKV_STATUS_BAD_POSITION);
  return pos < 0 ? 0 : p.n_pos - 1;
}

// Elements from the start of the cache to token t's row (all KV heads), -1 (flagged) where its slot is none.
__device__ __forceinline__ int64_t slot_row(const RotaryParams& p, uint32_t t) {
  const int slot = p.slots[t];
  const int page = slot >> p.log2_page;
  if (unsigned(page) >= unsigned(p.num_pages)) {
    flag_status(p.status, PKV_STATUS_BAD_PAGE);
    return -1;
  }
  return int64_t(page) * p.page_stride + int64_t(slot & ((1 << p.log2_page) - 1)) * p.n_kv * p.head_dim;
}

// One lane holds two 16-byte chunks of one head: half layout, the two halves of its pairs (behind the rotated
// part, chunks of the two halves of the rest); interleaved, chunks of the two halves of the head.  So the lanes of a
// head read and write 16 bytes next to each other with every instruction (two neighbouring chunks per lane, and in
// fp32 four, took 52 us where 5003 tokens of 32 heads now take 25).  A lane reads nothing that another
// writes, so the outputs may be the inputs; the norm's sum goes over the head's lanes by shuffles.  Lanes are
// counted over the heads of all tokens: a token's 2 + 14 or 16 + 40 heads leave no lane of a workgroup idle.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
  using C = Chunk<T>;
  constexpr int V = C::V;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  const uint32_t r = i >> p.log2_lanes;
  const int c = int(i & ((1u << p.log2_lanes) - 1));
  const uint32_t t = uint32_t((uint64_t(r) * p.magic) >> p.shift);
  int hh = int(r - t * p.rows);
  // the lanes past the last head, and those past a head whose chunks are no power of two, only take part in
  // the shuffles
  const bool live = t < p.tokens && 2 * V * c < p.head_dim;
  const bool is_v = hh >= p.n_heads + p.n_kv, is_k = hh >= p.n_heads;
  int o1 = V * c, o2 = p.head_dim / 2 + V * c;
  if (is_v) {
    if (live) {
      const uint16_t* src = p.v + t * p.v_st + (hh - p.n_heads - p.n_kv) * p.v_sh;
      const u32x4 v1 = ld16(src + o1), v2 = ld16(src + o2);
      const int64_t row = slot_row(p, t);
      if (row >= 0) {
        uint16_t* dst = p.v_cache + row + (hh - p.n_heads - p.n_kv) * p.head_dim;
        __builtin_nontemporal_store(v1, reinterpret_cast<u32x4*>(dst + o1));
        __builtin_nontemporal_store(v2, reinterpret_cast<u32x4*>(dst + o2));
      }
    }
    return;  // a head's lanes are of one kind, so none of a shuffle's partners leaves
  }
  const bool rotated = 2 * V * c < p.rotary;  // half layout
  if (!INTERLEAVED) {
    o1 = rotated ? V * c : p.rotary / 2 + V * c;
    o2 = o1 + (rotated ? p.rotary : p.head_dim - p.rotary) / 2;
  }
  hh -= is_k ? p.n_heads : 0;
  float x1[V], x2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) x1[e] = x2[e] = 0.f;
  int pos = 0;
  if (live) {
    const T* src = static_cast<const T*>(is_k ? p.k : p.q) + t * (is_k ? p.k_st : p.q_st) + hh * (is_k ? p.k_sh : p.q_sh);
    C::load(src + o1, x1);
    C::load(src + o2, x2);
    pos = table_row(p, t);
  }
  const T* nw = static_cast<const T*>(is_k ? p.k_norm_w : p.q_norm_w);
  if (nw) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) ss += x1[e] * x1[e] + x2[e] * x2[e];
    for (int off = 1; off < (1 << p.log2_lanes); off <<= 1) ss += __shfl_xor(ss, off, 64);
    const float rs = rsqrtf(ss / float(p.head_dim) + p.eps);
    if (live) {
      float w1[V], w2[V];
      C::load(nw + o1, w1);
      C::load(nw + o2, w2);
#pragma unroll
      for (int e = 0; e < V; ++e) x1[e] *= rs * w1[e], x2[e] *= rs * w2[e];
    }
  }
  if (!live) return;
  const float* ct = p.cos_tab + int64_t(pos) * (p.rotary / 2);
  const float* st = p.sin_tab + int64_t(pos) * (p.rotary / 2);
  if constexpr (INTERLEAVED) {
    float cs[V / 2], sn[V / 2];
    if (o1 < p.rotary) {
      load_table(ct + o1 / 2, cs);
      load_table(st + o1 / 2, sn);
      turn_pairs(x1, cs, sn);
    }
    if (o2 < p.rotary) {
      load_table(ct + o2 / 2, cs);
      load_table(st + o2 / 2, sn);
      turn_pairs(x2, cs, sn);
    }
  } else if (rotated) {
    float cs[V], sn[V];
    load_table(ct + o1, cs);
    load_table(st + o1, sn);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = x1[e], b = x2[e];
      x1[e] = a * cs[e] - b * sn[e];
      x2[e] = b * cs[e] + a * sn[e];
    }
  }
  if (!is_k) {
    T* dst = static_cast<T*>(p.q_out) + t * p.qo_st + hh * p.qo_sh;
    C::store(dst + o1, x1);
    C::store(dst + o2, x2);
    return;
  }
  if (p.k_out) {
    T* dst = static_cast<T*>(p.k_out) + t * p.ko_st + hh * p.ko_sh;
    C::store(dst + o1, x1);
    C::store(dst + o2, x2);
  }
  if constexpr (std::is_same<T, __bf16>::value) {
    if (p.k_cache) {
      const int64_t row = slot_row(p, t);
      if (row >= 0) {
        T* dst = reinterpret_cast<T*>(p.k_cache) + row + hh * p.head_dim;
        C::store(dst + o1, x1);
        C::store(dst + o2, x2);
      }
    }
  }
}

// The same for rows that 16-byte accesses do not fit (odd strides or addresses, a head or a rotated part that is
// no multiple of 16): one wave per head, one pair or one unrotated element per lane and step.  Accesses of one element
// bound it: 2048 tokens of 40 heads of 96 with 24 rotated, bf16, 21.9 us (1.4 TB/s; 31 with the norm), where 32 rotated
// take 6.4 in the kernel above; 48 heads of 128 in rows of odd strides 27 against 6.7.
template <typename T>
__global__ __launch_bounds__(256) void rotary_any_kernel(const RotaryParams p) {
  const uint32_t r = blockIdx.x * 4u + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const uint32_t t = uint32_t((uint64_t(r) * p.magic) >> p.shift);
  if (t >= p.tokens) return;
  int hh = int(r - t * p.rows);
  const bool is_k = hh >= p.n_heads;
  hh -= is_k ? p.n_heads : 0;
  const T* src = static_cast<const T*>(is_k ? p.k : p.q) + t * (is_k ? p.k_st : p.q_st) + hh * (is_k ? p.k_sh : p.q_sh);
  T* dst = static_cast<T*>(is_k ? p.k_out : p.q_out) + t * (is_k ? p.ko_st : p.qo_st) + hh * (is_k ? p.ko_sh : p.qo_sh);
  const T* nw = static_cast<const T*>(is_k ? p.k_norm_w : p.q_norm_w);
  float rs = 1.f;
  if (nw) {
    float ss = 0.f;
    for (int e = lane; e < p.head_dim; e += 64) {
      const float x = static_cast<float>(src[e]);
      ss += x * x;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) ss += __shfl_xor(ss, off, 64);
    rs = rsqrtf(ss / float(p.head_dim) + p.eps);
  }
  auto value = [&](int e) {
    const float x = static_cast<float>(src[e]);
    return nw ? x * (rs * static_cast<float>(nw[e])) : x;
  };
  const int half = p.rotary / 2;
  const int64_t row = int64_t(table_row(p, t)) * half;
  for (int e = lane; e < p.head_dim - half; e += 64) {
    if (e < half) {
      const int ia = p.interleaved ? 2 * e : e, ib = p.interleaved ? 2 * e + 1 : e + half;
      const float a = value(ia), b = value(ib), c = p.cos_tab[row + e], s = p.sin_tab[row + e];
      dst[ia] = static_cast<T>(a * c - b * s);
      dst[ib] = static_cast<T>(b * c + a * s);
    } else {
      dst[e + half] = static_cast<T>(value(e + half));
    }
  }
}

// Entry (t, i) of the tables: cos and sin of t freq[i] in 64 bits, times gain, rounded once.
constexpr int kTableFreqs = 128;  // frequencies of a launch: 1 KiB of its arguments
struct TableParams {
  double freq[kTableFreqs];
  double gain;
  float* cos_tab;
  float* sin_tab;
  int64_t entries;  // n_pos * count
  int count, half;
};
__global__ __launch_bounds__(256) void rotary_tables_kernel(const TableParams p) {
  const int64_t stride = int64_t(gridDim.x) * 256;
  for (int64_t e = int64_t(blockIdx.x) * 256 + threadIdx.x; e < p.entries; e += stride) {
    const int64_t t = e / p.count;
    const int i = int(e - t * p.count);
    double s, c;
    sincos(double(t) * p.freq[i], &s, &c);
    p.cos_tab[t * p.half + i] = float(c * p.gain);
    p.sin_tab[t * p.half + i] = float(s * p.gain);
  }
}

// Tokens go out in launches of fewer than 2^31 lanes, and pointers move on between them.
template <typename T>
static void launch_rotary(RotaryParams p, int64_t tokens, bool wide, hipStream_t stream) {
  // r / d for r < 2^31: see silu_mul_kernel's launch
  const int l = ilog2(p.rows);
  p.magic = uint32_t((uint64_t(1) << (31 + l)) / p.rows + 1);
  p.shift = 31 + l;
  const int64_t lanes = wide ? int64_t(1) << p.log2_lanes : 64;
  const int64_t slab = (int64_t(1) << 30) / (p.rows * lanes);
  auto at = [](auto* base, int64_t elems, size_t size) {
    using P = decltype(base);
    return base ? reinterpret_cast<P>(reinterpret_cast<uintptr_t>(base) + uintptr_t(elems) * size) : nullptr;
  };
  for (int64_t t0 = 0; t0 < tokens; t0 += slab) {
    RotaryParams s = p;
    s.tokens = uint32_t(tokens - t0 < slab ? tokens - t0 : slab);
    s.q = at(p.q, t0 * p.q_st, sizeof(T));
    s.k = at(p.k, t0 * p.k_st, sizeof(T));
    s.v = at(p.v, t0 * p.v_st, 2);
    s.q_out = at(p.q_out, t0 * p.qo_st, sizeof(T));
    s.k_out = at(p.k_out, t0 * p.ko_st, sizeof(T));
    s.positions = p.positions + t0;
    s.slots = p.slots ? p.slots + t0 : nullptr;
    const int64_t threads = int64_t(s.tokens) * p.rows * lanes;
    const unsigned grid = unsigned((threads + 255) / 256);
    if (!wide)
      rotary_any_kernel<T><<<grid, 256, 0, stream>>>(s);
    else if (p.interleaved)
      rotary_kernel<T, true><<<grid, 256, 0, stream>>>(s);
    else
      rotary_kernel<T, false><<<grid, 256, 0, stream>>>(s);
  }
}

static int check_rotary(const char* fn, int64_t tokens, int n_heads, int n_kv, int head_dim, int rotary_dim,
                        const void* cos_tab, const void* sin_tab, int n_pos, float eps) {
  if (tokens < 0 || n_heads <= 0 || n_kv < 0 || n_pos <= 0)
    return fail(PKV_EINVAL, "%s: bad sizes tokens=%lld n_heads=%d n_kv=%d n_pos=%d", fn, (long long)tokens, n_heads,
                n_kv, n_pos);
  if (int64_t(n_heads) + 2 * int64_t(n_kv) > 65536) return fail(PKV_EINVAL, "%s: more than 65536 heads", fn);
  if (head_dim <= 0 || head_dim > 1024) return fail(PKV_EINVAL, "%s: head_dim %d outside [1, 1024]", fn, head_dim);
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(PKV_EINVAL, "%s: rotary_dim %d must be even and within head_dim %d", fn, rotary_dim, head_dim);
  if (!cos_tab || !sin_tab) return fail(PKV_EINVAL, "%s: null cos/sin table", fn);
  if ((reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab)) & 3u)
    return fail(PKV_EINVAL, "%s: cos/sin tables not 4-byte aligned", fn);
  if (!(eps >= 0.f)) return fail(PKV_EINVAL, "%s: eps must be >= 0", fn);
  return PKV_OK;
}

// Lanes of a head, two chunks of 16 bytes each; at most a wave.
static int lanes_log2(int head_dim, int size) { return ilog2((head_dim * size + 31) / 32); }

}  // namespace pkv

extern "C" int pkv_rotary_tables(const double* freq_gain, int32_t half, int64_t n_pos, float* cos_tab, float* sin_tab,
                                 void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_rotary_tables";
  if (half <= 0 || n_pos <= 0 || n_pos > 0x7fffffff)
    return fail(PKV_EINVAL, "%s: bad sizes half=%d n_pos=%lld", fn, half, (long long)n_pos);
  if (!freq_gain || !cos_tab || !sin_tab) return fail(PKV_EINVAL, "%s: null argument", fn);
  if ((reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab)) & 3u)
    return fail(PKV_EINVAL, "%s: cos/sin tables not 4-byte aligned", fn);
  for (int i0 = 0; i0 < half; i0 += kTableFreqs) {
    TableParams p;
    p.count = half - i0 < kTableFreqs ? half - i0 : kTableFreqs;
    for (int i = 0; i < kTableFreqs; ++i) p.freq[i] = i < p.count ? freq_gain[i0 + i] : 0.0;
    p.gain = freq_gain[half];
    p.cos_tab = cos_tab + i0;
    p.sin_tab = sin_tab + i0;
    p.entries = n_pos * p.count;
    p.half = half;
    const int64_t blocks = (p.entries + 255) / 256;
    rotary_tables_kernel<<<unsigned(blocks < 16384 ? blocks : 16384), 256, 0, static_cast<hipStream_t>(stream)>>>(p);
  }
  return check_launch(fn);
}

extern "C" int pkv_rotate_qk(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh,
                             const int32_t* positions, const float* cos_tab, const float* sin_tab, int32_t n_pos,
                             const void* q_norm_w, const void* k_norm_w, float eps, void* q_out, int64_t qo_st,
                             int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh, int64_t tokens,
                             int32_t n_heads, int32_t n_kv, int32_t head_dim, int32_t rotary_dim,
                             int32_t interleaved, int32_t dtype, int32_t* status, void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_rotate_qk";
  int rc = check_rotary(fn, tokens, n_heads, n_kv, head_dim, rotary_dim, cos_tab, sin_tab, n_pos, eps);
  if (rc) return rc;
  if (dtype != PKV_BF16 && dtype != PKV_FP16 && dtype != PKV_FP32) return fail(PKV_EINVAL, "%s: bad dtype %d", fn, dtype);
  if (tokens == 0) return PKV_OK;
  if (!q || !q_out || !positions || (n_kv > 0 && (!k || !k_out))) return fail(PKV_EINVAL, "%s: null argument", fn);
  const int size = dtype == PKV_FP32 ? 4 : 2;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                          reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out) |
                          reinterpret_cast<uintptr_t>(q_norm_w) | reinterpret_cast<uintptr_t>(k_norm_w);
  if (bases & uintptr_t(size - 1)) return fail(PKV_EINVAL, "%s: a tensor is not aligned to its element", fn);
  const uintptr_t tables = reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab);
  const uint64_t strides = uint64_t(q_st) | uint64_t(q_sh) | uint64_t(k_st) | uint64_t(k_sh) | uint64_t(qo_st) |
                           uint64_t(qo_sh) | uint64_t(ko_st) | uint64_t(ko_sh);
  const int granule = 32 / size;  // two 16-byte chunks
  const bool wide = ((bases | tables) & 15u) == 0 && (strides * size) % 16 == 0 && head_dim % granule == 0 &&
                    head_dim <= 64 * granule &&
                    rotary_dim % granule == 0;
  RotaryParams p = {};
  p.q = q; p.q_st = q_st; p.q_sh = q_sh;
  p.k = k; p.k_st = k_st; p.k_sh = k_sh;
  p.q_out = q_out; p.qo_st = qo_st; p.qo_sh = qo_sh;
  p.k_out = k_out; p.ko_st = ko_st; p.ko_sh = ko_sh;
  p.positions = positions;
  p.cos_tab = cos_tab;
  p.sin_tab = sin_tab;
  p.n_pos = n_pos;
  p.q_norm_w = q_norm_w;
  p.k_norm_w = k_norm_w;
  p.eps = eps;
  p.n_heads = n_heads;
  p.n_kv = n_kv;
  p.head_dim = head_dim;
  p.rotary = rotary_dim;
  p.interleaved = interleaved ? 1 : 0;
  p.rows = uint32_t(n_heads + n_kv);
  p.log2_lanes = lanes_log2(head_dim, size);
  p.status = status;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == PKV_BF16)
    launch_rotary<__bf16>(p, tokens, wide, s);
  else if (dtype == PKV_FP16)
    launch_rotary<_Float16>(p, tokens, wide, s);
  else
    launch_rotary<float>(p, tokens, wide, s);
  return check_launch(fn);
}

extern "C" int pkv_packed_rope_append(const void* qkv, int64_t qkv_st, const int32_t* positions, const int32_t* slots,
                                      const float* cos_tab, const float* sin_tab, int32_t n_pos,
                                      const void* q_norm_w, const void* k_norm_w, float eps, void* q_out,
                                      int64_t qo_st, int64_t qo_sh, void* k_cache, void* v_cache,
                                      int64_t cache_page_stride, int64_t tokens, int32_t n_heads, int32_t n_kv,
                                      int32_t head_dim, int32_t rotary_dim, int32_t interleaved, int32_t page_size,
                                      int32_t num_pages, int32_t* status, void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_packed_rope_append";
  int rc = check_rotary(fn, tokens, n_heads, n_kv, head_dim, rotary_dim, cos_tab, sin_tab, n_pos, eps);
  if (rc) return rc;
  if (head_dim != 64 && head_dim != 128) return fail(PKV_EINVAL, "%s: head_dim %d unsupported (64 or 128)", fn, head_dim);
  if (rotary_dim % 16) return fail(PKV_EINVAL, "%s: rotary_dim %d must be a multiple of 16", fn, rotary_dim);
  if (n_kv <= 0 || num_pages <= 0) return fail(PKV_EINVAL, "%s: bad sizes n_kv=%d num_pages=%d", fn, n_kv, num_pages);
  if (!is_pow2(page_size) || page_size < 16)
    return fail(PKV_EINVAL, "%s: page_size %d must be a power of two >= 16", fn, page_size);
  if (int64_t(num_pages) * page_size > 0x7fffffff) return fail(PKV_EINVAL, "%s: more than 2^31 - 1 cache slots", fn);
  if (tokens == 0) return PKV_OK;
  if (!qkv || !positions || !slots || !q_out || !k_cache || !v_cache) return fail(PKV_EINVAL, "%s: null argument", fn);
  if (cache_page_stride < int64_t(page_size) * n_kv * head_dim || (cache_page_stride % 8) != 0)
    return fail(PKV_EINVAL, "%s: page stride %lld too small or not 16-byte aligned", fn, (long long)cache_page_stride);
  if (!aligned16(qkv) || (qkv_st % 8)) return fail(PKV_EINVAL, "%s: qkv rows must be 16-byte aligned", fn);
  if (!aligned16(k_cache) || !aligned16(v_cache)) return fail(PKV_EINVAL, "%s: k_cache/v_cache not 16-byte aligned", fn);
  if (!aligned16(cos_tab) || !aligned16(sin_tab)) return fail(PKV_EINVAL, "%s: cos/sin tables not 16-byte aligned", fn);
  if ((q_norm_w && !aligned16(q_norm_w)) || (k_norm_w && !aligned16(k_norm_w)))
    return fail(PKV_EINVAL, "%s: norm weights not 16-byte aligned", fn);
  if ((rc = validate_rows(fn, "q_out", q_out, 0, qo_st, qo_sh))) return rc;
  const uint16_t* x = static_cast<const uint16_t*>(qkv);
  RotaryParams p = {};
  p.q = x;
  p.k = x + int64_t(n_heads) * head_dim;
  p.v = x + (int64_t(n_heads) + n_kv) * head_dim;
  p.q_st = p.k_st = p.v_st = qkv_st;
  p.q_sh = p.k_sh = p.v_sh = head_dim;
  p.q_out = q_out; p.qo_st = qo_st; p.qo_sh = qo_sh;
  p.positions = positions;
  p.slots = slots;
  p.cos_tab = cos_tab;
  p.sin_tab = sin_tab;
  p.n_pos = n_pos;
  p.q_norm_w = q_norm_w;
  p.k_norm_w = k_norm_w;
  p.eps = eps;
  p.k_cache = static_cast<uint16_t*>(k_cache);
  p.v_cache = static_cast<uint16_t*>(v_cache);
  p.page_stride = cache_page_stride;
  p.log2_page = ilog2(page_size);
  p.num_pages = num_pages;
  p.n_heads = n_heads;
  p.n_kv = n_kv;
  p.head_dim = head_dim;
  p.rotary = rotary_dim;
  p.interleaved = interleaved ? 1 : 0;
  p.rows = uint32_t(n_heads + 2 * n_kv);
  p.log2_lanes = lanes_log2(head_dim, 2);
  p.status = status;
  launch_rotary<__bf16>(p, tokens, true, static_cast<hipStream_t>(stream));
  return check_launch(fn);
}
