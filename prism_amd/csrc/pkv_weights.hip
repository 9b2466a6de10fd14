// How much attention every cached key got from a packed step's new tokens, for eviction (pkv_key_weights).
//
//   w[slot(t), h]  (+)=  sum over rows r and heads i of h's group that see t  of  exp(scale q[r, i] . k[t, h] - lse[r, i])
//
// lse is what the attention returned, so the softmax needs no second pass and no running maximum: one product, one
// exponential and one sum per (row, key).  The sums run over query rows, so keys are independent of each other: every
// key is summed by one wave (or, for long prompts, by a fixed list of them), in an order that the work list fixes.
#include <algorithm>
#include <cmath>
#include <exception>
#include <vector>

#include "pkv_common.h"
#include "pkv_weights.h"

namespace pkv {
namespace {

struct WeightParams {
  const uint16_t* q;
  const uint16_t* k;
  const float* lse;
  float* w;
  const int32_t* bt;
  const WeightItem* items;
  float* parts;
  int32_t* status;
  int64_t q_st, q_sh, page_stride, lse_st, w_page, bt_stride;
  float scale2;  // softmax scale times log2 e
  int tokens, batch, n_kv, g, log2_page, num_pages, max_blocks, n_parts;
  uint32_t g_mul, g_shift;  // row / g
  uint32_t window;  // a row sees the keys with pos - t < window, unsigned
};

// row / g for 0 <= row < 2^30: with shift = log2 g, rounded up, and mul = ceil(2^(31 + shift) / g), less than 2^32, the product
// exceeds row * 2^(31 + shift) / g by less than row < 2^31, so by less than 1 / g of the quotient's unit.
__device__ __forceinline__ int token_of(const WeightParams& p, int row) {
  return int((uint64_t(uint32_t(row)) * p.g_mul) >> (31 + p.g_shift));
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 frag(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// Workgroups of weigh_few_kernel on a CU at once.  48 sequences of 2500 keys, 28 heads on 4: 2 of them 34 us, 4 30, 6 32
// (too few registers); 16 of 4000 keys with 20 query rows, 40 heads on 8: 31, 29 and 34.
constexpr int kFewPerCu = 4;
constexpr float kLog2e = 1.4426950408889634f;

// A row's denominator in log2; one that saw nothing (-inf) weighs nothing, as one of +inf does.
__device__ __forceinline__ float row_lse2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// The lists are the caller's memory: an item that does not fit the call is skipped.
__device__ __forceinline__ bool fits(const WeightItem& it, const WeightParams& p) {
  return it.tok0 >= 0 && it.n_tok > 0 && it.n_tok <= p.tokens && it.tok0 <= p.tokens - it.n_tok && it.pos0 >= 0 &&
         unsigned(it.seq) < unsigned(p.batch) && it.key0 >= 0 && it.keys > 0 &&
         it.key0 <= (int64_t(p.max_blocks) << p.log2_page) - it.keys && it.row0 >= 0 && it.rows >= 0 &&
         it.rows <= int64_t(it.n_tok) * p.g - it.row0;
}

// The page of key t, -1 where the table has none for it: such a key is not written, and flagged where it is seen.
__device__ __forceinline__ int page_of(const WeightParams& p, const int32_t* row, int t) {
  const int col = t >> p.log2_page;
  const int page = col < p.max_blocks ? row[col] : -1;
  return unsigned(page) < unsigned(p.num_pages) ? page : -1;
}

// Whether some row of positions [pos0, last] sees some key of [t0, t1).
__device__ __forceinline__ bool seen(int pos0, int last, uint32_t window, int t0, int t1) {
  return t0 <= last && t1 - 1 > pos0 - int(window);  // positions are not negative, windows at most 2^31 - 1
}

// Over the 16 lanes of a row, in every lane: rotations within the row, no way through LDS.
template <int CTRL>
__device__ __forceinline__ float add_rotated(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row16_sum(float x) {
  return add_rotated<0x121>(add_rotated<0x122>(add_rotated<0x124>(add_rotated<0x128>(x))));
}

// ---- few query rows: the keys stream past them ----
// Decode tokens and verify rows: the reading of K is all there is to do.  The item's query rows lie in LDS, every wave
// takes a run of 32-key tiles straight into the A operand (16 keys x 32 elements an instruction, a lane's 16 bytes
// of its key's row), the rows are the columns of the product: C[key, row], a lane has 4 keys of one row.  The next tile
// is on its way meanwhile, with its keys' weights so far (read at the end of a tile they cost decode tokens beside chunks
// 5 us of 75).  Memory bounds it: 48 sequences of 2500 keys (4 KV heads of 128, 135 MB) take 37 us, 3.7 TB/s, or 29 where
// the last-level cache holds some; 7 of 50 k keys on one KV head (106 MB) 25.6, 4.2 TB/s.  A large copy runs at 4.9.
template <int HD>
struct FewLds {
  u32x4 q[kWeightFewRows * (HD / 8)];
  float lse[kWeightFewRows];
  int pos[kWeightFewRows];
};
template <int HD>
__device__ __forceinline__ void weigh_few(const WeightParams& p, const WeightItem it, int h, FewLds<HD>& lds) {
  constexpr int KS = HD / 32, CH = HD / 8;  // steps of the contraction, 16-byte chunks of a row
  if (!fits(it, p) || it.rows > kWeightFewRows || it.keys > kWeightFewKeys) {  // also what keeps a wave's page ids in its lanes
    if (threadIdx.x == 0) flag_status(p.status, PKV_STATUS_BAD_PAGE);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* bt = p.bt + it.seq * p.bt_stride;
  const int cols = (it.rows + 15) & ~15;
  for (int i = threadIdx.x; i < cols * CH; i += 256) {
    const int r = i / CH, c = i % CH, row = it.row0 + min(r, it.rows - 1);
    const int j = token_of(p, row), tok = it.tok0 + j, head = h * p.g + row - j * p.g;
    lds.q[r * CH + (c ^ (r & 7))] = ld16(p.q + tok * p.q_st + head * p.q_sh + c * 8);
    if (c == 0) {
      lds.lse[r] = row_lse2(p.lse[tok * p.lse_st + head]);
      lds.pos[r] = r < it.rows ? it.pos0 + j : -(1 << 30);
    }
  }
  __syncthreads();
  // this wave's keys: whole tiles of 32 from the item's first key's tile on
  const int tile0 = it.key0 & ~31, end = it.key0 + it.keys;
  const int tiles = (end - tile0 + 31) >> 5, per = (tiles + 3) >> 2;
  const int first = tile0 + wave * per * 32, last = min(first + per * 32, end);
  if (first >= last) return;
  // page of each 16 keys, one a lane: at most 64 of them, as an item of 3968 keys has at most 125 tiles
  const int mine = page_of(p, bt, min(first + lane * 16, end - 1));
  const int n16 = lane & 15, quad = lane >> 4;
  const int64_t key_st = int64_t(p.n_kv) * HD;
  const int in_page = (1 << p.log2_page) - 1;
  const int last_pos = it.pos0 + it.n_tok - 1;

  // the weights so far come with the keys: lane (quad, i) of the first four of each row of lanes has key quad * 4 + i
  auto load = [&](int t0, u32x4 (&a)[2][KS], float (&old)[2]) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int page = __builtin_amdgcn_readlane(mine, ((t0 - first) >> 4) + s);
      const int row = ((t0 + s * 16) & in_page) + n16;
      const uint16_t* src = p.k + int64_t(max(page, 0)) * p.page_stride + row * key_st + h * HD + quad * 8;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) a[s][ks] = ld16(src + ks * 32);
      const int t = t0 + s * 16 + quad * 4 + n16;
      old[s] = 0.0f;
      if (n16 < 4 && page >= 0 && t < it.fresh) old[s] = p.w[page * p.w_page + (h << p.log2_page) + (t & in_page)];
    }
  };
  u32x4 a[2][KS];
  float old[2];
  load(first, a, old);
  for (int t0 = first; t0 < last; t0 += 32) {
    u32x4 next[2][KS];
    float next_old[2];
    if (t0 + 32 < last) load(t0 + 32, next, next_old);
    float sum[2][4] = {};
    for (int c0 = 0; c0 < cols; c0 += 16) {
      f32x4 acc[2] = {};
      const int r = c0 + n16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const bf16x8 b = frag(lds.q[r * CH + ((ks * 4 + quad) ^ (r & 7))]);
        acc[0] = mfma16(frag(a[0][ks]), b, acc[0]);
        acc[1] = mfma16(frag(a[1][ks]), b, acc[1]);
      }
      const float lse2 = lds.lse[r];
      const int ahead = lds.pos[r] - t0 - quad * 4;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[s][i], p.scale2, -lse2));
          sum[s][i] += uint32_t(ahead - s * 16 - i) < p.window ? e : 0.0f;
        }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[s][i] = row16_sum(sum[s][i]);
      const float got = n16 == 0 ? sum[s][0] : n16 == 1 ? sum[s][1] : n16 == 2 ? sum[s][2] : sum[s][3];
      const int group = t0 + s * 16, t = group + quad * 4 + n16;
      const int page = __builtin_amdgcn_readlane(mine, ((t0 - first) >> 4) + s);
      if (page < 0) {
        if (lane == 0 && group < end && seen(it.pos0, last_pos, p.window, max(group, it.key0), min(group + 16, end)))
          flag_status(p.status, PKV_STATUS_BAD_PAGE);
      } else if (n16 < 4 && t >= it.key0 && t < end) {
        p.w[page * p.w_page + (h << p.log2_page) + (t & in_page)] = t < it.fresh ? old[s] + got : got;
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      old[s] = next_old[s];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) a[s][ks] = next[s][ks];
    }
  }
}

// ---- many query rows: a block of keys stays, the rows go past it ----
// Prompt chunks: 4 waves hold 64 keys each as the A operand, 64 query rows at a time come through LDS (two buffers, one
// barrier a step; 32 a step take 4 % longer) as B, 32 a product: C[key, row], a lane has 16 keys of one row twice, so the
// row's lse is one value a lane and a key's sum stays in the lane until the end.  Exponentials bound it: of 32 x 32 scores
// the products take 256 cycles of the matrix pipe, their 16 multiply-adds, exponentials and sums a lane 384 of the vector
// ALU.  So the products of the second 32 keys are issued between the exponentials of the first, and the other wave of the
// SIMD fills the rest.  Four prompts of 2600 to 3400 tokens (28 heads of 128 on 4): 175 to
// 182 us, 0.76 to 0.79 PFLOP/s, or 198 repeated on one state.
constexpr int kStepRows = 64;
template <int HD>
struct ManyLds {
  u32x4 q[2][kStepRows * (HD / 8)];
  float lse[2][kStepRows];
  int pos[2][kStepRows];
};
template <int HD>
__device__ __forceinline__ void weigh_many(const WeightParams& p, const WeightItem it, int h, ManyLds<HD>& lds) {
  constexpr int KS = HD / 16, CH = HD / 8, LOADS = kStepRows * CH / 256;
  if (!fits(it, p) || it.keys > kWeightBlock || it.part >= p.n_parts) {
    if (threadIdx.x == 0) flag_status(p.status, PKV_STATUS_BAD_PAGE);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* bt = p.bt + it.seq * p.bt_stride;
  const int n32 = lane & 31, half = lane >> 5;
  const int64_t key_st = int64_t(p.n_kv) * HD;
  const int in_page = (1 << p.log2_page) - 1;
  const int end = it.key0 + it.keys, base = it.key0 + wave * 64;
  bf16x8 a[2][KS];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    // keys behind the block's last stand in for it: their sums are not written
    const int t = min(base + s * 32 + n32, end - 1);
    const int page = page_of(p, bt, t);
    const uint16_t* src = p.k + int64_t(max(page, 0)) * p.page_stride + (t & in_page) * key_st + h * HD + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) a[s][ks] = frag(ld16(src + ks * 16));
  }
  // waited for here: in the loop the wait would take in the rows on their way too
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(a[s][ks]));
  const int steps = (it.rows + kStepRows - 1) / kStepRows;
  // held in registers for the loop
  const int rows = __builtin_amdgcn_readfirstlane(it.rows), row0 = __builtin_amdgcn_readfirstlane(it.row0);
  const int pos0 = __builtin_amdgcn_readfirstlane(it.pos0);
  const float* const lse = p.lse + it.tok0 * p.lse_st + h * p.g;
  const uint32_t lse_st = uint32_t(p.lse_st);
  // A thread's rows are a step apart: (token, head) goes on by a quotient and a remainder, and wraps at the group's end.
  // Behind the last row it stays where it is: what it reads there is not counted.
  const int skip_j = kStepRows / p.g, skip_i = kStepRows - skip_j * p.g;
  const int64_t ahead = skip_j * p.q_st + skip_i * p.q_sh, wrap = p.q_st - p.g * p.q_sh;
  const uint16_t* src[LOADS];
  int head[LOADS], left[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int i = threadIdx.x + u * 256, r = i / CH, c = i % CH, row = row0 + max(min(r, rows - 1), 0), j = token_of(p, row);
    src[u] = p.q + (it.tok0 + j) * p.q_st + (h * p.g + row - j * p.g) * p.q_sh + c * 8;
    head[u] = row - j * p.g;
    left[u] = rows - r;  // rows from this one on
  }
  u32x4 stage[LOADS];
  float stage_lse;
  int stage_pos;
  auto fetch = [&](int step) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      stage[u] = ld16(src[u]);
      left[u] -= kStepRows;
      const bool more = left[u] > 0, over = head[u] + skip_i >= p.g;
      head[u] += over ? skip_i - p.g : skip_i;
      src[u] += more ? ahead + (over ? wrap : 0) : 0;
    }
    if (threadIdx.x < kStepRows) {
      const int r = step * kStepRows + threadIdx.x;
      const uint32_t row = row0 + min(r, rows - 1), j = token_of(p, row);
      stage_lse = lse[uint64_t(j) * lse_st + (row - j * p.g)];
      stage_pos = r < rows ? pos0 + int(j) : -(1 << 30);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = threadIdx.x + u * 256, r = i / CH, c = i % CH;
      lds.q[buf][r * CH + (c ^ (r & 7))] = stage[u];
    }
    if (threadIdx.x < kStepRows) {
      lds.lse[buf][threadIdx.x] = row_lse2(stage_lse);
      lds.pos[buf][threadIdx.x] = stage_pos;
    }
  };
  float sum[2][16] = {};
  // scores to weights, all of them or what a row sees
  auto weights = [&](f32x16& c, float lse2) {
#pragma unroll
    for (int i = 0; i < 16; ++i) c[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(c[i], p.scale2, -lse2));
  };
  auto weights_seen = [&](f32x16& c, float lse2, int ahead) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(c[i], p.scale2, -lse2));
      c[i] = uint32_t(ahead - (i & 3) - 8 * (i >> 2)) < p.window ? e : 0.0f;
    }
  };
  // one product, then two scores' worth of the vector ALU
  auto interleave = [] {
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, 32 / KS, 0);
    }
  };
  // Tiles of 32 rows that all see all 64 keys: from the first whose first row is past them to the last whose last row's
  // window still begins before them.
  const int64_t past = int64_t(base + 63 - pos0) * p.g - row0, before = (int64_t(base) + p.window - pos0) * p.g - row0;
  const int full0 = base < end ? int(min(max((past + 31) >> 5, int64_t(0)), int64_t(1 << 30))) : 1 << 30;
  const int full1 = int(min(max(before >> 5, int64_t(0)), int64_t(rows >> 5)));
  // chunk ks * 2 + half of a row lies at that number ^ (row & 7): the exclusive or reaches the lowest three bits alone
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = n32 * CH * 16 + (((i * 2 + half) ^ (n32 & 7)) << 4);
  if (steps > 0) {
    fetch(0);
    put(0);
  }
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    const int buf = step & 1;
    if (step + 1 < steps) fetch(step + 1);
#pragma unroll
    for (int sub = 0; sub < kStepRows / 32; ++sub) {
      const int tile = step * (kStepRows / 32) + sub;
      const float lse2 = lds.lse[buf][sub * 32 + n32];
      const char* const q_tile = reinterpret_cast<const char*>(lds.q[buf] + sub * 32 * CH);
      bf16x8 b[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) b[ks] = frag(*reinterpret_cast<const u32x4*>(q_tile + at[ks & 3] + (ks >> 2) * 128));
      f32x16 acc[2];
      if (tile >= full0 && tile < full1) {
        acc[0] = acc[1] = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc[0] = mfma32(a[0][ks], b[ks], acc[0]);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc[1] = mfma32(a[1][ks], b[ks], acc[1]);
        weights(acc[0], lse2);
        __builtin_amdgcn_sched_group_barrier(0x008, KS, 0);
        interleave();
        weights(acc[1], lse2);
      } else {
        // positions grow with the rows: the first and last row's say what the tile's rows see
        const int pos = lds.pos[buf][sub * 32 + n32];
        const int lo = max(__builtin_amdgcn_readlane(pos, 0), 0), hi = pos0 + token_of(p, row0 + min(tile * 32 + 31, rows - 1));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int t0 = base + s * 32;
          acc[s] = f32x16{};
          if (t0 >= end || !seen(lo, hi, p.window, t0, t0 + 32)) continue;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) acc[s] = mfma32(a[s][ks], b[ks], acc[s]);
          weights_seen(acc[s], lse2, pos - t0 - half * 4);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[s][i] += acc[s][i];
    }
    if (step + 1 < steps) put(buf ^ 1);
    __syncthreads();
  }
  // over the 32 rows of a half wave; then lane i of it has key (i & 3) + 8 (i >> 2) + 4 half of the first 16 sums
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float got = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float x = row16_sum(sum[s][i]);
      x += __shfl_xor(x, 16);
      if (n32 == i) got = x;
    }
    const int t = base + s * 32 + (n32 & 3) + 8 * ((n32 >> 2) & 3) + 4 * half;
    if (n32 >= 16 || t >= end) continue;
    if (it.part >= 0) {
      p.parts[(int64_t(it.part) * p.n_kv + h) * kWeightBlock + (t - it.key0)] = got;
      continue;
    }
    const int page = page_of(p, bt, t);
    if (page < 0) {
      if (seen(it.pos0, it.pos0 + it.n_tok - 1, p.window, t, t + 1)) flag_status(p.status, PKV_STATUS_BAD_PAGE);
      continue;
    }
    float* at = p.w + page * p.w_page + (h << p.log2_page) + (t & in_page);
    *at = t < it.fresh ? *at + got : got;
  }
}

template <int HD>
__global__ __launch_bounds__(256, kFewPerCu) void weigh_few_kernel(const WeightParams p) {
  __shared__ FewLds<HD> lds;
  weigh_few<HD>(p, p.items[blockIdx.x / p.n_kv], blockIdx.x % p.n_kv, lds);
}
template <int HD>
__global__ __launch_bounds__(256) void weigh_many_kernel(const WeightParams p) {
  __shared__ ManyLds<HD> lds;
  weigh_many<HD>(p, p.items[blockIdx.x / p.n_kv], blockIdx.x % p.n_kv, lds);
}
// Both, in turn: the blocks of many rows keep the matrix and vector units busy while the others read.  At the registers of
// the former (250 at head_dim 128) a CU holds two of either, where weigh_few_kernel has four; the list cuts for four.
template <int HD>
__global__ __launch_bounds__(256) void weigh_both_kernel(const WeightParams p, int n_few, int n_many) {
  __shared__ union {
    FewLds<HD> few;
    ManyLds<HD> many;
  } lds;
  const int i = blockIdx.x / p.n_kv, h = blockIdx.x % p.n_kv, pairs = min(n_few, n_many);
  const int at = i < 2 * pairs ? i >> 1 : i - pairs;
  if (i < 2 * pairs ? i & 1 : n_few > n_many)
    weigh_few<HD>(p, p.items[at], h, lds.few);
  else
    weigh_many<HD>(p, p.items[n_few + at], h, lds.many);
}

// The blocks whose rows were split: their partial sums, in the list's order.
__global__ __launch_bounds__(kWeightBlock) void weigh_merge_kernel(const WeightParams p) {
  const int h = blockIdx.x % p.n_kv;
  const WeightItem it = p.items[blockIdx.x / p.n_kv];
  if (!fits(it, p) || it.keys > kWeightBlock || it.part < 0 || it.count < 0 || it.count > p.n_parts - it.part) {
    if (threadIdx.x == 0) flag_status(p.status, PKV_STATUS_BAD_PAGE);
    return;
  }
  if (int(threadIdx.x) >= it.keys) return;
  float got = 0.0f;
  for (int i = 0; i < it.count; ++i) got += p.parts[(int64_t(it.part + i) * p.n_kv + h) * kWeightBlock + threadIdx.x];
  const int t = it.key0 + threadIdx.x;
  const int page = page_of(p, p.bt + it.seq * p.bt_stride, t);
  if (page < 0) {
    if (seen(it.pos0, it.pos0 + it.n_tok - 1, p.window, t, t + 1)) flag_status(p.status, PKV_STATUS_BAD_PAGE);
    return;
  }
  float* at = p.w + page * p.w_page + (h << p.log2_page) + (t & ((1 << p.log2_page) - 1));
  *at = t < it.fresh ? *at + got : got;
}

// ---- the host side ----
// Few rows: pieces of the keys for four workgroups per CU, of 128 keys at least (a tile per wave).
// Many rows: blocks of 256 keys, their rows in pieces for eight workgroups per CU (four prompts: 4 of them 203 us, 8 198,
// 16 212), of 12 steps of 32 rows at least, as a partial's way through memory has its price (4 steps: a prompt of 2048
// tokens 65 us in place of 45, decode tokens beside chunks 86 in place of 68, but one of 512 18 in place of 23; 24 steps:
// 45, 70 and 36).
constexpr int kManyPerCu = 8;
constexpr int kMinSteps = 12;

struct Lists {
  std::vector<WeightItem> few, many, merges;
  int partials = 0;
};

void weight_plan(const int32_t* new_lens, const int32_t* ctx_lens, const int32_t* weighed, int batch, int g, int n_kv,
                 int window, int rows, int cus, Lists& out) {
  struct Seq {
    WeightItem it;
    int first, end;  // its keys
  };
  std::vector<Seq> seqs;
  int64_t few_keys = 0, many_steps = 0;
  int tok0 = 0;
  // the rows of a block that see any of its keys: from the first that reaches its first key, to the last whose window does
  auto block_rows = [&](const Seq& s, int key0, int key1, int& r0, int& r1) {
    const int64_t from = std::max<int64_t>(int64_t(key0) - s.it.pos0, 0);
    int64_t to = s.it.n_tok;
    if (window > 0) to = std::min<int64_t>(to, int64_t(key1 - 1) + window - s.it.pos0);
    r0 = int(std::min<int64_t>(from, s.it.n_tok)) * g;
    r1 = int(std::max<int64_t>(to, 0)) * g;
    if (r1 < r0) r1 = r0;
  };
  for (int b = 0; b < batch; tok0 += new_lens[b], ++b) {
    const int n = new_lens[b], ctx = ctx_lens[b];
    if (n == 0) continue;
    const int count = rows > 0 ? std::min(rows, n) : n;
    Seq s = {};
    s.it.tok0 = tok0 + n - count;
    s.it.n_tok = count;
    s.it.pos0 = ctx + n - count;
    s.it.seq = b;
    s.it.fresh = weighed ? std::min(weighed[b], ctx) : ctx;
    s.it.rows = count * g;
    s.it.part = -1;
    s.first = window > 0 ? std::min<int>(std::max<int64_t>(int64_t(s.it.pos0) - window + 1, 0), s.it.fresh) : 0;
    s.end = ctx + n;
    seqs.push_back(s);
    if (s.it.rows <= kWeightFewRows) {
      few_keys += s.end - s.first;
    } else {
      for (int k = s.first & ~(kWeightBlock - 1); k < s.end; k += kWeightBlock) {
        int r0, r1;
        block_rows(s, std::max(k, s.first), std::min(k + kWeightBlock, s.end), r0, r1);
        many_steps += (r1 - r0 + 31) / 32;
      }
    }
  }
  // the shortest pieces, in whole tiles for each of four waves, that all run at once
  int piece = 128;
  if (few_keys > 0) {
    const int64_t slots = int64_t(cus) * kFewPerCu;
    piece = int(std::min<int64_t>((few_keys * n_kv / slots + 127) / 128 * 128, kWeightFewKeys));
    for (piece = std::max(piece, 128); piece < kWeightFewKeys; piece += 128) {
      int64_t count = 0;
      for (const Seq& s : seqs)
        if (s.it.rows <= kWeightFewRows) count += (s.end - (s.first & ~31) + piece - 1) / piece;
      if (count * n_kv <= slots) break;
    }
  }
  const int64_t many_share = std::max<int64_t>((many_steps * n_kv + int64_t(cus) * kManyPerCu - 1) / (int64_t(cus) * kManyPerCu), kMinSteps);
  for (const Seq& s : seqs) {
    if (s.it.rows <= kWeightFewRows) {
      for (int k = s.first; k < s.end;) {
        WeightItem it = s.it;
        it.key0 = k;
        it.keys = std::min(s.end, (k & ~31) + piece) - k;
        out.few.push_back(it);
        k += it.keys;
      }
      continue;
    }
    for (int k = s.first & ~(kWeightBlock - 1); k < s.end; k += kWeightBlock) {
      WeightItem it = s.it;
      it.key0 = std::max(k, s.first);
      it.keys = std::min(k + kWeightBlock, s.end) - it.key0;
      int r0, r1;
      block_rows(s, it.key0, it.key0 + it.keys, r0, r1);
      const int64_t steps = (r1 - r0 + 31) / 32;
      const int pieces = int(std::max<int64_t>(std::min((steps + many_share - 1) / many_share, steps / kMinSteps), 1));
      const int64_t per = ((steps + pieces - 1) / pieces + 1) / 2 * 64;
      it.row0 = r0;
      it.rows = r1 - r0;
      if (per >= r1 - r0) {
        out.many.push_back(it);
        continue;
      }
      WeightItem merge = it;
      merge.part = out.partials;
      for (int64_t r = r0; r < r1; r += per) {
        it.row0 = int(r);
        it.rows = int(std::min<int64_t>(per, r1 - r));
        it.part = out.partials++;
        out.many.push_back(it);
      }
      merge.count = out.partials - merge.part;
      out.merges.push_back(merge);
    }
  }
  // the longest first: what starts last is short
  std::stable_sort(out.many.begin(), out.many.end(), [](const WeightItem& a, const WeightItem& b) { return a.rows > b.rows; });
}

}  // namespace
}  // namespace pkv

extern "C" int pkv_key_weights_plan(const int32_t* new_lens, const int32_t* ctx_lens, const int32_t* weighed,
                                    int32_t batch, int32_t n_heads, int32_t n_kv, int32_t window, int32_t rows,
                                    int32_t compute_units, int32_t* items, int32_t max_items, int32_t* counts) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_key_weights_plan";
  if (batch < 0 || n_heads <= 0 || n_kv <= 0 || n_heads % n_kv || window < 0 || rows < 0 || compute_units <= 0)
    return fail(PKV_EINVAL, "%s: bad sizes batch=%d n_heads=%d n_kv=%d window=%d rows=%d compute_units=%d", fn, batch,
                n_heads, n_kv, window, rows, compute_units);
  if ((batch > 0 && (!new_lens || !ctx_lens)) || !counts) return fail(PKV_EINVAL, "%s: null argument", fn);
  int64_t tokens = 0;
  for (int b = 0; b < batch; ++b) {
    if (new_lens[b] < 0 || ctx_lens[b] < 0 || int64_t(new_lens[b]) + ctx_lens[b] > (int64_t(1) << 27))
      return fail(PKV_EINVAL, "%s: sequence %d has %d new and %d cached tokens: not negative, and at most 2^27 together",
                  fn, b, new_lens[b], ctx_lens[b]);
    if (weighed && weighed[b] < 0) return fail(PKV_EINVAL, "%s: sequence %d has %d weighed keys", fn, b, weighed[b]);
    tokens += new_lens[b];
  }
  if (tokens * n_heads > (int64_t(1) << 30)) return fail(PKV_EINVAL, "%s: more than 2^30 query rows", fn);
  try {
    Lists lists;
    weight_plan(new_lens, ctx_lens, weighed, batch, n_heads / n_kv, n_kv, window, rows, compute_units, lists);
    const std::vector<WeightItem>* all[] = {&lists.few, &lists.many, &lists.merges};
    int64_t total = 0;
    for (int i = 0; i < 3; ++i) {
      total += int64_t(all[i]->size());
      counts[i] = int32_t(all[i]->size());
    }
    counts[3] = lists.partials;
    if (!items) return PKV_OK;
    if (total > max_items)
      return fail(PKV_ENOSPC, "%s: %lld items do not fit %d", fn, (long long)total, max_items);
    WeightItem* at = reinterpret_cast<WeightItem*>(items);
    for (const auto* list : all) at = std::copy(list->begin(), list->end(), at);
  } catch (const std::exception& e) {  // no memory: no C++ exception leaves a C entry
    return fail(PKV_EINVAL, "%s: %s", fn, e.what());
  }
  return PKV_OK;
}

extern "C" size_t pkv_key_weights_workspace_bytes(int32_t partials, int32_t n_kv) {
  if (partials <= 0 || n_kv <= 0) return 0;
  return size_t(partials) * n_kv * pkv::kWeightBlock * sizeof(float);
}

extern "C" int pkv_key_weights(const void* q, int64_t q_st, int64_t q_sh, const void* k_cache, int64_t cache_page_stride,
                               const float* lse, int64_t lse_st, float* weights, int64_t weights_page_stride,
                               const int32_t* block_table, int64_t bt_stride, const int32_t* items, int32_t n_few,
                               int32_t n_many, int32_t n_merges, int32_t partials, void* workspace,
                               size_t workspace_bytes, int32_t tokens, int32_t batch, int32_t n_heads, int32_t n_kv,
                               int32_t head_dim, int32_t page_size, int32_t num_pages, int32_t max_blocks,
                               int32_t window, float softmax_scale, int32_t* status, void* stream) {
  using namespace pkv;
  clear_error();
  const char* fn = "pkv_key_weights";
  if (tokens < 0 || n_few < 0 || n_many < 0 || n_merges < 0 || partials < 0 || window < 0)
    return fail(PKV_EINVAL, "%s: bad sizes tokens=%d n_few=%d n_many=%d n_merges=%d partials=%d window=%d", fn, tokens,
                n_few, n_many, n_merges, partials, window);
  if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv)
    return fail(PKV_EINVAL, "%s: n_heads %d must be a multiple of n_kv %d", fn, n_heads, n_kv);
  int rc = validate_paged(fn, k_cache, k_cache, cache_page_stride, block_table, bt_stride, block_table, batch, n_kv,
                          head_dim, page_size, num_pages, max_blocks);
  if (rc) return rc;
  if ((rc = validate_rows(fn, "q", q, 0, q_st, q_sh))) return rc;
  if (!q || !lse || !weights) return fail(PKV_EINVAL, "%s: null q, lse or weights", fn);
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return fail(PKV_EINVAL, "%s: bad softmax_scale", fn);
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(weights)) & 3u)
    return fail(PKV_EINVAL, "%s: lse/weights not 4-byte aligned", fn);
  if (q_st < 0 || q_sh < 0 || q_st > 0x7fffffff || q_sh > 0x7fffffff || lse_st > 0x7fffffff)
    return fail(PKV_EINVAL, "%s: strides of q or lse past 2^31 elements", fn);
  if (lse_st < n_heads || weights_page_stride < int64_t(n_kv) * page_size)
    return fail(PKV_EINVAL, "%s: lse or weights rows overlap", fn);
  if (n_few + int64_t(n_many) + n_merges == 0) return PKV_OK;
  if (!items || !aligned16(items)) return fail(PKV_EINVAL, "%s: work list null or not 16-byte aligned", fn);
  if ((n_few + int64_t(n_many) + n_merges) * n_kv * 256 > 0x7fffffff) return fail(PKV_EINVAL, "%s: too many work items", fn);
  const size_t need = pkv_key_weights_workspace_bytes(partials, n_kv);
  if (need > 0 && (!workspace || !aligned16(workspace)))
    return fail(PKV_EINVAL, "%s: workspace null or not 16-byte aligned", fn);
  if (need > 0 && workspace_bytes < need)
    return fail(PKV_ENOSPC, "%s: workspace %zu bytes < %zu needed", fn, workspace_bytes, need);
  WeightParams p;
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k_cache);
  p.lse = lse;
  p.w = weights;
  p.bt = block_table;
  p.items = reinterpret_cast<const WeightItem*>(items);
  p.parts = static_cast<float*>(workspace);
  p.status = status;
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.page_stride = cache_page_stride;
  p.lse_st = lse_st;
  p.w_page = weights_page_stride;
  p.bt_stride = bt_stride;
  p.scale2 = float(double(softmax_scale) * 1.4426950408889634);
  p.tokens = tokens;
  p.batch = batch;
  p.n_kv = n_kv;
  p.g = n_heads / n_kv;
  p.g_shift = uint32_t(ilog2(p.g));
  p.g_mul = uint32_t(((uint64_t(1) << (31 + p.g_shift)) + p.g - 1) / p.g);
  p.log2_page = ilog2(page_size);
  p.num_pages = num_pages;
  p.max_blocks = max_blocks;
  p.n_parts = partials;
  p.window = window > 0 ? uint32_t(window) : 0x7fffffffu;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (n_few > 0 && n_many > 0) {
    auto* kernel = head_dim == 128 ? weigh_both_kernel<128> : weigh_both_kernel<64>;
    kernel<<<unsigned(n_few + n_many) * n_kv, 256, 0, s>>>(p, n_few, n_many);
  } else if (n_few > 0) {
    auto* kernel = head_dim == 128 ? weigh_few_kernel<128> : weigh_few_kernel<64>;
    kernel<<<unsigned(n_few) * n_kv, 256, 0, s>>>(p);
  } else if (n_many > 0) {
    auto* kernel = head_dim == 128 ? weigh_many_kernel<128> : weigh_many_kernel<64>;
    kernel<<<unsigned(n_many) * n_kv, 256, 0, s>>>(p);
  }
  p.items += n_few + n_many;
  if (n_merges > 0) weigh_merge_kernel<<<unsigned(n_merges) * n_kv, kWeightBlock, 0, s>>>(p);
  return check_launch(fn);
}
