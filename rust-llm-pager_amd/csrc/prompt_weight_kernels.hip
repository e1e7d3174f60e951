// Attention weights that the last `window` queries of a prompt give each of its tokens:
//
//   w[b, kv, j] = sum over queries i and the group's heads r of
//                 exp(s(r, i, j)) / sum_j' exp(s(r, i, j')),   s = scale q . k (softcapped),
//                 j and j' in [lo, tokens - window + i]
//
// Two sweeps over the scores, both on v_mfma_f32_32x32x16. The queries of a KV head's group make up
// its rows, query by query: row r = i * n_rep + head.
//   statistics  S^T[32 keys x 32 rows] = K . Q^T, the rows in registers, the keys through LDS: a
//               lane holds 16 keys of one row, so the running maximum and sum are its own scalars.
//   sums        S[32 rows x 32 keys] = Q . K^T, the keys in registers, the rows through LDS: a lane
//               holds 16 rows of one key and adds exp2(s - norm[row]) up, norm = m + log2(l).
// Nothing is added by atomics: the same inputs give the same sums.
//
// Bound by the matrix cores, the vector unit and LDS together: a score costs 2 D flops, one exponential
// (v_exp_f32, 8 cycles a wave) and two or three plain operations (4 cycles each), 544 and 590 cycles
// a wave and 2048 scores at head dim 128, and 8 KB of operands from LDS, which two waves per SIMD only
// partly overlap. 8192 tokens, all of them queries, 32/8 heads, D 128 (275 GF a sweep): 583 us a call,
// 0.94 PFLOP/s over both sweeps where a large matrix product of the library reaches 1.27 (the first form of
// these kernels: 2333 us). With parts taken out of the two sweeps (284 and 296 us then): no LDS operands 189
// and 197, no products 213 and 221, no exponentials 268 and 280, no staging 255 and 243.
// Where a step waits matters most: the operands of the next 32 rows are read under the fold of the last,
// the next tile goes to the other LDS buffer under the last step, and the exponentials come 16 at a time
// (one after the other each waited for its own). A window of few queries has few tiles a workgroup and is
// bound by latency, the start of a workgroup and a barrier a tile, by no unit: 65536 tokens and 64 queries,
// 32/4 heads, D 64: 33 + 4.7 + 32 us, matrix cores 18% and vector units 54% busy; two rows of 4133 tokens and 32
// queries, 28/4 heads, D 128: 10 + 3 + 10 us.
// With a softcap, a tanhf per score and sweep costs more than all else: these take 124 and 31 us a call (63 and 20
// without), the 8192 x 8192 scores 1768 (576).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "cache_device.h"

namespace pgr {
namespace {

constexpr int kTile = 128;  // keys (statistics) or rows (sums) in LDS

struct ScoreScale {
  float c;          // log2 units per unit of the (softcapped) score
  float cap_scale;  // softcap: scale / cap, else 0
};

// x / n_rep for 0 <= x < 2^32 / 16: exact with magic = floor(2^32 / n_rep) + 1 (0: n_rep is 1). An
// ordinary division is some thirty instructions, and a tile's rows take one per 16-byte piece.
__device__ __forceinline__ int div_rep(int x, uint32_t magic) {
  return magic == 0 ? x : (int)__umulhi((uint32_t)x, magic);
}
__device__ __forceinline__ uint32_t rep_magic(int n_rep) {
  return n_rep == 1 ? 0u : 0xffffffffu / (uint32_t)n_rep + 1u;
}

// The (softcapped) score in units of `c`.
template <bool kCap>
__device__ __forceinline__ float raw_score(float s, const ScoreScale& sc) {
  return kCap ? tanhf(s * sc.cap_scale) : s;
}

// One tile of rows on its way to LDS: 16-byte pieces in registers, so that a later tile's loads run
// under the current one's products.
template <int D>
struct Stage {
  static constexpr int kStride = D + 8, kPieces = D / 8, kPer = kTile * kPieces / 256;
  static constexpr int kRound = 256 / kPieces;  // rows that the workgroup reads at once
  u32x4 v[kPer];

  __device__ __forceinline__ static int first_row() { return (int)threadIdx.x / kPieces; }
  __device__ __forceinline__ static int element() { return (int)threadIdx.x % kPieces * 8; }

  // A whole tile whose rounds lie `step` elements apart; own: the thread's piece of the first one. An
  // addition a round instead of a division and two products a piece, which were a fifth of the vector
  // instructions of the sums: 302 -> 295 us at 8192 tokens and queries (32/8 heads, D 128), 30.5 -> 29.4 at
  // 65536 tokens and 64 queries (32/4, D 64). The keys' tiles have less to save: 297 with it and without.
  __device__ __forceinline__ void fetch_even(const uint16_t* own, uint64_t step) {
#pragma unroll
    for (int x = 0; x < kPer; ++x) v[x] = *reinterpret_cast<const u32x4_e*>(own + x * step);
  }
  // offset(i): element offset of row i from `base`; rows from `valid` on repeat the last one (what they
  // give is masked, or weighs nothing, or is not stored).
  template <class F>
  __device__ __forceinline__ void fetch(const uint16_t* base, int valid, F offset) {
#pragma unroll
    for (int x = 0; x < kPer; ++x)
      v[x] = *reinterpret_cast<const u32x4_e*>(base + offset(min(x * kRound + first_row(), valid - 1)) + element());
  }
  __device__ __forceinline__ void put(uint16_t* lds) const {
    uint16_t* const to = lds + first_row() * kStride + element();
#pragma unroll
    for (int x = 0; x < kPer; ++x) *reinterpret_cast<u32x4*>(to + x * kRound * kStride) = v[x];
  }
};

// The lane's part of 32 LDS rows: the first operand of a step's products. All of it is asked for at
// once, and a step ahead: the products then wait for nothing.
template <int D>
__device__ __forceinline__ void read_rows(u32x4 (&r)[D / 16], const uint16_t* lds_row) {
#pragma unroll
  for (int c = 0; c < D / 16; ++c) r[c] = *reinterpret_cast<const u32x4*>(lds_row + 16 * c);
}

template <class Ty, int D, int kN>
__device__ __forceinline__ void product(f32x16 (&s)[kN], const u32x4 (&rows)[D / 16], const u32x4 (&own)[kN][D / 16]) {
#pragma unroll
  for (int g = 0; g < kN; ++g) s[g] = f32x16{};
#pragma unroll
  for (int c = 0; c < D / 16; ++c)
#pragma unroll
    for (int g = 0; g < kN; ++g) s[g] = Ty::mma32(rows[c], own[g][c], s[g]);
}

template <int D>
__device__ __forceinline__ void load_own(u32x4 (&r)[D / 16], const uint16_t* row, int half) {
#pragma unroll
  for (int c = 0; c < D / 16; ++c) r[c] = *reinterpret_cast<const u32x4_e*>(row + 16 * c + 8 * half);
}

// The sum of 16 values, as four chains: one chain would wait for each addition.
__device__ __forceinline__ float sum16(const float (&p)[16]) {
  float t[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
  for (int x = 4; x < 16; ++x) t[x & 3] += p[x];
  return (t[0] + t[1]) + (t[2] + t[3]);
}

// p[x] = exp2(s[x] * c - ref(x)). The steps are kept apart: left to itself the compiler makes one
// value after the other in one register, and each waits for the exponential before it.
template <class F>
__device__ __forceinline__ void exp_all(float (&p)[16], const f32x16& s, float c, F ref) {
#pragma unroll
  for (int x = 0; x < 16; ++x) p[x] = fmaf(s[x], c, -ref(x));
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int x = 0; x < 16; ++x) p[x] = __builtin_amdgcn_exp2f(p[x]);
  __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// kRowWaves 4: the waves hold rows of their own and all take every key; 1: they hold the same rows
// and take a quarter of the keys each. Grid (batch x KV heads, key splits, row blocks): the KV head
// varies fastest, so that workgroups of one head tend to share an XCD's L2, and the blocks of the
// last rows, which attend to most, start first.
template <class Ty, int D, int kN, int kRowWaves, bool kCap>
__global__ __launch_bounds__(256) void prompt_stats_kernel(PromptWeightLaunch a, ScoreScale sc) {
  typedef Stage<D> S;
  constexpr int kSubs = kRowWaves == 4 ? kTile / 32 : 1;  // steps of a wave per tile
  __shared__ __align__(16) uint16_t lds[2][kTile * S::kStride];
  __shared__ float2 part[4][kN * 32];
  const int n_rep = a.hq / a.hkv, rows = a.window * n_rep;
  const uint32_t magic = rep_magic(n_rep), q_h = (uint32_t)a.qs.h, q_t = (uint32_t)a.qs.t, k_t = (uint32_t)a.ks.t;
  const int bh = blockIdx.x, b = bh / a.hkv, h = bh - b * a.hkv;
  const int wave = wave_index(), lane = threadIdx.x & 63, half = lane >> 5, j = lane & 31;
  const int lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
  const uint16_t* qb = static_cast<const uint16_t*>(a.q) + b * a.qs.b + (int64_t)h * n_rep * a.qs.h;
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.ks.b + h * a.ks.h;

  const int wg_row = (int)(gridDim.z - 1 - blockIdx.z) * kRowWaves * kN * 32;
  const int wave_row = wg_row + (kRowWaves == 4 ? wave * kN * 32 : 0);
  u32x4 own[kN][D / 16];
  int last[kN];  // the last column that the lane's row attends to (past the last row: that one again)
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    const int r = min(wave_row + g * 32 + j, rows - 1), i = div_rep(r, magic);
    last[g] = a.tokens - a.window + i;
    load_own<D>(own[g], qb + (uint64_t)(uint32_t)(r - i * n_rep) * q_h + (uint64_t)(uint32_t)i * q_t, half);
  }
  // The last keys that any row of the workgroup, any row of the wave, and every row of the wave attends to.
  auto last_of = [&](int r) { return a.tokens - a.window + div_rep(min(r, rows - 1), magic); };
  const int wg_last = last_of(wg_row + kRowWaves * kN * 32 - 1);
  const int any = last_of(wave_row + kN * 32 - 1), every = last_of(wave_row);

  // This split's tiles of [lo, wg_last].
  const int t_lo = lo / kTile, t_hi = wg_last / kTile + 1;
  const int per = (max(t_hi - t_lo, 0) + a.plan.key_splits - 1) / a.plan.key_splits;
  const int t_begin = t_lo + (int)blockIdx.y * per, t_end = min(t_begin + per, t_hi);

  float m[kN], l[kN];
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    m[g] = kMinusInf;
    l[g] = 0.f;
  }
  S st;
  auto fetch = [&](int tile) {
    st.fetch(kb + (int64_t)tile * kTile * a.ks.t, a.tokens - tile * kTile, [&](int i) { return (uint64_t)i * k_t; });
  };
  // Folds the scores of 32 keys into the rows' statistics; masked: some row does not attend to some key.
  auto fold = [&](f32x16 (&s)[kN], int k0, auto masked) {
#pragma unroll
    for (int g = 0; g < kN; ++g) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s[g][x] = raw_score<kCap>(s[g][x], sc);
        if constexpr (decltype(masked)::value) {
          const int key = k0 + 8 * (x / 4) + 4 * half + (x & 3);
          s[g][x] = key < lo || key > last[g] ? kMinusInf : s[g][x];
        }
      }
      float top = m[g], top2 = s[g][15];
#pragma unroll
      for (int x = 0; x < 14; x += 4) {
        top = fmaxf(fmaxf(top, s[g][x]), s[g][x + 1]);
        if (x + 3 < 15) top2 = fmaxf(fmaxf(top2, s[g][x + 2]), s[g][x + 3]);
      }
      top = fmaxf(fmaxf(top, top2), s[g][14]);
      const float ref = top == kMinusInf ? 0.f : top * sc.c;  // (scores may be -inf without a mask)
      float p[16];
      exp_all(p, s[g], sc.c, [&](int) { return ref; });
      l[g] = fmaf(l[g], __builtin_amdgcn_exp2f(fmaf(m[g], sc.c, -ref)), sum16(p));
      m[g] = top;
    }
  };
  u32x4 keys[D / 16];
  const int sub0 = kRowWaves == 4 ? 0 : wave, at = j * S::kStride + 8 * half;
  if (t_begin < t_end) fetch(t_begin);
#pragma unroll
  for (int g = 0; g < kN; ++g) arrived(own[g]);
  if (t_begin < t_end) {
    st.put(lds[0]);
    if (t_begin + 1 < t_end) fetch(t_begin + 1);
    __syncthreads();
    read_rows<D>(keys, lds[0] + sub0 * 32 * S::kStride + at);
  }
  for (int tile = t_begin; tile < t_end; ++tile) {
    uint16_t* const here = lds[(tile - t_begin) & 1];
    uint16_t* const there = lds[(tile - t_begin + 1) & 1];
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      const int k0 = tile * kTile + (sub0 + sub) * 32;
      const bool some = k0 <= any;  // otherwise no row of the wave attends to these keys
      f32x16 s[kN];
      if (some) product<Ty, D, kN>(s, keys, own);
      __builtin_amdgcn_sched_barrier(0);
      if (sub + 1 < kSubs) {
        read_rows<D>(keys, here + (sub + 1) * 32 * S::kStride + at);
      } else if (tile + 1 < t_end) {
        st.put(there);
        if (tile + 2 < t_end) fetch(tile + 2);
        __syncthreads();
        read_rows<D>(keys, there + sub0 * 32 * S::kStride + at);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (k0 < lo || k0 + 31 > every) {
        if (some) fold(s, k0, std::true_type{});
      } else {
        fold(s, k0, std::false_type{});
      }
    }
  }
  // The halves of the wave hold other keys of the same rows; so do the waves where they share rows.
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    const float m2 = __shfl_xor(m[g], 32), l2 = __shfl_xor(l[g], 32);
    const float mm = fmaxf(m[g], m2);
    const float ref = mm == kMinusInf ? 0.f : mm * sc.c;
    const float ll = l[g] * __builtin_amdgcn_exp2f(fmaf(m[g], sc.c, -ref)) +
                     l2 * __builtin_amdgcn_exp2f(fmaf(m2, sc.c, -ref));
    if (half == 0) part[wave][g * 32 + j] = float2{mm * sc.c, ll};
  }
  __syncthreads();
  float2* out = a.stats + ((int64_t)blockIdx.y * a.batch * a.hkv + bh) * rows;
  for (int i = threadIdx.x; i < kRowWaves * kN * 32; i += 256) {
    if (wg_row + i >= rows) continue;
    if (kRowWaves == 4) {
      out[wg_row + i] = part[i / (kN * 32)][i % (kN * 32)];
    } else {
      float mm = kMinusInf, ll = 0.f;
      for (int w = 0; w < 4; ++w) mm = fmaxf(mm, part[w][i].x);
      const float ref = mm == kMinusInf ? 0.f : mm;
      for (int w = 0; w < 4; ++w) ll += part[w][i].y * __builtin_amdgcn_exp2f(part[w][i].x - ref);
      out[wg_row + i] = float2{mm, ll};
    }
  }
}

// norm = m + log2(l) over splits from, from + step, ... of row i of n, eight loads in flight; as (m, l).
__device__ __forceinline__ float2 join_stats(const float2* stats, int64_t n, int64_t i, int splits, int from, int step) {
  float m = kMinusInf, l = 0.f;
  for (int s0 = from; s0 < splits; s0 += 8 * step) {
    float2 p[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int s = s0 + step * x;
      p[x] = stats[(s < splits ? s : s0) * n + i];
      if (s >= splits) p[x] = float2{kMinusInf, 0.f};
    }
    float top = m;
#pragma unroll
    for (int x = 0; x < 8; ++x) top = fmaxf(top, p[x].x);
    const float ref = top == kMinusInf ? 0.f : top;
    l *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
    for (int x = 0; x < 8; ++x) l += p[x].y * __builtin_amdgcn_exp2f(p[x].x - ref);
    m = top;
  }
  return float2{m, l};
}

// +inf for a row that attends to nothing. (One float for both: a row's weights share its rounding, up to 2^-20
// relative where it is 16 to 32. The sums of 32, 64 and 8192 queries are within 2.5e-7, 3.2e-7 and 2.5e-7 of 64
// bits, torch's float32 form within 4e-7, 1.4e-7 and 0.7e-7. Apart, each row would be two reads from LDS.)
__device__ __forceinline__ float norm_of(float2 p) {
  return p.y == 0.f ? -kMinusInf : (p.x == kMinusInf ? 0.f : p.x) + __builtin_amdgcn_logf(p.y);
}

// The norms of 64 rows a workgroup, each wave a quarter of the splits. (Two grid dimensions: one ends at 2^32
// threads, here 2^30 rows, and a launch past it runs too few workgroups without an error.)
__global__ __launch_bounds__(256) void prompt_norm_kernel(PromptWeightLaunch a, int64_t n) {
  __shared__ float2 part[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 64 + lane;
  part[wave][lane] = join_stats(a.stats, n, i < n ? i : n - 1, a.plan.key_splits, wave, 4);
  __syncthreads();
  if (wave != 0 || i >= n) return;
  a.norm[i] = norm_of(join_stats(&part[0][0], 64, lane, 4, 0, 1));
}

// Grid (batch x KV heads, row splits, key blocks): as above; the first keys, which most rows attend
// to, start first.
template <class Ty, int D, int kN, bool kCap>
__global__ __launch_bounds__(256) void prompt_sums_kernel(PromptWeightLaunch a, ScoreScale sc) {
  typedef Stage<D> S;
  constexpr int kSubs = kTile / 32, kNever = 0x7fffffff;
  __shared__ __align__(16) uint16_t lds[2][kTile * S::kStride];
  __shared__ __align__(16) float norm_s[2][kTile];
  const int n_rep = a.hq / a.hkv, rows = a.window * n_rep, before = a.tokens - a.window;
  const uint32_t magic = rep_magic(n_rep), q_h = (uint32_t)a.qs.h, q_t = (uint32_t)a.qs.t;
  const int bh = blockIdx.x, b = bh / a.hkv, h = bh - b * a.hkv;
  const int wave = wave_index(), lane = threadIdx.x & 63, half = lane >> 5, j = lane & 31;
  const int lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
  const uint16_t* qb = static_cast<const uint16_t*>(a.q) + b * a.qs.b + (int64_t)h * n_rep * a.qs.h;
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.ks.b + h * a.ks.h;
  const float* norm = a.norm + (int64_t)bh * rows;
  const float2* stats = a.stats + (int64_t)bh * rows;

  const int wg_key = (int)blockIdx.z * 4 * kN * 32, wave_key = wg_key + wave * kN * 32;
  u32x4 own[kN][D / 16];
  float sum[kN];
  int from[kN];  // the first row that attends to the lane's key (padding: none, whatever the key holds)
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    const int key = wave_key + g * 32 + j;
    load_own<D>(own[g], kb + min(key, a.tokens - 1) * a.ks.t, half);
    sum[g] = 0.f;
    from[g] = key < lo || key >= a.tokens ? kNever : max(key - before, 0) * n_rep;
  }
  // The first rows that attend to the workgroup's first key, to the wave's first and to all of the wave's.
  const int first = max(wg_key - before, 0) * n_rep, any = max(wave_key - before, 0) * n_rep;
  const int every = wave_key < lo ? kNever : max(wave_key + kN * 32 - 1 - before, 0) * n_rep;
  const int t_lo = first / kTile, t_hi = (rows + kTile - 1) / kTile;
  const int per = (max(t_hi - t_lo, 0) + a.plan.row_splits - 1) / a.plan.row_splits;
  const int t_begin = t_lo + (int)blockIdx.y * per, t_end = min(t_begin + per, t_hi);

  S st;
  float nm_next = 0.f;
  auto row_offset = [&](int r) {
    const int i = div_rep(r, magic);
    return (uint64_t)(uint32_t)(r - i * n_rep) * q_h + (uint64_t)(uint32_t)i * q_t;
  };
  // Rounds of whole queries lie evenly: heads that divide a round's rows.
  const int round_queries = div_rep(S::kRound, magic);
  const bool even = round_queries * n_rep == S::kRound;
  const uint16_t* const mine = qb + row_offset(S::first_row()) + S::element();
  auto fetch = [&](int tile) {
    const int row0 = tile * kTile;
    if (even && row0 + kTile <= rows) {
      const uint64_t step = (uint64_t)(uint32_t)round_queries * q_t;
      st.fetch_even(mine + (uint64_t)(uint32_t)(tile * S::kPer) * step, step);
    } else {
      st.fetch(qb, rows - row0, [&](int i) { return row_offset(row0 + i); });
    }
    if (threadIdx.x < kTile) {
      const int r = min(row0 + (int)threadIdx.x, rows - 1);
      if (a.plan.norm_apart)
        nm_next = norm[r];
      else
        nm_next = norm_of(join_stats(stats, (int64_t)a.batch * a.hkv * rows, r, a.plan.key_splits, 0, 1));
      if (row0 + (int)threadIdx.x >= rows) nm_next = -kMinusInf;
    }
  };
  auto put = [&](int buffer) {
    st.put(lds[buffer]);
    if (threadIdx.x < kTile) norm_s[buffer][threadIdx.x] = nm_next;
  };
  // Adds the probabilities of 32 rows up; masked: some row does not attend to some key.
  auto fold = [&](const f32x16 (&s)[kN], const f32x4 (&nm)[4], int r0, auto masked) {
#pragma unroll
    for (int g = 0; g < kN; ++g) {
      float p[16];
      f32x16 x16;
#pragma unroll
      for (int x = 0; x < 16; ++x) x16[x] = raw_score<kCap>(s[g][x], sc);
      exp_all(p, x16, sc.c, [&](int x) { return nm[x / 4][x & 3]; });
      if constexpr (decltype(masked)::value) {
#pragma unroll
        for (int x = 0; x < 16; ++x) p[x] = r0 + 8 * (x / 4) + 4 * half + (x & 3) < from[g] ? 0.f : p[x];
      }
      sum[g] += sum16(p);  // 16 rows at a time, so that long sums of small terms lose less
    }
  };
  u32x4 q[D / 16];
  const int at = j * S::kStride + 8 * half;
  if (t_begin < t_end) fetch(t_begin);
#pragma unroll
  for (int g = 0; g < kN; ++g) arrived(own[g]);
  if (t_begin < t_end) {
    put(0);
    if (t_begin + 1 < t_end) fetch(t_begin + 1);
    __syncthreads();
    read_rows<D>(q, lds[0] + at);
  }
  for (int tile = t_begin; tile < t_end; ++tile) {
    const int here = (tile - t_begin) & 1, there = here ^ 1;
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub) {
      const int r0 = tile * kTile + sub * 32;
      const bool some = r0 + 31 >= any;  // otherwise none of these rows attends to a key of the wave
      f32x16 s[kN];
      f32x4 nm[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) nm[x] = *reinterpret_cast<const f32x4*>(norm_s[here] + sub * 32 + 8 * x + 4 * half);
      if (some) product<Ty, D, kN>(s, q, own);
      __builtin_amdgcn_sched_barrier(0);
      if (sub + 1 < kSubs) {
        read_rows<D>(q, lds[here] + (sub + 1) * 32 * S::kStride + at);
      } else if (tile + 1 < t_end) {
        put(there);
        if (tile + 2 < t_end) fetch(tile + 2);
        __syncthreads();
        read_rows<D>(q, lds[there] + at);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (r0 < every) {
        if (some) fold(s, nm, r0, std::true_type{});
      } else {
        fold(s, nm, r0, std::false_type{});
      }
    }
  }
  float* out = a.plan.row_splits == 1 ? a.out : a.partial + (int64_t)blockIdx.y * a.batch * a.hkv * a.tokens;
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    const float total = sum[g] + __shfl_xor(sum[g], 32);
    const int key = wave_key + g * 32 + j;
    if (half == 0 && key < a.tokens) out[(int64_t)bh * a.tokens + key] = total;
  }
}

__global__ __launch_bounds__(256) void prompt_join_kernel(PromptWeightLaunch a, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float x = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.plan.row_splits; ++s) x += a.partial[s * n + i];
  a.out[i] = x;
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

template <class Ty, int D, int kN, bool kCap>
hipError_t run(const PromptWeightLaunch& p, const ScoreScale& sc, hipStream_t stream) {
  const int rows = p.window * (p.hq / p.hkv), own = kN * 32;
  const unsigned bh = (unsigned)(p.batch * p.hkv);
  const dim3 stats(bh, (unsigned)p.plan.key_splits, (unsigned)ceil_div(rows, p.plan.row_waves * own));
  if (p.plan.row_waves == 1)
    prompt_stats_kernel<Ty, D, kN, 1, kCap><<<stats, 256, 0, stream>>>(p, sc);
  else
    prompt_stats_kernel<Ty, D, kN, 4, kCap><<<stats, 256, 0, stream>>>(p, sc);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.plan.norm_apart) {
    const int64_t n = (int64_t)bh * rows;
    const int64_t blocks = (n + 63) / 64, most = 1 << 20;
    const dim3 grid((unsigned)std::min(blocks, most), (unsigned)ceil_div(blocks, most));
    prompt_norm_kernel<<<grid, 256, 0, stream>>>(p, n);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const dim3 sums(bh, (unsigned)p.plan.row_splits, (unsigned)ceil_div(p.tokens, 4 * own));
  prompt_sums_kernel<Ty, D, kN, kCap><<<sums, 256, 0, stream>>>(p, sc);
  e = hipGetLastError();
  if (e != hipSuccess || p.plan.row_splits == 1) return e;
  const int64_t m = (int64_t)bh * p.tokens;
  prompt_join_kernel<<<(unsigned)((m + 255) / 256), 256, 0, stream>>>(p, m);
  return hipGetLastError();
}

template <class Ty, int D>
hipError_t run_cap(const PromptWeightLaunch& p, hipStream_t stream) {
  const bool cap = p.softcap > 0.f;
  const ScoreScale sc = cap ? ScoreScale{p.softcap * kLog2e, p.scale / p.softcap} : ScoreScale{p.scale * kLog2e, 0.f};
  if constexpr (D == 128) {
    if (p.plan.groups == 2) return cap ? run<Ty, D, 2, true>(p, sc, stream) : run<Ty, D, 2, false>(p, sc, stream);
  }
  return cap ? run<Ty, D, 1, true>(p, sc, stream) : run<Ty, D, 1, false>(p, sc, stream);
}

template <class Ty>
hipError_t run_dim(const PromptWeightLaunch& p, hipStream_t stream) {
  switch (p.d) {
    case 16: return run_cap<Ty, 16>(p, stream);
    case 32: return run_cap<Ty, 32>(p, stream);
    case 64: return run_cap<Ty, 64>(p, stream);
    case 128: return run_cap<Ty, 128>(p, stream);
    default: return run_cap<Ty, 256>(p, stream);
  }
}

}  // namespace

PromptWeightPlan prompt_weight_plan(int batch, int hq, int hkv, int tokens, int window, int d) {
  PromptWeightPlan plan;
  const int64_t rows = (int64_t)window * (hq / hkv), bh = (int64_t)batch * hkv;
  // Two groups of 32 per wave at head dim 128 where that still leaves two workgroups for every CU:
  // each operand read from LDS then feeds two products (8192 tokens and queries, 32/8 heads: 341 + 356
  // us against 402 + 427 with one group; two batch rows of 4133 tokens and 32 queries, 28/4 heads, where
  // it does not: 12.1 + 12.3 against 10.4 + 11.1). At head dim 64 one group is as fast (35 + 36 against
  // 42 + 35 us at 65536 tokens and 64 queries, 32/4 heads).
  plan.groups = d == 128 && ceil_div(rows, 256) * bh * ceil_div(tokens, 2048) >= 512 ? 2 : 1;
  const int64_t own = 32 * plan.groups;
  // Rows that one wave holds are shared by the four, a quarter of the keys each: 4 rows a KV head, 4096
  // tokens (32/8, D 128) 11.4 us against 13.1, 32768 tokens 41.1 against 44.6; 64 rows, two blocks so,
  // 50.2 against 44.3.
  plan.row_waves = rows <= own ? 1 : 4;
  // Parts of two tiles or more. Where every part is as long as the others, the choice among whole rounds of
  // the workgroups that the chip holds (by LDS) with the fewest tiles one after the other, half a tile
  // for a workgroup's start: 65536 tokens and 64 queries (32/4, D 64), statistics in 32 / 48 / 64 / 96 / 128
  // parts 36.6 / 33.6 / 31.4 / 33.8 / 31.4 us. Where the window is more than a quarter of the prompt the
  // causal bound makes them unequal, and about 1536 workgroups, the longest first, fill up evenly.
  const bool even = (int64_t)window * 4 <= tokens;
  const int64_t slots = 256 * std::min<int64_t>(6, 160 * 1024 / (2 * kTile * (d + 8) * 2 + 2048));
  auto parts = [&](int64_t workgroups, int64_t tiles) {
    const int64_t most = std::max<int64_t>((tiles + 1) / 2, 1);
    if (!even) return (int)std::min<int64_t>(most, (1536 + workgroups - 1) / workgroups);
    int64_t best = 1, best_cost = INT64_MAX;
    for (int64_t rounds = 1; rounds <= 8; ++rounds) {
      const int64_t n = std::clamp<int64_t>(slots * rounds / workgroups, 1, most);
      const int64_t per = (tiles + n - 1) / n, used = (tiles + per - 1) / per;
      const int64_t cost = (workgroups * used + slots - 1) / slots * (2 * per + 1);
      if (cost < best_cost) best = used, best_cost = cost;
    }
    return (int)best;
  };
  plan.key_splits = parts(ceil_div(rows, plan.row_waves * own) * bh, ceil_div(tokens, kTile));
  plan.row_splits = parts(ceil_div(tokens, 4 * own) * bh, ceil_div(rows, kTile));
  // Up to 8 parts of a row's statistics are joined by every workgroup of the sums for itself, without a
  // launch: 1000 tokens and 32 queries (32/8, D 128; 4 parts) 12.1 us against 14.3 apart; 17 parts (4133
  // tokens, 28/4) 20.4 against 20.2, 64 and more (16384 tokens, 32/4, D 64) 22.8 against 17.2. Where a
  // workgroup sums many tiles of rows (8192 queries: 602 us against 591), the launch is the smaller part.
  plan.norm_apart = plan.key_splits > 8 || rows > 1024;
  return plan;
}

hipError_t launch_prompt_weights(int dtype, const PromptWeightLaunch& p, hipStream_t stream) {
  return dtype == kF16 ? run_dim<HalfT>(p, stream) : run_dim<Bf16T>(p, stream);
}

}  // namespace pgr
