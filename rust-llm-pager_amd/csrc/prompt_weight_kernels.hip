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
#include <hip/hip_runtime.h>

#include "cache_device.h"

namespace pgr {
namespace {

constexpr int kTile = 128;  // keys (statistics) or rows (sums) in LDS

// Groups of 32 rows (statistics) or keys (sums) that a wave holds in registers.
template <int D>
constexpr int groups() {
  return D <= 128 ? 2 : 1;
}

struct ScoreScale {
  float c;          // log2 units per unit of the (softcapped) score
  float cap_scale;  // softcap: scale / cap, else 0
  float cap;
};

// The (softcapped) score in units of `c`.
template <bool kCap>
__device__ __forceinline__ float raw_score(float s, const ScoreScale& sc) {
  return kCap ? tanhf(s * sc.cap_scale) : s;
}

// kTile rows of D elements into LDS, `row_ptr(i)` giving row i's address (null: zeros).
template <int D, class F>
__device__ __forceinline__ void stage(uint16_t* lds, F row_ptr) {
  constexpr int kStride = D + 8, kPieces = D / 8;
#pragma unroll
  for (int x = 0; x < kTile * kPieces / 256; ++x) {
    const int id = x * 256 + (int)threadIdx.x, i = id / kPieces, e = (id - i * kPieces) * 8;
    const uint16_t* p = row_ptr(i);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (p != nullptr) v = *reinterpret_cast<const u32x4_e*>(p + e);
    *reinterpret_cast<u32x4*>(lds + i * kStride + e) = v;
  }
}

template <class Ty, int D>
__device__ __forceinline__ f32x16 product(const uint16_t* lds_row, const u32x4 (&own)[D / 16]) {
  f32x16 s = {};
#pragma unroll
  for (int c = 0; c < D / 16; ++c) s = Ty::mma32(*reinterpret_cast<const u32x4*>(lds_row + 16 * c), own[c], s);
  return s;
}

template <int D>
__device__ __forceinline__ void load_own(u32x4 (&r)[D / 16], const uint16_t* row, int half) {
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    r[c] = u32x4{0u, 0u, 0u, 0u};
    if (row != nullptr) r[c] = *reinterpret_cast<const u32x4_e*>(row + 16 * c + 8 * half);
  }
}

// kRowWaves 4: the waves hold rows of their own and all take every key; 1: they hold the same rows
// and take a quarter of the keys each.
template <class Ty, int D, int kRowWaves, bool kCap>
__global__ __launch_bounds__(256) void prompt_stats_kernel(PromptWeightLaunch a, ScoreScale sc) {
  constexpr int kN = groups<D>();
  constexpr int kStride = D + 8;
  __shared__ __align__(16) uint16_t lds[kTile * kStride];
  const int n_rep = a.hq / a.hkv, rows = a.window * n_rep;
  const int bh = blockIdx.z, b = bh / a.hkv, h = bh - b * a.hkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5, j = lane & 31;
  const int lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
  const uint16_t* qb = static_cast<const uint16_t*>(a.q) + b * a.qs.b + (int64_t)h * n_rep * a.qs.h;
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.ks.b + h * a.ks.h;

  const int wg_row = blockIdx.x * kRowWaves * kN * 32;
  const int wave_row = wg_row + (kRowWaves == 4 ? wave * kN * 32 : 0);
  u32x4 own[kN][D / 16];
  int last[kN];  // the last column that the lane's row attends to (-1: no such row)
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    const int r = wave_row + g * 32 + j, i = r / n_rep;
    last[g] = r < rows ? a.tokens - a.window + i : -1;
    load_own<D>(own[g], r < rows ? qb + (r - i * n_rep) * a.qs.h + i * a.qs.t : nullptr, half);
  }
  // Keys that any row of the workgroup, and every row of the wave, attends to.
  const int wg_last = a.tokens - a.window + min(wg_row + kRowWaves * kN * 32, rows) / n_rep;
  const int every = a.tokens - a.window + wave_row / n_rep;

  // This split's tiles of [lo, wg_last].
  const int t_lo = lo / kTile, t_hi = min(wg_last, a.tokens - 1) / kTile + 1;
  const int per = (max(t_hi - t_lo, 0) + a.plan.key_splits - 1) / a.plan.key_splits;
  const int t_begin = t_lo + (int)blockIdx.y * per, t_end = min(t_begin + per, t_hi);

  float m[kN], l[kN];
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    m[g] = kMinusInf;
    l[g] = 0.f;
  }
  for (int tile = t_begin; tile < t_end; ++tile) {
    const int key0 = tile * kTile;
    __syncthreads();
    stage<D>(lds, [&](int i) { return key0 + i < a.tokens ? kb + (key0 + i) * a.ks.t : nullptr; });
    __syncthreads();
    for (int sub = kRowWaves == 4 ? 0 : wave; sub < kTile / 32; sub += kRowWaves == 4 ? 1 : 4) {
      const int k0 = key0 + sub * 32;
      const bool edge = k0 < lo || k0 + 31 > every;
#pragma unroll
      for (int g = 0; g < kN; ++g) {
        f32x16 s = product<Ty, D>(lds + (sub * 32 + j) * kStride + 8 * half, own[g]);
        float top = kMinusInf;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          s[x] = raw_score<kCap>(s[x], sc);
          if (edge) {
            const int key = k0 + 8 * (x / 4) + 4 * half + (x & 3);
            if (key < lo || key > last[g]) s[x] = kMinusInf;
          }
          top = fmaxf(top, s[x]);
        }
        const float m_new = fmaxf(m[g], top);
        const float ref = m_new == kMinusInf ? 0.f : m_new * sc.c;
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) sum += __builtin_amdgcn_exp2f(fmaf(s[x], sc.c, -ref));
        l[g] = l[g] * __builtin_amdgcn_exp2f(fmaf(m[g], sc.c, -ref)) + sum;
        m[g] = m_new;
      }
    }
  }
  // The halves of the wave hold other keys of the same rows; so do the waves where they share rows.
  __shared__ float2 part[4][kN * 32];
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

// norm = m + log2(l) over the splits of each row; +inf for a row that attends to nothing.
__global__ __launch_bounds__(256) void prompt_norm_kernel(PromptWeightLaunch a, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float m = kMinusInf;
  for (int s = 0; s < a.plan.key_splits; ++s) m = fmaxf(m, a.stats[s * n + i].x);
  const float ref = m == kMinusInf ? 0.f : m;
  float l = 0.f;
  for (int s = 0; s < a.plan.key_splits; ++s) {
    const float2 p = a.stats[s * n + i];
    l += p.y * __builtin_amdgcn_exp2f(p.x - ref);
  }
  a.norm[i] = l == 0.f ? -kMinusInf : ref + __builtin_amdgcn_logf(l);
}

template <class Ty, int D, bool kCap>
__global__ __launch_bounds__(256) void prompt_sums_kernel(PromptWeightLaunch a, ScoreScale sc) {
  constexpr int kN = groups<D>();
  constexpr int kStride = D + 8;
  __shared__ __align__(16) uint16_t lds[kTile * kStride];
  __shared__ __align__(16) float norm_s[kTile];
  const int n_rep = a.hq / a.hkv, rows = a.window * n_rep;
  const int bh = blockIdx.z, b = bh / a.hkv, h = bh - b * a.hkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5, j = lane & 31;
  const int lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
  const uint16_t* qb = static_cast<const uint16_t*>(a.q) + b * a.qs.b + (int64_t)h * n_rep * a.qs.h;
  const uint16_t* kb = static_cast<const uint16_t*>(a.k) + b * a.ks.b + h * a.ks.h;
  const float* norm = a.norm + (int64_t)bh * rows;

  const int wg_key = blockIdx.x * 4 * kN * 32, wave_key = wg_key + wave * kN * 32;
  u32x4 own[kN][D / 16];
  float sum[kN];
#pragma unroll
  for (int g = 0; g < kN; ++g) {
    const int key = wave_key + g * 32 + j;
    load_own<D>(own[g], key < a.tokens ? kb + key * a.ks.t : nullptr, half);
    sum[g] = 0.f;
  }
  // The first row that attends to the workgroup's first key, and this split's tiles from there on.
  const int first = max(wg_key - (a.tokens - a.window), 0) * n_rep;
  const int t_lo = first / kTile, t_hi = (rows + kTile - 1) / kTile;
  const int per = (max(t_hi - t_lo, 0) + a.plan.row_splits - 1) / a.plan.row_splits;
  const int t_begin = t_lo + (int)blockIdx.y * per, t_end = min(t_begin + per, t_hi);
  for (int tile = t_begin; tile < t_end; ++tile) {
    const int row0 = tile * kTile;
    __syncthreads();
    stage<D>(lds, [&](int i) {
      const int r = row0 + i, qi = r / n_rep;
      return r < rows ? qb + (r - qi * n_rep) * a.qs.h + qi * a.qs.t : nullptr;
    });
    if (threadIdx.x < kTile)
      norm_s[threadIdx.x] = row0 + (int)threadIdx.x < rows ? norm[row0 + threadIdx.x] : -kMinusInf;
    __syncthreads();
    for (int sub = 0; sub < kTile / 32; ++sub) {
      const int r0 = row0 + sub * 32;
      // Rows that do not attend to every key of the wave.
      const bool edge = wave_key < lo || wave_key + kN * 32 - 1 > a.tokens - a.window + r0 / n_rep;
#pragma unroll
      for (int g = 0; g < kN; ++g) {
        const f32x16 s = product<Ty, D>(lds + (sub * 32 + j) * kStride + 8 * half, own[g]);
        const int key = wave_key + g * 32 + j;
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
          const f32x4 nm = *reinterpret_cast<const f32x4*>(norm_s + sub * 32 + 2 * x + 4 * half);
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            float p = __builtin_amdgcn_exp2f(fmaf(raw_score<kCap>(s[x + y], sc), sc.c, -nm[y]));
            if (edge) {
              const int r = r0 + 2 * x + 4 * half + y;
              if (key < lo || key > a.tokens - a.window + r / n_rep) p = 0.f;
            }
            sum[g] += p;
          }
        }
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
  for (int s = 0; s < a.plan.row_splits; ++s) x += a.partial[s * n + i];
  a.out[i] = x;
}

bool shared_rows(int rows) { return rows <= 128; }

template <class Ty, int D, bool kCap>
hipError_t run(const PromptWeightLaunch& p, const ScoreScale& sc, hipStream_t stream) {
  const int rows = p.window * (p.hq / p.hkv), own = groups<D>() * 32;
  const unsigned bh = (unsigned)(p.batch * p.hkv);
  if (shared_rows(rows)) {
    const dim3 grid((unsigned)((rows + own - 1) / own), (unsigned)p.plan.key_splits, bh);
    prompt_stats_kernel<Ty, D, 1, kCap><<<grid, 256, 0, stream>>>(p, sc);
  } else {
    const dim3 grid((unsigned)((rows + 4 * own - 1) / (4 * own)), (unsigned)p.plan.key_splits, bh);
    prompt_stats_kernel<Ty, D, 4, kCap><<<grid, 256, 0, stream>>>(p, sc);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t n = (int64_t)bh * rows;
  prompt_norm_kernel<<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(p, n);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)((p.tokens + 4 * own - 1) / (4 * own)), (unsigned)p.plan.row_splits, bh);
  prompt_sums_kernel<Ty, D, kCap><<<grid, 256, 0, stream>>>(p, sc);
  e = hipGetLastError();
  if (e != hipSuccess || p.plan.row_splits == 1) return e;
  const int64_t m = (int64_t)bh * p.tokens;
  prompt_join_kernel<<<(unsigned)((m + 255) / 256), 256, 0, stream>>>(p, m);
  return hipGetLastError();
}

template <class Ty, int D>
hipError_t run_cap(const PromptWeightLaunch& p, hipStream_t stream) {
  ScoreScale sc;
  if (p.softcap > 0.f) {
    sc = {p.softcap * kLog2e, p.scale / p.softcap, p.softcap};
    return run<Ty, D, true>(p, sc, stream);
  }
  sc = {p.scale * kLog2e, 0.f, 0.f};
  return run<Ty, D, false>(p, sc, stream);
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
  const int64_t rows = (int64_t)window * (hq / hkv), own = d <= 128 ? 64 : 32, bh = (int64_t)batch * hkv;
  const int64_t row_blocks = shared_rows((int)rows) ? (rows + own - 1) / own : (rows + 4 * own - 1) / (4 * own);
  auto parts = [](int64_t workgroups, int64_t tiles) {  // about 1024 workgroups, two tiles each
    int64_t n = (1024 + workgroups - 1) / workgroups;
    const int64_t most = (tiles + 1) / 2;
    if (n > most) n = most;
    return (int)(n < 1 ? 1 : n);
  };
  plan.key_splits = parts(row_blocks * bh, (tokens + kTile - 1) / kTile);
  plan.row_splits = parts((tokens + 4 * own - 1) / (4 * own) * bh, (rows + kTile - 1) / kTile);
  return plan;
}

hipError_t launch_prompt_weights(int dtype, const PromptWeightLaunch& p, hipStream_t stream) {
  return dtype == kF16 ? run_dim<HalfT>(p, stream) : run_dim<Bf16T>(p, stream);
}

}  // namespace pgr
