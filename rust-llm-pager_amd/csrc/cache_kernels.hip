// The bounded cache: append with eviction, weighted decode attention, prompt selection.
//
// A row (batch row x KV head) holds up to `capacity` tokens in slots: key, value, accumulated
// attention weight, and its number among the row's tokens (order). lengths and seen are kept per
// row and on the device: each workgroup owns the rows it changes, and a captured step replays.
#include <hip/hip_runtime.h>

#include "cache_device.h"

namespace pgr {
namespace {

// ---------------------------------------------------------------------------------------
// Weights in their order as unsigned numbers: a heavier token has the larger key, -0 and 0 are
// equal, and NaN (one key for all of them) is the heaviest. 0 and 0xffffffff are no weight's key.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xfffffffeu;
  const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t min_u64(uint64_t a, uint64_t b) { return a < b ? a : b; }

__device__ __forceinline__ uint64_t shuffle_xor(uint64_t x, int mask) {
  const uint32_t lo = __shfl_xor((uint32_t)x, mask), hi = __shfl_xor((uint32_t)(x >> 32), mask);
  return (uint64_t)hi << 32 | lo;
}

// Element i of a head after the turn; cs, sn: the pairs' cosines and sines.
template <class Ty>
__device__ __forceinline__ typename Ty::Raw turned(const typename Ty::Raw* x, int i, const RotaryForm& f,
                                                   const float* cs, const float* sn) {
  if (i >= 2 * f.half) return x[i];
  const bool first = f.interleaved ? (i & 1) == 0 : i < f.half;
  const int pair = f.interleaved ? i >> 1 : (first ? i : i - f.half);
  const int mate = f.interleaved ? i ^ 1 : (first ? i + f.half : i - f.half);
  const float own = Ty::to_f(x[i]), other = Ty::to_f(x[mate]);
  return Ty::cvt(first ? turned_x(own, other, cs[pair], sn[pair]) : turned_y(other, own, cs[pair], sn[pair]));
}

typedef float f32x4_e __attribute__((ext_vector_type(4), aligned(4)));
typedef int32_t i32x4_e __attribute__((ext_vector_type(4), aligned(4)));

// One workgroup per row: the new token's slot (the next free one, or in a full row the lightest
// token's that is neither among the first keep_first nor among the last keep_recent, the new one
// counted), its turned key, its value, and the turned queries of the row's heads.
//
// Latency-bound: a full row's weights and orders are 8 bytes a slot. The first 4096 slots' are asked for
// 16 bytes at a time before anything else, and the angles and queries are done under them. 512 rows
// (64 x 8 KV heads, 32 heads, D 128), three quarters of them full with 4096 slots: 8.9 us (11.7 with one
// slot a thread at a time and an angle per element); one row of 256 slots: 4.7 us, a launch.
template <class Ty>
__global__ __launch_bounds__(256) void hh_append_kernel(HHAppendLaunch a) {
  typedef typename Ty::Raw Raw;
  constexpr int kAhead = 4;  // times 4 slots a thread
  __shared__ uint64_t best_s[4];
  __shared__ float cs[128], sn[128];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const HHCache& c = a.c;
  const int64_t row = (int64_t)b * c.hkv + h;
  const int seen = c.seen[row];
  const int length = min(max(c.lengths[row], 0), c.capacity);
  const bool full = length == c.capacity;
  float* w = c.weights + row * c.capacity;
  int32_t* order = c.order + row * c.capacity;

  // (A row of less than four slots is read one by one.)
  const int groups = full ? c.capacity / 4 : 0;
  f32x4_e wa[kAhead];
  i32x4_e oa[kAhead];
#pragma unroll
  for (int x = 0; x < kAhead; ++x) {
    const int i = 4 * min(tid + x * 256, groups - 1);
    if (groups > 0) {
      wa[x] = *reinterpret_cast<const f32x4_e*>(w + i);
      oa[x] = *reinterpret_cast<const i32x4_e*>(order + i);
    }
  }

  const int d = c.d, n_rep = c.hq / c.hkv;
  const Raw* k = static_cast<const Raw*>(a.k) + b * a.ks.b + h * a.ks.h;
  const Raw* v = static_cast<const Raw*>(a.v) + b * a.vs.b + h * a.vs.h;
  if (tid < a.form.half) {
    const int64_t pos = a.positions != nullptr ? load_position(a.positions, a.positions64, b) : (int64_t)seen;
    float x, y;
    turn(pos, a.form.inv_freq[tid], x, y);
    cs[tid] = x * a.form.factor;
    sn[tid] = y * (a.form.factor * a.form.sign);
  }
  __syncthreads();  // (also: every thread has read the row's length and number)
  Raw k_new{}, v_new{};
  if (tid < d) {
    k_new = turned<Ty>(k, tid, a.form, cs, sn);
    v_new = v[tid];
  }
  if (a.q_out != nullptr) {
    Raw* qo = static_cast<Raw*>(a.q_out) + ((int64_t)b * c.hq + (int64_t)h * n_rep) * d;
    const Raw* q = static_cast<const Raw*>(a.q) + b * a.qs.b + (int64_t)h * n_rep * a.qs.h;
    for (int i = tid; i < n_rep * d; i += 256) {
      const int r = i / d;
      qo[i] = turned<Ty>(q + r * a.qs.h, i - r * d, a.form, cs, sn);
    }
  }

  int slot = length;
  if (full) {
    const int64_t recent = (int64_t)seen + 1 - c.keep_recent;
    uint64_t best = ~0ull;
    auto look = [&](int i, float x, int32_t o) {
      const uint64_t held = o < c.keep_first || o >= recent;
      best = min_u64(best, held << 63 | (uint64_t)weight_key(x) << 31 | (uint64_t)i);
    };
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      if (tid + x * 256 >= groups) continue;
#pragma unroll
      for (int y = 0; y < 4; ++y) look(4 * (tid + x * 256) + y, wa[x][y], oa[x][y]);
    }
#pragma unroll 2
    for (int g = tid + kAhead * 256; g < groups; g += 256) {
      const f32x4_e x = *reinterpret_cast<const f32x4_e*>(w + 4 * g);
      const i32x4_e o = *reinterpret_cast<const i32x4_e*>(order + 4 * g);
#pragma unroll
      for (int y = 0; y < 4; ++y) look(4 * g + y, x[y], o[y]);
    }
    const int i = 4 * groups + tid;
    if (i < c.capacity) look(i, w[i], order[i]);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) best = min_u64(best, shuffle_xor(best, m));
    if ((tid & 63) == 0) best_s[tid >> 6] = best;
    __syncthreads();
    best = min_u64(min_u64(best_s[0], best_s[1]), min_u64(best_s[2], best_s[3]));
    slot = (int)(best & 0x7fffffffu);
  }

  const int64_t to = (row * c.capacity + slot) * d;
  if (tid < d) {
    static_cast<Raw*>(c.keys)[to + tid] = k_new;
    static_cast<Raw*>(c.values)[to + tid] = v_new;
  }
  if (tid == 0) {  // (in a full row every thread is past its reads: the barrier above)
    w[slot] = 0.f;
    order[slot] = seen;
    c.seen[row] = seen + 1;
    c.lengths[row] = full ? length : length + 1;
  }
}

// ---------------------------------------------------------------------------------------
// Attention of one new token. Each wave folds tiles of 32 tokens, two halves of 16, on
// v_mfma_f32_16x16x32:
//     S^T[16 tok x 16 heads] = K . Q^T,   O^T[D x 16 heads] += V^T[D x 32 tok] . P^T[32 tok x 16 heads]
// Lane (g, n) holds tokens 4g..4g+3 of each half for query head n, which is the P^T operand as it
// stands (contraction slot 8g + e: token 4g + e of the first half, 4g + e - 4 of the second), and every
// O^T value of a lane belongs to head n as well: the softmax state is a scalar of the lane.
// P goes in as two numbers of the K/V type, P.V in two products each: with one, rounded, the output of 24 like
// tokens was off by up to seven times what its other roundings explain, and the products are free beside the
// loads (the sizes below take the same time either way).
// A lane reads 16-byte pieces 4c + g of K row n, so that an instruction covers 64 bytes of each of
// 16 rows, and of V the D/16 elements n of its eight rows, transposed in registers (v_perm_b32).
//
// Bound by HBM. The next tile's K is loaded as soon as the scores of this one are taken, its V after
// P.V, without a second set of registers. The scores go to memory once (4 bytes a head and token,
// beside 4 D of K and V), since the weights need each head's final maximum and sum: the merge launch adds
// them up. 32 full rows x 8192 tokens, 32/8 heads, D 128: 206 + 13 us for 1.08 GB (5.2 TB/s in the first
// launch; a copy reaches 5.1, a plain read in this order 6.25, this launch without its stores 5.8). Tiles
// of 16 tokens, one load after the other: 221 us; 256 to 8192 workgroups, non-temporal loads or not: 205-212.
// What a head's scores are taken against for their probabilities, in log2 units. +inf where nothing has weight
// (no tokens, or scores of -inf only): the head then gives zeros, and nothing to the weights.
__device__ __forceinline__ float norm_of(float m, float l) {
  return l == 0.f ? -kMinusInf : m + __builtin_amdgcn_logf(l);
}

// Tokens [begin, end) of a row of `length` that split `split` of n_split takes: whole 32-token
// tiles, evenly.
constexpr int kTileTokens = 32;
__device__ __forceinline__ int split_tiles(int length, int n_split) {
  const int tiles = (length + kTileTokens - 1) / kTileTokens;
  return (tiles + n_split - 1) / n_split;
}

// Rows of up to kOneTokens slots (half of that at head dim 256): the workgroup holds the whole row, its
// scores in LDS, and finishes it without a merge launch. 28/4 heads, D 128, one row of 64 / 256 / 512
// tokens: 4.8 / 6.6 / 8.4 us against 9.2 / 9.8 / 10.0 split; 32/8 heads, 64 and 128 rows of 512: 28.8 and
// 55.3 against 37.7 and 65.4; at head dim 256 (8/1, 8 rows of 512) 14.7 against 12.1.
constexpr int kOneTokens = 512;
constexpr int kMostSplits = 1024;

template <class Ty, int D, int kW, bool kOne>
__global__ __launch_bounds__(64 * kW) void hh_attend_kernel(HHAttendLaunch a, AttendScale sc) {
  typedef KVTile<D> T;
  constexpr int kThreads = 64 * kW;
  __shared__ float sm_m[kW][kMaxRep], sm_l[kW][kMaxRep];
  __shared__ float sm_acc[kW][kMaxRep][D + 1];
  __shared__ __align__(16) float sm_logits[kOne ? kMaxRep * kOneTokens : 1];
  __shared__ float norm_s[kMaxRep];
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const HHCache& c = a.c;
  const int n_rep = c.hq / c.hkv;
  const int64_t row = (int64_t)b * c.hkv + h;
  const int length = min(max(c.lengths[row], 0), c.capacity);
  const int per = kOne ? length : split_tiles(length, a.n_split) * kTileTokens;
  const int begin = min(split * per, length), end = min(begin + per, length);
  // Uniform: nothing to fold. (The merge reads only the splits that hold tokens; a row that is
  // finished here and holds none still has its zeros to write.)
  if (!kOne && begin >= end) return;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const bool real = n < n_rep;
  const uint16_t* kp = static_cast<const uint16_t*>(c.keys) + (row * c.capacity + begin) * D;
  const uint16_t* vp = static_cast<const uint16_t*>(c.values) + (row * c.capacity + begin) * D;
  const int tokens = end - begin, tiles = (tokens + kTileTokens - 1) / kTileTokens;

  T t;
  // Rows past the split's end read its last row; what they hold is masked.
  auto fetch_k = [&](int ti) {
    const int most = tokens - 1 - ti * kTileTokens;
    const uint16_t* p = kp + (int64_t)ti * kTileTokens * D;
#pragma unroll
    for (int x = 0; x < 2; ++x) load_pieces<D>(t.k[x], p + min(16 * x + n, most) * D, g);
  };
  auto fetch_v = [&](int ti) {
    const int most = tokens - 1 - ti * kTileTokens;
    const uint16_t* p = vp + (int64_t)ti * kTileTokens * D;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) load_v<D>(t.v[x][i], p + min(16 * x + 4 * g + i, most) * D, n);
  };
  u32x4 q[T::KP];
#pragma unroll
  for (int i = 0; i < T::KP; ++i) q[i] = u32x4{0u, 0u, 0u, 0u};
  if (real)
    load_pieces<D>(q, static_cast<const uint16_t*>(a.q) + b * a.qs.b + ((int64_t)h * n_rep + n) * a.qs.h, g);
  if (wave < tiles) {
    fetch_k(wave);
    fetch_v(wave);
  }
  arrived(q);

  float m_run = kMinusInf, l_run = 0.f;
  f32x4 acc[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Scores of a tile lie together, head by head (32 tokens: 128 bytes): whole lines, one after the other.
  float* lg = kOne ? sm_logits : a.logits + (row * hh_attend_stride(c.capacity) + begin) * n_rep;
  lg += n * kTileTokens + 4 * g;

  auto scores = [&](f32x4 (&s)[2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (D == 16) {
        s[x] = Ty::mma16(u32x2{t.k[x][0].x, t.k[x][0].y}, u32x2{q[0].x, q[0].y}, s[x]);
      } else {
#pragma unroll
        for (int i = 0; i < T::KP; ++i) s[x] = Ty::mma16x32(t.k[x][i], q[i], s[x]);
      }
    }
  };
  auto fold = [&](f32x4 (&s)[2], int ti) {
    float p[8], top = kMinusInf;
    if (sc.cap_log2 > 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i / 4][i & 3] = sc.cap_log2 * tanhf(s[i / 4][i & 3] * sc.cap_scale);
    } else {
#pragma unroll
      for (int x = 0; x < 2; ++x) s[x] *= sc.scale_log2;
    }
    if ((ti + 1) * kTileTokens > tokens) {  // uniform: the last tile, ragged
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (ti * kTileTokens + 16 * x + 4 * g + i < tokens) continue;
          s[x][i] = kMinusInf;
#pragma unroll
          for (int j = 0; j < T::VD; ++j) t.v[x][i][j] = 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i / 4][i & 3]);
    const float m_new = fmaxf(m_run, max_g(top));
    const float ref = m_new == kMinusInf ? 0.f : m_new;  // (scores of -inf weigh nothing, those of NaN stay NaN)
    if (__any(m_new > m_run)) {  // (otherwise the factor is 1)
      const float alpha = __builtin_amdgcn_exp2f(m_run - ref);
      l_run *= alpha;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) acc[j] *= alpha;
      m_run = m_new;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(s[i / 4][i & 3] - ref);
    l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x, y;
      Ty::split(p[2 * i], p[2 * i + 1], x, y);
      hi[i] = x;
      lo[i] = y;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
      const int e = j >> 1;
      u32x4 vt;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        vt[2 * x] = __builtin_amdgcn_perm(t.v[x][1][e], t.v[x][0][e], sel);
        vt[2 * x + 1] = __builtin_amdgcn_perm(t.v[x][3][e], t.v[x][2][e], sel);
      }
      acc[j] = Ty::mma16x32(vt, lo, acc[j]);
      acc[j] = Ty::mma16x32(vt, hi, acc[j]);
    }
  };
  // After the next tile's loads, which are waited for in the order of all memory operations.
  auto store = [&](const f32x4 (&s)[2], int ti) {
    if (real) {
#pragma unroll
      for (int x = 0; x < 2; ++x) *reinterpret_cast<f32x4*>(lg + (int64_t)ti * kTileTokens * n_rep + 16 * x) = s[x];
    }
  };
  int ti = wave;
  for (; ti + kW < tiles; ti += kW) {
    f32x4 s[2];
    scores(s);
    fetch_k(ti + kW);
    fold(s, ti);
    fetch_v(ti + kW);
    __builtin_amdgcn_sched_barrier(0);
    store(s, ti);
  }
  if (ti < tiles) {
    f32x4 s[2];
    scores(s);
    fold(s, ti);
    store(s, ti);
  }

  const float l_wave = sum_g(l_run);
  if (g == 0) {
    sm_m[wave][n] = m_run;
    sm_l[wave][n] = l_wave;
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sm_acc[wave][n][(D / 4) * g + (D / 16) * i + j] = acc[j][i] * Ty::kUnit;
  __syncthreads();
  const int64_t part = (row * a.n_split + split) * n_rep;
  for (int i = threadIdx.x; i < n_rep * D; i += kThreads) {
    const int r = i / D, e = i - r * D;
    float m = kMinusInf;
#pragma unroll
    for (int w = 0; w < kW; ++w) m = fmaxf(m, sm_m[w][r]);
    float x = 0.f, l = 0.f;
    const float ref = m == kMinusInf ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm_m[w][r] - ref);
      x += sm_acc[w][r][e] * f;
      l += sm_l[w][r] * f;
    }
    if constexpr (kOne) {
      static_cast<uint16_t*>(a.out)[(row * n_rep + r) * D + e] = Ty::cvt(l == 0.f ? 0.f : x / l);
      if (e == 0) norm_s[r] = norm_of(m, l);
    } else {
      a.pacc[part * D + i] = x;
      if (e == 0) {
        a.pm[part + r] = m;
        a.pl[part + r] = l;
      }
    }
  }
  if constexpr (kOne) {
    __syncthreads();
    float* w = c.weights + row * c.capacity;
    for (int i = threadIdx.x; i < length; i += kThreads) {
      float sum = 0.f;
      const float* y = sm_logits + i / kTileTokens * kTileTokens * n_rep + i % kTileTokens;
      for (int r = 0; r < n_rep; ++r) sum += __builtin_amdgcn_exp2f(y[r * kTileTokens] - norm_s[r]);
      w[i] += sum;
    }
  }
}

// Joins the splits. Workgroups x < n_rep of a row write the output of query head x; the others add
// the probabilities of 1024 tokens each, summed over the row's heads in their order, to the weights.
// The splits' maxima and sums are read by a wave at once, the splits' outputs by groups of d / 4 threads
// (32 splits of 32 rows: 5.6 us; 21.1 with a thread's loop over the splits).
template <class Ty>
__global__ __launch_bounds__(256) void hh_attend_merge_kernel(HHAttendLaunch a) {
  __shared__ float norm_s[kMaxRep], f_s[kMostSplits];
  __shared__ __align__(16) float sum_s[256 * 4];
  const HHCache& c = a.c;
  const int n_rep = c.hq / c.hkv, d = c.d, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t row = blockIdx.y;
  const int length = min(max(c.lengths[row], 0), c.capacity);
  const int tiles = (length + kTileTokens - 1) / kTileTokens, per = split_tiles(length, a.n_split);
  const int used = per > 0 ? (tiles + per - 1) / per : 0;
  const float* pm = a.pm + row * a.n_split * n_rep;
  const float* pl = a.pl + row * a.n_split * n_rep;
  // (m, l) of head r over the splits, in every lane of the calling wave.
  auto head_stats = [&](int r, float& m, float& l) {
    m = kMinusInf;
    l = 0.f;
    for (int s = lane; s < used; s += 64) {
      const float ms = pm[s * n_rep + r], ls = pl[s * n_rep + r], top = fmaxf(m, ms);
      if (top != kMinusInf) l = l * __builtin_amdgcn_exp2f(m - top) + ls * __builtin_amdgcn_exp2f(ms - top);
      else l += ls;
      m = top;
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) {
      const float m2 = __shfl_xor(m, x), l2 = __shfl_xor(l, x), top = fmaxf(m, m2);
      if (top != kMinusInf) l = l * __builtin_amdgcn_exp2f(m - top) + l2 * __builtin_amdgcn_exp2f(m2 - top);
      else l += l2;
      m = top;
    }
  };
  const int x = blockIdx.x;
  if (x < n_rep) {
    float m, l;
    head_stats(x, m, l);
    for (int s = tid; s < used; s += 256) f_s[s] = m == kMinusInf ? 0.f : __builtin_amdgcn_exp2f(pm[s * n_rep + x] - m);
    __syncthreads();
    const int cols = d / 4, groups = 256 / cols, g = tid / cols, e = (tid - g * cols) * 4;
    const float* pacc = a.pacc + (row * a.n_split * n_rep + x) * d + e;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = g; s < used; s += groups) o += *reinterpret_cast<const f32x4*>(pacc + (int64_t)s * n_rep * d) * f_s[s];
    *reinterpret_cast<f32x4*>(sum_s + 4 * tid) = o;
    __syncthreads();
    if (tid < d) {
      float y = 0.f;
      for (int k = 0; k < min(groups, used); ++k) y += sum_s[k * d + tid];
      static_cast<uint16_t*>(a.out)[(row * n_rep + x) * d + tid] = Ty::cvt(l == 0.f ? 0.f : y / l);
    }
    return;
  }
  const int first = (x - n_rep) * 1024;
  if (first >= length) return;
  for (int r = wave; r < n_rep; r += 4) {
    float m, l;
    head_stats(r, m, l);
    if (lane == 0) norm_s[r] = norm_of(m, l);
  }
  const int t = first + 4 * tid;
  float* w = c.weights + row * c.capacity + t;
  const float* lg = a.logits + (row * hh_attend_stride(c.capacity) + t / kTileTokens * kTileTokens) * n_rep +
                    t % kTileTokens;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  __syncthreads();
  if (t >= length) return;
#pragma unroll 4
  for (int r = 0; r < n_rep; ++r) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(lg + r * kTileTokens);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += __builtin_amdgcn_exp2f(y[i] - norm_s[r]);
  }
  if (t + 3 < length) {
    f32x4_e* to = reinterpret_cast<f32x4_e*>(w);
    *to = *to + sum;
  } else {  // slots from the length on stay as they are
    for (int i = 0; i < length - t; ++i) w[i] += sum[i];
  }
}

// ---------------------------------------------------------------------------------------
// Which of a prompt's tokens stay, where a row has more than slots: the `capacity` heaviest, the
// lowest column first among equals, where the first keep_first and the last keep_recent tokens count as
// heavier than any other. The key of the last one taken (`last`; of those equal to it the first `need`
// are taken) is found from its top 11 bits down: 11, 11, 10, a count per class, then a scan over the
// classes from the heaviest. Then every token above it, and every equal one of low enough rank, has
// its slot from the counts before it.
//
// Latency-bound: the weights are few bytes (256 KB a row at 65536 tokens), the passes and their barriers
// many. Up to kSelShort tokens one workgroup per row does it all, its keys in registers (2 / 32 / 512 rows
// of 8192 tokens, the copy of short records included: 11.4 / 12.9 / 31.7 us against 16.5 / 18.2 / 41.5 in
// parts). Longer rows are dealt out in parts of kSelPart tokens over three launches: the parts' counts of the
// top 11 bits; from all of a row's counts the class of the last token, whose members go to the row's list; and
// from that list the last key and each part's slots. 16 rows of 65536 tokens, 4096 kept, weights over many
// binades (the list is a hundredth of the row): 4.4 + 6.8 + 9.6 us; one workgroup per row took 71 us (129 with
// 8-bit classes and without registers), the fetching of its unrolled code included, on 16 of the 256 CUs.
// Every part reads the row's whole list, up to three times, and the list is as long as weights are alike: of a
// prompt's attention weights (64 queries, D 128) 4% of the row with queries of scale 2, 44-49% at scale 1 and
// 0.5, where the last launch takes 12 and 42-46 us (at 131072 tokens and 8192 kept 16 and 70-77); 114 us
// if all weights are equal. 8 rows of 1023 tokens in one launch: 9.3 us (31.8).
//
// Counts of one class are added one after the other; where all of a wave's tokens are of one class
// (equal weights), one lane adds them up.
constexpr int kSelThreads = 1024, kSelShort = 8192;
constexpr int kPartThreads = 512, kSelPart = 4096, kPartKeys = kSelPart / kPartThreads;

// The sum of x over the threads before this one; *all: over the workgroup. `part`: a value per wave.
template <int kWaveCount>
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* part, uint32_t* all) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t incl = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 63) part[wave] = incl;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWaveCount; ++w) {
    const uint32_t y = part[w];
    before += w < wave ? y : 0u;
    total += y;
  }
  __syncthreads();
  *all = total;
  return before + incl - x;
}

// Adds 1 to hist[digit] for the calling lanes.
__device__ __forceinline__ void count_class(uint32_t* hist, uint32_t digit) {
  const uint32_t first = __builtin_amdgcn_readfirstlane(digit);
  const uint64_t here = __ballot(true), same = __ballot(digit == first);
  if (same == here) {
    if (__builtin_ctzll(here) == (int)(threadIdx.x & 63)) atomicAdd(&hist[digit], (uint32_t)__popcll(here));
  } else {
    atomicAdd(&hist[digit], 1u);
  }
}

// The class that holds the need-th heaviest of 2048 counted classes: thread t holds the counts of the
// kN classes from 2047 - kN * t down. out: class, how many of its members are taken, whether all are.
// The caller synchronizes before it reads out.
template <int kN, int kWaveCount>
__device__ __forceinline__ void pick_class(const uint32_t (&count)[kN], uint32_t need, uint32_t* part, uint32_t* out) {
  uint32_t mine = 0, total;
#pragma unroll
  for (int x = 0; x < kN; ++x) mine += count[x];
  uint32_t before = scan_before<kWaveCount>(mine, part, &total);
  if (before < need && need <= before + mine) {
#pragma unroll
    for (int x = 0; x < kN; ++x) {
      if (before < need && need <= before + count[x]) {
        out[0] = 2047 - kN * threadIdx.x - x;
        out[1] = need - before;
        out[2] = need - before == count[x];
      }
      before += count[x];
    }
  }
}

struct SelectRow {
  int lo, n, mid0, mid1;
  const float* w;
  __device__ __forceinline__ SelectRow(const HHLoadLaunch& a, int64_t row) {
    const int b = (int)(row / a.c.hkv);
    lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
    n = a.tokens - lo;
    mid0 = a.c.keep_first;
    mid1 = n - a.c.keep_recent;
    w = a.weights + row * a.tokens + lo;
  }
  // Token i's key: 0xffffffff for one that is kept in any case, 0 past the row's end.
  __device__ __forceinline__ uint32_t key(int i) const {
    const uint32_t k = weight_key(w[min(i, n - 1)]);
    return i >= n ? 0u : i < mid0 || i >= mid1 ? 0xffffffffu : k;
  }
};

__device__ __forceinline__ void keep_token(const HHLoadLaunch& a, const SelectRow& r, int64_t row, uint32_t at, int i) {
  if (at >= (uint32_t)a.c.capacity) return;
  const int64_t to = row * a.c.capacity + at;
  a.kept[to] = r.lo + i;
  a.c.weights[to] = r.w[i];
  a.c.order[to] = i;
}

// A row that fits: every token stays. Also sets the row's length.
__device__ __forceinline__ bool keep_all(const HHLoadLaunch& a, const SelectRow& r, int64_t row, int part, int parts) {
  if (part == 0 && threadIdx.x == 0) {
    a.c.lengths[row] = min(r.n, a.c.capacity);
    a.c.seen[row] = r.n;
  }
  if (r.n > a.c.capacity) return false;
  for (int i = part * (int)blockDim.x + threadIdx.x; i < r.n; i += parts * (int)blockDim.x)
    keep_token(a, r, row, (uint32_t)i, i);
  return true;
}

__global__ __launch_bounds__(kSelThreads) void hh_select_kernel(HHLoadLaunch a) {
  constexpr int kPer = kSelShort / kSelThreads, kWaveCount = kSelThreads / 64, kGroups = kPer * kWaveCount;
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t ups[kGroups], eqs[kGroups];  // per group of 64: tokens above the key, equal to it
  __shared__ uint32_t part[kWaveCount], picked[3];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const SelectRow r(a, row);
  if (keep_all(a, r, row, 0, 1)) return;
  uint32_t keys[kPer];
#pragma unroll
  for (int y = 0; y < kPer; ++y) keys[y] = r.key(y * kSelThreads + tid);

  uint32_t need = (uint32_t)a.c.capacity, last = 0;
#pragma unroll 1
  for (int shift = 21, above = 32; above > 0; above = shift, shift = shift == 21 ? 10 : 0) {
    hist[tid] = 0;
    hist[tid + 1024] = 0;
    __syncthreads();
#pragma unroll
    for (int y = 0; y < kPer; ++y)
      if (((uint64_t)(keys[y] ^ last) >> above) == 0) count_class(hist, keys[y] >> shift & (above == 10 ? 1023u : 2047u));
    __syncthreads();
    const uint32_t counts[2] = {hist[2047 - 2 * tid], hist[2046 - 2 * tid]};
    pick_class<2, kWaveCount>(counts, need, part, picked);
    __syncthreads();
    last |= picked[0] << shift;
    need = picked[1];
    if (picked[2] != 0) {  // the whole class is taken: all above its lowest key less one (no class holds key 0)
      last -= 1;
      need = 0;
      break;
    }
  }

#pragma unroll
  for (int y = 0; y < kPer; ++y) {
    const uint32_t u = (uint32_t)__popcll(__ballot(keys[y] > last)), e = (uint32_t)__popcll(__ballot(keys[y] == last));
    if (lane == 0) {
      ups[y * kWaveCount + wave] = u;  // the columns' order
      eqs[y * kWaveCount + wave] = e;
    }
  }
  __syncthreads();
  // (At most 8192 of either: both in one scan.)
  uint32_t all;
  const uint32_t ue = scan_before<kWaveCount>(tid < kGroups ? ups[tid] << 16 | eqs[tid] : 0u, part, &all);
  if (tid < kGroups) {
    ups[tid] = ue >> 16;
    eqs[tid] = ue & 0xffffu;
  }
  __syncthreads();
#pragma unroll
  for (int y = 0; y < kPer; ++y) {
    const uint64_t um = __ballot(keys[y] > last), em = __ballot(keys[y] == last), below = (1ull << lane) - 1;
    const uint32_t rank = eqs[y * kWaveCount + wave] + (uint32_t)__popcll(em & below);
    if (keys[y] > last || (keys[y] == last && rank < need))
      keep_token(a, r, row, ups[y * kWaveCount + wave] + (uint32_t)__popcll(um & below) + min(rank, need),
                 y * kSelThreads + tid);
  }
}

// A thread's keys of a part, all asked for at once: kPartKeys groups of 64 tokens a wave, in order.
__device__ __forceinline__ int part_column(int part, int y) {
  return part * kSelPart + ((int)threadIdx.x >> 6) * (64 * kPartKeys) + 64 * y + ((int)threadIdx.x & 63);
}
__device__ __forceinline__ void part_keys(uint32_t (&keys)[kPartKeys], const SelectRow& r, int part) {
#pragma unroll
  for (int y = 0; y < kPartKeys; ++y) keys[y] = r.key(part_column(part, y));
}

// Long rows, first launch: the counts of the top 11 bits of each part's keys.
__global__ __launch_bounds__(kPartThreads) void hh_part_count_kernel(HHLoadLaunch a) {
  __shared__ uint32_t hist[2048];
  const int64_t row = blockIdx.y;
  const int part = blockIdx.x, tid = threadIdx.x;
  const SelectRow r(a, row);
  if (keep_all(a, r, row, part, gridDim.x)) return;
  uint32_t keys[kPartKeys];
  part_keys(keys, r, part);
  for (int x = tid; x < 2048; x += kPartThreads) hist[x] = 0;
  if (part == 0 && tid == 0) a.rows[row].listed = 0;
  __syncthreads();
#pragma unroll
  for (int y = 0; y < kPartKeys; ++y) count_class(hist, keys[y] >> 21);
  __syncthreads();
  uint32_t* out = reinterpret_cast<uint32_t*>(a.part_counts) + (row * gridDim.x + part) * 1024;  // 16 bits a class
  for (int x = tid; x < 1024; x += kPartThreads) out[x] = hist[2 * x] | hist[2 * x + 1] << 16;
}

// Second launch: the class of the last taken token, from the counts of all parts of the row (every
// workgroup finds it for itself). Its members go to the row's list, in any order, each with its part; the
// part's tokens above it are counted.
__global__ __launch_bounds__(kPartThreads) void hh_part_list_kernel(HHLoadLaunch a) {
  constexpr int kWaveCount = kPartThreads / 64, kWords = 1024 / kPartThreads;
  __shared__ uint32_t wave_part[kWaveCount], wave_mine[kWaveCount], picked[3], higher, first;
  const int64_t row = blockIdx.y;
  const int part = blockIdx.x, parts = gridDim.x, tid = threadIdx.x, lane = tid & 63;
  const SelectRow r(a, row);
  if (r.n <= a.c.capacity) return;
  uint32_t keys[kPartKeys];
  part_keys(keys, r, part);
  uint32_t counts[2 * kWords] = {};
  const uint32_t* in = reinterpret_cast<const uint32_t*>(a.part_counts) + row * parts * 1024 + 1024 - kWords * (tid + 1);
#pragma unroll 8
  for (int p = 0; p < parts; ++p) {
#pragma unroll
    for (int y = 0; y < kWords; ++y) {
      const uint32_t x = in[p * 1024 + kWords - 1 - y];
      counts[2 * y] += x >> 16;
      counts[2 * y + 1] += x & 0xffffu;
    }
  }
  if (tid == 0) higher = 0;
  pick_class<2 * kWords, kWaveCount>(counts, (uint32_t)a.c.capacity, wave_part, picked);
  __syncthreads();
  const uint32_t cls = picked[0];
  if (part == 0 && tid == 0) {
    a.rows[row].cls = cls;
    a.rows[row].need = picked[1];
    a.rows[row].whole = picked[2];
  }
  u32x2* list = reinterpret_cast<u32x2*>(a.listed) + row * parts * kSelPart;
  uint32_t above = 0, mine = 0;
#pragma unroll
  for (int y = 0; y < kPartKeys; ++y) {
    above += (uint32_t)__popcll(__ballot(keys[y] >> 21 > cls));
    mine += (uint32_t)__popcll(__ballot(keys[y] >> 21 == cls));
  }
  if (lane == 0) {
    wave_mine[tid >> 6] = mine;
    if (above != 0) atomicAdd(&higher, above);
  }
  __syncthreads();
  if (tid == 0) {  // (one addition per workgroup: the row's 16 parts wait for each other)
    uint32_t sum = 0;
#pragma unroll
    for (int v = 0; v < kWaveCount; ++v) {
      const uint32_t x = wave_mine[v];
      wave_mine[v] = sum;
      sum += x;
    }
    first = sum != 0 ? atomicAdd(&a.rows[row].listed, sum) : 0u;
    a.part_above[row * parts + part] = higher;
  }
  __syncthreads();
  uint32_t base = first + wave_mine[tid >> 6];
#pragma unroll
  for (int y = 0; y < kPartKeys; ++y) {
    const bool in_class = keys[y] >> 21 == cls;
    const uint64_t mask = __ballot(in_class);
    if (in_class) list[base + (uint32_t)__popcll(mask & ((1ull << lane) - 1))] = u32x2{keys[y], (uint32_t)part};
    base += (uint32_t)__popcll(mask);
  }
}

// Third launch: the last key from the row's list, the part's first slot, its tokens' slots.
__global__ __launch_bounds__(kPartThreads) void hh_part_keep_kernel(HHLoadLaunch a) {
  constexpr int kWaveCount = kPartThreads / 64, kPer = 2048 / kPartThreads;
  __shared__ uint32_t hist[2048];
  __shared__ uint32_t wave_part[kWaveCount], picked[3], base_u, base_e, wave_u[kWaveCount], wave_e[kWaveCount];
  const int64_t row = blockIdx.y;
  const int part = blockIdx.x, parts = gridDim.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const SelectRow r(a, row);
  if (r.n <= a.c.capacity) return;
  uint32_t keys[kPartKeys];
  part_keys(keys, r, part);
  const HHSelectRow info = a.rows[row];
  const u32x2* list = reinterpret_cast<const u32x2*>(a.listed) + row * parts * kSelPart;
  const int m = (int)info.listed;
  uint32_t last = info.cls << 21, need = info.need;
  bool whole = info.whole != 0;
  uint32_t u = 0, e = 0;  // tokens of the parts before this one above the key, and equal to it
  for (int p = tid; p < part; p += kPartThreads) u += a.part_above[row * parts + p];
  if (tid == 0) base_u = base_e = 0;
#pragma unroll 1
  for (int shift = 10, above = 21; above > 0 && !whole; above = shift, shift = 0) {
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kPer; ++x) hist[tid + x * kPartThreads] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < m; i += kPartThreads) {
      const uint32_t key = list[i].x;
      if ((key ^ last) >> above == 0) count_class(hist, key >> shift & (above == 10 ? 1023u : 2047u));
    }
    __syncthreads();
    uint32_t counts[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) counts[x] = hist[2047 - kPer * tid - x];
    pick_class<kPer, kWaveCount>(counts, need, wave_part, picked);
    __syncthreads();
    last |= picked[0] << shift;
    need = picked[1];
    whole = picked[2] != 0;
  }
  if (whole) {  // the whole class is taken: all above its lowest key less one (no class holds key 0)
    last -= 1;
    need = 0;
  }
#pragma unroll 4
  for (int i = tid; i < m; i += kPartThreads) {
    const u32x2 x = list[i];
    if ((int)x.y < part) {
      u += x.x > last;
      e += x.x == last;
    }
  }
  __syncthreads();
  if (u != 0) atomicAdd(&base_u, u);
  if (e != 0) atomicAdd(&base_e, e);
  u = e = 0;
#pragma unroll
  for (int y = 0; y < kPartKeys; ++y) {
    u += (uint32_t)__popcll(__ballot(keys[y] > last));
    e += (uint32_t)__popcll(__ballot(keys[y] == last));
  }
  if (lane == 0) {
    wave_u[wave] = u;
    wave_e[wave] = e;
  }
  __syncthreads();
  u = base_u;
  e = base_e;
  for (int v = 0; v < wave; ++v) {
    u += wave_u[v];
    e += wave_e[v];
  }
#pragma unroll
  for (int y = 0; y < kPartKeys; ++y) {
    const uint64_t um = __ballot(keys[y] > last), em = __ballot(keys[y] == last), below = (1ull << lane) - 1;
    const uint32_t rank = e + (uint32_t)__popcll(em & below);
    // Before this token: those above the key, and of the equal ones as many as are taken.
    if (keys[y] > last || (keys[y] == last && rank < need))
      keep_token(a, r, row, u + (uint32_t)__popcll(um & below) + min(rank, need), part_column(part, y));
    u += (uint32_t)__popcll(um);
    e += (uint32_t)__popcll(em);
  }
}

// Keys and values of the kept columns, 16 bytes a thread.
__global__ __launch_bounds__(256) void hh_gather_kernel(HHLoadLaunch a) {
  const HHCache& c = a.c;
  const int64_t row = blockIdx.y;
  const int b = (int)(row / c.hkv), h = (int)(row - (int64_t)b * c.hkv);
  const int pieces = c.d / 8;  // 16-byte pieces of a token
  const int lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
  const int m = min(a.tokens - lo, c.capacity);
  const uint16_t* k = static_cast<const uint16_t*>(a.k) + b * a.ks.b + h * a.ks.h;
  const uint16_t* v = static_cast<const uint16_t*>(a.v) + b * a.vs.b + h * a.vs.h;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(id / pieces), e = (int)(id - (int64_t)i * pieces) * 8;
  if (i >= m) return;
  const int64_t t = a.kept[row * c.capacity + i];
  const u32x4 x = *reinterpret_cast<const u32x4_e*>(k + t * a.ks.t + e);
  const u32x4 y = *reinterpret_cast<const u32x4_e*>(v + t * a.vs.t + e);
  const int64_t to = (row * c.capacity + i) * c.d + e;
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(c.keys) + to) = x;
  *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(c.values) + to) = y;
}

template <class Ty, int D>
hipError_t attend_dim(const HHAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  const HHCache& c = p.c;
  const dim3 grid((unsigned)p.n_split, (unsigned)c.hkv, (unsigned)c.batch);
  if (p.n_split == 0) {  // one workgroup finishes a row
    constexpr int kW = D == 256 ? 4 : 8;
    hh_attend_kernel<Ty, D, kW, true><<<dim3(1, grid.y, grid.z), 64 * kW, 0, stream>>>(p, sc);
    return hipGetLastError();
  }
  hh_attend_kernel<Ty, D, 4, false><<<grid, 256, 0, stream>>>(p, sc);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 merge((unsigned)(c.hq / c.hkv + (c.capacity + 1023) / 1024), (unsigned)(c.batch * c.hkv));
  hh_attend_merge_kernel<Ty><<<merge, 256, 0, stream>>>(p);
  return hipGetLastError();
}

template <class Ty>
hipError_t attend(const HHAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  switch (p.c.d) {
    case 16: return attend_dim<Ty, 16>(p, sc, stream);
    case 32: return attend_dim<Ty, 32>(p, sc, stream);
    case 64: return attend_dim<Ty, 64>(p, sc, stream);
    case 128: return attend_dim<Ty, 128>(p, sc, stream);
    default: return attend_dim<Ty, 256>(p, sc, stream);
  }
}

}  // namespace

hipError_t launch_hh_append(int dtype, const HHAppendLaunch& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.c.hkv, (unsigned)p.c.batch);
  if (dtype == kF16)
    hh_append_kernel<HalfT><<<grid, 256, 0, stream>>>(p);
  else
    hh_append_kernel<Bf16T><<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

int hh_attend_splits(int batch, int hkv, int capacity, int d) {
  const int rows = batch * hkv;
  if (capacity <= (d == 256 ? kOneTokens / 2 : kOneTokens)) return 0;
  const int most = (capacity + 4 * kTileTokens - 1) / (4 * kTileTokens);  // a tile for each wave
  int n = (2048 + rows - 1) / rows;
  if (n > most) n = most;
  return n < 1 ? 1 : n > kMostSplits ? kMostSplits : n;
}

hipError_t launch_hh_attend(int dtype, const HHAttendLaunch& p, hipStream_t stream) {
  AttendScale sc;
  sc.scale_log2 = p.scale * kLog2e;
  sc.cap_scale = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  sc.cap_log2 = p.softcap > 0.f ? p.softcap * kLog2e : 0.f;
  return dtype == kF16 ? attend<HalfT>(p, sc, stream) : attend<Bf16T>(p, sc, stream);
}

int hh_select_parts(int tokens) { return (tokens + kSelPart - 1) / kSelPart; }
size_t hh_select_part_tokens() { return kSelPart; }

hipError_t launch_hh_load(const HHLoadLaunch& p, hipStream_t stream) {
  const unsigned rows = (unsigned)(p.c.batch * p.c.hkv);
  hipError_t e = hipSuccess;
  if (p.tokens <= kSelShort || p.tokens <= p.c.capacity) {
    hh_select_kernel<<<rows, kSelThreads, 0, stream>>>(p);
    e = hipGetLastError();
  } else {
    const dim3 grid((unsigned)hh_select_parts(p.tokens), rows);
    hh_part_count_kernel<<<grid, kPartThreads, 0, stream>>>(p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hh_part_list_kernel<<<grid, kPartThreads, 0, stream>>>(p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hh_part_keep_kernel<<<grid, kPartThreads, 0, stream>>>(p);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const int most = p.tokens < p.c.capacity ? p.tokens : p.c.capacity;
  const int64_t pieces = (int64_t)most * (p.c.d / 8);
  if (pieces == 0) return hipSuccess;
  hh_gather_kernel<<<dim3((unsigned)((pieces + 255) / 256), rows), 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace pgr
