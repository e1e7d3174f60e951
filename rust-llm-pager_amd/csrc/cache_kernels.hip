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
// equal, and NaN (one key for all of them) is the heaviest.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint64_t min_u64(uint64_t a, uint64_t b) { return a < b ? a : b; }

__device__ __forceinline__ uint64_t shuffle_xor(uint64_t x, int mask) {
  const uint32_t lo = __shfl_xor((uint32_t)x, mask), hi = __shfl_xor((uint32_t)(x >> 32), mask);
  return (uint64_t)hi << 32 | lo;
}

// Element i of a head's rotary part (or of its copied part) after the turn.
template <class Ty>
__device__ __forceinline__ float turned(const typename Ty::Raw* x, int i, const RotaryForm& f, int64_t pos) {
  const float own = Ty::to_f(x[i]);
  if (i >= 2 * f.half) return own;
  const bool first = f.interleaved ? (i & 1) == 0 : i < f.half;
  const int pair = f.interleaved ? i >> 1 : (first ? i : i - f.half);
  const int mate = f.interleaved ? i ^ 1 : (first ? i + f.half : i - f.half);
  float cs, sn;
  turn(pos, f.inv_freq[pair], cs, sn);
  cs *= f.factor;
  sn *= f.factor * f.sign;
  const float other = Ty::to_f(x[mate]);
  return first ? turned_x(own, other, cs, sn) : turned_y(other, own, cs, sn);
}

// One workgroup per row: the new token's slot (the next free one, or in a full row the lightest
// token's that is neither among the first keep_first nor among the last keep_recent, the new one
// counted), its turned key, its value, and the turned queries of the row's heads.
template <class Ty>
__global__ __launch_bounds__(256) void hh_append_kernel(HHAppendLaunch a) {
  typedef typename Ty::Raw Raw;
  __shared__ uint64_t best_s[4];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const HHCache& c = a.c;
  const int64_t row = (int64_t)b * c.hkv + h;
  const int seen = c.seen[row];
  const int length = min(max(c.lengths[row], 0), c.capacity);
  const bool full = length == c.capacity;
  float* w = c.weights + row * c.capacity;
  int32_t* order = c.order + row * c.capacity;

  int slot = length;
  if (full) {
    uint64_t best = ~0ull;
    const int64_t recent = (int64_t)seen + 1 - c.keep_recent;
    for (int i = tid; i < c.capacity; i += 256) {
      const int32_t o = order[i];
      const uint64_t held = o < c.keep_first || o >= recent;
      best = min_u64(best, held << 63 | (uint64_t)weight_key(w[i]) << 31 | (uint64_t)i);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) best = min_u64(best, shuffle_xor(best, m));
    if ((tid & 63) == 0) best_s[tid >> 6] = best;
    __syncthreads();
    best = min_u64(min_u64(best_s[0], best_s[1]), min_u64(best_s[2], best_s[3]));
    slot = (int)(best & 0x7fffffffu);
  }

  const int64_t pos =
      a.positions != nullptr ? load_position(a.positions, a.positions64, b) : (int64_t)seen;
  const int d = c.d, n_rep = c.hq / c.hkv;
  const Raw* k = static_cast<const Raw*>(a.k) + b * a.ks.b + h * a.ks.h;
  const Raw* v = static_cast<const Raw*>(a.v) + b * a.vs.b + h * a.vs.h;
  Raw* ko = static_cast<Raw*>(c.keys) + (row * c.capacity + slot) * d;
  Raw* vo = static_cast<Raw*>(c.values) + (row * c.capacity + slot) * d;
  for (int i = tid; i < d; i += 256) {
    ko[i] = a.form.inv_freq != nullptr ? Ty::cvt(turned<Ty>(k, i, a.form, pos)) : k[i];
    vo[i] = v[i];
  }
  if (a.q_out != nullptr) {
    Raw* qo = static_cast<Raw*>(a.q_out) + ((int64_t)b * c.hq + (int64_t)h * n_rep) * d;
    for (int i = tid; i < n_rep * d; i += 256) {
      const int r = i / d, e = i - r * d;
      const Raw* q = static_cast<const Raw*>(a.q) + b * a.qs.b + ((int64_t)h * n_rep + r) * a.qs.h;
      qo[i] = a.form.inv_freq != nullptr ? Ty::cvt(turned<Ty>(q, e, a.form, pos)) : q[e];
    }
  }
  __syncthreads();  // every thread has read the row's state
  if (tid == 0) {
    w[slot] = 0.f;
    order[slot] = seen;
    c.seen[row] = seen + 1;
    c.lengths[row] = full ? length : length + 1;
  }
}

// ---------------------------------------------------------------------------------------
// Attention of one new token. MFMA tiles as in the decode kernels: a 16-token tile is
//     S^T[16 tok x 16 heads] = K . Q^T,   O^T[D x 16 heads] += V^T . P^T
// lane (g, n) holding tokens 4g..4g+3 of query head n, so the softmax state is a per-lane scalar.
template <int D>
struct KVTile {
  static constexpr int KD = D / 8;                     // dwords: D/4 elements of K row n
  static constexpr int VD = D >= 32 ? D / 32 : 1;      // dwords: D/16 elements of each of 4 V rows
  uint32_t k[KD];
  uint32_t v[4][VD];
};

template <int N>
__device__ __forceinline__ void load_dwords(uint32_t (&r)[N], const uint16_t* src) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 x = *reinterpret_cast<const u32x4_e*>(src + 8 * i);
#pragma unroll
      for (int c = 0; c < 4; ++c) r[4 * i + c] = x[c];
    }
  } else {
    typedef uint32_t u32_e __attribute__((aligned(2)));
    typedef uint32_t u32x2_e __attribute__((ext_vector_type(2), aligned(2)));
    if constexpr (N == 2) {
      const u32x2 x = *reinterpret_cast<const u32x2_e*>(src);
      r[0] = x.x;
      r[1] = x.y;
    } else {
      static_assert(N == 1, "1, 2 or a multiple of 4 dwords");
      r[0] = *reinterpret_cast<const u32_e*>(src);
    }
  }
}

__device__ __forceinline__ float max_g(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_g(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Scores in log2 units: scale_log2 = scale * log2(e), or with a softcap cap * log2(e).
__device__ __forceinline__ float log2_score(float s, float scale_log2, float cap_scale, float cap_log2) {
  return cap_log2 > 0.f ? cap_log2 * tanhf(s * cap_scale) : s * scale_log2;
}

struct AttendScale {
  float scale_log2, cap_scale, cap_log2;
};

// Tokens [begin, end) of a row of `length` that split `split` of n_split takes: whole 16-token
// tiles, evenly.
__device__ __forceinline__ void split_range(int length, int split, int n_split, int& begin, int& end) {
  const int tiles = (length + 15) / 16, per = (tiles + n_split - 1) / n_split;
  begin = min(split * per, tiles) * 16;
  end = min(min((split + 1) * per, tiles) * 16, length);
}

template <class Ty, int D>
__global__ __launch_bounds__(256) void hh_attend_kernel(HHAttendLaunch a, AttendScale sc) {
  typedef KVTile<D> T;
  constexpr int kRep = kMaxRep;
  __shared__ float sm_m[kWaves][kRep], sm_l[kWaves][kRep];
  __shared__ float sm_acc[kWaves][kRep][D + 1];
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const HHCache& c = a.c;
  const int n_rep = c.hq / c.hkv;
  const int64_t row = (int64_t)b * c.hkv + h;
  const int length = min(max(c.lengths[row], 0), c.capacity);
  int begin, end;
  split_range(length, split, a.n_split, begin, end);
  if (begin >= end) return;  // uniform; the merge reads the splits that hold tokens
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const bool real = n < n_rep;
  const uint16_t* kp = static_cast<const uint16_t*>(c.keys) + row * c.capacity * D;
  const uint16_t* vp = static_cast<const uint16_t*>(c.values) + row * c.capacity * D;
  const int tiles = (end - begin + 15) / 16;

  auto fetch = [&](T& t, int ti) {
    const int t0 = begin + ti * 16;
    load_dwords(t.k, kp + (int64_t)min(t0 + n, end - 1) * D + (D / 4) * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t* p = vp + (int64_t)min(t0 + 4 * g + i, end - 1) * D + (D / 16) * n;
      if constexpr (D < 32)
        t.v[i][0] = *p;
      else
        load_dwords(t.v[i], p);
    }
  };

  uint32_t q[T::KD];
#pragma unroll
  for (int i = 0; i < T::KD; ++i) q[i] = 0u;
  if (real)
    load_dwords(q, static_cast<const uint16_t*>(a.q) + b * a.qs.b + ((int64_t)h * n_rep + n) * a.qs.h + (D / 4) * g);

  float m_run = kMinusInf, l_run = 0.f;
  f32x4 acc[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t stride = hh_attend_stride(c.capacity);
  float* lg = a.logits + ((int64_t)b * c.hq + (int64_t)h * n_rep + n) * stride;

  for (int ti = wave; ti < tiles; ti += kWaves) {
    T t;
    fetch(t, ti);
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < T::KD; i += 2) s = Ty::mma16(u32x2{t.k[i], t.k[i + 1]}, u32x2{q[i], q[i + 1]}, s);
    const int tok = begin + ti * 16 + 4 * g;
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool ok = tok + i < end;
      x[i] = ok ? log2_score(s[i], sc.scale_log2, sc.cap_scale, sc.cap_log2) : kMinusInf;
      if (!ok) {
#pragma unroll
        for (int j = 0; j < T::VD; ++j) t.v[i][j] = 0u;
      }
    }
    if (real) *reinterpret_cast<f32x4*>(lg + tok) = x;
    const float m_new = fmaxf(m_run, max_g(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]))));
    const bool none = m_new == kMinusInf;
    const float alpha = none ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = none ? 0.f : __builtin_amdgcn_exp2f(x[i] - m_new);
    l_run = l_run * alpha + ((p[0] + p[1]) + (p[2] + p[3]));
    // P is rounded to the K/V type for the matrix cores, as in the framework's other decode kernels.
    const u32x2 pb = {Ty::pack(p[0], p[1]), Ty::pack(p[2], p[3])};
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
      const int e = j >> 1;
      const u32x2 vt = {__builtin_amdgcn_perm(t.v[1][e], t.v[0][e], sel),
                        __builtin_amdgcn_perm(t.v[3][e], t.v[2][e], sel)};
      acc[j] = Ty::mma16(vt, pb, acc[j] * alpha);
    }
    m_run = m_new;
  }

  const float l_wave = sum_g(l_run);
  if (g == 0) {
    sm_m[wave][n] = m_run;
    sm_l[wave][n] = l_wave;
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sm_acc[wave][n][(D / 4) * g + (D / 16) * i + j] = acc[j][i];
  __syncthreads();
  const int64_t part = (row * a.n_split + split) * n_rep;
  for (int i = threadIdx.x; i < n_rep * D; i += 256) {
    const int r = i / D, e = i - r * D;
    float m = kMinusInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, sm_m[w][r]);
    float x = 0.f, l = 0.f;
    if (m != kMinusInf) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(sm_m[w][r] - m);
        x += sm_acc[w][r][e] * f;
        l += sm_l[w][r] * f;
      }
    }
    a.pacc[part * D + i] = x;
    if (e == 0) {
      a.pm[part + r] = m;
      a.pl[part + r] = l;
    }
  }
}

// Joins the splits. Workgroups x < n_rep of a row write the output of query head x; the others add
// the probabilities of 1024 tokens each, summed over the row's heads in their order, to the weights.
template <class Ty>
__global__ __launch_bounds__(256) void hh_attend_merge_kernel(HHAttendLaunch a) {
  typedef typename Ty::Raw Raw;
  __shared__ float norm_s[kMaxRep];
  const HHCache& c = a.c;
  const int n_rep = c.hq / c.hkv, d = c.d, tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const int b = (int)(row / c.hkv), h = (int)(row - (int64_t)b * c.hkv);
  const int length = min(max(c.lengths[row], 0), c.capacity);
  const int tiles = (length + 15) / 16, per = (tiles + a.n_split - 1) / a.n_split;
  const int used = per > 0 ? (tiles + per - 1) / per : 0;
  const float* pm = a.pm + row * a.n_split * n_rep;
  const float* pl = a.pl + row * a.n_split * n_rep;
  const int x = blockIdx.x;
  if (x < n_rep) {
    float m = kMinusInf;
    for (int s = 0; s < used; ++s) m = fmaxf(m, pm[s * n_rep + x]);
    float l = 0.f;
    for (int s = 0; s < used; ++s) l += m == kMinusInf ? 0.f : pl[s * n_rep + x] * __builtin_amdgcn_exp2f(pm[s * n_rep + x] - m);
    const float* pacc = a.pacc + (row * a.n_split * n_rep + x) * d;
    Raw* out = static_cast<Raw*>(a.out) + ((int64_t)b * c.hq + (int64_t)h * n_rep + x) * d;
    for (int e = tid; e < d; e += 256) {
      float o = 0.f;
      for (int s = 0; s < used; ++s)
        o += m == kMinusInf ? 0.f : pacc[(int64_t)s * n_rep * d + e] * __builtin_amdgcn_exp2f(pm[s * n_rep + x] - m);
      out[e] = Ty::cvt(used > 0 ? o / l : 0.f);
    }
    return;
  }
  const int first = (x - n_rep) * 1024;
  if (first >= length) return;
  if (tid < n_rep) {
    float m = kMinusInf;
    for (int s = 0; s < used; ++s) m = fmaxf(m, pm[s * n_rep + tid]);
    float l = 0.f;
    for (int s = 0; s < used; ++s) l += m == kMinusInf ? 0.f : pl[s * n_rep + tid] * __builtin_amdgcn_exp2f(pm[s * n_rep + tid] - m);
    norm_s[tid] = m + __builtin_amdgcn_logf(l);  // log2
  }
  __syncthreads();
  const int64_t stride = hh_attend_stride(c.capacity);
  const float* lg = a.logits + ((int64_t)b * c.hq + (int64_t)h * n_rep) * stride;
  for (int t = first + tid; t < min(first + 1024, length); t += 256) {
    float sum = 0.f;
    for (int r = 0; r < n_rep; ++r) sum += __builtin_amdgcn_exp2f(lg[r * stride + t] - norm_s[r]);
    c.weights[row * c.capacity + t] += sum;
  }
}

// ---------------------------------------------------------------------------------------
// Which of a prompt's tokens stay. One workgroup per row. More tokens than slots: the first
// keep_first and the last keep_recent, and of those between the capacity's remainder by weight,
// the lowest column first among equals. The weight of the last one taken is found byte by byte
// from the top (four counts of 256 classes), then one pass writes the kept columns in order.
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

__global__ __launch_bounds__(kSelThreads) void hh_select_kernel(HHLoadLaunch a) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t picked[2];  // class taken in this round, tokens still to take in it
  __shared__ int base_s[kSelWaves][2];
  const HHCache& c = a.c;
  const int64_t row = blockIdx.x;
  const int b = (int)(row / c.hkv), tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int lo = a.lo != nullptr ? min(max(a.lo[b], 0), a.tokens) : 0;
  const int n = a.tokens - lo;
  const float* w = a.weights + row * a.tokens + lo;
  int32_t* kept = a.kept + row * c.capacity;
  float* wo = c.weights + row * c.capacity;
  int32_t* order = c.order + row * c.capacity;
  if (tid == 0) {
    c.lengths[row] = min(n, c.capacity);
    c.seen[row] = n;
  }
  if (n <= c.capacity) {
    for (int i = tid; i < n; i += kSelThreads) {
      kept[i] = lo + i;
      wo[i] = w[i];
      order[i] = i;
    }
    return;
  }
  const int mid0 = c.keep_first, mid1 = n - c.keep_recent;  // mid1 - mid0 > need, since n > capacity
  uint32_t need = (uint32_t)(c.capacity - c.keep_first - c.keep_recent);
  uint32_t prefix = 0, mask = 0;  // of the last taken token's key
  if (need > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = mid0 + tid; i < mid1; i += kSelThreads) {
        const uint32_t key = weight_key(w[i]);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t left = need;
        int cls = 255;
        while (hist[cls] < left) left -= hist[cls--];
        picked[0] = (uint32_t)cls;
        picked[1] = left;
      }
      __syncthreads();
      prefix |= picked[0] << shift;
      mask |= 255u << shift;
      need = picked[1];
    }
  }
  // `need` tokens of key == prefix are taken, and every one above it. Each wave takes a stretch of
  // columns, 64 at a time; its first slot and first equal token come from the waves before it.
  const bool none = c.capacity == c.keep_first + c.keep_recent;
  const int chunk = ((n + kSelWaves - 1) / kSelWaves + 63) / 64 * 64;
  const int from = min(wave * chunk, n), to = min(from + chunk, n);
  int above = 0, equal = 0;
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    bool up = false, eq = false;
    if (i < to) {
      if (i < mid0 || i >= mid1) {
        up = true;
      } else if (!none) {
        const uint32_t key = weight_key(w[i]);
        up = key > prefix;
        eq = key == prefix;
      }
    }
    above += __popcll(__ballot(up));
    equal += __popcll(__ballot(eq));
  }
  if (lane == 0) {
    base_s[wave][0] = above;
    base_s[wave][1] = equal;
  }
  __syncthreads();
  int slot = 0, rank = 0;
  for (int v = 0; v < wave; ++v) {
    slot += base_s[v][0];
    rank += base_s[v][1];
  }
  slot += min(rank, (int)need);
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    bool up = false, eq = false;
    float x = 0.f;
    if (i < to) {
      x = w[i];
      if (i < mid0 || i >= mid1) {
        up = true;
      } else if (!none) {
        const uint32_t key = weight_key(x);
        up = key > prefix;
        eq = key == prefix;
      }
    }
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t eqs = __ballot(eq);
    const bool take = up || (eq && rank + __popcll(eqs & below) < (int)need);
    const uint64_t takes = __ballot(take);
    const int at = slot + __popcll(takes & below);
    if (take && at < c.capacity) {
      kept[at] = lo + i;
      wo[at] = x;
      order[at] = i;
    }
    rank += __popcll(eqs);
    slot += __popcll(takes);
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

template <class Ty>
hipError_t attend(const HHAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  const HHCache& c = p.c;
  const dim3 grid((unsigned)p.n_split, (unsigned)c.hkv, (unsigned)c.batch);
  switch (c.d) {
    case 16: hh_attend_kernel<Ty, 16><<<grid, 256, 0, stream>>>(p, sc); break;
    case 32: hh_attend_kernel<Ty, 32><<<grid, 256, 0, stream>>>(p, sc); break;
    case 64: hh_attend_kernel<Ty, 64><<<grid, 256, 0, stream>>>(p, sc); break;
    case 128: hh_attend_kernel<Ty, 128><<<grid, 256, 0, stream>>>(p, sc); break;
    default: hh_attend_kernel<Ty, 256><<<grid, 256, 0, stream>>>(p, sc); break;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int n_rep = c.hq / c.hkv;
  const dim3 merge((unsigned)(n_rep + (c.capacity + 1023) / 1024), (unsigned)(c.batch * c.hkv));
  hh_attend_merge_kernel<Ty><<<merge, 256, 0, stream>>>(p);
  return hipGetLastError();
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

int hh_attend_splits(int batch, int hkv, int capacity) {
  const int most = (capacity + 63) / 64;  // a tile for each wave
  const int want = (1024 + batch * hkv - 1) / (batch * hkv);
  const int n = most < want ? most : want;
  return n < 1 ? 1 : n;
}

hipError_t launch_hh_attend(int dtype, const HHAttendLaunch& p, hipStream_t stream) {
  AttendScale sc;
  sc.scale_log2 = p.scale * kLog2e;
  sc.cap_scale = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  sc.cap_log2 = p.softcap > 0.f ? p.softcap * kLog2e : 0.f;
  return dtype == kF16 ? attend<HalfT>(p, sc, stream) : attend<Bf16T>(p, sc, stream);
}

hipError_t launch_hh_load(const HHLoadLaunch& p, hipStream_t stream) {
  const unsigned rows = (unsigned)(p.c.batch * p.c.hkv);
  hh_select_kernel<<<rows, kSelThreads, 0, stream>>>(p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int most = p.tokens < p.c.capacity ? p.tokens : p.c.capacity;
  const int64_t pieces = (int64_t)most * (p.c.d / 8);
  if (pieces == 0) return hipSuccess;
  hh_gather_kernel<<<dim3((unsigned)((pieces + 255) / 256), rows), 256, 0, stream>>>(p);
  return hipGetLastError();
}

}  // namespace pgr
