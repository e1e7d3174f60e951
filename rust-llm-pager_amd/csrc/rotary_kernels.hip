// Rotary position embedding of q and k.
//
//   (x, y) -> factor * (x cos a - y sin a, x sin a + y cos a),   a = position * inv_freq[i]
//
// for the pairs (i, i + half) or (2i, 2i + 1) of each head's first 2 * half dims; the rest of the
// head is copied. Memory-bound: every element is read and written once.
#include <hip/hip_runtime.h>

#include "cache_device.h"

namespace pgr {
namespace {

template <class Ty, int kV>
struct Vec {
  typedef typename Ty::Raw Raw;
  Raw e[kV];
};

template <class Ty, int kV>
__device__ __forceinline__ Vec<Ty, kV> load_vec(const typename Ty::Raw* p) {
  Vec<Ty, kV> v;
  if constexpr (kV == 1) {
    v.e[0] = *p;
  } else {
    static_assert(sizeof(v) == 16, "one 16-byte access");
    const u32x4 x = *reinterpret_cast<const u32x4_e*>(p);
    v = __builtin_bit_cast(Vec<Ty, kV>, x);
  }
  return v;
}

template <class Ty, int kV>
__device__ __forceinline__ void store_vec(typename Ty::Raw* p, const Vec<Ty, kV>& v) {
  if constexpr (kV == 1)
    *p = v.e[0];
  else
    *reinterpret_cast<u32x4_e*>(p) = __builtin_bit_cast(u32x4, v);
}

// A thread owns one unit of one token (two vectors of kV elements: kV pairs, or a piece of the
// part that is copied) and walks `per` heads with it, so that its angles are taken once.
template <class Ty, int kV, bool kInterleaved>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryLaunch a, int64_t n_units, int per) {
  typedef typename Ty::Raw Raw;
  const int half = a.form.half, rest = a.d - 2 * half;
  const int turning = half / kV, units = turning + (rest + 2 * kV - 1) / (2 * kV);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= n_units) return;
  const int64_t token = id / units;
  const int u = (int)(id - token * units);
  const int b = (int)(token / a.tokens), t = (int)(token - (int64_t)b * a.tokens);

  int first, second;  // element offsets of the unit's two vectors
  bool two = true;
  float cs[kV], sn[kV];
  const bool turns = u < turning;
  if (turns) {
    first = kInterleaved ? 2 * u * kV : u * kV;
    second = kInterleaved ? first + kV : half + first;
    const int64_t pos = load_position(a.positions, a.positions64, b * a.pos_b + t * a.pos_t);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      turn(pos, a.form.inv_freq[u * kV + i], cs[i], sn[i]);
      cs[i] *= a.form.factor;
      sn[i] *= a.form.factor * a.form.sign;
    }
  } else {
    first = 2 * half + (u - turning) * 2 * kV;
    second = first + kV;
    two = second < a.d;
    if (!two) second = first;
  }

  const int total = a.heads[0] + a.heads[1];
  const int h_begin = blockIdx.y * per, h_end = min(h_begin + per, total);
#pragma unroll 4
  for (int h = h_begin; h < h_end; ++h) {
    const int s = h >= a.heads[0];
    const int hh = s ? h - a.heads[0] : h;
    const Raw* x = static_cast<const Raw*>(a.x[s]) + b * a.xs[s].b + hh * a.xs[s].h + t * a.xs[s].t;
    Raw* y = static_cast<Raw*>(a.y[s]) + (((int64_t)b * a.heads[s] + hh) * a.tokens + t) * a.d;
    Vec<Ty, kV> p = load_vec<Ty, kV>(x + first), q = load_vec<Ty, kV>(x + second);
    if (turns) {
      if constexpr (kInterleaved && kV > 1) {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          Vec<Ty, kV>& w = i < kV / 2 ? p : q;
          const int j = 2 * (i % (kV / 2));
          const float c = Ty::to_f(w.e[j]), d = Ty::to_f(w.e[j + 1]);
          w.e[j] = Ty::cvt(turned_x(c, d, cs[i], sn[i]));
          w.e[j + 1] = Ty::cvt(turned_y(c, d, cs[i], sn[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          const float c = Ty::to_f(p.e[i]), d = Ty::to_f(q.e[i]);
          p.e[i] = Ty::cvt(turned_x(c, d, cs[i], sn[i]));
          q.e[i] = Ty::cvt(turned_y(c, d, cs[i], sn[i]));
        }
      }
    }
    store_vec<Ty, kV>(y + first, p);
    if (two) store_vec<Ty, kV>(y + second, q);
  }
}

template <class Ty, int kV>
hipError_t rotary(const RotaryLaunch& p, hipStream_t stream) {
  const int rest = p.d - 2 * p.form.half;
  const int units = p.form.half / kV + (rest + 2 * kV - 1) / (2 * kV);
  const int64_t n = (int64_t)p.batch * p.tokens * units;
  const int total = p.heads[0] + p.heads[1];
  if (n == 0 || total == 0) return hipSuccess;
  const int64_t blocks = (n + 255) / 256;
  int64_t parts = (2048 + blocks - 1) / blocks;  // head parts: about 2048 workgroups
  if (parts > total) parts = total;
  const int per = (int)((total + parts - 1) / parts);
  const dim3 grid((unsigned)blocks, (unsigned)((total + per - 1) / per));
  if (p.form.interleaved)
    rotary_kernel<Ty, kV, true><<<grid, 256, 0, stream>>>(p, n, per);
  else
    rotary_kernel<Ty, kV, false><<<grid, 256, 0, stream>>>(p, n, per);
  return hipGetLastError();
}

template <class Ty>
hipError_t rotary_any(const RotaryLaunch& p, hipStream_t stream) {
  constexpr int kV = 16 / (int)sizeof(typename Ty::Raw);
  // 16-byte pieces where both the rotary half and the copied part are whole numbers of them.
  if (p.form.half % kV == 0 && (p.d - 2 * p.form.half) % kV == 0) return rotary<Ty, kV>(p, stream);
  return rotary<Ty, 1>(p, stream);
}

}  // namespace

hipError_t launch_rotary(int dtype, const RotaryLaunch& p, hipStream_t stream) {
  if (dtype == kF16) return rotary_any<HalfT>(p, stream);
  if (dtype == kBF16) return rotary_any<Bf16T>(p, stream);
  return rotary_any<FloatT>(p, stream);
}

}  // namespace pgr
