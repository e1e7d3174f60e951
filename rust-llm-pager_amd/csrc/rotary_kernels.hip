// Rotary position embedding of q and k.
//
//   (x, y) -> factor * (x cos a - y sin a, x sin a + y cos a),   a = position * inv_freq[i]
//
// for the pairs (i, i + half) or (2i, 2i + 1) of each head's first 2 * half dims; the rest of the
// head is copied. Memory-bound: every element is read and written once, in 16-byte pieces that
// neighbouring threads read side by side. 4 x 8191 tokens, 32/8 heads, D 128, 64 dims turned in adjacent
// pairs, fp16: 138 us for 671 MB (4.9 TB/s; a copy reaches 5.1), 152 us with two pieces 32 bytes apart per
// thread. One token of 14/2 heads: 4.1 us, a launch.
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

// A thread owns one unit of one token and walks `per` heads with it, so that its angles are taken
// once. A unit is what 16 bytes allow (kV elements): kV pairs of the half layout, in two places; kV / 2
// neighbouring pairs, or kV elements of the part that is copied, in one.
template <class Ty, int kV, bool kInterleaved>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryLaunch a, int64_t n_units, int units, int per) {
  typedef typename Ty::Raw Raw;
  constexpr int kPairs = kInterleaved && kV > 1 ? kV / 2 : kV;
  const int half = a.form.half, turning = half / kPairs;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= n_units) return;
  const int64_t token = id / units;
  const int u = (int)(id - token * units);
  const int b = (int)(token / a.tokens), t = (int)(token - (int64_t)b * a.tokens);

  // Element offsets of the unit; a unit in one place has no second.
  const bool turns = u < turning;
  const bool two = turns && (!kInterleaved || kV == 1);
  const int first = !turns ? 2 * half + (u - turning) * kV : kInterleaved ? 2 * u * kPairs : u * kPairs;
  const int second = kInterleaved ? first + 1 : first + half;
  float cs[kPairs], sn[kPairs];
  if (turns) {
    const int64_t pos = load_position(a.positions, a.positions64, b * a.pos_b + t * a.pos_t);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      turn(pos, a.form.inv_freq[u * kPairs + i], cs[i], sn[i]);
      cs[i] *= a.form.factor;
      sn[i] *= a.form.factor * a.form.sign;
    }
  }

  const int h_begin = blockIdx.y * per, h_end = min(h_begin + per, a.heads[0] + a.heads[1]);
#pragma unroll
  for (int s = 0; s < 2; ++s) {  // q's heads of [h_begin, h_end), then k's
    const int from = s == 0 ? h_begin : max(h_begin - a.heads[0], 0);
    const int to = s == 0 ? min(h_end, a.heads[0]) : h_end - a.heads[0];
    const Raw* x = static_cast<const Raw*>(a.x[s]) + b * a.xs[s].b + t * a.xs[s].t;
    Raw* y = static_cast<Raw*>(a.y[s]) + ((int64_t)b * a.heads[s] * a.tokens + t) * a.d;
    const int64_t step = (int64_t)a.tokens * a.d;
#pragma unroll 4
    for (int h = from; h < to; ++h) {
      const Raw* xh = x + h * a.xs[s].h;
      Raw* yh = y + h * step;
      Vec<Ty, kV> p = load_vec<Ty, kV>(xh + first), q = p;
      if (two) q = load_vec<Ty, kV>(xh + second);
      if (turns) {
        if constexpr (kInterleaved && kV > 1) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float c = Ty::to_f(p.e[2 * i]), d = Ty::to_f(p.e[2 * i + 1]);
            p.e[2 * i] = Ty::cvt(turned_x(c, d, cs[i], sn[i]));
            p.e[2 * i + 1] = Ty::cvt(turned_y(c, d, cs[i], sn[i]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            const float c = Ty::to_f(p.e[i]), d = Ty::to_f(q.e[i]);
            p.e[i] = Ty::cvt(turned_x(c, d, cs[i], sn[i]));
            q.e[i] = Ty::cvt(turned_y(c, d, cs[i], sn[i]));
          }
        }
      }
      store_vec<Ty, kV>(yh + first, p);
      if (two) store_vec<Ty, kV>(yh + second, q);
    }
  }
}

template <class Ty, int kV>
hipError_t rotary(const RotaryLaunch& p, hipStream_t stream) {
  const int pairs = p.form.interleaved && kV > 1 ? kV / 2 : kV;
  const int units = p.form.half / pairs + (p.d - 2 * p.form.half) / kV;
  const int64_t n = (int64_t)p.batch * p.tokens * units;
  const int total = p.heads[0] + p.heads[1];
  if (n == 0 || total == 0) return hipSuccess;
  const int64_t blocks = (n + 255) / 256;
  int64_t parts = (2048 + blocks - 1) / blocks;  // head parts: about 2048 workgroups
  if (parts > total) parts = total;
  const int per = (int)((total + parts - 1) / parts);
  const dim3 grid((unsigned)blocks, (unsigned)((total + per - 1) / per));
  if (p.form.interleaved)
    rotary_kernel<Ty, kV, true><<<grid, 256, 0, stream>>>(p, n, units, per);
  else
    rotary_kernel<Ty, kV, false><<<grid, 256, 0, stream>>>(p, n, units, per);
  return hipGetLastError();
}

template <class Ty>
hipError_t rotary_any(const RotaryLaunch& p, hipStream_t stream) {
  constexpr int kV = 16 / (int)sizeof(typename Ty::Raw);
  // 16-byte pieces where the rotary part (half layout: each half) and the copied part are whole numbers
  // of them.
  const int piece = p.form.interleaved ? 2 * p.form.half : p.form.half;
  if (piece % kV == 0 && (p.d - 2 * p.form.half) % kV == 0) return rotary<Ty, kV>(p, stream);
  return rotary<Ty, 1>(p, stream);
}

}  // namespace

hipError_t launch_rotary(int dtype, const RotaryLaunch& p, hipStream_t stream) {
  if (dtype == kF16) return rotary_any<HalfT>(p, stream);
  if (dtype == kBF16) return rotary_any<Bf16T>(p, stream);
  return rotary_any<FloatT>(p, stream);
}

}  // namespace pgr
