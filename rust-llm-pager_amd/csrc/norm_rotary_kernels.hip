// RMS norm of each head of q and k and their rotary embedding in one pass, into new tensors or, with v, into
// the pages of a cache.
//
//   y = R(position) (x / sqrt(mean(x^2) + eps) * weight)
//
// in float32 from the operands' elements to one rounding at the end; R as in the rotary embedding.
// Memory-bound: every element is read and written once. A head is held by the lanes of a group, two
// 16-byte pieces each: the pieces of a pair's halves where the pairs are (i, i + half), pieces a group's
// width apart otherwise, so that neighbouring lanes read side by side. The mean is summed over the group
// by lane exchanges; the angles and weights are taken once for all heads a thread walks, four heads' pieces asked
// for at a time. 4 x 8191 tokens, 32/8 heads, D 128, bf16: 137 us for 671 MB (4.9 TB/s; a copy reaches 5.1), 145 with
// one head after the other; the append of as many, up to 3/8 of a row's columns not its own: 154 us for 704 MB, 173
// where those columns are read all the same.
#include <hip/hip_runtime.h>

#include "cache_device.h"
#include "page_table_kernels.h"

namespace pgr {
namespace {

// Where a new token goes: its row of the pool (keys' and values' elements from head 0 on), or -1 where it has
// no place: behind the row's new tokens or the table's end, or in a page that the pool does not have.
__device__ __forceinline__ int64_t slot_of(const PTPages& c, const PTRows& r, int b, int64_t token) {
  const int64_t page = token >> c.page_shift;
  if (token < 0 || page >= r.width) return -1;
  const int32_t p = r.table[b * r.table_stride + page];
  if (p < 0 || p >= c.pages) return -1;
  const int64_t in = token & (((int64_t)1 << c.page_shift) - 1);
  return (((int64_t)p * c.hkv << c.page_shift) + in) * c.d;
}

// A token of the call: its position, its place in the pool, whether it is one of its row's new ones.
struct Token {
  int64_t pos, slot;
  bool has;
};

template <bool kPages>
__device__ __forceinline__ Token token_of(const NormRotaryLaunch& a, int b, int t) {
  Token k;
  k.has = true;
  k.slot = -1;
  int64_t length = 0;
  if constexpr (kPages) {
    length = max(a.r.lengths[b], 0);
    k.has = a.r.counts == nullptr || t < a.r.counts[b];
    if (k.has) k.slot = slot_of(a.c, a.r, b, length + t);
  }
  if (!kPages || a.positions != nullptr)
    k.pos = a.form.half > 0 ? load_position(a.positions, a.positions64, b * a.pos_b + t * a.pos_t) : 0;
  else
    k.pos = length + (a.depths != nullptr ? max(a.depths[(int64_t)b * a.tokens + t], 0) : t);
  return k;
}

template <class Ty>
__device__ __forceinline__ float weight_of(const HeadNorm& n, int which, int i) {
  return n.weight_f32 ? static_cast<const float*>(n.weight[which])[i]
                      : Ty::to_f(static_cast<const typename Ty::Raw*>(n.weight[which])[i]);
}

// Destination of head h of q (0), k (1) or v (2); null: nowhere.
template <bool kPages>
__device__ __forceinline__ char* target(const NormRotaryLaunch& a, const Token& k, int which, int b, int h, int t,
                                        int elem) {
  if (!kPages || which == 0)
    return static_cast<char*>(a.y[which]) + (((int64_t)b * a.heads[which] + h) * a.tokens + t) * a.d * elem;
  if (k.slot < 0) return nullptr;
  return static_cast<char*>(which == 1 ? a.c.keys : a.c.values) + (k.slot + ((int64_t)h * a.d << a.c.page_shift)) * elem;
}

template <class Ty>
struct Piece {
  static constexpr int kV = 16 / (int)sizeof(typename Ty::Raw);
  typename Ty::Raw e[kV];
};

// kNorm, kPages as the launch asks; kAhead heads are asked for at a time; 2^log_lanes lanes hold a head, the first d / (2 kV) of them.
template <class Ty, bool kInterleaved, bool kNorm, bool kPages, int kAhead>
__global__ __launch_bounds__(256) void norm_rotary_kernel(NormRotaryLaunch a, int log_lanes, int per) {
  typedef typename Ty::Raw Raw;
  constexpr int kV = Piece<Ty>::kV;
  const int lanes = a.d / (2 * kV);
  const int64_t id = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> log_lanes;
  const int u = threadIdx.x & ((1 << log_lanes) - 1);
  // (Lanes without a piece or a token take part in the exchanges, on element 0 of the last token.)
  const bool live = u < lanes && id < (int64_t)a.batch * a.tokens;
  const int64_t tok = min(id, (int64_t)a.batch * a.tokens - 1);
  const int b = (int)(tok / a.tokens), t = (int)(tok - (int64_t)b * a.tokens);

  const int half = a.form.half, turning = half / kV;  // (kInterleaved: not used)
  const bool first_turns = live && (kInterleaved ? u * kV < 2 * half : u < turning);
  const bool second_turns = live && (kInterleaved ? (u + lanes) * kV < 2 * half : u < turning);
  int first, second;  // the lane's elements
  if constexpr (kInterleaved) {
    first = u * kV;
    second = (u + lanes) * kV;
  } else if (u < turning) {
    first = u * kV;
    second = first + half;
  } else {
    first = (u + turning) * kV;
    second = (u + lanes) * kV;
  }
  if (!live) first = second = 0;

  const Token k = token_of<kPages>(a, b, t);
  float cs[kV], sn[kV];
  if (first_turns) {
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      int pair;
      if constexpr (kInterleaved)
        pair = ((i < kV / 2 ? first : second) >> 1) + i % (kV / 2);
      else
        pair = first + i;
      if (kInterleaved && i >= kV / 2 && !second_turns) continue;
      turn(k.pos, a.form.inv_freq[pair], cs[i], sn[i]);
      cs[i] *= a.form.factor;
      sn[i] *= a.form.factor;
    }
  }

  const int total = a.heads[0] + (kPages ? 2 : 1) * a.heads[1];
  const int h_begin = blockIdx.y * per, h_end = min(h_begin + per, total);
  float w[2][kV];
#pragma unroll
  for (int s = 0; s < (kPages ? 3 : 2); ++s) {  // q's heads of [h_begin, h_end), then k's, then v's
    const int before = s == 0 ? 0 : s == 1 ? a.heads[0] : a.heads[0] + a.heads[1];
    const int from = max(h_begin - before, 0), to = min(h_end - before, a.heads[s == 0 ? 0 : 1]);
    if (from >= to) continue;
    if (kNorm && s < 2) {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        w[0][i] = weight_of<Ty>(a.norm, s, first + i);
        w[1][i] = weight_of<Ty>(a.norm, s, second + i);
      }
    }
    const Raw* x = static_cast<const Raw*>(a.x[s]) + b * a.xs[s].b + t * a.xs[s].t;
    if (kPages && !k.has) {  // (a token's lanes go together)
      if (s == 0 && live) {
        for (int h = from; h < to; ++h) {
          Raw* y = reinterpret_cast<Raw*>(target<kPages>(a, k, s, b, h, t, (int)sizeof(Raw)));
          *reinterpret_cast<u32x4_e*>(y + first) = u32x4{0u, 0u, 0u, 0u};
          *reinterpret_cast<u32x4_e*>(y + second) = u32x4{0u, 0u, 0u, 0u};
        }
      }
      continue;
    }
    for (int h0 = from; h0 < to; h0 += kAhead) {
      // (Stores keep the compiler from asking for the next heads' pieces before this one's are written.)
      u32x4 piece[2 * kAhead];
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        if (h0 + z >= to) break;  // uniform
        const Raw* xh = x + (h0 + z) * a.xs[s].h;
        piece[2 * z] = *reinterpret_cast<const u32x4_e*>(xh + first);
        piece[2 * z + 1] = *reinterpret_cast<const u32x4_e*>(xh + second);
      }
#pragma unroll
      for (int z = 0; z < kAhead; ++z) {
        const int h = h0 + z;
        if (h >= to) break;  // uniform
        Piece<Ty> p = __builtin_bit_cast(Piece<Ty>, piece[2 * z]), q = __builtin_bit_cast(Piece<Ty>, piece[2 * z + 1]);
        if (s < 2) {
          float f[kV], g[kV];
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            f[i] = Ty::to_f(p.e[i]);
            g[i] = Ty::to_f(q.e[i]);
          }
          if constexpr (kNorm) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kV; ++i) sum = fmaf(f[i], f[i], fmaf(g[i], g[i], sum));
            sum = live ? sum : 0.f;
            for (int m = 1 << log_lanes >> 1; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
            const float r = 1.f / sqrtf(sum / (float)a.d + a.norm.eps);
#pragma unroll
            for (int i = 0; i < kV; ++i) {
              f[i] = f[i] * r * w[0][i];
              g[i] = g[i] * r * w[1][i];
            }
          }
          if constexpr (kInterleaved) {
            if (first_turns) {
#pragma unroll
              for (int i = 0; i < kV / 2; ++i) {
                const float c = f[2 * i], d = f[2 * i + 1];
                f[2 * i] = turned_x(c, d, cs[i], sn[i]);
                f[2 * i + 1] = turned_y(c, d, cs[i], sn[i]);
              }
            }
            if (second_turns) {
#pragma unroll
              for (int i = 0; i < kV / 2; ++i) {
                const float c = g[2 * i], d = g[2 * i + 1];
                g[2 * i] = turned_x(c, d, cs[kV / 2 + i], sn[kV / 2 + i]);
                g[2 * i + 1] = turned_y(c, d, cs[kV / 2 + i], sn[kV / 2 + i]);
              }
            }
          } else if (first_turns) {
#pragma unroll
            for (int i = 0; i < kV; ++i) {
              const float c = f[i], d = g[i];
              f[i] = turned_x(c, d, cs[i], sn[i]);
              g[i] = turned_y(c, d, cs[i], sn[i]);
            }
          }
          if (kNorm || first_turns) {
#pragma unroll
            for (int i = 0; i < kV; ++i) p.e[i] = Ty::cvt(f[i]);
          }
          if (kNorm || second_turns) {
#pragma unroll
            for (int i = 0; i < kV; ++i) q.e[i] = Ty::cvt(g[i]);
          }
        }
        Raw* y = reinterpret_cast<Raw*>(target<kPages>(a, k, s, b, h, t, (int)sizeof(Raw)));
        if (live && y != nullptr) {
          *reinterpret_cast<u32x4_e*>(y + first) = __builtin_bit_cast(u32x4, p);
          *reinterpret_cast<u32x4_e*>(y + second) = __builtin_bit_cast(u32x4, q);
        }
      }
    }
  }
}

// Heads that are no whole number of 16-byte pieces, or whose rotary part is none: a wave per head, element by
// element, read twice, with angles of its own. Simple, and far from what the bytes would take: 8 x 8191 tokens, 32/8 heads,
// bf16, D 16 of which 8 turn 1274 us (39 where all turn), 4 x 4096 tokens, D 96 of which 24 turn 362 (49 at a copy's rate).
template <class Ty, bool kPages>
__global__ __launch_bounds__(256) void norm_rotary_any_kernel(NormRotaryLaunch a, int64_t n, int total) {
  typedef typename Ty::Raw Raw;
  const int lane = threadIdx.x & 63;
  for (int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); id < n; id += (int64_t)gridDim.x * 4) {
    const int64_t tok = id / total;
    int h = (int)(id - tok * total);
    const int b = (int)(tok / a.tokens), t = (int)(tok - (int64_t)b * a.tokens);
    const int s = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
    h -= s == 0 ? 0 : s == 1 ? a.heads[0] : a.heads[0] + a.heads[1];
    const Token k = token_of<kPages>(a, b, t);
    const Raw* x = static_cast<const Raw*>(a.x[s]) + b * a.xs[s].b + t * a.xs[s].t + h * a.xs[s].h;
    Raw* y = reinterpret_cast<Raw*>(target<kPages>(a, k, s, b, h, t, (int)sizeof(Raw)));
    if (y == nullptr) continue;
    if (s == 2 || (kPages && s == 0 && !k.has)) {
      for (int i = lane; i < a.d; i += 64) y[i] = s == 2 ? x[i] : Raw{};
      continue;
    }
    const bool norm = a.norm.weight[s] != nullptr;
    float r = 1.f;
    if (norm) {
      float sum = 0.f;
      for (int i = lane; i < a.d; i += 64) sum = fmaf(Ty::to_f(x[i]), Ty::to_f(x[i]), sum);
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
      r = 1.f / sqrtf(sum / (float)a.d + a.norm.eps);
    }
    auto value = [&](int i) {
      const float f = Ty::to_f(x[i]);
      return norm ? f * r * weight_of<Ty>(a.norm, s, i) : f;
    };
    const int half = a.form.half;
    for (int i = lane; i < half; i += 64) {
      const int i0 = a.form.interleaved ? 2 * i : i, i1 = a.form.interleaved ? 2 * i + 1 : i + half;
      float cs, sn;
      turn(k.pos, a.form.inv_freq[i], cs, sn);
      cs *= a.form.factor;
      sn *= a.form.factor;
      const float c = value(i0), d = value(i1);
      y[i0] = Ty::cvt(turned_x(c, d, cs, sn));
      y[i1] = Ty::cvt(turned_y(c, d, cs, sn));
    }
    for (int i = 2 * half + lane; i < a.d; i += 64) y[i] = norm ? Ty::cvt(value(i)) : x[i];
  }
}

template <class Ty, bool kPages, bool kNorm, bool kInterleaved>
hipError_t pieces(const NormRotaryLaunch& p, hipStream_t stream) {
  constexpr int kV = Piece<Ty>::kV;
  const int lanes = p.d / (2 * kV), total = p.heads[0] + (kPages ? 2 : 1) * p.heads[1];
  int log_lanes = 0;
  while (1 << log_lanes < lanes) ++log_lanes;
  const int64_t blocks = (((int64_t)p.batch * p.tokens << log_lanes) + 255) / 256;
  int64_t parts = (2048 + blocks - 1) / blocks;  // head parts: about 2048 workgroups
  if (parts > total) parts = total;
  const int per = (int)((total + parts - 1) / parts);
  const dim3 grid((unsigned)blocks, (unsigned)((total + per - 1) / per));
  if (per >= 4)
    norm_rotary_kernel<Ty, kInterleaved, kNorm, kPages, 4><<<grid, 256, 0, stream>>>(p, log_lanes, per);
  else  // (a call of few tokens)
    norm_rotary_kernel<Ty, kInterleaved, kNorm, kPages, 1><<<grid, 256, 0, stream>>>(p, log_lanes, per);
  return hipGetLastError();
}

template <class Ty, bool kPages>
hipError_t norm_rotary(const NormRotaryLaunch& p, hipStream_t stream) {
  constexpr int kV = Piece<Ty>::kV;
  const int total = p.heads[0] + (kPages ? 2 : 1) * p.heads[1];
  const int64_t n = (int64_t)p.batch * p.tokens * total;
  if (n == 0) return hipSuccess;
  // Two pieces a lane, at most 64 lanes, and a rotary part of whole pieces (half layout: each half).
  const int part = p.form.interleaved ? 2 * p.form.half : p.form.half;
  if (p.d % (2 * kV) != 0 || p.d > 128 * kV || part % kV != 0) {
    norm_rotary_any_kernel<Ty, kPages><<<(unsigned)(n < 4 << 20 ? (n + 3) / 4 : 1 << 20), 256, 0, stream>>>(p, n, total);
    return hipGetLastError();
  }
  const bool norm = p.norm.weight[0] != nullptr || p.norm.weight[1] != nullptr;
  if (p.form.interleaved) {
    if (norm) return pieces<Ty, kPages, true, true>(p, stream);
    if constexpr (kPages) return pieces<Ty, kPages, false, true>(p, stream);
  } else {
    if (norm) return pieces<Ty, kPages, true, false>(p, stream);
    if constexpr (kPages) return pieces<Ty, kPages, false, false>(p, stream);
  }
  return hipErrorInvalidValue;  // (a call outside a cache always norms)
}

}  // namespace

hipError_t launch_norm_rotary(int dtype, const NormRotaryLaunch& p, hipStream_t stream) {
  if (dtype == kF16) return norm_rotary<HalfT, false>(p, stream);
  if (dtype == kBF16) return norm_rotary<Bf16T, false>(p, stream);
  return norm_rotary<FloatT, false>(p, stream);
}

hipError_t launch_pt_append(int dtype, const NormRotaryLaunch& p, hipStream_t stream) {
  return dtype == kF16 ? norm_rotary<HalfT, true>(p, stream) : norm_rotary<Bf16T, true>(p, stream);
}

}  // namespace pgr
