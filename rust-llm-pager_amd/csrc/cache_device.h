// Device-side pieces shared by the rotary and bounded-cache kernels.
#pragma once

#include <hip/hip_runtime.h>

#include "cache_kernels.h"

namespace pgr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Operands are only as aligned as their elements (a caller's view may start anywhere).
typedef uint32_t u32x4_e __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr float kMinusInf = -__builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

// Weights w in [0, 1] of a product with V, which the matrix cores take as numbers of the K/V type, go in as two
// of them, so that what a rounding to one would lose is kept: hi, w lowered by half a step u and cut off, and
// lo, the rest w - hi (exact in float32, at most 3 u w), rounded: hi + lo is within 3 u^2 w of w (2^-14.4 w in
// bf16, 2^-20.4 w in fp16). Lowered first, so that neither part of a weight is 0: 0 times an infinite V is NaN.
// Both are 1 / kUnit times the weight's, which keeps lo above fp16's smallest number down to weights of 2^-39;
// the caller takes the sum of the products times kUnit.

struct HalfT {
  typedef uint16_t Raw;
  static __device__ __forceinline__ float to_f(Raw x) { return (float)__builtin_bit_cast(_Float16, x); }
  static __device__ __forceinline__ Raw cvt(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const f16x2 h = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, h);
  }
  static constexpr float kUnit = 0x1p-14f;
  static constexpr float kSlack = 1.f;  // log2 of what split's weights may be above 1
  static __device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    constexpr float kLower = (1.f - 0x1p-11f) / kUnit;
    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x * kLower, y * kLower));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = pack(fmaf(x, 1.f / kUnit, -(float)h.x), fmaf(y, 1.f / kUnit, -(float)h.y));
  }
  static __device__ __forceinline__ f32x4 mma16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0,
                                                 0);
  }
  static __device__ __forceinline__ f32x4 mma16x32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
};

struct Bf16T {
  typedef uint16_t Raw;
  static __device__ __forceinline__ float to_f(Raw x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
  static __device__ __forceinline__ Raw cvt(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const bf16x2 h = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, h);
  }
  static constexpr float kUnit = 1.f;
  static constexpr float kSlack = 8.f;
  static __device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
    constexpr float kLower = 1.f - 0x1p-8f;
    const uint32_t a = __builtin_bit_cast(uint32_t, x * kLower), b = __builtin_bit_cast(uint32_t, y * kLower);
    hi = __builtin_amdgcn_perm(b, a, 0x07060302u);
    lo = pack(x - __builtin_bit_cast(float, a & 0xffff0000u), y - __builtin_bit_cast(float, b & 0xffff0000u));
  }
  static __device__ __forceinline__ f32x4 mma16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c, 0,
                                                     0, 0);
  }
  static __device__ __forceinline__ f32x4 mma16x32(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  static __device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
};

struct FloatT {
  typedef float Raw;
  static __device__ __forceinline__ float to_f(Raw x) { return x; }
  static __device__ __forceinline__ Raw cvt(float x) { return x; }
};

__device__ __forceinline__ int64_t load_position(const void* p, int is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

// cos and sin of position * inv_freq. The angle is taken in 64 bits and reduced to a part of one
// turn there: in 32 bits its error at position 2^17 would be 2^-7 rad, as large as the rotation
// between neighbouring positions of the slower pairs. From the reduced turn on 32 bits suffice.
// (No contraction: every kernel that inlines this gets the same bits.)
__device__ __forceinline__ void turn(int64_t position, float inv_freq, float& cs, float& sn) {
#pragma clang fp contract(off)
  const double turns = (double)position * (double)inv_freq * 0.15915494309189535;  // 1 / (2 pi)
  const float part = (float)(turns - __builtin_rint(turns));
  sincospif(2.f * part, &sn, &cs);
}

// Registers loaded before a loop, complete here: otherwise the compiler, which counts outstanding loads
// in their order, waits in the loop for whatever was asked for after them.
template <int N>
__device__ __forceinline__ void arrived(u32x4 (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(r[i]));
}

// A tile of 32 tokens as the attention kernels hold it in registers: lane (g, n) has pieces 8g.. of K rows n and
// 16 + n, and elements (D/16) n.. of V rows 4g + i and 16 + 4g + i.
template <int D>
struct KVTile {
  static constexpr int KP = D >= 32 ? D / 32 : 1;  // 16-byte pieces of a K row (D 16: one of 8 bytes)
  static constexpr int VD = D >= 32 ? D / 32 : 1;  // dwords of each V row (D 16: half of one)
  u32x4 k[2][KP];
  uint32_t v[2][4][VD];
};

typedef uint32_t u32x2_e __attribute__((ext_vector_type(2), aligned(2)));

// The lane's pieces of a K row (or of a query).
template <int D>
__device__ __forceinline__ void load_pieces(u32x4 (&r)[KVTile<D>::KP], const uint16_t* row, int g) {
  if constexpr (D == 16) {
    const u32x2 x = *reinterpret_cast<const u32x2_e*>(row + 4 * g);
    r[0] = u32x4{x.x, x.y, 0u, 0u};
  } else {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) r[c] = *reinterpret_cast<const u32x4_e*>(row + 32 * c + 8 * g);
  }
}

// Elements (D/16) n.. of a V row.
template <int D>
__device__ __forceinline__ void load_v(uint32_t (&r)[KVTile<D>::VD], const uint16_t* row, int n) {
  const uint16_t* p = row + (D / 16) * n;
  if constexpr (D == 16) {
    r[0] = *p;
  } else if constexpr (D == 32) {
    typedef uint32_t u32_e __attribute__((aligned(2)));
    r[0] = *reinterpret_cast<const u32_e*>(p);
  } else if constexpr (D == 64) {
    const u32x2 x = *reinterpret_cast<const u32x2_e*>(p);
    r[0] = x.x;
    r[1] = x.y;
  } else {
#pragma unroll
    for (int c = 0; c < D / 128; ++c) {
      const u32x4 x = *reinterpret_cast<const u32x4_e*>(p + 8 * c);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[4 * c + i] = x[i];
    }
  }
}

// Max and sum over the four lane groups g.
__device__ __forceinline__ float max_g(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_g(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Scores in log2 units: scale_log2 = scale * log2(e), or with a softcap cap * log2(e).
struct AttendScale {
  float scale_log2, cap_scale, cap_log2;
};

// The pair (x, y) turned, as fused multiply-adds with a float32 result of their own (the empty
// statement keeps the conversion to fp16 from being fused into them, which rounds once instead of
// twice): every kernel gets the same bits.
__device__ __forceinline__ float turned_x(float x, float y, float cs, float sn) {
  float r = fmaf(x, cs, -(y * sn));
  asm("" : "+v"(r));
  return r;
}
__device__ __forceinline__ float turned_y(float x, float y, float cs, float sn) {
  float r = fmaf(y, cs, x * sn);
  asm("" : "+v"(r));
  return r;
}

}  // namespace
}  // namespace pgr
