// The cache of pages: attention of a row's new tokens (one, a tree of drafts, a prompt's chunk) over the pages
// its table names, the move of accepted drafts to the front, and the masks of a tree.
//
// Lengths, counts, tables, masks and paths are read on the device. A page index outside the pool stands for
// a page that is not there: its tokens are not seen. So no value in them can lead an access astray.
#include <hip/hip_runtime.h>

#include "cache_device.h"
#include "page_table_kernels.h"

namespace pgr {
namespace {

constexpr int kTile = 32;  // tokens of a wave's tile: whole halves of 16, each in one page

// What a block of rows (row = new token * n_rep + query head) reads: tokens [begin, end), begin on a tile's
// border; and the tokens of its batch row.
struct Span {
  int length, n;   // tokens held, new tokens (those that the table has room for)
  int first, begin, end;  // the first token that some row sees; the first tile; behind the last token
};

__device__ __forceinline__ Span span_of(const PTAttendLaunch& a, int b, int r0, int rows, int n_rep) {
  Span s;
  const int capacity = a.r.width << a.c.page_shift;
  s.length = min(max(a.r.lengths[b], 0), capacity);
  s.n = min(a.r.counts != nullptr ? min(max(a.r.counts[b], 0), a.r.tokens) : a.r.tokens, capacity - s.length);
  const int t0 = r0 / n_rep, t1 = min((r0 + rows - 1) / n_rep, s.n - 1);
  s.first = s.begin = s.end = 0;
  if (t0 >= s.n) return s;
  s.end = a.masks != nullptr ? s.length + s.n : s.length + t1 + 1;
  if (a.window > 0) {
    s.first = max(s.length + (a.masks != nullptr ? 0 : t0) - a.window + 1, 0);
    s.begin = s.first & ~(kTile - 1);
  }
  return s;
}

// Tiles that a split takes of a block's: evenly, a tile for each wave at least.
__device__ __forceinline__ int tiles_per_split(const Span& s, int n_split, int waves) {
  const int tiles = (s.end - s.begin + kTile - 1) / kTile;
  return max((tiles + n_split - 1) / n_split, waves);
}

// Which tokens a row sees.
struct Row {
  int lo;         // first held token (and, in order, first new one)
  int t;          // its own number among the new ones
  uint64_t mask;  // with a tree: the new ones it sees
};

__device__ __forceinline__ Row row_of(const PTAttendLaunch& a, const Span& s, int b, int t) {
  Row r;
  r.t = t;
  r.mask = 0;
  int depth = t;
  const int at = max(min(t, s.n - 1), 0);
  if (a.masks != nullptr) {
    const int64_t row = (int64_t)b * a.r.tokens;
    r.mask = a.masks[row + at];
    if (s.n < 64) r.mask &= (1ull << s.n) - 1;
    depth = min(max(a.depths[row + at], 0), kMostDrafts - 1);
    if (a.window > 0)
      for (int j = 0; j < s.n; ++j)
        if (min(max(a.depths[row + j], 0), kMostDrafts - 1) <= depth - a.window) r.mask &= ~(1ull << j);
  }
  r.lo = a.window > 0 ? s.length + depth - a.window + 1 : 0;
  return r;
}

// (Without branches: selects of a few comparisons.)
__device__ __forceinline__ bool sees(const PTAttendLaunch& a, const Span& s, const Row& r, int c) {
  const int j = c - s.length;
  const bool bit = (r.mask >> (j & 63)) & 1, since = c >= r.lo;
  const bool fresh = a.masks != nullptr ? bit & (j < s.n) : (j <= r.t) & since;
  return j < 0 ? since : fresh;
}

// The block, split, KV head and batch row of a workgroup. Blocks that read the same tokens are neighbours on one
// XCD (workgroups go to the eight XCDs in turn), so that its L2 serves all but the first.
struct Work {
  int block, split, h, b;
};
__device__ __forceinline__ bool work_of(const PTAttendLaunch& a, Work& w) {
  const unsigned id = blockIdx.x, rest = id >> 3;
  const unsigned p = rest / a.plan.blocks * 8 + (id & 7);
  w.block = a.plan.blocks - 1 - (int)(rest % a.plan.blocks);  // the longest first
  if (p >= (unsigned)(a.r.batch * a.c.hkv * a.plan.n_split)) return false;
  w.split = (int)(p % a.plan.n_split);
  const unsigned bh = p / a.plan.n_split;
  w.h = (int)(bh % a.c.hkv);
  w.b = (int)(bh / a.c.hkv);
  return true;
}

// ---------------------------------------------------------------------------------------
// Attention of few rows a KV head. As in the bounded cache's attention each wave folds tiles of 32 tokens,
// two halves of 16, on v_mfma_f32_16x16x32,
//     S^T[16 tok x 16 rows] = K . Q^T,   O^T[D x 16 rows] += V^T[D x 32 tok] . P^T[32 tok x 16 rows],
// here for kG groups of 16 rows, which share a tile's K and its transposed V. The waves take tiles in turn and
// are joined at the end. A half lies in one page (pages are multiples of 16 tokens), whose index is one
// scalar load, two tiles ahead. P goes into the product with V as two numbers of the cache's type: rounded to
// one, the output's error is several times what its other roundings explain where sums all but cancel.
template <class Ty, int D, int kG, int kW>
__global__ __launch_bounds__(64 * kW) void pt_attend_kernel(PTAttendLaunch a, AttendScale sc) {
  typedef KVTile<D> T;
  constexpr int kThreads = 64 * kW, kRows = 16 * kG;
  __shared__ float sm_m[kW][kRows], sm_l[kW][kRows];
  __shared__ float sm_acc[kW][kRows][D + 1];
  Work wk;
  if (!work_of(a, wk)) return;
  const PTPages& c = a.c;
  const int b = wk.b, h = wk.h, n_rep = c.hq / c.hkv, r0 = wk.block * kRows;
  const Span sp = span_of(a, b, r0, kRows, n_rep);
  const int per = tiles_per_split(sp, a.plan.n_split, kW);
  const int begin = min(sp.begin + wk.split * per * kTile, sp.end), end = min(begin + per * kTile, sp.end);
  // (The merge reads only the splits that hold tokens; a block that is finished here writes its zeros.)
  if (a.plan.n_split > 1 && begin >= end) return;
  const int tiles = (end - begin + kTile - 1) / kTile;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int32_t* table = a.r.table + b * a.r.table_stride;
  const int in_page = (1 << c.page_shift) - 1;
  const uint16_t* kp = static_cast<const uint16_t*>(c.keys) + ((int64_t)h * D << c.page_shift);
  const uint16_t* vp = static_cast<const uint16_t*>(c.values) + ((int64_t)h * D << c.page_shift);

  // A tile's pages; halves past the end read its last one.
  struct Places {
    int32_t page[2];
  };
  auto places = [&](int ti) {
    Places p;
#pragma unroll
    for (int x = 0; x < 2; ++x) p.page[x] = table[min(begin + ti * kTile + 16 * x, end - 1) >> c.page_shift];
    return p;
  };
  auto there = [&](int32_t page) { return page >= 0 && page < c.pages; };
  // Element offset of a half's first token. A page that is not there is read at page 0 and masked.
  auto place = [&](const Places& p, int ti, int x) {
    const int t = min(begin + ti * kTile + 16 * x, (end - 1) & ~15);
    return (((int64_t)(there(p.page[x]) ? p.page[x] : 0) * c.hkv << c.page_shift) + (t & in_page)) * D;
  };
  T t;
  auto fetch_k = [&](const Places& p, int ti) {
#pragma unroll
    for (int x = 0; x < 2; ++x) load_pieces<D>(t.k[x], kp + place(p, ti, x) + n * D, g);
  };
  auto fetch_v = [&](const Places& p, int ti) {
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < 4; ++i) load_v<D>(t.v[x][i], vp + place(p, ti, x) + (4 * g + i) * D, n);
  };

  Row row[kG];
  u32x4 q[kG][T::KP];
  int lo_most = 0;
#pragma unroll
  for (int y = 0; y < kG; ++y) {
    const int r = r0 + 16 * y + n, tok = r / n_rep, e = r - tok * n_rep;
    row[y] = row_of(a, sp, b, tok);
    lo_most = max(lo_most, row[y].lo);
#pragma unroll
    for (int i = 0; i < T::KP; ++i) q[y][i] = u32x4{0u, 0u, 0u, 0u};
    if (tok < sp.n)
      load_pieces<D>(q[y], static_cast<const uint16_t*>(a.q) + b * a.qs.b + ((int64_t)h * n_rep + e) * a.qs.h +
                               tok * a.qs.t, g);
  }
  Places now{}, next{};
  if (wave < tiles) {
    now = places(wave);
    fetch_k(now, wave);
    fetch_v(now, wave);
    next = places(min(wave + kW, tiles - 1));
  }
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) lo_most = max(lo_most, __shfl_xor(lo_most, m));
  lo_most = __builtin_amdgcn_readfirstlane(lo_most);
#pragma unroll
  for (int y = 0; y < kG; ++y) arrived(q[y]);

  float m_run[kG], l_run[kG];
  f32x4 acc[kG][D / 16];
#pragma unroll
  for (int y = 0; y < kG; ++y) {
    m_run[y] = kMinusInf;
    l_run[y] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) acc[y][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto scores = [&](f32x4 (&s)[kG][2]) {
#pragma unroll
    for (int y = 0; y < kG; ++y)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        s[y][x] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (D == 16) {
          s[y][x] = Ty::mma16(u32x2{t.k[x][0].x, t.k[x][0].y}, u32x2{q[y][0].x, q[y][0].y}, s[y][x]);
        } else {
#pragma unroll
          for (int i = 0; i < T::KP; ++i) s[y][x] = Ty::mma16x32(t.k[x][i], q[y][i], s[y][x]);
        }
      }
  };
  auto fold = [&](f32x4 (&s)[kG][2], int ti, const Places& at) {
    const int c0 = begin + ti * kTile;
    // Uniform: some row may not see some token of the tile.
    const bool masked = c0 < lo_most || c0 + kTile > min(sp.length, end) || !there(at.page[0]) || !there(at.page[1]);
    if (masked) {  // values that no row sees may be anything: NaN times a weight of 0 is NaN
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = c0 + 16 * x + 4 * g + i;
          if (tok >= sp.first && tok < end && there(at.page[x])) continue;
#pragma unroll
          for (int j = 0; j < T::VD; ++j) t.v[x][i][j] = 0u;
        }
    }
    u32x4 hi[kG], lo[kG];
#pragma unroll
    for (int y = 0; y < kG; ++y) {
      float p[8], top = kMinusInf;
      if (sc.cap_log2 > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = sc.cap_log2 * tanhf(s[y][i / 4][i & 3] * sc.cap_scale);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = s[y][i / 4][i & 3] * sc.scale_log2;
      }
      if (masked) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int tok = c0 + 16 * (i / 4) + 4 * g + (i & 3);
          const bool seen = (tok < end) & there(at.page[i / 4]) & sees(a, sp, row[y], tok);
          p[i] = seen ? p[i] : kMinusInf;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, p[i]);
      const float m_new = fmaxf(m_run[y], max_g(top));
      const float ref = m_new == kMinusInf ? 0.f : m_new;  // (scores of -inf weigh nothing, those of NaN stay NaN)
      if (__any(m_new > m_run[y])) {  // (otherwise the factor is 1)
        const float alpha = __builtin_amdgcn_exp2f(m_run[y] - ref);
        l_run[y] *= alpha;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc[y][j] *= alpha;
        m_run[y] = m_new;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(p[i] - ref);
      l_run[y] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t u, v;
        Ty::split(p[2 * i], p[2 * i + 1], u, v);
        hi[y][i] = u;
        lo[y][i] = v;
      }
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
#pragma unroll
      for (int y = 0; y < kG; ++y) {
        acc[y][j] = Ty::mma16x32(vt, lo[y], acc[y][j]);
        acc[y][j] = Ty::mma16x32(vt, hi[y], acc[y][j]);
      }
    }
  };
  int ti = wave;
  for (; ti + kW < tiles; ti += kW) {
    const Places then = places(min(ti + 2 * kW, tiles - 1));
    f32x4 s[kG][2];
    scores(s);
    fetch_k(next, ti + kW);
    fold(s, ti, now);
    fetch_v(next, ti + kW);
    now = next;
    next = then;
  }
  if (ti < tiles) {
    f32x4 s[kG][2];
    scores(s);
    fold(s, ti, now);
  }

#pragma unroll
  for (int y = 0; y < kG; ++y) {
    const float l_wave = sum_g(l_run[y]);
    if (g == 0) {
      sm_m[wave][16 * y + n] = m_run[y];
      sm_l[wave][16 * y + n] = l_wave;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sm_acc[wave][16 * y + n][(D / 4) * g + (D / 16) * i + j] = acc[y][j][i] * Ty::kUnit;
  }
  __syncthreads();
  const int64_t part = ((((int64_t)b * c.hkv + h) * a.plan.blocks + wk.block) * a.plan.n_split + wk.split) * kRows;
  for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
    const int r = i / D, e = i - r * D, tok = (r0 + r) / n_rep;
    if (tok >= a.r.tokens) break;
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
    if (a.plan.n_split == 1) {
      const int64_t head = ((int64_t)b * a.r.tokens + tok) * c.hq + h * n_rep + (r0 + r - tok * n_rep);
      static_cast<uint16_t*>(a.out)[head * D + e] = Ty::cvt(tok >= sp.n || l == 0.f ? 0.f : x / l);
    } else {
      a.pacc[part * D + i] = x;
      if (e == 0) {
        a.pm[part + r] = m;
        a.pl[part + r] = l;
      }
    }
  }
}

// Joins the splits: groups of d / 4 threads take a row each.
template <class Ty>
__global__ __launch_bounds__(256) void pt_merge_kernel(PTAttendLaunch a, int waves) {
  const PTPages& c = a.c;
  const int d = c.d, n_rep = c.hq / c.hkv, cols = d / 4, b = blockIdx.z, h = blockIdx.y;
  const int r = blockIdx.x * (256 / cols) + threadIdx.x / cols, e = threadIdx.x % cols * 4;
  const int tok = r / n_rep;
  if (tok >= a.r.tokens) return;
  const int block = r / a.plan.rows, in = r - block * a.plan.rows;
  const Span sp = span_of(a, b, block * a.plan.rows, a.plan.rows, n_rep);
  const int tiles = (sp.end - sp.begin + kTile - 1) / kTile, per = tiles_per_split(sp, a.plan.n_split, waves);
  const int used = (tiles + per - 1) / per;
  const int64_t part = (((int64_t)b * c.hkv + h) * a.plan.blocks + block) * a.plan.n_split * a.plan.rows + in;
  float m = kMinusInf, l = 0.f;
  for (int s = 0; s < used; ++s) m = fmaxf(m, a.pm[part + (int64_t)s * a.plan.rows]);
  const float ref = m == kMinusInf ? 0.f : m;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < used; ++s) {
    const int64_t at = part + (int64_t)s * a.plan.rows;
    const float f = __builtin_amdgcn_exp2f(a.pm[at] - ref);
    l += a.pl[at] * f;
    x += *reinterpret_cast<const f32x4*>(a.pacc + at * d + e) * f;
  }
  const bool none = tok >= sp.n || l == 0.f;
  uint16_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = Ty::cvt(none ? 0.f : x[i] / l);
  const int64_t head = ((int64_t)b * a.r.tokens + tok) * c.hq + h * n_rep + (r - tok * n_rep);
  *reinterpret_cast<u32x2_e*>(static_cast<uint16_t*>(a.out) + head * d + e) =
      u32x2{(uint32_t)y[0] | (uint32_t)y[1] << 16, (uint32_t)y[2] | (uint32_t)y[3] << 16};
}

// ---------------------------------------------------------------------------------------
// The accepted path to the front: token length + j of each row becomes token length + path[j], as all were
// before the call. A workgroup moves the keys (z even) or the values of one layer, row and KV head, in
// 16-byte pieces: all of them are read before the first is written. Entries outside [0, 64) move nothing, nor do
// those that are in their place. Memory-bound, in short pieces.
constexpr int kKeepMost = kMostDrafts * 32 / 256;  // pieces a thread: 64 tokens of up to 32 pieces

__global__ __launch_bounds__(256) void pt_keep_kernel(PTKeepLaunch a) {
  __shared__ int64_t from_s[kMostDrafts], to_s[kMostDrafts];
  const PTPages& c = a.c;
  const int h = blockIdx.x % c.hkv, b = blockIdx.x / c.hkv, tid = threadIdx.x, tokens = a.r.tokens;
  const int layer = blockIdx.y;
  auto cell = [&](int64_t token) {
    const int64_t page = token >> c.page_shift;
    if (page >= a.r.width) return (int64_t)-1;
    const int32_t p = a.r.table[b * a.r.table_stride + page];
    if (p < 0 || p >= c.pages) return (int64_t)-1;
    return (((int64_t)p * c.hkv + h << c.page_shift) + (token & (((int64_t)1 << c.page_shift) - 1))) * c.d;
  };
  bool moves = false;
  if (tid < tokens) {
    const int64_t length = max(a.r.lengths[b], 0);
    const int p = a.path[(int64_t)b * tokens + tid];
    int64_t from = -1, to = -1;
    if (p >= 0 && p < kMostDrafts && p != tid) {
      from = cell(length + p);
      to = cell(length + tid);
    }
    moves = from >= 0 && to >= 0;
    from_s[tid] = moves ? from : -1;
    to_s[tid] = to;
  }
  if (!__syncthreads_or(moves)) return;
  const int pieces = c.d / 8, n = tokens * pieces;
  uint16_t* const pool = static_cast<uint16_t*>(blockIdx.z == 0 ? c.keys : c.values) +
                         (((int64_t)layer * c.pages * c.hkv << c.page_shift) * c.d);
  u32x4 x[kKeepMost];
#pragma unroll
  for (int i = 0; i < kKeepMost; ++i) {
    const int at = tid + i * 256, j = at / pieces;
    x[i] = u32x4{0u, 0u, 0u, 0u};
    if (at < n && from_s[j] >= 0) x[i] = *reinterpret_cast<const u32x4*>(pool + from_s[j] + (at - j * pieces) * 8);
  }
  arrived(x);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kKeepMost; ++i) {
    const int at = tid + i * 256, j = at / pieces;
    if (at < n && from_s[j] >= 0) *reinterpret_cast<u32x4*>(pool + to_s[j] + (at - j * pieces) * 8) = x[i];
  }
}

// ---------------------------------------------------------------------------------------
// Each token's ancestors and itself as bits, and its depth. A wave per row, a token a lane: six steps of
// doubling, after each of which a lane knows twice as many ancestors. A parent that is not an earlier token
// makes a root.
__global__ __launch_bounds__(64) void draft_tree_kernel(const int32_t* parents, int tokens, uint64_t* masks,
                                                        int32_t* depths) {
  const int lane = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * tokens;
  int up = lane < tokens ? parents[row + lane] : -1;
  if (up < 0 || up >= lane) up = -1;
  uint32_t low = lane < 32 ? 1u << lane : 0u, high = lane >= 32 ? 1u << (lane - 32) : 0u;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const int at = up < 0 ? lane : up;
    const uint32_t l = __shfl(low, at), h = __shfl(high, at);
    const int u = __shfl(up, at);
    if (up >= 0) {
      low |= l;
      high |= h;
      up = u;
    }
  }
  if (lane < tokens) {
    masks[row + lane] = (uint64_t)high << 32 | low;
    depths[row + lane] = __popc(low) + __popc(high) - 1;
  }
}

template <class Ty, int D, int kG>
hipError_t attend_dim(const PTAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  const int64_t parts = (int64_t)p.r.batch * p.c.hkv * p.plan.n_split;
  const dim3 grid((unsigned)((parts + 7) / 8 * 8 * p.plan.blocks));
  pt_attend_kernel<Ty, D, kG, 4><<<grid, 256, 0, stream>>>(p, sc);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.plan.n_split == 1) return e;
  const int rows = p.r.tokens * (p.c.hq / p.c.hkv), each = 256 / (D / 4);
  const dim3 merge((unsigned)((rows + each - 1) / each), (unsigned)p.c.hkv, (unsigned)p.r.batch);
  pt_merge_kernel<Ty><<<merge, 256, 0, stream>>>(p, 4);
  return hipGetLastError();
}

template <class Ty, int D>
hipError_t attend_rows(const PTAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  if constexpr (D < 256)
    if (p.plan.rows == 32) return attend_dim<Ty, D, 2>(p, sc, stream);
  return attend_dim<Ty, D, 1>(p, sc, stream);
}

template <class Ty>
hipError_t attend(const PTAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  switch (p.c.d) {
    case 16: return attend_rows<Ty, 16>(p, sc, stream);
    case 32: return attend_rows<Ty, 32>(p, sc, stream);
    case 64: return attend_rows<Ty, 64>(p, sc, stream);
    case 128: return attend_rows<Ty, 128>(p, sc, stream);
    default: return attend_rows<Ty, 256>(p, sc, stream);
  }
}

}  // namespace

PTAttendPlan pt_attend_plan(int batch, int tokens, int hq, int hkv, int64_t capacity, int d) {
  PTAttendPlan p;
  const int rows = tokens * (hq / hkv);
  p.rows = rows > 16 && d < 256 ? 32 : 16;
  p.blocks = (rows + p.rows - 1) / p.rows;
  const int64_t groups = (int64_t)batch * hkv * p.blocks;
  const int64_t most = (capacity + 4 * kTile - 1) / (4 * kTile);  // a tile for each wave
  int64_t n = (1024 + groups - 1) / groups;
  if (n > most) n = most;
  p.n_split = n < 1 ? 1 : (int)n;
  return p;
}

hipError_t launch_pt_attend(int dtype, const PTAttendLaunch& p, hipStream_t stream) {
  AttendScale sc;
  sc.scale_log2 = p.scale * kLog2e;
  sc.cap_scale = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  sc.cap_log2 = p.softcap > 0.f ? p.softcap * kLog2e : 0.f;
  return dtype == kF16 ? attend<HalfT>(p, sc, stream) : attend<Bf16T>(p, sc, stream);
}

hipError_t launch_pt_keep(const PTKeepLaunch& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.r.batch * p.c.hkv), (unsigned)p.layers, 2);
  pt_keep_kernel<<<grid, 256, 0, stream>>>(p);
  return hipGetLastError();
}

hipError_t launch_draft_tree(const int32_t* parents, int batch, int tokens, uint64_t* masks, int32_t* depths,
                             hipStream_t stream) {
  draft_tree_kernel<<<(unsigned)batch, 64, 0, stream>>>(parents, tokens, masks, depths);
  return hipGetLastError();
}

}  // namespace pgr
