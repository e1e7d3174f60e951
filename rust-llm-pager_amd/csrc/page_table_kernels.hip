// The cache of pages: attention of a row's new tokens (one, a tree of drafts, a prompt's chunk) over the pages
// its table names, the move of accepted drafts to the front, and the masks of a tree.
//
// Lengths, counts, tables, masks and paths are read on the device. A page index outside the pool stands for
// a page that is not there: its tokens are not seen. So no value in them can lead an access astray.
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>

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

__device__ __forceinline__ int tiles_of(const PTAttendPlan& p, const Span& s) {
  return (s.end - s.begin + p.tile - 1) / p.tile;
}

// Tiles of the longest of a batch row's blocks, at least.
__device__ __forceinline__ int row_tiles(const PTAttendLaunch& a, int b) {
  const int capacity = a.r.width << a.c.page_shift;
  const int length = min(max(a.r.lengths[b], 0), capacity);
  const int n = min(a.r.counts != nullptr ? min(max(a.r.counts[b], 0), a.r.tokens) : a.r.tokens, capacity - length);
  // (A window begins up to kTile - 1 tokens early, on a tile's border.)
  const int held = a.window > 0 ? min(length, a.window + kTile - 1) : length;
  return n <= 0 ? 0 : (held + n + a.plan.tile - 1) / a.plan.tile;
}

// The wave's sums up to each lane, by lane shifts within rows of 16 and then across them.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

// A workgroup's work: a block of rows, a KV head, a batch row and which `per` tiles of the block's (whole: all of them).
struct Work {
  int block, h, b, split, per;
  bool whole;
};

// The batch's rows are cut into parts of one size, `per` tiles: the least with which there are no more parts than
// plan.slots, so that long rows have more of them and all workgroups about as much to do (8 rows of 13 drafted tokens
// over 0 to 8191, D 64, softcapped: 27 us, 36 with as many parts for a short row as for a long one). Every wave finds
// that size and its part by itself; the first workgroup leaves both for the merge. (In large batches a launch before this
// one has listed the parts.) A row of one part is finished by its workgroup; without slots every row is.
//
// Blocks that read the same tokens are neighbours on one XCD (workgroups go to the eight XCDs in turn), so that its L2
// serves all but the first; the longest block is first.
__device__ __forceinline__ bool work_of(const PTAttendLaunch& a, Work& w) {
  const unsigned id = blockIdx.x, rest = id >> 3, blocks = a.plan.blocks, hkv = a.c.hkv;
  const unsigned p = rest / blocks * 8 + (id & 7);
  w.block = (int)(blocks - 1 - rest % blocks);
  w.h = (int)(p % hkv);
  const int part = (int)(p / hkv);
  w.per = 0;
  w.split = 0;
  w.b = part;
  w.whole = true;
  if (a.plan.slots == 0) return part < a.r.batch;
  if (part >= a.plan.slots) return false;
  if (a.parts != nullptr) {
    const int2 listed = a.parts[part];
    if (listed.x < 0) return false;
    w.b = listed.x;
    w.split = listed.y;
    w.per = a.meta[w.b].y;
    w.whole = row_tiles(a, w.b) <= w.per;
    return true;
  }
  if (a.r.batch == 1) {
    w.per = max((row_tiles(a, 0) + a.plan.slots - 1) / a.plan.slots, a.plan.least);
    w.split = part;
    w.b = 0;
    w.whole = row_tiles(a, 0) <= w.per;
    if (w.whole && part > 0) return false;
    if (id == 0 && threadIdx.x == 0) a.meta[0] = int2{0, w.per};
    return true;
  }
  const int lane = threadIdx.x & 63, mine = lane < a.r.batch ? row_tiles(a, lane) : 0;
  int all = mine;
  for (int b = lane + 64; b < a.r.batch; b += 64) all += row_tiles(a, b);
  int per = max((__builtin_amdgcn_readlane(wave_scan(all), 63) + a.plan.slots - 1) / a.plan.slots, a.plan.least);
  // Parts of all rows at `size` tiles a part; upto: of the first 64 rows up to the lane's.
  int upto = 0;
  auto parts_at = [&](int size) {
    upto = wave_scan((mine + size - 1) / size);
    int parts = __builtin_amdgcn_readlane(upto, 63);
    for (int b0 = 64; b0 < a.r.batch; b0 += 64)
      parts += __builtin_amdgcn_readlane(wave_scan(b0 + lane < a.r.batch ? (row_tiles(a, b0 + lane) + size - 1) / size : 0), 63);
    return parts;
  };
  int parts = parts_at(per);
  if (parts > a.plan.slots) {
    int few = per;  // too small a size; then one that is not (there are as many slots as rows: one part each ends it)
#pragma unroll 1
    for (int i = 0; parts > a.plan.slots; ++i) {
      few = per;
      per = i < 8 ? max(per + 1, (int)min((int64_t)1 << 30, ((int64_t)per * parts + a.plan.slots - 1) / a.plan.slots)) : 1 << 30;
      parts = parts_at(per);
    }
#pragma unroll 1
    while (per - few > 1 + (per >> 6)) {  // within a 64th of the least
      const int size = (few + per) >> 1;
      if (parts_at(size) > a.plan.slots)
        few = size;
      else
        per = size;
    }
    parts_at(per);
  }
  w.per = per;
  w.b = -1;
  int before = 0;  // parts of the rows before b0
  for (int b0 = 0; b0 < a.r.batch; b0 += 64) {
    const int own = b0 == 0 ? (mine + per - 1) / per
                            : b0 + lane < a.r.batch ? (row_tiles(a, b0 + lane) + per - 1) / per : 0;
    const int last = before + (b0 == 0 ? upto : wave_scan(own));  // behind the lane's row
    if (id == 0 && threadIdx.x < 64 && b0 + lane < a.r.batch) a.meta[b0 + lane] = int2{last - own, per};
    const uint64_t later = __ballot(last > part);
    if (w.b < 0 && later != 0) {
      const int at = __builtin_ctzll(later);
      w.b = b0 + at;
      const int parts_of_row = __builtin_amdgcn_readlane(own, at);
      w.split = part - (__builtin_amdgcn_readlane(last, at) - parts_of_row);
      w.whole = parts_of_row == 1;
      if (id != 0) break;
    }
    before = __builtin_amdgcn_readlane(last, 63);
  }
  return w.b >= 0;
}

// The parts of a large batch, listed once: the size of a part as above, each row's first part and each part's row. One
// workgroup, a thread for so many rows that follow each other. Any size from total / (slots - batch) on leaves no more than
// `slots` parts, since a row has at most one that is not full; a dozen sums over the batch find the least. Latency alone.
constexpr int kListThreads = 1024;

__global__ __launch_bounds__(kListThreads) void pt_list_kernel(PTAttendLaunch a) {
  __shared__ int tiles_s[kMostListed];
  __shared__ int wave_s[kListThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, batch = a.r.batch, slots = a.plan.slots;
  const int each = (batch + kListThreads - 1) / kListThreads, first = min(tid * each, batch), last = min(first + each, batch);
  // Sum over the threads; `before`: over those before this one.
  auto sum = [&](int x, int& before) {
    const int upto = wave_scan(x);
    __syncthreads();
    if (lane == 63) wave_s[wave] = upto;
    __syncthreads();
    int all = 0;
    before = upto - x;
    for (int w = 0; w < kListThreads / 64; ++w) {
      before += w < wave ? wave_s[w] : 0;
      all += wave_s[w];
    }
    return all;
  };
  int mine = 0, before;
  for (int b = first; b < last; ++b) {
    tiles_s[b] = row_tiles(a, b);
    mine += tiles_s[b];
  }
  const int total = sum(mine, before);
  auto own_at = [&](int size) {
    int parts = 0;
    for (int b = first; b < last; ++b) parts += (tiles_s[b] + size - 1) / size;
    return parts;
  };
  int few = max((total + slots - 1) / slots, a.plan.least) - 1, per = max((total - 1) / (slots - batch) + 1, few + 1);
#pragma unroll 1
  while (per - few > 1 + (per >> 6)) {  // few: too small, or not tried; per: not too small
    const int size = (few + per) >> 1;
    if (sum(own_at(size), before) > slots)
      few = size;
    else
      per = size;
  }
  const int all = sum(own_at(per), before);
  for (int b = first; b < last; ++b) {
    const int n = (tiles_s[b] + per - 1) / per;
    a.meta[b] = int2{before, per};
    for (int i = 0; i < n; ++i) a.parts[before + i] = int2{b, i};
    before += n;
  }
  for (int i = all + tid; i < slots; i += kListThreads) a.parts[i] = int2{-1, 0};
}

// The first row of a part's results: [hkv, blocks, slots, rows], a batch row's parts one after the other.
__device__ __forceinline__ int64_t slot_of_part(const PTAttendLaunch& a, const Work& w, int rows) {
  const int part = (int)((blockIdx.x >> 3) / a.plan.blocks * 8 + (blockIdx.x & 7)) / a.c.hkv;
  return (((int64_t)w.h * a.plan.blocks + w.block) * a.plan.slots + part) * rows;
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
    depth = max(a.depths[row + at], 0);  // (none below 0: what a block reads begins a window before depth 0)
    if (a.window > 0)
      for (int j = 0; j < s.n; ++j)
        if (max(a.depths[row + j], 0) <= depth - a.window) r.mask &= ~(1ull << j);
  }
  // (64 bits, and cut off behind all tokens: a depth may be any number.)
  r.lo = a.window > 0 ? (int)min((int64_t)s.length + depth - a.window + 1, (int64_t)s.end) : 0;
  return r;
}

__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// Bit i: whether the row sees token first + i (of those before its block's end).
__device__ __forceinline__ uint64_t sees(const PTAttendLaunch& a, const Span& s, const Row& r, int first) {
  const int at = first - s.length;  // bit 0's number among the new tokens
  const uint64_t since = ~low_bits(r.lo - first);
  if (a.masks == nullptr) return low_bits(r.t + 1 - at) & since;
  const uint64_t fresh = at >= 64 || at <= -64 ? 0ull : at >= 0 ? r.mask >> at : r.mask << -at;
  return (low_bits(-at) & since) | fresh;
}

// Scores x to cap * log2(e) * tanh(y), y = x * scale / cap, by z = 2 log2(e) y (x * cap_scale here): 1 - 2 / (1 + 2^z), whose error
// is that of numbers about 1, and below kNear (y below 0.6) z times a polynomial in z^2, whose error goes by the score. The
// polynomial is fitted to an even relative error of 2^-23.5; with float32's roundings it is within 4 half steps of the
// score, the other within 5 of the score and 3 of the cap (a unit in the last place each for the exponential and the
// reciprocal counted in). Caps lie far above most scores, and where all of a wave's are near, the polynomial takes no
// longer than the exponential would: 13 drafted tokens over 8 x 8191, 32/4 heads, D 64, 37 us without a cap, 41 with the
// exponential alone, 43 so, and 50 under a cap of 5 that many scores pass; a chunk of 2048 tokens over 16384, 32/8,
// D 128, 830, 980, 984 and 1202.
constexpr float kNear = 1.73f;

__device__ __forceinline__ float capped_near(float z) {
  const float z2 = z * z;
  return z * fmaf(z2, fmaf(z2, fmaf(z2, fmaf(z2, 1.1262515e-06f, -3.135718e-05f), 0.000665667001f), -0.013875721f), 0.346573591f);
}

template <int N, class V>
__device__ __forceinline__ void capped(V& s, const AttendScale& sc) {
  float most = 0.f;
  float near[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] *= sc.cap_scale;
    near[i] = capped_near(s[i]);
    most = fmaxf(most, fabsf(s[i]));
  }
  if (__any(most >= kNear)) {  // (NaN is NaN either way)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[i])), 1.f);
      near[i] = fabsf(s[i]) >= kNear ? far : near[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = sc.cap_log2 * near[i];
}

// ---------------------------------------------------------------------------------------
// Attention of few rows a KV head. As in the bounded cache's attention each wave folds tiles of 32 tokens,
// two halves of 16, on v_mfma_f32_16x16x32,
//     S^T[16 tok x 16 rows] = K . Q^T,   O^T[D x 16 rows] += V^T[D x 32 tok] . P^T[32 tok x 16 rows],
// here for kG groups of 16 rows, which share a tile's K and its transposed V. The waves take tiles in turn and
// are joined at the end. A half lies in one page (pages are multiples of 16 tokens), whose index is one
// scalar load, two tiles ahead. P goes into the product with V as two numbers of the cache's type, which costs
// nothing beside the loads: rounded to one, the output's error is several times what its other roundings explain
// where sums all but cancel.
//
// Bound by HBM, and for a few rows by the two launches' latency. 8 rows x 8192 tokens, 32/8 heads, D 128, one token: 55 us
// for 268 MB (4.9 TB/s; a copy reaches 5.1), 8 drafted tokens 61; 2 x 65536 tokens: 102 us for 537 MB. Parts for 256
// workgroups against 512 / 1024: 54.6 / 54.9 / 56.7 us (one token), 61.9 / 65.0 / 72.9 (eight), one row of 28/4 heads
// 14.4 either way, 16 rows of 4096 tokens, D 64: 19.5 / 21.0 / 21.8. Short rows are finished by one workgroup of
// eight waves, without a merge: 256 tokens, D 64 6.7 us against 9.4, D 128 8.2 against 10.4; at 1000 and 500 tokens
// (D 64 and 128) the two are even.
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
  const bool whole = wk.whole;
  // (64 bits: a part's border may lie past any row.)
  const int begin = whole ? sp.begin : (int)min((int64_t)sp.end, sp.begin + (int64_t)wk.split * wk.per * kTile);
  const int end = whole ? sp.end : (int)min((int64_t)sp.end, begin + (int64_t)wk.per * kTile);
  // (The merge reads only the parts that hold tokens; a block that is finished here writes its zeros.)
  if (!whole && begin >= end) return;
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
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = s[y][i / 4][i & 3];
      if (sc.cap_log2 > 0.f) {
        capped<8>(p, sc);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] *= sc.scale_log2;
      }
      if (masked) {
        const uint32_t here = (there(at.page[0]) ? 0xffffu : 0u) | (there(at.page[1]) ? 0xffff0000u : 0u);
        const uint32_t seen = (uint32_t)sees(a, sp, row[y], c0 + 4 * g) & (uint32_t)low_bits(end - c0 - 4 * g) & here >> 4 * g;
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = seen >> (16 * (i / 4) + (i & 3)) & 1 ? p[i] : kMinusInf;
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
  const int64_t part = slot_of_part(a, wk, kRows);
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
    if (whole) {
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

// Max and sum over the lanes l and l + 32.
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// ---------------------------------------------------------------------------------------
// Attention of many rows a KV head (trees of several heads, a prompt's chunks): bound by arithmetic, so each wave
// holds 32 rows on v_mfma_f32_32x32x16 and all waves fold the same tile of kTok tokens, which passes through LDS
// once for all of them:
//     S^T[32 tok x 32 rows] = K . Q^T,   O^T[32 dims x 32 rows] += V^T[32 dims x 16 tok] . P^T[16 tok x 32 rows].
// Lane (h, n) = (l / 32, l % 32) holds tokens 8 (i / 4) + 4 h + i % 4, i < 16, of row n, which is the P^T operand as it
// stands; V^T comes from V's rows by the transposing LDS read, four tokens at a time. The 16-byte pieces of a row
// lie in LDS at their number XORed with bits of the row's, so that neither the 16 rows that an operand of K
// takes one piece of, nor the four rows of a transposing read, meet in one bank. The next tile's loads are under way
// in registers while this one is folded.
//
// kTwo: P as two numbers, as above, unless the caller has said that one will do (rounded to one number of the cache's type
// P is off by half a step of each weight: in bf16 the output is then 0.0023 of its norm from 64 bits, 0.0017 with two): here
// the second product is half as much arithmetic again. A chunk of 2048 tokens over 16384, 32/8 heads, D 128: 826 us with
// two numbers, 622 with one (939 TFLOP/s; a library's matrix product reaches 1244); the kernel above took 1265. Trees of
// 64 tokens over 8 rows of 32768, 28/4: 387 and 302 us (598). In the chunk the matrix cores are busy 0.50 of the cycles and
// the vector units 0.57 (0.42 and 0.52 with one number), one after the other: the two waves of a SIMD go through products
// and softmax together. With one number: half of the waves half a tile behind the others (676 us), a barrier every second
// tile (641), raised wave priorities over either product (637 to 653): no better. Eight waves (one workgroup a CU) against
// four: 664 and 752 us, 323 and 355; 128 rows, 8 x 8192 tokens: 74 and 76; few workgroups (448 rows, 1000 tokens) 15.4 and
// 13.5. Up to 32 rows the kernel above is as fast or faster (32 rows, 8 x 8192 tokens: 61 us; 48 rows here 65, there 80).
template <int D>
struct Staged {
  static constexpr int kPieces = D / 8;  // 16-byte pieces of a token
  static __device__ __forceinline__ int k_at(int token, int piece) {
    const int f = kPieces >= 16 ? token & 15 : token / (16 / kPieces) & (kPieces - 1);
    return token * kPieces + (piece ^ f);
  }
  static __device__ __forceinline__ int v_at(int token, int piece) {
    const int f = kPieces >= 16 ? (token & 3) << 2 : kPieces == 8 ? (token >> 1 & 1) << 2 : 0;
    return token * kPieces + (piece ^ f);
  }
};

typedef short i16x4_t __attribute__((ext_vector_type(4)));

template <class Ty, int D, int kW, bool kTwo>
__global__ __launch_bounds__(64 * kW, D == 256 ? 1 : 2) void pt_attend_wide_kernel(PTAttendLaunch a, AttendScale sc) {
  typedef Staged<D> L;
  constexpr int kTok = D == 256 ? 32 : 64, kThreads = 64 * kW, kRows = 32 * kW, kHalves = kTok / 32;
  constexpr int kTilePieces = kTok * L::kPieces, kEach = kTilePieces / kThreads;
  static_assert(kTilePieces % kThreads == 0 && kThreads % L::kPieces == 0, "whole pieces a thread, in one column");
  __shared__ u32x4 k_s[2][kTilePieces], v_s[2][kTilePieces];
  __shared__ uint32_t held_s[2][kTok];  // whether the tile's token is one that the block reads
  Work wk;
  if (!work_of(a, wk)) return;
  const PTPages& c = a.c;
  const int b = wk.b, h_kv = wk.h, n_rep = c.hq / c.hkv;
  const Span sp = span_of(a, b, wk.block * kRows, kRows, n_rep);
  const bool whole = wk.whole;
  const int begin = whole ? sp.begin : (int)min((int64_t)sp.end, sp.begin + (int64_t)wk.split * wk.per * kTok);
  const int end = whole ? sp.end : (int)min((int64_t)sp.end, begin + (int64_t)wk.per * kTok);
  if (!whole && begin >= end) return;
  const int tiles = (end - begin + kTok - 1) / kTok;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int h = lane >> 5, n = lane & 31;
  const int32_t* table = a.r.table + b * a.r.table_stride;
  const int in_page = (1 << c.page_shift) - 1;

  // Loads: thread tid takes piece tid % kPieces of tokens tid / kPieces + i * (kThreads / kPieces).
  const int piece = tid % L::kPieces, first_token = tid / L::kPieces;
  constexpr int kApart = kThreads / L::kPieces;
  const uint16_t* kp = static_cast<const uint16_t*>(c.keys) + ((int64_t)h_kv * D << c.page_shift) + piece * 8;
  const uint16_t* vp = static_cast<const uint16_t*>(c.values) + ((int64_t)h_kv * D << c.page_shift) + piece * 8;
  int32_t page[kEach];
  u32x4 kr[kEach], vr[kEach];
  uint32_t held = 0;  // bit i: token i of the thread's is read
  auto pages = [&](int ti) {
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      page[i] = table[min(begin + ti * kTok + first_token + i * kApart, end - 1) >> c.page_shift];
  };
  auto fetch = [&](int ti) {
    held = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int tok = begin + ti * kTok + first_token + i * kApart;
      const bool there = page[i] >= 0 && page[i] < c.pages;
      held |= (there & (tok >= sp.first) & (tok < end)) ? 1u << i : 0u;
      // (Behind the end: its last token; a page that is not there: the pool's first.)
      const int64_t at = (((int64_t)(there ? page[i] : 0) * c.hkv << c.page_shift) + (min(tok, end - 1) & in_page)) * D;
      kr[i] = *reinterpret_cast<const u32x4*>(kp + at);
      vr[i] = *reinterpret_cast<const u32x4*>(vp + at);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int t = first_token + i * kApart;
      const bool ok = held >> i & 1;
      k_s[buf][L::k_at(t, piece)] = kr[i];
      v_s[buf][L::v_at(t, piece)] = ok ? vr[i] : u32x4{0u, 0u, 0u, 0u};  // (NaN times a weight of 0 is NaN)
      if (piece == 0) held_s[buf][t] = ok;
    }
  };
  if (tiles > 0) {
    pages(0);
    fetch(0);
    pages(min(1, tiles - 1));
  }

  // The wave's rows.
  const int r0 = wk.block * kRows + 32 * wave, r = r0 + n, tok = r / n_rep, head = h_kv * n_rep + (r - tok * n_rep);
  const int t_first = r0 / n_rep, t_last = min((r0 + 31) / n_rep, sp.n - 1);
  const bool busy = t_first < sp.n;  // uniform
  const Row row = row_of(a, sp, b, tok);
  u32x4 q[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) q[i] = u32x4{0u, 0u, 0u, 0u};
  if (tok < sp.n) {
    const uint16_t* p = static_cast<const uint16_t*>(a.q) + b * a.qs.b + head * a.qs.h + tok * a.qs.t + 8 * h;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = *reinterpret_cast<const u32x4_e*>(p + 16 * i);
  }
  int lo_most = row.lo;
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) lo_most = max(lo_most, __shfl_xor(lo_most, m));
  lo_most = __builtin_amdgcn_readfirstlane(lo_most);
  const int seen_by_all = a.masks != nullptr ? sp.length : sp.length + t_first + 1;
  const int seen_by_none = a.masks != nullptr ? sp.end : sp.length + t_last + 1;

  if (tiles > 0) put(0);
  __syncthreads();
  arrived(q);

  float m_run = kMinusInf, l_run = 0.f;
  f32x16 acc[D / 32];
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[j][i] = 0.f;

  // The lane's places in a tile: of K piece h of token n (piece 2 i + h: XOR 2 i), of V its part of the transposing reads
  // of the first 32 dims (j: XOR 32 j elements, where a row is wider than that).
  const int k_first = L::k_at(n, h);
  const int v_first = L::v_at(4 * h + ((lane & 15) >> 2), 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) * 8 + 4 * (lane & 1);

  auto fold = [&](int ti, int buf) {
    const int c0 = begin + ti * kTok;
    int k_at = k_first, v_at = v_first;  // (taken apart anew for each tile: a dozen registers less over the loop)
    asm volatile("" : "+v"(k_at), "+v"(v_at));
    f32x16 s[kHalves];
#pragma unroll
    for (int x = 0; x < kHalves; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[x][i] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int x = 0; x < kHalves; ++x) s[x] = Ty::mma32(k_s[buf][(k_at ^ 2 * i) + 32 * x * L::kPieces], q[i], s[x]);
    const uint64_t here = __ballot(held_s[buf][lane & (kTok - 1)] != 0);
    // Uniform: some row of the wave may not see some token of the tile.
    const bool masked = ~here != 0 || c0 < lo_most || c0 + kTok > seen_by_all;
    // (Scores stay as the products left them, `unit` of them in log2 units: one multiply-add before the exponential.)
    float top = kMinusInf, unit = sc.scale_log2;
    if (sc.cap_log2 > 0.f) {
      unit = 1.f;
#pragma unroll
      for (int x = 0; x < kHalves; ++x) capped<16>(s[x], sc);
    }
    if (masked) {
      const uint64_t seen = sees(a, sp, row, c0 + 4 * h) & here >> 4 * h;
#pragma unroll
      for (int x = 0; x < kHalves; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[x][i] = (uint32_t)(seen >> 32 * x) >> (8 * (i / 4) + i % 4) & 1 ? s[x][i] : kMinusInf;
    }
#pragma unroll
    for (int x = 0; x < kHalves; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[x][i]);
    top = max_halves(top) * unit;
    // The reference of the weights follows the maximum where that is more than kSlack above it: weights are up to
    // 2^kSlack then, which both parts of P hold.
    if (__any(top > m_run + Ty::kSlack)) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == kMinusInf ? 0.f : m_new));
      l_run *= alpha;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) acc[j] *= alpha;
      m_run = m_new;
    }
    const float ref = m_run == kMinusInf ? 0.f : m_run;  // (scores of -inf weigh nothing, those of NaN stay NaN)
#pragma unroll
    for (int x = 0; x < kHalves; ++x) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[x][i] = __builtin_amdgcn_exp2f(fmaf(s[x][i], unit, -ref));
      float sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = (s[x][4 * i] + s[x][4 * i + 1]) + (s[x][4 * i + 2] + s[x][4 * i + 3]);
      l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        u32x4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p0 = s[x][8 * y + 2 * i], p1 = s[x][8 * y + 2 * i + 1];
          if constexpr (kTwo) {
            uint32_t u, v;
            Ty::split(p0, p1, u, v);
            hi[i] = u;
            lo[i] = v;
          } else {
            hi[i] = Ty::pack(p0 * (1.f / Ty::kUnit), p1 * (1.f / Ty::kUnit));
          }
        }
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          typedef __attribute__((address_space(3))) i16x4_t Lds;
          const uint16_t* at = reinterpret_cast<const uint16_t*>(v_s[buf]) + (v_at ^ 32 * j) + (32 * x + 16 * y) * D;
          const i16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)at);
          const i16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(at + 8 * D));
          const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
          const u32x4 vt = {w0.x, w0.y, w1.x, w1.y};
          if constexpr (kTwo) acc[j] = Ty::mma32(vt, lo, acc[j]);
          acc[j] = Ty::mma32(vt, hi, acc[j]);
        }
      }
    }
  };

  for (int ti = 0; ti < tiles; ++ti) {
    const int buf = ti & 1;
    if (ti + 1 < tiles) {
      fetch(ti + 1);
      pages(min(ti + 2, tiles - 1));
    }
    if (busy && begin + ti * kTok < seen_by_none) fold(ti, buf);
    if (ti + 1 < tiles) put(buf ^ 1);
    __syncthreads();
  }

  const float l = sum_halves(l_run);
  if (tok >= a.r.tokens) return;
  if (whole) {
    uint16_t* out = static_cast<uint16_t*>(a.out) + (((int64_t)b * a.r.tokens + tok) * c.hq + head) * D + 4 * h;
    const bool none = tok >= sp.n || l == 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = Ty::cvt(none ? 0.f : acc[j][4 * i + e] * Ty::kUnit / l);
        *reinterpret_cast<u32x2_e*>(out + 32 * j + 8 * i) = u32x2{y[0] | y[1] << 16, y[2] | y[3] << 16};
      }
    return;
  }
  const int64_t part = slot_of_part(a, wk, kRows) + 32 * wave + n;
  if (h == 0) {
    a.pm[part] = m_run;
    a.pl[part] = l;
  }
  float* to = a.pacc + part * D + 4 * h;
#pragma unroll
  for (int j = 0; j < D / 32; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<f32x4*>(to + 32 * j + 8 * i) =
          f32x4{acc[j][4 * i], acc[j][4 * i + 1], acc[j][4 * i + 2], acc[j][4 * i + 3]} * Ty::kUnit;
}

// Joins the parts of a row: `groups` groups of d / 4 threads take parts in turn, four dims a thread, under a maximum
// of their own, and are joined through LDS. Rows and groups fill a workgroup.
template <class Ty>
__global__ __launch_bounds__(256) void pt_merge_kernel(PTAttendLaunch a, int groups) {
  __shared__ float m_s[256], l_s[256];
  __shared__ f32x4 x_s[256];
  const PTPages& c = a.c;
  const int d = c.d, n_rep = c.hq / c.hkv, cols = d / 4, b = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  const int unit = tid / cols, e = (tid - unit * cols) * 4, g = unit % groups;
  const int r = blockIdx.x * (256 / cols / groups) + unit / groups, tok = r / n_rep;
  const bool real = tok < a.r.tokens;
  const int block = r / a.plan.rows, in = r - block * a.plan.rows;
  const Span sp = span_of(a, b, block * a.plan.rows, a.plan.rows, n_rep);
  const int2 meta = a.meta[b];  // the row's first part, a part's tiles
  const int tiles = row_tiles(a, b);
  if (tiles > 0 && tiles <= meta.y) return;  // (a row of one part is finished by its workgroup)
  // (Within the workspace, whatever the lengths have become since.)
  const int most = max(a.plan.slots - max(meta.x, 0), 0);
  const int used = real ? min((tiles_of(a.plan, sp) + meta.y - 1) / max(meta.y, 1), most) : 0;
  const int64_t part = (((int64_t)h * a.plan.blocks + block) * a.plan.slots + meta.x) * a.plan.rows + in;
  float m = kMinusInf, l = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < used; s += groups) {  // (one pass: the loads of several parts are under way together)
    const int64_t at = part + (int64_t)s * a.plan.rows;
    const float ms = a.pm[at], ls = a.pl[at];
    const f32x4 xs = *reinterpret_cast<const f32x4*>(a.pacc + at * d + e);
    const float top = fmaxf(m, ms), ref = top == kMinusInf ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f(m - ref), fs = __builtin_amdgcn_exp2f(ms - ref);
    l = l * f + ls * fs;
    x = x * f + xs * fs;
    m = top;
  }
  if (groups > 1) {
    m_s[tid] = m;
    l_s[tid] = l;
    x_s[tid] = x;
    __syncthreads();
    if (g != 0) return;
    for (int k = 1; k < groups; ++k) m = fmaxf(m, m_s[tid + k * cols]);
    const float all = m == kMinusInf ? 0.f : m;
    l = 0.f;
    x = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < groups; ++k) {
      const float f = __builtin_amdgcn_exp2f(m_s[tid + k * cols] - all);
      l += l_s[tid + k * cols] * f;
      x += x_s[tid + k * cols] * f;
    }
  }
  if (!real) return;
  const bool none = tok >= sp.n || l == 0.f;
  uint32_t y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = Ty::cvt(none ? 0.f : x[i] / l);
  const int64_t head = ((int64_t)b * a.r.tokens + tok) * c.hq + h * n_rep + (r - tok * n_rep);
  *reinterpret_cast<u32x2_e*>(static_cast<uint16_t*>(a.out) + head * d + e) = u32x2{y[0] | y[1] << 16, y[2] | y[3] << 16};
}

// ---------------------------------------------------------------------------------------
// The accepted path to the front: token length + j of each row becomes token length + path[j], as all were
// before the call. A workgroup finds the moves of one row once and makes them for its share of the row's planes (a
// plane: one KV head's keys or values in one layer), in 16-byte pieces. A move never reads what another plane's
// writes, so a workgroup takes as many planes at a time as its registers hold, reads all of their pieces and writes
// them behind a barrier. Entries outside [0, 64) move nothing, nor do those that are in their place. Memory-bound: 1774
// tokens moved in 64 rows, 8 KV heads, D 128, 32 layers: 101 us for 465 MB (4.6 TB/s); 291 with a workgroup that finds
// the moves anew for every plane.
constexpr int kKeepThreads = 512, kKeepEach = 4;  // pieces a thread holds: 64 tokens of up to 32 are one plane's at most

__global__ __launch_bounds__(kKeepThreads) void pt_keep_kernel(PTKeepLaunch a, int planes, int share) {
  __shared__ int64_t from_s[kMostDrafts], to_s[kMostDrafts];
  __shared__ int moves_s;
  const PTPages& c = a.c;
  const int b = blockIdx.y, tid = threadIdx.x, tokens = a.r.tokens;
  // A token's element in its plane's first page (head 0 of layer 0), or -1.
  auto cell = [&](int64_t token) {
    const int64_t page = token >> c.page_shift;
    if (page >= a.r.width) return (int64_t)-1;
    const int32_t p = a.r.table[b * a.r.table_stride + page];
    if (p < 0 || p >= c.pages) return (int64_t)-1;
    return (((int64_t)p * c.hkv << c.page_shift) + (token & (((int64_t)1 << c.page_shift) - 1))) * c.d;
  };
  if (tid < 64) {
    int64_t from = -1, to = -1;
    if (tid < tokens) {
      const int64_t length = max(a.r.lengths[b], 0);
      const int p = a.path[(int64_t)b * tokens + tid];
      if (p >= 0 && p < kMostDrafts && p != tid) {
        from = cell(length + p);
        to = cell(length + tid);
      }
    }
    const bool moves = from >= 0 && to >= 0;
    const uint64_t all = __ballot(moves);
    if (moves) {
      const int at = __popcll(all & ((1ull << tid) - 1));
      from_s[at] = from;
      to_s[at] = to;
    }
    if (tid == 0) moves_s = __popcll(all);
  }
  __syncthreads();
  const int pieces = c.d / 8, n = moves_s * pieces;  // of a plane
  if (n == 0) return;
  const int held = kKeepThreads * kKeepEach / n;  // planes at a time
  const int first = blockIdx.x * share, last = min(first + share, planes);
  const int64_t page = (int64_t)c.d << c.page_shift, layer = page * c.hkv * c.pages;
  for (int p0 = first; p0 < last; p0 += held) {
    const int count = min(held, last - p0) * n;
    u32x4 x[kKeepEach];
    uint16_t* to[kKeepEach];
#pragma unroll
    for (int i = 0; i < kKeepEach; ++i) {
      const int at = min(tid + i * kKeepThreads, count - 1), p = at / n, in = at - p * n, j = in / pieces;
      const int plane = p0 + p, half = plane >> 1, l = half / c.hkv, h = half - l * c.hkv;
      uint16_t* const pool = static_cast<uint16_t*>(plane & 1 ? c.values : c.keys) + l * layer + h * page + (in - j * pieces) * 8;
      to[i] = pool + to_s[j];
      x[i] = *reinterpret_cast<const u32x4*>(pool + from_s[j]);
    }
    arrived(x);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKeepEach; ++i)
      if (tid + i * kKeepThreads < count) *reinterpret_cast<u32x4*>(to[i]) = x[i];
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

template <class Ty, int D>
hipError_t attend_dim(const PTAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  const int64_t parts = (int64_t)p.c.hkv * (p.plan.slots == 0 ? p.r.batch : p.plan.slots);
  const dim3 grid((unsigned)((parts + 7) / 8 * 8 * p.plan.blocks));
  if (p.plan.listed) {
    pt_list_kernel<<<1, kListThreads, 0, stream>>>(p);
    const hipError_t listed = hipGetLastError();
    if (listed != hipSuccess) return listed;
  }
  if (p.plan.waves == 0) {
    if (p.plan.rows == 16 && p.plan.share == 4) pt_attend_kernel<Ty, D, 1, 4><<<grid, 256, 0, stream>>>(p, sc);
    if constexpr (D < 256) {
      if (p.plan.rows == 16 && p.plan.share == 8) pt_attend_kernel<Ty, D, 1, 8><<<grid, 512, 0, stream>>>(p, sc);
      if (p.plan.rows == 32) pt_attend_kernel<Ty, D, 2, 4><<<grid, 256, 0, stream>>>(p, sc);
    }
  } else if constexpr (D >= 32) {
    if (p.plan.waves == 4) {
      if (p.exact)
        pt_attend_wide_kernel<Ty, D, 4, true><<<grid, 256, 0, stream>>>(p, sc);
      else
        pt_attend_wide_kernel<Ty, D, 4, false><<<grid, 256, 0, stream>>>(p, sc);
    }
    if constexpr (D == 64 || D == 128) {
      if (p.plan.waves == 8) {
        if (p.exact)
          pt_attend_wide_kernel<Ty, D, 8, true><<<grid, 512, 0, stream>>>(p, sc);
        else
          pt_attend_wide_kernel<Ty, D, 8, false><<<grid, 512, 0, stream>>>(p, sc);
      }
    }
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.plan.slots == 0) return e;
  const int rows = p.r.tokens * (p.c.hq / p.c.hkv);
  int groups = 1;
  while (2 * groups * p.r.batch <= p.plan.slots && 2 * groups <= 256 / (D / 4) &&
         (int64_t)rows * p.c.hkv * p.r.batch * (D / 4) * groups < 256 * 512)
    groups *= 2;
  const int each = 256 / (D / 4) / groups;
  const dim3 merge((unsigned)((rows + each - 1) / each), (unsigned)p.c.hkv, (unsigned)p.r.batch);
  pt_merge_kernel<Ty><<<merge, 256, 0, stream>>>(p, groups);
  return hipGetLastError();
}

template <class Ty>
hipError_t attend(const PTAttendLaunch& p, const AttendScale& sc, hipStream_t stream) {
  switch (p.c.d) {
    case 16: return attend_dim<Ty, 16>(p, sc, stream);
    case 32: return attend_dim<Ty, 32>(p, sc, stream);
    case 64: return attend_dim<Ty, 64>(p, sc, stream);
    case 128: return attend_dim<Ty, 128>(p, sc, stream);
    default: return attend_dim<Ty, 256>(p, sc, stream);
  }
}

}  // namespace

PTAttendPlan pt_attend_plan(int batch, int tokens, int hq, int hkv, int64_t capacity, int d) {
  PTAttendPlan p;
  const int64_t rows = (int64_t)tokens * (hq / hkv), units = (int64_t)batch * hkv;
  int64_t target = 256;  // workgroups that the card holds at once, or that fill it
  if (rows > 32 && d >= 32) {
    p.tile = d == 256 ? 32 : 64;
    p.least = 2;
    p.waves = 4;
    if (rows > 64 && (d == 64 || d == 128) && units * ((rows + 255) / 256) * (capacity / 128) >= 256) p.waves = 8;
    if (p.waves == 4 && d < 256) target = 512;
    p.rows = 32 * p.waves;
  } else {
    p.rows = rows > 16 && d < 256 ? 32 : 16;
  }
  p.blocks = (int)((rows + p.rows - 1) / p.rows);
  if (p.rows == 16 && capacity * (d < 64 ? 64 : d) <= 1 << 15) {  // one workgroup finishes a row
    if (d < 256) p.share = p.least = 8;
    return p;
  }
  // The device adds the batch's tiles up in 32 bits: beyond, rows are left whole (2^35 tokens; such a table is
  // one that rows share).
  if (batch * ((capacity + p.tile - 1) / p.tile) >= (int64_t)1 << 30) return p;
  const int64_t groups = units * p.blocks, most = (capacity + p.least * p.tile - 1) / (p.least * p.tile),
                once = target / ((int64_t)hkv * p.blocks);
  // Places for a part of each row and for those of long rows. (None where a row's results are many: it has blocks enough
  // then.)
  const int64_t places = batch + (once > 8 ? once : 8);
  const bool few = places * hkv * p.blocks * p.rows * d * 4 <= (int64_t)128 << 20;
  if (batch > 256) {
    // Parts that every workgroup finds by walking the batch cost more than they gain here (one token, 16/1 heads, D 32, rows
    // of 0 to 4096 tokens, walked and whole: 300 rows 35 and 25 us, 1025 166 and 50, 4097 1729 and 202), so they are
    // listed once, by a launch of their own, and only where a row can be so long that it would hold the call up: one of
    // 60000 tokens among 299 of 200, 32/8 heads, D 128, 653 us whole, 167 walked, 110 listed; among 999 708, 1049, 222. Rows
    // alike under such a table pay for the launches: 300 of 1000 tokens 218 us whole, 245 walked, 232 listed; 16/1 heads,
    // D 32, 12, 25 and 20.
    p.listed = few && batch <= kMostListed && most >= 64;
    if (p.listed) p.slots = (int)places;
    return p;
  }
  // Parts a row on average: as many as fill the card once.
  int64_t n = target / groups;
  if (2 * groups > target) {
    // The blocks all but fill the card, or more: cut where whole rounds of workgroups come nearer by more than the parts
    // cost. The unit is a round of the longest block. Blocks of a prompt's tokens shorten from the last to the first, the
    // longest start first: they end after their mean work and the shortest block, or after whole rounds. A part's results
    // are written and read once more, which takes as long as two tokens for each of its rows, and 300 tokens at most (where
    // arithmetic bounds a token takes longer). 256 MiB of them at most: a token more must not ask for gigabytes.
    // Whole, in 2 and in 4 parts (P as one number): a prompt of 8193 tokens, 32/8 heads, D 128, 619, 720 and 777 us (8192: 665,
    // 740, 780), one of 2100 over 16384 1101, 853, 736; 9 rows of 130 over 900, 32/4, D 64, 31, 49, 52; 65 rows of one
    // token over 4096, 32/8, 222, 209, 208.
    const double round = (double)groups / target, last = tokens < capacity ? 1. - tokens / (double)capacity : 0.,
                 mean = 0.5 * (1. + last);
    const double each = 2. * rows / p.blocks < 300. ? 2. * rows / p.blocks : 300.;
    double best = 1e30;
    for (int k = 1; k <= 4; ++k) {
      const double whole = (double)((groups * k + target - 1) / target) / k;
      const double even = round * mean + (k == 1 ? last : 1. / k);
      double cost = even < whole ? even : whole;
      if (cost < 1. / k) cost = 1. / k;
      if (k > 1) {
        if (groups * k * p.rows * (d + 2) * 4 > (int64_t)256 << 20) break;
        cost += 0.05 + 0.01 * k + k * round * each / (capacity * mean);
      }
      if (cost < best) {
        best = cost;
        n = k;
      }
    }
  }
  if (n > most) n = most;
  if (n > 1) {
    p.slots = (int)(batch > 1 && once > n * batch ? once : n * batch);
  } else if (batch > 1 && most >= 32) {
    // The rows fill the card, but one that is much longer than the others would hold the call up: one of 60000 tokens and
    // 63 of 200 (32/8 heads, D 128) 635 us whole, 78 cut; 64 of 4096 tokens, none of them cut, 184 and 188.
    if (few) p.slots = (int)places;
  }
  return p;
}

hipError_t launch_pt_attend(int dtype, const PTAttendLaunch& p, hipStream_t stream) {
  AttendScale sc;
  constexpr double kLog2 = 1.4426950408889634;  // (of e; each factor rounded once)
  sc.scale_log2 = (float)(p.scale * kLog2);
  // (Scores are far below 2^88, so that a cap of 2^96 changes none of them by half a step, and larger ones pass float32's range
  // here; under the smallest caps the quotient must not, since 0 times infinity is NaN.)
  const bool capped = p.softcap > 0.f && p.softcap < 0x1p96f;
  sc.cap_scale = capped ? (float)std::fmin(p.scale / (double)p.softcap * (2. * kLog2), (double)FLT_MAX) : 0.f;
  sc.cap_log2 = capped ? (float)(p.softcap * kLog2) : 0.f;
  return dtype == kF16 ? attend<HalfT>(p, sc, stream) : attend<Bf16T>(p, sc, stream);
}

hipError_t launch_pt_keep(const PTKeepLaunch& p, hipStream_t stream) {
  const int planes = 2 * p.layers * p.c.hkv;
  int parts = (2048 + p.r.batch - 1) / p.r.batch;  // about 2048 workgroups
  if (parts > planes) parts = planes;
  const int share = (planes + parts - 1) / parts;
  pt_keep_kernel<<<dim3((unsigned)((planes + share - 1) / share), (unsigned)p.r.batch), kKeepThreads, 0, stream>>>(p, planes, share);
  return hipGetLastError();
}

hipError_t launch_draft_tree(const int32_t* parents, int batch, int tokens, uint64_t* masks, int32_t* depths,
                             hipStream_t stream) {
  draft_tree_kernel<<<(unsigned)batch, 64, 0, stream>>>(parents, tokens, masks, depths);
  return hipGetLastError();
}

}  // namespace pgr
