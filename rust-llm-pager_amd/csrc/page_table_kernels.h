// Launchers of the normed rotary embedding and of the cache of pages (implemented in
// norm_rotary_kernels.hip and page_table_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "cache_kernels.h"

namespace pgr {

// One layer of a cache of pages (pgr_pt_cache_t): keys and values [pages, hkv, 2^page_shift, d].
struct PTPages {
  void* keys = nullptr;
  void* values = nullptr;
  int pages = 0, hq = 0, hkv = 0, page_shift = 0, d = 0;
};

// The rows of a call: which pages hold their tokens, how many are held, how many are new.
struct PTRows {
  const int32_t* table = nullptr;  // [batch, width], the rows table_stride apart
  int64_t table_stride = 0;
  int width = 0;
  const int32_t* lengths = nullptr;  // [batch]
  const int32_t* counts = nullptr;   // [batch]; null: `tokens` each
  int batch = 0, tokens = 0;
};

// The RMS norm of each head before its turn: x / sqrt(mean(x^2) + eps) * weight. Weights null: no norm.
struct HeadNorm {
  const void* weight[2] = {nullptr, nullptr};  // q's and k's, [d]
  int weight_f32 = 0;                          // float32 instead of the operands' type
  float eps = 0.f;
};

struct NormRotaryLaunch {
  const void* x[3] = {nullptr, nullptr, nullptr};  // q, k and (append) v
  void* y[2] = {nullptr, nullptr};                 // [batch, heads, tokens, d] contiguous; append: q's alone
  Strides xs[3];
  int heads[2] = {0, 0};
  const void* positions = nullptr;  // append: null: the row's length plus the depth
  int positions64 = 0;
  int64_t pos_b = 0, pos_t = 0;
  RotaryForm form;
  HeadNorm norm;
  int batch = 0, tokens = 0, d = 0;
  // append:
  PTPages c;
  PTRows r;
  const int32_t* depths = nullptr;  // [batch, tokens]; null: a token's number
};
hipError_t launch_norm_rotary(int dtype, const NormRotaryLaunch& p, hipStream_t stream);
hipError_t launch_pt_append(int dtype, const NormRotaryLaunch& p, hipStream_t stream);

// How an attend call is dealt out.
struct PTAttendPlan {
  int waves = 0;    // of a workgroup whose waves hold 32 rows each; 0: one whose waves share its rows
  int share = 4;    // waves that share their rows (4 or 8)
  int rows = 16;    // rows (new token x query head of a KV head) of a workgroup
  int blocks = 1;   // blocks of rows
  int slots = 0;    // parts that the batch's rows are cut into at most (0: whole rows, no merge launch)
  int tile = 32;    // tokens
  int least = 4;    // tiles of a part at least
  bool listed = false;  // a launch of its own finds the parts
};
PTAttendPlan pt_attend_plan(int batch, int tokens, int hq, int hkv, int64_t capacity, int d);

struct PTAttendLaunch {
  PTPages c;
  PTRows r;
  const void* q = nullptr;
  Strides qs;
  void* out = nullptr;               // [batch, tokens, hq, d]
  const uint64_t* masks = nullptr;   // [batch, tokens]; null: in order
  const int32_t* depths = nullptr;   // with masks
  int window = 0;                    // 0: none
  float scale = 1.f, softcap = 0.f;
  int exact = 1;  // P as two numbers; 0: one where that is faster
  PTAttendPlan plan;
  int2* meta = nullptr;   // [batch]: a row's first part, a part's tiles
  int2* parts = nullptr;  // plan.listed: [slots]: a part's batch row (-1: no part) and its number in the row
  float* pm = nullptr;    // [hkv, blocks, slots, rows]
  float* pl = nullptr;
  float* pacc = nullptr;  // [..., d]
};
hipError_t launch_pt_attend(int dtype, const PTAttendLaunch& p, hipStream_t stream);

struct PTKeepLaunch {
  PTPages c;  // layer 0's
  PTRows r;   // tokens: the path's length
  int layers = 0;
  const int32_t* path = nullptr;  // [batch, tokens]
};
hipError_t launch_pt_keep(const PTKeepLaunch& p, hipStream_t stream);

hipError_t launch_draft_tree(const int32_t* parents, int batch, int tokens, uint64_t* masks, int32_t* depths,
                             hipStream_t stream);

// New tokens of a row that a tree's masks cover, and tokens of a path.
constexpr int kMostDrafts = 64;
// Rows of a batch whose parts are listed.
constexpr int kMostListed = 8192;

}  // namespace pgr
