// Launchers of the rotary and bounded-cache kernels (implemented in rotary_kernels.hip,
// cache_kernels.hip and prompt_weight_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "pgr_common.h"

namespace pgr {

// Element strides of a [batch, heads, tokens, head_dim] operand (head_dim has stride 1).
struct Strides {
  int64_t b = 0, h = 0, t = 0;
};

// How a head's rotary part is paired and turned.
struct RotaryForm {
  const float* inv_freq = nullptr;  // half values; null: nothing is turned
  int half = 0;                     // pairs
  int interleaved = 0;              // pairs (2i, 2i + 1) instead of (i, i + half)
  float factor = 1.f;               // of cos and sin
  float sign = 1.f;                 // -1: the inverse turn
};

struct RotaryLaunch {
  const void* x[2] = {nullptr, nullptr};  // q, k
  void* y[2] = {nullptr, nullptr};        // [batch, heads, tokens, d] contiguous
  Strides xs[2];
  int heads[2] = {0, 0};
  const void* positions = nullptr;
  int positions64 = 0;
  int64_t pos_b = 0, pos_t = 0;
  RotaryForm form;
  int batch = 0, tokens = 0, d = 0;
};
hipError_t launch_rotary(int dtype, const RotaryLaunch& p, hipStream_t stream);

// The buffers of a bounded cache (pgr_hh_cache_t).
struct HHCache {
  void* keys = nullptr;      // [batch, hkv, capacity, d]
  void* values = nullptr;
  float* weights = nullptr;  // [batch, hkv, capacity]
  int32_t* order = nullptr;
  int32_t* lengths = nullptr;  // [batch, hkv]
  int32_t* seen = nullptr;
  int batch = 0, hq = 0, hkv = 0, capacity = 0, d = 0;
  int keep_first = 0, keep_recent = 1;
};

struct HHAppendLaunch {
  HHCache c;
  const void *q = nullptr, *k = nullptr, *v = nullptr;
  Strides qs, ks, vs;  // t unused
  void* q_out = nullptr;
  const void* positions = nullptr;
  int positions64 = 0;
  RotaryForm form;
};
hipError_t launch_hh_append(int dtype, const HHAppendLaunch& p, hipStream_t stream);

// Splits of a cache row that an attend call makes (0: one workgroup per row, no merge launch), and the
// tokens of a row's scores (padded to whole tiles).
int hh_attend_splits(int batch, int hkv, int capacity, int d);
__host__ __device__ inline int64_t hh_attend_stride(int capacity) { return ((int64_t)capacity + 31) / 32 * 32; }

struct HHAttendLaunch {
  HHCache c;
  const void* q = nullptr;
  Strides qs;  // t unused
  void* out = nullptr;
  float scale = 1.f, softcap = 0.f;
  int n_split = 1;
  float* logits = nullptr;  // [batch, hq, hh_attend_stride]
  float* pm = nullptr;      // [batch, hkv, n_split, n_rep]
  float* pl = nullptr;
  float* pacc = nullptr;    // [batch, hkv, n_split, n_rep, d]
};
hipError_t launch_hh_attend(int dtype, const HHAttendLaunch& p, hipStream_t stream);

// What the launches of a long row's selection tell each other.
struct HHSelectRow {
  uint32_t cls, need, whole;  // the last taken token's class, how many of it are taken, whether all are
  uint32_t listed;            // its members
};

struct HHLoadLaunch {
  HHCache c;
  const void *k = nullptr, *v = nullptr;
  Strides ks, vs;
  const float* weights = nullptr;  // [batch, hkv, tokens]
  const int32_t* lo = nullptr;
  int tokens = 0;
  int32_t* kept = nullptr;  // [batch, hkv, capacity]
  // Long rows, dealt out in parts:
  uint16_t* part_counts = nullptr;  // [batch, hkv, parts, 2048]: tokens of each class
  uint32_t* part_above = nullptr;   // [batch, hkv, parts]: tokens of classes above the last one
  uint32_t* listed = nullptr;       // [batch, hkv, parts * hh_select_part_tokens()] (key, part)
  HHSelectRow* rows = nullptr;      // [batch, hkv]
};
int hh_select_parts(int tokens);
size_t hh_select_part_tokens();
hipError_t launch_hh_load(const HHLoadLaunch& p, hipStream_t stream);

// Geometry of a prompt_weights call.
struct PromptWeightPlan {
  int groups = 1;      // groups of 32 rows (statistics) or keys (sums) that a wave holds
  int row_waves = 4;   // waves of a statistics workgroup with rows of their own (1 or 4)
  int key_splits = 1;  // statistics pass: parts of the prompt per block of queries
  int row_splits = 1;  // sums pass: parts of the queries per block of keys
  bool norm_apart = true;  // the statistics' parts are joined by a launch of their own
};
PromptWeightPlan prompt_weight_plan(int batch, int hq, int hkv, int tokens, int window, int d);

struct PromptWeightLaunch {
  const void *q = nullptr, *k = nullptr;
  Strides qs, ks;
  const int32_t* lo = nullptr;
  float* out = nullptr;  // [batch, hkv, tokens]
  int batch = 0, hq = 0, hkv = 0, tokens = 0, window = 0, d = 0;
  float scale = 1.f, softcap = 0.f;
  PromptWeightPlan plan;
  float2* stats = nullptr;   // [key_splits][batch, hkv, rows]: (m, l) in log2 units
  float* norm = nullptr;     // [batch, hkv, rows]: m + log2(l), +inf where nothing is valid
  float* partial = nullptr;  // [row_splits][batch, hkv, tokens] (row_splits > 1)
};
hipError_t launch_prompt_weights(int dtype, const PromptWeightLaunch& p, hipStream_t stream);

// Head dims of the cache kernels: 16, 32, 64, 128, 256.
inline bool hh_head_dim_supported(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }

}  // namespace pgr
