// pkv_step.h -- argument structs and launchers of a serving step's operators: rotation
// with append, attention over packed prompts, attention over shared prefixes.
#pragma once
#include "pkv_launch.h"

namespace pkv {

struct RopeAppendArgs {
  Geo g;
  uint8_t *pool;
  int64_t num_pages;
  const uint16_t *qkv;  // rows of heads + 2 * hk heads of dim elements, row_stride elements apart
  int64_t row_stride;
  int rows, heads, batch;
  int tokens;  // row_starts NULL: sequence b has rows b * tokens ...
  const int32_t *row_starts, *widths, *start_pos;
  const int32_t *positions;  // [axes][rows], or NULL
  const int32_t *axis;       // [half], or NULL for axis 0
  int axes;
  const float *inv_freq;  // [half]
  int half;               // rotated pairs of a head
  const int32_t *table;
  int max_pages;
  uint16_t *q, *k, *v;  // packed [rows][heads][dim], or by sequence [batch][heads][tokens][dim]; k, v may be NULL
};

hipError_t launch_rope_append(hipStream_t stream, const RopeAppendArgs &a);

struct PromptArgs {
  const uint16_t *q, *k, *v;  // rows, stride elements apart; head h at h * dim
  int64_t q_stride, k_stride, v_stride;
  int float_kind, rows, batch, heads, kv_heads, gqa, dim;
  const int32_t *row_starts;
  float scale_log2;
  uint16_t *out;  // [rows][heads][dim]
};

hipError_t launch_prompt_attention(hipStream_t stream, const PromptArgs &a);

struct SharedArgs {
  Geo g;
  const uint8_t *pool;
  int64_t num_pages;
  const uint16_t *q;  // [B][H][nq][D]
  int batch, heads, nq, gqa, rows;  // rows = nq * gqa per KV head: row r is query r / gqa of head r % gqa
  const int32_t *table;
  int max_pages;
  const int32_t *seq_lens, *q_pos, *widths;
  float scale;
  int groups, count;  // members in all groups
  const int32_t *members, *group_starts, *prefix_lens;
  void *workspace;
  uint16_t *out;  // as q
};

constexpr int kMaxShared = 1024;  // sequences, and groups
// Query rows per block of the kernel, and the most a sequence may have per KV head.
constexpr int shared_rows(int dp) { return dp > 128 ? 16 : 32; }
int64_t shared_workspace(const Geo &g, int batch, int rows, int groups);
hipError_t launch_shared_attention(hipStream_t stream, const SharedArgs &a);

}  // namespace pkv
