// pkv_step.h -- argument structs and launchers of a serving step's operators: rotation
// with append, attention over packed prompts, attention over shared prefixes.
#pragma once
#include "pkv_launch.h"

namespace pkv {

// What values that are not finite add to a sum: `count` holds how many are +inf, -inf and
// NaN, in digits of 64.
__device__ __forceinline__ float seen_kinds(float count) {
  const int n = (int)count;
  const bool plus = n & 63, minus = n >> 6 & 63, nan = n >> 12;
  return nan || (plus && minus) ? __builtin_nanf("") : plus ? INFINITY : minus ? -INFINITY : 0.0f;
}

// Sixteen bytes of each active lane from memory to LDS at `to` + 16 lane (`to` alike for the
// wave).  Written as an instruction, which has no result register: for the builtin the compiler
// waits for every copy under way before any read of LDS.  The caller waits (vmcnt) before it
// reads what was copied.  The second form reads at base + offset, base alike for the wave.
typedef __attribute__((address_space(3))) uint8_t ldsbyte;
__device__ __forceinline__ void copy_to_lds(const uint8_t *from, uint8_t *to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ldsbyte *)to);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(at) : "memory", "m0");
}
__device__ __forceinline__ void copy_to_lds(const uint8_t *base, uint32_t offset, uint8_t *to) {
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(ldsbyte *)to);
  // (a request reads scalars that a vector instruction wrote five wait states later at the soonest)
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(at) : "memory", "m0");
}

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
  int zero_others;  // the rows of sequences that no group names become zeros
};

constexpr int kMaxShared = 1024;  // sequences, and groups
// Query rows per block of the kernel, and the most a sequence may have per KV head.
constexpr int shared_rows(int dp) { return dp > 128 ? 16 : 32; }
int64_t shared_workspace(const Geo &g, int batch, int rows, int groups);
hipError_t launch_shared_attention(hipStream_t stream, const SharedArgs &a);

}  // namespace pkv
