// pkv_cache_ops.h -- argument structs and launchers of the operators that decide
// which cached state lives on: attention mass, eviction, beam selection and
// reordering.
#pragma once
#include "pkv_launch.h"

namespace pkv {

struct MassArgs {
  Geo g;
  const uint8_t *pool;
  int64_t num_pages;
  const uint16_t *q;  // [B][H][nq][D]
  int batch, heads, nq, gqa, rows;  // rows = nq * gqa per KV head: row r is query r / gqa of head r % gqa
  const int32_t *table;
  int max_pages;
  const int32_t *seq_lens, *q_pos, *widths;
  float scale;
  const float *mass;  // [mass_rows][HK][width] sums so far, or NULL
  const int32_t *counted, *out_rows;
  int mass_rows;
  int64_t width;
  float *out;  // as mass
  void *workspace;
};

int64_t mass_workspace(const Geo &g, int batch, int rows, int max_pages);
hipError_t launch_mass(hipStream_t stream, const MassArgs &a);

struct EvictSelectArgs {
  const float *mass;  // [layers][mass_rows][HK][width]
  int layers, mass_rows, hk;
  int64_t width;
  const int32_t *rows, *seq_lens, *keep;  // [B] each; rows and keep may be NULL
  int batch, max_keep, sinks, recent;
  int32_t *kept;      // [layers][B][HK][max_keep]
  int32_t *new_lens;  // [B]
  float *new_mass;    // [layers][mass_rows][HK][new_width], or NULL; may be mass
  int64_t new_width;
};

hipError_t launch_evict_select(hipStream_t stream, const EvictSelectArgs &a);

struct EvictPagesArgs {
  Geo g;
  uint8_t *pools[kMaxArenaPools];
  int num_pools;
  int64_t num_pages;
  const int32_t *kept;  // [num_pools][B][HK][max_keep]
  const int32_t *new_lens;
  int batch, max_keep;
  const int32_t *src_table, *dst_table;
  int src_pages, dst_pages;
};

hipError_t launch_evict_pages(hipStream_t stream, const EvictPagesArgs &a);

struct BeamArgs {
  const void *logits;
  int kind;  // 0 = bf16, 1 = f16, 2 = f32
  int groups, beams, vocab;
  int64_t group_stride, beam_stride;  // elements
  const float *scores;   // [groups][beams]
  const uint8_t *done;   // [groups][beams], or NULL
  int pad_token, count;
  void *workspace;
  float *out_scores;     // [groups][count]
  int32_t *parents, *tokens;
};

constexpr int kMaxBeams = 64, kMaxBeamCount = 64;
int64_t beam_workspace(int groups, int beams, int vocab, int count);
hipError_t launch_beam(hipStream_t stream, const BeamArgs &a);

struct ReorderArgs {
  uint8_t *state;  // [outer][num_rows][row_bytes]
  int64_t outer, row_bytes;
  int num_rows;
  const int32_t *targets, *sources;
  int count;
};

constexpr int kMaxReorder = 8192, kMaxArenaReorder = 4096;
hipError_t launch_reorder_rows(hipStream_t stream, const ReorderArgs &a);

struct ArenaReorderArgs {
  int32_t *state;
  int capacity;
  int32_t *table;
  int num_slots, max_pages;
  int32_t *lens;
  const int32_t *slots, *sources;
  int count;
  int32_t *workspace;
};

int64_t arena_reorder_workspace(int count, int max_pages);
hipError_t launch_arena_reorder(hipStream_t stream, const ArenaReorderArgs &a);

}  // namespace pkv
