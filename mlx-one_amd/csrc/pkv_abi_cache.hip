// pkv_abi_cache.hip -- extern "C" entry points of the operators that decide which
// cached state lives on (declared in include/pkv.h): attention mass, eviction, beam
// selection, reordering.  Validation and errors as in pkv_abi.hip; no entry point
// lets an exception out.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "pkv.h"

#include "pkv_cache_ops.h"
#include "pkv_error.h"

namespace {

using pkv::check_launch;
using pkv::fail;
using pkv::geometry;

// An entry point's body, with what it throws (no memory for an error text) as a
// status, or as a size of -1.
template <typename F>
auto guarded(F body) noexcept -> decltype(body()) {
  try {
    return body();
  } catch (...) {
    return sizeof(body()) == sizeof(int64_t) ? -1 : PKV_LAUNCH_FAILED;
  }
}

// The bounds below keep every grid under 2^32 threads.
constexpr int64_t kMaxRows = 1 << 24;  // query rows per KV head of a call

// Kernels count tokens in 32 bits up to the end of a row's last part: of 1024 tokens
// (attention mass), 16384 logits (beams), 32768 sums (select).
constexpr int64_t kMaxMassTokens = (int64_t)INT32_MAX - 1023;
constexpr int64_t kMaxVocab = (int64_t)INT32_MAX - ((1 << 15) - 1), kMaxSelectTokens = (int64_t)INT32_MAX - ((1 << 16) - 1);

// Kernels read and write their workspace 16 bytes at a time.
bool aligned(const void *workspace) { return (uintptr_t)workspace % 16 == 0; }

int mass_shape(const pkv_layout *layout, int32_t num_heads, int32_t num_queries, int32_t batch, int32_t max_pages,
               pkv_geometry *g) {
  if (int rc = geometry(layout, g)) return rc;
  if (batch < 0 || num_heads < 1 || num_queries < 0 || max_pages < 0)
    return fail(PKV_INVALID_ARGUMENT, "invalid attention mass shape");
  if (num_heads % g->hk) return fail(PKV_INVALID_ARGUMENT, "num_heads must be a multiple of num_kv_heads");
  if ((int64_t)num_queries * (num_heads / g->hk) > kMaxRows)
    return fail(PKV_UNSUPPORTED, "at most 2^24 query rows per KV head");
  if ((int64_t)max_pages * g->page > INT32_MAX) return fail(PKV_INVALID_ARGUMENT, "block table too wide");
  if ((int64_t)max_pages * g->page > kMaxMassTokens) return fail(PKV_UNSUPPORTED, "block tables of at most 2^31 - 1024 tokens");
  if ((int64_t)batch * g->hk > 65535) return fail(PKV_UNSUPPORTED, "at most 65535 (sequence, KV head) pairs");
  if ((int64_t)batch * g->hk * max_pages > (1 << 30))
    return fail(PKV_UNSUPPORTED, "at most 2^30 pages of (sequence, KV head) pairs");
  if ((int64_t)batch * g->hk * num_queries * (num_heads / g->hk) > (1 << 27))
    return fail(PKV_UNSUPPORTED, "at most 2^27 query rows");
  return PKV_OK;
}

int beam_shape(int32_t groups, int32_t beams, int32_t vocab, int32_t count) {
  if (groups < 0 || beams < 1 || vocab < 1 || count < 1) return fail(PKV_INVALID_ARGUMENT, "invalid beam shape");
  if (beams > pkv::kMaxBeams || count > pkv::kMaxBeamCount)
    return fail(PKV_UNSUPPORTED, "at most 64 beams and 64 selected pairs per group");
  if (vocab > kMaxVocab || (int64_t)beams * vocab > INT32_MAX || groups > (1 << 21) || (int64_t)groups * beams > (1 << 22) ||
      (int64_t)groups * beams * vocab > ((int64_t)1 << 36))
    return fail(PKV_UNSUPPORTED, "at most 2^31 - 2^15 tokens, 2^31 - 1 (beam, token) pairs per group, 2^21 groups, 2^22 beams and 2^36 pairs");
  if (count > (int64_t)beams * vocab) return fail(PKV_INVALID_ARGUMENT, "fewer (beam, token) pairs than the count");
  return PKV_OK;
}

int reorder_shape(int32_t count, int32_t max_pages) {
  if (count < 0 || max_pages < 1) return fail(PKV_INVALID_ARGUMENT, "invalid reorder shape");
  if (count > pkv::kMaxArenaReorder) return fail(PKV_UNSUPPORTED, "at most 4096 slots are reordered in a call");
  if (max_pages > (1 << 23)) return fail(PKV_UNSUPPORTED, "slot tables of at most 2^23 pages");
  return PKV_OK;
}

}  // namespace

extern "C" {

int64_t pkv_attention_mass_workspace_bytes(const pkv_layout *layout, int32_t num_heads, int32_t num_queries,
                                           int32_t batch, int32_t max_pages) {
  return guarded([&]() -> int64_t {
    pkv_geometry g;
    if (int rc = mass_shape(layout, num_heads, num_queries, batch, max_pages, &g)) return -rc;
    return pkv::mass_workspace(pkv::to_geo(g), batch, num_queries * (num_heads / g.hk), max_pages);
  });
}

int pkv_attention_mass(void *stream, const pkv_layout *layout, const void *pool, int64_t num_pages,
                       const void *queries, int32_t batch, int32_t num_heads, int32_t num_queries,
                       const int32_t *block_table, int32_t max_pages, const int32_t *seq_lens, const int32_t *q_pos,
                       const int32_t *widths, float scale, const float *mass, const int32_t *counted,
                       const int32_t *rows, int32_t mass_rows, int64_t mass_width, void *workspace,
                       int64_t workspace_bytes, float *out) {
  return guarded([&]() -> int {
    pkv_geometry g;
    if (int rc = mass_shape(layout, num_heads, num_queries, batch, max_pages, &g)) return rc;
    if (!std::isfinite(scale)) return fail(PKV_INVALID_ARGUMENT, "the softmax scale must be finite");
    if (num_pages < 0 || mass_rows < 0 || mass_width < 0 || (!rows && batch > mass_rows))
      return fail(PKV_INVALID_ARGUMENT, "invalid attention mass shape");
    if (batch == 0 || max_pages == 0 || mass_width == 0) return PKV_OK;
    if (!pool || !block_table || !seq_lens || !out || (num_queries > 0 && !queries))
      return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    pkv::MassArgs a;
    a.g = pkv::to_geo(g);
    a.gqa = num_heads / g.hk;
    a.rows = num_queries * a.gqa;
    const int64_t need = pkv::mass_workspace(a.g, batch, a.rows, max_pages);
    if (need > 0 && (!workspace || workspace_bytes < need))
      return fail(PKV_OUT_OF_MEMORY, "attention mass workspace too small: need " + std::to_string(need) + " bytes");
    if (need > 0 && !aligned(workspace)) return fail(PKV_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
    a.pool = (const uint8_t *)pool;
    a.num_pages = num_pages;
    a.q = (const uint16_t *)queries;
    a.batch = batch;
    a.heads = num_heads;
    a.nq = num_queries;
    a.table = block_table;
    a.max_pages = max_pages;
    a.seq_lens = seq_lens;
    a.q_pos = q_pos;
    a.widths = widths;
    a.scale = scale;
    a.mass = mass;
    a.counted = counted;
    a.out_rows = rows;
    a.mass_rows = mass_rows;
    a.width = mass_width;
    a.out = out;
    a.workspace = workspace;
    return check_launch(pkv::launch_mass((hipStream_t)stream, a), "attention mass launch");
  });
}

int pkv_evict_select(void *stream, const float *mass, int32_t layers, int32_t mass_rows, int32_t kv_heads,
                     int64_t mass_width, const int32_t *rows, const int32_t *seq_lens, int32_t batch,
                     const int32_t *keep, int32_t max_keep, int32_t sinks, int32_t recent, int32_t *kept,
                     int32_t *new_lens, float *new_mass, int64_t new_width) {
  return guarded([&]() -> int {
    if (layers < 0 || mass_rows < 0 || kv_heads < 1 || mass_width < 0 || mass_width > INT32_MAX || batch < 0 ||
        max_keep < 0 || (!rows && batch > mass_rows))
      return fail(PKV_INVALID_ARGUMENT, "invalid eviction shape");
    if (sinks < 0 || recent < 0) return fail(PKV_INVALID_ARGUMENT, "negative count of protected tokens");
    if (new_mass && new_width < max_keep)
      return fail(PKV_INVALID_ARGUMENT, "the kept sums need room for max_keep tokens");
    if (mass_width > kMaxSelectTokens || max_keep > kMaxSelectTokens)
      return fail(PKV_UNSUPPORTED, "at most 2^31 - 2^16 tokens");
    if ((int64_t)layers * batch * kv_heads > (1 << 21))
      return fail(PKV_UNSUPPORTED, "at most 2^21 (layer, sequence, KV head) rows");
    if (layers == 0 || batch == 0) return PKV_OK;
    const bool sums = mass_rows > 0 && mass_width > 0;  // (else no row has a token)
    if ((!mass && sums) || !seq_lens || !new_lens || (!kept && max_keep > 0))
      return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    pkv::EvictSelectArgs a;
    a.mass = mass;
    a.layers = layers;
    a.mass_rows = mass_rows;
    a.hk = kv_heads;
    a.width = mass_width;
    a.rows = rows;
    a.seq_lens = seq_lens;
    a.keep = keep;
    a.batch = batch;
    a.max_keep = max_keep;
    a.sinks = sinks;
    a.recent = recent;
    a.kept = kept;
    a.new_lens = new_lens;
    a.new_mass = new_mass;
    a.new_width = new_width;
    return check_launch(pkv::launch_evict_select((hipStream_t)stream, a), "eviction select launch");
  });
}

int pkv_evict_pages(void *stream, const pkv_layout *layout, void *const *pools, int32_t num_pools, int64_t num_pages,
                    const int32_t *kept, const int32_t *new_lens, int32_t batch, int32_t max_keep,
                    const int32_t *src_table, int32_t src_pages, const int32_t *dst_table, int32_t dst_pages) {
  return guarded([&]() -> int {
    pkv_geometry g;
    if (int rc = geometry(layout, &g)) return rc;
    if (num_pools < 0 || num_pools > pkv::kMaxArenaPools)
      return fail(PKV_INVALID_ARGUMENT, "pools must number 0..128");
    if (num_pages < 0 || batch < 0 || max_keep < 0 || src_pages < 0 || dst_pages < 0 ||
        (int64_t)src_pages * g.page > INT32_MAX || (int64_t)dst_pages * g.page > INT32_MAX)
      return fail(PKV_INVALID_ARGUMENT, "invalid eviction shape");
    if ((int64_t)batch * g.hk > 65535) return fail(PKV_UNSUPPORTED, "at most 65535 (sequence, KV head) pairs");
    if (max_keep > (1 << 29)) return fail(PKV_UNSUPPORTED, "at most 2^29 kept tokens");
    if (num_pools == 0 || batch == 0 || max_keep == 0 || src_pages == 0 || dst_pages == 0) return PKV_OK;
    if (!pools || !kept || !new_lens || !src_table || !dst_table) return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    pkv::EvictPagesArgs a;
    a.g = pkv::to_geo(g);
    for (int l = 0; l < num_pools; ++l) {
      if (!pools[l]) return fail(PKV_INVALID_ARGUMENT, "NULL pool");
      a.pools[l] = (uint8_t *)pools[l];
    }
    a.num_pools = num_pools;
    a.num_pages = num_pages;
    a.kept = kept;
    a.new_lens = new_lens;
    a.batch = batch;
    a.max_keep = max_keep;
    a.src_table = src_table;
    a.dst_table = dst_table;
    a.src_pages = src_pages;
    a.dst_pages = dst_pages;
    return check_launch(pkv::launch_evict_pages((hipStream_t)stream, a), "eviction pages launch");
  });
}

int64_t pkv_beam_workspace_bytes(int32_t groups, int32_t beams, int32_t vocab, int32_t count) {
  return guarded([&]() -> int64_t {
    if (int rc = beam_shape(groups, beams, vocab, count)) return -rc;
    return pkv::beam_workspace(groups, beams, vocab, count);
  });
}

int pkv_beam_select(void *stream, const void *logits, int32_t kind, int32_t groups, int32_t beams, int32_t vocab,
                    int64_t group_stride, int64_t beam_stride, const float *scores, const uint8_t *done,
                    int32_t pad_token, int32_t count, void *workspace, int64_t workspace_bytes, float *out_scores,
                    int32_t *parents, int32_t *tokens) {
  return guarded([&]() -> int {
    if (kind < 0 || kind > 2) return fail(PKV_INVALID_ARGUMENT, "logits must be bf16 (0), f16 (1) or f32 (2)");
    if (int rc = beam_shape(groups, beams, vocab, count)) return rc;
    if (group_stride < 0 || beam_stride < 0) return fail(PKV_INVALID_ARGUMENT, "negative logits stride");
    if (done && (pad_token < 0 || pad_token >= vocab))
      return fail(PKV_INVALID_ARGUMENT, "the pad token must lie in the vocabulary");
    if (groups == 0) return PKV_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens) return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    const int64_t need = pkv::beam_workspace(groups, beams, vocab, count);
    if (!workspace || workspace_bytes < need)
      return fail(PKV_OUT_OF_MEMORY, "beam workspace too small: need " + std::to_string(need) + " bytes");
    if (!aligned(workspace)) return fail(PKV_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
    pkv::BeamArgs a;
    a.logits = logits;
    a.kind = kind;
    a.groups = groups;
    a.beams = beams;
    a.vocab = vocab;
    a.group_stride = group_stride;
    a.beam_stride = beam_stride;
    a.scores = scores;
    a.done = done;
    a.pad_token = pad_token;
    a.count = count;
    a.workspace = workspace;
    a.out_scores = out_scores;
    a.parents = parents;
    a.tokens = tokens;
    return check_launch(pkv::launch_beam((hipStream_t)stream, a), "beam select launch");
  });
}

int pkv_reorder_rows(void *stream, void *state, int64_t outer, int32_t num_rows, int64_t row_bytes,
                     const int32_t *targets, const int32_t *sources, int32_t count) {
  return guarded([&]() -> int {
    if (outer < 0 || num_rows < 0 || row_bytes < 0 || count < 0)
      return fail(PKV_INVALID_ARGUMENT, "invalid reorder shape");
    if (count > pkv::kMaxReorder) return fail(PKV_UNSUPPORTED, "at most 8192 rows are reordered in a call");
    if (outer > 65535) return fail(PKV_UNSUPPORTED, "at most 65535 outer slices");
    if (row_bytes > ((int64_t)1 << 31)) return fail(PKV_UNSUPPORTED, "rows of at most 2^31 bytes");
    if (row_bytes * count > ((int64_t)1 << 37)) return fail(PKV_UNSUPPORTED, "rows of at most 2^37 bytes in a slice");
    if (outer == 0 || num_rows == 0 || row_bytes == 0 || count == 0) return PKV_OK;
    if (!state || !targets || !sources) return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    pkv::ReorderArgs a;
    a.state = (uint8_t *)state;
    a.outer = outer;
    a.row_bytes = row_bytes;
    a.num_rows = num_rows;
    a.targets = targets;
    a.sources = sources;
    a.count = count;
    return check_launch(pkv::launch_reorder_rows((hipStream_t)stream, a), "reorder launch");
  });
}

int64_t pkv_arena_reorder_workspace_bytes(int32_t count, int32_t max_pages) {
  return guarded([&]() -> int64_t {
    if (int rc = reorder_shape(count, max_pages)) return -rc;
    return count == 0 ? 0 : pkv::arena_reorder_workspace(count, max_pages);
  });
}

int pkv_arena_reorder(void *stream, void *state, int32_t capacity_pages, int32_t page_tokens, int32_t *slot_table,
                      int32_t num_slots, int32_t max_pages, int32_t *slot_lens, const int32_t *slots,
                      const int32_t *sources, int32_t count, void *workspace, int64_t workspace_bytes) {
  return guarded([&]() -> int {
    if (capacity_pages < 1 || capacity_pages > (1 << 30))
      return fail(PKV_INVALID_ARGUMENT, "arena capacity must be 1..2^30 pages");
    if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128)
      return fail(PKV_INVALID_ARGUMENT, "page_tokens must be 16, 32, 64 or 128");
    if (num_slots < 1 || max_pages < 1 || (int64_t)max_pages * page_tokens > INT32_MAX)
      return fail(PKV_INVALID_ARGUMENT, "invalid slot table shape");
    if (int rc = reorder_shape(count, max_pages)) return rc;
    if (!state || !slot_table || !slot_lens || (count > 0 && (!slots || !sources)))
      return fail(PKV_INVALID_ARGUMENT, "NULL arena tensor");
    if (count == 0) return PKV_OK;
    const int64_t need = pkv::arena_reorder_workspace(count, max_pages);
    if (!workspace || workspace_bytes < need)
      return fail(PKV_OUT_OF_MEMORY, "reorder workspace too small: need " + std::to_string(need) + " bytes");
    if (!aligned(workspace)) return fail(PKV_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
    pkv::ArenaReorderArgs a;
    a.state = (int32_t *)state;
    a.capacity = capacity_pages;
    a.table = slot_table;
    a.num_slots = num_slots;
    a.max_pages = max_pages;
    a.lens = slot_lens;
    a.slots = slots;
    a.sources = sources;
    a.count = count;
    a.workspace = (int32_t *)workspace;
    return check_launch(pkv::launch_arena_reorder((hipStream_t)stream, a), "arena reorder launch");
  });
}

}  // extern "C"
