// pkv_abi_step.hip -- extern "C" entry points of a serving step's operators (declared in
// include/pkv.h): rotation with append, attention over packed prompts, attention over
// shared prefixes.  Validation and errors as in pkv_abi.hip; no entry point lets an
// exception out.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "pkv.h"

#include "pkv_error.h"
#include "pkv_step.h"

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

int shared_shape(const pkv_layout *layout, int32_t num_heads, int32_t num_queries, int32_t num_members,
                 int32_t num_groups, pkv_geometry *g) {
  if (int rc = geometry(layout, g)) return rc;
  if (num_heads < 1 || num_queries < 1 || num_members < 0 || num_groups < 0)
    return fail(PKV_INVALID_ARGUMENT, "invalid shared attention shape");
  if (num_heads % g->hk) return fail(PKV_INVALID_ARGUMENT, "num_heads must be a multiple of num_kv_heads");
  const int64_t rows = (int64_t)num_queries * (num_heads / g->hk);
  if (rows > pkv::shared_rows(g->dp))
    return fail(PKV_UNSUPPORTED, "shared attention serves at most 32 query rows per KV head of a sequence (16 beyond "
                                 "head dim 128)");
  if (num_members > pkv::kMaxShared || num_groups > pkv::kMaxShared)
    return fail(PKV_UNSUPPORTED, "shared attention serves at most 1024 sequences and groups");
  if ((int64_t)num_members * g->hk > (1 << 16))
    return fail(PKV_UNSUPPORTED, "at most 65536 (sequence, KV head) pairs");
  return PKV_OK;
}

}  // namespace

extern "C" {

int pkv_rope_append(void *stream, const pkv_layout *layout, void *pool, int64_t num_pages, const void *qkv,
                    int64_t row_stride, int32_t rows, int32_t num_heads, int32_t batch, int32_t tokens,
                    const int32_t *row_starts, const int32_t *widths, const int32_t *start_pos,
                    const int32_t *positions, int32_t num_axes, const float *inv_freq, int32_t num_freqs,
                    const int32_t *axis, const int32_t *block_table, int32_t max_pages, void *q, void *k, void *v) {
  return guarded([&]() -> int {
    pkv_geometry g;
    if (int rc = geometry(layout, &g)) return rc;
    if (rows < 0 || batch < 0 || tokens < 0 || num_heads < 1 || num_pages < 0 || max_pages < 0)
      return fail(PKV_INVALID_ARGUMENT, "invalid rotation and append shape");
    if (num_freqs < 0 || 2 * (int64_t)num_freqs > g.dim)
      return fail(PKV_INVALID_ARGUMENT, "at most head_dim / 2 frequencies");
    if (num_axes < 1 || num_axes > 8) return fail(PKV_INVALID_ARGUMENT, "1 to 8 position axes");
    if (axis && !positions) return fail(PKV_INVALID_ARGUMENT, "axes need positions");
    if (row_starts && widths) return fail(PKV_INVALID_ARGUMENT, "packed rows take no widths");
    if (!row_starts && (int64_t)batch * tokens != rows)
      return fail(PKV_INVALID_ARGUMENT, "rows of a padded batch must be batch * tokens");
    const int64_t all = (int64_t)num_heads + 2 * (int64_t)g.hk;
    if (all > 65536) return fail(PKV_UNSUPPORTED, "at most 65536 heads of a row");
    if (row_stride < all * g.dim) return fail(PKV_INVALID_ARGUMENT, "rows overlap: row_stride is below the row's elements");
    if (row_stride > ((int64_t)1 << 40)) return fail(PKV_UNSUPPORTED, "row strides of at most 2^40 elements");
    if (rows > (1 << 23) || batch > (1 << 20)) return fail(PKV_UNSUPPORTED, "at most 2^23 rows and 2^20 sequences");
    if ((int64_t)rows * ((all + 3) / 4) > ((int64_t)1 << 23) * 256)
      return fail(PKV_UNSUPPORTED, "at most 2^33 (row, head) pairs");
    if ((int64_t)max_pages * g.page > INT32_MAX) return fail(PKV_INVALID_ARGUMENT, "block table too wide");
    if (rows == 0 || batch == 0) return PKV_OK;
    if (!qkv || !start_pos || !q || (num_freqs > 0 && !inv_freq) || (num_pages > 0 && !pool) ||
        (max_pages > 0 && !block_table))
      return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    if (!k != !v) return fail(PKV_INVALID_ARGUMENT, "k and v come out together");
    pkv::RopeAppendArgs a;
    a.g = pkv::to_geo(g);
    a.pool = (uint8_t *)pool;
    a.num_pages = num_pages;
    a.qkv = (const uint16_t *)qkv;
    a.row_stride = row_stride;
    a.rows = rows;
    a.heads = num_heads;
    a.batch = batch;
    a.tokens = tokens;
    a.row_starts = row_starts;
    a.widths = widths;
    a.start_pos = start_pos;
    a.positions = positions;
    a.axis = axis;
    a.axes = num_axes;
    a.inv_freq = inv_freq;
    a.half = num_freqs;
    a.table = block_table;
    a.max_pages = max_pages;
    a.q = (uint16_t *)q;
    a.k = (uint16_t *)k;
    a.v = (uint16_t *)v;
    return check_launch(pkv::launch_rope_append((hipStream_t)stream, a), "rotation and append launch");
  });
}

int pkv_prompt_attention(void *stream, const void *queries, int64_t q_stride, const void *keys, int64_t k_stride,
                         const void *values, int64_t v_stride, int32_t float_kind, int32_t rows, int32_t batch,
                         const int32_t *row_starts, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                         float scale, void *out) {
  return guarded([&]() -> int {
    if (float_kind != 0 && float_kind != 1) return fail(PKV_INVALID_ARGUMENT, "float_kind must be 0 or 1");
    if (rows < 0 || batch < 0 || num_heads < 1 || num_kv_heads < 1 || head_dim < 1)
      return fail(PKV_INVALID_ARGUMENT, "invalid prompt attention shape");
    if (num_heads % num_kv_heads) return fail(PKV_INVALID_ARGUMENT, "num_heads must be a multiple of num_kv_heads");
    if (head_dim > 256 || head_dim % 8)
      return fail(PKV_UNSUPPORTED, "prompt attention supports head dimensions 8, 16, ... 256");
    if (!std::isfinite(scale)) return fail(PKV_INVALID_ARGUMENT, "the softmax scale must be finite");
    if (q_stride < (int64_t)num_heads * head_dim || k_stride < (int64_t)num_kv_heads * head_dim ||
        v_stride < (int64_t)num_kv_heads * head_dim)
      return fail(PKV_INVALID_ARGUMENT, "rows overlap: a stride is below its row's elements");
    if ((q_stride | k_stride | v_stride) % 8) return fail(PKV_INVALID_ARGUMENT, "strides must be multiples of 8 elements");
    if (std::max(q_stride, std::max(k_stride, v_stride)) > (1 << 23))
      return fail(PKV_UNSUPPORTED, "strides of at most 2^23 elements");
    if (rows > (1 << 24) || batch > (1 << 20)) return fail(PKV_UNSUPPORTED, "at most 2^24 rows and 2^20 sequences");
    if (((int64_t)rows + 63 * (int64_t)std::min(rows, batch)) / 32 * num_heads > (1 << 23))
      return fail(PKV_UNSUPPORTED, "at most 2^28 (row, head) pairs");
    if (rows == 0 || batch == 0) return PKV_OK;
    if (!queries || !keys || !values || !row_starts || !out) return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    if (((uintptr_t)queries | (uintptr_t)keys | (uintptr_t)values | (uintptr_t)out) % 16)
      return fail(PKV_INVALID_ARGUMENT, "tensors must be 16-byte aligned");
    pkv::PromptArgs a;
    a.q = (const uint16_t *)queries;
    a.k = (const uint16_t *)keys;
    a.v = (const uint16_t *)values;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.float_kind = float_kind;
    a.rows = rows;
    a.batch = batch;
    a.heads = num_heads;
    a.kv_heads = num_kv_heads;
    a.gqa = num_heads / num_kv_heads;
    a.dim = head_dim;
    a.row_starts = row_starts;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.out = (uint16_t *)out;
    return check_launch(pkv::launch_prompt_attention((hipStream_t)stream, a), "prompt attention launch");
  });
}

int64_t pkv_shared_attention_workspace_bytes(const pkv_layout *layout, int32_t num_heads, int32_t num_queries,
                                             int32_t num_members, int32_t num_groups) {
  return guarded([&]() -> int64_t {
    pkv_geometry g;
    if (int rc = shared_shape(layout, num_heads, num_queries, num_members, num_groups, &g)) return -rc;
    return pkv::shared_workspace(pkv::to_geo(g), num_members, num_queries * (num_heads / g.hk), num_groups);
  });
}

int pkv_shared_attention(void *stream, const pkv_layout *layout, const void *pool, int64_t num_pages,
                         const void *queries, int32_t batch, int32_t num_heads, int32_t num_queries,
                         const int32_t *block_table, int32_t max_pages, const int32_t *seq_lens, const int32_t *q_pos,
                         const int32_t *widths, int32_t num_groups, const int32_t *members, int32_t num_members,
                         const int32_t *group_starts, const int32_t *prefix_lens, float scale, void *workspace,
                         int64_t workspace_bytes, void *out, int32_t zero_others) {
  return guarded([&]() -> int {
    pkv_geometry g;
    if (int rc = shared_shape(layout, num_heads, num_queries, num_members, num_groups, &g)) return rc;
    if (batch < 0 || num_pages < 0 || max_pages < 0) return fail(PKV_INVALID_ARGUMENT, "invalid shared attention shape");
    if (batch > (1 << 20)) return fail(PKV_UNSUPPORTED, "at most 2^20 sequences");
    if ((int64_t)batch * num_heads * num_queries > (1 << 25)) return fail(PKV_UNSUPPORTED, "at most 2^25 query rows");
    if ((int64_t)max_pages * g.page > INT32_MAX) return fail(PKV_INVALID_ARGUMENT, "block table too wide");
    if ((int64_t)max_pages * g.page > INT32_MAX - 4096) return fail(PKV_UNSUPPORTED, "block tables of at most 2^31 - 4097 tokens");
    if (!std::isfinite(scale)) return fail(PKV_INVALID_ARGUMENT, "the softmax scale must be finite");
    if (batch == 0 || num_members == 0 || num_groups == 0) return PKV_OK;
    if (!pool || !queries || !block_table || !seq_lens || !members || !group_starts || !prefix_lens || !out)
      return fail(PKV_INVALID_ARGUMENT, "NULL tensor");
    if (num_pages < 1 || max_pages < 1) return fail(PKV_INVALID_ARGUMENT, "empty page pool or block table");
    pkv::SharedArgs a;
    a.g = pkv::to_geo(g);
    a.gqa = num_heads / g.hk;
    a.rows = num_queries * a.gqa;
    const int64_t need = pkv::shared_workspace(a.g, num_members, a.rows, num_groups);
    if (!workspace || workspace_bytes < need)
      return fail(PKV_OUT_OF_MEMORY, "shared attention workspace too small: need " + std::to_string(need) + " bytes");
    if ((uintptr_t)workspace % 16) return fail(PKV_INVALID_ARGUMENT, "the workspace must be 16-byte aligned");
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
    a.groups = num_groups;
    a.count = num_members;
    a.members = members;
    a.group_starts = group_starts;
    a.prefix_lens = prefix_lens;
    a.workspace = workspace;
    a.out = (uint16_t *)out;
    a.zero_others = zero_others;
    return check_launch(pkv::launch_shared_attention((hipStream_t)stream, a), "shared attention launch");
  });
}

}  // extern "C"
