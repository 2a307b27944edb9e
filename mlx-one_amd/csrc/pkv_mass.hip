// pkv_mass.hip -- the attention weight that a call's queries put on each cached token.
//
//   out[h, t] = old[h, t] + sum over query rows r of KV head h of softmax_t(scale * q_r . k_t)
//
// over the tokens t that row r sees (t <= its position, t < the sequence's
// length).  Two passes: the log-sum-exp of each row, then the weights summed
// over the rows of a token, in row order.
#include "pkv_cache_ops.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;

// Element d (< dp) of token `slot` of a head block's K side, dequantized.
__device__ __forceinline__ float k_element(const Geo &g, const uint8_t *head, int slot, int d) {
  const uint8_t *tile = head + (int64_t)(slot / PKV_TILE) * g.tile_bytes;
  const int lane = slot % PKV_TILE + 16 * ((d % 32) / 8), kb = d / 32, e = d % 8;
  if (g.bits == 16)
    return bits_to_float(*(const uint16_t *)(tile + payload_offset(lane, 2 * (8 * kb + e), g.chunk)), g.float_kind);
  int code;
  if (g.bits == 8) {
    code = tile[payload_offset(lane, 8 * kb + e, g.chunk)];
  } else {
    const int nib = k4_nibble(e);
    code = (tile[payload_offset(lane, 4 * kb + nib / 2, g.chunk)] >> (4 * (nib & 1))) & 15;
  }
  const uint32_t w = *(const uint32_t *)(head + g.kmeta_offset + ((int64_t)slot * g.ng + d / g.group) * 4);
  return (float)code * f16_bits_to_f32(w) + f16_bits_to_f32(w >> 16);
}

__device__ __forceinline__ const uint8_t *token_head(const MassArgs &a, int b, int kh, int t) {
  const int p = t / a.g.page;
  const int id = p < a.max_pages ? a.table[(int64_t)b * a.max_pages + p] : -1;
  if (id < 0 || id >= a.num_pages) return nullptr;
  return a.pool + (int64_t)id * a.g.page_bytes + (int64_t)kh * a.g.head_bytes;
}

__device__ __forceinline__ float score(const MassArgs &a, const uint8_t *head, int t, const float *q) {
  float s = 0.0f;
  for (int d = 0; d < a.g.dim; ++d) s += q[d] * k_element(a.g, head, t % a.g.page, d);
  return s * a.scale;
}

// The tokens of sequence b that count, and the tokens its row qi sees.
__device__ __forceinline__ int mass_len(const MassArgs &a, int b) {
  const int64_t most = min((int64_t)a.max_pages * a.g.page, a.width);
  return (int)min((int64_t)a.seq_lens[b], most);
}
__device__ __forceinline__ int row_sees(const MassArgs &a, int b, int qi, int L) {
  const int w = a.widths ? a.widths[b] : a.nq;
  if (qi >= w) return 0;
  const int pos = a.q_pos ? a.q_pos[(int64_t)b * a.nq + qi] : a.seq_lens[b] - w + qi;
  return pos >= L ? L : pos + 1;
}

__device__ __forceinline__ void load_query(const MassArgs &a, int b, int kh, int row, float *q) {
  const int qi = row / a.gqa, h = kh * a.gqa + row % a.gqa;
  const uint16_t *src = a.q + (((int64_t)b * a.heads + h) * a.nq + qi) * a.g.dim;
  for (int d = threadIdx.x; d < a.g.dim; d += kThreads) q[d] = bits_to_float(src[d], a.g.float_kind);
}

__global__ __launch_bounds__(kThreads) void mass_lse_kernel(const MassArgs a) {
  __shared__ float q[256], part[2][kThreads];
  const int row = blockIdx.x % a.rows, seg = blockIdx.x / a.rows;
  const int b = seg / a.g.hk, kh = seg % a.g.hk;
  const int L = mass_len(a, b), see = row_sees(a, b, row / a.gqa, L);
  load_query(a, b, kh, row, q);
  __syncthreads();
  float m = -INFINITY, l = 0.0f;
  for (int t = threadIdx.x; t < see; t += kThreads) {
    const uint8_t *head = token_head(a, b, kh, t);
    if (!head) continue;
    const float s = score(a, head, t, q);
    const float n = fmaxf(m, s);
    l = l * expf(m - n) + expf(s - n);
    m = n;
  }
  part[0][threadIdx.x] = m;
  part[1][threadIdx.x] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    float mm = -INFINITY, ll = 0.0f;
    for (int i = 0; i < kThreads; ++i) mm = fmaxf(mm, part[0][i]);
    for (int i = 0; i < kThreads; ++i)
      if (part[1][i] != 0.0f) ll += part[1][i] * expf(part[0][i] - mm);
    ((float *)a.workspace)[blockIdx.x] = ll == 0.0f ? INFINITY : mm + logf(ll);  // a row that sees nothing weighs nothing
  }
}

__global__ __launch_bounds__(kThreads) void mass_sum_kernel(const MassArgs a) {
  __shared__ float q[256];
  const int seg = blockIdx.y, b = seg / a.g.hk, kh = seg % a.g.hk;
  const int L = mass_len(a, b);
  const int t0 = blockIdx.x * kThreads, t = t0 + threadIdx.x;
  const int out_row = a.out_rows ? a.out_rows[b] : b;
  if (t0 >= L || out_row < 0 || out_row >= a.mass_rows) return;
  const uint8_t *head = t < L ? token_head(a, b, kh, t) : nullptr;
  float sum = 0.0f;
  for (int row = 0; row < a.rows; ++row) {
    const int see = row_sees(a, b, row / a.gqa, L);
    __syncthreads();
    load_query(a, b, kh, row, q);
    __syncthreads();
    if (head && t < see) sum += expf(score(a, head, t, q) - ((const float *)a.workspace)[seg * a.rows + row]);
  }
  if (t < L) {
    const int64_t at = ((int64_t)out_row * a.g.hk + kh) * a.width + t;
    const bool old = a.mass && (!a.counted || t < a.counted[b]);
    a.out[at] = (old ? a.mass[at] : 0.0f) + sum;
  }
}

}  // namespace

int64_t mass_workspace(const Geo &g, int batch, int rows, int /*max_pages*/) {
  return (int64_t)batch * g.hk * rows * 4;
}

hipError_t launch_mass(hipStream_t stream, const MassArgs &a) {
  const int segs = a.batch * a.g.hk;
  const int64_t tokens = min((int64_t)a.max_pages * a.g.page, a.width);
  hipLaunchKernelGGL(mass_lse_kernel, dim3(segs * a.rows), dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL(mass_sum_kernel, dim3((tokens + kThreads - 1) / kThreads, segs), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace pkv
