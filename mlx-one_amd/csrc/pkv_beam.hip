// pkv_beam.hip -- a beam step's selection over beams and vocabulary.
//
//   c[w, v] = score[w] + x[w, v] - log sum_v' exp(x[w, v'])
//
// and the `count` best of a group's (w, v), ties to the lowest w * V + v.  A
// finished beam has one candidate, its pad token at its score; a beam whose score
// or log-sum-exp is not finite has none.  Places past the candidates there are
// hold -inf and the lowest pairs that are no candidates.
//
// Which of two beams' tokens comes first hangs on the last digits of their
// log-sum-exps, so those, and the comparison, are in 64 bits; within a beam the
// logits themselves give the order.
#include "pkv_cache_ops.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;

struct RowBest {
  double log_sum;  // of exp(x - most); not finite: the row has no candidates
  float most;      // apart from the sum, which it would swallow where it is large
  int32_t n;       // its best tokens, in order
};

struct BeamParts {
  RowBest *row;
  float *value;
  int32_t *token;
  __device__ BeamParts(const BeamArgs &a) {
    const int64_t rows = (int64_t)a.groups * a.beams;
    row = (RowBest *)a.workspace;
    value = (float *)(row + rows);
    token = (int32_t *)(value + rows * a.count);
  }
};

__device__ __forceinline__ float logit(const BeamArgs &a, int64_t base, int v) {
  if (a.kind == 2) return ((const float *)a.logits)[base + v];
  return bits_to_float(((const uint16_t *)a.logits)[base + v], a.kind);
}

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T *s, F f) {
  __syncthreads();
  s[threadIdx.x] = v;
  for (int k = kThreads / 2; k > 0; k /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < k) s[threadIdx.x] = f(s[threadIdx.x], s[threadIdx.x + k]);
  }
  __syncthreads();
  return s[0];
}

__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// One workgroup per row: its log-sum-exp, then its best tokens one after another.
__global__ __launch_bounds__(kThreads) void beam_row_kernel(const BeamArgs a) {
  __shared__ double s_sum[kThreads];
  __shared__ float s_max[kThreads];
  __shared__ uint64_t s_key[kThreads];
  const BeamParts p(a);
  const int64_t row = blockIdx.x;
  const int64_t base = row / a.beams * a.group_stride + row % a.beams * a.beam_stride;
  float m = -INFINITY;
  bool nan = false;
  for (int v = threadIdx.x; v < a.vocab; v += kThreads) {
    const float x = logit(a, base, v);
    nan = nan || x != x;
    m = fmaxf(m, x);
  }
  m = block_reduce(nan ? INFINITY : m, s_max, [](float x, float y) { return fmaxf(x, y); });
  double sum = 0.0;
  const bool dead = !(fabsf(m) < INFINITY);
  if (!dead)
    for (int v = threadIdx.x; v < a.vocab; v += kThreads) sum += exp((double)logit(a, base, v) - (double)m);
  sum = block_reduce(sum, s_sum, [](double x, double y) { return x + y; });
  // order: the logit, then the lowest token; 0 is no token
  uint64_t last = ~0ull;
  int n = 0;
  for (; n < a.count && !dead; ++n) {
    uint64_t best = 0;
    for (int v = threadIdx.x; v < a.vocab; v += kThreads) {
      const float x = logit(a, base, v);
      const uint64_t key = (uint64_t)order_key(x) << 32 | (uint32_t)(~v);
      if (x > -INFINITY && key < last && key > best) best = key;
    }
    best = block_reduce(best, s_key, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
    if (best == 0) break;
    last = best;
    if (threadIdx.x == 0) {
      p.value[row * a.count + n] = key_value((uint32_t)(best >> 32));
      p.token[row * a.count + n] = (int32_t)~(uint32_t)best;
    }
  }
  if (threadIdx.x == 0) p.row[row] = RowBest{dead ? (double)INFINITY : log(sum), m, n};
}

// One thread per group: the rows' lists are in order, so the best of their heads
// is the next of all.
__global__ void beam_merge_kernel(const BeamArgs a) {
  const int group = blockIdx.x * blockDim.x + threadIdx.x;
  if (group >= a.groups) return;
  const BeamParts p(a);
  int at[kMaxBeams];
  for (int w = 0; w < a.beams; ++w) at[w] = 0;
  const int64_t out = (int64_t)group * a.count;
  int n = 0;
  for (; n < a.count; ++n) {
    double best = -INFINITY;
    int bw = -1, bt = 0;
    for (int w = 0; w < a.beams; ++w) {
      const int64_t row = (int64_t)group * a.beams + w;
      const float score = a.scores[row];
      if (!(fabsf(score) < INFINITY)) continue;
      double c;
      int t;
      if (a.done && a.done[row]) {
        if (at[w] > 0) continue;
        c = score;
        t = a.pad_token;
      } else {
        const RowBest best_of = p.row[row];
        if (!(fabs(best_of.log_sum) < INFINITY) || at[w] >= best_of.n) continue;
        c = (double)score - best_of.log_sum + ((double)p.value[row * a.count + at[w]] - (double)best_of.most);
        t = p.token[row * a.count + at[w]];
      }
      if (c > best) {
        best = c;
        bw = w;
        bt = t;
      }
    }
    if (bw < 0) break;
    ++at[bw];
    a.out_scores[out + n] = (float)best;
    a.parents[out + n] = bw;
    a.tokens[out + n] = bt;
  }
  const int found = n;
  for (int64_t f = 0; n < a.count; ++f) {  // the lowest pairs that were not taken
    const int w = (int)(f / a.vocab), t = (int)(f % a.vocab);
    bool taken = false;
    for (int k = 0; k < found; ++k) taken = taken || (a.parents[out + k] == w && a.tokens[out + k] == t);
    if (taken) continue;
    a.out_scores[out + n] = -INFINITY;
    a.parents[out + n] = w;
    a.tokens[out + n] = t;
    ++n;
  }
}

}  // namespace

int64_t beam_workspace(int groups, int beams, int /*vocab*/, int count) {
  return (int64_t)groups * beams * ((int64_t)sizeof(RowBest) + (int64_t)count * 8);
}

hipError_t launch_beam(hipStream_t stream, const BeamArgs &a) {
  hipLaunchKernelGGL(beam_row_kernel, dim3(a.groups * a.beams), dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL(beam_merge_kernel, dim3((a.groups + 63) / 64), dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace pkv
