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
// log-sum-exps, so those are joined, and candidates compared, in 64 bits.  What they are
// joined from is float32: hardware exponentials and each thread's sum of 32 or 64 of them,
// which leaves a log-sum-exp off by up to 2^-21, and 2^-23 times the mean of max - x under
// the softmax; closer beams come in the order of these sums.  Within a beam the logits
// themselves give the order.
//
// One launch reads the logits, in chunks of a row held in registers: the chunk's
// maximum and sum of exponentials, and its `count` best tokens.  Each wave finds
// the count-th largest of its lanes' maxima, by bisection on the bits of the order;
// what reaches the largest of the waves' bounds, a few times `count`, goes to LDS
// and is ranked there.  A second launch joins the chunks' sums and does the same
// with the lists' entries.  One read of the logits: 128 rows of 128256 bfloat16 (33
// MB) take 13.8 us (2.4 TB/s: all chunks resident at once, one round of loads, sums,
// bisection and ranks, half of it the issue of instructions) and the merge 8.6 us, a chain of dependent steps; 768 rows of 104543
// float16, 21 selected (161 MB), 62 us (2.6 TB/s) and 14.
#include <cfloat>

#include "pkv_cache_ops.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMergeList = 512;  // candidates of a group in LDS
constexpr int kHeld = 16384;  // candidates of a group whose order is kept in LDS
constexpr int kList = 256;  // candidates in LDS, per wave

// Order of float32 as unsigned numbers (none is 0, which callers take for nothing).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Of a chunk: its sum of exp(x - most) and its maximum (NaN where there is a NaN).
struct Chunk {
  double sum;
  float most;
};

// Workspace: [groups][beams][chunks] Chunk, then as many lists [count] of (order, token).
struct BeamParts {
  int chunks;
  uint32_t by_count, by_chunks;  // floor(2^32 / d) + 1: __umulhi(e, it) = e / d for e < 2^32 / d
  int64_t lists, total;
  __host__ __device__ BeamParts(int groups, int beams, int vocab, int count, int vectors) {
    const int chunk = 8 * vectors * kThreads;
    chunks = (vocab + chunk - 1) / chunk;
    const int64_t n = (int64_t)groups * beams * chunks;
    by_count = (uint32_t)(((uint64_t)1 << 32) / count) + 1;
    by_chunks = (uint32_t)(((uint64_t)1 << 32) / chunks) + 1;
    lists = n * (int64_t)sizeof(Chunk);
    total = lists + n * count * 8;
  }
};

// Eight logits from v on (-inf from the end of the row on), wherever they lie: as
// they are in memory.
template <int KIND>
struct Eight {
  uint32_t w[KIND == 2 ? 8 : 4];

  __device__ __forceinline__ void load(const BeamArgs &a, int64_t base, int v) {
    if (v + 8 <= a.vocab) {
      if constexpr (KIND == 2) __builtin_memcpy(w, (const float *)a.logits + base + v, 32);
      else __builtin_memcpy(w, (const uint16_t *)a.logits + base + v, 16);
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = v + e < a.vocab;
      if constexpr (KIND == 2) {
        w[e] = in ? ((const uint32_t *)a.logits)[base + v + e] : 0xFF800000u;
      } else {
        const uint32_t x = in ? ((const uint16_t *)a.logits)[base + v + e] : KIND == 0 ? 0xFF80u : 0xFC00u;
        w[e / 2] = e % 2 ? w[e / 2] | x << 16 : x;
      }
    }
  }
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (KIND == 2) return __uint_as_float(w[e]);
    else if constexpr (KIND == 0) return __uint_as_float(e % 2 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    else return f16_bits_to_f32(e % 2 ? w[e / 2] >> 16 : w[e / 2]);
  }
};

// The largest bound that `count` of the wave's N x 64 keys reach, to BITS bits from
// the top (the rest 0); 0 where fewer than `count` are above 0.
template <int BITS, int N>
__device__ __forceinline__ uint32_t wave_bound(const uint32_t (&key)[N], int count) {
  uint32_t at = 0;
#pragma unroll
  for (int bit = 31; bit >= 32 - BITS; --bit) {
    const uint32_t next = at | 1u << bit;
    int reach = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) reach += __popcll(__ballot(key[j] >= next));
    if (reach >= count) at = next;
  }
  return at;
}

// Lane exchanges of a 64-bit value, as two halves, without LDS.
template <int CTRL>
__device__ __forceinline__ double row_xchg64(double v) {
  const u2 h = __builtin_bit_cast(u2, v);
  return __builtin_bit_cast(double, u2{(uint32_t)__builtin_amdgcn_mov_dpp((int)h.x, CTRL, 0xF, 0xF, false),
                                       (uint32_t)__builtin_amdgcn_mov_dpp((int)h.y, CTRL, 0xF, 0xF, false)});
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += row_xchg64<0xB1>(v);
  v += row_xchg64<0x4E>(v);
  v += row_xchg64<0x141>(v);
  v += row_xchg64<0x140>(v);
  const u2 h = __builtin_bit_cast(u2, v);
  const auto x = __builtin_amdgcn_permlane16_swap(h.x, h.x, false, false), y = __builtin_amdgcn_permlane16_swap(h.y, h.y, false, false);
  v = __builtin_bit_cast(double, u2{x[0], y[0]}) + __builtin_bit_cast(double, u2{x[1], y[1]});
  const u2 g = __builtin_bit_cast(u2, v);
  const auto z = __builtin_amdgcn_permlane32_swap(g.x, g.x, false, false), t = __builtin_amdgcn_permlane32_swap(g.y, g.y, false, false);
  return __builtin_bit_cast(double, u2{z[0], t[0]}) + __builtin_bit_cast(double, u2{z[1], t[1]});
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, row_xchg<0xB1>(v));
  v = fmaxf(v, row_xchg<0x4E>(v));
  v = fmaxf(v, row_xchg<0x141>(v));
  v = fmaxf(v, row_xchg<0x140>(v));
  return xor32_max(xor16_max(v));
}

// Lanes of the wave before this one that are in `mask`.
__device__ __forceinline__ int lanes_before(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Sum over four neighbouring lanes.
__device__ __forceinline__ int sum4(int v) {
  v += __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false);
  return v + __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false);
}

// V vectors of eight logits per thread
template <int KIND, int V>
__global__ __launch_bounds__(kThreads, V > 4 ? 4 : 6) void beam_chunk_kernel(const BeamArgs a, const BeamParts w) {
  constexpr int kChunk = 8 * V * kThreads;
  __shared__ uint64_t s_list[kWaves][kList];  // (order << 32 | ~token), what each wave found
  __shared__ double s_sum[kWaves];
  __shared__ float s_most[kWaves];
  __shared__ uint32_t s_bound[kWaves];
  __shared__ int s_n[kWaves], s_nan;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / w.chunks;
  if (a.done && a.done[row]) return;  // its logits are not asked for
  const int64_t base = row / a.beams * a.group_stride + row % a.beams * a.beam_stride;
  const int v0 = (int)(blockIdx.x % w.chunks) * kChunk + threadIdx.x * 8;
  Eight<KIND> x[V];
  float vm[V];
#pragma unroll
  for (int j = 0; j < V; ++j) x[j].load(a, base, v0 + j * 8 * kThreads);
  if (threadIdx.x == 0) s_nan = 0;
  bool nan = false;
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    vm[j] = x[j][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) vm[j] = __builtin_elementwise_maximum(vm[j], x[j][e]);  // NaN stays
    m = __builtin_elementwise_maximum(m, vm[j]);
  }
  nan = m != m;
  // A bound from the lanes' maxima; for many tokens from those of their vectors,
  // which also do where masks leave lanes without a token.  bfloat16's order has 16
  // bits, float16's 19, of float32's 24 are enough.
  constexpr int kBits = KIND == 0 ? 16 : KIND == 1 ? 19 : 24;
  auto key_of = [](float v) { return v == -INFINITY ? 0u : order_key(v); };
  uint32_t bound;
  if (a.count <= 16) {
    const uint32_t key[1] = {key_of(m)};
    bound = wave_bound<kBits>(key, a.count);
  } else {
    uint32_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = key_of(vm[j]);
    bound = wave_bound<kBits>(key, a.count);
  }
  const float most = wave_max(m);
  // exp(x - most) as 2^(x L - R), L = log2(e) in float32 and R the integer next to
  // most L: the product is not rounded, R is exact, and 2^(R - most L) makes up for it
  constexpr float kL = 1.4426950408889634f;
  const float from = rintf(most * kL);
  // From 8e6 on float32 holds no such R (and one that is off by hundreds leaves a sum of
  // inf or 0).  Logits there lie half a unit apart at least, so x - most is exact where
  // its exponential is not 0.  Masks of -1e9 to -1e38 come here, and rows without a sum.
  const bool flat = __builtin_amdgcn_readfirstlane(!(fabsf(most) < 8e6f));
  float sum = 0.0f;
  if (flat) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += __builtin_amdgcn_exp2f((x[j][e] - most) * kL);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += __builtin_amdgcn_exp2f(fmaf(x[j][e], kL, -from));
  }
  const double total = wave_sum64((double)sum) * (flat ? 1.0 : exp2((double)from - (double)most * (double)kL));
  if (lane == 0) {
    s_sum[wave] = total;
    s_most[wave] = most;
    s_bound[wave] = bound;
  }
  __syncthreads();
  if (nan) s_nan = 1;
  // what reaches the highest bound: `count` tokens at least, if there are as many
  uint32_t least = 1;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) least = max(least, s_bound[k]);
  const float reach = fmaxf(key_value(least), -FLT_MAX);
  int found = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (__ballot(vm[j] >= reach) == 0) continue;  // (in a row with a NaN nothing matters)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = x[j][e] >= reach;
      const unsigned long long mask = __ballot(in);
      if (mask == 0) continue;
      const int at = found + lanes_before(mask);
      if (in && at < kList)
        s_list[wave][at] = (uint64_t)order_key(x[j][e]) << 32 | (uint32_t)~(v0 + j * 8 * kThreads + e);
      found += __popcll(mask);
    }
  }
  if (lane == 0) s_n[wave] = found;
  __syncthreads();
  uint2 *list = (uint2 *)((char *)a.workspace + w.lists) + (int64_t)blockIdx.x * a.count;
  int n = 0, longest = 0;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    n += s_n[k];
    longest = max(longest, s_n[k]);
  }
  if (longest > kList) {
    // more equal (or adjacent) tokens than the list holds: one after another
    uint64_t last = ~0ull;
    __shared__ uint64_t s_best[kWaves];
    for (n = 0; n < a.count; ++n) {
      uint64_t best = 0;
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint64_t k = (uint64_t)order_key(x[j][e]) << 32 | (uint32_t)~(v0 + j * 8 * kThreads + e);
          if (x[j][e] > -INFINITY && k < last && k > best) best = k;
        }
#pragma unroll
      for (int k = 1; k < 64; k *= 2) {
        const uint64_t other = __shfl_xor((unsigned long long)best, k, 64);
        best = other > best ? other : best;
      }
      __syncthreads();
      if (lane == 0) s_best[wave] = best;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kWaves; ++k) best = s_best[k] > best ? s_best[k] : best;
      if (best == 0) break;
      last = best;
      if (threadIdx.x == 0) list[n] = uint2{(uint32_t)(best >> 32), ~(uint32_t)best};
    }
  } else {
    // a rank is the number of larger ones (no two are equal), counted by four lanes,
    // one of the waves' finds each
    for (int i0 = 0; i0 < n; i0 += kThreads / 4) {
      int i = i0 + (int)threadIdx.x / 4, from = 0;
      const bool mine = i < n;
#pragma unroll
      for (int k = 0; k < kWaves - 1; ++k)
        if (mine && from == k && i >= s_n[k]) {
          i -= s_n[k];
          ++from;
        }
      const uint64_t key = mine ? s_list[from][i] : 0;
      const int other = threadIdx.x % 4, most = s_n[other];
      int rank = 0;
#pragma unroll 8
      for (int k = 0; k < most; ++k) rank += s_list[other][k] > key;
      rank = sum4(rank);
      if (mine && other == 0 && rank < a.count) list[rank] = uint2{(uint32_t)(key >> 32), ~(uint32_t)key};
    }
    n = min(n, a.count);
  }
  for (int k = n + (int)threadIdx.x; k < a.count; k += kThreads) list[k] = uint2{0u, 0u};  // 0: none
  if (wave == kWaves - 1 && lane < kWaves) {  // four lanes of the last wave, which has the least to rank
    const float part = s_most[lane];
    float all = fmaxf(part, row_xchg<0xB1>(part));
    all = fmaxf(all, row_xchg<0x4E>(all));
    double sums = part > -INFINITY ? s_sum[lane] * exp((double)part - (double)all) : 0.0;
    sums += row_xchg64<0xB1>(sums);
    sums += row_xchg64<0x4E>(sums);
    if (lane == 0) ((Chunk *)a.workspace)[blockIdx.x] = Chunk{sums, s_nan ? NAN : all};
  }
}

// One workgroup per group of beams.
template <int kMergeThreads>
__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(const BeamArgs a, const BeamParts w) {
  constexpr int kMergeWaves = kMergeThreads / 64;
  struct Pair {
    double c;
    uint32_t key;  // the logit's: the order within a beam
    int32_t beam, token;
  };
  __shared__ Pair s_list[kMergeList], s_best[kMergeWaves];
  __shared__ double s_c[kMergeList];
  __shared__ uint64_t s_tie[kMergeList];  // order of equal ones but for the token: (beam, the logit's falling)
  __shared__ uint32_t s_order[kHeld];
  __shared__ double s_offset[kMaxBeams];  // score - log of the sum; -inf: no candidates
  __shared__ float s_most[kMaxBeams];
  __shared__ int s_reach[2][3][kMergeWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr double kNone = -(double)INFINITY;
  const int64_t row0 = (int64_t)blockIdx.x * a.beams, out = (int64_t)blockIdx.x * a.count;
  const Chunk *chunk = (const Chunk *)a.workspace + row0 * w.chunks;
  const uint2 *lists = (const uint2 *)((const char *)a.workspace + w.lists) + row0 * w.chunks * a.count;
  auto done = [&](int beam) { return a.done && a.done[row0 + beam]; };
  const int entries = a.beams * w.chunks * a.count;  // (less than 2^31 pairs per group: so are these)
  // a row's sum: lanes beside each other take its chunks
  int width = 1;
  while (width < 64 && width < w.chunks && width * 2 * a.beams <= kMergeThreads) width *= 2;
  const int beam = threadIdx.x / width, slice = threadIdx.x % width;
  if (beam < a.beams) {
    const float score = a.scores[row0 + beam];
    bool dead = !(fabsf(score) < INFINITY);
    float most = -INFINITY;
    double sum = 0.0;
    if (!done(beam)) {
      for (int k = slice; k < w.chunks; k += width) {
        const float x = chunk[beam * w.chunks + k].most;
        dead = dead || x != x;
        most = fmaxf(most, x);
      }
      for (int k = 1; k < width; k *= 2) {
        most = fmaxf(most, __shfl_xor(most, k, 64));
        dead = __shfl_xor((int)dead, k, 64) || dead;
      }
      dead = dead || !(fabsf(most) < INFINITY);
      for (int k = slice; k < w.chunks && !dead; k += width) {
        const Chunk c = chunk[beam * w.chunks + k];
        if (c.most > -INFINITY) sum += c.sum * exp((double)c.most - (double)most);
      }
      for (int k = 1; k < width; k *= 2) sum += __shfl_xor(sum, k, 64);
    }
    if (slice == 0) {
      s_most[beam] = most;
      s_offset[beam] = dead ? kNone : done(beam) ? (double)score : (double)score - log(sum);
    }
  }
  __syncthreads();
  // entry e, as loaded, as a candidate: false past its list's end
  auto candidate = [&](int e, uint2 x, Pair &p) {
    // (quotients by 1 are no multiples of 2^32 / 1)
    const bool near = e < kHeld && w.chunks < 1 << 16;
    const int list = a.count == 1 ? e : near ? (int)__umulhi(e, w.by_count) : e / a.count;
    const int b = w.chunks == 1 ? list : near ? (int)__umulhi(list, w.by_chunks) : list / w.chunks;
    p = Pair{s_offset[b], x.x, b, (int)x.y};
    if (p.c == kNone) return false;
    if (done(b)) {
      p.key = 0u;
      p.token = a.pad_token;
      return e == b * w.chunks * a.count;  // (lists of rows that are done hold anything)
    }
    if (x.x == 0) return false;
    p.c += (double)key_value(x.x) - (double)s_most[b];
    return p.c > kNone;
  };
  // A bound that `count` candidates reach and few others: bisection on the bits of
  // the candidates' order in float32 (rounding keeps it), until the rest fits easily.
  // (Loops, not unrolled code: with one workgroup per group, instruction fetch counts.)
  Pair p;
  auto order_of = [&](int e) { return candidate(e, lists[e], p) ? order_key((float)p.c) : 0u; };
  // candidates that reach the bound: in the waves before this one, and in all
  uint32_t least = 1;
  int first = 0, n = 0;
  auto counted = [&](const int (&reach)[kMergeWaves], int &before) {
    // lanes 0..15 of a row hold the waves' counts
    int v = lane < kMergeWaves ? reach[lane] : 0;
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    if (kMergeWaves > 4) {
      v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
      v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    }
    before = wave > 0 ? __builtin_amdgcn_readlane(v, wave - 1) : 0;
    return __builtin_amdgcn_readlane(v, kMergeWaves - 1);
  };
  {
    int reach = 0;
#pragma unroll 1
    for (int e0 = 0; e0 < entries; e0 += kMergeThreads) {
      const int e = e0 + threadIdx.x;
      const uint32_t key = e < entries ? order_of(e) : 0u;
      if (e < min(entries, kHeld)) s_order[e] = key;
      reach += __popcll(__ballot(key > 0));
    }
    if (lane == 0) s_reach[1][0][wave] = reach;
    __syncthreads();
    n = counted(s_reach[1][0], first);
  }
  uint32_t at = 0;
#pragma unroll 1
  for (int shift = 30, step = 0; shift >= 0 && n > a.count + 48; shift -= 2, ++step) {  // two bits at a time
    int reach[3] = {0, 0, 0};
#pragma unroll 1
    for (int e0 = 0; e0 < entries; e0 += kMergeThreads) {
      const int e = e0 + threadIdx.x;
      const uint32_t key = e >= entries ? 0u : e < kHeld ? s_order[e] : order_of(e);
#pragma unroll
      for (int d = 0; d < 3; ++d) reach[d] += __popcll(__ballot(key >= (at | (d + 1u) << shift)));
    }
    if (lane == 0)
#pragma unroll
      for (int d = 0; d < 3; ++d) s_reach[step & 1][d][wave] = reach[d];
    __syncthreads();
#pragma unroll
    for (int d = 2; d >= 0; --d) {
      int before;
      const int sum = counted(s_reach[step & 1][d], before);
      if (sum < a.count) continue;
      at |= (d + 1u) << shift;
      least = at;
      first = before;
      n = sum;
      break;
    }
  }
#pragma unroll 1
  for (int e0 = 0; e0 < entries && n <= kMergeList; e0 += kMergeThreads) {
    const int e = e0 + threadIdx.x;
    const bool in = e < entries && (e < kHeld ? s_order[e] : order_of(e)) >= least;
    const unsigned long long mask = __ballot(in);
    if (mask == 0) continue;
    if (in) {
      candidate(e, lists[e], p);
      const int to = first + lanes_before(mask);
      s_list[to] = p;
      s_c[to] = p.c;
      s_tie[to] = (uint64_t)p.beam << 32 | ~p.key;
    }
    first += __popcll(mask);
  }
  __syncthreads();
  auto before = [](const Pair &x, const Pair &y) {
    if (x.c != y.c) return x.c > y.c;
    if (x.beam != y.beam) return x.beam < y.beam;
    return x.key != y.key ? x.key > y.key : x.token < y.token;
  };
  auto put = [&](int rank, const Pair &p) {
    a.out_scores[out + rank] = (float)p.c;
    a.parents[out + rank] = p.beam;
    a.tokens[out + rank] = p.token;
  };
  if (n > kMergeList) {
    // more than LDS holds (then there are `count` of them): one after another
    Pair last{(double)INFINITY, 0u, 0, 0};
    for (int rank = 0; rank < a.count; ++rank) {
      Pair best{kNone, 0u, INT32_MAX, 0};
      for (int e = threadIdx.x; e < entries; e += kMergeThreads)
        if (candidate(e, lists[e], p) && before(last, p) && before(p, best)) best = p;
      for (int k = 1; k < 64; k *= 2) {
        Pair other;
        other.c = __shfl_xor(best.c, k, 64);
        other.key = __shfl_xor(best.key, k, 64);
        other.beam = __shfl_xor(best.beam, k, 64);
        other.token = __shfl_xor(best.token, k, 64);
        if (before(other, best)) best = other;
      }
      __syncthreads();
      if (lane == 0) s_best[wave] = best;
      __syncthreads();
      for (int k = 0; k < kMergeWaves; ++k)
        if (before(s_best[k], best)) best = s_best[k];
      last = best;
      if (threadIdx.x == 0) put(rank, best);
    }
    return;
  }
  // ranks, by four lanes a candidate
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += kMergeThreads / 4) {
    const int i = i0 + (int)threadIdx.x / 4;
    const Pair pair = s_list[min(i, n - 1)];
    const uint64_t tie = (uint64_t)pair.beam << 32 | ~pair.key;
    int rank = 0;
#pragma unroll 4
    for (int k = threadIdx.x % 4; k < n; k += 4) {
      const double c = s_c[k];
      const uint64_t t = s_tie[k];
      const int token = s_list[k].token;
      rank += c > pair.c || (c == pair.c && (t < tie || (t == tie && token < pair.token)));
    }
    rank = sum4(rank);
    if (i < n && threadIdx.x % 4 == 0 && rank < a.count) put(rank, pair);
  }
  if (threadIdx.x == 0 && n < a.count) {
    // the lowest pairs that are no candidates
    int at = n;
    for (int64_t f = 0; at < a.count; ++f) {
      const int b = (int)(f / a.vocab), t = (int)(f % a.vocab);
      bool taken = false;
      for (int k = 0; k < n; ++k) taken = taken || (s_list[k].beam == b && s_list[k].token == t);
      if (!taken) put(at++, Pair{kNone, 0u, b, t});
    }
  }
}

// Vectors per thread: 4 (chunks of 8192 logits), or 8 where the grid is large anyhow
// and many lists of a group are to be merged: fewer lists against fewer waves that hide
// loads, which float32's 32 bytes a vector need more.  Both launches by 8 over by 4, 16,384
// to 152,064 logits, 64 to 1,024 rows, 1 to 32 selected, grids of 1,024 chunks or more
// (median, a tenth below and above):
//   candidates of a group   up to 511           512 to 8191         from 8192 on
//   bfloat16                1.02 (0.93, 1.08)   0.97 (0.90, 1.06)   0.84 (0.60, 0.91)
//   float32                 1.05 (0.95, 1.23)   1.04 (0.94, 1.23)   0.96 (0.67, 1.11)
// and 1.02, 1.01 for smaller grids.
int chunk_vectors(int kind, int groups, int beams, int vocab, int count) {
  const int64_t chunks = (vocab + 8191) / 8192;
  return groups * beams * chunks >= 1024 && beams * chunks * count >= (kind == 2 ? 8192 : 512) ? 8 : 4;
}

template <int V>
void start_chunks(hipStream_t stream, const BeamArgs &a, const BeamParts &w) {
  const dim3 grid((unsigned)((int64_t)a.groups * a.beams * w.chunks));
  if (a.kind == 0) hipLaunchKernelGGL((beam_chunk_kernel<0, V>), grid, dim3(kThreads), 0, stream, a, w);
  else if (a.kind == 1) hipLaunchKernelGGL((beam_chunk_kernel<1, V>), grid, dim3(kThreads), 0, stream, a, w);
  else hipLaunchKernelGGL((beam_chunk_kernel<2, V>), grid, dim3(kThreads), 0, stream, a, w);
}

}  // namespace

int64_t beam_workspace(int groups, int beams, int vocab, int count) {
  return BeamParts(groups, beams, vocab, count, 4).total;  // (chunks of 16384 need less)
}

hipError_t launch_beam(hipStream_t stream, const BeamArgs &a) {
  const int vectors = chunk_vectors(a.kind, a.groups, a.beams, a.vocab, a.count);
  const BeamParts w(a.groups, a.beams, a.vocab, a.count, vectors);
  if (vectors == 8) start_chunks<8>(stream, a, w);
  else start_chunks<4>(stream, a, w);
  // us by 256 and by 1024 threads: 128 candidates of a group 7.4 and 8.5, 512 10.1 and
  // 10.2, 2048 18.9 and 11.4
  if (a.beams * w.chunks * a.count <= 1024)
    hipLaunchKernelGGL(beam_merge_kernel<256>, dim3(a.groups), dim3(256), 0, stream, a, w);
  else
    hipLaunchKernelGGL(beam_merge_kernel<1024>, dim3(a.groups), dim3(1024), 0, stream, a, w);
  return hipGetLastError();
}

}  // namespace pkv
