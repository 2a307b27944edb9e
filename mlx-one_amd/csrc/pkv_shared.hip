// pkv_shared.hip -- attention of a batch whose sequences share prefixes, over paged KV.
//
// A group's sequences hold the same first tokens.  Attention over them is one product
// for the group's query rows together; over each sequence's own tokens one per
// sequence; the parts of a row are joined by their log-sum-exps:
//   M = max m_i,  o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// so a prefix is read once per 32 of the group's query rows per KV head (16 beyond head dim
// 128) instead of once per sequence.
//
// Every workgroup first lays out the call's work from the lengths on the device: the
// prefix of a (group, KV head, block of rows) and the own tokens of a (sequence, KV
// head) are segments of 16-token tiles, cut into runs so that there are about as many
// runs as workgroups.  Its four waves take pairs of a run's tiles in turn:
//   S^T = K.Q^T      v_mfma_f32_16x16x32, one tile: lane (row, jj) holds tokens 4jj + r
//   O^T += V^T.P^T   v_mfma_f32_16x16x32, the pair's 32 tokens
// K and V go from the pages straight to operand registers, codes as float16 (one rounding of
// 2^-11 where scale and bias are applied, as the output's, or better), queries of quantized
// pages as float16 scaled by a power of two per row, which is exact for what their scores
// keep.  Scores, maxima, sums and parts are float32.  Weights are rounded to the operand type
// (bfloat16 pages: as the sum of two), and summed as they enter the product.
//
// A token past a sequence's end or on an unmapped page is absent; one that a row may not see
// yet changes nothing for it, not even where it is not finite.
#include <algorithm>

#include "pkv_mfma.h"
#include "pkv_step.h"

namespace pkv {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTarget = 512;  // runs to aim at beyond one per segment: two for each of 256 CUs

// Workspace: [member][8] descriptors, then per run its rows' (m, l) and sums of V.
struct SharedParts {
  int rows, runs, segs;  // rows per run, most runs, most segments
  int64_t ml, acc, total;
  SharedParts(const Geo &g, int batch, int rows_per_seq, int groups) {
    rows = shared_rows(g.dp);
    const int64_t blocks = ((int64_t)batch * rows_per_seq + rows - 1) / rows + std::min(groups, batch);
    segs = (int)(g.hk * (blocks + batch));
    runs = segs + kTarget;
    ml = (int64_t)batch * 32;
    acc = ml + (int64_t)runs * rows * 8;
    total = acc + (int64_t)runs * rows * g.dp * 4;
  }
};

struct SharedWork {
  int most;    // runs that there is room for
  int32_t *desc;
  float *ml, *acc;
};

// The call's work, laid out in LDS.
struct SharedPlan {
  int group_first[kMaxShared + 1];  // first member
  int group_tiles[kMaxShared];      // shared tiles
  int group_run[kMaxShared + 1];    // first run
  int own_run[kMaxShared + 1];      // a member's first run, counted behind the groups'
  int reduce[2 * kWaves];
  int long_run, own_long;           // tiles per run
};

__device__ __forceinline__ int seq_length(const SharedArgs &a, int b) {
  return (int)min((int64_t)max(a.seq_lens[b], 0), (int64_t)a.max_pages * a.g.page);
}
__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + PKV_TILE - 1) / PKV_TILE; }

__device__ __forceinline__ int64_t block_sum(SharedPlan &p, int64_t v, int tid) {
  // (two halves: every sum is below 2^46)
  const int lo = wave_sum((int)(v & 0x7FFFFF)), hi = wave_sum((int)(v >> 23));
  __syncthreads();
  if ((tid & 63) == 63) {
    p.reduce[2 * (tid >> 6)] = lo;
    p.reduce[2 * (tid >> 6) + 1] = hi;
  }
  __syncthreads();
  int64_t s = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += (int64_t)p.reduce[2 * w] + ((int64_t)p.reduce[2 * w + 1] << 23);
  return s;
}

// In-place exclusive sums of v[0..n), v[n] = the total.
__device__ __forceinline__ void block_scan(SharedPlan &p, int *v, int n, int tid) {
  int carry = 0;
  for (int base = 0; base < n; base += kThreads) {
    const int i = base + tid;
    const int x = i < n ? v[i] : 0;
    const int incl = wave_scan_incl(x, 0);
    __syncthreads();
    if ((tid & 63) == 63) p.reduce[tid >> 6] = incl;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < (tid >> 6)) before += p.reduce[w];
      carry += p.reduce[w];
    }
    if (i < n) v[i] = before + incl - x;
  }
  if (tid == 0) v[n] = carry;
  __syncthreads();
}

// The last i with v[i] <= x, 0 <= i < n (v[0] <= x).
__device__ __forceinline__ int last_at_most(const int *v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int row_blocks(const SharedArgs &a, const SharedPlan &p, int g, int per) {
  return (max(0, p.group_first[g + 1] - p.group_first[g]) * a.rows + per - 1) / per;
}

__device__ void lay_out(const SharedArgs &a, const SharedWork &w, SharedPlan &p, int per, int tid) {
  for (int g = tid; g <= a.groups; g += kThreads) p.group_first[g] = min(max(a.group_starts[g], 0), a.count);
  __syncthreads();
  int64_t shared = 0, own = 0;
  for (int g = tid; g < a.groups; g += kThreads) {
    const int first = p.group_first[g], n = p.group_first[g + 1] - first;
    int tiles = 0;
    if (n > 1) {  // (one sequence shares nothing)
      const int b = a.members[first];
      if (b >= 0 && b < a.batch) tiles = max(0, min(a.prefix_lens[g], seq_length(a, b))) / PKV_TILE;
    }
    p.group_tiles[g] = tiles;
    shared += (int64_t)tiles * row_blocks(a, p, g, per) * a.g.hk;
  }
  __syncthreads();
  const int last = p.group_first[a.groups];
  for (int j = tid; j < a.count; j += kThreads) {
    int tiles = 0;
    if (j >= p.group_first[0] && j < last) {
      const int b = a.members[j];
      if (b >= 0 && b < a.batch)
        tiles = max(0, tiles_of(seq_length(a, b)) - p.group_tiles[last_at_most(p.group_first, a.groups, j)]);
    }
    p.own_run[j] = tiles;
    own += (int64_t)tiles * a.g.hk;
  }
  shared = block_sum(p, shared, tid);
  own = block_sum(p, own, tid);
  // a shared tile's rows are many: it counts twice
  const int64_t cost = (2 * shared + own + kTarget - 1) / kTarget;
  const int step = 2 * kWaves;
  const int long_run = (int)((cost / 2 + step) / step * step), own_long = (int)((cost + step) / step * step);
  __syncthreads();
  for (int g = tid; g < a.groups; g += kThreads)
    p.group_run[g] = row_blocks(a, p, g, per) * a.g.hk * ((p.group_tiles[g] + long_run - 1) / long_run);
  for (int j = tid; j < a.count; j += kThreads) p.own_run[j] = a.g.hk * ((p.own_run[j] + own_long - 1) / own_long);
  if (tid == 0) {
    p.long_run = long_run;
    p.own_long = own_long;
  }
  __syncthreads();
  block_scan(p, p.group_run, a.groups, tid);
  block_scan(p, p.own_run, a.count, tid);
}

// A zero accumulator in registers: an inline constant 0 as an MFMA's accumulator has
// given wrong results where its destination partly overlaps an operand.
__device__ __forceinline__ f4 register_zero() {
  f4 z = {0.0f, 0.0f, 0.0f, 0.0f};
  asm volatile("" : "+v"(z));
  return z;
}

__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

template <int BITS, int DP, int G, int FK>
struct SharedCfg : Cfg<BITS, DP, G, 1, FK, 1> {
  using Base = Cfg<BITS, DP, G, 1, FK, 1>;
  static constexpr bool F16 = Base::QUANT || FK == 1;  // operand type
  using T = typename std::conditional<F16, h8, b8>::type;
  using E = typename std::conditional<F16, _Float16, __bf16>::type;
  static constexpr uint16_t INF = F16 ? 0x7C00 : 0x7F80;
  static constexpr int PAGE_BITS = BITS, GROUP = G;
};

// One run of a segment: its tiles, rows and where they come from.
struct Run {
  int kh, t0, t1;      // tiles [t0, t1)
  int b;               // the sequence whose block table is read
  int L;               // its tokens
  int member, row0;    // first member of the rows, first row counted from it
  int rows;            // live rows
  int slot;
};

// A pair of tiles in flight.
template <typename C>
struct Pair {
  uint32_t k[2][C::LW], v[2][C::LW];
  uint32_t km[2][C::NG], vm[2][C::QUANT ? 4 * C::NG : 1];
};

template <typename C, int RB>
__device__ __forceinline__ void run_tiles(const SharedArgs &a, const SharedWork &w, const Run &run, int lane, int wave,
                                          float *s_acc, float (*s_ml)[shared_rows(64)][2]) {
  using T = typename C::T;
  using E = typename C::E;
  constexpr int KB = C::KB, NB = C::NB, NG = C::NG, DP = 32 * KB;
  const Geo &g = a.g;
  const int col = lane & 15, jj = lane >> 4;
  const int tpp = g.page / PKV_TILE;

  // ---- rows: operands, how far each sees
  T q[RB][KB];
  float mult[RB];
  int lim[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = run.row0 + rb * 16 + col;
    const bool there = rb * 16 + col < run.rows;
    const int member = run.member + (there ? r / a.rows : 0), in = there ? r % a.rows : 0;
    int b = a.members[member];
    const bool known = there && b >= 0 && b < a.batch;
    b = known ? b : 0;
    const int qi = in / a.gqa, h = run.kh * a.gqa + in % a.gqa;
    const int L = seq_length(a, b), width = a.widths ? a.widths[b] : a.nq;
    const int pos = a.q_pos ? a.q_pos[(int64_t)b * a.nq + qi] : a.seq_lens[b] - width + qi;
    lim[rb] = known && qi < width ? min(pos, L - 1) : -1;
    const uint16_t *src = a.q + (((int64_t)b * a.heads + h) * a.nq + qi) * g.dim;
    uint16_t raw[KB][8];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int d0 = 32 * kb + 8 * jj;
      if ((g.dim & 7) == 0 && ((uintptr_t)a.q & 15) == 0) {
        u4 x = {0, 0, 0, 0};
        if (lim[rb] >= 0 && d0 < g.dim) x = *(const u4 *)(src + d0);
        __builtin_memcpy(raw[kb], &x, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[kb][e] = lim[rb] >= 0 && d0 + e < g.dim ? src[d0 + e] : (uint16_t)0;
      }
    }
    mult[rb] = a.scale * kLog2e;
    if constexpr (!C::QUANT) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) __builtin_memcpy(&q[rb][kb], raw[kb], 16);
    } else {
      // float16 operands: a row's largest element to [2^7, 2^8)
      float most = 0.0f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(bits_to_float(raw[kb][e], g.float_kind)));
      most = xor32_max(xor16_max(most));
      const int shift = most > 0.0f && most < INFINITY ? 8 - __builtin_amdgcn_frexp_expf(most) : 0;
      mult[rb] = ldexpf(mult[rb], -shift);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[rb][kb][e] = (_Float16)ldexpf(bits_to_float(raw[kb][e], g.float_kind), shift);
    }
  }
  int least = 0x7FFFFFFF;  // every live row sees the tokens up to it
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) least = min(least, lim[rb] < 0 ? 0x7FFFFFFF : lim[rb]);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
  least = __builtin_amdgcn_readfirstlane(least);

  float m[RB], thr[RB];
  f4 O[RB][NB], sum[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m[rb] = 0.0f;
    thr[rb] = -INFINITY;
    sum[rb] = f4{0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < NB; ++n) O[rb][n] = f4{0, 0, 0, 0};
  }
  const f4 zero = register_zero();
  T ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (E)1.0f;

  // ---- the wave's pairs: tiles t0 + 2 (wave + 4 i), + 1.  Lane l keeps the page of its
  // tile l (of pair l / 2) among 32 pairs.
  const int pairs = (run.t1 - run.t0 + 1) / 2;
  int pages = -1;
  auto window = [&](int i0) __attribute__((always_inline)) {
    const int t = run.t0 + 2 * (wave + kWaves * (i0 + lane / 2)) + (lane & 1);
    pages = t < run.t1 ? a.table[(int64_t)run.b * a.max_pages + t / tpp] : -1;
    if (pages >= a.num_pages) pages = -1;
  };
  Pair<C> next;
  int next_there = 0;
  auto fetch = [&](int i) __attribute__((always_inline)) {
    next_there = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int id = __builtin_amdgcn_readlane(pages, 2 * (i & 31) + s);
      if (id >= 0) next_there |= 1 << s;
      const int t = run.t0 + 2 * (wave + kWaves * i) + s;
      const uint8_t *head = a.pool + (int64_t)max(id, 0) * g.page_bytes + (int64_t)run.kh * g.head_bytes;
      const int tip = t % tpp;
      load_payload<C>(next.k[s], head + tip * g.tile_bytes, lane);
      load_payload<C>(next.v[s], head + g.v_offset + tip * g.tile_bytes, lane);
      if constexpr (C::QUANT) {
        const uint32_t *km = (const uint32_t *)(head + g.kmeta_offset) + (tip * PKV_TILE + col) * NG;
#pragma unroll
        for (int x = 0; x < NG; ++x) next.km[s][x] = km[x];
        const u4 *vm = (const u4 *)(head + g.vmeta_offset + (tip * PKV_TILE + 4 * jj) * NG * 4);
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const u4 y = vm[x];
          next.vm[s][4 * x] = y.x; next.vm[s][4 * x + 1] = y.y; next.vm[s][4 * x + 2] = y.z; next.vm[s][4 * x + 3] = y.w;
        }
      }
    }
  };
  if (wave < pairs) {
    window(0);
    fetch(0);
  }
  for (int i = 0; wave + kWaves * i < pairs; ++i) {
    Pair<C> p = next;
    const int there = next_there;
    if (wave + kWaves * (i + 1) < pairs) {
      if (((i + 1) & 31) == 0) window(i + 1);
      fetch(i + 1);
    }
    const int tok0 = (run.t0 + 2 * (wave + kWaves * i)) * PKV_TILE;  // the pair's first token
    const bool masked = there != 3 || tok0 + 2 * PKV_TILE - 1 > least;
    if (masked) {
      // absent tokens hold zeros
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const bool here = there >> s & 1;
        const int t = tok0 + s * PKV_TILE;
        if constexpr (C::QUANT) {
          const bool kt = here && t + col < run.L;
#pragma unroll
          for (int x = 0; x < NG; ++x) p.km[s][x] = kt ? p.km[s][x] : 0u;
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < NG; ++x) p.vm[s][e * NG + x] = here && t + 4 * jj + e < run.L ? p.vm[s][e * NG + x] : 0u;
        } else {
          const uint32_t kmask = here && t + col < run.L ? 0xFFFFFFFFu : 0u;
          uint32_t vmask[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            vmask[e] = (here && t + 4 * jj + 2 * e < run.L ? 0xFFFFu : 0u) |
                       (here && t + 4 * jj + 2 * e + 1 < run.L ? 0xFFFF0000u : 0u);
#pragma unroll
          for (int x = 0; x < C::LW; ++x) {
            p.k[s][x] &= kmask;
            p.v[s][x] &= vmask[x & 1];
          }
        }
      }
    }

    // S^T = K.Q^T
    f4 S[2][RB];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) S[s][rb] = zero;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        T k;
        if constexpr (C::QUANT) {
          const h2 sb = __builtin_bit_cast(h2, p.km[s][32 * kb / C::GROUP]);
          const h8 c = Conv<C::PAGE_BITS>::kop(p.k[s], kb) - (h8)(_Float16)1024.0f;
          k = __builtin_elementwise_fma(c, (h8)sb.x, (h8)sb.y);
        } else {
          k = __builtin_bit_cast(T, u4{p.k[s][4 * kb], p.k[s][4 * kb + 1], p.k[s][4 * kb + 2], p.k[s][4 * kb + 3]});
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) S[s][rb] = mma(k, q[rb][kb], S[s][rb]);
      }

    // softmax: a lane's 8 tokens of its row
    float x[RB][8];
    float mx[RB];
    bool need = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[rb][e] = __builtin_fmaf(S[e >> 2][rb][e & 3], mult[rb], -m[rb]);
      if (masked) {
        const int sees = lim[rb] - tok0 - 4 * jj;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool vis = (there >> (e >> 2) & 1) && PKV_TILE * (e >> 2) + (e & 3) <= sees;
          x[rb][e] = vis ? x[rb][e] : -INFINITY;
        }
      }
      mx[rb] = x[rb][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx[rb] = __builtin_elementwise_maximum(mx[rb], x[rb][e]);
      need |= mx[rb] > thr[rb];
    }
    if (__any(need)) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float up = xor32_max(xor16_max(mx[rb]));
        const bool moves = up > thr[rb];
        const float by = moves ? up : 0.0f;
        const float alpha = !moves ? 1.0f : thr[rb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-up);
        m[rb] += by;
        thr[rb] = moves ? kTau : thr[rb];
        sum[rb] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[rb][e] -= by;
#pragma unroll
        for (int n = 0; n < NB; ++n) O[rb][n] *= alpha;
      }
    }
    constexpr bool SPLIT = !C::F16;  // bfloat16 weights as the sum of two
    T P[RB], low[SPLIT ? RB : 1];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f(x[rb][e]);
        P[rb][e] = (E)y;
        if constexpr (SPLIT) low[rb][e] = (E)(y - (float)P[rb][e]);
      }
      sum[rb] = mma(ones, P[rb], sum[rb]);
      if constexpr (SPLIT) sum[rb] = mma(ones, low[rb], sum[rb]);
    }

    // O^T += V^T.P^T
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      T v;
      if constexpr (C::QUANT) {
        constexpr int per = C::GROUP / 16;
        h4 half[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          h4 sc, bi;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const h2 sb = __builtin_bit_cast(h2, p.vm[s][e * NG + n / per]);
            sc[e] = sb.x;
            bi[e] = sb.y;
          }
          half[s] = __builtin_elementwise_fma(Conv<C::PAGE_BITS>::vop(p.v[s], n) - (h4)(_Float16)1024.0f, sc, bi);
        }
        v = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        v = __builtin_bit_cast(T, u4{p.v[0][2 * n], p.v[0][2 * n + 1], p.v[1][2 * n], p.v[1][2 * n + 1]});
      }
      bool odd = false;
      if (masked) {
        const u4 bits = __builtin_bit_cast(u4, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (bits[e] & 0x7FFFu) >= C::INF || (bits[e] >> 16 & 0x7FFFu) >= C::INF;
      }
      if (!__any(odd)) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          O[rb][n] = mma(v, P[rb], O[rb][n]);
          if constexpr (SPLIT) O[rb][n] = mma(v, low[rb], O[rb][n]);
        }
      } else {
        // infinities and NaN: their products with a hidden token's zero weight must not be
        // NaN.  The finite values go through the product; of the others, kind by kind,
        // the tokens that a row sees are counted by one.
        uint16_t bits[8];
        __builtin_memcpy(bits, &v, 16);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const int sees = lim[rb] - tok0 - 4 * jj;
          T part, seen;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            part[e] = (bits[e] & 0x7FFF) >= C::INF ? (E)0.0f : v[e];
            seen[e] = PKV_TILE * (e >> 2) + (e & 3) <= sees ? (E)1.0f : (E)0.0f;
          }
          O[rb][n] = mma(part, P[rb], O[rb][n]);
          if constexpr (SPLIT) O[rb][n] = mma(part, low[rb], O[rb][n]);
#pragma unroll 1
          for (int kind = 0; kind < 3; ++kind) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const bool hit = kind == 2 ? (bits[e] & 0x7FFF) > C::INF : bits[e] == (C::INF | (kind << 15));
              part[e] = hit ? (E)1.0f : (E)0.0f;
            }
            const f4 count = mma(part, seen, zero);
            const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
            for (int e = 0; e < 4; ++e) O[rb][n][e] += count[e] > 0.0f ? what : 0.0f;
          }
        }
      }
    }
  }

  // ---- the four waves' parts joined, 16 rows at a time, and written
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
    if (jj == 0) {
      // (a row that sees nothing has none, whatever went through its lanes)
      s_ml[wave][rb * 16 + col][0] = thr[rb] == -INFINITY || lim[rb] < 0 ? -INFINITY : m[rb];
      s_ml[wave][rb * 16 + col][1] = sum[rb][0];
    }
  __syncthreads();
  constexpr int ROW = DP + 4;
  const int tid = wave * 64 + lane;
  float *acc = w.acc + (int64_t)run.slot * shared_rows(DP) * DP;
  float *ml = w.ml + (int64_t)run.slot * shared_rows(DP) * 2;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kWaves; ++x) top = fmaxf(top, s_ml[x][rb * 16 + col][0]);
    const float mine = s_ml[wave][rb * 16 + col][0];
    const float scale = mine == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mine - top);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      // (a wave without tokens has zeros, also where the maximum is NaN)
      const f4 y = mine == -INFINITY ? f4{0, 0, 0, 0} : O[rb][n] * scale;
      *(f4 *)(s_acc + (wave * 16 + col) * ROW + 16 * n + 4 * jj) = y;
    }
    __syncthreads();
    if (rb * 16 < run.rows) {
      for (int u = tid; u < 16 * DP / 4; u += kThreads) {
        const int row = u / (DP / 4), d = u % (DP / 4) * 4;
        f4 y = *(const f4 *)(s_acc + row * ROW + d);
#pragma unroll
        for (int x = 1; x < kWaves; ++x) y += *(const f4 *)(s_acc + (x * 16 + row) * ROW + d);
        if (rb * 16 + row < run.rows) *(f4 *)(acc + (int64_t)(rb * 16 + row) * DP + d) = y;
      }
      if (tid < 16 && rb * 16 + tid < run.rows) {
        float l = 0.0f, best = -INFINITY;
#pragma unroll
        for (int x = 0; x < kWaves; ++x) best = fmaxf(best, s_ml[x][rb * 16 + tid][0]);
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
          const float mx = s_ml[x][rb * 16 + tid][0];
          if (mx != -INFINITY) l += s_ml[x][rb * 16 + tid][1] * __builtin_amdgcn_exp2f(mx - best);
        }
        ml[2 * (rb * 16 + tid)] = best;
        ml[2 * (rb * 16 + tid) + 1] = l;
      }
    }
    __syncthreads();
  }
}

template <int BITS, int DP, int G, int FK>
__global__ __launch_bounds__(kThreads, 1) void shared_kernel(const SharedArgs a, const SharedWork w) {
  using C = SharedCfg<BITS, DP, G, FK>;
  constexpr int PER = shared_rows(DP);
  __shared__ SharedPlan plan;
  __shared__ __attribute__((aligned(16))) float s_acc[kWaves * 16 * (DP + 4)];
  __shared__ float s_ml[kWaves][shared_rows(64)][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  lay_out(a, w, plan, PER, tid);
  const int shared_runs = plan.group_run[a.groups], runs = shared_runs + plan.own_run[a.count];
  if (blockIdx.x == 0) {
    // where a member's parts are, for the merge: its group's first run and runs per
    // segment, its first row in the group; its own first run and runs per KV head
    for (int j = tid; j < a.count; j += kThreads) {
      const bool in = j >= plan.group_first[0] && j < plan.group_first[a.groups];
      const int g = in ? last_at_most(plan.group_first, a.groups, j) : 0;
      int32_t *d = w.desc + 8 * j;
      d[0] = plan.group_run[g];
      d[1] = in ? (plan.group_tiles[g] + plan.long_run - 1) / plan.long_run : 0;
      d[2] = (j - plan.group_first[g]) * a.rows;
      d[3] = shared_runs + plan.own_run[j];
      d[4] = (plan.own_run[j + 1] - plan.own_run[j]) / a.g.hk;
      d[5] = in;
    }
  }
  for (int u = blockIdx.x; u < runs && u < w.most; u += gridDim.x) {
    Run run;
    run.slot = u;
    if (u < shared_runs) {
      const int g = last_at_most(plan.group_run, a.groups, u);
      const int n = (plan.group_tiles[g] + plan.long_run - 1) / plan.long_run, at = u - plan.group_run[g];
      const int seg = at / n, c = at - seg * n, blk = seg / a.g.hk;
      run.kh = seg - blk * a.g.hk;
      run.t0 = c * plan.long_run;
      run.t1 = min(plan.group_tiles[g], run.t0 + plan.long_run);
      run.member = plan.group_first[g];
      run.row0 = blk * PER;
      run.rows = min(PER, (plan.group_first[g + 1] - run.member) * a.rows - run.row0);
    } else {
      const int j = last_at_most(plan.own_run, a.count, u - shared_runs);
      const int n = (plan.own_run[j + 1] - plan.own_run[j]) / a.g.hk, at = u - shared_runs - plan.own_run[j];
      const int g = last_at_most(plan.group_first, a.groups, j);
      run.kh = at / n;
      const int c = at - run.kh * n;
      run.t0 = plan.group_tiles[g] + c * plan.own_long;
      run.t1 = min(tiles_of(seq_length(a, a.members[j])), run.t0 + plan.own_long);
      run.member = j;
      run.row0 = 0;
      run.rows = a.rows;
    }
    run.b = __builtin_amdgcn_readfirstlane(a.members[run.member]);
    run.L = __builtin_amdgcn_readfirstlane(seq_length(a, run.b));
    run.kh = __builtin_amdgcn_readfirstlane(run.kh);
    run.t0 = __builtin_amdgcn_readfirstlane(run.t0);
    run.t1 = __builtin_amdgcn_readfirstlane(run.t1);
    run.member = __builtin_amdgcn_readfirstlane(run.member);
    run.row0 = __builtin_amdgcn_readfirstlane(run.row0);
    run.rows = __builtin_amdgcn_readfirstlane(run.rows);
    if (run.rows <= 16) run_tiles<C, 1>(a, w, run, lane, wave, s_acc, s_ml);
    else if constexpr (PER > 16) run_tiles<C, 2>(a, w, run, lane, wave, s_acc, s_ml);
  }
}

// One wave per (member, KV head, row): the row's parts joined.
template <int DP>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(const SharedArgs a, const SharedWork w) {
  constexpr int PER = shared_rows(DP), EPL = DP / 64;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  const int per_member = a.g.hk * a.rows;
  if (unit >= (int64_t)a.count * per_member) return;
  const int j = (int)(unit / per_member), in = (int)(unit % per_member), kh = in / a.rows, r = in % a.rows;
  const int b = a.members[j];
  const int32_t *d = w.desc + 8 * j;
  if (b < 0 || b >= a.batch || !d[5]) return;
  const int row = d[2] + r, shared = d[1], own = d[4];
  const int first = d[0] + (row / PER * a.g.hk + kh) * shared, own_first = d[3] + kh * own;
  const int n = shared + own;
  auto at = [&](int i) {  // the part's row among all runs' rows
    return i < shared ? (int64_t)(first + i) * PER + row % PER : (int64_t)(own_first + i - shared) * PER + r;
  };
  float top = -INFINITY;
  for (int i = lane; i < n; i += 64) top = __builtin_elementwise_maximum(top, w.ml[2 * at(i)]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o, 64));
  float l = 0.0f, acc[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) acc[e] = 0.0f;
  for (int i = 0; i < n; ++i) {
    const int64_t p = at(i);
    const float m = w.ml[2 * p];
    if (m == -INFINITY) continue;
    const float scale = __builtin_amdgcn_exp2f(m - top);
    l += w.ml[2 * p + 1] * scale;
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] += w.acc[p * DP + lane * EPL + e] * scale;
  }
  const float inv = top == -INFINITY ? 0.0f : 1.0f / l;
  const int qi = r / a.gqa, h = kh * a.gqa + r % a.gqa;
  uint16_t *o = a.out + (((int64_t)b * a.heads + h) * a.nq + qi) * a.g.dim;
#pragma unroll
  for (int e = 0; e < EPL; ++e)
    if (lane * EPL + e < a.g.dim) o[lane * EPL + e] = float_to_bits(acc[e] * inv, a.g.float_kind);
}

}  // namespace

int64_t shared_workspace(const Geo &g, int batch, int rows, int groups) {
  return SharedParts(g, batch, rows, groups).total;
}

hipError_t launch_shared_attention(hipStream_t stream, const SharedArgs &a) {
  if (a.count == 0 || a.groups == 0) return hipSuccess;
  const SharedParts parts(a.g, a.count, a.rows, a.groups);
  SharedWork w;
  w.most = parts.runs;
  w.desc = (int32_t *)a.workspace;
  w.ml = (float *)((uint8_t *)a.workspace + parts.ml);
  w.acc = (float *)((uint8_t *)a.workspace + parts.acc);
  const dim3 block(kThreads), grid((unsigned)parts.runs);
  hipError_t e = hipErrorInvalidValue;
#define PKV_SHARED(DP_, G_, BITS_, FK_)                                                     \
  if (a.g.dp == DP_ && a.g.bits == BITS_ && (BITS_ == 16 ? a.g.float_kind == FK_ : a.g.group == G_)) { \
    hipLaunchKernelGGL((shared_kernel<BITS_, DP_, G_, FK_>), grid, block, 0, stream, a, w); \
    e = hipGetLastError();                                                                  \
  }
#define PKV_SHARED_F(DP_) PKV_SHARED(DP_, 32, 16, 0) PKV_SHARED(DP_, 32, 16, 1)
#define PKV_SHARED_Q(DP_, G_) PKV_SHARED(DP_, G_, 4, 0) PKV_SHARED(DP_, G_, 8, 0)
  PKV_SHARED_F(64) PKV_SHARED_F(128) PKV_SHARED_F(256)
  PKV_SHARED_Q(64, 32) PKV_SHARED_Q(64, 64)
  PKV_SHARED_Q(128, 32) PKV_SHARED_Q(128, 64) PKV_SHARED_Q(128, 128)
  PKV_SHARED_Q(256, 32) PKV_SHARED_Q(256, 64) PKV_SHARED_Q(256, 128)
#undef PKV_SHARED_F
#undef PKV_SHARED_Q
#undef PKV_SHARED
  if (e != hipSuccess) return e;
  const dim3 rows((unsigned)(((int64_t)a.count * a.g.hk * a.rows + kWaves - 1) / kWaves));
  if (a.g.dp == 64) hipLaunchKernelGGL((shared_merge_kernel<64>), rows, block, 0, stream, a, w);
  else if (a.g.dp == 128) hipLaunchKernelGGL((shared_merge_kernel<128>), rows, block, 0, stream, a, w);
  else hipLaunchKernelGGL((shared_merge_kernel<256>), rows, block, 0, stream, a, w);
  return hipGetLastError();
}

}  // namespace pkv
