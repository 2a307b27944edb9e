// pkv_mass.hip -- the attention weight that a call's queries put on each cached token.
//
//   out[h, t] = old[h, t] + sum over query rows r of KV head h of softmax_t(scale * q_r . k_t)
//
// over the tokens t that row r sees (t <= its position, t < the sequence's
// length).  A row's weights need its log-sum-exp over all its tokens first, so K
// is gone through twice, or once and its scores kept:
//
//  * few rows (at most 16 per KV head: decode and verify steps): one pass over K
//    writes every score (float32) and the rows' (max, sum) of each run of tokens; a
//    second launch reads the scores back.  16 bytes per token written and read at up
//    to 4 rows, 32 at up to 8, 64 beyond, where K itself is 136 (8-bit, head_dim 128).
//  * more rows: a pass over K for the log-sum-exps, a launch that joins their
//    parts, and a second pass over K that sums the weights.
//
// Scores come from the matrix cores.  Quantized K enters as its exact codes (f16),
// queries as f16 with each row scaled by a power of two, so that its largest
// element lies in [2^7, 2^8): bfloat16 queries are exact then down to 2^-24 of that,
// and what is lost below is smaller than the float32 accumulator's own rounding.  A
// group's scale is applied to its accumulator in float32 and its bias to the sum of
// the row's elements in the group, so a score is a float32 sum of exact products.
#include <algorithm>

#include "pkv_cache_ops.h"
#include "pkv_mfma.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kFewRows = 16;
constexpr float kLog2e = 1.4426950408889634f;

// ---- sequences, rows, units ---------------------------------------------------------

// The tokens of sequence b that count, and the tokens its row qi sees.
__device__ __forceinline__ int mass_len(const MassArgs &a, int b) {
  const int64_t most = min((int64_t)a.max_pages * a.g.page, a.width);
  return (int)min((int64_t)a.seq_lens[b], most);
}
__device__ __forceinline__ int row_sees(const MassArgs &a, int b, int qi, int L) {
  const int w = a.widths ? a.widths[b] : a.nq;
  if (qi >= w) return 0;
  const int pos = a.q_pos ? a.q_pos[(int64_t)b * a.nq + qi] : a.seq_lens[b] - w + qi;
  return max(0, pos >= L ? L : pos + 1);
}

// The units of a launch: parts of `size` tokens of every sequence, for each KV
// head; a workgroup walks unit blockIdx.x, + gridDim.x, ...  Lane l of every wave
// keeps the running count of parts of sequence base + l.
struct Units {
  int base, carry, incl, len;
  int b, kh, part, L;

  __device__ __forceinline__ void load(const MassArgs &a, int size, int lane) {
    len = base + lane < a.batch ? max(0, mass_len(a, base + lane)) : 0;
    incl = carry + wave_scan_incl((len + size - 1) / size, lane);
  }
  __device__ __forceinline__ void start(const MassArgs &a, int size, int lane) {
    base = carry = 0;
    load(a, size, lane);
  }
  // The whole wave calls, with rising units.  False past the last one.
  __device__ __forceinline__ bool find(const MassArgs &a, int size, int64_t unit, int lane) {
    const int64_t u = unit / a.g.hk;
    kh = (int)(unit % a.g.hk);
    for (;;) {
      const unsigned long long hit = __ballot(incl > u);
      if (hit) {
        const int f = __ffsll((long long)hit) - 1;
        L = __builtin_amdgcn_readlane(len, f);
        b = base + f;
        part = (int)u - (__builtin_amdgcn_readlane(incl, f) - (L + size - 1) / size);
        return true;
      }
      if (base + 64 >= a.batch) return false;
      carry = __builtin_amdgcn_readlane(incl, 63);
      base += 64;
      load(a, size, lane);
    }
  }
};

// The same units in the order (sequence, KV head, part), shared out as equal runs of
// consecutive ones over the workgroups: a run's units of one (sequence, KV head) share
// their query operands and their running (max, sum).
struct Runs {
  int total;             // units of the launch (fewer than 2^31)
  int each, more;        // units per run, and one more in the first `more` runs
  int b, kh, part, L;    // where the run stands
  int parts;             // of sequence b

  // The units of the sequences before b, in parts of one KV head.
  static __device__ __forceinline__ int parts_before(const MassArgs &a, int size, int lane, int b) {
    int sum = 0;
    for (int base = 0; base < b; base += 64) {
      const int n = base + lane < b ? (max(0, mass_len(a, base + lane)) + size - 1) / size : 0;
      sum += wave_sum(n);
    }
    return sum;
  }
  __device__ __forceinline__ void share(int units, int grid) {
    total = units;
    each = total / grid;
    more = total - each * grid;
  }
  // First unit of workgroup w, and the workgroup of unit u.
  __device__ __forceinline__ int first(int w) const { return w * each + min(w, more); }
  __device__ __forceinline__ int owner(int u) const {
    const int longer = more * (each + 1);
    return u < longer ? u / (each + 1) : more + (u - longer) / each;
  }
  __device__ __forceinline__ void set(const MassArgs &a, int size, int to) {
    b = to;
    L = mass_len(a, b);
    parts = (max(0, L) + size - 1) / size;
  }
  // Stands at unit u < total.
  __device__ __forceinline__ void seek(const MassArgs &a, int size, int lane, int u) {
    int carry = 0;
    for (int base = 0;; base += 64) {
      const int n = base + lane < a.batch ? (max(0, mass_len(a, base + lane)) + size - 1) / size : 0;
      const int incl = wave_scan_incl(n, lane);
      const unsigned long long hit = __ballot((carry + incl) * a.g.hk > u);
      if (hit || base + 64 >= a.batch) {
        const int f = hit ? __ffsll((long long)hit) - 1 : 0;
        parts = __builtin_amdgcn_readlane(n, f);
        const int r = u - (carry + __builtin_amdgcn_readlane(incl, f) - parts) * a.g.hk;
        b = base + f;
        L = mass_len(a, b);
        kh = r / max(parts, 1);
        part = r - kh * parts;
        return;
      }
      carry += __builtin_amdgcn_readlane(incl, 63);
    }
  }
  // The next unit (there is one); true where it is of another (sequence, KV head).
  __device__ __forceinline__ bool next(const MassArgs &a, int size) {
    if (++part < parts) return false;
    part = 0;
    if (++kh < a.g.hk) return true;
    kh = 0;
    do set(a, size, b + 1);
    while (parts == 0);
    return true;
  }
};

// ---- tiles and query rows -------------------------------------------------------------

template <int BITS, int DP, int G, int FK>
struct MassCfg : Cfg<BITS, DP, G, 1, FK, 1> {
  using Base = Cfg<BITS, DP, G, 1, FK, 1>;
  static constexpr int PAGE_BITS = BITS;
  static constexpr int OPS = BITS == 16 ? FK : 1;  // operand type: f16 for codes
  using KT = typename FloatOps<OPS>::KT;
  static constexpr int GB = Base::QUANT ? G / 32 : Base::KB;  // 32-element blocks per accumulator
};

// A zero accumulator in registers: an inline constant 0 as an MFMA's accumulator has
// given wrong results where its destination partly overlaps an operand.
__device__ __forceinline__ f4 register_zero() {
  f4 z = {0.0f, 0.0f, 0.0f, 0.0f};
  asm volatile("" : "+v"(z));
  return z;
}

// Page ids of the N tiles from token t0 of sequence b: lane l's for tile l % N.
template <int N>
__device__ __forceinline__ int tile_page(const MassArgs &a, int b, int t0, int L, int lane) {
  const int t = t0 + (lane % N) * PKV_TILE;
  if (t >= L) return -1;
  const int id = a.table[(int64_t)b * a.max_pages + t / a.g.page];
  return id >= 0 && id < a.num_pages ? id : -1;
}

// A lane's K operands of a tile: codes as exact f16, or the float elements.
template <typename C>
__device__ __forceinline__ typename C::KT k_operand(const uint32_t (&w)[C::LW], int kb) {
  if constexpr (C::QUANT) {
    const h8 biased = Conv<C::PAGE_BITS>::kop(w, kb);  // 1024 + code
    return biased - (h8)(_Float16)1024.0f;
  } else {
    return __builtin_bit_cast(typename C::KT, u4{w[4 * kb], w[4 * kb + 1], w[4 * kb + 2], w[4 * kb + 3]});
  }
}

// One query row's elements d = 32 kb + 8 jj + e as operands (zeros without a row or
// past the head dim), its multiplier (of a raw score, to log2 units) and its sums
// per group.  The whole wave calls: lanes l, l ^ 16, l ^ 32 share a row.
template <typename C>
__device__ __forceinline__ void query_operands(const MassArgs &a, int b, int kh, int row, int jj,
                                               typename C::KT (&op)[C::KB], float &mult, float (&qs)[C::NG]) {
  const bool there = row < a.rows;
  const int qi = there ? row / a.gqa : 0, h = kh * a.gqa + (there ? row % a.gqa : 0);
  const uint16_t *src = a.q + (((int64_t)b * a.heads + h) * a.nq + qi) * a.g.dim;
  uint16_t raw[C::KB][8];
#pragma unroll
  for (int kb = 0; kb < C::KB; ++kb) {
    const int d0 = 32 * kb + 8 * jj;
    if ((a.g.dim & 7) == 0 && ((uintptr_t)a.q & 15) == 0) {
      u4 x = {0, 0, 0, 0};
      if (there && d0 < a.g.dim) x = *(const u4 *)(src + d0);
      __builtin_memcpy(raw[kb], &x, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[kb][e] = there && d0 + e < a.g.dim ? src[d0 + e] : (uint16_t)0;
    }
  }
  // a multiplier of at least 0: the scale's sign goes to the elements
  const uint16_t sign = a.scale < 0.0f ? 0x8000u : 0u;
  mult = fabsf(a.scale) * kLog2e;
#pragma unroll
  for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
    for (int e = 0; e < 8; ++e) raw[kb][e] ^= sign;
  if constexpr (!C::QUANT) {
#pragma unroll
    for (int kb = 0; kb < C::KB; ++kb) __builtin_memcpy(&op[kb], raw[kb], 16);
    qs[0] = 0.0f;
  } else {
    const int fk = a.g.float_kind;
    float most = 0.0f;
#pragma unroll
    for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(bits_to_float(raw[kb][e], fk)));
    most = xor32_max(xor16_max(most));
    const int shift = most > 0.0f && most < INFINITY ? 8 - __builtin_amdgcn_frexp_expf(most) : 0;
    mult = ldexpf(mult, -shift);
#pragma unroll
    for (int g = 0; g < C::NG; ++g) qs[g] = 0.0f;
#pragma unroll
    for (int kb = 0; kb < C::KB; ++kb)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const _Float16 x = (_Float16)ldexpf(bits_to_float(raw[kb][e], fk), shift);
        op[kb][e] = x;
        qs[kb / C::GB] += (float)x;
      }
#pragma unroll
    for (int g = 0; g < C::NG; ++g) qs[g] = xor32_add(xor16_add(qs[g]));
  }
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// (m, l) with another pair of the same row; an empty one is (-inf, 0).
__device__ __forceinline__ void join(float &m, float &l, float m2, float l2) {
  const float n = fmaxf(m, m2), z = n == -INFINITY ? 0.0f : n;
  l = l * exp2_fast(m - z) + l2 * exp2_fast(m2 - z);
  m = n;
}

// ---- few rows: scores kept --------------------------------------------------------------

constexpr int kPart = 256;  // tokens per unit: four tiles per wave
constexpr int kTiles = kPart / PKV_TILE / kWaves;

// Rows by fours, as the kernels are built: 1, 2 or 4.
__host__ __device__ inline int quads(int rows) { return rows > 8 ? 4 : rows > 4 ? 2 : 1; }

// Workspace: [scores: segment][quad][tokens][4] f32, [segment][k][16] (m, l) of the
// k-th workgroup that had units of the segment (k < its parts).
struct FewParts {
  int64_t tokens, parts, scores, total;
  int grid;  // workgroups of the first launch
  __host__ __device__ FewParts(int64_t segs, int rows, int64_t cap) {
    tokens = (cap + kPart - 1) / kPart * kPart;
    parts = tokens / kPart;
    scores = segs * quads(rows) * tokens * 16;
    total = scores + segs * parts * kFewRows * 8;
    grid = 0;
  }
};

// S = Q K^T with query row 4 r + jj in row 4 jj + r of the 16x16 tile: its four
// rows per lane are then the lane's registers r, and a call of at most 4 rows has
// one score per lane and tile, a call of 8 two.  Memory-bound: 32 sequences of 4.6K
// tokens in the mean, 8 KV heads, 8-bit pages, read 160 MB and write 19 in 38.5 us
// (4.6 TB/s; 31 us without the stores).  Runs of units against strided ones 42.5 us;
// four waves per SIMD (128 registers) against three 37.4 and 43.9.
template <typename C, int NR>
__global__ __launch_bounds__(kThreads, C::KB > 4 ? 2 : NR > 2 ? 3 : 4) void mass_scores_kernel(const MassArgs a, const FewParts w) {
  __shared__ float s_ml[kWaves][NR * 4][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, jj = lane >> 4, col = lane & 15;
  const Geo &g = a.g;
  const f4 zero = register_zero();
  Runs run;
  run.share(Runs::parts_before(a, kPart, lane, a.batch) * g.hk, gridDim.x);
  int unit = run.first(blockIdx.x);
  const int end = run.first(blockIdx.x + 1);
  if (unit >= end) return;
  run.seek(a, kPart, lane, unit);
  auto pages = [&]() { return tile_page<kTiles>(a, run.b, run.part * kPart + wave * (kTiles * PKV_TILE), run.L, lane); };
  int ids = pages();
  bool fresh = true;
  typename C::KT q[C::KB];
  float qs[NR][C::NG], mult[NR], m[NR], l[NR];
  int sees[NR];
  for (; unit < end; ++unit) {
    const int b = run.b, kh = run.kh, part = run.part;
    const int t0 = part * kPart + wave * (kTiles * PKV_TILE);
    const int64_t seg = (int64_t)b * g.hk + kh;
    uint32_t kw[kTiles][C::LW], mw[kTiles][C::NG];
    bool there[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int id = __builtin_amdgcn_readlane(ids, i);
      there[i] = id >= 0;
      const int slot = (t0 + i * PKV_TILE) % g.page;
      const uint8_t *head = a.pool + (int64_t)max(id, 0) * g.page_bytes + (int64_t)kh * g.head_bytes;
#pragma unroll
      for (int k = 0; k < C::LW; ++k) kw[i][k] = 0;
#pragma unroll
      for (int k = 0; k < C::NG; ++k) mw[i][k] = 0;
      if (there[i]) {
        load_payload<C, true>(kw[i], head + (slot / PKV_TILE) * g.tile_bytes, lane);
        if constexpr (C::QUANT) {
          const uint32_t *meta = (const uint32_t *)(head + g.kmeta_offset) + (slot + col) * C::NG;
#pragma unroll
          for (int k = 0; k < C::NG; ++k) mw[i][k] = meta[k];
        }
      }
    }
    if (fresh) {
      float qs_row[C::NG], mult_row;
      query_operands<C>(a, b, kh, 4 * (col & 3) + (col >> 2), jj, q, mult_row, qs_row);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const int row = 4 * r + jj;
        sees[r] = row < a.rows ? row_sees(a, b, row / a.gqa, run.L) : 0;
        mult[r] = __shfl(mult_row, 4 * jj + r, 64);
#pragma unroll
        for (int k = 0; k < C::NG; ++k) qs[r][k] = __shfl(qs_row[k], 4 * jj + r, 64);
        m[r] = -INFINITY;
        l[r] = 0.0f;
      }
    }
    // the next unit's page ids are under way while this one's tiles are used
    const bool last = unit + 1 >= end;
    fresh = last || run.next(a, kPart);
    if (!last) ids = pages();
    float s[NR][kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      f4 acc[C::NG];
#pragma unroll
      for (int k = 0; k < C::NG; ++k) acc[k] = zero;
#pragma unroll
      for (int kb = 0; kb < C::KB; ++kb)
        acc[kb / C::GB] = FloatOps<C::OPS>::qk(q[kb], k_operand<C>(kw[i], kb), acc[kb / C::GB]);
      const int t = t0 + i * PKV_TILE + col;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float x = 0.0f;
        if constexpr (C::QUANT) {
#pragma unroll
          for (int k = 0; k < C::NG; ++k) x = fmaf(f16_bits_to_f32(mw[i][k] >> 16), qs[r][k], x);
#pragma unroll
          for (int k = 0; k < C::NG; ++k) x = fmaf(f16_bits_to_f32(mw[i][k]), acc[k][r], x);
        } else {
          x = acc[0][r];
        }
        s[r][i] = there[i] && t < sees[r] ? x * mult[r] : -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float *to = (float *)a.workspace + ((seg * quads(a.rows) + r) * w.tokens + t0 + col) * 4 + jj;
      float n = m[r];
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        n = fmaxf(n, s[r][i]);
        to[i * PKV_TILE * 4] = s[r][i];  // (the row of parts is whole: nothing past it is written)
      }
      const float z = n == -INFINITY ? 0.0f : n;
      l[r] = m[r] == -INFINITY ? l[r] : l[r] * exp2_fast(m[r] - z);  // (0, or NaN, stays)
#pragma unroll
      for (int i = 0; i < kTiles; ++i) l[r] += exp2_fast(s[r][i] - z);
      m[r] = n;
    }
    if (!fresh) continue;
    // the end of the segment's units here: its rows' (m, l) over the lanes and waves
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float mm = m[r];
      mm = fmaxf(mm, row_xchg<0xB1>(mm));
      mm = fmaxf(mm, row_xchg<0x4E>(mm));
      mm = fmaxf(mm, row_xchg<0x141>(mm));
      mm = fmaxf(mm, row_xchg<0x140>(mm));
      float ll = m[r] == -INFINITY ? l[r] : l[r] * exp2_fast(m[r] - mm);
      ll += row_xchg<0xB1>(ll);
      ll += row_xchg<0x4E>(ll);
      ll += row_xchg<0x141>(ll);
      ll += row_xchg<0x140>(ll);
      if (col == 0) {
        s_ml[wave][4 * r + jj][0] = mm;
        s_ml[wave][4 * r + jj][1] = ll;
      }
    }
    __syncthreads();
    if (threadIdx.x < NR * 4) {
      float mm = -INFINITY, ll = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) join(mm, ll, s_ml[k][threadIdx.x][0], s_ml[k][threadIdx.x][1]);
      // of the segment's workgroups, this is the one after those before its first unit here
      const int owner = run.owner(unit - part);
      float *to = (float *)((char *)a.workspace + w.scores) +
                  ((seg * w.parts + (blockIdx.x - owner)) * kFewRows + threadIdx.x) * 2;
      to[0] = mm;
      to[1] = ll;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ void store_mass(const MassArgs &a, int b, int kh, int row, int t, float sum) {
  const int64_t at = ((int64_t)row * a.g.hk + kh) * a.width + t;
  const bool old = a.mass && (!a.counted || t < a.counted[b]);
  a.out[at] = (old ? a.mass[at] : 0.0f) + sum;
}
__device__ __forceinline__ int mass_row(const MassArgs &a, int b) {
  const int row = a.out_rows ? a.out_rows[b] : b;
  return row >= 0 && row < a.mass_rows ? row : -1;
}

// The second launch: 19 MB of scores and 9 of sums in 7.7 us at the size above.
constexpr int kSumPart = 1024;  // tokens per unit

template <int NR>
__global__ __launch_bounds__(kThreads) void mass_weights_kernel(const MassArgs a, const FewParts w) {
  const int lane = threadIdx.x & 63;
  auto parts_of = [](int len) { return (len + kPart - 1) / kPart; };
  Units u;
  u.start(a, kSumPart, lane);
  // the first launch's units: of the sequences before u.base, and of all
  int before = 0, total = wave_sum(parts_of(u.len));
  if (a.batch > 64) total = Runs::parts_before(a, kPart, lane, a.batch);
  Runs run;
  run.share(total * a.g.hk, w.grid);
  for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
    const int base = u.base;
    if (!u.find(a, kSumPart, unit, lane)) return;
    if (u.base != base) before = Runs::parts_before(a, kPart, lane, u.base);  // (also where the row is skipped)
    const int row = mass_row(a, u.b);
    if (row < 0) continue;
    const int64_t seg = (int64_t)u.b * a.g.hk + u.kh;
    // everything is requested before any of it is used
    const float *scores = (const float *)a.workspace + seg * quads(a.rows) * w.tokens * 4;
    float4 s[NR][4];
    float old[4];
    const int counted = !a.mass ? 0 : a.counted ? a.counted[u.b] : u.L;
    const int64_t to = ((int64_t)row * a.g.hk + u.kh) * a.width;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = u.part * kSumPart + i * kThreads + threadIdx.x;
      const int at = min(t, u.L - 1);
#pragma unroll
      for (int r = 0; r < NR; ++r) s[r][i] = *(const float4 *)(scores + ((int64_t)r * w.tokens + at) * 4);
      old[i] = t < min(counted, u.L) ? a.mass[to + t] : 0.0f;
    }
    // the rows' log-sum-exps from the workgroups' (m, l): lane 16 k + r the k-th's of row r
    float lse;
    {
      const int n1 = parts_of(u.len), f = u.b - u.base, parts = __builtin_amdgcn_readlane(n1, f);
      const int upto = __builtin_amdgcn_readlane(wave_scan_incl(n1, lane), f);
      const int first = (before + upto - parts) * a.g.hk + u.kh * parts;
      const int n = run.owner(first + parts - 1) - run.owner(first) + 1;
      const float2 *ml = (const float2 *)((const char *)a.workspace + w.scores) + seg * w.parts * kFewRows;
      float m = -INFINITY, l = 0.0f;
      for (int k = lane / 16; k < n; k += 4)
        if (lane % 16 < NR * 4) {
          const float2 x = ml[k * kFewRows + lane % 16];
          join(m, l, x.x, x.y);
        }
#pragma unroll
      for (int k = 16; k < 64; k *= 2) join(m, l, __shfl_xor(m, k, 64), __shfl_xor(l, k, 64));
      lse = l == 0.0f ? INFINITY : m + __builtin_amdgcn_logf(l);  // a row that sees nothing weighs nothing
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = u.part * kSumPart + i * kThreads + threadIdx.x;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float x[4] = {s[r][i].x, s[r][i].y, s[r][i].z, s[r][i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {  // a token that the row does not see adds 0 also where the row's sum is NaN
          const float of_row = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lse), 4 * r + k));
          sum += x[k] == -INFINITY ? 0.0f : exp2_fast(x[k] - of_row);
        }
      }
      if (t < u.L) a.out[to + t] = old[i] + sum;
    }
  }
}

// ---- many rows: K twice -----------------------------------------------------------------
//
// Rows in blocks of 16.  A workgroup of eight waves holds a unit's K tiles in
// registers, two per wave, and goes through the row blocks, which it stages in LDS
// few at a time, the next ones under way while these are used.  Bound by the issue of
// vector instructions (group scales, exponentials at quarter rate) and matrix ones (80
// cycles per 16x16 tile at head_dim 128), which add up.  256 rows per KV head, 4
// sequences of 28K tokens, 4 KV heads, 4-bit: 75 us for the (max, sum), 63 for the
// weights (the biases by float32 matrix instructions: 80 and 70).

constexpr int kManyWaves = 8, kManyThreads = 64 * kManyWaves;
constexpr int kManyTiles = 2;  // per wave
constexpr int kManyPart = kManyWaves * kManyTiles * PKV_TILE;

// A block's record: query operands [KB][64 lanes] 16 bytes; then [16 rows] f32 each:
// multiplier, log-sum-exp, tokens seen (int), and a last one: the most and the least
// that its rows see; then, for quantized pages, the operands [64 lanes] 16 bytes of
// the groups' sums.
template <typename C>
struct Record {
  static constexpr int MULT = C::KB * 1024, LSE = MULT + 64, SEES = LSE + 64, RANGE = SEES + 64, SUMS = RANGE + 64,
                       BYTES = SUMS + (C::QUANT ? 1024 : 0);
  static constexpr int STAGE = C::KB > 4 ? 2 : 4;  // records per stage
};

// Workspace: records [segment][block], parts [segment][part][rows] (m, l).
struct ManyParts {
  int64_t blocks, parts, record, ml, total;
  __host__ __device__ ManyParts(int64_t segs, int rows, int64_t cap, int dp, int ng) {
    blocks = rows > 0 ? (rows + 15) / 16 : 1;  // (no rows: one block that sees nothing)
    parts = (cap + kManyPart - 1) / kManyPart;
    record = dp * 32 + 4 * 64 + (ng > 0 ? 1024 : 0);
    ml = segs * blocks * record + 4 * record;  // (a stage's last copy reads past the last record)
    total = ml + segs * parts * blocks * 16 * 8;
  }
};

template <typename C>
__global__ __launch_bounds__(kThreads) void mass_prepare_kernel(const MassArgs a, const ManyParts w) {
  using R = Record<C>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, jj = lane >> 4, col = lane & 15;
  const int64_t n = (int64_t)blockIdx.x * kWaves + wave;  // (segment, block)
  if (n >= w.blocks * a.batch * a.g.hk) return;
  const int64_t seg = n / w.blocks;
  const int block = (int)(n % w.blocks), b = (int)(seg / a.g.hk), kh = (int)(seg % a.g.hk);
  const int row = block * 16 + col, L = max(0, mass_len(a, b));
  typename C::KT q[C::KB];
  float qs[C::NG], mult;
  query_operands<C>(a, b, kh, row, jj, q, mult, qs);
  const int sees = row < a.rows ? row_sees(a, b, row / a.gqa, L) : 0;
  if (sees == 0) {  // a row that is not live may hold anything
#pragma unroll
    for (int kb = 0; kb < C::KB; ++kb) q[kb] = typename C::KT{};
#pragma unroll
    for (int k = 0; k < C::NG; ++k) qs[k] = 0.0f;
    mult = 0.0f;
  }
  char *record = (char *)a.workspace + n * R::BYTES;
#pragma unroll
  for (int kb = 0; kb < C::KB; ++kb) *(u4 *)(record + (kb * 64 + lane) * 16) = __builtin_bit_cast(u4, q[kb]);
  int most = sees, least = sees > 0 ? sees : INT32_MAX;  // (rows that see nothing weigh nothing in any case)
#pragma unroll
  for (int k = 1; k < 16; k *= 2) {
    most = max(most, __shfl_xor(most, k, 64));
    least = min(least, __shfl_xor(least, k, 64));
  }
  if (jj == 0) {
    ((float *)(record + R::MULT))[col] = mult;
    ((float *)(record + R::LSE))[col] = 0.0f;
    ((int *)(record + R::SEES))[col] = sees;
    ((int *)(record + R::RANGE))[col] = col == 0 ? most : col == 1 ? least : 0;
  }
  if constexpr (C::QUANT) {
    // a group's sum (at most 2^15, float32) as three float16 that add up to it: their
    // products with the bias are exact, and one matrix instruction takes eight groups
    h8 sums = {};
#pragma unroll
    for (int k = 0; k < C::NG; ++k) {
      const _Float16 hi = (_Float16)qs[k], mid = (_Float16)(qs[k] - (float)hi);
      const _Float16 lo = (_Float16)(qs[k] - (float)hi - (float)mid);
      const bool finite = fabsf(qs[k]) < INFINITY;
      if (k / 2 == jj) {
        sums[k % 2 * 3] = hi;
        sums[k % 2 * 3 + 1] = finite ? mid : (_Float16)0.0f;
        sums[k % 2 * 3 + 2] = finite ? lo : (_Float16)0.0f;
      }
    }
    *(u4 *)(record + R::SUMS + lane * 16) = __builtin_bit_cast(u4, sums);
  }
}

// The pass over a launch's units.  SUM false: the (max, sum) of each row over the
// unit's tokens, from S^T = K Q^T (a lane has one query row, its column, and four
// tokens of each tile).  SUM true: the weights summed over the rows, from S = Q K^T
// (a lane has one token of each tile and four rows).
template <typename C, bool SUM>
__global__ __launch_bounds__(kManyThreads, C::KB > 4 ? 2 : 4) void mass_pass_kernel(const MassArgs a, const ManyParts w) {
  using R = Record<C>;
  constexpr int N = kManyTiles, S = R::STAGE, kUnits = (S * R::BYTES + 15) / 16;
  constexpr int kCopies = (kUnits + kManyThreads - 1) / kManyThreads;
  __shared__ __align__(16) char s_rec[2][S * R::BYTES];
  __shared__ float2 s_ml[SUM ? 1 : 2][SUM ? 1 : kManyWaves][SUM ? 1 : S * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), jj = lane >> 4,
            col = lane & 15;
  const Geo &g = a.g;
  const f4 zero = register_zero();
  Units u;
  u.start(a, kManyPart, lane);
  for (int64_t unit = blockIdx.x; u.find(a, kManyPart, unit, lane); unit += gridDim.x) {
    const int first = u.part * kManyPart, t0 = first + wave * (N * PKV_TILE);
    const int out_row = SUM ? mass_row(a, u.b) : 0;
    if (SUM && out_row < 0) continue;
    const int64_t seg = (int64_t)u.b * g.hk + u.kh;
    const char *records = (const char *)a.workspace + seg * w.blocks * R::BYTES;
    // the records of S blocks from b0 on straight to LDS, 16 bytes per lane (what lies
    // past the last block is in the workspace and not used)
    auto fetch = [&](int64_t b0, int buffer) {
#pragma unroll
      for (int k = 0; k < kCopies; ++k) {
        const int unit0 = (wave + k * kManyWaves) * 64;
        if (unit0 < kUnits) {
          const char *from = records + b0 * R::BYTES + (int64_t)(unit0 + lane) * 16;
          if (unit0 + lane < kUnits)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)from,
                                             (__attribute__((address_space(3))) uint32_t *)(s_rec[buffer] + unit0 * 16),
                                             16, 0, 0);
        }
      }
    };
    fetch(0, 0);

    // the wave's tiles
    typename C::KT kt[N][C::KB];
    bool there[N], all = true;
    float scale[N][SUM ? 1 : 4][C::NG];  // of the lane's token, or its four
    h8 bias[N];  // operand: thrice that of groups 2 jj and 2 jj + 1 of token col
    const int ids = tile_page<N>(a, u.b, t0, u.L, lane);
    uint32_t kw[N][C::LW];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = __builtin_amdgcn_readlane(ids, i);
      there[i] = id >= 0;
      all = all && there[i];
      const int slot = (t0 + i * PKV_TILE) % g.page;
      const uint8_t *head = a.pool + (int64_t)max(id, 0) * g.page_bytes + (int64_t)u.kh * g.head_bytes;
      const uint8_t *meta = head + g.kmeta_offset + (int64_t)slot * C::NG * 4;
#pragma unroll
      for (int j = 0; j < C::LW; ++j) kw[i][j] = 0;
      if (there[i]) load_payload<C>(kw[i], head + (slot / PKV_TILE) * g.tile_bytes, lane);
      if constexpr (C::QUANT) {
        uint32_t b0 = 0, b1 = 0;
        if (there[i] && 2 * jj < C::NG) b0 = ((const uint32_t *)meta)[col * C::NG + 2 * jj] >> 16;
        if (there[i] && 2 * jj + 1 < C::NG) b1 = ((const uint32_t *)meta)[col * C::NG + 2 * jj + 1] >> 16;
        bias[i] = __builtin_bit_cast(h8, u4{b0 | b0 << 16, b0 | b1 << 16, b1 | b1 << 16, 0u});
        if constexpr (SUM) {
#pragma unroll
          for (int j = 0; j < C::NG; ++j)
            scale[i][0][j] = there[i] ? f16_bits_to_f32(((const uint32_t *)meta)[col * C::NG + j]) : 0.0f;
        } else {
          uint32_t mw[4 * C::NG];
#pragma unroll
          for (int k = 0; k < C::NG; ++k) {
            u4 x = {0, 0, 0, 0};
            if (there[i]) x = ((const u4 *)meta)[jj * C::NG + k];
            mw[4 * k] = x.x; mw[4 * k + 1] = x.y; mw[4 * k + 2] = x.z; mw[4 * k + 3] = x.w;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < C::NG; ++j) scale[i][SUM ? 0 : r][j] = f16_bits_to_f32(mw[r * C::NG + j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int kb = 0; kb < C::KB; ++kb) kt[i][kb] = k_operand<C>(kw[i], kb);
    float sum[N];
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] = 0.0f;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the records have arrived
    __syncthreads();

    int buffer = 0;
    for (int64_t b0 = 0; b0 < w.blocks; b0 += S, buffer ^= 1) {
      const bool more = b0 + S < w.blocks;
      if (more) fetch(b0 + S, buffer ^ 1);
      const int nb = (int)min((int64_t)S, w.blocks - b0);
      for (int k = 0; k < nb; ++k) {
        const char *rec = s_rec[buffer] + k * R::BYTES;
        const int most = __builtin_amdgcn_readfirstlane(((const int *)(rec + R::RANGE))[0]);
        const int least = __builtin_amdgcn_readfirstlane(((const int *)(rec + R::RANGE))[1]);
        if (most <= t0) {  // no row sees any of the wave's tokens
          if (!SUM && jj == 0) s_ml[buffer & (SUM ? 0 : 1)][SUM ? 0 : wave][SUM ? 0 : k * 16 + col] = float2{-INFINITY, 0.0f};
          continue;
        }
        typename C::KT q[C::KB];
#pragma unroll
        for (int kb = 0; kb < C::KB; ++kb) q[kb] = __builtin_bit_cast(typename C::KT, *(const u4 *)(rec + (kb * 64 + lane) * 16));
        h8 qs = {};
        if constexpr (C::QUANT) qs = __builtin_bit_cast(h8, *(const u4 *)(rec + R::SUMS + lane * 16));
        float x[N][4];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          f4 acc[C::NG];
          f4 base = zero;  // the biases' part
          if constexpr (C::QUANT) base = SUM ? FloatOps<1>::qk(qs, bias[i], zero) : FloatOps<1>::qk(bias[i], qs, zero);
#pragma unroll
          for (int j = 0; j < C::NG; ++j) acc[j] = zero;
#pragma unroll
          for (int kb = 0; kb < C::KB; ++kb)
            acc[kb / C::GB] = SUM ? FloatOps<C::OPS>::qk(q[kb], kt[i][kb], acc[kb / C::GB])
                                  : FloatOps<C::OPS>::qk(kt[i][kb], q[kb], acc[kb / C::GB]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[i][r] = C::QUANT ? base[r] : acc[0][r];
            if constexpr (C::QUANT)
#pragma unroll
              for (int j = 0; j < C::NG; ++j)
                x[i][r] = fmaf(scale[i][SUM ? 0 : r][j], acc[j][r], x[i][r]);
          }
        }
        const bool masked = !all || least < t0 + N * PKV_TILE;  // not every row sees every token
        if constexpr (SUM) {
          const f4 mult = *(const f4 *)(rec + R::MULT + jj * 16), lse = *(const f4 *)(rec + R::LSE + jj * 16);
          f4 p[N];
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) p[i][r] = exp2_fast(fmaf(x[i][r], mult[r], -lse[r]));
          if (masked) {
            const int4 sees = *(const int4 *)(rec + R::SEES + jj * 16);
            const int see[4] = {sees.x, sees.y, sees.z, sees.w};
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (!there[i] || t0 + i * PKV_TILE + col >= see[r]) p[i][r] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < N; ++i) sum[i] += (p[i][0] + p[i][1]) + (p[i][2] + p[i][3]);
        } else {
          const float mult = ((const float *)(rec + R::MULT))[col];
          if (masked) {
            const int sees = ((const int *)(rec + R::SEES))[col];
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (!there[i] || t0 + i * PKV_TILE + 4 * jj + r >= sees) x[i][r] = -INFINITY;
          }
          // raw scores, one multiplier (not negative) for the row
          float m = -INFINITY, l = 0.0f;
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) m = fmaxf(m, x[i][r]);
          m = xor32_max(xor16_max(m));
          const float z = m == -INFINITY ? 0.0f : m * mult;
          if (!masked) {
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) l += exp2_fast(fmaf(x[i][r], mult, -z));
          } else {  // (-inf times a multiplier of 0 is no number)
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) l += x[i][r] == -INFINITY ? 0.0f : exp2_fast(fmaf(x[i][r], mult, -z));
          }
          l = xor32_add(xor16_add(l));
          if (jj == 0) s_ml[SUM ? 0 : buffer][SUM ? 0 : wave][SUM ? 0 : k * 16 + col] = float2{m == -INFINITY ? m : z, l};
        }
      }
      // the next records have arrived
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
      const int mine = (int)threadIdx.x - (int)(b0 / S % kManyWaves) * 64;  // another wave at each stage
      if (!SUM && mine >= 0 && mine < nb * 16) {
        // (these are written again two stages on, behind another barrier)
        float m = -INFINITY, l = 0.0f;
        float2 y[kManyWaves];
#pragma unroll
        for (int k = 0; k < kManyWaves; ++k) {
          y[k] = s_ml[SUM ? 0 : buffer][SUM ? 0 : k][SUM ? 0 : mine];
          m = fmaxf(m, y[k].x);
        }
        const float z = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int k = 0; k < kManyWaves; ++k) l += y[k].y * exp2_fast(y[k].x - z);
        ((float2 *)((char *)a.workspace + w.ml))[((seg * w.parts + u.part) * w.blocks + b0) * 16 + mine] = float2{m, l};
      }
    }
    if constexpr (SUM) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float total = xor32_add(xor16_add(sum[i]));
        const int t = t0 + i * PKV_TILE + col;
        if (jj == 0 && t < u.L) store_mass(a, u.b, u.kh, out_row, t, total);
      }
    }
    __syncthreads();  // the buffers and sums are used again
  }
}

// Each row's log-sum-exp from its parts: 16 rows of 16 lanes per workgroup.
__global__ __launch_bounds__(kThreads) void mass_join_kernel(const MassArgs a, const ManyParts w, int at_lse, int at_sees) {
  const int64_t rows = w.blocks * 16;
  const int64_t seg = blockIdx.x / w.blocks, block = blockIdx.x % w.blocks, row = block * 16 + threadIdx.x % 16;
  __shared__ float s_ml[2][16][17];
  const int parts = (max(0, mass_len(a, (int)(seg / a.g.hk))) + kManyPart - 1) / kManyPart, slice = threadIdx.x / 16;
  const float2 *ml = (const float2 *)((const char *)a.workspace + w.ml) + seg * w.parts * rows + row;
  float m = -INFINITY, l = 0.0f;
  for (int p = slice; p < parts; p += 16) {
    const float2 x = ml[p * rows];
    join(m, l, x.x, x.y);
  }
  s_ml[0][slice][threadIdx.x % 16] = m;
  s_ml[1][slice][threadIdx.x % 16] = l;
  __syncthreads();
  if (slice == 0) {
    for (int k = 1; k < 16; ++k) join(m, l, s_ml[0][k][threadIdx.x], s_ml[1][k][threadIdx.x]);
    char *record = (char *)a.workspace + (seg * w.blocks + block) * w.record;
    // a row that sees nothing weighs nothing
    const bool none = ((const int *)(record + at_sees))[threadIdx.x] == 0 || l == 0.0f;
    ((float *)(record + at_lse))[threadIdx.x] = none ? INFINITY : m + __builtin_amdgcn_logf(l);
  }
}

// ---- launches -----------------------------------------------------------------------------

// Scores are kept for up to 16 rows where they take no more than this (the size goes
// by the block table's width).  32 sequences of 1K..8K tokens, 8 KV heads, head_dim
// 128, kept against K read twice, us: 8-bit pages, 4 rows 46 and 134, 8 rows 55 and
// 133, 16 rows 79 and 134; 4-bit pages, 4 rows 38 and 120, 12 rows 60 and 122; bf16
// pages, 16 rows 100 and 136.  Past 16 rows the first kernel has no registers for them.
constexpr int64_t kMostScores = (int64_t)2 << 30;

bool keeps_scores(const Geo &g, int64_t segs, int rows, int64_t cap) {
  return rows <= kFewRows && FewParts(segs, rows, cap).scores <= kMostScores;
}

// Workgroups of a walk over `units` units: no more than stay resident.
int walkers(int64_t units) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(units, 8 * (int64_t)std::max(1, device_cus())));
}

// Workgroups that share out at most `units` units: as many as stay resident at the
// registers that the kernel needs (four of four waves per CU).
int runs(int64_t units) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(units, 4 * (int64_t)std::max(1, device_cus())));
}

template <typename C>
void launch(hipStream_t stream, const MassArgs &a, int64_t cap) {
  const int64_t segs = (int64_t)a.batch * a.g.hk;
  if (keeps_scores(a.g, segs, a.rows, cap)) {
    FewParts w(segs, a.rows, cap);
    w.grid = runs(segs * w.parts);
    const dim3 grid(w.grid), second(walkers(segs * ((cap + kSumPart - 1) / kSumPart)));
    if (quads(a.rows) == 1) {
      hipLaunchKernelGGL((mass_scores_kernel<C, 1>), grid, dim3(kThreads), 0, stream, a, w);
      hipLaunchKernelGGL((mass_weights_kernel<1>), second, dim3(kThreads), 0, stream, a, w);
    } else if (quads(a.rows) == 2) {
      hipLaunchKernelGGL((mass_scores_kernel<C, 2>), grid, dim3(kThreads), 0, stream, a, w);
      hipLaunchKernelGGL((mass_weights_kernel<2>), second, dim3(kThreads), 0, stream, a, w);
    } else {
      hipLaunchKernelGGL((mass_scores_kernel<C, 4>), grid, dim3(kThreads), 0, stream, a, w);
      hipLaunchKernelGGL((mass_weights_kernel<4>), second, dim3(kThreads), 0, stream, a, w);
    }
    return;
  }
  using R = Record<C>;
  const ManyParts w(segs, a.rows, cap, a.g.dp, a.g.ng);
  static_assert(R::BYTES == C::KB * 1024 + 4 * 64 + (C::QUANT ? 1024 : 0), "as ManyParts has it");
  const dim3 grid(walkers(segs * w.parts));
  const unsigned blocks = (unsigned)(segs * w.blocks);
  hipLaunchKernelGGL((mass_prepare_kernel<C>), dim3((blocks + kWaves - 1) / kWaves), dim3(kThreads), 0, stream, a, w);
  hipLaunchKernelGGL((mass_pass_kernel<C, false>), grid, dim3(kManyThreads), 0, stream, a, w);
  hipLaunchKernelGGL(mass_join_kernel, dim3(blocks), dim3(kThreads), 0, stream, a, w, R::LSE, R::SEES);
  hipLaunchKernelGGL((mass_pass_kernel<C, true>), grid, dim3(kManyThreads), 0, stream, a, w);
}

template <int BITS, int DP>
void launch_group(hipStream_t stream, const MassArgs &a, int64_t cap) {
  if (a.g.group == 32) return launch<MassCfg<BITS, DP, 32, 1>>(stream, a, cap);
  if (a.g.group == 64) return launch<MassCfg<BITS, DP, 64, 1>>(stream, a, cap);
  if constexpr (DP >= 128) launch<MassCfg<BITS, DP, 128, 1>>(stream, a, cap);
}

template <int BITS>
void launch_dim(hipStream_t stream, const MassArgs &a, int64_t cap) {
  if (a.g.dp == 64) launch_group<BITS, 64>(stream, a, cap);
  else if (a.g.dp == 128) launch_group<BITS, 128>(stream, a, cap);
  else launch_group<BITS, 256>(stream, a, cap);
}

template <int FK>
void launch_float(hipStream_t stream, const MassArgs &a, int64_t cap) {
  if (a.g.dp == 64) launch<MassCfg<16, 64, 32, FK>>(stream, a, cap);
  else if (a.g.dp == 128) launch<MassCfg<16, 128, 32, FK>>(stream, a, cap);
  else launch<MassCfg<16, 256, 32, FK>>(stream, a, cap);
}

}  // namespace

int64_t mass_workspace(const Geo &g, int batch, int rows, int max_pages) {
  const int64_t segs = (int64_t)batch * g.hk, cap = (int64_t)max_pages * g.page;
  if (keeps_scores(g, segs, rows, cap)) return FewParts(segs, rows, cap).total;
  return ManyParts(segs, rows, cap, g.dp, g.ng).total;
}

hipError_t launch_mass(hipStream_t stream, const MassArgs &a) {
  const int64_t cap = (int64_t)a.max_pages * a.g.page;  // as the workspace is sized, whatever the mass's width
  if (a.g.bits == 8) launch_dim<8>(stream, a, cap);
  else if (a.g.bits == 4) launch_dim<4>(stream, a, cap);
  else if (a.g.float_kind == 0) launch_float<0>(stream, a, cap);
  else launch_float<1>(stream, a, cap);
  return hipGetLastError();
}

}  // namespace pkv
