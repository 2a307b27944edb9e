// pkv_shared.hip -- attention of a batch whose sequences share prefixes, over paged KV.
//
// A group's sequences hold the same first tokens.  Attention over them is one product
// for the group's query rows together; over each sequence's own tokens one per
// sequence; the parts of a row are joined by their log-sum-exps:
//   M = max m_i,  o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i
// so a prefix is read once per 32 of the group's query rows per KV head (16 beyond head dim
// 128) instead of once per sequence.
//
// Every workgroup (up to 64 sequences every wave) first lays out the call's work from the
// lengths on the device: the prefix of a (group, KV head, block of rows) and the own tokens of
// a (sequence, KV head) are segments of 16-token tiles, cut into runs so that all are in flight together.  Its
// four waves take pairs of a run's tiles in turn:
//   S^T = K.Q^T      v_mfma_f32_16x16x32, one tile: lane (row, jj) holds tokens 4jj + r
//   O^T += V^T.P^T   v_mfma_f32_16x16x32, the pair's 32 tokens
// What bounds it are the instructions that turn codes into operands (a pair takes about 400, and
// 560 for two blocks of 16 rows), then the way from the lengths to the first tile, about 6 us.
// So two waves share a SIMD: one block of rows keeps the next pair in registers; two, which
// need those for sums, copy it to LDS.  (In registers at one wave per SIMD: 69 us for 32
// sequences behind 4096 tokens int8, 87 us for eight answers to each of four 24000-token documents
// int4, 47 us for five queries each of 16 sequences; now 32, 55 and 31 us, with the merge.)
//
// Quantized K enters as its codes (1024 + c, exact in float16; queries as float16, bfloat16 ones
// with each row scaled by a power of two), group scales and biases are applied to the float32
// scores:  s = sum_g scale_g (q_g . c'_g) + (bias_g - 1024 scale_g) sum(q_g).  Quantized V is
// rounded once to float16 (2^-11); a row that sees a value past float16's range, which pages can
// hold, is computed anew by the kernel that joins the parts (where all 1,024 rows of 4,160 tokens
// do: 560 us instead of 40).  Weights are rounded to the operand type, or, where that would show in
// the result (bfloat16 pages, float16 results of quantized ones), enter as the sum of two; they
// are summed as they enter.  (Float16 ones of less than 2^-21 of the largest have a fixed step of
// 2^-31 of that.)  Scores, maxima, sums and parts are float32.
//
// A token past a sequence's end or on an unmapped page is absent; one that a row may not see
// yet changes nothing for it, not even where it is not finite.  (An infinity that it sees may
// come out as NaN where weights are two operands.)
#include <algorithm>

#include "pkv_mfma.h"
#include "pkv_step.h"
#include "pkv_token.h"

namespace pkv {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
// Runs to aim at: two workgroups for each of 256 CUs.  A shared tile serves 32 rows, one of a
// sequence's own a few: costs of 3 and 2 (32 sequences behind 4096 tokens: 34 us; 5 and 3: 38; 2
// and 1: 40).
constexpr int kTarget = 512, kSharedCost = 3, kOwnCost = 2;

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
  int sequence[kMaxShared];         // a member's sequence, -1 for none
  int length[kMaxShared];           // its tokens
  int reduce[3 * kWaves];
  int long_run, own_long;           // tiles per run
};

__device__ __forceinline__ int seq_length(const SharedArgs &a, int b) {
  return (int)min((int64_t)max(a.seq_lens[b], 0), (int64_t)a.max_pages * a.g.page);
}
__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + PKV_TILE - 1) / PKV_TILE; }

// Runs of a segment, of about `most` tiles each.
__device__ __forceinline__ int runs_of(int tiles, int most) { return (tiles + most - 1) / most; }
// Tiles of each of n runs: whole turns of the waves' pairs.
__device__ __forceinline__ int run_length(int tiles, int n) {
  constexpr int turn = 2 * kWaves;
  return ((tiles + n - 1) / n + turn - 1) / turn * turn;
}

// Sums over the workgroup.
__device__ __forceinline__ void block_sum(SharedPlan &p, int64_t &v, int &x, int tid) {
  // (v in two halves: it is below 2^46)
  const int part[3] = {wave_sum((int)(v & 0x7FFFFF)), wave_sum((int)(v >> 23)), wave_sum(x)};
  __syncthreads();
  if ((tid & 63) == 63)
    for (int k = 0; k < 3; ++k) p.reduce[3 * (tid >> 6) + k] = part[k];
  __syncthreads();
  v = 0;
  x = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    v += (int64_t)p.reduce[3 * w] + ((int64_t)p.reduce[3 * w + 1] << 23);
    x += p.reduce[3 * w + 2];
  }
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

// The last i with v[i] <= x, 0 <= i < n (v[0] <= x; v does not fall).
__device__ __forceinline__ int last_at_most(const int *v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}
// The same, x alike for the wave.
__device__ __forceinline__ int last_at_most_uniform(const int *v, int n, int x, int lane) {
  int i = 0;
  while (i + 64 < n && __builtin_amdgcn_readfirstlane(v[i + 64]) <= x) i += 64;
  return i + __popcll(__ballot(i + lane < n && v[min(i + lane, n - 1)] <= x)) - 1;
}

__device__ __forceinline__ int row_blocks(const SharedArgs &a, const SharedPlan &p, int g, int per) {
  return (max(0, p.group_first[g + 1] - p.group_first[g]) * a.rows + per - 1) / per;
}

// The lengths of runs by the k-th allowance for the segments' ends.
__device__ __forceinline__ void run_lengths(int64_t cost, int segs, int own_cost, int k, int &long_run, int &own_long) {
  const float each = (float)cost / (float)max(kTarget - (int)((int64_t)segs * (k + 1) / kWaves), kTarget / 4);
  long_run = (int)fminf(each * (1.0f / kSharedCost), 1e9f) + 1;
  own_long = (int)fminf(each / (float)own_cost, 1e9f) + 1;
}

__device__ __forceinline__ void lay_out(const SharedArgs &a, SharedPlan &p, int per, int tid) {
  for (int g = tid; g <= a.groups; g += kThreads) p.group_first[g] = min(max(a.group_starts[g], 0), a.count);
  for (int g = tid; g < a.groups; g += kThreads) p.group_tiles[g] = a.prefix_lens[g];
  for (int j = tid; j < a.count; j += kThreads) {
    const int b = a.members[j];
    const bool known = b >= 0 && b < a.batch;
    p.sequence[j] = known ? b : -1;
    p.length[j] = p.own_run[j] = known ? seq_length(a, b) : 0;
  }
  __syncthreads();
  const int own_cost = a.rows > 16 ? kSharedCost : kOwnCost;  // (two blocks of rows)
  int64_t cost = 0;
  bool falls = false;
  for (int g = tid; g < a.groups; g += kThreads) {
    const int first = p.group_first[g], n = p.group_first[g + 1] - first;
    falls |= n < 0;
    // (one sequence shares nothing)
    const int tiles = n > 1 ? max(0, min(p.group_tiles[g], p.own_run[first])) / PKV_TILE : 0;
    p.group_tiles[g] = tiles;
    cost += kSharedCost * (int64_t)tiles * row_blocks(a, p, g, per) * a.g.hk;
  }
  if (__syncthreads_or(falls)) {  // groups that would overlap: none
    cost = 0;
    for (int g = tid; g <= a.groups; g += kThreads) p.group_first[g] = 0;
    for (int g = tid; g < a.groups; g += kThreads) p.group_tiles[g] = 0;
    __syncthreads();
  }
  const int last = p.group_first[a.groups];
  for (int j = tid; j < a.count; j += kThreads) {
    const bool in = j >= p.group_first[0] && j < last;
    const int tiles = in ? tiles_of(p.own_run[j]) - p.group_tiles[last_at_most(p.group_first, a.groups, j)] : 0;
    p.own_run[j] = max(0, tiles);
    cost += own_cost * (int64_t)p.own_run[j] * a.g.hk;
  }
  // Long enough runs that all of them are in flight together, as short as that allows: a
  // segment's length is rounded up to whole runs, so each wave tries another allowance.
  int segs = 0;
  for (int g = tid; g < a.groups; g += kThreads) segs += p.group_tiles[g] > 0 ? row_blocks(a, p, g, per) * a.g.hk : 0;
  for (int j = tid; j < a.count; j += kThreads) segs += p.own_run[j] > 0 ? a.g.hk : 0;
  block_sum(p, cost, segs, tid);
  int long_run, own_long, count = 0;
  run_lengths(cost, segs, own_cost, tid >> 6, long_run, own_long);
  for (int g = tid & 63; g < a.groups; g += 64) count += row_blocks(a, p, g, per) * runs_of(p.group_tiles[g], long_run);
  for (int j = tid & 63; j < a.count; j += 64) count += runs_of(p.own_run[j], own_long);
  count = wave_sum(count);
  __syncthreads();
  if ((tid & 63) == 63) p.reduce[tid >> 6] = count;
  __syncthreads();
  int k = 0;
  while (k < kWaves - 1 && (int64_t)p.reduce[k] * a.g.hk > kTarget) ++k;
  run_lengths(cost, segs, own_cost, k, long_run, own_long);
  for (int g = tid; g < a.groups; g += kThreads)
    p.group_run[g] = row_blocks(a, p, g, per) * a.g.hk * runs_of(p.group_tiles[g], long_run);
  for (int j = tid; j < a.count; j += kThreads) p.own_run[j] = a.g.hk * runs_of(p.own_run[j], own_long);
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
  // weights as 2^LIFT of themselves, the largest 2^(kTau + LIFT) then: float16's have fewer bits
  // below 2^-14
  static constexpr float LIFT = F16 ? 7.0f : 0.0f;
  static constexpr int PAGE_BITS = BITS, GROUP = G;
};

// Bytes of one side of a pair of tiles: payloads and metadata.
template <typename C>
constexpr int side_bytes() { return 2 * 256 * C::LW + (C::QUANT ? 2 * 64 * C::NG : 0); }

// Until at most N of the wave's requests to memory are under way; until LDS has been read.
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The lane, made anew: kept over the loop it goes to scratch memory, and reading it back there
// waits for the requests before.
__device__ __forceinline__ int lane_again() {
  uint32_t l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(l));
  return (int)l;
}

// One run of a segment: its tiles, rows and where they come from.
struct Run {
  int kh, t0, t1;      // tiles [t0, t1)
  int b;               // the sequence whose block table is read
  int L;               // its tokens
  int member, row0;    // first member of the rows, first row counted from it
  int rows;            // live rows
  int slot;
};

struct __attribute__((aligned(16))) TilePlace {
  int64_t head;
  int tip;
};

// A pair of tiles in flight: payloads, and the metadata of a lane's four tokens.
template <typename C>
struct Pair {
  uint32_t k[2][C::LW], v[2][C::LW];
  uint32_t km[2][C::MW], vm[2][C::MW];
};

template <typename C, int RB>
__device__ __forceinline__ void run_tiles(const SharedArgs &a, const SharedWork &w, const int *sequence,
                                          const int *length, const Run &run, int lane, int wave, TilePlace *where,
                                          uint8_t *lds, float (*s_ml)[shared_rows(64)][2]) {
  using T = typename C::T;
  using E = typename C::E;
  constexpr int KB = C::KB, NB = C::NB, NG = C::NG, DP = 32 * KB;
  constexpr int GB = C::QUANT ? C::GROUP / 32 : KB;  // 32-element blocks per accumulator
  const Geo &g = a.g;
  const int col = lane & 15, jj = lane >> 4;
  const int tpp = g.page / PKV_TILE;

  // ---- the wave's pairs: tiles t0 + 2 (wave + 4 i), + 1.  LDS keeps where 32 pairs' tiles
  // are: the tile in its page, -1 for none, and the page's head.
  constexpr int kTileBytes = 256 * C::LW;
  const int pairs = (run.t1 - run.t0 + 1) / 2;
  auto window = [&](int i0) __attribute__((always_inline)) {
    const int t = run.t0 + 2 * (wave + kWaves * (i0 + lane / 2)) + (lane & 1), page = t / tpp;
    int id = -1;
    if (t < run.t1) id = a.table[(int64_t)run.b * a.max_pages + page];
    const bool there = id >= 0 && id < a.num_pages;
    where[lane].head = (int64_t)(there ? id : 0) * g.page_bytes + (int64_t)run.kh * g.head_bytes;
    where[lane].tip = there ? t - page * tpp : -1;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  // A pair's K and V are requested a pair ahead: into registers of their own for one block of
  // rows; for two, whose accumulators take that room, into LDS, each side as soon as the pair
  // before has been read from there.
  constexpr bool STAGED = RB > 1;
  Pair<C> p, next;
  int next_there = 0;
  const uint8_t *heads[2];  // the requested pair's tiles
  int tips[2];
  auto locate = [&](int i) __attribute__((always_inline)) {
    next_there = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const TilePlace at = where[2 * (i & 31) + s];
      const int tip = __builtin_amdgcn_readfirstlane(at.tip);
      const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)at.head);
      const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(at.head >> 32));
      if (tip >= 0) next_there |= 1 << s;
      tips[s] = max(tip, 0);
      heads[s] = a.pool + (int64_t)((uint64_t)hi << 32 | lo);
    }
  };
  auto fetch = [&](Pair<C> &to) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      load_payload<C, true>(to.k[s], heads[s] + tips[s] * kTileBytes, lane);
      load_payload<C, true>(to.v[s], heads[s] + g.v_offset + tips[s] * kTileBytes, lane);
      if constexpr (C::QUANT) {
        load_meta<C, true>(to.km[s], heads[s] + g.kmeta_offset + tips[s] * (PKV_TILE * NG * 4) + 16 * NG * jj);
        load_meta<C, true>(to.vm[s], heads[s] + g.vmeta_offset + tips[s] * (PKV_TILE * NG * 4) + 16 * NG * jj);
      }
    }
  };
  // One side of a pair: two tiles' payloads, then two tiles' metadata.
  constexpr int kSide = side_bytes<C>(), kCopies = C::LW / 2 + (C::QUANT ? 1 : 0);
  uint8_t *const ring = lds + wave * 2 * kSide;
  auto stage = [&](int64_t payload, int64_t meta, uint8_t *to) __attribute__((always_inline)) {
    const int lane = lane_again();
#pragma unroll
    for (int c = 0; c < C::LW / 2; ++c) {
      if constexpr (kTileBytes >= 1024) {
        const int s = c * 1024 / kTileBytes;
        copy_to_lds(heads[s] + (payload + tips[s] * kTileBytes + c * 1024 % kTileBytes), lane * 16, to + c * 1024);
      } else {
        copy_to_lds(lane < 32 ? heads[0] + (payload + tips[0] * kTileBytes) + lane * 16
                              : heads[1] + (payload + tips[1] * kTileBytes) + (lane - 32) * 16, to + c * 1024);
      }
    }
    if constexpr (C::QUANT) {
      constexpr int per = 4 * NG;  // lanes for a tile's
      const uint8_t *from = lane < per ? heads[0] + (meta + tips[0] * (16 * per)) + lane * 16
                                       : heads[1] + (meta + tips[1] * (16 * per)) + (lane - per) * 16;
      if (lane < 2 * per) copy_to_lds(from, to + 2 * kTileBytes);
    }
  };
  auto stage_k = [&]() __attribute__((always_inline)) { stage(0, g.kmeta_offset, ring); };
  auto stage_v = [&]() __attribute__((always_inline)) { stage(g.v_offset, g.vmeta_offset, ring + kSide); };
  auto take = [&](const uint8_t *from, uint32_t (&words)[2][C::LW], uint32_t (&meta)[2][C::MW])
      __attribute__((always_inline)) {
    const int lane = lane_again(), jj = lane >> 4;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      load_payload<C, false>(words[s], from + s * kTileBytes, lane);
      if constexpr (C::QUANT) load_meta<C, false>(meta[s], from + 2 * kTileBytes + (s * 4 + jj) * (16 * NG));
    }
  };
  if (wave < pairs) window(0);

  // ---- rows: operands, how far each sees
  T q[RB][KB];  // (two blocks of rows: kept in LDS)
  float mult[RB], qs[RB][NG];
  int lim[RB];
  uint16_t raw[RB][KB][8];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = run.row0 + rb * 16 + col;
    const bool there = rb * 16 + col < run.rows;
    const int member = there ? r / a.rows : 0, in = there ? r - member * a.rows : 0;
    const int b = sequence[run.member + member];
    const int qi = in / a.gqa, h = run.kh * a.gqa + in - qi * a.gqa, at = max(b, 0);
    const int L = length[run.member + member];
    const int width = a.widths ? a.widths[at] : a.nq;
    const int pos = a.q_pos ? a.q_pos[(int64_t)at * a.nq + qi] : a.seq_lens[at] - width + qi;
    lim[rb] = there && b >= 0 && qi < width ? min(pos, L - 1) : -1;
    const uint16_t *src = a.q + (((int64_t)at * a.heads + h) * a.nq + qi) * g.dim;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int d0 = 32 * kb + 8 * jj;
      if ((g.dim & 7) == 0 && ((uintptr_t)a.q & 15) == 0) {
        u4 x = {0, 0, 0, 0};
        if (there && d0 < g.dim) x = *(const u4 *)(src + d0);
        __builtin_memcpy(raw[rb][kb], &x, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[rb][kb][e] = there && d0 + e < g.dim ? src[d0 + e] : (uint16_t)0;
      }
    }
  }
  if constexpr (STAGED) __syncthreads();  // (a plan's memory is taken)
  if (wave < pairs) {
    locate(0);
    if constexpr (STAGED) {
      stage_k();
      stage_v();
    } else {
      fetch(next);
    }
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    mult[rb] = a.scale * kLog2e;
    if constexpr (!C::QUANT) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) __builtin_memcpy(&q[rb][kb], raw[rb][kb], 16);
      qs[rb][0] = 0.0f;
    } else {
      if (g.float_kind == 1) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) __builtin_memcpy(&q[rb][kb], raw[rb][kb], 16);
      } else {
        // bfloat16 to float16: a row's largest element to [2^7, 2^8)
        typedef uint16_t us2 __attribute__((ext_vector_type(2)));
        us2 tops = {0, 0};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 8; e += 2)
            tops = __builtin_elementwise_max(tops, us2{raw[rb][kb][e], raw[rb][kb][e + 1]} & (uint16_t)0x7FFF);
        const float most = xor32_max(xor16_max(bits_to_float(max(tops.x, tops.y), 0)));
        const int shift = most > 0.0f && most < INFINITY ? min(8 - __builtin_amdgcn_frexp_expf(most), 126) : 0;
        mult[rb] = ldexpf(mult[rb], -shift);
        const float by = __int_as_float((127 + shift) << 23);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            // (exact down to float16's smallest step, 2^-31 of the row's largest)
            const auto two = __builtin_amdgcn_cvt_pkrtz(bits_to_float(raw[rb][kb][e], 0) * by,
                                                        bits_to_float(raw[rb][kb][e + 1], 0) * by);
            q[rb][kb][e] = (_Float16)two[0];
            q[rb][kb][e + 1] = (_Float16)two[1];
          }
      }
#pragma unroll
      for (int x = 0; x < NG; ++x) qs[rb][x] = 0.0f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          qs[rb][kb / GB] = __builtin_amdgcn_fdot2(h2{q[rb][kb][e], q[rb][kb][e + 1]},
                                                   h2{(_Float16)1.0f, (_Float16)1.0f}, qs[rb][kb / GB], false);
#pragma unroll
      for (int x = 0; x < NG; ++x) qs[rb][x] = xor32_add(xor16_add(qs[rb][x]));
    }
  }
  const uint32_t q_at = (uint32_t)lane * 8;  // operand (rb, kb): kept[(rb * KB + kb) * 512 + q_at]
  uint16_t *kept = (uint16_t *)(lds + kWaves * 2 * kSide);
  if constexpr (RB > 1) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      if (wave == rb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) *(T *)(kept + (rb * KB + kb) * 512 + q_at) = q[rb][kb];
    __syncthreads();
  }
  int least = 0x7FFFFFFF;  // every live row sees the tokens up to it
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) least = min(least, lim[rb] < 0 ? 0x7FFFFFFF : lim[rb]);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
  least = __builtin_amdgcn_readfirstlane(least);

  float m[RB], thr[RB];
  f4 O[RB][NB];
  float sum[RB];  // the lane's tokens'
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m[rb] = 0.0f;
    thr[rb] = -INFINITY;
    sum[rb] = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n) O[rb][n] = f4{0, 0, 0, 0};
  }
  const f4 zero = register_zero();
  // whether weights enter as the sum of two operands
  const bool split = C::QUANT ? g.float_kind == 1 : !C::F16;

  // One pair.  CAREFUL: tokens of it are absent, or hidden from some row.
  auto pair = [&](int i, auto careful) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(careful)::value;
    const bool more = wave + kWaves * (i + 1) < pairs;
    const int there = next_there;
    if constexpr (!STAGED) {
      p = next;
      if (more) {
        if (((i + 1) & 31) == 0) window(i + 1);
        locate(i + 1);
        fetch(next);
      }
    } else {
      wait_loads<kCopies>();
      take(ring, p.k, p.km);
    }
    const int tok0 = (run.t0 + 2 * (wave + kWaves * i)) * PKV_TILE;  // the pair's first token

    // S^T = K.Q^T, and the scores from it
    const uint32_t q_at = RB > 1 ? lane_again() * 8 : 0;  // (read again for each pair)
    auto query = [&](int rb, int kb) __attribute__((always_inline)) {
      if constexpr (RB > 1) return *(const T *)(kept + (rb * KB + kb) * 512 + q_at);
      else return q[rb][kb];
    };
    float x[RB][8];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      f4 S[RB][NG];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        T k;
        if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);
        if constexpr (C::QUANT) k = Conv<C::PAGE_BITS>::kop(p.k[s], kb);  // 1024 + code
        else k = __builtin_bit_cast(T, u4{p.k[s][4 * kb], p.k[s][4 * kb + 1], p.k[s][4 * kb + 2], p.k[s][4 * kb + 3]});
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          S[rb][kb / GB] = mma(k, query(rb, kb), kb % GB == 0 ? zero : S[rb][kb / GB]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (C::QUANT) {
#pragma unroll
          for (int x_ = 0; x_ < NG; ++x_) {
            const h2 sb = __builtin_bit_cast(h2, p.km[s][e * NG + x_]);
            const float sc = (float)sb.x, off = __builtin_fmaf(-1024.0f, sc, (float)sb.y);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
              x[rb][4 * s + e] = __builtin_fmaf(S[rb][x_][e], sc, x_ == 0 ? off * qs[rb][x_]
                                                                          : __builtin_fmaf(off, qs[rb][x_], x[rb][4 * s + e]));
          }
        } else {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) x[rb][4 * s + e] = S[rb][0][e];
        }
      }
    }

    if constexpr (STAGED) {
      if (more) {
        if (((i + 1) & 31) == 0) window(i + 1);
        locate(i + 1);
        wait_lds();
        stage_k();
      }
    }

    // softmax: a lane's 8 tokens of its row
    float mx[RB];
    bool need = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[rb][e] = __builtin_fmaf(x[rb][e], mult[rb], -m[rb]);
      if constexpr (CAREFUL) {
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
      need |= !(mx[rb] <= thr[rb]);  // (also where they are NaN: a row of NaN is one, not none)
    }
    if (__builtin_expect(__any(need), 0)) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float up = xor32_max(xor16_max(mx[rb]));
        const bool moves = !(up <= thr[rb]);
        const float by = moves ? up - C::LIFT : 0.0f;
        const float alpha = !moves ? 1.0f : thr[rb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-by);
        m[rb] += by;
        thr[rb] = moves ? kTau + C::LIFT : thr[rb];
        sum[rb] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[rb][e] -= by;
#pragma unroll
        for (int n = 0; n < NB; ++n) O[rb][n] *= alpha;
      }
    }
    // (the sum is that of the weights as they enter the product)
    T P[RB], low[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[rb][e] = __builtin_amdgcn_exp2f(x[rb][e]);
        P[rb][e] = (E)x[rb][e];
      }
    if (split) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          low[rb][e] = (E)(x[rb][e] - (float)P[rb][e]);
          sum[rb] += (float)P[rb][e] + (float)low[rb][e];
        }
    } else {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[rb] += (float)P[rb][e];
    }

    if constexpr (STAGED) {
      if (more) wait_loads<kCopies>();
      else wait_loads<0>();
      take(ring + kSide, p.v, p.vm);
    }
    // V's operand of dims 16n ..
    auto value = [&](int n) __attribute__((always_inline)) {
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
        return (T)__builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        return __builtin_bit_cast(T, u4{p.v[0][2 * n], p.v[0][2 * n + 1], p.v[1][2 * n], p.v[1][2 * n + 1]});
      }
    };
    [[maybe_unused]] bool odd = false;
    if constexpr (CAREFUL) {
      // absent tokens hold zeros; are there infinities or NaN among the others?
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int t = (there >> s & 1) ? run.L - tok0 - s * PKV_TILE - 4 * jj : 0;  // the lane's tokens there
        if constexpr (C::QUANT) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x_ = 0; x_ < NG; ++x_) p.vm[s][e * NG + x_] = e < t ? p.vm[s][e * NG + x_] : 0u;
        } else {
#pragma unroll
          for (int x_ = 0; x_ < C::LW; ++x_)
            p.v[s][x_] &= (2 * (x_ & 1) < t ? 0xFFFFu : 0u) | (2 * (x_ & 1) + 1 < t ? 0xFFFF0000u : 0u);
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const u4 bits = __builtin_bit_cast(u4, value(n));
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (bits[e] & 0x7FFFu) >= C::INF || (bits[e] >> 16 & 0x7FFFu) >= C::INF;
      }
    }

    // O^T += V^T.P^T
    if (CAREFUL && __builtin_expect(__any(odd), 0)) {
      // infinities and NaN: their products with a hidden token's zero weight must not be
      // NaN.  The finite values go through the product; the others are counted over the
      // tokens that a row sees, kind by kind in digits of 64 (there are 32 tokens).
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        T v = value(n), kind;
        uint16_t bits[8];
        __builtin_memcpy(bits, &v, 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool bad = (bits[e] & 0x7FFF) >= C::INF;
          kind[e] = !bad ? (E)0.0f : bits[e] == C::INF ? (E)1.0f : bits[e] == (C::INF | 0x8000) ? (E)64.0f : (E)4096.0f;
          v[e] = bad ? (E)0.0f : v[e];
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const int sees = lim[rb] - tok0 - 4 * jj;
          T seen;
#pragma unroll
          for (int e = 0; e < 8; ++e) seen[e] = PKV_TILE * (e >> 2) + (e & 3) <= sees ? (E)1.0f : (E)0.0f;
          O[rb][n] = mma(v, P[rb], O[rb][n]);
          if (split) O[rb][n] = mma(v, low[rb], O[rb][n]);
          const f4 count = mma(kind, seen, zero);
#pragma unroll
          for (int e = 0; e < 4; ++e) O[rb][n][e] += seen_kinds(count[e]);
        }
      }
    } else if (split) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);
        const T v = value(n);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) O[rb][n] = mma(v, low[rb], mma(v, P[rb], O[rb][n]));
      }
    } else {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (RB > 1) __builtin_amdgcn_sched_barrier(0);
        const T v = value(n);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) O[rb][n] = mma(v, P[rb], O[rb][n]);
      }
    }
    if constexpr (STAGED) {
      if (more) {
        wait_lds();
        stage_v();
      }
    }
  };
  // (the pairs that need care are a run's last, but for missing pages)
  int i = 0;
  for (; wave + kWaves * i < pairs; ++i) {
    const int last_token = (run.t0 + 2 * (wave + kWaves * i)) * PKV_TILE + 2 * PKV_TILE - 1;
    if (__builtin_expect(next_there != 3 || last_token > least, 0)) break;
    pair(i, std::false_type());
  }
  for (; wave + kWaves * i < pairs; ++i) pair(i, std::true_type());

  // ---- the four waves' parts joined, 16 rows at a time, and written
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    sum[rb] = xor32_add(xor16_add(sum[rb]));
    if (jj == 0) {
      // (a row that sees nothing has none, whatever went through its lanes)
      s_ml[wave][rb * 16 + col][0] = thr[rb] == -INFINITY || lim[rb] < 0 ? -INFINITY : m[rb];
      s_ml[wave][rb * 16 + col][1] = sum[rb];
    }
  }
  __syncthreads();
  constexpr int ROW = DP + 4;
  float *s_acc = (float *)lds;
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
        for (int x = 0; x < kWaves; ++x) best = __builtin_elementwise_maximum(best, s_ml[x][rb * 16 + tid][0]);
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

// Run u of the call and, in the first workgroup, what the merge needs: by a plan in LDS.
__device__ __forceinline__ bool planned_run(const SharedArgs &a, const SharedWork &w, SharedPlan &plan, int per, int u,
                                            int tid, Run &run) {
  const int lane = tid & 63;
  lay_out(a, plan, per, tid);
  const int shared_runs = plan.group_run[a.groups], runs = shared_runs + plan.own_run[a.count];
  if (blockIdx.x == 0) {
    // where a member's parts are, for the merge: its group's first run and runs per
    // segment, its first row in the group; its own first run and runs per KV head; whose
    // table the group's tiles are read through, and how many there are
    for (int j = tid; j < a.count; j += kThreads) {
      const bool in = j >= plan.group_first[0] && j < plan.group_first[a.groups];
      const int g = in ? last_at_most(plan.group_first, a.groups, j) : 0;
      int32_t *d = w.desc + 8 * j;
      d[0] = plan.group_run[g];
      d[1] = in ? runs_of(plan.group_tiles[g], plan.long_run) : 0;
      d[2] = (j - plan.group_first[g]) * a.rows;
      d[3] = shared_runs + plan.own_run[j];
      d[4] = (plan.own_run[j + 1] - plan.own_run[j]) / a.g.hk;
      d[5] = in;
      d[6] = in ? plan.sequence[plan.group_first[g]] : -1;
      d[7] = plan.group_tiles[g];
    }
  }
  if (u >= runs) return false;
  run.slot = u;
  if (u < shared_runs) {
    const int g = last_at_most_uniform(plan.group_run, a.groups, u, lane);
    const int tiles = plan.group_tiles[g], n = runs_of(tiles, plan.long_run), at = u - plan.group_run[g];
    const int seg = at / n, blk = seg / a.g.hk, len = run_length(tiles, n);
    run.kh = seg - blk * a.g.hk;
    run.t0 = min((at - seg * n) * len, tiles);
    run.t1 = min(tiles, run.t0 + len);
    run.member = plan.group_first[g];
    run.row0 = blk * per;
    run.rows = min(per, (plan.group_first[g + 1] - run.member) * a.rows - run.row0);
  } else {
    const int j = last_at_most_uniform(plan.own_run, a.count, u - shared_runs, lane);
    const int n = (plan.own_run[j + 1] - plan.own_run[j]) / a.g.hk, at = u - shared_runs - plan.own_run[j];
    const int g = last_at_most_uniform(plan.group_first, a.groups, j, lane);
    run.kh = at / n;
    const int first = plan.group_tiles[g], end = tiles_of(plan.length[j]), len = run_length(end - first, n);
    run.t0 = min(first + (at - run.kh * n) * len, end);
    run.t1 = min(end, run.t0 + len);
    run.member = j;
    run.row0 = 0;
    run.rows = a.rows;
  }
  return true;
}

// The same for at most 64 members and 63 groups, by each wave for itself: lane l has member l and
// group l.  (No barrier: 2.9 us until the run is known instead of 4.8, for 16 sequences in four
// groups.)
__device__ __forceinline__ bool small_run(const SharedArgs &a, const SharedWork &w, int per, int u, int wave, int lane,
                                          int *sequence, int *length, Run &run) {
  const int hk = a.g.hk;
  int first = min(max(a.group_starts[min(lane, a.groups)], 0), a.count);
  int tiles = lane < a.groups ? a.prefix_lens[lane] : 0;
  const int b = lane < a.count ? a.members[lane] : -1;
  const bool known = b >= 0 && b < a.batch;
  const int len = known ? seq_length(a, b) : 0;
  sequence[lane] = known ? b : -1;
  length[lane] = len;
  const int next = __shfl(first, min(lane + 1, 63), 64);
  int n = lane < a.groups ? next - first : 0;
  if (__any(n < 0)) first = n = tiles = 0;  // groups that would overlap: none
  const int held = __shfl(len, min(first, 63), 64);
  tiles = n > 1 ? max(0, min(tiles, held)) / PKV_TILE : 0;  // (one sequence shares nothing)
  const int blocks = (n * a.rows + per - 1) / per;
  const int last = __builtin_amdgcn_readlane(first, a.groups);
  int g = -1;  // the member's group
  for (int k = 0; k < a.groups; ++k) g += lane >= __builtin_amdgcn_readlane(first, k);
  const bool in = g >= 0 && lane < last;
  g = max(g, 0);
  const int skipped = __shfl(tiles, g, 64);
  const int own = in ? max(0, tiles_of(len) - skipped) : 0;
  const int own_cost = a.rows > 16 ? kSharedCost : kOwnCost;
  const int64_t mine = ((int64_t)kSharedCost * tiles * blocks + (int64_t)own_cost * own) * hk;
  const int lo = wave_sum((int)(mine & 0x7FFFFF));
  const int hi = wave_sum((int)(mine >> 23));
  const int64_t cost = lo + ((int64_t)hi << 23);
  const int segs = wave_sum((tiles > 0 ? blocks : 0) + (own > 0 ? 1 : 0)) * hk;
  int long_run = 0, own_long = 0, shared_n = 0, own_n = 0;  // a segment's runs
  for (int k = 0; k < kWaves; ++k) {
    run_lengths(cost, segs, own_cost, k, long_run, own_long);
    shared_n = runs_of(tiles, long_run);
    own_n = runs_of(own, own_long);
    if ((int64_t)wave_sum(blocks * shared_n + own_n) * hk <= kTarget) break;
  }
  const int group_runs = blocks * hk * shared_n, own_runs = hk * own_n;
  const int group_end = wave_scan_incl(group_runs, lane), own_end = wave_scan_incl(own_runs, lane);
  const int group_run = group_end - group_runs, own_run = own_end - own_runs;
  const int shared_runs = __builtin_amdgcn_readlane(group_end, 63);
  const int runs = shared_runs + __builtin_amdgcn_readlane(own_end, 63);
  if (blockIdx.x == 0) {
    const int d0 = __shfl(group_run, g, 64), d1 = __shfl(shared_n, g, 64), at = __shfl(first, g, 64);
    const int leader = __shfl(known ? b : -1, min(at, 63), 64);
    if (wave == 0 && lane < a.count) {
      int32_t *d = w.desc + 8 * lane;
      d[0] = d0;
      d[1] = in ? d1 : 0;
      d[2] = (lane - at) * a.rows;
      d[3] = shared_runs + own_run;
      d[4] = own_n;
      d[5] = in;
      d[6] = leader;
      d[7] = skipped;
    }
  }
  if (u >= runs) return false;
  run.slot = u;
  if (u < shared_runs) {
    const int k = __popcll(__ballot(lane < a.groups && group_run <= u)) - 1;
    const int total = __builtin_amdgcn_readlane(tiles, k), c = __builtin_amdgcn_readlane(shared_n, k);
    const int at = u - __builtin_amdgcn_readlane(group_run, k), seg = at / c, blk = seg / hk, size = run_length(total, c);
    run.kh = seg - blk * hk;
    run.t0 = min((at - seg * c) * size, total);
    run.t1 = min(total, run.t0 + size);
    run.member = __builtin_amdgcn_readlane(first, k);
    run.row0 = blk * per;
    run.rows = min(per, __builtin_amdgcn_readlane(n, k) * a.rows - run.row0);
  } else {
    const int k = __popcll(__ballot(lane < a.count && own_run <= u - shared_runs)) - 1;
    const int c = __builtin_amdgcn_readlane(own_n, k), at = u - shared_runs - __builtin_amdgcn_readlane(own_run, k);
    const int from = __builtin_amdgcn_readlane(skipped, k), end = tiles_of(__builtin_amdgcn_readlane(len, k));
    const int size = run_length(end - from, c);
    run.kh = at / c;
    run.t0 = min(from + (at - run.kh * c) * size, end);
    run.t1 = min(end, run.t0 + size);
    run.member = k;
    run.row0 = 0;
    run.rows = a.rows;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return true;
}

template <int BITS, int DP, int G, int FK>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void shared_kernel(const SharedArgs a, const SharedWork w) {
  using C = SharedCfg<BITS, DP, G, FK>;
  constexpr int PER = shared_rows(DP);
  // the plan; behind it the copies and the rows of two blocks; behind those the sums
  constexpr int kRing = PER > 16 ? kWaves * 2 * side_bytes<C>() + 2 * C::KB * 1024 : 0;
  constexpr int kSums = kWaves * 16 * (DP + 4) * 4;
  constexpr int kLds = std::max({(int)sizeof(SharedPlan), kRing, kSums});
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
  SharedPlan &plan = *(SharedPlan *)lds;
  __shared__ float s_ml[kWaves][shared_rows(64)][2];
  __shared__ TilePlace s_place[kWaves][64];
  __shared__ int s_members[kWaves][2][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int u = blockIdx.x;
  Run run;
  const int *sequence = plan.sequence, *length = plan.length;
  bool found;
  if (a.count <= 64 && a.groups < 64) {
    found = small_run(a, w, PER, u, wave, lane, s_members[wave][0], s_members[wave][1], run);
    sequence = s_members[wave][0];
    length = s_members[wave][1];
  } else {
    found = planned_run(a, w, plan, PER, u, tid, run);
  }
  if (found && u < w.most) {
    // (a member that is no sequence has no tokens; the first of a group with a prefix is one)
    run.b = max(0, __builtin_amdgcn_readfirstlane(sequence[run.member]));
    run.L = __builtin_amdgcn_readfirstlane(length[run.member]);
    run.kh = __builtin_amdgcn_readfirstlane(run.kh);
    run.t0 = __builtin_amdgcn_readfirstlane(run.t0);
    run.t1 = __builtin_amdgcn_readfirstlane(run.t1);
    run.member = __builtin_amdgcn_readfirstlane(run.member);
    run.row0 = __builtin_amdgcn_readfirstlane(run.row0);
    run.rows = __builtin_amdgcn_readfirstlane(run.rows);
    if (run.rows <= 16) run_tiles<C, 1>(a, w, sequence, length, run, lane, wave, s_place[wave], lds, s_ml);
    else if constexpr (PER > 16) run_tiles<C, 2>(a, w, sequence, length, run, lane, wave, s_place[wave], lds, s_ml);
  }
}

// Row r of (sequence b, KV head kh) by itself, a tile at a time in 32 bits: the sums of
// p_t v_t (the lane's dims) and of p_t = 2^(s_t - top).  The first `shared` tiles are read through
// `leader`'s table.  q: the row's queries as float32, in LDS.  The whole wave calls.
template <int DP>
__device__ __forceinline__ float row_alone(const SharedArgs &a, int b, int leader, int shared, int kh, int qi,
                                           const float *q, float top, int lane, float (&acc)[DP / 64]) {
  constexpr int EPL = DP / 64;
  const Geo &g = a.g;
  const int t = lane & 15, jj = lane >> 4, tpp = g.page / PKV_TILE;
  const int width = a.widths ? a.widths[b] : a.nq;
  const int pos = a.q_pos ? a.q_pos[(int64_t)b * a.nq + qi] : a.seq_lens[b] - width + qi;
  const int last = qi < width ? min(pos, seq_length(a, b) - 1) : -1;
#pragma unroll
  for (int e = 0; e < EPL; ++e) acc[e] = 0.0f;
  float total = 0.0f;
  for (int tile = 0; tile * PKV_TILE <= last; ++tile) {
    const int page = a.table[(int64_t)(tile < shared ? leader : b) * a.max_pages + tile / tpp];
    if (page < 0 || page >= a.num_pages) continue;
    const uint8_t *head = a.pool + (int64_t)page * g.page_bytes + (int64_t)kh * g.head_bytes;
    const uint8_t *k = head + (int64_t)(tile % tpp) * g.tile_bytes, *v = k + g.v_offset;
    auto word = [&](int64_t meta, int tt, int d) __attribute__((always_inline)) {
      return *(const uint32_t *)(head + meta + ((int64_t)(tile % tpp * PKV_TILE + tt) * g.ng + d / g.group) * 4);
    };
    const bool bytes = g.bits == 8;
    // K: the lane's share of the payload, elements 32 kb + 8 jj + 0..7 of token t
    float s = 0.0f;
#pragma unroll
    for (int kb = 0; kb < DP / 32; ++kb) {
      const int d0 = 32 * kb + 8 * jj;  // (a group holds whole eights)
      const uint32_t m = word(g.kmeta_offset, t, d0);
      const uint32_t w0 = *(const uint32_t *)(k + payload_offset(lane, bytes ? 8 * kb : 4 * kb, g.chunk));
      const uint32_t w1 = bytes ? *(const uint32_t *)(k + payload_offset(lane, 8 * kb + 4, g.chunk)) : 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t code = bytes ? (e < 4 ? w0 : w1) >> (8 * (e & 3)) & 255u : w0 >> (4 * k4_nibble(e)) & 15u;
        s = __builtin_fmaf(__builtin_fmaf((float)code, f16_bits_to_f32(m), f16_bits_to_f32(m >> 16)), q[d0 + e], s);
      }
    }
    s = xor32_add(xor16_add(s));
    float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s, a.scale * kLog2e, -top));
    if (tile * PKV_TILE + t > last) p = 0.0f;
    // V: the lane's dims, four tokens to a word
    const int d = lane * EPL;  // (all of them in one group)
#pragma unroll
    for (int four = 0; four < 4; ++four) {
      uint32_t w[EPL], m[4];
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int n = (d + e) / 16;
        w[e] = *(const uint32_t *)(v + payload_offset((d + e) % 16 + 16 * four, bytes ? 4 * n : n / 2 * 4, g.chunk));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) m[r] = word(g.vmeta_offset, 4 * four + r, d);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(p), 4 * four + r));
        total += x;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const uint32_t code = bytes ? w[e] >> (8 * r) & 255u : w[e] >> (8 * v4_byte(r) + 4 * ((d + e) / 16 % 2)) & 15u;
          const float y = __builtin_fmaf((float)code, f16_bits_to_f32(m[r]), f16_bits_to_f32(m[r] >> 16));
          // (what follows the last token may be anything)
          acc[e] = __builtin_fmaf(tile * PKV_TILE + 4 * four + r <= last ? y : 0.0f, x, acc[e]);
        }
      }
    }
  }
  return total;
}

// One wave per (sequence, KV head, row): the row's parts joined.  Lane l weighs part l (of 64 at
// a time); the parts' rows are read eight at a time.
template <int DP>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(const SharedArgs a, const SharedWork w) {
  constexpr int PER = shared_rows(DP), EPL = DP / 64, KEPT = 8;
  const int lane = threadIdx.x & 63;
  const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  const int per_row = a.g.hk * a.rows;
  const int b = unit / per_row, in = unit - b * per_row, kh = in / a.rows, r = in - kh * a.rows;
  if (b >= a.batch) return;
  // the sequence's member
  int j = -1;
  for (int c = 0; c < a.count && j < 0; c += 64) {
    const unsigned long long hit = __ballot(c + lane < a.count && a.members[c + lane] == b);
    if (hit) j = c + __ffsll((long long)hit) - 1;
  }
  const int32_t *d = w.desc + 8 * max(j, 0);
  const int qi = r / a.gqa, h = kh * a.gqa + r % a.gqa;
  uint16_t *o = a.out + (((int64_t)b * a.heads + h) * a.nq + qi) * a.g.dim;
  if (j < 0 || !d[5]) {
    if (a.zero_others)
      for (int e = lane; e < a.g.dim; e += 64) o[e] = 0;
    return;
  }
  const int row = d[2] + r, shared = d[1], own = d[4];
  // the first parts' rows among all runs' rows
  const int64_t first = (int64_t)(d[0] + (row / PER * a.g.hk + kh) * shared) * PER + row % PER;
  const int64_t own_first = (int64_t)(d[3] + kh * own) * PER + r;
  const int n = shared + own;
  auto at = [&](int i) { return i < shared ? first + (int64_t)i * PER : own_first + (int64_t)(i - shared) * PER; };
  float x[KEPT][EPL];
  auto request = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) x[i][e] = 0.0f;
      if (i0 + i < n) __builtin_memcpy(x[i], w.acc + at(i0 + i) * DP + lane * EPL, 4 * EPL);
    }
  };
  request(0);
  float top = -INFINITY, m = -INFINITY, l = 0.0f;  // m and l: lane's part of the first 64
  for (int i = lane; i < n; i += 64) {
    float2 ml;
    __builtin_memcpy(&ml, w.ml + 2 * at(i), 8);
    if (i == lane) {
      m = ml.x;
      l = ml.y;
    }
    top = __builtin_elementwise_maximum(top, ml.x);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o, 64));
  float total = 0.0f, acc[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) acc[e] = 0.0f;
  for (int c = 0; c < n; c += 64) {
    if (c > 0) {
      m = -INFINITY;
      l = 0.0f;
      if (c + lane < n) {
        m = w.ml[2 * at(c + lane)];
        l = w.ml[2 * at(c + lane) + 1];
      }
    }
    // (a part without a visible token has weight 0, whatever the maximum)
    const float weight = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    total += l * weight;
    for (int i = c; i < n && i < c + 64; i += KEPT) {
      if (i > 0) request(i);
#pragma unroll
      for (int y = 0; y < KEPT; ++y) {
        const float wy = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), i - c + y));
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] = wy == 0.0f ? acc[e] : __builtin_fmaf(x[y][e], wy, acc[e]);
      }
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o, 64);
  // Values of quantized pages go up to 2^24, past float16's range: an operand that has become an
  // infinity leaves sums that are not finite, and the row is computed by itself.
  bool lost = false;
#pragma unroll
  for (int e = 0; e < EPL; ++e) lost |= !(fabsf(acc[e]) < INFINITY);
  if (__builtin_expect(a.g.bits != 16 && fabsf(top) < INFINITY && __any(lost), 0)) {
    __shared__ float s_q[kWaves][DP];
    float *q = s_q[threadIdx.x >> 6];
    const uint16_t *src = a.q + (((int64_t)b * a.heads + h) * a.nq + qi) * a.g.dim;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const int i = lane + 64 * e;
      q[i] = i < a.g.dim ? bits_to_float(src[i], a.g.float_kind) : 0.0f;
    }
    wave_lds_sync();
    total = row_alone<DP>(a, b, max(d[6], 0), d[6] < 0 ? 0 : d[7], kh, qi, q, top, lane, acc);
  }
  const float inv = top == -INFINITY ? 0.0f : 1.0f / total;
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
  const dim3 rows((unsigned)(((int64_t)a.batch * a.g.hk * a.rows + kWaves - 1) / kWaves));
  if (a.g.dp == 64) hipLaunchKernelGGL((shared_merge_kernel<64>), rows, block, 0, stream, a, w);
  else if (a.g.dp == 128) hipLaunchKernelGGL((shared_merge_kernel<128>), rows, block, 0, stream, a, w);
  else hipLaunchKernelGGL((shared_merge_kernel<256>), rows, block, 0, stream, a, w);
  return hipGetLastError();
}

}  // namespace pkv
