// pkv_prompt.hip -- causal attention within every sequence of packed rows.
//
//   o_i = sum_{j <= i} softmax_j(scale * q_i . k_j) v_j     per sequence and head
//
// A chunk is 32 consecutive queries of one head; the chunks of a (sequence, KV head) are
// ordered by position, then head, and the four waves of a workgroup take consecutive ones:
// with a few heads per KV head they end at nearly the same key.  Keys come in stages of 64 (32
// beyond head dim 128), K and V copied straight to LDS in rows (global_load_lds), a stage ahead.
//
//   S^T = K.Q^T       v_mfma_f32_32x32x16, 32 keys x 32 queries: a lane has one query
//   O^T += V^T.P^T    the same; V^T comes out of V's rows by transposing LDS reads
//
// The contraction over keys takes a lane's scores as they lie (keys 8g + 4h + r in slot
// 8h + 4(g & 1) + r), so P never crosses lanes.  Softmax in the exp2 domain with float32
// maximum and sum; P is rounded once to the activation type, as the operand of its product
// (2^-8 relative for bfloat16, beside the output's own rounding of the same size; 2^-11 for float16,
// and from 2^-21 of the largest weight down half of a fixed step, 2^-32 of that weight), and summed
// as rounded, so that weights still add up to one: a channel of V that is the same for all rows
// comes out as it is.  (bfloat16 weights as the sum of two operands, as attention over bfloat16
// pages takes them, put half as many products more beside the scores': 16,000 rows 1.90 ms ->
// 2.68, mixed prompts 250 us -> 317.  What they save is 12% of the error of 30 rows of ordinary
// values and 22% of that of 2,000, beside the output's rounding.)
//
// Only the last tile of a wave, on the diagonal, is masked.  There a masked key's V may be
// anything: where it is not finite those elements are taken apart (a rare branch).
//
// Bound by the issue of matrix and vector instructions: a tile's weights and product are
// issued beside the next tile's scores, and two waves share a SIMD (one beyond head dim 128,
// where two would spill: 355 us against 144 then for 16 heads of 256).  16,000 rows of 32 heads of 128: 1.93
// ms, 1.09 PFLOP/s (86% of an 8192^3 product); 16 prompts of 100 to 2,000 rows 0.23 ms.
#include <type_traits>

#include "pkv_mfma.h"
#include "pkv_step.h"

namespace pkv {

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

template <int FK>
struct Wide;
template <>
struct Wide<0> {
  typedef b8 T;
  typedef __bf16 E;
  static __device__ __forceinline__ f16v mma(b8 a, b8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // sum + the pair's two values
  static __device__ __forceinline__ float add(__bf16 x, __bf16 y, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(b2{x, y}, b2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
  }
  static constexpr uint16_t kInf = 0x7F80;
  static constexpr float kLift = 0.0f;
};
template <>
struct Wide<1> {
  typedef h8 T;
  typedef _Float16 E;
  static __device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add(_Float16 x, _Float16 y, float sum) {
    return __builtin_amdgcn_fdot2(h2{x, y}, h2{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
  }
  static constexpr uint16_t kInf = 0x7C00;
  // weights as 2^kLift of themselves, the largest 2^(kTau + kLift) then: those of less than
  // 2^-14 have fewer bits
  static constexpr float kLift = 7.0f;
};

template <int DP>
struct PromptShape {
  static constexpr int UNITS = DP / 8;                // 16-byte units per row
  static constexpr int TILES = DP > 128 ? 1 : 2;      // 32-key tiles per stage
  static constexpr int KEYS = 32 * TILES;
  static constexpr int SIDE = KEYS * DP * 2;          // bytes of a stage's K (or V)
  static constexpr int COPIES = KEYS * UNITS / 256;   // 16-byte units per thread and side
  // a tile's product with V runs beside the next tile's scores: V stays a stage longer
  static constexpr int KBUF = 2, VBUF = 3;
  static constexpr int BYTES = (KBUF + VBUF) * SIDE;
};

// Where unit u of row m of a stage's K sits, so that the operand reads (one unit of 32 rows)
// meet no bank twice: LDS serves 16 lanes of a 16-byte read at once, 0-7 and 16-23, then
// 8-15 and 24-31, over 64 banks.
template <int DP>
__device__ __forceinline__ int k_unit(int m, int u) {
  if constexpr (DP == 64) return u ^ (((m >> 1) & 3) | (((m >> 4) & 1) << 2));
  else return u ^ ((m & 7) | (((m >> 4) & 1) << 3));
}
// The same for V, whose transposing reads take 64 bytes of four consecutive rows.
template <int DP>
__device__ __forceinline__ int v_unit(int m, int u) {
  if constexpr (DP == 64) return u ^ (((m >> 1) & 1) << 2);
  else return u ^ ((m & 3) << 2);
}

// Rows of sequence b: first and count.
__device__ __forceinline__ int prompt_rows(const PromptArgs &a, int b, int &first) {
  first = min(max(a.row_starts[b], 0), a.rows);
  return min(a.row_starts[b + 1], a.rows) - first;
}

// Workgroups of a sequence of n rows, per KV head.
constexpr int kChunks = 4;
__device__ __forceinline__ int prompt_blocks(int n, int gqa) {
  return n <= 0 ? 0 : ((n + 31) / 32 * gqa + kChunks - 1) / kChunks;
}

// The workgroup's (sequence, block), and the sequence's rows: the longest blocks of all
// sequences first for 4 to 12 sequences, else sequence by sequence, each from its end.  (All
// together end more evenly, but take longer to find, and the work passes through more
// sequences at once.  Prompts of 100 to 2,000 rows, all together and by sequence: 2 prompts 40
// and 41 us, 4 46 and 49, 6 92 and 106, 8 108 and 109, 12 263 and 263, 13 207 and 204, 16 230
// and 231, 24 383 and 377, 32 504 and 479, 64 1,074 and 962; of up to 500 rows, 4 17.1 and 16.7,
// 8 25.8 and 25.3, 12 37 and 36, 16 37 and 34, 64 142 and 127.  One of 8,000 rows as the last of 4
// to 64 short ones: within 1% up to 24, 619 and 602 for 64.)  The whole wave calls.
__device__ __forceinline__ bool find_block(const PromptArgs &a, int rank, int lane, int &b, int &blk, int &first,
                                           int &n) {
  int carry = 0;
  for (int c = 0; c < a.batch; c += 64) {
    int start = 0;
    const int rows = c + lane < a.batch ? prompt_rows(a, c + lane, start) : 0;
    const int mine = prompt_blocks(rows, a.gqa);
    int f;
    if (a.batch >= 4 && a.batch <= 12) {
      if (rank >= wave_sum(mine)) return false;
      // the largest level of which more than `rank` blocks are at or above
      int lo = 0, hi = 1;
      while (__ballot(mine >= hi)) hi <<= 1;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (wave_sum(max(0, mine - mid)) > rank) lo = mid;
        else hi = mid;
      }
      unsigned long long at = __ballot(mine > lo);
      for (int i = rank - wave_sum(max(0, mine - lo - 1)); i > 0; --i) at &= at - 1;
      f = __ffsll((long long)at) - 1;
      blk = lo;
    } else {
      const int incl = wave_scan_incl(mine, lane) + carry;
      const unsigned long long hit = __ballot(incl > rank);
      carry = __builtin_amdgcn_readlane(incl, 63);
      if (!hit) continue;
      f = __ffsll((long long)hit) - 1;
      blk = __builtin_amdgcn_readlane(incl, f) - 1 - rank;
    }
    b = c + f;
    first = __builtin_amdgcn_readlane(start, f);
    n = __builtin_amdgcn_readlane(rows, f);
    return true;
  }
  return false;
}

__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}

// A lane's V^T operand (dim 32 nb + col, 16 keys) out of V's rows in LDS.
template <int DP, typename T>
__device__ __forceinline__ T v_operand(const ldsbyte *src) {
  typedef short s4v __attribute__((ext_vector_type(4)));
  struct { s4v lo, hi; } v;
  v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)src);
  v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)(src + 8 * DP * 2));
  return __builtin_bit_cast(T, v);
}

template <int DP, int FK>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void prompt_kernel(const PromptArgs a) {
  using W = Wide<FK>;
  using T = typename W::T;
  using E = typename W::E;
  using S = PromptShape<DP>;
  constexpr int KS = DP / 16, NB = DP / 32;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int kh = blockIdx.x % a.kv_heads;
  int b, blk, first, n;
  if (!find_block(a, blockIdx.x / a.kv_heads, lane, b, blk, first, n)) return;
  const int chunks = (n + 31) / 32 * a.gqa;

  // the wave's chunk: 32 queries from 32 * place on, of one head (place -1: none)
  const int chunk = blk * kChunks + wave;
  const int place = chunk < chunks ? chunk / a.gqa : -1, head = kh * a.gqa + chunk % a.gqa;
  const int last = (min(chunks, (blk + 1) * kChunks) - 1) / a.gqa;  // 32-key tile of the block's last chunk
  const int stages = last / S::TILES + 1;

  // ---- K and V rows to LDS: thread tid copies unit tid + 256 i of a stage
  const uint8_t *kbase = (const uint8_t *)(a.k + (int64_t)first * a.k_stride + kh * a.dim);
  const uint8_t *vbase = (const uint8_t *)(a.v + (int64_t)first * a.v_stride + kh * a.dim);
  // Copies i are STEP rows apart: V's units keep their places, K's are moved by bit 4 of
  // the row alone.
  constexpr int STEP = 256 / S::UNITS;
  const int crow = tid / S::UNITS, vu = v_unit<DP>(crow, tid % S::UNITS);
  int ku[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) ku[f] = k_unit<DP>((crow & ~16) | (((crow >> 4) ^ f) & 1) << 4, tid % S::UNITS);
  const uint32_t vat = crow * (uint32_t)a.v_stride * 2 + vu * 16;
  uint32_t kat[2];
#pragma unroll
  for (int f = 0; f < 2; ++f) kat[f] = crow * (uint32_t)a.k_stride * 2 + ku[f] * 16;
  auto copy = [&](int s) __attribute__((always_inline)) {
    uint8_t *kdst = lds + s % S::KBUF * S::SIDE + wave * 1024;
    uint8_t *vdst = lds + (S::KBUF + s % S::VBUF) * S::SIDE + wave * 1024;
    const uint8_t *ksrc = kbase + (int64_t)s * S::KEYS * a.k_stride * 2;
    const uint8_t *vsrc = vbase + (int64_t)s * S::KEYS * a.v_stride * 2;
    if (a.dim == DP && (s + 1) * S::KEYS <= n) {  // whole rows, all of them there
#pragma unroll
      for (int i = 0; i < S::COPIES; ++i) {
        copy_to_lds(ksrc + (int64_t)i * STEP * a.k_stride * 2, kat[i * STEP / 16 % 2], kdst + i * 4096);
        copy_to_lds(vsrc + (int64_t)i * STEP * a.v_stride * 2, vat, vdst + i * 4096);
      }
      return;
    }
    // rows past the last one read it again (their keys are masked)
    const int rows = n - s * S::KEYS;
#pragma unroll
    for (int i = 0; i < S::COPIES; ++i) {
      const int f = i * STEP / 16 % 2;
      const int64_t back = i * STEP - max(crow + i * STEP - (rows - 1), 0);
      if (ku[f] < a.dim / 8) copy_to_lds(ksrc + back * a.k_stride * 2 + kat[f], kdst + i * 4096);
      if (vu < a.dim / 8) copy_to_lds(vsrc + back * a.v_stride * 2 + vat, vdst + i * 4096);
    }
  };
  if (a.dim < DP) {  // the units past the head dim hold zeros
    for (int i = tid; i < S::BYTES / 16; i += 256) *((u4 *)lds + i) = u4{0, 0, 0, 0};
    barrier();
  }

  copy(0);

  // ---- queries: lane (col, half) holds elements 16 ks + 8 half + e of query col
  T q[KS];
  {
    const int64_t row = first + min(max(place, 0) * 32 + col, n - 1);
    const uint16_t *src = a.q + row * a.q_stride + (int64_t)head * a.dim;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = 16 * ks + 8 * half;
      u4 x = {0, 0, 0, 0};
      if (d < a.dim && place >= 0) x = *(const u4 *)(src + d);
      q[ks] = __builtin_bit_cast(T, x);
    }
  }

  float m = 0.0f, thr = -INFINITY, l = 0.0f;
  f16v O[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) O[j][e] = 0.0f;

  // (a swizzle moves a unit within 16: beyond head dim 128 the second half lies 256 bytes on)
  constexpr int KO = KS < 8 ? KS : 8, VO = NB < 4 ? NB : 4;
  uint32_t koff[KO], voff[VO];
#pragma unroll
  for (int ks = 0; ks < KO; ++ks) koff[ks] = (col * S::UNITS + k_unit<DP>(col, 2 * ks + half)) * 16;
  {
    const int i = lane & 15, j = (lane >> 4) & 1, r = 4 * half + i / 4;
#pragma unroll
    for (int nb = 0; nb < VO; ++nb)
      voff[nb] = (r * S::UNITS + v_unit<DP>(r, 4 * nb + 2 * j + (i & 3) / 2)) * 16 + 8 * (i & 1);
  }

  // S^T = K.Q^T of a tile.  (From zeros in registers: an MFMA with an inline constant 0 as
  // its accumulator has given wrong results where its destination partly overlaps an operand.)
  f16v zero = {0};
  asm volatile("" : "+v"(zero));
  ldsbyte *const base = (ldsbyte *)lds;
  auto scores = [&](uint32_t ktile, f16v &x) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const u4 k = *(const __attribute__((address_space(3))) u4 *)(base + (koff[ks % KO] + ktile) + ks / KO * 256);
      x = W::mma(__builtin_bit_cast(T, k), q[ks], ks == 0 ? zero : x);
    }
  };
  // the exponents, less the running maximum and plus kLift: it moves when a score passes it by
  // kTau
  auto settle = [&](auto masks, f16v &x) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __builtin_fmaf(x[e], a.scale_log2, -m);
    // on the diagonal, key 8g + 4 half + r is seen by the queries from it on
    if constexpr (decltype(masks)::value) {
      const int sees = col - 4 * half;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = 8 * (e / 4) + e % 4 <= sees ? x[e] : -INFINITY;
    }
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = __builtin_elementwise_maximum(mx, x[e]);
    if (__builtin_expect(__any(mx > thr), 0)) {
      const float up = xor32_max(mx);
      const bool moves = up > thr;
      const float by = moves ? up - W::kLift : 0.0f;
      const float alpha = !moves ? 1.0f : thr == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-by);
      m += by;
      thr = moves ? kTau + W::kLift : thr;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] -= by;
#pragma unroll
      for (int j = 0; j < NB; ++j) O[j] *= alpha;
    }
  };
  // the weights as operands, and their sum
  auto weights = [&](const f16v &x, T (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      const E r0 = (E)__builtin_amdgcn_exp2f(x[e]), r1 = (E)__builtin_amdgcn_exp2f(x[e + 1]);
      p[e / 8][e % 8] = r0;
      p[e / 8][e % 8 + 1] = r1;
      l = W::add(r0, r1, l);
    }
  };
  auto product = [&](uint32_t vtile, const T (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        O[nb] = W::mma(v_operand<DP, T>(base + (voff[nb % VO] + vtile) + kk * 16 * DP * 2 + nb / VO * 256), p[kk], O[nb]);
  };
  // where tile `at` lies: uniform offsets (of a stage, then of its second tile)
  auto ktile = [&](int at) __attribute__((always_inline)) {
    return (uint32_t)__builtin_amdgcn_readfirstlane(at / S::TILES % S::KBUF * S::SIDE + at % S::TILES * (32 * DP * 2));
  };
  auto vtile = [&](int at) __attribute__((always_inline)) {
    return (uint32_t)__builtin_amdgcn_readfirstlane((S::KBUF + at / S::TILES % S::VBUF) * S::SIDE +
                                                    at % S::TILES * (32 * DP * 2));
  };
  // stage s is here; everyone is done with the scores of stage s - 1 and the products of
  // stage s - 2, whose places the next stage takes
  auto turn = [&](int s) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    barrier();
    if (s + 1 < stages) copy(s + 1);
  };

  // ---- the wave's tiles: a tile's weights and product go beside the next one's scores;
  // the last one, on the diagonal, is masked
  if (place >= 0) {
    f16v x, y;
    T p[2];
    turn(0);
    scores(ktile(0), x);
    if (place == 0) {
      settle(std::true_type{}, x);
    } else {
      settle(std::false_type{}, x);
      int at = 1;
      for (; at + 1 < place; at += 2) {
        if (S::TILES == 1) turn(at);
        scores(ktile(at), y);
        weights(x, p);
        product(vtile(at - 1), p);
        settle(std::false_type{}, y);
        turn((at + 1) / S::TILES);
        scores(ktile(at + 1), x);
        weights(y, p);
        product(vtile(at), p);
        settle(std::false_type{}, x);
      }
      if (at < place) {
        if (S::TILES == 1) turn(at);
        scores(ktile(at), y);
        weights(x, p);
        product(vtile(at - 1), p);
        settle(std::false_type{}, y);
        x = y;
      }
      if (place % S::TILES == 0) turn(place / S::TILES);
      scores(ktile(place), y);
      weights(x, p);
      product(vtile(place - 1), p);
      settle(std::true_type{}, y);
      x = y;
    }
    weights(x, p);
    const uint32_t vlast = vtile(place);
    bool odd = false;  // infinities or NaN among the tile's values?
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const u4 w = __builtin_bit_cast(u4, v_operand<DP, T>(base + (voff[nb % VO] + vlast) + kk * 16 * DP * 2 + nb / VO * 256));
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (w[e] & 0x7FFFu) >= W::kInf || (w[e] >> 16 & 0x7FFFu) >= W::kInf;
      }
    if (__builtin_expect(!__any(odd), 1)) {
      product(vlast, p);
    } else {
      // their products with the masked keys' zero weights must not be NaN: the finite
      // values go through the product; the others are counted over the keys that a query
      // sees, kind by kind in digits of 64
      const int sees = col - 4 * half;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        T seen;
#pragma unroll
        for (int e = 0; e < 8; ++e) seen[e] = 8 * (2 * kk + e / 4) + e % 4 <= sees ? (E)1.0f : (E)0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          T v = v_operand<DP, T>(base + (voff[nb % VO] + vlast) + kk * 16 * DP * 2 + nb / VO * 256), kind;
          uint16_t w[8];
          __builtin_memcpy(w, &v, 16);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const bool bad = (w[e] & 0x7FFF) >= W::kInf;
            kind[e] = !bad ? (E)0.0f : w[e] == W::kInf ? (E)1.0f : w[e] == (W::kInf | 0x8000) ? (E)64.0f : (E)4096.0f;
            v[e] = bad ? (E)0.0f : v[e];
          }
          O[nb] = W::mma(v, p[kk], O[nb]);
          const f16v count = W::mma(kind, seen, zero);
#pragma unroll
          for (int e = 0; e < 16; ++e) O[nb][e] += seen_kinds(count[e]);
        }
      }
    }
  }

  // the block's other waves may go further
  for (int st = place < 0 ? 0 : place / S::TILES + 1; st < stages; ++st) turn(st);

  const int row = place * 32 + col;
  const float inv = 1.0f / xor32_add(l);
  if (place < 0) return;
  const bool there = row < n;
  uint16_t *dst = a.out + ((int64_t)(first + row) * a.heads + head) * a.dim;
  // (a lane's four dims beside the other half's: 16 bytes a store, g even from half 0 and g + 1
  // from half 1)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      u2 w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        E r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (E)(O[nb][4 * (g + i) + e] * inv);
        __builtin_memcpy(&w[i], r, 8);
      }
      const auto x = __builtin_amdgcn_permlane32_swap(w[0].x, w[1].x, false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[0].y, w[1].y, false, false);
      const int d = 32 * nb + 8 * (g + half);
      if (there && d < a.dim) *(u4 *)(dst + d) = u4{x[0], y[0], x[1], y[1]};
    }
}

}  // namespace

hipError_t launch_prompt_attention(hipStream_t stream, const PromptArgs &a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  // workgroups, at most: every sequence's last one may be short
  const int64_t seqs = a.batch < a.rows ? a.batch : a.rows;
  const int64_t blocks = (((int64_t)a.rows + 31 * seqs) / 32 * a.gqa / kChunks + seqs) * a.kv_heads;
  const dim3 grid((unsigned)blocks), block(256);
#define PKV_PROMPT(DP_, FK_)                                                     \
  if (a.dim <= DP_ && a.float_kind == FK_) {                                     \
    hipLaunchKernelGGL((prompt_kernel<DP_, FK_>), grid, block, 0, stream, a);    \
    return hipGetLastError();                                                    \
  }
  PKV_PROMPT(64, 0) PKV_PROMPT(64, 1)
  PKV_PROMPT(128, 0) PKV_PROMPT(128, 1)
  PKV_PROMPT(256, 0) PKV_PROMPT(256, 1)
#undef PKV_PROMPT
  return hipErrorInvalidValue;
}

}  // namespace pkv
