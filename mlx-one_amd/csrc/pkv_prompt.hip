// pkv_prompt.hip -- causal attention within every sequence of packed rows.
//
//   o_i = sum_{j <= i} softmax_j(scale * q_i . k_j) v_j     per sequence and head
//
// A chunk is 32 consecutive queries of one head; the chunks of a (sequence, KV head) are
// ordered by position, then head, and a workgroup of four waves takes 4 * QB consecutive
// ones, a wave QB: with a few heads per KV head a workgroup's chunks end at nearly the same
// key.  Keys come in stages of 64 (32 beyond head dim 128), K and V copied straight to LDS
// in rows (global_load_lds), a stage ahead.
//
//   S^T = K.Q^T       v_mfma_f32_32x32x16, 32 keys x 32 queries: a lane has one query
//   O^T += V^T.P^T    the same; V^T comes out of V's rows by transposing LDS reads
//
// The contraction over keys takes a lane's scores as they lie (keys 8g + 4h + r in slot
// 8h + 4(g & 1) + r), so P never crosses lanes.  Softmax in the exp2 domain with float32
// maximum and sum; P is rounded once to the activation type, as the operand of its product
// (2^-9 relative for bfloat16, beside the output's own rounding of the same size), and summed as
// rounded, so that weights still add up to one.
//
// Only the last tiles of a wave, on the diagonal, are masked.  There a masked key's V may be
// anything: where it is not finite those elements are taken apart (a rare branch).
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
__device__ __forceinline__ int prompt_blocks(int n, int gqa, int per) {
  return n <= 0 ? 0 : ((n + 31) / 32 * gqa + per - 1) / per;
}

// The workgroup's (sequence, block): longest blocks first where the batch fits a wave's
// lanes, else sequence by sequence.  The whole wave calls.
__device__ __forceinline__ bool find_block(const PromptArgs &a, int rank, int per, int lane, int &b, int &blk) {
  if (a.batch <= 64) {
    int first;
    const int mine = lane < a.batch ? prompt_blocks(prompt_rows(a, lane, first), a.gqa, per) : 0;
    if (rank >= wave_sum(mine)) return false;
    // the largest level of which more than `rank` blocks are at or above
    int lo = 0, hi = 1;
    while (__ballot(mine >= hi)) hi <<= 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (wave_sum(max(0, mine - mid)) > rank) lo = mid;
      else hi = mid;
    }
    const int above = wave_sum(max(0, mine - lo - 1));
    unsigned long long at = __ballot(mine > lo);
    for (int i = rank - above; i > 0; --i) at &= at - 1;
    b = __ffsll((long long)at) - 1;
    blk = lo;
    return true;
  }
  int carry = 0;
  for (int c = 0; c < a.batch; c += 64) {
    int first;
    const int mine = c + lane < a.batch ? prompt_blocks(prompt_rows(a, c + lane, first), a.gqa, per) : 0;
    const int incl = wave_scan_incl(mine, lane) + carry;
    const unsigned long long hit = __ballot(incl > rank);
    if (hit) {
      const int f = __ffsll((long long)hit) - 1;
      b = c + f;
      blk = __builtin_amdgcn_readlane(incl, f) - 1 - rank;
      return true;
    }
    carry = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

__device__ __forceinline__ void barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}

// A lane's V^T operand (dim 32 nb + col, 16 keys) out of V's rows in LDS.
template <int DP, typename T>
__device__ __forceinline__ T v_operand(const uint8_t *src) {
  typedef short s4v __attribute__((ext_vector_type(4)));
  struct { s4v lo, hi; } v;
  v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)src);
  v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)(src + 8 * DP * 2));
  return __builtin_bit_cast(T, v);
}

template <int DP, int FK, int QB>
__global__ __launch_bounds__(256, 1) void prompt_kernel(const PromptArgs a) {
  using W = Wide<FK>;
  using T = typename W::T;
  using E = typename W::E;
  using S = PromptShape<DP>;
  constexpr int KS = DP / 16, NB = DP / 32, PER = 4 * QB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[S::BYTES];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int kh = blockIdx.x % a.kv_heads;
  int b, blk;
  if (!find_block(a, blockIdx.x / a.kv_heads, PER, lane, b, blk)) return;
  b = __builtin_amdgcn_readfirstlane(b);
  blk = __builtin_amdgcn_readfirstlane(blk);
  int first;
  const int n = prompt_rows(a, b, first);
  const int chunks = (n + 31) / 32 * a.gqa;

  // the wave's chunks, rising; -1: none
  int place[QB], head[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int c = blk * PER + wave * QB + i;
    place[i] = c < chunks ? c / a.gqa : -1;
    head[i] = kh * a.gqa + c % a.gqa;
  }
  const int last = (min(chunks, (blk + 1) * PER) - 1) / a.gqa;  // 32-key tile of the block's last chunk
  const int stages = last / S::TILES + 1;
  // the wave's last tile, and its first with a mask (a wave without chunks has no tile)
  const int top = max(place[0], place[QB - 1]), clear = place[0];

  // ---- K and V rows to LDS: thread tid copies unit tid + 256 i of a stage
  const uint8_t *kbase = (const uint8_t *)(a.k + (int64_t)first * a.k_stride + kh * a.dim);
  const uint8_t *vbase = (const uint8_t *)(a.v + (int64_t)first * a.v_stride + kh * a.dim);
  uint32_t krow[S::COPIES], kat[S::COPIES], vat[S::COPIES];  // row; byte offsets from the stage's first row
  uint32_t live = 0;                                         // units within the head dim
#pragma unroll
  for (int i = 0; i < S::COPIES; ++i) {
    const int at = tid + 256 * i, m = at / S::UNITS;
    const int ku = k_unit<DP>(m, at % S::UNITS), vu = v_unit<DP>(m, at % S::UNITS);
    krow[i] = m;
    kat[i] = m * (uint32_t)a.k_stride * 2 + ku * 16;
    vat[i] = m * (uint32_t)a.v_stride * 2 + vu * 16;
    live |= (ku < a.dim / 8 ? 1u : 0u) << (2 * i) | (vu < a.dim / 8 ? 2u : 0u) << (2 * i);
  }
  auto copy = [&](int s) __attribute__((always_inline)) {
    uint8_t *kdst = lds + s % S::KBUF * S::SIDE + wave * 1024;
    uint8_t *vdst = lds + (S::KBUF + s % S::VBUF) * S::SIDE + wave * 1024;
    const uint8_t *ksrc = kbase + (int64_t)s * S::KEYS * a.k_stride * 2;
    const uint8_t *vsrc = vbase + (int64_t)s * S::KEYS * a.v_stride * 2;
    auto unit = [](const uint8_t *from, uint8_t *to) __attribute__((always_inline)) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)from,
                                       (__attribute__((address_space(3))) uint32_t *)to, 16, 0, 0);
    };
    if (a.dim == DP && (s + 1) * S::KEYS <= n) {  // whole rows, all of them there
#pragma unroll
      for (int i = 0; i < S::COPIES; ++i) {
        unit(ksrc + kat[i], kdst + i * 4096);
        unit(vsrc + vat[i], vdst + i * 4096);
      }
      return;
    }
    // rows past the last one read it again (their keys are masked)
    const int rows = n - s * S::KEYS;
#pragma unroll
    for (int i = 0; i < S::COPIES; ++i) {
      const int64_t past = max((int)krow[i] - (rows - 1), 0);
      if (live >> (2 * i) & 1) unit(ksrc + kat[i] - past * a.k_stride * 2, kdst + i * 4096);
      if (live >> (2 * i) & 2) unit(vsrc + vat[i] - past * a.v_stride * 2, vdst + i * 4096);
    }
  };
  if (a.dim < DP) {  // the units past the head dim hold zeros
    for (int i = tid; i < S::BYTES / 16; i += 256) *((u4 *)lds + i) = u4{0, 0, 0, 0};
    barrier();
  }

  copy(0);

  // ---- queries: lane (col, half) holds elements 16 ks + 8 half + e of query col
  T q[QB][KS];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int64_t row = first + min(max(place[i], 0) * 32 + col, n - 1);
    const uint16_t *src = a.q + row * a.q_stride + (int64_t)head[i] * a.dim;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d = 16 * ks + 8 * half;
      u4 x = {0, 0, 0, 0};
      if (d < a.dim && place[i] >= 0) x = *(const u4 *)(src + d);
      q[i][ks] = __builtin_bit_cast(T, x);
      // (accumulation registers: the MFMAs take them from there as operands, and the vector
      // registers are left to O and the scores)
      asm("" : "+a"(q[i][ks]));
    }
  }

  float m[QB], thr[QB], l[QB];
  f16v O[QB][NB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    m[i] = l[i] = 0.0f;
    thr[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) O[i][j][e] = 0.0f;
  }
  int koff[KS], voff[NB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) koff[ks] = (col * S::UNITS + k_unit<DP>(col, 2 * ks + half)) * 16;
  {
    const int i = lane & 15, j = (lane >> 4) & 1, r = 4 * half + i / 4;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      voff[nb] = (r * S::UNITS + v_unit<DP>(r, 4 * nb + 2 * j + (i & 3) / 2)) * 16 + 8 * (i & 1);
  }

  // S^T = K.Q^T of a tile.  (From zeros in registers: an MFMA with an inline constant 0 as
  // its accumulator has given wrong results where its destination partly overlaps an operand.)
  f16v zero = {0};
  asm volatile("" : "+v"(zero));
  auto scores = [&](const uint8_t *ktile, f16v (&x)[QB]) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const T k = __builtin_bit_cast(T, *(const u4 *)(ktile + koff[ks]));
#pragma unroll
      for (int i = 0; i < QB; ++i) x[i] = W::mma(k, q[i][ks], ks == 0 ? zero : x[i]);
    }
  };
  // the exponents, less the running maximum: it moves when a score passes it by kTau
  auto settle = [&](auto masks, f16v (&x)[QB], int at) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[i][e] = __builtin_fmaf(x[i][e], a.scale_log2, -m[i]);
    // key 8g + 4 half + r of the tile is seen by the queries from it on
    if constexpr (decltype(masks)::value) {
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        const int sees = (place[i] - at) * 32 + col - 4 * half;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[i][e] = 8 * (e / 4) + e % 4 <= sees ? x[i][e] : -INFINITY;
      }
    }
    float mx[QB];
    bool need = false;
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      mx[i] = x[i][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx[i] = __builtin_elementwise_maximum(mx[i], x[i][e]);
      need |= mx[i] > thr[i];
    }
    if (__builtin_expect(__any(need), 0)) {
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        const float up = xor32_max(mx[i]);
        const bool moves = up > thr[i];
        const float by = moves ? up : 0.0f;
        const float alpha = !moves ? 1.0f : thr[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-up);
        m[i] += by;
        thr[i] = moves ? kTau : thr[i];
        l[i] *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[i][e] -= by;
#pragma unroll
        for (int j = 0; j < NB; ++j) O[i][j] *= alpha;
      }
    }
  };
  // the weights as operands, and their sums
  auto weights = [&](const f16v (&x)[QB], T (&p)[QB][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < QB; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const E r0 = (E)__builtin_amdgcn_exp2f(x[i][e]), r1 = (E)__builtin_amdgcn_exp2f(x[i][e + 1]);
        p[i][e / 8][e % 8] = r0;
        p[i][e / 8][e % 8 + 1] = r1;
        l[i] = W::add(r0, r1, l[i]);
      }
  };
  auto product = [&](const uint8_t *vtile, const T (&p)[QB][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const T v = v_operand<DP, T>(vtile + kk * 16 * DP * 2 + voff[nb]);
#pragma unroll
        for (int i = 0; i < QB; ++i) O[i][nb] = W::mma(v, p[i][kk], O[i][nb]);
      }
  };
  auto ktile = [&](int at) __attribute__((always_inline)) {
    return lds + at / S::TILES % S::KBUF * S::SIDE + at % S::TILES * 32 * DP * 2;
  };
  auto vtile = [&](int at) __attribute__((always_inline)) {
    return lds + (S::KBUF + at / S::TILES % S::VBUF) * S::SIDE + at % S::TILES * 32 * DP * 2;
  };
  // stage s is here; everyone is done with the scores of stage s - 1 and the products of
  // stage s - 2, whose places the next stage takes
  auto turn = [&](int s) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    barrier();
    if (s + 1 < stages) copy(s + 1);
  };

  // ---- tiles that the wave's queries see whole, two at a time: a tile's weights and
  // product go beside the next one's scores
  const int whole = max(clear, 0) & ~1;
  if (whole > 0) {
    f16v x[QB];
    turn(0);
    scores(ktile(0), x);
    settle(std::false_type{}, x, 0);
    f16v y[QB];
    T p[QB][2];
    int at = 1;
    for (; at + 1 < whole; at += 2) {
      if (S::TILES == 1) turn(at);
      scores(ktile(at), y);
      weights(x, p);
      product(vtile(at - 1), p);
      settle(std::false_type{}, y, at);
      turn((at + 1) / S::TILES);
      scores(ktile(at + 1), x);
      weights(y, p);
      product(vtile(at), p);
      settle(std::false_type{}, x, at + 1);
    }
    if (S::TILES == 1) turn(at);
    scores(ktile(at), y);
    weights(x, p);
    product(vtile(at - 1), p);
    settle(std::false_type{}, y, at);
    weights(y, p);
    product(vtile(at), p);
  }
  // ---- and the rest
  for (int at = whole; at < stages * S::TILES; ++at) {
    if (at % S::TILES == 0) turn(at / S::TILES);
    if (at > top) continue;
    f16v x[QB];
    T p[QB][2];
    scores(ktile(at), x);
    settle(std::true_type{}, x, at);
    weights(x, p);
    bool odd = false;  // infinities or NaN among the tile's values?
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const u4 w = __builtin_bit_cast(u4, v_operand<DP, T>(vtile(at) + kk * 16 * DP * 2 + voff[nb]));
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= (w[e] & 0x7FFFu) >= W::kInf || (w[e] >> 16 & 0x7FFFu) >= W::kInf;
      }
    if (__builtin_expect(!__any(odd), 1)) {
      product(vtile(at), p);
    } else {
      // their products with the masked keys' zero weights must not be NaN: the finite
      // values go through the product; of the others, kind by kind, the keys that a
      // query sees are counted by one
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        const int sees = (place[i] - at) * 32 + col - 4 * half;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          T seen;
#pragma unroll
          for (int e = 0; e < 8; ++e) seen[e] = 8 * (2 * kk + e / 4) + e % 4 <= sees ? (E)1.0f : (E)0.0f;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const T v = v_operand<DP, T>(vtile(at) + kk * 16 * DP * 2 + voff[nb]);
            uint16_t w[8];
            __builtin_memcpy(w, &v, 16);
            T part = v;
#pragma unroll
            for (int e = 0; e < 8; ++e) part[e] = (w[e] & 0x7FFF) >= W::kInf ? (E)0.0f : part[e];
            O[i][nb] = W::mma(part, p[i][kk], O[i][nb]);
#pragma unroll 1
            for (int kind = 0; kind < 3; ++kind) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const bool hit = kind == 2 ? (w[e] & 0x7FFF) > W::kInf : w[e] == (W::kInf | (kind << 15));
                part[e] = hit ? (E)1.0f : (E)0.0f;
              }
              const f16v count = W::mma(part, seen, zero);
              const float what = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : __builtin_nanf("");
#pragma unroll
              for (int e = 0; e < 16; ++e) O[i][nb][e] += count[e] > 0.0f ? what : 0.0f;
            }
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int row = place[i] * 32 + col;
    const float inv = 1.0f / xor32_add(l[i]);
    if (place[i] < 0 || row >= n) continue;
    uint16_t *dst = a.out + ((int64_t)(first + row) * a.heads + head[i]) * a.dim;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * nb + 8 * g + 4 * half;
        if (d >= a.dim) continue;
        E r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (E)(O[i][nb][4 * g + e] * inv);
        u2 w;
        __builtin_memcpy(&w, r, 8);
        *(u2 *)(dst + d) = w;
      }
  }
}

template <int QB>
hipError_t launch(hipStream_t stream, const PromptArgs &a, int64_t blocks) {
  const dim3 grid((unsigned)blocks), block(256);
#define PKV_PROMPT(DP_, FK_, QB_)                                                            \
  if (a.dim <= DP_ && a.float_kind == FK_) {                                                 \
    hipLaunchKernelGGL((prompt_kernel<DP_, FK_, QB_>), grid, block, 0, stream, a);           \
    return hipGetLastError();                                                                \
  }
  PKV_PROMPT(64, 0, QB) PKV_PROMPT(64, 1, QB)
  PKV_PROMPT(128, 0, QB) PKV_PROMPT(128, 1, QB)
  PKV_PROMPT(256, 0, 1) PKV_PROMPT(256, 1, 1)
#undef PKV_PROMPT
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_prompt_attention(hipStream_t stream, const PromptArgs &a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  // workgroups, at most: every sequence's last one may be short
  auto blocks = [&](int per) {
    const int64_t seqs = a.batch < a.rows ? a.batch : a.rows;
    return (((int64_t)a.rows + 31 * seqs) / 32 * a.gqa / per + seqs) * a.kv_heads;
  };
  const bool wide = a.dim <= 128 && blocks(8) >= 512;
  if (wide) return launch<2>(stream, a, blocks(8));
  return launch<1>(stream, a, blocks(4));
}

}  // namespace pkv
