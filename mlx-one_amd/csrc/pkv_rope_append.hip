// pkv_rope_append.hip -- rotate the q and k heads of a fused projection, store k and v
// into the sequences' pages and q (k, v) beside them, in one pass over the projection.
//
//   angle_i = p_{axis(i)} * inv_freq_i                     i < half, in 64 bits
//   y_i = x_i cos - x_{i+half} sin, y_{i+half} = x_{i+half} cos + x_i sin
//
// cos and sin are rounded to 32 bits once, products and sums rounded one by one in
// 32 bits, the result once to the activation type; k is quantized from that, so a page
// holds what append_quantize makes of the k that comes out.  (Angles in 32 bits are
// off by up to 2^-24 of themselves, 0.008 rad at position 131072.)
//
// Memory-bound: a row of (H + 2 HK) D elements is read once, H D elements and the
// pages' bytes are written.  Two kernels, as for the append:
//  * rows kernel: a wave per (row, q head) or (row, KV head).  Any dims and strides.
//  * tiles kernel: a workgroup per 16-token tile of the cache and run of heads; 16-byte
//    loads and stores, K and V tiles stored in whole payload chunks.
// 24K rows of 48 heads into 8-bit pages, k and v returned: 154 us, 4.35 TB/s (a copy: 4.9); 64
// next tokens: 5.8 us on the device.
#include <algorithm>

#include "pkv_step.h"
#include "pkv_tile_store.h"

namespace pkv {

namespace {

// cos and sin of x (any finite x below 2^52), each rounded to 32 bits.  Cody-Waite
// reduction by pi/2 in two parts (106 bits) and the Taylor polynomials on
// [-pi/4, pi/4], to x^15 and x^16 (remainders below 5e-17): the error in 64 bits is about
// 2e-16, so the rounding to 32 bits is the correct one but for a few in 10^8.
__device__ __forceinline__ void cos_sin(double x, float &c, float &s) {
  const double k = __builtin_rint(x * 0.63661977236758134308);
  double r = __builtin_fma(-k, 1.57079632679489655800, x);
  r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double p = -1.0 / 1307674368000.0;                 // 15!
  p = __builtin_fma(p, z, 1.0 / 6227020800.0);       // 13!
  p = __builtin_fma(p, z, -1.0 / 39916800.0);        // 11!
  p = __builtin_fma(p, z, 1.0 / 362880.0);           // 9!
  p = __builtin_fma(p, z, -1.0 / 5040.0);            // 7!
  p = __builtin_fma(p, z, 1.0 / 120.0);              // 5!
  p = __builtin_fma(p, z, -1.0 / 6.0);
  const double sine = __builtin_fma(p * z, r, r);
  double q = 1.0 / 20922789888000.0;                 // 16!
  q = __builtin_fma(q, z, -1.0 / 87178291200.0);     // 14!
  q = __builtin_fma(q, z, 1.0 / 479001600.0);        // 12!
  q = __builtin_fma(q, z, -1.0 / 3628800.0);         // 10!
  q = __builtin_fma(q, z, 1.0 / 40320.0);            // 8!
  q = __builtin_fma(q, z, -1.0 / 720.0);
  q = __builtin_fma(q, z, 1.0 / 24.0);
  q = __builtin_fma(q, z, -0.5);
  const double cosine = __builtin_fma(q, z, 1.0);
  const int quarter = (int)(k - 4.0 * __builtin_floor(k * 0.25));
  const double a = quarter & 1 ? sine : cosine, b = quarter & 1 ? cosine : sine;
  c = (float)((quarter + 1) & 2 ? -a : a);
  s = (float)(quarter & 2 ? -b : b);
}

// y = (x0, x1) turned; every product and sum rounded by itself.
__device__ __forceinline__ void turn(float x0, float x1, float c, float s, float &y0, float &y1) {
#pragma clang fp contract(off)
  y0 = x0 * c - x1 * s;
  y1 = x1 * c + x0 * s;
}

// Rows of sequence b: first one and count, and the cache position of the first.  No
// rows where positions would not be numbers of a cache.
__device__ __forceinline__ int seq_rows(const RopeAppendArgs &a, int b, int &first, int &start) {
  int n;
  if (a.row_starts) {
    first = min(max(a.row_starts[b], 0), a.rows);
    n = min(a.row_starts[b + 1], a.rows) - first;
  } else {
    first = b * a.tokens;
    n = a.widths ? min(a.widths[b], a.tokens) : a.tokens;
  }
  start = a.start_pos[b];
  return start < 0 || start > 0x7FFFFFFF - max(n, 0) ? 0 : n;
}

// The position of row `row` (token i of a sequence that starts at `start`) for pair j.
__device__ __forceinline__ int pair_position(const RopeAppendArgs &a, int row, int at, int j) {
  if (!a.positions) return at;
  const int axis = a.axis ? a.axis[j] : 0;
  return a.positions[(int64_t)min(max(axis, 0), a.axes - 1) * a.rows + row];
}

// Where head h of token i of sequence b goes in an output of `heads` heads.
__device__ __forceinline__ int64_t out_at(const RopeAppendArgs &a, int heads, int b, int row, int i, int h) {
  const int64_t place = a.row_starts ? (int64_t)row * heads + h : ((int64_t)b * heads + h) * a.tokens + i;
  return place * a.g.dim;
}

// ---- a wave per (row, q head) or (row, KV head) ----------------------------------------

constexpr int kMaxPairs = 2;  // pairs per lane: head dims of at most 256

template <int DP, int BITS>
__global__ __launch_bounds__(256) void rope_append_rows_kernel(const RopeAppendArgs a) {
  constexpr int EPL = DP / 64;
  __shared__ __attribute__((aligned(16))) uint16_t s_row[4][DP];
  __shared__ __attribute__((aligned(16))) uint8_t s_codes[4][2][DP];
  __shared__ uint32_t s_meta[4][2][8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Geo &g = a.g;
  const int row = blockIdx.x;
  const int item = blockIdx.y * 4 + wave;  // q heads, then KV heads
  if (item >= a.heads + g.hk) return;
  const int kh = item - a.heads;
  const uint16_t *src = a.qkv + (int64_t)row * a.row_stride + (int64_t)item * g.dim;
  // the head's pairs (and, for a KV head, v): requested before the row's place is known
  uint16_t x0[kMaxPairs], x1[kMaxPairs], rest[EPL], vraw[EPL];
#pragma unroll
  for (int j = 0; j < kMaxPairs; ++j) {
    const int i = lane + 64 * j;
    x0[j] = i < a.half ? src[i] : (uint16_t)0;
    x1[j] = i < a.half ? src[i + a.half] : (uint16_t)0;
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int d = 2 * a.half + lane + 64 * j;
    rest[j] = d < g.dim ? src[d] : (uint16_t)0;
    const int e = lane * EPL + j;
    vraw[j] = kh >= 0 && e < g.dim ? src[(int64_t)g.hk * g.dim + e] : (uint16_t)0;
  }
  // the row's sequence: the starts at or below the row, counted
  int b;
  if (a.row_starts) {
    int n = 0;
    for (int c = 0; c < a.batch; c += 64)
      n += __popcll(__ballot(c + lane < a.batch && a.row_starts[c + lane] <= row));
    b = n - 1;
    // (empty sequences share their successor's start: the last one at or below has the row)
    if (b < 0) return;
  } else {
    b = row / a.tokens;
  }
  int first, start;
  const int n = seq_rows(a, b, first, start);
  const int i = row - first;
  if (i < 0 || i >= n) return;
  const int pos = start + i;
  int page = -1;
  if (kh >= 0 && pos / g.page < a.max_pages) page = a.table[(int64_t)b * a.max_pages + pos / g.page];
  uint16_t *dst = nullptr;
  if (kh < 0) dst = a.q + out_at(a, a.heads, b, row, i, item);
  else if (a.k) dst = a.k + out_at(a, g.hk, b, row, i, kh);
#pragma unroll
  for (int j = 0; j < kMaxPairs; ++j) {
    const int p = lane + 64 * j;
    if (p >= a.half) continue;
    float c, s, y0, y1;
    cos_sin((double)pair_position(a, row, pos, p) * (double)a.inv_freq[p], c, s);
    turn(bits_to_float(x0[j], g.float_kind), bits_to_float(x1[j], g.float_kind), c, s, y0, y1);
    const uint16_t r0 = float_to_bits(y0, g.float_kind), r1 = float_to_bits(y1, g.float_kind);
    if (dst) {
      dst[p] = r0;
      dst[p + a.half] = r1;
    }
    s_row[wave][p] = r0;
    s_row[wave][p + a.half] = r1;
  }
#pragma unroll
  for (int j = 0; j < EPL; ++j) {
    const int d = 2 * a.half + lane + 64 * j;
    if (d >= DP) continue;
    s_row[wave][d] = rest[j];  // zeros past the head dim
    if (dst && d < g.dim) dst[d] = rest[j];
  }
  if (kh < 0) return;
  if (a.v) {
    uint16_t *vdst = a.v + out_at(a, g.hk, b, row, i, kh);
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (lane * EPL + j < g.dim) vdst[lane * EPL + j] = vraw[j];
  }
  if (page < 0 || page >= a.num_pages) return;
  wave_lds_sync();
  uint16_t kraw[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) kraw[j] = s_row[wave][lane * EPL + j];
  const int slot = pos % g.page, tt = slot % PKV_TILE;
  uint8_t *head = a.pool + (int64_t)page * g.page_bytes + (int64_t)kh * g.head_bytes;
  if constexpr (BITS == 16) {
    uint8_t *ktile = head + (int64_t)(slot / PKV_TILE) * g.tile_bytes, *vtile = ktile + g.v_offset;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int d = lane * EPL + j;
      *(uint16_t *)(ktile + payload_offset(tt + 16 * (d % 32 / 8), 2 * (8 * (d / 32) + d % 8), 16)) = kraw[j];
      *(uint16_t *)(vtile + payload_offset(d % 16 + 16 * (tt / 4), 2 * (4 * (d / 16) + tt % 4), 16)) = vraw[j];
    }
  } else {
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      float x[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) x[j] = bits_to_float(side ? vraw[j] : kraw[j], g.float_kind);
      quantize_row<EPL>(x, lane, g.group, BITS, s_codes[wave][side], s_meta[wave][side]);
    }
    wave_lds_sync();
    store_token<DP, BITS>(g, head, slot, s_codes[wave][0], s_codes[wave][1], s_meta[wave][0], s_meta[wave][1], lane);
  }
}

// ---- a workgroup per 16-token tile and run of heads ------------------------------------------

// The tile-th tile that new tokens touch, counted over the sequences; false past the
// last.  The whole wave calls.
__device__ __forceinline__ bool find_tile(const RopeAppendArgs &a, int tile, int lane, int &b, int &nth) {
  int carry = 0;
  for (int c = 0; c < a.batch; c += 64) {
    int count = 0;
    if (c + lane < a.batch) {
      int first, start;
      const int n = seq_rows(a, c + lane, first, start);
      if (n > 0) count = (start + n - 1) / PKV_TILE - start / PKV_TILE + 1;
    }
    const int incl = wave_scan_incl(count, lane) + carry;
    const unsigned long long hit = __ballot(incl > tile);
    if (hit) {
      const int f = __ffsll((long long)hit) - 1;
      b = c + f;
      nth = tile - (__builtin_amdgcn_readlane(incl, f) - __builtin_amdgcn_readlane(count, f));
      return true;
    }
    carry = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// u / d for u < 2^11 by one product: inv = ceil(2^20 / d) is off by less than d <= 2^7 of 2^-20.
__device__ __forceinline__ uint32_t inverse(int d) { return d > 0 ? ((1u << 20) + d - 1) / d : 0; }
__device__ __forceinline__ int over(int u, uint32_t inv) { return (int)((uint32_t)u * inv >> 20); }

template <int DP, int G, int BITS, int FK>
__global__ __launch_bounds__(256) void rope_append_tiles_kernel(const RopeAppendArgs a, int per_wave) {
  constexpr int KB = DP / 32;
  constexpr int ROW = DP + 8;  // rows of a K tile in LDS, 16 bytes apart
  constexpr int VW = tile_row_words<DP, BITS>();
  // a token's angles: the first four of every eight, then the last four, so that units are 16
  // bytes apart; rows a quarter of the banks further on
  __shared__ __attribute__((aligned(16))) float s_cos[PKV_TILE][DP / 2 + 16], s_sin[PKV_TILE][DP / 2 + 16];
  __shared__ __attribute__((aligned(16))) uint32_t s_buf[4][16 * (ROW / 2 > VW ? ROW / 2 : VW)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Geo g = a.g;
  g.float_kind = FK;
  int b, nth;
  if (!find_tile(a, blockIdx.x, lane, b, nth)) return;
  int first, start;
  const int n = seq_rows(a, b, first, start);
  const int pos0 = (start / PKV_TILE + nth) * PKV_TILE;
  const int rel = pos0 - start;  // the tile's token t is the sequence's new token rel + t
  const int page = pos0 / g.page < a.max_pages ? a.table[(int64_t)b * a.max_pages + pos0 / g.page] : -1;
  const uint32_t by_half = inverse(a.half);
  for (int u = threadIdx.x; u < PKV_TILE * a.half; u += 256) {
    const int t = over(u, by_half), j = u - t * a.half;
    if (rel + t < 0 || rel + t >= n) continue;
    const int at = (j & 4 ? a.half / 2 : 0) + (j >> 3) * 4 + (j & 3);
    cos_sin((double)pair_position(a, first + rel + t, pos0 + t, j) * (double)a.inv_freq[j], s_cos[t][at], s_sin[t][at]);
  }
  __syncthreads();
  const int lo = max(0, -rel), hi = min(PKV_TILE, n - rel);  // the tile's new tokens
  const int pairs = a.half / 8, plain = (g.dim - 2 * a.half) / 8;  // 16-byte units per token
  const uint32_t by_pairs = inverse(pairs), by_plain = inverse(plain);
  const int all = a.heads + 2 * g.hk;
  for (int i = 0; i < per_wave; ++i) {
    const int h = (blockIdx.y * per_wave + i) * 4 + wave;
    if (h >= all) return;
    const uint16_t *src0 = a.qkv + (int64_t)(first + rel) * a.row_stride + (int64_t)h * g.dim;
    const int kh = h < a.heads + g.hk ? h - a.heads : h - a.heads - g.hk;
    const bool is_q = h < a.heads, is_v = h >= a.heads + g.hk;
    uint16_t *out = is_q ? a.q : is_v ? a.v : a.k;
    const int out_heads = is_q ? a.heads : g.hk, out_head = is_q ? h : kh;
    uint8_t *head = a.pool + (int64_t)max(page, 0) * g.page_bytes + (int64_t)max(kh, 0) * g.head_bytes;
    const bool mapped = page >= 0 && page < a.num_pages;
    const int t16 = lane & 15, jj = lane >> 4;
    u4 raw[KB];
    if (is_v) {
      const bool mine = t16 >= lo && t16 < hi;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int d0 = 32 * kb + 8 * jj;
        raw[kb] = u4{0, 0, 0, 0};
        if (mine && d0 < g.dim) raw[kb] = *(const u4 *)(src0 + (int64_t)t16 * a.row_stride + d0);
      }
      if (out && mine) {
        uint16_t *dst = out + out_at(a, out_heads, b, first + rel + t16, rel + t16, out_head);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          if (32 * kb + 8 * jj < g.dim) *(u4 *)(dst + 32 * kb + 8 * jj) = raw[kb];
      }
    } else {
      uint16_t *rows = (uint16_t *)s_buf[wave];
      if (!is_q) wave_lds_sync();  // (the last head's reads of the buffer are done)
      // (two units' loads under way at a time)
      for (int u0 = lane; u0 < PKV_TILE * pairs; u0 += 128) {
        int t[2], c[2];
        bool mine[2];
        u4 w[2][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int u = u0 + 64 * k;
          t[k] = over(u, by_pairs);
          c[k] = u - t[k] * pairs;
          mine[k] = t[k] >= lo && t[k] < hi;
          if (!mine[k]) continue;
          const uint16_t *src = src0 + (int64_t)t[k] * a.row_stride + 8 * c[k];
          w[k][0] = *(const u4 *)src;
          w[k][1] = *(const u4 *)(src + a.half);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (!mine[k]) continue;
          uint16_t x0[8], x1[8], y0[8], y1[8];
          __builtin_memcpy(x0, &w[k][0], 16);
          __builtin_memcpy(x1, &w[k][1], 16);
          f4 cs[2], sn[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            cs[i] = *(const f4 *)&s_cos[t[k]][i * (a.half / 2) + 4 * c[k]];
            sn[i] = *(const f4 *)&s_sin[t[k]][i * (a.half / 2) + 4 * c[k]];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float f0, f1;
            turn(bits_to_float(x0[e], FK), bits_to_float(x1[e], FK), cs[e / 4][e % 4], sn[e / 4][e % 4], f0, f1);
            y0[e] = float_to_bits(f0, FK);
            y1[e] = float_to_bits(f1, FK);
          }
          u4 o0, o1;
          __builtin_memcpy(&o0, y0, 16);
          __builtin_memcpy(&o1, y1, 16);
          if (out) {
            uint16_t *dst = out + out_at(a, out_heads, b, first + rel + t[k], rel + t[k], out_head) + 8 * c[k];
            *(u4 *)dst = o0;
            *(u4 *)(dst + a.half) = o1;
          }
          if (!is_q) {
            *(u4 *)(rows + t[k] * ROW + 8 * c[k]) = o0;
            *(u4 *)(rows + t[k] * ROW + a.half + 8 * c[k]) = o1;
          }
        }
      }
      for (int u = lane; u < PKV_TILE * plain; u += 64) {
        const int t = over(u, by_plain), d = 2 * a.half + 8 * (u - t * plain);
        if (t < lo || t >= hi) continue;
        const u4 w = *(const u4 *)(src0 + (int64_t)t * a.row_stride + d);
        if (out) *(u4 *)(out + out_at(a, out_heads, b, first + rel + t, rel + t, out_head) + d) = w;
        if (!is_q) *(u4 *)(rows + t * ROW + d) = w;
      }
      if (is_q) continue;
      wave_lds_sync();
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int d0 = 32 * kb + 8 * jj;
        raw[kb] = u4{0, 0, 0, 0};
        if (t16 >= lo && t16 < hi && d0 < g.dim) raw[kb] = *(const u4 *)(rows + t16 * ROW + d0);
      }
      wave_lds_sync();
    }
    if (mapped) store_tile_side<DP, G, BITS>(g, head, pos0 % g.page, is_v ? 1 : 0, raw, rel, n, s_buf[wave], lane);
    wave_lds_sync();
  }
}

}  // namespace

// Workgroups to leave of a tile kernel's launch.  10K rows of 20 heads (670 tiles): 30 us at two
// workgroups to a tile, 31 at three, 36 at five; 24K rows of 48 heads (1524): 168 at one, 162 at
// two, 166 at three.
constexpr int kLeast = 1536;

hipError_t launch_rope_append(hipStream_t stream, const RopeAppendArgs &a) {
  if (a.rows == 0 || a.batch == 0) return hipSuccess;
  const dim3 block(256);
  // 16-byte units: heads, halves and rows of whole ones at aligned addresses
  const uintptr_t at = (uintptr_t)a.qkv | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
  const bool vec = a.g.dim % 8 == 0 && a.half % 8 == 0 && a.row_stride % 8 == 0 && (at & 15) == 0;
  // Tiles from 8 rows a sequence and 128 in all: 64 sequences of 4 rows 10.3 us by tiles and 8.5 by rows,
  // of 8 rows 11.1 and 13.5, of 32 rows 19.2 and 41.8; 4 sequences of 16 rows 7.0 and 5.2, of 64 7.6 and
  // 8.5 (8-bit pages, 32 and 8 heads of 128).
  if (vec && a.rows >= 128 && (int64_t)a.rows >= 8 * (int64_t)a.batch) {
    const int tiles = (a.rows + PKV_TILE - 1) / PKV_TILE + 2 * (a.batch < a.rows ? a.batch : a.rows);
    const int all = a.heads + 2 * a.g.hk;
    // A workgroup computes its tile's angles for all its heads: as many heads as leave
    // kLeast workgroups, so that six may be on each CU.
    int per_wave = 1;
    while (4 * per_wave < all && (int64_t)tiles * ((all + 4 * per_wave + 3) / (4 * per_wave + 4)) >= kLeast) ++per_wave;
    const dim3 grid(tiles, (all + 4 * per_wave - 1) / (4 * per_wave));
#define PKV_TILES(DP_, G_, BITS_)                                                                    \
  if (a.g.dp == DP_ && a.g.bits == BITS_ && (BITS_ == 16 || a.g.group == G_)) {                      \
    if (a.g.float_kind == 1)                                                                         \
      hipLaunchKernelGGL((rope_append_tiles_kernel<DP_, G_, BITS_, 1>), grid, block, 0, stream, a, per_wave); \
    else                                                                                             \
      hipLaunchKernelGGL((rope_append_tiles_kernel<DP_, G_, BITS_, 0>), grid, block, 0, stream, a, per_wave); \
    return hipGetLastError();                                                                        \
  }
#define PKV_TILES_Q(DP_, G_) PKV_TILES(DP_, G_, 4) PKV_TILES(DP_, G_, 8)
    PKV_TILES(64, 32, 16) PKV_TILES(128, 32, 16) PKV_TILES(256, 32, 16)
    PKV_TILES_Q(64, 32) PKV_TILES_Q(64, 64)
    PKV_TILES_Q(128, 32) PKV_TILES_Q(128, 64) PKV_TILES_Q(128, 128)
    PKV_TILES_Q(256, 32) PKV_TILES_Q(256, 64) PKV_TILES_Q(256, 128)
#undef PKV_TILES_Q
#undef PKV_TILES
    return hipErrorInvalidValue;
  }
  const dim3 grid(a.rows, (a.heads + a.g.hk + 3) / 4);
#define PKV_ROWS(DP_, BITS_)                                                              \
  if (a.g.dp == DP_ && a.g.bits == BITS_) {                                               \
    hipLaunchKernelGGL((rope_append_rows_kernel<DP_, BITS_>), grid, block, 0, stream, a); \
    return hipGetLastError();                                                             \
  }
  PKV_ROWS(64, 4) PKV_ROWS(64, 8) PKV_ROWS(64, 16)
  PKV_ROWS(128, 4) PKV_ROWS(128, 8) PKV_ROWS(128, 16)
  PKV_ROWS(256, 4) PKV_ROWS(256, 8) PKV_ROWS(256, 16)
#undef PKV_ROWS
  return hipErrorInvalidValue;
}

}  // namespace pkv
