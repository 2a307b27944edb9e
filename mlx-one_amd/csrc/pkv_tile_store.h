// pkv_tile_store.h -- quantize one side (K or V) of a 16-token page tile and store
// it, one wave per tile side (device functions shared by the append kernels).
#pragma once
#include "pkv_token.h"

namespace pkv {

// Quantize the lane's share of its token's row: meta words of every storage
// group and the codes, 8 per kb, as two words of four bytes.  The whole wave
// calls.
template <int DP, int G, int BITS, int FK>
__device__ __forceinline__ void quantize_share(const u4 (&raw)[DP / 32], uint32_t (&meta)[DP / G],
                                               uint32_t (&codes)[DP / 16]) {
  constexpr int NG = DP / G, KPG = G / 32;
  const float levels = (float)((1 << BITS) - 1);
  float lo[NG], hi[NG], bias[NG], scale[NG];
  auto affine = [&](int gi) __attribute__((always_inline)) {
    const uint16_t b16 = f32_to_f16_bits(lo[gi]);
    bias[gi] = f16_bits_to_f32(b16);
    const uint16_t s16 = f32_to_f16_bits(fmaxf(__fdiv_rn(hi[gi] - bias[gi], levels), 1e-6f));
    scale[gi] = f16_bits_to_f32(s16);
    meta[gi] = (uint32_t)s16 | ((uint32_t)b16 << 16);
  };
  // min and max by the NaN-propagating three-input forms (half the operations
  // of fminf / fmaxf, and no canonicalisation)
  bool odd = false;
#pragma unroll
  for (int gi = 0; gi < NG; ++gi) {
    float l = 0.0f, h = 0.0f;
#pragma unroll
    for (int k = 0; k < KPG; ++k) {
      float x[8];
      unpack8<FK>(raw[gi * KPG + k], x);
      if (k == 0) l = h = x[0];
      minmax8(x, l, h);
    }
    l = __builtin_elementwise_minimum(l, __shfl_xor(l, 16, 64));
    h = __builtin_elementwise_maximum(h, __shfl_xor(h, 16, 64));
    lo[gi] = __builtin_elementwise_minimum(l, __shfl_xor(l, 32, 64));
    hi[gi] = __builtin_elementwise_maximum(h, __shfl_xor(h, 32, 64));
    affine(gi);
    odd |= !(fabsf(bias[gi]) < INFINITY && scale[gi] < INFINITY && hi[gi] - lo[gi] < INFINITY);
  }
  if (__any(odd)) {  // rare: infinities, NaN, or a range past f16: the row kernel's operations
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      float l = 0.0f, h = 0.0f;
#pragma unroll
      for (int k = 0; k < KPG; ++k) {
        float x[8];
        unpack8<FK>(raw[gi * KPG + k], x);
        if (k == 0) l = h = x[0];
#pragma unroll
        for (int e = 0; e < 8; ++e) { l = fminf(l, x[e]); h = fmaxf(h, x[e]); }
      }
      lo[gi] = xor32_min(xor16_min(l));
      hi[gi] = xor32_max(xor16_max(h));
      affine(gi);
    }
#pragma unroll
    for (int kb = 0; kb < DP / 32; ++kb) {
      float x[8];
      unpack8<FK>(raw[kb], x);
      codes8_div(x, bias[kb / KPG], scale[kb / KPG], levels, codes[2 * kb], codes[2 * kb + 1]);
    }
    return;
  }
  float rcp[NG];
#pragma unroll
  for (int gi = 0; gi < NG; ++gi) rcp[gi] = __fdiv_rn(1.0f, scale[gi]);
#pragma unroll
  for (int kb = 0; kb < DP / 32; ++kb) {
    const int gi = kb / KPG;
    float x[8];
    unpack8<FK>(raw[kb], x);
    codes8(x, bias[gi], scale[gi], rcp[gi], levels, codes[2 * kb], codes[2 * kb + 1]);
  }
}

// Words per token row of a wave's V staging buffer (rows apart by 16 bytes).
template <int DP, int BITS>
constexpr int tile_row_words() { return BITS == 16 ? DP / 2 + 4 : DP / 4 + 4; }

// Store one side of the tile at slots slot0 .. slot0 + 15 of a head block: lane
// (t, jj) holds the elements d = 32*kb + 8*jj + e of token t in raw (zeros past the
// head dim).  The tile's token t is number rel + t of `width` new ones; tokens
// outside them stay as they are.  vbuf: the wave's own LDS, 16 rows of
// tile_row_words.  The whole wave calls.
template <int DP, int G, int BITS>
__device__ __forceinline__ void store_tile_side(const Geo &g, uint8_t *head, int slot0, int side,
                                                const u4 (&raw)[DP / 32], int rel, int width, uint32_t *vbuf,
                                                int lane) {
  constexpr int KB = DP / 32, NB = DP / 16;
  constexpr int ROWW = tile_row_words<DP, BITS>();
  const int t = lane & 15, jj = lane >> 4;
  const bool mine = rel + t >= 0 && rel + t < width;
  const int64_t toff = (int64_t)(slot0 / PKV_TILE) * g.tile_bytes;
  uint8_t *ktile = head + toff, *vtile = head + g.v_offset + toff;
  uint32_t *vrow = vbuf + t * ROWW;
  if constexpr (BITS == 16) {
    if (side == 0) {
      if (mine) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) *(u4 *)(ktile + kb * 1024 + lane * 16) = raw[kb];
      }
      return;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) *(u4 *)(vrow + 16 * kb + 4 * jj) = raw[kb];
  } else {
    constexpr int NG = DP / G;
    uint32_t meta[NG], codes[2 * KB];
    if (g.float_kind == 0) quantize_share<DP, G, BITS, 0>(raw, meta, codes);
    else quantize_share<DP, G, BITS, 1>(raw, meta, codes);
    if (mine) {
      // the token's (scale, bias) words: group gi by lane jj = gi % 4
      uint32_t *m = (uint32_t *)(head + (side ? g.vmeta_offset : g.kmeta_offset)) + (slot0 + t) * NG;
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
        if (gi % 4 == jj) m[gi] = meta[gi];
    }
    if (side == 0) {
      // K: the lane's payload, 16-byte chunks (8 bytes where it holds no more)
      constexpr int LW = DP * BITS / 128;
      uint32_t w[LW];
#pragma unroll
      for (int i = 0; i < LW; ++i) {
        if constexpr (BITS == 8) {
          w[i] = codes[i];
        } else {
          // nibble (e odd ? 4 : 0) + e / 2 holds element e
          const uint32_t c0 = codes[2 * i], c1 = codes[2 * i + 1];
          const uint32_t ev = (c0 & 15u) | ((c0 >> 12) & 0xF0u) | ((c1 & 15u) << 8) | ((c1 >> 4) & 0xF000u);
          const uint32_t od = ((c0 >> 8) & 15u) | ((c0 >> 20) & 0xF0u) | (c1 & 0xF00u) | ((c1 >> 12) & 0xF000u);
          w[i] = ev | (od << 16);
        }
      }
      if (mine) {
        if constexpr (LW >= 4) {
#pragma unroll
          for (int c = 0; c < LW / 4; ++c)
            *(u4 *)(ktile + c * 1024 + lane * 16) = u4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
        } else {
          *(u2 *)(ktile + lane * 8) = u2{w[0], w[1]};
        }
      }
      return;
    }
    // codes of d = 32*kb + 8*jj + 0..7: words 8*kb + 2*jj, + 1 of the row
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) *(u2 *)(vrow + 8 * kb + 2 * jj) = u2{codes[2 * kb], codes[2 * kb + 1]};
  }
  wave_lds_sync();
  // V: lane (col, jj) takes column d = 16*n + col of tokens 4*jj .. 4*jj + 3
  const int col = t;
  const int first = rel + 4 * jj;  // token 4*jj of the tile, among the new ones
  const bool all4 = first >= 0 && first + 3 < width;
  const uint32_t *vcol = vbuf + 4 * jj * ROWW;
  if constexpr (BITS == 16) {
    const uint32_t sel = (col & 1) ? 0x07060302u : 0x05040100u;
    uint32_t w[2 * NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = vcol[i * ROWW + 8 * n + (col >> 1)];
      w[2 * n] = __builtin_amdgcn_perm(r[1], r[0], sel);
      w[2 * n + 1] = __builtin_amdgcn_perm(r[3], r[2], sel);
    }
    if (all4) {
#pragma unroll
      for (int c = 0; c < NB / 2; ++c)
        *(u4 *)(vtile + c * 1024 + lane * 16) = u4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (first + i < 0 || first + i >= width) continue;
#pragma unroll
        for (int n = 0; n < NB; ++n)
          *(uint16_t *)(vtile + (n / 2) * 1024 + lane * 16 + 8 * (n & 1) + 2 * i) =
              (uint16_t)(w[2 * n + i / 2] >> (16 * (i & 1)));
      }
    }
  } else {
    // a word's bytes: tokens 0..3 of a column (8-bit), or 0, 2, 1, 3 with the
    // odd block's codes in the high nibbles (4-bit)
    const uint32_t cb = col & 3;
    const uint32_t sel = cb | ((4 + cb) << 8) | 0x0C0C0000u;  // bytes cb of both sources
    uint32_t w[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = vcol[i * ROWW + 4 * n + (col >> 2)];
      const uint32_t p01 = __builtin_amdgcn_perm(r[BITS == 8 ? 1 : 2], r[0], sel);
      const uint32_t p23 = __builtin_amdgcn_perm(r[3], r[BITS == 8 ? 2 : 1], sel);
      w[n] = p01 | (p23 << 16);
    }
    constexpr int LW = DP * BITS / 128;
    uint32_t o[LW];
#pragma unroll
    for (int i = 0; i < LW; ++i) o[i] = BITS == 8 ? w[i] : w[2 * i] | (w[2 * i + 1] << 4);
    if (all4) {
      if constexpr (LW >= 4) {
#pragma unroll
        for (int c = 0; c < LW / 4; ++c)
          *(u4 *)(vtile + c * 1024 + lane * 16) = u4{o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]};
      } else {
        *(u2 *)(vtile + lane * 8) = u2{o[0], o[1]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (first + i < 0 || first + i >= width) continue;
        const int byte = BITS == 8 ? i : v4_byte(i);
#pragma unroll
        for (int x = 0; x < LW; ++x)
          vtile[payload_offset(lane, 4 * x + byte, LW >= 4 ? 16 : 8)] = (uint8_t)(o[x] >> (8 * byte));
      }
    }
  }
}

}  // namespace pkv
