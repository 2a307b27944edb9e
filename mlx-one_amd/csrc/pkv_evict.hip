// pkv_evict.hip -- eviction from the paged cache by accumulated attention weight.
//
// select: of a sequence's L tokens the n = min(L, budget) that stay are, per
// (layer, KV head), the last r = min(recent, n), the first s = min(sinks, n - r)
// and the n - r - s of largest sum among the rest (ties: the lowest index), in
// ascending order.
//
// pages: the kept tokens' K and V, codes and metadata bit for bit, to positions
// 0..n-1 of other pages.
#include "pkv_cache_ops.h"

namespace pkv {

namespace {

// ---- select ------------------------------------------------------------------------
//
// One workgroup per (layer, sequence, KV head).  The need-th largest key is found by
// its digits from the top, 11, 11 and 10 bits, each by a histogram in LDS of the keys
// that agree so far; as a rule the second digit's bin is to be taken whole and the
// third is not needed.  The row's keys stay in registers up to 32 per thread (a longer
// row is read again for each step); protected tokens have a key of their own above
// all others, so no step looks at positions (32 rows of 32700 sums: 26.4 -> 20.2 us).
// Bound by the steps of one workgroup, vector instructions first (a quarter LDS
// atomics): 256 rows of up to 8191 sums 12.4 us.  Four copies of each bin changed
// nothing.

constexpr int kVectors = 8;  // of four values, per thread
constexpr int kBins = 2048;

// Unsigned key of the order: a NaN above every number, -0 equal to +0.  No key is 0
// (no token) or kStays (a protected one).
constexpr uint32_t kStays = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t order_key(uint32_t bits) {
  const float x = __uint_as_float(bits);
  if (x != x) return kStays - 1;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the workgroup; *total the sum.
template <int NT>
__device__ __forceinline__ int block_scan(int v, int *s_wave, int *total) {
  const int incl = wave_scan_incl(v, 0), wave = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s_wave[wave] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) {
    before += k < wave ? s_wave[k] : 0;
    sum += s_wave[k];
  }
  *total = sum;
  return before + incl - v;
}

template <int NT>
__global__ __launch_bounds__(NT) void evict_select_kernel(const EvictSelectArgs a) {
  constexpr int kWaves = NT / 64, kChunk = NT * kVectors * 4;
  __shared__ int s_wave[kWaves], s_bins[kBins], s_found[3], s_sums[kVectors][kWaves];
  const int kh = blockIdx.x % a.hk, b = blockIdx.x / a.hk % a.batch, layer = blockIdx.x / a.hk / a.batch;
  const int row = a.rows ? a.rows[b] : b;
  const int L = (int)max((int64_t)0, min((int64_t)a.seq_lens[b], a.width));
  int n = min(L, a.max_keep);
  if (a.keep) n = max(0, min(n, a.keep[b]));
  const bool there = row >= 0 && row < a.mass_rows;
  if (!there) n = 0;  // no such row: nothing is kept of it
  if (layer == 0 && kh == 0 && threadIdx.x == 0) a.new_lens[b] = n;
  int32_t *kept = a.kept + (int64_t)blockIdx.x * a.max_keep;
  const int64_t base = ((int64_t)layer * a.mass_rows + row) * a.hk + kh;
  const float *mass = a.mass + base * a.width;
  float *new_mass = a.new_mass && there ? a.new_mass + base * a.new_width : nullptr;
  const int r = min(a.recent, n), s = min(a.sinks, n - r);
  const int lo = s, hi = L - r;  // the tokens lo..hi-1 are ordered by their sums
  const int chunks = n > 0 ? (L + kChunk - 1) / kChunk : 0;

  // keys of chunk c: this thread's vectors, four tokens from c * kChunk + (j * NT + thread) * 4 on
  uint32_t keys[kVectors][4];
  auto first = [&](int c, int j) { return c * kChunk + (j * NT + (int)threadIdx.x) * 4; };
  auto live = [&](int c, int j) { return c * kChunk + j * NT * 4 < L; };
  auto read = [&](int c, int j) {
    const int t = first(c, j);
    if (t + 4 <= L) {
      __builtin_memcpy(keys[j], mass + t, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) keys[j][e] = t + e < L ? __float_as_uint(mass[t + e]) : 0u;
    }
  };
  auto load = [&](int c) {
#pragma unroll
    for (int j = 0; j < kVectors; ++j)
      if (live(c, j)) read(c, j);
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      if (!live(c, j)) break;
      const int t = first(c, j);
#pragma unroll
      for (int e = 0; e < 4; ++e) keys[j][e] = order_key(keys[j][e]);
      if (t < lo || t + 4 > hi) {
#pragma unroll
        for (int e = 0; e < 4; ++e) keys[j][e] = t + e >= L ? 0u : t + e < lo || t + e >= hi ? kStays : keys[j][e];
      }
    }
  };
  if (chunks > 0) load(0);

  uint32_t least = 0;  // keys above it stay, and `room` of those that are equal to it
  int room = INT32_MAX;
  if (n > 0 && n < L) {
    int left = n, shift = 21;
    for (;;) {
      for (int k = threadIdx.x; k < kBins; k += NT) s_bins[k] = 0;
      __syncthreads();
      const uint32_t digits = shift > 0 ? kBins - 1 : 1023;  // the last digit has 10 bits
      for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) load(c);
#pragma unroll
        for (int j = 0; j < kVectors; ++j) {
          if (!live(c, j)) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t key = keys[j][e];
            const bool same = shift == 21 || key >> (shift == 10 ? 21 : 10) == least >> (shift == 10 ? 21 : 10);
            if (same) atomicAdd(&s_bins[key >> shift & digits], 1);
          }
        }
      }
      __syncthreads();
      // the bin of the left-th from the top: thread i has the bins below those of i - 1
      int mine = 0;
#pragma unroll
      for (int k = 0; k < kBins / NT; ++k) mine += s_bins[kBins - 1 - (int)threadIdx.x * (kBins / NT) - k];
      int total;
      int above = block_scan<NT>(mine, s_wave, &total);
      if (above < left && above + mine >= left)
#pragma unroll
        for (int k = 0; k < kBins / NT; ++k) {
          const int bin = kBins - 1 - (int)threadIdx.x * (kBins / NT) - k;
          if (above < left && above + s_bins[bin] >= left) {
            s_found[0] = bin;
            s_found[1] = left - above;
            s_found[2] = s_bins[bin];
          }
          above += s_bins[bin];
        }
      __syncthreads();
      least |= (uint32_t)s_found[0] << shift;
      left = s_found[1];
      if (left == s_found[2]) break;  // the whole bin stays: everything from its lowest key on
      room = left;
      if (shift == 0) break;
      room = INT32_MAX;
      shift = shift == 21 ? 10 : 0;
      __syncthreads();
    }
    if (room == INT32_MAX && least > 0) --least;  // "above it" is then all that stays
  }
  int done = 0;
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
    // which of its tokens each thread keeps: a bit each, and how many its wave's
    // lanes before it keep of the vector
    uint32_t keep[kVectors];
    // s_sums, as the waves' counts of each vector, becomes what comes before them
    auto prefix = [&]() {
      __syncthreads();
      if (threadIdx.x < 64) {
        constexpr int kPer = (kVectors * kWaves + 63) / 64;
        int *sums = &s_sums[0][0], v[kPer], all = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int i = (int)threadIdx.x * kPer + k;
          v[k] = i < kVectors * kWaves ? sums[i] : 0;
          all += v[k];
        }
        const int incl = wave_scan_incl(all, 0);
        int at = incl - all;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          const int i = (int)threadIdx.x * kPer + k;
          if (i < kVectors * kWaves) sums[i] = at;
          at += v[k];
        }
        if (threadIdx.x == 63) s_found[0] = incl;
      }
      __syncthreads();
    };
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) keep[j] = 0;
    if (room != INT32_MAX) {
      // ties: the lowest indices
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        uint32_t tie = 0;
        if (live(c, j))
#pragma unroll
          for (int e = 0; e < 4; ++e) tie |= (uint32_t)(keys[j][e] == least) << e;
        const int incl = wave_scan_incl(__popc(tie), 0);
        if ((threadIdx.x & 63) == 63) s_sums[j][wave] = incl;
        keep[j] = tie | (uint32_t)(incl - __popc(tie)) << 8;
      }
      prefix();
      const int ties = s_found[0];
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        int at = s_sums[j][wave] + (int)(keep[j] >> 8);
        uint32_t taken = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (keep[j] >> e & 1) taken |= (uint32_t)(at++ < room) << e;
        keep[j] = taken;
      }
      room -= min(room, ties);
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      if (live(c, j))
#pragma unroll
        for (int e = 0; e < 4; ++e) keep[j] |= (uint32_t)(keys[j][e] > least) << e;
      const int incl = wave_scan_incl(__popc(keep[j]), 0);
      if ((threadIdx.x & 63) == 63) s_sums[j][wave] = incl;
      keep[j] |= (uint32_t)(incl - __popc(keep[j])) << 8;
    }
    // the chunk's sums again, here before any are written: new_mass may be mass
    if (new_mass) {
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
        if (live(c, j)) read(c, j);
#pragma unroll
      for (int j = 0; j < kVectors; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(keys[j][e]));
    }
    prefix();
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      if (!live(c, j)) break;
      int at = done + s_sums[j][wave] + (int)(keep[j] >> 8);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (keep[j] >> e & 1) {
          if (at < a.max_keep) {
            kept[at] = first(c, j) + e;
            if (new_mass) new_mass[at] = __uint_as_float(keys[j][e]);
          }
          ++at;
        }
    }
    done += s_found[0];
    __syncthreads();
  }
  for (int i = n + threadIdx.x; i < a.max_keep; i += NT) {
    kept[i] = -1;
    if (new_mass) new_mass[i] = 0.0f;
  }
}

// ---- pages -------------------------------------------------------------------------

// One wave per 16-token tile of the new pages.  A K lane's bytes belong to one
// token, so they move as they are; a V lane holds four tokens of a column, so it
// gathers four source lanes and takes one token's bytes of each.  Memory-bound by
// lines: 128 bytes of K hold a chunk of eight tokens and 512 of V four tokens, so
// with a quarter kept most of every page is fetched.  1024 of 4.6K tokens (32
// sequences, 8 KV heads, 8-bit): 71 MB kept and as much written in 68 us, with 233 MB
// of lines fetched for it (4.5 TB/s).
template <int BITS, int DP>
__global__ __launch_bounds__(256) void evict_pages_kernel(const EvictPagesArgs a) {
  constexpr int LB = DP * BITS / 32, CS = LB < 16 ? LB : 16, NCH = LB / CS, W = CS / 4;
  const Geo &g = a.g;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = (blockIdx.x * 4 + wave) * PKV_TILE;
  const int kh = blockIdx.y % g.hk, b = blockIdx.y / g.hk;
  const int n = min(a.new_lens[b], a.max_keep);
  if (t0 >= n || t0 / g.page >= a.dst_pages) return;
  const int dst_id = a.dst_table[(int64_t)b * a.dst_pages + t0 / g.page];
  if (dst_id < 0 || dst_id >= a.num_pages) return;
  uint8_t *pool = a.pools[blockIdx.z];
  uint8_t *dst_head = pool + (int64_t)dst_id * g.page_bytes + (int64_t)kh * g.head_bytes;
  const int dst_slot = t0 % g.page;
  const int64_t dst_tile = (int64_t)(dst_slot / PKV_TILE) * g.tile_bytes;

  // this lane's token: lane % 16 of the tile
  const int i = t0 + lane % 16;
  int slot = -1, id = -1;
  if (i < n) {
    const int t = a.kept[(((int64_t)blockIdx.z * a.batch + b) * g.hk + kh) * a.max_keep + i];
    if (t >= 0 && t / g.page < a.src_pages) {
      id = a.src_table[(int64_t)b * a.src_pages + t / g.page];
      slot = t % g.page;
      if (id < 0 || id >= a.num_pages) id = -1;
    }
  }
  auto head_of = [&](int page) { return pool + (int64_t)page * g.page_bytes + (int64_t)kh * g.head_bytes; };
  if (id >= 0) {
    const uint8_t *src = head_of(id) + (int64_t)(slot / PKV_TILE) * g.tile_bytes;
    const int from = slot % PKV_TILE + (lane & 48);
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if constexpr (CS == 16)
        *(u4 *)(dst_head + dst_tile + c * 1024 + lane * 16) = *(const u4 *)(src + c * 1024 + from * 16);
      else
        *(u2 *)(dst_head + dst_tile + lane * 8) = *(const u2 *)(src + from * 8);
    }
    // its metadata words, groups lane / 16, lane / 16 + 4, ...
    if (BITS != 16)
      for (int gi = lane / 16; gi < g.ng; gi += 4) {
        const int64_t from_w = ((int64_t)slot * g.ng + gi) * 4, to_w = ((int64_t)(dst_slot + lane % 16) * g.ng + gi) * 4;
        *(uint32_t *)(dst_head + g.kmeta_offset + to_w) = *(const uint32_t *)(head_of(id) + g.kmeta_offset + from_w);
        *(uint32_t *)(dst_head + g.vmeta_offset + to_w) = *(const uint32_t *)(head_of(id) + g.vmeta_offset + from_w);
      }
  }
  int id4[4], slot4[4];
  bool all = true, any = false;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    id4[r] = __shfl(id, (lane >> 4) * 4 + r, 64);
    slot4[r] = __shfl(slot, (lane >> 4) * 4 + r, 64);
    all = all && id4[r] >= 0;
    any = any || id4[r] >= 0;
  }
  if (!any) return;
  uint8_t *dst = dst_head + g.v_offset + dst_tile;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    uint32_t out[W] = {};
    const int64_t at = (int64_t)c * 64 * CS;
    if (!all)  // positions without a kept token stay as they are
#pragma unroll
      for (int w = 0; w < W; ++w) out[w] = *(const uint32_t *)(dst + at + lane * CS + 4 * w);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (id4[r] < 0) continue;
      const int t = slot4[r] % PKV_TILE;
      const uint8_t *src = head_of(id4[r]) + g.v_offset + (int64_t)(slot4[r] / PKV_TILE) * g.tile_bytes + at +
                           (lane % 16 + 16 * (t / 4)) * CS;
      const int q = t % 4;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if constexpr (BITS == 16) {
          // dwords (2n, 2n+1) hold tokens (0, 1) and (2, 3) of block n
          if ((w & 1) != r / 2) continue;
          const uint32_t x = *(const uint32_t *)(src + 4 * ((w & ~1) + q / 2));
          const uint32_t h = q & 1 ? x >> 16 : x & 0xFFFFu;
          out[w] = r & 1 ? (out[w] & 0xFFFFu) | h << 16 : (out[w] & 0xFFFF0000u) | h;
        } else {
          const int bq = BITS == 4 ? v4_byte(q) : q, br = BITS == 4 ? v4_byte(r) : r;
          const uint32_t x = *(const uint32_t *)(src + 4 * w);
          out[w] = (out[w] & ~(0xFFu << (8 * br))) | ((x >> (8 * bq)) & 0xFFu) << (8 * br);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) *(uint32_t *)(dst + at + lane * CS + 4 * w) = out[w];
  }
}

template <int BITS>
void start_pages(hipStream_t stream, const EvictPagesArgs &a, dim3 grid) {
  if (a.g.dp == 64) hipLaunchKernelGGL((evict_pages_kernel<BITS, 64>), grid, dim3(256), 0, stream, a);
  else if (a.g.dp == 128) hipLaunchKernelGGL((evict_pages_kernel<BITS, 128>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((evict_pages_kernel<BITS, 256>), grid, dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_evict_select(hipStream_t stream, const EvictSelectArgs &a) {
  const dim3 grid(a.layers * a.batch * a.hk);
  // us by 256, 512 and 1024 threads: 64 rows of 1000 sums 7.3, 7.9 and 10.8, of 4000
  // 9.9, 8.8 and 9.7; 512 rows of 2000 9.9, 9.4 and 19.6; 256 rows of up to 8191 14.3,
  // 12.4 and 13.2.  Past 16384, 512 threads would read a row again for each digit.
  if (a.width <= 1024) hipLaunchKernelGGL(evict_select_kernel<256>, grid, dim3(256), 0, stream, a);
  else if (a.width <= 16384) hipLaunchKernelGGL(evict_select_kernel<512>, grid, dim3(512), 0, stream, a);
  else hipLaunchKernelGGL(evict_select_kernel<1024>, grid, dim3(1024), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_evict_pages(hipStream_t stream, const EvictPagesArgs &a) {
  const dim3 grid((a.max_keep + 4 * PKV_TILE - 1) / (4 * PKV_TILE), a.batch * a.g.hk, a.num_pools);
  if (a.g.bits == 4) start_pages<4>(stream, a, grid);
  else if (a.g.bits == 8) start_pages<8>(stream, a, grid);
  else start_pages<16>(stream, a, grid);
  return hipGetLastError();
}

}  // namespace pkv
