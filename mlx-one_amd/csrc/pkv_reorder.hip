// pkv_reorder.hip -- rows of a state tensor, or sequence slots of the page arena,
// become others' copies, all at once: row targets[i] gets what row sources[i] held
// before the call.
//
// A workgroup owns a block of columns of every row in the call: it reads them all
// before it writes any, so rows that are sources and targets need no second
// buffer.
#include "pkv_cache_ops.h"

namespace pkv {

namespace {

constexpr int kThreads = 256;

// ---- rows of a tensor ------------------------------------------------------------------
//
// A workgroup holds its columns of all the rows in registers: PER units of 16 bytes
// per thread, 2^log_columns units beside each other of every row, read before the
// barrier and written after it.  Where a row ends inside a unit (TAIL), the threads
// of its last whole unit also move its last 16 bytes, which overlap that one.
// Memory-bound, one read and one write of the rows that move, 67 MB in 11.4 us (5.9
// TB/s); rows at odd addresses are read and written unaligned: 512 of 66666 bytes in
// 10.8 us.

typedef u4 __attribute__((aligned(1))) Unit;  // 16 bytes anywhere

template <int PER, int NT, bool TAIL>
__global__ __launch_bounds__(NT) void reorder_rows_kernel(const ReorderArgs a, int log_columns) {
  uint8_t *state = a.state + (int64_t)blockIdx.y * a.num_rows * a.row_bytes;
  const int columns = 1 << log_columns, step = NT >> log_columns;
  const int64_t units = a.row_bytes / 16;
  const int64_t c = (int64_t)blockIdx.x * columns + (threadIdx.x & (columns - 1));  // this thread's column
  const int64_t at = min(c, units - 1) * 16, end = a.row_bytes - 16;
  const bool tail = TAIL && c == units - 1;
  int to[PER], from[PER];
  u4 v[PER], w[TAIL ? PER : 1];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = min((int)(threadIdx.x >> log_columns) + k * step, a.count - 1);
    to[k] = a.targets[i];
    from[k] = a.sources[i];
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const bool moves = to[k] >= 0 && to[k] < a.num_rows && from[k] >= 0 && from[k] < a.num_rows && to[k] != from[k] &&
                       (int)(threadIdx.x >> log_columns) + k * step < a.count && c < units;
    if (!moves) to[k] = -1;
    const uint8_t *row = state + (moves ? from[k] : 0) * a.row_bytes;  // (a load without a branch)
    v[k] = *(const Unit *)(row + at);
    if constexpr (TAIL) w[k] = *(const Unit *)(row + (tail ? end : at));
  }
  // the loads have returned, not only been issued, before any wave stores
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    asm volatile("" : "+v"(v[k]));
    if constexpr (TAIL) asm volatile("" : "+v"(w[k]));
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < PER; ++k)
    if (to[k] >= 0) {
      uint8_t *row = state + to[k] * a.row_bytes;
      *(Unit *)(row + at) = v[k];
      if (tail) *(Unit *)(row + end) = w[TAIL ? k : 0];
    }
}

// Rows of fewer than 16 bytes, one thread a row.
__global__ __launch_bounds__(1024) void reorder_short_kernel(const ReorderArgs a) {
  uint8_t *state = a.state + (int64_t)blockIdx.x * a.num_rows * a.row_bytes;
  const int bytes = (int)a.row_bytes;
  uint32_t v[kMaxReorder / 1024][4];
#pragma unroll
  for (int k = 0; k < kMaxReorder / 1024; ++k) {
    const int i = threadIdx.x + k * 1024;
    const int s = i < a.count ? a.sources[i] : -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] = 0;
    if (s >= 0 && s < a.num_rows)
#pragma unroll
      for (int e = 0; e < 15; ++e)
        if (e < bytes) v[k][e / 4] |= (uint32_t)state[s * a.row_bytes + e] << (e % 4 * 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(v[k][e]));  // returned before any wave stores
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kMaxReorder / 1024; ++k) {
    const int i = threadIdx.x + k * 1024;
    const int t = i < a.count ? a.targets[i] : -1, s = i < a.count ? a.sources[i] : -1;
    if (t >= 0 && t < a.num_rows && s >= 0 && s < a.num_rows)
#pragma unroll
      for (int e = 0; e < 15; ++e)
        if (e < bytes) state[t * a.row_bytes + e] = (uint8_t)(v[k][e / 4] >> (e % 4 * 8));
  }
}

// ---- arena slots -----------------------------------------------------------------------

// Columns of the page table per workgroup, [count][columns] page ids before and
// after in LDS.
int arena_columns(int count, int max_pages) {
  int c = 16;
  while (c > 1 && count * c > 4096) c /= 2;
  return c < max_pages ? c : max_pages;
}

// The tables' entries and the pages' reference counts.  A page sits at the same
// place in every table that holds it, so all its references that change are in
// one workgroup: the new ones are counted before the old ones are dropped, and a
// page that none is left of goes to the workgroup's list of free pages, by the
// first of its droppers, in their order.
__global__ __launch_bounds__(kThreads) void arena_reorder_kernel(const ArenaReorderArgs a, int columns) {
  extern __shared__ int32_t s_ids[];
  __shared__ int s_wave[kThreads / 64];
  int32_t *s_old = s_ids, *s_new = s_ids + a.count * columns;
  int32_t *err = a.state + 1, *ref = a.state + kArenaHeaderWords + a.capacity;
  const int c0 = blockIdx.x * columns, total = a.count * columns;
  auto valid = [&](int id) { return id >= 0 && id < a.capacity; };
  for (int e = threadIdx.x; e < total; e += kThreads) {
    const int c = c0 + e % columns, to = a.slots[e / columns], from = a.sources[e / columns];
    int was = -1, is = -1;
    if (to < 0 || to >= a.num_slots || from < 0 || from >= a.num_slots) {
      atomicOr(err, kArenaBadArgument);
    } else if (c < a.max_pages) {
      was = a.table[(int64_t)to * a.max_pages + c];
      is = a.table[(int64_t)from * a.max_pages + c];
    }
    s_old[e] = was;
    s_new[e] = is;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < total; e += kThreads) {
    const int was = s_old[e], is = s_new[e];
    if (was == is) continue;
    a.table[(int64_t)a.slots[e / columns] * a.max_pages + c0 + e % columns] = is;
    if (valid(is)) atomicAdd(&ref[is], 1);
    else if (is != -1) atomicOr(err, kArenaCorrupt);
  }
  __threadfence();
  __syncthreads();
  for (int e = threadIdx.x; e < total; e += kThreads) {
    const int was = s_old[e];
    if (was == s_new[e]) s_old[e] = -1;  // nothing dropped
    else if (!valid(was)) {
      if (was != -1) atomicOr(err, kArenaCorrupt);
      s_old[e] = -1;
    } else if (atomicSub(&ref[was], 1) < 1) {
      atomicOr(err, kArenaCorrupt);
      atomicAdd(&ref[was], 1);
      s_old[e] = -1;
    }
  }
  __threadfence();
  __syncthreads();
  // the first dropper of a page without references claims it
  for (int e = threadIdx.x; e < total; e += kThreads) {
    const int was = s_old[e];
    if (was >= 0 && atomicAdd(&ref[was], 0) > 0) s_old[e] = -1;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < total; e += kThreads)
    if (s_old[e] >= 0) atomicMin(&ref[s_old[e]], e - 0x40000000);
  __threadfence();
  __syncthreads();
  for (int e = threadIdx.x; e < total; e += kThreads)
    if (s_old[e] >= 0 && atomicAdd(&ref[s_old[e]], 0) != e - 0x40000000) s_old[e] = -1;
  __syncthreads();
  int32_t *list = a.workspace + gridDim.x + (int64_t)blockIdx.x * total;
  int freed = 0;
  for (int e0 = 0; e0 < total; e0 += kThreads) {
    const int e = e0 + threadIdx.x;
    const bool mine = e < total && s_old[e] >= 0;
    const int incl = wave_scan_incl(mine, 0), wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 63) s_wave[wave] = incl;
    __syncthreads();
    int before = 0, sum = 0;
    for (int k = 0; k < kThreads / 64; ++k) {
      before += k < wave ? s_wave[k] : 0;
      sum += s_wave[k];
    }
    if (mine) {
      list[freed + before + incl - 1] = s_old[e];
      ref[s_old[e]] = 0;
    }
    freed += sum;
    __syncthreads();
  }
  if (threadIdx.x == 0) a.workspace[blockIdx.x] = freed;
}

// One workgroup: the lists onto the free stack, in the workgroups' order, and the
// slots' lengths.
__global__ __launch_bounds__(1024) void arena_reorder_finish_kernel(const ArenaReorderArgs a, int columns, int blocks) {
  __shared__ int s_len[kMaxArenaReorder];
  int32_t *stack = a.state + kArenaHeaderWords;
  for (int i = threadIdx.x; i < a.count; i += 1024) {
    const int from = a.sources[i];
    s_len[i] = from >= 0 && from < a.num_slots ? a.lens[from] : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.count; i += 1024) {
    const int to = a.slots[i];
    if (to >= 0 && to < a.num_slots && s_len[i] >= 0) a.lens[to] = s_len[i];
  }
  int top = a.state[0];
  for (int k = 0; k < blocks; ++k) {
    const int n = a.workspace[k];
    const int32_t *list = a.workspace + blocks + (int64_t)k * a.count * columns;
    for (int i = threadIdx.x; i < n; i += 1024) {
      if (top + i < a.capacity) stack[top + i] = list[i];
      else atomicOr(a.state + 1, kArenaCorrupt);
    }
    top = min(top + n, a.capacity);
  }
  __syncthreads();
  if (threadIdx.x == 0) a.state[0] = top;
}

int arena_blocks(int count, int max_pages) {
  const int c = arena_columns(count, max_pages);
  return (max_pages + c - 1) / c;
}

}  // namespace

template <int PER, int NT>
void start_rows(hipStream_t stream, const ReorderArgs &a, int log_columns) {
  const int64_t units = a.row_bytes / 16;
  const dim3 grid((unsigned)((units + (1 << log_columns) - 1) >> log_columns), (unsigned)a.outer);
  if (a.row_bytes % 16)
    hipLaunchKernelGGL((reorder_rows_kernel<PER, NT, true>), grid, dim3(NT), 0, stream, a, log_columns);
  else
    hipLaunchKernelGGL((reorder_rows_kernel<PER, NT, false>), grid, dim3(NT), 0, stream, a, log_columns);
}

hipError_t launch_reorder_rows(hipStream_t stream, const ReorderArgs &a) {
  if (a.row_bytes < 16) {
    hipLaunchKernelGGL(reorder_short_kernel, dim3((unsigned)a.outer), dim3(1024), 0, stream, a);
  } else if (a.count <= 512) {
    // at least 4 columns (64 bytes of a row) beside each other; us by 256 and by 1024
    // threads: 32 rows 11.4 and 14.4, 512 rows 6.1 and 6.6, 1024 rows 33.0 and 12.3
    int log_columns = 2;
    while (log_columns < 8 && (a.count << (log_columns + 1)) <= 8 * kThreads) ++log_columns;
    start_rows<8, kThreads>(stream, a, log_columns);
  } else {
    int log_columns = 0;
    while (log_columns < 6 && (a.count << (log_columns + 1)) <= 8 * 1024) ++log_columns;
    start_rows<8, 1024>(stream, a, log_columns);
  }
  return hipGetLastError();
}

int64_t arena_reorder_workspace(int count, int max_pages) {
  const int64_t blocks = arena_blocks(count, max_pages);
  return 4 * (blocks + blocks * count * arena_columns(count, max_pages));
}

hipError_t launch_arena_reorder(hipStream_t stream, const ArenaReorderArgs &a) {
  const int columns = arena_columns(a.count, a.max_pages), blocks = arena_blocks(a.count, a.max_pages);
  hipLaunchKernelGGL(arena_reorder_kernel, dim3(blocks), dim3(kThreads), 8 * a.count * columns, stream, a, columns);
  hipLaunchKernelGGL(arena_reorder_finish_kernel, dim3(1), dim3(1024), 0, stream, a, columns, blocks);
  return hipGetLastError();
}

}  // namespace pkv
