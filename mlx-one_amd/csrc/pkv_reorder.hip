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

__device__ __forceinline__ bool pair_moves(const ReorderArgs &a, int i, int &to, int &from) {
  to = a.targets[i];
  from = a.sources[i];
  return to >= 0 && to < a.num_rows && from >= 0 && from < a.num_rows && to != from;
}

// One byte column per thread and step, through LDS: [count][columns].
__global__ __launch_bounds__(kThreads) void reorder_rows_kernel(const ReorderArgs a, int columns) {
  extern __shared__ uint8_t s_bytes[];
  uint8_t *state = a.state + (int64_t)blockIdx.y * a.num_rows * a.row_bytes;
  const int64_t c0 = (int64_t)blockIdx.x * columns;
  for (int e = threadIdx.x; e < a.count * columns; e += kThreads) {
    int to, from;
    const int64_t c = c0 + e % columns;
    if (c < a.row_bytes && pair_moves(a, e / columns, to, from)) s_bytes[e] = state[from * a.row_bytes + c];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.count * columns; e += kThreads) {
    int to, from;
    const int64_t c = c0 + e % columns;
    if (c < a.row_bytes && pair_moves(a, e / columns, to, from)) state[to * a.row_bytes + c] = s_bytes[e];
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
  __shared__ int s_len[kMaxReorder];
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

hipError_t launch_reorder_rows(hipStream_t stream, const ReorderArgs &a) {
  int columns = 256;
  while (columns > 1 && a.count * columns > 65536) columns /= 2;
  const dim3 grid((unsigned)((a.row_bytes + columns - 1) / columns), (unsigned)a.outer);
  hipLaunchKernelGGL(reorder_rows_kernel, grid, dim3(kThreads), a.count * columns, stream, a, columns);
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
