// Block tables and maps of a serving step, built on the device from the requests' lengths.
//
// A step holds n requests. Request i sits in row rows[i] of the block table, has cached[i] tokens in the cache and brings new[i] more. Two
// things follow from these lengths and a prefix sum over them, and neither needs the host:
//   b200_extend_block_tables   row i lists ceil(cached / bs) blocks and needs ceil(lens / bs); what is missing comes off a list of
//                              free blocks in the order of the requests
//   b200_step_maps             for every token its position, cache row and place in the pool (block * bs + offset); first token of each
//                              request, last token, and the tiles of at most 64 rows that the attention kernels take
//
// Bound: the launch. 64 requests read 1 KB and write 2; a step of 60 prompt pieces (60 000 tokens) writes 1 MB, 0.15 us at the memory's
// rate. The tables take 3.4 us (of 200 requests with 800 000 tokens 4.3), the maps 3.3 (of that step 4.4), about what a kernel of two loads that
// depend on each other takes; a call is 12 and 23 us, most of it the host's. So each of them is one launch whose CTAs ask each other nothing: a CTA
// takes kReq requests and adds up the lengths of all requests before them by itself (n values from L2 instead of a pass over the CTAs), then its threads
// share out the tokens of its requests, kChunk to a CTA: a long prompt is spread over the grid's second dimension. Sums stop at 2^31 - 1: what lies that
// far behind is behind the end of every table, and nothing is written there.
#include "common.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kReq = 32;            // requests of a CTA: one warp scans their lengths
constexpr int kChunk = 1024;        // tokens (or blocks) of them that a CTA writes
constexpr int kMapThreads = 256;
constexpr int kMapTile = 64;        // rows of an attention tile

__device__ __forceinline__ int blocks_of(int tokens, int bs) { return tokens > 0 ? (int)(((long long)tokens + bs - 1) / bs) : 0; }

constexpr unsigned kMost = 0x7fffffffu;

// a + b of numbers that are not negative, kMost at most: in any order the same
__device__ __forceinline__ int add_up(int a, int b) { return (int)min((unsigned)a + (unsigned)b, kMost); }
// a warp's values, by halves of 16 bits, whose sums fit
__device__ __forceinline__ int add_up_warp(int v) {
  const unsigned long long lo = __reduce_add_sync(0xffffffffu, (unsigned)v & 0xffffu), hi = __reduce_add_sync(0xffffffffu, (unsigned)v >> 16);
  return (int)min((hi << 16) + lo, (unsigned long long)kMost);
}

// Sums of value(i) >= 0 over requests before this CTA's and, in cu[0 .. kReq], over its own; n requests, blockIdx.x * kReq the first
template <typename F>
__device__ __forceinline__ int scan_requests(int n, int* cu, int* red, F value) {
  const int first = blockIdx.x * kReq, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int i = threadIdx.x; i < first; i += kMapThreads) before = add_up(before, value(i));
  before = add_up_warp(before);
  if (lane == 0) red[warp] = before;
  if (warp == 0) {
    int v = first + lane < n ? value(first + lane) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = add_up(v, u);
    }
    cu[lane + 1] = v;
    if (lane == 0) cu[0] = 0;
  }
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < kMapThreads / 32; ++w) before = add_up(before, red[w]);
  return before;
}

// the request (of kReq) that item k belongs to: the last one that starts at or before it
__device__ __forceinline__ int owner_of(const int* cu, int k) {
  int lo = 0;
#pragma unroll
  for (int step = kReq / 2; step > 0; step >>= 1)
    if (cu[lo + step] <= k) lo += step;
  return lo;
}

__global__ void __launch_bounds__(kMapThreads)
extend_tables_kernel(int* __restrict__ table, long long table_stride, int table_rows, int width, const int* __restrict__ rows,
                     const int* __restrict__ cached, const int* __restrict__ lens, const int* __restrict__ blocks, int n_blocks, int* __restrict__ used,
                     int n, int bs) {
  __shared__ int cu[kReq + 1], red[kMapThreads / 32];
  auto need = [&](int i) { return max(blocks_of(lens[i], bs) - blocks_of(cached[i], bs), 0); };
  const int before = scan_requests(n, cu, red, need);
  const int total = cu[kReq], live = min(total, max(n_blocks - before, 0));      // blocks that the list still has for them
  for (unsigned k = blockIdx.y * kChunk + threadIdx.x; k < (unsigned)live; k += gridDim.y * kChunk) {
#pragma unroll
    for (int u = 0; u < kChunk; u += kMapThreads) {
      if (k + u >= (unsigned)live) break;
      const int kk = (int)(k + u);
      const int j = owner_of(cu, kk), i = blockIdx.x * kReq + j;
      const int row = rows[i], col = blocks_of(cached[i], bs) + kk - cu[j];
      // a list that ended too early, or a row that is too short, leaves the rest of the row as it was
      if ((unsigned)row < (unsigned)table_rows && (unsigned)col < (unsigned)width)
        table[row * table_stride + col] = blocks[before + kk];
    }
  }
  if (used && blockIdx.y == 0 && blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *used = add_up(before, total);
}

struct StepMapsOut {
  int *cu, *pos, *slot, *tiles, *tile_of, *runs, *run_tiles;      // tiles .. run_tiles: all or none
  long long *place, *last;
};

__global__ void __launch_bounds__(kMapThreads)
step_maps_kernel(const int* __restrict__ table, long long table_stride, int table_rows, int width, const int* __restrict__ rows,
                 const int* __restrict__ cached, const int* __restrict__ fresh, int n, int bs, int total, int n_tiles, const StepMapsOut out) {
  __shared__ int cu[kReq + 1], ct[kReq + 1], red[kMapThreads / 32], red2[kMapThreads / 32];
  const int first = blockIdx.x * kReq;
  const int before = scan_requests(n, cu, red, [&](int i) { return max(fresh[i], 0); });
  const int mine = cu[kReq], live = min(mine, max(total - before, 0));           // tokens that the tables have room for
  for (unsigned k0 = blockIdx.y * kChunk; k0 < (unsigned)live; k0 += gridDim.y * kChunk) {
#pragma unroll
    for (int u = 0; u < kChunk; u += kMapThreads) {
      if (k0 + u + threadIdx.x >= (unsigned)live) break;
      const int k = (int)(k0 + u + threadIdx.x), t = before + k;
      const int j = owner_of(cu, k), i = first + j;
      const int p = (int)((unsigned)cached[i] + (unsigned)(k - cu[j])), row = rows[i];      // behind 2^31 - 1: negative, and in no table
      out.pos[t] = p;
      out.slot[t] = row;
      long long at = -1;                                   // a place that no table entry gives
      if (p >= 0 && (unsigned)row < (unsigned)table_rows && p / bs < width) at = (long long)table[row * table_stride + p / bs] * bs + p % bs;
      out.place[t] = at;
    }
  }
  if (blockIdx.y == 0 && threadIdx.x < kReq && first + threadIdx.x < n) {
    const int i = first + threadIdx.x, end = add_up(before, cu[threadIdx.x + 1]);
    if (i == 0) out.cu[0] = 0;
    out.cu[i + 1] = end;
    out.last[i] = (long long)end - 1;
  }
  if (n_tiles == 0) return;
  const int tiles_before = scan_requests(n, ct, red2, [&](int i) { return blocks_of(fresh[i], kMapTile); });
  const int my_tiles = ct[kReq], live_tiles = min(my_tiles, max(n_tiles - tiles_before, 0));
  int4* tiles = reinterpret_cast<int4*>(out.tiles);
  int4* tile_of = reinterpret_cast<int4*>(out.tile_of);
  for (unsigned kt = blockIdx.y * kMapThreads + threadIdx.x; kt < (unsigned)live_tiles; kt += gridDim.y * kMapThreads) {
    const int k = (int)kt, t = tiles_before + k;
    const int j = owner_of(ct, k), i = first + j, place = k - ct[j];
    const int row0 = place * kMapTile, rows_i = max(fresh[i], 0);
    tiles[t] = make_int4(add_up(add_up(before, cu[j]), row0), min(kMapTile, rows_i - row0), (int)((unsigned)cached[i] + (unsigned)row0), rows[i]);
    tile_of[t] = make_int4(i, place, blocks_of(rows_i, kMapTile), tiles_before + ct[j]);
  }
  if (blockIdx.y == 0 && threadIdx.x < kReq && first + threadIdx.x < n) {
    const int j = threadIdx.x, i = first + j;
    reinterpret_cast<int4*>(out.runs)[i] = make_int4(add_up(before, cu[j]), max(fresh[i], 0), cached[i], rows[i]);
    reinterpret_cast<int4*>(out.run_tiles)[i] = make_int4(add_up(tiles_before, ct[j]), blocks_of(fresh[i], kMapTile), 0, 0);
  }
  // tiles that the caller's bound has too many of are of no rows
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0)
    for (unsigned t = (unsigned)add_up(tiles_before, my_tiles) + threadIdx.x; t < (unsigned)n_tiles; t += kMapThreads) tiles[t] = tile_of[t] = make_int4(0, 0, 0, 0);
}

// chunks along the second dimension: enough for kReq requests to hold all of `items`, at most 256 (the rest in turn)
static unsigned map_chunks(long long items, int per) {
  const long long c = (items + per - 1) / per;
  return (unsigned)(c < 1 ? 1 : c > 256 ? 256 : c);
}

}  // namespace b200
using namespace b200;

B200_API int b200_extend_block_tables(void* table, long long table_stride, int table_rows, int width, const void* rows, const void* cached,
                                      const void* lens, const void* blocks, int n_blocks, void* used, int n, int block_size, void* stream) {
  if (n < 0 || table_rows < 0 || width < 0 || n_blocks < 0 || block_size < 1) return B200_ERR_BAD_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  if (n == 0) {
    if (used) B200_CHECK(cudaMemsetAsync(used, 0, sizeof(int), st));
    return 0;
  }
  const dim3 grid(ceil_div(n, kReq), map_chunks(n_blocks, kChunk));
  extend_tables_kernel<<<grid, kMapThreads, 0, st>>>((int*)table, table_stride, table_rows, width, (const int*)rows, (const int*)cached,
                                                     (const int*)lens, (const int*)blocks, n_blocks, (int*)used, n, block_size);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_step_maps(const void* table, long long table_stride, int table_rows, int width, const void* rows, const void* cached,
                            const void* fresh, int n, int block_size, int total, int n_tiles, void* cu, void* pos, void* slot, void* place,
                            void* last, void* tiles, void* tile_of, void* runs, void* run_tiles, void* stream) {
  if (n < 1 || table_rows < 0 || width < 0 || block_size < 1 || total < 0 || n_tiles < 0) return B200_ERR_BAD_SHAPE;
  if (n_tiles > 0) {
    if (!tiles || !tile_of || !runs || !run_tiles) return B200_ERR_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(tiles) | reinterpret_cast<uintptr_t>(tile_of) | reinterpret_cast<uintptr_t>(runs) |
         reinterpret_cast<uintptr_t>(run_tiles)) & 15) return B200_ERR_BAD_ALIGN;
  }
  const StepMapsOut out = {(int*)cu, (int*)pos, (int*)slot, (int*)tiles, (int*)tile_of, (int*)runs, (int*)run_tiles, (long long*)place, (long long*)last};
  const dim3 grid(ceil_div(n, kReq), map_chunks(total, kChunk));
  step_maps_kernel<<<grid, kMapThreads, 0, (cudaStream_t)stream>>>((const int*)table, table_stride, table_rows, width, (const int*)rows,
                                                                   (const int*)cached, (const int*)fresh, n, block_size, total, n_tiles, out);
  B200_LAUNCH_CHECK();
  return 0;
}
