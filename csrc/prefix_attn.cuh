// What the kernels of prefix_attn.cu and prefix_attn_tc.cu share: their arguments, and how the shared keys are cut into ranges.
#pragma once

#include "common.cuh"

namespace b200 {

constexpr int kPxKeys = 64;                     // keys of a block
constexpr float kPxLog2e = 1.4426950408889634f;

struct PrefixParams {
  const void *q, *ck, *cv;
  long long q_stride;
  const int *pos, *slot, *table;
  long long table_stride;
  int table_rows, width, n_pages;               // block table [table_rows, width], pages in the pools
  const int *groups, *of;                       // [n_groups, 4] = (first token, tokens, shared keys, -), [T] group of a token or -1
  int n_groups, longest;                        // tokens of a group that the shared part takes; those behind them see to all keys by themselves
  const float* sinks;
  void* out;
  float *part_o, *part_ml;                      // [T, H, nsplit, D], [T, H, nsplit, 2] (maximum in powers of two, sum)
  int T, H, G, D, bs_log2, nsplit;
  long long beside;                             // CTAs of the tcgen05 kernel, none: 0
  int most_own;                                 // keys that a token sees to by itself, at most: chooses how they are cut
  float scale_log2;
};

// A group as the kernels use it; nothing in it reaches outside the batch or the table
struct PrefixGroup { int first, tokens, shared; };
__device__ __forceinline__ PrefixGroup prefix_group(const PrefixParams& p, int j) {
  PrefixGroup g;
  g.first = p.groups[4 * j]; g.tokens = p.groups[4 * j + 1]; g.shared = p.groups[4 * j + 2];
  if (g.first < 0 || g.first >= p.T) g.tokens = g.first = 0;
  g.tokens = min(max(g.tokens, 0), min(p.T - g.first, p.longest));
  g.shared = (int)min((long long)max(g.shared, 0), (long long)p.width << p.bs_log2);
  return g;
}
// ranges of the shared keys, in blocks of kPxKeys: how many each takes, and how many there are
__device__ __forceinline__ int range_blocks(const PrefixParams& p, int shared) { return (ceil_div(shared, kPxKeys) + p.nsplit - 1) / p.nsplit; }
__device__ __forceinline__ int ranges_used(const PrefixParams& p, int shared) {
  return shared > 0 ? ceil_div(ceil_div(shared, kPxKeys), range_blocks(p, shared)) : 0;
}
// the page of key k in a table row, or -1: pages outside the pool are not read
__device__ __forceinline__ int page_of(const PrefixParams& p, const int* row, int k) {
  const int page = row[k >> p.bs_log2];
  return (unsigned)page < (unsigned)p.n_pages ? page : -1;
}

// Launch attribute of the two kernels that run side by side: an SM whose memory was cut for the one alone has less room for the other, and is cut anew only when
// it is empty. 64 tokens, 2000 shared and up to 300 own keys, 16 / 8 heads of 64: 15.0 -> 11.7 us; 100 with 8000 and 100, 12 / 2 heads: 19.0 -> 16.6
inline cudaLaunchAttribute most_shared_memory() {
  cudaLaunchAttribute a = {};
  a.id = cudaLaunchAttributePreferredSharedMemoryCarveout;
  a.val.sharedMemCarveout = cudaSharedmemCarveoutMaxShared;
  return a;
}

// The shared keys on tcgen05 (prefix_attn_tc.cu): part_o and part_ml of every row and range, as the mma.sync kernel leaves them. Tokens of a tile, 0 where the
// kernel does not take the call.
int prefix_tc_tokens(int H, int G, int D);
int prefix_shared_tc(const PrefixParams& p, int dtype, cudaStream_t st);

}  // namespace b200
