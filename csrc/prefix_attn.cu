// Attention of a decode batch whose sequences share their first keys (a system prompt, one long document).
//
// Token t of group j sees keys 0 .. pos[t] of its sequence; the first shared_j of them are the same for the whole group. With the scores
// s = scale q . k and a sink z (a logit that only takes part in the sum),
//   m = max over both parts (and z),  out = (sum_shared e^(s-m) v + sum_own e^(s-m) v) / (sum_shared e^(s-m) + sum_own e^(s-m) + e^(z-m))
// so each part may be summed up against a maximum of its own and the two joined: (m1, l1, o1), (m2, l2, o2) -> m = max(m1, m2),
// l = l1 e^(m1-m) + l2 e^(m2-m), the same for o. All maxima, sums and partial results are 32 bits; the weights are rounded to the cache's
// 16 bits for the tensor cores' second product, as in the other attention kernels.
//
//   shared keys  for each group and KV head ONE product of all its rows (tokens x heads of the KV head) with the keys: they are read
//                once for 64 rows (mma.sync, here) or 128 (tcgen05, prefix_attn_tc.cu) instead of once a sequence. The keys are cut into nsplit
//                ranges, so that few rows still fill the GPU; a range leaves (m, l, o) per row
//   own keys     a CTA for a token and KV head (or a cluster, where tokens are few), whose warps have rings of 16 keys by TMA and mma.sync products; at its end
//                it takes up the ranges of the shared keys and the sink, and writes the result: no third kernel (one beside both took 36 us where this took 31). It
//                starts while the first kernel runs and waits for it only there
//
// Bound: memory, until the rows of a group are so many that the tensor cores are. 64 tokens, 32 / 8 heads of 128, 4096 shared and 300 own keys on average:
// 17 MB of shared keys and 78 MB of own ones (15 us at 6.5 TB/s), 4.6 GFLOP (3 us); read once a sequence they were 1.15 GB. It takes 28 us, about 16 of them beside the
// shared keys. 10 of them are there without any work: two launches, for the shared keys the way from a row number to the first product and back to memory, and the
// joining. There a CTA's own steps count: four loads one after another (row, group, page numbers, keys), its blocks, two waits to join the parts. What finds no room
// beside the shared keys takes these steps after them (own_warps): 31 us with four warps to each token. 128 tokens, 16384 shared and 256 own keys: 68 us, 39 of them the
// shared keys (prefix_attn_tc.cu), which fill the SMs. 4 tokens, 512 shared and 20 own keys: 6 + 5 us, of which 8 remain as the second starts early.
#include "common.cuh"
#include "mma_sync.cuh"
#include "prefix_attn.cuh"
#include "tma_host.h"
#include <type_traits>
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kPxRows = 64;

template <typename T> __device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_bf16_16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
template <> __device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <> __device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <> __device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ------------------------------------------------------------------------------------------------------------------
// shared keys on mma.sync: 64 rows x 64 keys at a time, 4 warps of 16 rows, keys and values double-buffered by cp.async
// ------------------------------------------------------------------------------------------------------------------
template <typename T, int DK>                         // head size = 16 * DK
__global__ void __launch_bounds__(128, 3)
prefix_shared_mma_kernel(const PrefixParams p) {
  constexpr int D = 16 * DK, LD = D + 8, CH = D / 8;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  T* sk = reinterpret_cast<T*>(smem_raw);             // [2][64][LD]
  T* sv = sk + 2 * kPxKeys * LD;                      // [2][64][LD]
  T* sq = sk + kPxKeys * LD;                          // Q is staged in K buffer 1 until its fragments are read
  pdl_launch_dependents();
  const PrefixGroup grp = prefix_group(p, blockIdx.z);
  const int rep = p.H / p.G, tiles = gridDim.y / p.G;
  const int g = blockIdx.y / tiles, row0 = (blockIdx.y % tiles) * kPxRows, nrows = min(kPxRows, grp.tokens * rep - row0);
  const int per = range_blocks(p, grp.shared), k_lo = blockIdx.x * per * kPxKeys, k_hi = min(grp.shared, k_lo + per * kPxKeys);
  if (nrows <= 0 || k_lo >= k_hi) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slot = p.slot[grp.first];
  const int* trow = (unsigned)slot < (unsigned)p.table_rows ? p.table + slot * p.table_stride : nullptr;
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* ck = reinterpret_cast<const T*>(p.ck);
  const T* cv = reinterpret_cast<const T*>(p.cv);
  const int nkb = ceil_div(k_hi - k_lo, kPxKeys), bs_mask = (1 << p.bs_log2) - 1;

  auto load_kv = [&](int buf, int kb) {               // two threads per key row, alternating 16-byte chunks
    const int r = tid >> 1, half = tid & 1, k = k_lo + kb * kPxKeys + r;
    T* dk = sk + (buf * kPxKeys + r) * LD;
    T* dv = sv + (buf * kPxKeys + r) * LD;
    const int page = k < k_hi && trow ? page_of(p, trow, k) : -1;
    if (page >= 0) {
      const long long off = ((((long long)page * p.G + g) << p.bs_log2) + (k & bs_mask)) * D;
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) {
        const int col = (half + 2 * i) * 8;
        cp_async16(smem_u32(dk + col), ck + off + col);
        cp_async16(smem_u32(dv + col), cv + off + col);
      }
    } else {                                          // also rows behind the shared keys: another sequence's, a NaN perhaps
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) {
        const int col = (half + 2 * i) * 8;
        *reinterpret_cast<uint4*>(dk + col) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dv + col) = make_uint4(0, 0, 0, 0);
      }
    }
  };

  for (int c = tid; c < kPxRows * CH; c += 128) {
    const int r = c / CH, col = (c % CH) * 8, rr = row0 + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < nrows) v = *reinterpret_cast<const uint4*>(q + (long long)(grp.first + rr / rep) * p.q_stride + (long long)(g * rep + rr % rep) * D + col);
    *reinterpret_cast<uint4*>(sq + r * LD + col) = v;
  }
  load_kv(0, 0);
  cp_async_commit();
  __syncthreads();
  uint32_t qa[DK][4];
#pragma unroll
  for (int k = 0; k < DK; ++k)
    ldsm_x4(smem_u32(sq + (warp * 16 + (lane & 15)) * LD + k * 16 + (lane >> 4) * 8), qa[k][0], qa[k][1], qa[k][2], qa[k][3]);
  __syncthreads();                                    // every warp has its Q fragments: buffer 1 may be refilled with keys

  const float sl2 = p.scale_log2;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float o[2 * DK][4];
#pragma unroll
  for (int i = 0; i < 2 * DK; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  for (int kb = 0; kb < nkb; ++kb) {
    const int buf = kb & 1;
    if (kb + 1 < nkb) load_kv(buf ^ 1, kb + 1);
    cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    const T* bk = sk + buf * kPxKeys * LD;
    const T* bv = sv + buf * kPxKeys * LD;
    float s[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < DK; ++k) {                    // eight key tiles of a step are independent sums
      uint32_t b[8][2];
#pragma unroll
      for (int n = 0; n < 8; ++n) ldsm_x2(smem_u32(bk + (n * 8 + (lane & 7)) * LD + k * 16 + ((lane >> 3) & 1) * 8), b[n][0], b[n][1]);
#pragma unroll
      for (int n = 0; n < 8; ++n) mma_16816<T>(s[n], qa[k], b[n][0], b[n][1]);
    }
    const int left = k_hi - k_lo - kb * kPxKeys;      // keys of this block
    if (left < kPxKeys) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n * 8 + 2 * (lane & 3) + (j & 1) >= left) s[n][j] = -INFINITY;
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      mx0 = fmaxf(mx0, fmaxf(s[n][0], s[n][1]));
      mx1 = fmaxf(mx1, fmaxf(s[n][2], s[n][3]));
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, x));
      mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, x));
    }
    const float mn0 = fmaxf(m0, mx0 * sl2), mn1 = fmaxf(m1, mx1 * sl2);      // the scale is above zero (checked by the launcher)
    const float e0 = mn0 == -INFINITY ? 0.f : mn0, e1 = mn1 == -INFINITY ? 0.f : mn1;
    const float r0 = ex2_approx(m0 - e0), r1 = ex2_approx(m1 - e1);
    m0 = mn0; m1 = mn1;
    l0 *= r0; l1 *= r1;
#pragma unroll
    for (int i = 0; i < 2 * DK; ++i) { o[i][0] *= r0; o[i][1] *= r0; o[i][2] *= r1; o[i][3] *= r1; }
    uint32_t pa[4][4];                                // P as A fragments: 4 k-steps of 16 keys
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const float p0 = ex2_approx(fmaf(s[n][0], sl2, -e0)), p1 = ex2_approx(fmaf(s[n][1], sl2, -e0));
      const float p2 = ex2_approx(fmaf(s[n][2], sl2, -e1)), p3 = ex2_approx(fmaf(s[n][3], sl2, -e1));
      l0 += p0 + p1;
      l1 += p2 + p3;
      pa[n >> 1][(n & 1) * 2] = pack_pair<T>(p0, p1);
      pa[n >> 1][(n & 1) * 2 + 1] = pack_pair<T>(p2, p3);
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
      for (int n = 0; n < 2 * DK; n += 2) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4_trans(smem_u32(bv + (kk * 16 + (lane & 15)) * LD + n * 8 + (lane >> 4) * 8), b0, b1, b2, b3);
        mma_16816<T>(o[n], pa[kk], b0, b1);
        mma_16816<T>(o[n + 1], pa[kk], b2, b3);
      }
    }
    __syncthreads();                                  // everyone is done with `buf` before the next prefetch lands in it
  }
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = warp * 16 + (lane >> 2) + 8 * half, rr = row0 + r;
    if (r >= nrows || p.of[grp.first + rr / rep] != (int)blockIdx.z) continue;          // a row's ranges have one writer
    const long long at = ((long long)(grp.first + rr / rep) * p.H + g * rep + rr % rep) * p.nsplit + blockIdx.x;
    if ((lane & 3) == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = half ? make_float2(m1, l1) : make_float2(m0, l0);
#pragma unroll
    for (int n = 0; n < 2 * DK; ++n)
      *reinterpret_cast<float2*>(p.part_o + at * D + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// own keys, and both parts together
// ------------------------------------------------------------------------------------------------------------------
// A CTA owns one token and up to eight query heads of one KV head; its warps take blocks of 16 keys in turn, each with a ring of its own that its
// first lane refills by TMA (one box per page and 64 dimensions, 128-byte swizzle). On mma.sync: S^T = K Q^T, the keys the first operand and the
// heads the eight columns, then O^T = V^T P^T with V turned by ldmatrix; P changes sides by movmatrix. Rings against 16-byte loads into registers: 64 tokens with
// 300 keys of their own 33 -> 20 us. How many warps: own_warps. Rings of three blocks instead of two 37 us (three warps) against 32; five warps of two 34.
constexpr int kPxOwn = 16, kPxStages = 2, kPxCluster = 4, kPxClusterWarps = 8 * kPxCluster;

__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int DK, int W> struct OwnSmem {
  static constexpr int kHalves = (DK + 3) / 4, LD = 64 * kHalves + 4;       // LD: floats of a row of O
  static constexpr int kBlock = kHalves * 2048, kStage = 2 * kBlock;        // 16 keys, 16 keys and their values
  static constexpr int kRing = kPxStages * kStage, kBytes = W * kRing + 8 * W * kPxStages;
  static_assert(8 * LD * 4 <= kRing, "a warp's O is joined where its ring was");
};

template <typename T, int DK, int W>                  // head size = 16 * DK, warps
__global__ void __launch_bounds__(32 * W)
prefix_own_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const PrefixParams p, const int cl) {
  using L = OwnSmem<DK, W>;
  constexpr int D = 16 * DK, LD = L::LD;
  extern __shared__ __align__(1024) uint8_t smem_own[];
  __shared__ float sml[W][8][2], sw[8][kPxClusterWarps + 32], sinv[8];  // of each head: weights of the cluster's warps and of up to 32 ranges
  const int rep = p.H / p.G, passes = ceil_div(rep, 8);
  // cl CTAs, a cluster, share the keys of a token
  const int t = blockIdx.x / cl, rank = blockIdx.x % cl, kvh = blockIdx.y / passes, h0 = kvh * rep + (blockIdx.y % passes) * 8, nh = min(8, kvh * rep + rep - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t ring = smem_u32(smem_own) + warp * L::kRing, bars = smem_u32(smem_own) + W * L::kRing + warp * kPxStages * 8;
  if (lane == 0) {
    for (int s = 0; s < kPxStages; ++s) mbar_init(bars + 8 * s, 1);
    fence_mbar_init();
  }
  const int slot = p.slot[t], j = p.of[t], pos = p.pos[t];
  const bool listed = (unsigned)slot < (unsigned)p.table_rows;
  const int* trow = p.table + (listed ? slot : 0) * p.table_stride;
  const int k_hi = listed ? (int)min((long long)pos + 1, (long long)p.width << p.bs_log2) : 0;
  // the shared part holds for this token if it is one of the group's and sees all of it
  int k_lo = 0, used = 0;
  if ((unsigned)j < (unsigned)p.n_groups) {
    const PrefixGroup grp = prefix_group(p, j);
    if (t >= grp.first && t < grp.first + grp.tokens && k_hi >= grp.shared) { k_lo = grp.shared; used = ranges_used(p, grp.shared); }
  }
  // this warp's blocks: n of them, the i-th at key_at(i). They start at multiples of 16, so that each lies in one page (pages of 8: in two)
  const int stride = W * cl * kPxOwn, base = (k_lo & ~(kPxOwn - 1)) + (rank * W + warp) * kPxOwn, n = base < k_hi ? (k_hi - base + stride - 1) / stride : 0;
  auto key_at = [&](int i) { return base + i * stride; };
  const int psl = min(p.bs_log2, 4), pieces = kPxOwn >> psl, pool_rows = (p.n_pages * p.G) << p.bs_log2;
  // Lane x holds the pool row of piece x % pieces of block (first of a set) + x / pieces. A piece behind the token's keys, or on a page outside the
  // pools, is asked for behind the pools' last row: zeros
  const int set = 32 / pieces;
  auto rows_of = [&](int first) {
    const int i = first + lane / pieces, k = key_at(i) + (lane % pieces << psl);
    const int page = i < n && k < k_hi ? page_of(p, trow, k) : -1;
    return page >= 0 ? ((page * p.G + kvh) << p.bs_log2) + (k & ((1 << p.bs_log2) - 1)) : pool_rows;
  };
  int rows = rows_of(0), have = 0;                    // for blocks have .. have + set - 1
  auto fetch = [&](int i) {                           // whole warp
    if (i >= n) return;
    if (i - have >= set) { have += set; rows = rows_of(have); }
    const int s = i % kPxStages;
    const uint32_t bar = bars + 8 * s, at = ring + s * L::kStage;
    if (lane == 0) mbar_arrive_expect_tx(bar, L::kStage);
    __syncwarp();
    for (int x = 0; x < pieces; ++x) {
      const int row = __shfl_sync(0xffffffffu, rows, (i - have) * pieces + x);
      if (lane < L::kHalves) tma_load_2d(at + lane * 2048 + (x << psl) * 128, &tk, bar, lane * 64, row);
      else if (lane < 2 * L::kHalves) tma_load_2d(at + lane * 2048 + (x << psl) * 128, &tv, bar, (lane - L::kHalves) * 64, row);
    }
  };
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPxStages; ++i) fetch(i);
  // Q^T as the second operand of S^T
  uint32_t qf[DK][2];
  {
    const T* q = reinterpret_cast<const T*>(p.q) + (long long)t * p.q_stride + (long long)(h0 + min(g, nh - 1)) * D + 2 * c;
#pragma unroll
    for (int i = 0; i < DK; ++i) {
      qf[i][0] = g < nh ? *reinterpret_cast<const uint32_t*>(q + 16 * i) : 0u;
      qf[i][1] = g < nh ? *reinterpret_cast<const uint32_t*>(q + 16 * i + 8) : 0u;
    }
  }
  float o[DK][4];
#pragma unroll
  for (int i = 0; i < DK; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;     // heads 2 c and 2 c + 1
  const float sl2 = p.scale_log2;
  // where a lane's rows of ldmatrix are: keys by rows of 16 and chunk, values (turned) by groups of 8 keys and chunk
  const int kr = lane & 15, kc = lane >> 4, vr = (lane & 7) + 8 * (lane >> 4), vc = (lane >> 3) & 1;
  for (int i = 0; i < n; ++i) {
    const int st = i % kPxStages, kb = key_at(i);
    const uint32_t ka = ring + st * L::kStage + kr * 128, va = ring + st * L::kStage + L::kBlock + vr * 128;
    mbar_wait_warp(bars + 8 * st, (uint32_t)(i / kPxStages) & 1u);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < DK; ++x) {
      uint32_t a[4];
      ldsm_x4(ka + (x >> 2) * 2048 + ((((x & 3) * 2 + kc) ^ (kr & 7)) << 4), a[0], a[1], a[2], a[3]);
      mma_16816<T>(s, a, qf[x][0], qf[x][1]);
    }
    uint32_t keep0 = ~0u, keep1 = ~0u;                // pairs of values of this lane's keys
    const bool ragged = kb < k_lo || kb + kPxOwn > k_hi;
    if (ragged) {
      auto out = [&](int k) { return kb + k < k_lo || kb + k >= k_hi; };
      if (out(g)) s[0] = s[1] = -INFINITY;
      if (out(g + 8)) s[2] = s[3] = -INFINITY;
      // values of keys that are not the token's own become zeros: a weight of zero does not undo a NaN
      keep0 = (out(2 * c) ? 0u : 0xffffu) | (out(2 * c + 1) ? 0u : 0xffff0000u);
      keep1 = (out(2 * c + 8) ? 0u : 0xffffu) | (out(2 * c + 9) ? 0u : 0xffff0000u);
    }
    float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) {
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, x));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, x));
    }
    const float n0 = fmaxf(m0, x0 * sl2), n1 = fmaxf(m1, x1 * sl2);
    const float e0 = n0 == -INFINITY ? 0.f : n0, e1 = n1 == -INFINITY ? 0.f : n1;
    const float r0 = ex2_approx(m0 - e0), r1 = ex2_approx(m1 - e1);
    m0 = n0; m1 = n1;
    const float p0 = ex2_approx(fmaf(s[0], sl2, -e0)), p1 = ex2_approx(fmaf(s[1], sl2, -e1));
    const float p2 = ex2_approx(fmaf(s[2], sl2, -e0)), p3 = ex2_approx(fmaf(s[3], sl2, -e1));
    l0 = fmaf(l0, r0, p0 + p2);
    l1 = fmaf(l1, r1, p1 + p3);
    const uint32_t b0 = turn8x8(pack_pair<T>(p0, p1)), b1 = turn8x8(pack_pair<T>(p2, p3));
#pragma unroll
    for (int x = 0; x < DK; ++x) {
      uint32_t a[4];
      ldsm_x4_trans(va + (x >> 2) * 2048 + ((((x & 3) * 2 + vc) ^ (vr & 7)) << 4), a[0], a[1], a[2], a[3]);
      if (ragged) { a[0] &= keep0; a[1] &= keep0; a[2] &= keep1; a[3] &= keep1; }
      o[x][0] *= r0; o[x][1] *= r1; o[x][2] *= r0; o[x][3] *= r1;
      mma_16816<T>(o[x], a, b0, b1);
    }
    __syncwarp();                                     // every lane has read the stage
    fetch(i + kPxStages);
  }
  // ---- the warps' parts, the ranges of the shared keys and the sink ----
#pragma unroll
  for (int x = 4; x <= 16; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  if (g == 0) {
    sml[warp][2 * c][0] = m0; sml[warp][2 * c][1] = l0;
    sml[warp][2 * c + 1][0] = m1; sml[warp][2 * c + 1][1] = l1;
  }
  float* so = reinterpret_cast<float*>(smem_own + warp * L::kRing);
#pragma unroll
  for (int i = 0; i < DK; ++i) {
    so[2 * c * LD + 16 * i + g] = o[i][0];
    so[(2 * c + 1) * LD + 16 * i + g] = o[i][1];
    so[2 * c * LD + 16 * i + g + 8] = o[i][2];
    so[(2 * c + 1) * LD + 16 * i + g + 8] = o[i][3];
  }
  pdl_wait();
  if (cl > 1) cluster_sync_all();
  else __syncthreads();
  const int warps = cl * W;                           // up to 32: one to a lane
  auto of_warp = [&](int w, const void* mine) { return mapa_shared(smem_u32(mine), w / W); };
  auto load2 = [](uint32_t at) { float2 x; asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(at) : "memory"); return x; };
  auto load4 = [](uint32_t at) {
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
    return x;
  };
  for (int hh = warp; hh < nh; hh += W) {             // a lane for each range and each warp's part
    const long long at = ((long long)t * p.H + h0 + hh) * p.nsplit + lane;
    const float2 ml = lane < used ? *reinterpret_cast<const float2*>(p.part_ml + 2 * at) : make_float2(-INFINITY, 0.f);
    const float2 own = lane < warps ? load2(of_warp(lane, &sml[lane % W][hh][0])) : make_float2(-INFINITY, 0.f);
    const float sink = p.sinks ? p.sinks[h0 + hh] * kPxLog2e : -INFINITY;
    const float top = fmaxf(warp_max(fmaxf(ml.x, own.x)), sink), e = top == -INFINITY ? 0.f : top;
    const float w1 = ex2_approx(own.x - e), w2 = ex2_approx(ml.x - e);
    const float total = warp_sum(own.y * w1 + ml.y * w2) + ex2_approx(sink - e);
    if (lane < warps) sw[hh][lane] = w1;
    if (lane < used) sw[hh][kPxClusterWarps + lane] = w2;
    if (lane == 0) sinv[hh] = total == 0.f ? 0.f : 1.f / total;      // a row that sees no key is zero
  }
  __syncthreads();
  for (int i = rank * (32 * W) + threadIdx.x; i < nh * (D / 4); i += cl * (32 * W)) {
    const int hh = i / (D / 4), d = i % (D / 4) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    auto take = [&](const float4 x, float w) { a.x = fmaf(x.x, w, a.x); a.y = fmaf(x.y, w, a.y); a.z = fmaf(x.z, w, a.z); a.w = fmaf(x.w, w, a.w); };
#pragma unroll 4
    for (int w = 0; w < warps; ++w) take(load4(of_warp(w, smem_own + (w % W) * L::kRing + (hh * LD + d) * 4)), sw[hh][w]);
    const float4* part = reinterpret_cast<const float4*>(p.part_o + ((long long)t * p.H + h0 + hh) * p.nsplit * D + d);
    for (int r0 = 0; r0 < used; r0 += 8) {            // eight at a time, the last ones too: one after another each is a wait of its own
      float4 x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r0 + r < used) x[r] = part[(long long)(r0 + r) * (D / 4)];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r0 + r < used) take(x[r], sw[hh][kPxClusterWarps + r0 + r]);
    }
    const float inv = sinv[hh];
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + ((long long)t * p.H + h0 + hh) * D + d) =
        make_uint2(pack_pair<T>(a.x * inv, a.y * inv), pack_pair<T>(a.z * inv, a.w * inv));
  }
  if (cl > 1) cluster_sync_all();                     // its shared memory has been read by the others
}

template <typename T, int DK>
static int launch_shared_mma(const PrefixParams& p, dim3 grid, cudaStream_t st) {
  const size_t smem = (size_t)(4 * kPxKeys) * (16 * DK + 8) * sizeof(T);
  auto kern = prefix_shared_mma_kernel<T, DK>;
  // per call: the attribute belongs to the current device, and a process may use several
  if (smem > 48 * 1024) B200_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute room = most_shared_memory();
  cfg.gridDim = grid; cfg.blockDim = dim3(128); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cfg.attrs = &room;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, p);
}

// The second kernel starts while the first one ends: it waits for it (griddepcontrol.wait) before it takes up the ranges, its own keys, queries and
// tables are of launches that were complete when the first one began.
template <typename T, int DK, int W>
static int launch_own_by(const PrefixParams& p, dim3 grid, int cl, cudaStream_t st) {
  using L = OwnSmem<DK, W>;
  // rows of the pools, boxes of 64 dimensions (those behind the head size come as zeros) and up to 16 keys
  const uint64_t dims[2] = {16 * DK, (uint64_t)((p.n_pages * p.G) << p.bs_log2)}, str[1] = {32 * DK};
  const uint32_t box[2] = {64, (uint32_t)(p.bs_log2 < 4 ? 1 << p.bs_log2 : kPxOwn)};
  CUtensorMap tk, tv;
  if (int rc = make_tensor_map(&tk, p.ck, 2, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&tv, p.cv, 2, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  auto kern = prefix_own_kernel<T, DK, W>;
  // per call: the attribute belongs to the current device, and a process may use several
  B200_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(32 * W); cfg.dynamicSmemBytes = L::kBytes; cfg.stream = st;
  cudaLaunchAttribute attr[3];
  int na = 1;
  attr[0] = most_shared_memory();
  if (cl > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = cl; attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
    ++na;
  }
  if (p.n_groups > 0 && p.longest > 0) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  return (int)cudaLaunchKernelEx(&cfg, kern, tk, tv, p, cl);
}
// Warps of a CTA that has a token to itself, heads of 128. Those that run beside the tcgen05 kernel end only after it, and what no SM has room for until then starts from
// the beginning: two waves. So where four warps to a CTA leave some out, three or two, if then all have room. beside: CTAs of that kernel, one to an SM.
// 40 tokens, 4096 shared and up to 600 own keys, four warps 25.9 us, three 22.2, two 25.8; 64 tokens (three leave some out) 30.8, 31.5, 28; with one own key 19.9, 19.2,
// 18.2. Two warps are slower at own keys alone: up to 2400 of them 74 us, three 62, four 62; 64 tokens, 4096 shared and up to 1000 own keys 40.3, four 39.8.
constexpr int kPxTwoWarps = 800;                      // own keys, at most, for two
static int own_warps(long long ctas, long long beside, int most_own, bool* room = nullptr) {
  const bool one = beside <= kNumSMs, four = one && ctas <= 3 * kNumSMs - 2 * beside, three = one && ctas <= 4 * kNumSMs - 2 * beside,
             two = one && ctas <= 6 * kNumSMs - 3 * beside && most_own <= kPxTwoWarps;
  if (room) *room = four || three || two;
  return four ? 4 : three ? 3 : two ? 2 : 4;
}
template <typename T, int DK>
static int launch_own(const PrefixParams& p, dim3 grid, cudaStream_t st) {
  // Where there are fewer CTAs than SMs, eight warps to each (four otherwise: then three CTAs fit an SM), and up to four CTAs to a token, while each warp has
  // two blocks. 32 / 8 heads of 128, own keys of up to 3000 for 2 tokens 37.9 -> 12.9 us (with eight CTAs to a token 21.9), of 2000 for 8 30.7 -> 21.5; 16 / 4
  // heads, 8000 keys for 4 tokens 99 -> 22; 64 tokens by eight warps 29.7 -> 37.5, 4 tokens with 40 keys 7.7 -> 7.9.
  const long long ctas = (long long)grid.x * grid.y;
  if (ctas > kNumSMs || p.most_own <= 256) {
    if constexpr (DK == 8) {
      const int w = own_warps(ctas, p.beside, p.most_own);
      if (w == 2) return launch_own_by<T, DK, 2>(p, grid, 1, st);
      if (w == 3) return launch_own_by<T, DK, 3>(p, grid, 1, st);
    }
    return launch_own_by<T, DK, 4>(p, grid, 1, st);
  }
  int cl = 1;
  while (cl < kPxCluster && ctas * cl * 2 <= kNumSMs && p.most_own >= 256 * cl) cl *= 2;
  grid.x *= cl;
  return launch_own_by<T, DK, 8>(p, grid, cl, st);
}

template <typename T>
static int prefix_attn(const PrefixParams& p, bool tc, cudaStream_t st) {
  const int rep = p.H / p.G;
  if (p.n_groups > 0 && p.longest > 0) {
    int rc = B200_ERR_UNSUPPORTED;
    const dim3 grid(p.nsplit, p.G * ceil_div(p.longest * rep, kPxRows), p.n_groups);
#define SHARED(DK) case DK: rc = launch_shared_mma<T, DK>(p, grid, st); break
    if (tc) rc = prefix_shared_tc(p, std::is_same<T, __nv_bfloat16>::value ? B200_DT_BF16 : B200_DT_FP16, st);
    else switch (p.D / 16) { SHARED(1); SHARED(2); SHARED(3); SHARED(4); SHARED(5); SHARED(6); SHARED(7); SHARED(8); }
#undef SHARED
    if (rc) return rc;
  }
#define OWN(DK) case DK: return launch_own<T, DK>(p, dim3(p.T, p.G * ceil_div(rep, 8)), st)
  switch (p.D / 16) { OWN(1); OWN(2); OWN(3); OWN(4); OWN(5); OWN(6); OWN(7); OWN(8); }
#undef OWN
  return B200_ERR_UNSUPPORTED;
}

}  // namespace b200
using namespace b200;

// How the shared keys of a call are worked on: the number of ranges (1 .. 32), plus kPxTc where tcgen05 does it.
// Which kernel: tcgen05 for the head sizes that it has, but for up to 32 rows a group and 1024 keys (device time with up to 20 own keys, each kernel at its best number
// of ranges; 32 / 8 heads of 128, one token, 600 keys: 9.6 us, 7.6 on mma.sync; 4096 keys: 12.1 and 13.4, 16000: 21.9 and 32; 32 rows, 1024 keys: 9.9 and 9.6, 2048:
// 10.8 and 11.4; 64 rows, 16000 keys: 22.6 and 37; 128 rows: 24 and 60).
// How many ranges: those that a cost makes cheapest, in us: the blocks of a CTA, each of which takes longer where an SM has more CTAs (0.72 and 1.15
// for one and two on tcgen05, 1.7 for each on mma.sync), rounds of CTAs, the ranges' way through L2, written and read at 4 TB/s, a wait for each eight of them where they are joined, and
// where not all CTAs of own keys have room beside the shared ones (own_warps) their first steps once more. 64 x 4096 keys with 32 / 8 heads and up to 600 own ones:
// 4, 6, 7, 8, 9 ranges 28, 28, 28, 31, 31 us (chosen: 7); 40 x 3000 and up to 512, 16 / 2 heads: 4, 8, 11, 24 ranges 17, 13.3, 13, 17 (8); 128 x 16384 and up to 512: 4, 8,
// 9, 12 ranges 80, 68, 69, 83 (9); 100 x 8000 and up to 512, 12 / 2 heads of 64: 4, 9, 12, 14, 18 ranges 30, 19.5, 18, 17.2, 17.5 (14).
// These are plans of the batch as it is. A captured step has to plan for every batch that it may replay: up to four groups as long as the batch, the cache's longest
// sequences, own keys unknown. 64 x 4096 and up to 600: 32 instead of 28 us; 40 x 4096: 26.6 and 22.9; 128 x 16384: 78 and 69; 4 x 512 and up to 40 (on tcgen05): 11.3 and 7.9.
constexpr int kPxTc = 256;
// CTAs of the shared keys' kernel for one range: tiles of the longest group for each, but no more than the batch can fill
static long long shared_items(int T, int n_groups, int longest, int rep, int G, int tc_tokens) {
  const long long of_longest = tc_tokens > 0 ? ceil_div(longest, tc_tokens) : ceil_div64((int64_t)longest * rep, kPxRows);
  const long long of_batch = (tc_tokens > 0 ? T / tc_tokens : (long long)T * rep / kPxRows) + n_groups;
  return G * (n_groups * of_longest < of_batch ? n_groups * of_longest : of_batch);
}
B200_API int b200_prefix_attn_plan(int T, int n_groups, int longest, int max_shared, int most_own, int H, int G, int D) {
  if (T < 1 || n_groups < 1 || longest < 1 || max_shared < 1 || H < 1 || G < 1 || H % G) return 1;
  const int rep = H / G, tokens = prefix_tc_tokens(H, G, D);
  const bool tc = tokens > 0 && !((long long)longest * rep <= 32 && max_shared <= 1024);
  const long long items = shared_items(T, n_groups, longest, rep, G, tc ? tokens : 0), blocks = ceil_div64(max_shared, kPxKeys);
  const long long own = (long long)T * G * ceil_div(rep, 8);
  const int resident = tc ? 2 : 3;
  const double pass = (double)T * H * D * 8 / 4e6;
  int best = 1;
  double least = 0;
  for (int n = 1; n <= 32 && n <= blocks; ++n) {
    const long long ctas = items * n, rounds = ceil_div64(ctas, resident * kNumSMs);
    const int beside = ctas > resident * kNumSMs ? resident : (int)ceil_div64(ctas, kNumSMs);
    double cost = rounds * ceil_div64(blocks, n) * (tc ? 0.29 + 0.43 * beside : 1.7 * beside) + n * pass;
    cost += ceil_div(n, 8);
    bool room = true;
    if (tc && D == 128) own_warps(own, ctas, most_own > 0 ? most_own : 0x7fffffff, &room);
    if (!room) cost += 3;
    if (n == 1 || cost < least) { best = n; least = cost; }
  }
  return best + (tc ? kPxTc : 0);
}

B200_API int b200_prefix_attn(const void* q, long long q_stride, const void* ck, const void* cv, int n_pages, const int* pos, const int* slot,
                              const int* table, long long table_stride, int table_rows, int width, const int* groups, const int* of, int n_groups,
                              int longest, const float* sinks, void* out, float* part, int plan, int most_own, int T, int H, int G, int D, int block_size,
                              float scale, int dtype, void* stream) {
  if (T <= 0) return 0;
  if ((dtype != B200_DT_BF16 && dtype != B200_DT_FP16) || D % 16 || D < 16 || D > 128 || !(scale > 0.f)) return B200_ERR_UNSUPPORTED;
  const bool tc = plan >= kPxTc;
  const int nsplit = tc ? plan - kPxTc : plan;
  if (H < 1 || G < 1 || H % G || n_pages < 0 || table_rows < 1 || width < 1 || n_groups < 0 || nsplit < 1 || nsplit > 32 || block_size < 1 ||
      q_stride < (long long)H * D) return B200_ERR_BAD_SHAPE;
  if (n_groups > 65535 || (long long)G * ceil_div64((int64_t)(longest < 1 ? 1 : longest) * (H / G), kPxRows) > 65535 || H > 65535) return B200_ERR_TOO_LARGE;
  if (q_stride % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(ck) | reinterpret_cast<uintptr_t>(cv) |
                        reinterpret_cast<uintptr_t>(part)) & 15)) return B200_ERR_BAD_ALIGN;
  PrefixParams p = {};
  while ((1 << p.bs_log2) < block_size) ++p.bs_log2;
  // a swizzled box starts on a group of eight rows, and rows of the pools and keys of a sequence are counted in 32 bits
  if ((1 << p.bs_log2) != block_size || block_size < 8 || n_pages < 1 || (long long)n_pages * G * block_size >= 0x7fffff00LL ||
      (long long)width * block_size >= 0x7ffff000LL) return B200_ERR_UNSUPPORTED;
  if (n_groups > 0 && longest > 0 && !part) return B200_ERR_BAD_SHAPE;
  if (tc && prefix_tc_tokens(H, G, D) < 1) return B200_ERR_UNSUPPORTED;
  p.q = q; p.ck = ck; p.cv = cv; p.q_stride = q_stride; p.pos = pos; p.slot = slot; p.table = table; p.table_stride = table_stride;
  p.table_rows = table_rows; p.width = width; p.n_pages = n_pages; p.groups = groups; p.of = of; p.n_groups = n_groups;
  p.longest = longest; p.sinks = sinks; p.out = out; p.T = T; p.H = H; p.G = G; p.D = D; p.nsplit = nsplit;
  p.part_o = part; p.part_ml = part ? part + (long long)T * H * nsplit * D : nullptr;
  p.most_own = most_own > 0 ? most_own : 0x7fffffff;
  p.beside = tc ? shared_items(T, n_groups, longest, H / G, G, prefix_tc_tokens(H, G, D)) * nsplit : 0;
  p.scale_log2 = scale * kPxLog2e;
  return dtype == B200_DT_BF16 ? prefix_attn<__nv_bfloat16>(p, tc, (cudaStream_t)stream) : prefix_attn<__half>(p, tc, (cudaStream_t)stream);
}
