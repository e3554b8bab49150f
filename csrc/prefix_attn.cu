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
//                once for 64 rows instead of once a sequence. The keys are cut into nsplit ranges, so that few rows still
//                fill the GPU; a range leaves (m, l, o) per row
//   own keys     a CTA for a token and KV head, 16-byte loads, every lane with keys of its own; at its end it takes up the ranges of the
//                shared keys and the sink, and writes the result: no third kernel
//
// Bound: memory, until the rows of a group are so many that the tensor cores are. 64 tokens, 32 / 8 heads of 128, 4096 shared and 300 own keys:
// 17 MB of shared keys and 78 MB of own ones (15 us at 6.5 TB/s), 4.6 GFLOP (3 us); read once a sequence they were 1.15 GB.
#include "common.cuh"
#include "mma_sync.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kPxRows = 64, kPxKeys = 64;
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
// A CTA owns one token and up to HB query heads of one KV head. A lane is (key, 16-byte chunk): the CP lanes of a key read its row and the
// same row of the values with one load each; every lane keeps (max, sum, acc) for the keys it has seen.
template <typename T, int HB>
__global__ void __launch_bounds__(128)
prefix_own_kernel(const PrefixParams p, int CP, int CPR) {
  extern __shared__ float sm[];                       // [4 warps][HB][D + 2]
  const int D = p.D, rep = p.H / p.G, passes = ceil_div(rep, HB);
  const int t = blockIdx.x, g = blockIdx.y / passes, h0 = g * rep + (blockIdx.y % passes) * HB, nh = min(HB, g * rep + rep - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int KPI = 32 / CP, kk = lane / CP, c = lane % CP;
  const bool live = c < CPR;
  const int slot = p.slot[t];
  const bool listed = (unsigned)slot < (unsigned)p.table_rows;
  const int* trow = p.table + (listed ? slot : 0) * p.table_stride;
  const int k_hi = listed ? (int)min((long long)p.pos[t] + 1, (long long)p.width << p.bs_log2) : 0;
  // the shared part holds for this token if it is one of the group's and sees all of it
  const int j = p.of[t];
  int k_lo = 0, used = 0;
  if ((unsigned)j < (unsigned)p.n_groups) {
    const PrefixGroup grp = prefix_group(p, j);
    if (t >= grp.first && t < grp.first + grp.tokens && k_hi >= grp.shared) { k_lo = grp.shared; used = ranges_used(p, grp.shared); }
  }
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* ck = reinterpret_cast<const T*>(p.ck);
  const T* cv = reinterpret_cast<const T*>(p.cv);
  float qv[HB][8], acc[HB][8], m[HB], l[HB];
#pragma unroll
  for (int hh = 0; hh < HB; ++hh) {
    m[hh] = -INFINITY;
    l[hh] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      acc[hh][e] = 0.f;
      qv[hh][e] = (live && hh < nh) ? to_f32<T>(q[(long long)t * p.q_stride + (long long)(h0 + hh) * D + c * 8 + e]) * p.scale_log2 : 0.f;
    }
  }
  const int bs_mask = (1 << p.bs_log2) - 1, stride = 4 * KPI;
  constexpr int U = HB >= 4 ? 2 : 4;                  // keys in flight per lane
  for (int kb = k_lo; kb < k_hi; kb += stride * U) {
    uint4 kr[U], vr[U];
    bool valid[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k0 = kb + u * stride + warp * KPI + kk;
      valid[u] = k0 < k_hi;
      kr[u] = vr[u] = make_uint4(0, 0, 0, 0);
      if (valid[u] && live) {
        const int page = page_of(p, trow, k0);
        if (page >= 0) {
          const long long off = ((((long long)page * p.G + g) << p.bs_log2) + (k0 & bs_mask)) * D + c * 8;
          kr[u] = *reinterpret_cast<const uint4*>(ck + off);
          vr[u] = *reinterpret_cast<const uint4*>(cv + off);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb + u * stride >= k_hi) break;             // uniform over the CTA: no lane has a key in this or a later slot
      float kf[8], vf[8];
      const T* kp = reinterpret_cast<const T*>(&kr[u]);
      const T* vp = reinterpret_cast<const T*>(&vr[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) { kf[e] = to_f32<T>(kp[e]); vf[e] = to_f32<T>(vp[e]); }
#pragma unroll
      for (int hh = 0; hh < HB; ++hh) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(qv[hh][e], kf[e], s);
        for (int o = CP >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (valid[u]) {
          const float mn = fmaxf(m[hh], s), e0 = mn == -INFINITY ? 0.f : mn;
          const float r = ex2_approx(m[hh] - e0), pj = ex2_approx(s - e0);
          m[hh] = mn;
          l[hh] = l[hh] * r + pj;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[hh][e] = fmaf(pj, vf[e], acc[hh][e] * r);
        }
      }
    }
  }
  // the key groups of the warp, then the warps, the ranges of the shared keys and the sink
#pragma unroll
  for (int hh = 0; hh < HB; ++hh) {
    for (int o = CP; o < 32; o <<= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m[hh], o), l2 = __shfl_xor_sync(0xffffffffu, l[hh], o);
      const float mn = fmaxf(m[hh], m2), e0 = mn == -INFINITY ? 0.f : mn;
      const float w1 = ex2_approx(m[hh] - e0), w2 = ex2_approx(m2 - e0);
      l[hh] = l[hh] * w1 + l2 * w2;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[hh][e] = acc[hh][e] * w1 + __shfl_xor_sync(0xffffffffu, acc[hh][e], o) * w2;
      m[hh] = mn;
    }
    if (kk == 0 && live) {
      float* w = sm + (warp * HB + hh) * (D + 2);
      if (c == 0) { w[0] = m[hh]; w[1] = l[hh]; }
#pragma unroll
      for (int e = 0; e < 8; ++e) w[2 + c * 8 + e] = acc[hh][e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * D; i += 128) {
    const int hh = i / D, d = i % D, h = h0 + hh;
    const long long at = ((long long)t * p.H + h) * p.nsplit;
    const float sink = p.sinks ? p.sinks[h] * kPxLog2e : -INFINITY;
    float mt = sink;
#pragma unroll
    for (int w = 0; w < 4; ++w) mt = fmaxf(mt, sm[(w * HB + hh) * (D + 2)]);
    for (int s = 0; s < used; ++s) mt = fmaxf(mt, p.part_ml[2 * (at + s)]);
    const float e0 = mt == -INFINITY ? 0.f : mt;
    float lt = ex2_approx(sink - e0), ot = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float* ws = sm + (w * HB + hh) * (D + 2);
      const float e = ex2_approx(ws[0] - e0);
      lt += ws[1] * e;
      ot += ws[2 + d] * e;
    }
    for (int s = 0; s < used; ++s) {
      const float e = ex2_approx(p.part_ml[2 * (at + s)] - e0);
      lt += p.part_ml[2 * (at + s) + 1] * e;
      ot += p.part_o[(at + s) * D + d] * e;
    }
    // a row that sees no key is zero
    reinterpret_cast<T*>(p.out)[((long long)t * p.H + h) * D + d] = from_f32<T>(lt == 0.f ? 0.f : ot / lt);
  }
}

template <typename T, int DK>
static int launch_shared_mma(const PrefixParams& p, dim3 grid, cudaStream_t st) {
  const size_t smem = (size_t)(4 * kPxKeys) * (16 * DK + 8) * sizeof(T);
  auto kern = prefix_shared_mma_kernel<T, DK>;
  // per call: the attribute belongs to the current device, and a process may use several
  if (smem > 48 * 1024) B200_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kern<<<grid, 128, smem, st>>>(p);
  B200_LAUNCH_CHECK();
  return 0;
}

template <typename T>
static int prefix_attn(const PrefixParams& p, cudaStream_t st) {
  const int rep = p.H / p.G;
  if (p.n_groups > 0 && p.longest > 0) {
    const dim3 grid(p.nsplit, p.G * ceil_div(p.longest * rep, kPxRows), p.n_groups);
    int rc = B200_ERR_UNSUPPORTED;
#define SHARED(DK) case DK: rc = launch_shared_mma<T, DK>(p, grid, st); break
    switch (p.D / 16) { SHARED(1); SHARED(2); SHARED(3); SHARED(4); SHARED(5); SHARED(6); SHARED(7); SHARED(8); }
#undef SHARED
    if (rc) return rc;
  }
  const int CPR = p.D / 8;
  int CP = 1;
  while (CP < CPR) CP <<= 1;
  const int HB = rep >= 4 ? 4 : rep >= 2 ? 2 : 1;
  const dim3 grid(p.T, p.G * ceil_div(rep, HB));
  const size_t smem = (size_t)4 * HB * (p.D + 2) * sizeof(float);
  if (HB == 4) prefix_own_kernel<T, 4><<<grid, 128, smem, st>>>(p, CP, CPR);
  else if (HB == 2) prefix_own_kernel<T, 2><<<grid, 128, smem, st>>>(p, CP, CPR);
  else prefix_own_kernel<T, 1><<<grid, 128, smem, st>>>(p, CP, CPR);
  B200_LAUNCH_CHECK();
  return 0;
}

}  // namespace b200
using namespace b200;

// Ranges that the shared keys of a call are cut into: enough CTAs for three on every SM, of no fewer than 256 keys each
B200_API int b200_prefix_attn_splits(int n_groups, int longest, int max_shared, int H, int G) {
  if (n_groups < 1 || longest < 1 || max_shared < 1 || H < 1 || G < 1 || H % G) return 1;
  const long long items = (long long)n_groups * G * ceil_div64((int64_t)longest * (H / G), kPxRows);
  long long n = ceil_div64(3 * kNumSMs, items);
  const long long most = ceil_div64(max_shared, 256);
  if (n > most) n = most;
  return (int)(n > 32 ? 32 : n);
}

B200_API int b200_prefix_attn(const void* q, long long q_stride, const void* ck, const void* cv, int n_pages, const int* pos, const int* slot,
                              const int* table, long long table_stride, int table_rows, int width, const int* groups, const int* of, int n_groups,
                              int longest, const float* sinks, void* out, float* part, int nsplit, int T, int H, int G, int D, int block_size,
                              float scale, int dtype, void* stream) {
  if (T <= 0) return 0;
  if ((dtype != B200_DT_BF16 && dtype != B200_DT_FP16) || D % 16 || D < 16 || D > 128 || !(scale > 0.f)) return B200_ERR_UNSUPPORTED;
  if (H < 1 || G < 1 || H % G || n_pages < 0 || table_rows < 1 || width < 1 || n_groups < 0 || nsplit < 1 || block_size < 1) return B200_ERR_BAD_SHAPE;
  if (n_groups > 65535 || (long long)G * ceil_div64((int64_t)(longest < 1 ? 1 : longest) * (H / G), kPxRows) > 65535 || H > 65535) return B200_ERR_TOO_LARGE;
  if (q_stride % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(ck) | reinterpret_cast<uintptr_t>(cv) |
                        reinterpret_cast<uintptr_t>(part)) & 15)) return B200_ERR_BAD_ALIGN;
  PrefixParams p = {};
  while ((1 << p.bs_log2) < block_size) ++p.bs_log2;
  if ((1 << p.bs_log2) != block_size) return B200_ERR_UNSUPPORTED;
  if (n_groups > 0 && longest > 0 && !part) return B200_ERR_BAD_SHAPE;
  p.q = q; p.ck = ck; p.cv = cv; p.q_stride = q_stride; p.pos = pos; p.slot = slot; p.table = table; p.table_stride = table_stride;
  p.table_rows = table_rows; p.width = width; p.n_pages = n_pages; p.groups = groups; p.of = of; p.n_groups = n_groups;
  p.longest = longest; p.sinks = sinks; p.out = out; p.T = T; p.H = H; p.G = G; p.D = D; p.nsplit = nsplit;
  p.part_o = part; p.part_ml = part ? part + (long long)T * H * nsplit * D : nullptr;
  p.scale_log2 = scale * kPxLog2e;
  return dtype == B200_DT_BF16 ? prefix_attn<__nv_bfloat16>(p, (cudaStream_t)stream) : prefix_attn<__half>(p, (cudaStream_t)stream);
}
