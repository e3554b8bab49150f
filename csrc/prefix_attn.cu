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
#include "prefix_attn.cuh"
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
// A CTA owns one token and up to eight query heads of one KV head; its warps take blocks of 16 keys in turn. Keys and values go from memory
// straight into the registers that mma.sync reads, 16 bytes to a load, whole rows side by side: the keys are the first operand of S^T = K Q^T and
// the values, turned in pairs of rows, that of O^T = V^T P^T, the heads the eight columns of both. For that the dimensions are taken in
// the order in which they lie in the lanes, the same for Q and K, and undone where O is written; P changes sides by movmatrix. Against a lane per
// key and chunk with FMAs, which kept two keys in flight per lane and spent 140 instructions on each pair of keys: 64 tokens with 300 own keys each, 32 / 8
// heads of 128 (78 MB).
constexpr int kPxOwn = 16;

__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T, int KC>                         // KC: head size in chunks of 32, rounded up
__global__ void __launch_bounds__(128, 3)
prefix_own_kernel(const PrefixParams p) {
  constexpr int VC = (KC + 1) / 2, LD = 64 * VC + 4;
  __shared__ __align__(16) float so[4][8][LD];
  __shared__ float sml[4][8][2], sw[8][36], sinv[8];  // of each head: weights of the four warps and of up to 32 ranges
  const int D = p.D, rep = p.H / p.G, passes = ceil_div(rep, 8);
  const int t = blockIdx.x, kvh = blockIdx.y / passes, h0 = kvh * rep + (blockIdx.y % passes) * 8, nh = min(8, kvh * rep + rep - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
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
  const T* ck = reinterpret_cast<const T*>(p.ck);
  const T* cv = reinterpret_cast<const T*>(p.cv);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  uint4 qf[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int d = i * 32 + c * 8;
    qf[i] = g < nh && d < D ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.q) + (long long)t * p.q_stride + (long long)(h0 + g) * D + d) : zero;
  }
  const int bs_mask = (1 << p.bs_log2) - 1;
  const bool one_page = p.bs_log2 >= 4;               // a block lies in one page
  auto page_at = [&](int kb) { return kb < k_hi ? page_of(p, trow, kb) : -1; };
  // row of key k in the pools, -1: not read
  auto row_of = [&](int k, int page) -> long long {
    if (k < k_lo || k >= k_hi) return -1;
    if (!one_page) page = page_of(p, trow, k);
    return page < 0 ? -1 : (((long long)page * p.G + kvh) << p.bs_log2) + (k & bs_mask);
  };
  uint4 kr[KC][2], vr[VC][4];
  auto load_k = [&](int kb, int page) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const long long row = row_of(kb + g + 8 * r, page);
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const int d = i * 32 + c * 8;
        kr[i][r] = row >= 0 && d < D ? *reinterpret_cast<const uint4*>(ck + row * D + d) : zero;
      }
    }
  };
  auto load_v = [&](int kb, int page) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long long row = row_of(kb + 2 * c + (r & 1) + 8 * (r >> 1), page);
#pragma unroll
      for (int i = 0; i < VC; ++i) {
        const int d = i * 64 + g * 8;
        vr[i][r] = row >= 0 && d < D ? *reinterpret_cast<const uint4*>(cv + row * D + d) : zero;
      }
    }
  };
  float o[4 * VC][4];
#pragma unroll
  for (int i = 0; i < 4 * VC; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;     // heads 2 c and 2 c + 1
  const float sl2 = p.scale_log2;
  int kb = (k_lo & ~(kPxOwn - 1)) + warp * kPxOwn;    // blocks start at multiples of 16: with larger pages each lies in one
  int page = page_at(kb), next = page_at(kb + 4 * kPxOwn);
  if (kb < k_hi) { load_k(kb, page); load_v(kb, page); }
  for (; kb < k_hi; kb += 4 * kPxOwn) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      const uint32_t a0[4] = {kr[i][0].x, kr[i][1].x, kr[i][0].y, kr[i][1].y}, a1[4] = {kr[i][0].z, kr[i][1].z, kr[i][0].w, kr[i][1].w};
      mma_16816<T>(s, a0, qf[i].x, qf[i].y);
      mma_16816<T>(s, a1, qf[i].z, qf[i].w);
    }
    const int after = page_at(kb + 8 * kPxOwn);
    if (kb + 4 * kPxOwn < k_hi) load_k(kb + 4 * kPxOwn, next);   // under way while this block is worked on; V's as soon as its registers are read
    if (kb < k_lo || kb + kPxOwn > k_hi) {
      if (kb + g < k_lo || kb + g >= k_hi) s[0] = s[1] = -INFINITY;
      if (kb + g + 8 < k_lo || kb + g + 8 >= k_hi) s[2] = s[3] = -INFINITY;
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
    for (int i = 0; i < VC; ++i) {
      const uint32_t* v[4] = {&vr[i][0].x, &vr[i][1].x, &vr[i][2].x, &vr[i][3].x};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a[4] = {__byte_perm(v[0][w], v[1][w], 0x5410), __byte_perm(v[0][w], v[1][w], 0x7632),
                               __byte_perm(v[2][w], v[3][w], 0x5410), __byte_perm(v[2][w], v[3][w], 0x7632)};
        float (&oo)[4] = o[4 * i + w];
        oo[0] *= r0; oo[1] *= r1; oo[2] *= r0; oo[3] *= r1;
        mma_16816<T>(oo, a, b0, b1);
      }
    }
    if (kb + 4 * kPxOwn < k_hi) load_v(kb + 4 * kPxOwn, next);
    next = after;
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
#pragma unroll
  for (int i = 0; i < 4 * VC; ++i) {
    const int d = (i >> 2) * 64 + g * 8 + (i & 3) * 2;
    *reinterpret_cast<float2*>(&so[warp][2 * c][d]) = make_float2(o[i][0], o[i][2]);
    *reinterpret_cast<float2*>(&so[warp][2 * c + 1][d]) = make_float2(o[i][1], o[i][3]);
  }
  __syncthreads();
  for (int hh = warp; hh < nh; hh += 4) {             // a lane for each range; the first four take a warp's part each as well
    const long long at = ((long long)t * p.H + h0 + hh) * p.nsplit + lane;
    const float2 ml = lane < used ? *reinterpret_cast<const float2*>(p.part_ml + 2 * at) : make_float2(-INFINITY, 0.f);
    const float wm = lane < 4 ? sml[lane][hh][0] : -INFINITY, wl = lane < 4 ? sml[lane][hh][1] : 0.f;
    const float sink = p.sinks ? p.sinks[h0 + hh] * kPxLog2e : -INFINITY;
    const float top = fmaxf(warp_max(fmaxf(ml.x, wm)), sink), e = top == -INFINITY ? 0.f : top;
    const float w1 = ex2_approx(wm - e), w2 = ex2_approx(ml.x - e);
    const float total = warp_sum(wl * w1 + ml.y * w2) + ex2_approx(sink - e);
    if (lane < 4) sw[hh][lane] = w1;
    if (lane < used) sw[hh][4 + lane] = w2;
    if (lane == 0) sinv[hh] = total == 0.f ? 0.f : 1.f / total;      // a row that sees no key is zero
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * (D / 2); i += 128) {
    const int hh = i / (D / 2), d = i % (D / 2) * 2;
    float2 a = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float2 x = *reinterpret_cast<const float2*>(&so[w][hh][d]);
      a.x = fmaf(x.x, sw[hh][w], a.x);
      a.y = fmaf(x.y, sw[hh][w], a.y);
    }
    const float2* part = reinterpret_cast<const float2*>(p.part_o + ((long long)t * p.H + h0 + hh) * p.nsplit * D + d);
#pragma unroll 4
    for (int r = 0; r < used; ++r) {
      const float2 x = part[(long long)r * (D / 2)];
      a.x = fmaf(x.x, sw[hh][4 + r], a.x);
      a.y = fmaf(x.y, sw[hh][4 + r], a.y);
    }
    *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + ((long long)t * p.H + h0 + hh) * D + d) = pack_pair<T>(a.x * sinv[hh], a.y * sinv[hh]);
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
  const dim3 grid(p.T, p.G * ceil_div(rep, 8));
  switch ((p.D + 31) / 32) {
    case 1: prefix_own_kernel<T, 1><<<grid, 128, 0, st>>>(p); break;
    case 2: prefix_own_kernel<T, 2><<<grid, 128, 0, st>>>(p); break;
    case 3: prefix_own_kernel<T, 3><<<grid, 128, 0, st>>>(p); break;
    default: prefix_own_kernel<T, 4><<<grid, 128, 0, st>>>(p); break;
  }
  B200_LAUNCH_CHECK();
  return 0;
}

}  // namespace b200
using namespace b200;

// How the shared keys of a call are worked on: the number of ranges (1 .. 32), plus kPxTc where tcgen05 does it.
constexpr int kPxTc = 256;
B200_API int b200_prefix_attn_plan(int n_groups, int longest, int max_shared, int H, int G, int D, int block_size, int n_pages) {
  if (n_groups < 1 || longest < 1 || max_shared < 1 || H < 1 || G < 1 || H % G || block_size < 1 || n_pages < 0) return 1;
  const int rep = H / G, tokens = prefix_tc_tokens(H, G, D, block_size);
  const bool tc = tokens > 0 && (long long)longest * rep > 32 && (long long)n_pages * G * block_size < 0x7fffff00LL;
  const long long items = (long long)n_groups * G * (tc ? ceil_div(longest, tokens) : ceil_div64((int64_t)longest * rep, kPxRows));
  long long n = ceil_div64(tc ? 2 * kNumSMs : 3 * kNumSMs, items);
  const long long most = ceil_div64(max_shared, 256);
  if (n > most) n = most;
  return (int)(n > 32 ? 32 : n) + (tc ? kPxTc : 0);
}

B200_API int b200_prefix_attn(const void* q, long long q_stride, const void* ck, const void* cv, int n_pages, const int* pos, const int* slot,
                              const int* table, long long table_stride, int table_rows, int width, const int* groups, const int* of, int n_groups,
                              int longest, const float* sinks, void* out, float* part, int plan, int T, int H, int G, int D, int block_size,
                              float scale, int dtype, void* stream) {
  if (T <= 0) return 0;
  if ((dtype != B200_DT_BF16 && dtype != B200_DT_FP16) || D % 16 || D < 16 || D > 128 || !(scale > 0.f)) return B200_ERR_UNSUPPORTED;
  const bool tc = plan >= kPxTc;
  const int nsplit = tc ? plan - kPxTc : plan;
  if (H < 1 || G < 1 || H % G || n_pages < 0 || table_rows < 1 || width < 1 || n_groups < 0 || nsplit < 1 || nsplit > 32 || block_size < 1) return B200_ERR_BAD_SHAPE;
  if (n_groups > 65535 || (long long)G * ceil_div64((int64_t)(longest < 1 ? 1 : longest) * (H / G), kPxRows) > 65535 || H > 65535) return B200_ERR_TOO_LARGE;
  if (q_stride % 8 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(ck) | reinterpret_cast<uintptr_t>(cv) |
                        reinterpret_cast<uintptr_t>(part)) & 15)) return B200_ERR_BAD_ALIGN;
  PrefixParams p = {};
  while ((1 << p.bs_log2) < block_size) ++p.bs_log2;
  if ((1 << p.bs_log2) != block_size) return B200_ERR_UNSUPPORTED;
  if (n_groups > 0 && longest > 0 && !part) return B200_ERR_BAD_SHAPE;
  if (tc && (prefix_tc_tokens(H, G, D, block_size) < 1 || n_pages < 1 || (long long)n_pages * G * block_size >= 0x7fffff00LL)) return B200_ERR_UNSUPPORTED;
  p.q = q; p.ck = ck; p.cv = cv; p.q_stride = q_stride; p.pos = pos; p.slot = slot; p.table = table; p.table_stride = table_stride;
  p.table_rows = table_rows; p.width = width; p.n_pages = n_pages; p.groups = groups; p.of = of; p.n_groups = n_groups;
  p.longest = longest; p.sinks = sinks; p.out = out; p.T = T; p.H = H; p.G = G; p.D = D; p.nsplit = nsplit;
  p.part_o = part; p.part_ml = part ? part + (long long)T * H * nsplit * D : nullptr;
  p.scale_log2 = scale * kPxLog2e;
  return dtype == B200_DT_BF16 ? prefix_attn<__nv_bfloat16>(p, tc, (cudaStream_t)stream) : prefix_attn<__half>(p, tc, (cudaStream_t)stream);
}
