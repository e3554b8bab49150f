// Shared keys of a prefix-attention call on the 5th-generation tensor cores (see prefix_attn.cu for the mathematics and the other kernels).
//
//   CTA = up to 128 rows (tokens x heads of one KV head) and one range of the group's shared keys, 192 threads: warps 0 - 3 softmax (thread = row,
//   TMEM lane = row, so that a row's maximum and sum need no shuffles), warp 4 TMA producer, warp 5 tcgen05 issuer (the whole warp runs
//   the loop, elect.sync picks the lane). Two CTAs per SM fill each other's gaps.
//   TMEM (256 columns): S of even blocks [0, 64), of odd ones [64, 128), O [128, 128 + D).
//   per block j of 64 keys:  S_j = Q K_j^T, issued one block ahead of the softmax; P = exp2(c S - m) over S_j in TMEM, 16 bits;
//                            O += P V_j with P from TMEM and V as it lies in its pages (MN-major)
//   Q comes by one box of (64 dimensions, heads of the KV head, tokens) for each half of a row; keys and values by one box for each page (or 64 rows of one).
// At its end a CTA turns O through shared memory and writes whole lines.
//
// Bound: the softmax warps' chain for a block (TMEM load, maximum, exponentials and conversions, TMEM store) beside the tensor pipe, as in the flash forward
// (flash_tc.cu). 128 tokens x 16384 keys, 32 / 8 heads of 128 (34 GFLOP, 21 us at the 1638 TFLOP/s of a GEMM): 39 us in 9 ranges, 288 CTAs, 0.9 PFLOP/s; the
// exponentials' unit is busy for 47 % of it, the tensor pipe for 46. 64 tokens x 4096 keys: 16 us (mma.sync 33), mostly the first loads and the joining.
#include "common.cuh"
#include "prefix_attn.cuh"
#include "tma_host.h"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kPtRows = 128, kPtThreads = 192;
constexpr uint32_t kPtCols = 256, kPtO = 128;
// How far a row's maximum may run ahead of the number that its weights refer to before O is scaled (an exponent of two). With 32 rows to a warp one of
// them has a new maximum in almost every block: with no slack 128 x 16384 keys, 32 / 8 heads of 128, and up to 512 own ones take 79 us, with 2^8 69. A weight of
// up to 256 is rounded like one of up to 1, relative to itself, and sums are in 32 bits.
constexpr float kPtSlack = 8.f;

template <int D> struct PtSmem {
  static constexpr uint32_t kHalves = D / 64, kStage = 8192 * kHalves;
  static constexpr int NK = D == 64 ? 4 : 3, NV = D == 64 ? 4 : 2;      // two CTAs fit an SM; K's stage is free a whole softmax before V's
  static constexpr uint32_t kQ = 0, kK = 16384 * kHalves, kV = kK + NK * kStage, kBar = kV + NV * kStage, kBytes = kBar + 256;
  static_assert(kQ + kPtRows * D * 4 <= kV, "O is turned where Q and the keys were");
};

// tcgen05 from converged code of a whole warp, one lane of which issues it
__device__ __forceinline__ void pt_mma_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pt_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float pt_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pt_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool BF16> __device__ __forceinline__ uint32_t pt_pack(float a, float b) {
  if (BF16) return pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPtThreads, 2)
prefix_shared_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                        const PrefixParams p, const int tile_tokens) {
  using L = PtSmem<D>;
  constexpr int kHalves = L::kHalves, NK = L::NK, NV = L::NV;
  extern __shared__ __align__(1024) uint8_t smem_pt[];
  const uint32_t sbase = smem_u32(smem_pt);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  const PrefixGroup grp = prefix_group(p, blockIdx.z);
  const int rep = p.H / p.G, tiles = gridDim.y / p.G, kvh = blockIdx.y / tiles, tok0 = blockIdx.y % tiles * tile_tokens;
  const int nrows = min(tile_tokens, grp.tokens - tok0) * rep;
  const int per = range_blocks(p, grp.shared), k_lo = blockIdx.x * per * kPxKeys, k_hi = min(grp.shared, k_lo + per * kPxKeys);
  if (nrows <= 0 || k_lo >= k_hi) return;
  const int nit = ceil_div(k_hi - k_lo, kPxKeys);

  const uint32_t bar = sbase + L::kBar;
  const uint32_t q_full = bar, o_done = bar + 8, s_full0 = bar + 16, p_full0 = bar + 32, tmem_slot = bar + 48;
  auto k_full = [&](int j) { return bar + 64 + 8u * ((uint32_t)j % NK); };
  auto k_empty = [&](int j) { return bar + 64 + 8u * (NK + (uint32_t)j % NK); };
  auto v_full = [&](int j) { return bar + 64 + 8u * (2 * NK + (uint32_t)j % NV); };
  auto v_empty = [&](int j) { return bar + 64 + 8u * (2 * NK + NV + (uint32_t)j % NV); };
  auto k_phase = [&](int j) { return ((uint32_t)j / NK) & 1u; };
  auto v_phase = [&](int j) { return ((uint32_t)j / NV) & 1u; };
  auto k_at = [&](int j) { return sbase + L::kK + ((uint32_t)j % NK) * L::kStage; };
  auto v_at = [&](int j) { return sbase + L::kV + ((uint32_t)j % NV) * L::kStage; };
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tq); tma_prefetch_desc(&tk); tma_prefetch_desc(&tv);
    mbar_init(q_full, 1); mbar_init(o_done, 1);
    for (int s = 0; s < 2; ++s) { mbar_init(s_full0 + 8 * s, 1); mbar_init(p_full0 + 8 * s, 4); }
    for (int s = 0; s < NK; ++s) { mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); }
    for (int s = 0; s < NV; ++s) { mbar_init(v_full(s), 1); mbar_init(v_empty(s), 1); }
    fence_mbar_init();
  }
  if (warp == 5) { tmem_alloc(tmem_slot, kPtCols); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem_base;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot));

  if (warp == 4) {
    if (lane == 0) {
      // rows of the box that lie behind the batch come as zeros; those of the tile that the box does not have are nobody's
      mbar_arrive_expect_tx(q_full, (uint32_t)(tile_tokens * rep) * 128u * kHalves);
      for (int half = 0; half < kHalves; ++half) tma_load_3d(sbase + L::kQ + half * 16384, &tq, q_full, half * 64, kvh * rep, grp.first + tok0);
    }
    __syncwarp();
    // a block is `pieces` boxes of `psize` rows; lane i looks up and fetches piece i, its page number one block ahead. A piece behind the range, or on a
    // page outside the pools, is asked for behind the pools' last row: zeros
    const int slot = p.slot[grp.first];
    const int* trow = (unsigned)slot < (unsigned)p.table_rows ? p.table + slot * p.table_stride : nullptr;
    const int psl = min(p.bs_log2, 6), psize = 1 << psl, pieces = kPxKeys >> psl, pool_rows = (p.n_pages * p.G) << p.bs_log2;
    auto row_of = [&](int it) {
      const int k = k_lo + it * kPxKeys + lane * psize;
      const int page = it < nit && lane < pieces && k < k_hi && trow ? page_of(p, trow, k) : -1;
      return page >= 0 ? ((page * p.G + kvh) << p.bs_log2) + (k & ((1 << p.bs_log2) - 1)) : pool_rows;
    };
    // block it's keys, then the values of the block before it: a K stage is free long before a V stage
    int row = row_of(0), row_v = 0;
    for (int it = 0; it <= nit; ++it) {
      if (it < nit) {
        if (lane == 0) {
          mbar_wait(k_empty(it), k_phase(it) ^ 1u);
          mbar_arrive_expect_tx(k_full(it), L::kStage);
        }
        __syncwarp();
        if (lane < pieces)
          for (int half = 0; half < kHalves; ++half) tma_load_2d(k_at(it) + half * 8192 + lane * psize * 128, &tk, k_full(it), half * 64, row);
      }
      const int next = row_of(it + 1);
      if (it > 0) {
        const int j = it - 1;
        if (lane == 0) {
          mbar_wait(v_empty(j), v_phase(j) ^ 1u);
          mbar_arrive_expect_tx(v_full(j), L::kStage);
        }
        __syncwarp();
        if (lane < pieces)
          for (int half = 0; half < kHalves; ++half) tma_load_2d(v_at(j) + half * 8192 + lane * psize * 128, &tv, v_full(j), half * 64, row_v);
      }
      row_v = row;
      row = next;
    }
    __syncwarp();
  } else if (warp == 5) {
    // descriptors: hi word = SBO 1024 | version 1 | 128B swizzle; lo word = address >> 4 (| LBO << 16 for MN-major)
    constexpr uint32_t kHi = (1024u >> 4) | (1u << 14) | (kSwizzle128B << 29);
    constexpr uint32_t kLoK = (16u >> 4) << 16, kLoMN = (8192u >> 4) << 16;
    auto desc = [](uint32_t lo) { return ((uint64_t)kHi << 32) | (uint64_t)lo; };
    const uint32_t idesc_qk = make_idesc_f16(kPtRows, kPxKeys, BF16, false, false);
    const uint32_t idesc_pv = make_idesc_f16(kPtRows, D, BF16, false, true);
    const uint32_t tS = tmem_base, tO = tmem_base + kPtO;
    const uint32_t qlo = ((sbase + L::kQ) >> 4) | kLoK;
    auto issue_qk = [&](int j) {
      const int s = j & 1;
      const uint32_t klo = (k_at(j) >> 4) | kLoK;
#pragma unroll
      for (int half = 0; half < kHalves; ++half)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          pt_mma_ss(tS + s * kPxKeys, desc(qlo + half * (16384u >> 4) + ks * 2u), desc(klo + half * (8192u >> 4) + ks * 2u), idesc_qk, (half | ks) ? 1u : 0u);
      pt_commit(s_full0 + 8 * s);
      pt_commit(k_empty(j));
    };
    mbar_wait_spin(q_full, 0);
    mbar_wait_spin(k_full(0), 0);
    __syncwarp();                                     // each lane has looked for itself
    tc_fence_after();
    issue_qk(0);
    for (int j = 0; j < nit; ++j) {
      const int s = j & 1;
      if (j + 1 < nit) {
        mbar_wait_spin(k_full(j + 1), k_phase(j + 1));
        __syncwarp();
        // buffer (j + 1) & 1 held P of block j - 1, whose product was issued before this one: the pipe runs in order
        tc_fence_after();
        issue_qk(j + 1);
      }
      mbar_wait_spin(v_full(j), v_phase(j));
      mbar_wait_spin(p_full0 + 8 * s, ((uint32_t)j >> 1) & 1u);     // P is written, and O scaled where a row needed it
      __syncwarp();
      tc_fence_after();
      const uint32_t vlo = (v_at(j) >> 4) | kLoMN;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        pt_mma_ts(tO, tS + s * kPxKeys + ks * 8, desc(vlo + ks * (2048u >> 4)), idesc_pv, (j | ks) ? 1u : 0u);
      pt_commit(o_done);
      pt_commit(v_empty(j));
    }
  } else {
    // ================= softmax: thread = row =================
    const int r = warp * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(warp * 32) << 16;
    const uint32_t tS = tmem_base + lane_addr, tO = tmem_base + lane_addr + kPtO;
    const float sl = p.scale_log2;
    float m = -INFINITY, l = 0.f;
    uint32_t v[64];
    for (int j = 0; j < nit; ++j) {
      const int sb = j & 1, left = k_hi - k_lo - j * kPxKeys;
      mbar_wait_warp(s_full0 + 8 * sb, ((uint32_t)j >> 1) & 1u);
      tc_fence_after();
      tmem_ld_32x32(tS + sb * kPxKeys, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
      tmem_ld_32x32(tS + sb * kPxKeys + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
      tmem_ld_wait();
      if (left < kPxKeys) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (i >= left) v[i] = 0xff800000u;          // -inf
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 64; i += 8)
#pragma unroll
        for (int c = 0; c < 4; ++c) m4[c] = pt_max3(m4[c], __uint_as_float(v[i + 2 * c]), __uint_as_float(v[i + 2 * c + 1]));
      const float mn = fmaxf(m, fmaxf(pt_max3(m4[0], m4[1], m4[2]), m4[3]) * sl);      // the scale is above zero (checked by the launcher)
      const bool raise = mn > m + kPtSlack;
      const float alpha = raise ? pt_ex2(m - mn) : 1.f;
      if (raise) m = mn;
      const float e = m == -INFINITY ? 0.f : m;
      const bool any_raise = j > 0 && __any_sync(0xffffffffu, raise);
      // The product of block j - 1 is complete: O may be read. A parity tells phase c from c + 1, not from c + 2; S(j) proves that the product
      // of j - 2 is complete, so a warp that skipped this for a while is at most one phase behind here, and the last block always waits.
      if (j > 0 && (any_raise || j == nit - 1)) {
        mbar_wait_warp(o_done, (uint32_t)(j - 1) & 1u);
        tc_fence_after();
      }
      if (any_raise) {
        uint32_t o[32];
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          tmem_ld_32x32(tO + c * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32(tO + c * 32, o);
        }
      }
      float2 rs = make_float2(0.f, 0.f);
      const float2 nm = make_float2(-e, -e), sl2 = make_float2(sl, sl);
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float2 x = __ffma2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sl2, nm);
        x.x = pt_ex2(x.x); x.y = pt_ex2(x.y);
        rs = __fadd2_rn(rs, x);
        w[i] = pt_pack<BF16>(x.x, x.y);
      }
      tmem_st_32x32(tS + sb * kPxKeys, w);
      if (left < kPxKeys) {                           // values behind the shared part, in its last page, become zeros: a weight of zero does not undo a NaN
        mbar_wait_warp(v_full(j), v_phase(j));
        for (int i = threadIdx.x; i < (kPxKeys - left) * 8 * kHalves; i += 128) {
          const int row = left + i / (8 * kHalves), c = i % (8 * kHalves);
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v_at(j) + (c >> 3) * 8192 + row * 128 + (c & 7) * 16), "r"(0) : "memory");
        }
        fence_proxy_async_smem();                     // generic-proxy stores -> visible to tcgen05.mma
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full0 + 8 * sb);
      l = fmaf(l, alpha, rs.x + rs.y);
    }
    // ---- O to the range's place: through shared memory (Q and the keys have been read), 16-byte pieces turned by the row, whole rows out ----
    mbar_wait_warp(o_done, (uint32_t)(nit - 1) & 1u);
    tc_fence_after();
    constexpr int CH = D / 4;                         // 16-byte pieces of a row of O
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      tmem_ld_32x32(tO + c * 32, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 8; ++i)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(sbase + (uint32_t)r * (D * 4u) + (((uint32_t)(c * 8 + i) ^ ((uint32_t)r & 7u)) << 4)),
                     "r"(o[4 * i]), "r"(o[4 * i + 1]), "r"(o[4 * i + 2]), "r"(o[4 * i + 3]) : "memory");
    }
    // where this row's part goes; -1: nowhere (no row, or one of another group)
    const int token = grp.first + tok0 + r / rep;
    const long long at = r < nrows && p.of[token] == (int)blockIdx.z
                             ? ((long long)token * p.H + kvh * rep + r % rep) * p.nsplit + blockIdx.x : -1;
    if (at >= 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, l);
    __syncwarp();
#pragma unroll 4
    for (int i = 0; i < CH; ++i) {                    // a row of 128: a warp's 32 pieces; of 64: two rows at a time
      const int rr = i * (32 / CH) + lane / CH, piece = lane % CH, row = warp * 32 + rr;
      const long long to = __shfl_sync(0xffffffffu, at, rr);
      uint4 x;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                   : "r"(sbase + (uint32_t)row * (D * 4u) + (((uint32_t)piece ^ ((uint32_t)row & 7u)) << 4)));
      if (to >= 0) *reinterpret_cast<uint4*>(p.part_o + to * D + piece * 4) = x;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kPtCols);
  }
}

int prefix_tc_tokens(int H, int G, int D) {
  const int rep = H / G;
  return (D == 64 || D == 128) && rep <= kPtRows ? kPtRows / rep : 0;
}

template <int D, bool BF16>
static int launch_shared_tc(const PrefixParams& p, cudaStream_t st) {
  const int rep = p.H / p.G, tokens = kPtRows / rep;
  const long long pool_rows = ((long long)p.n_pages * p.G) << p.bs_log2;
  CUtensorMap tq, tk, tv;
  {
    uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.H, (uint64_t)p.T}, str[2] = {(uint64_t)D * 2, (uint64_t)p.q_stride * 2};
    uint32_t box[3] = {64, (uint32_t)rep, (uint32_t)tokens};
    if (int rc = make_tensor_map(&tq, p.q, 2, 3, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  }
  uint64_t dims[2] = {(uint64_t)D, (uint64_t)pool_rows}, str[1] = {(uint64_t)D * 2};
  uint32_t box[2] = {64, (uint32_t)(p.bs_log2 < 6 ? 1 << p.bs_log2 : 64)};
  if (int rc = make_tensor_map(&tk, p.ck, 2, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  if (int rc = make_tensor_map(&tv, p.cv, 2, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  auto kern = prefix_shared_tc_kernel<D, BF16>;
  // per call: the attribute belongs to the current device, and a process may use several
  B200_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PtSmem<D>::kBytes));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute room = most_shared_memory();
  cfg.gridDim = dim3(p.nsplit, p.G * ceil_div(p.longest, tokens), p.n_groups); cfg.blockDim = dim3(kPtThreads); cfg.dynamicSmemBytes = PtSmem<D>::kBytes; cfg.stream = st;
  cfg.attrs = &room;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, tq, tk, tv, p, tokens);
}

int prefix_shared_tc(const PrefixParams& p, int dtype, cudaStream_t st) {
  const bool bf = dtype == B200_DT_BF16;
  return p.D == 64 ? (bf ? launch_shared_tc<64, true>(p, st) : launch_shared_tc<64, false>(p, st))
                   : (bf ? launch_shared_tc<128, true>(p, st) : launch_shared_tc<128, false>(p, st));
}

}  // namespace b200
