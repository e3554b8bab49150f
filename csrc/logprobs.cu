// Log probabilities of given tokens, with the entropy of their rows, their rank and the most probable alternatives, and the gradient of the
// first two. With y = l / T, p = softmax(y), t the row's token:
//     lp = y_t - log sum e^y,   H = -sum p log p,   rank = 1 + #{ l_j > l_t },   the k largest l, lowest ids first among equals
//     dl_j = 1/T ( g (d_jt - p_j) - h p_j (log p_j + H) )      for gradients g of lp and h of H
// One pass over a row keeps, of what it has seen, the largest logit m, and with x = (l - m) log2(e) / T the sums s = sum 2^x and u = sum 2^x x, so that
//     lp = (l_t - m) / T - log s,   H = log s - log(2) u / s.
// Differences of logits come first, before any product: a row of the type's lowest values is uniform, and log probabilities near zero keep their bits. A row
// without a token of the vocabulary is passed over: zeros, no alternatives, no gradient. A row of minus infinities alone, or with a NaN or
// plus infinity, gives NaN as log_softmax does.
//
//   lp_rows        logits [B, V] -> lp, H, rank, alternatives, and (m, 1 / s, log s, H) for the backward pass; a CTA or a cluster a row
//   lp_rows_grad   logits, (m, 1 / s, log s, H), g, h -> dl, in one pass
// and for logits x w^T that are never stored (gemm_tcgen05.cu: sums and gradients in the epilogues of the product):
//   lp_finish      lp, H and what the backward pass needs, from the sums of a row's tiles
//   lp_active, lp_gather, lp_return   rows whose tokens are not passed over, side by side, and their gradients back where they belong
//   lp_scale, lp_cast   a power of two for fp16's gradients of single logits, and back
// Rows of logits are bound by HBM where log probabilities alone are asked for (3000 x 151936 in bf16 139 us, 6.6 TB/s; gradients of 4096 rows 385, 6.5 TB/s): 5.1 instructions
// and an exponential a 16-bit logit are just behind it (issue slots 43 % busy, exponential unit 76 %). With entropies, ranks and alternatives it is 9.2 instructions
// and a row's last steps that 16-bit rows wait for (187 us), while rows of 32 bits stay near HBM (1000 x 151936 93 us, with all of them 106).
#include "logprob_math.cuh"
#include "../include/b200_ops.h"
#include <type_traits>

namespace b200 {

constexpr int kLpThreads = 256, kLpMaxTop = 32, kLpMaxCluster = 8;

// What a CTA of NT threads knows of its slice of a row, where the others of its cluster read it.
template <int NT> struct LpSums {
  float red[3][NT / 32];
  int redi[NT / 32];
  float4 sums;                                   // m, s, u, logits above the token's
};
template <int NT> struct LpShared : LpSums<NT> {
  static constexpr int kList = NT == 64 ? 512 : 1280, kSegments = NT == 64 ? 1 : 2048;
  unsigned long long best[kLpMaxTop];            // the slice's alternatives in order
  unsigned long long list[kList];
  float segment[kSegments];                      // the largest of each 128 vectors, or 32
  uint32_t group[64];
  int chosen[kLpMaxTop];
  unsigned long long bound;
  int n, more;
};

template <typename T> struct LpVec { static constexpr int N = 16 / sizeof(T); };

// Two values of a vector's word (one of 32 bits).
template <typename T> __device__ __forceinline__ float2 lp_word(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// The largest of G vectors' values (NaN aside).
template <typename T, int G>
__device__ __forceinline__ float lp_largest(const uint4 (&raw)[G]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = fmaxf(m, __uint_as_float((&raw[g].x)[j]));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m = *reinterpret_cast<const T2*>(&raw[0].x);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = __hmax2(m, *reinterpret_cast<const T2*>(&(&raw[g].x)[j]));
    return fmaxf(to_f32<T>(m.x), to_f32<T>(m.y));
  }
}
// lp_join of G vectors, of which m is the largest value: unpacked two at a time as they are used, so that a thread holds the vectors and little else.
template <typename T, bool ENT, int G>
__device__ __forceinline__ void lp_join_vectors(LpSum& a, const uint4 (&raw)[G], float m, float c) {
  if (m > a.m) {
    const float x = (a.m - m) * c, f = lp_exp2(x);
    if constexpr (ENT) a.u = f * (a.u + a.s * lp_factor(x));
    a.s *= f;
    a.m = m;
  }
  const float base = a.m == -INFINITY ? 0.f : a.m;
  const unsigned long long nb = lp_pair(-base, -base), cc = lp_pair(c, c);
  unsigned long long s = 0, u = 0;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int j = 0; j < (sizeof(T) == 4 ? 2 : 4); ++j) {
      const float2 v = sizeof(T) == 4 ? make_float2(__uint_as_float((&raw[g].x)[2 * j]), __uint_as_float((&raw[g].x)[2 * j + 1])) : lp_word<T>((&raw[g].x)[j & 3]);
      const unsigned long long x = lp_mul2(lp_add2(lp_pair(v.x, v.y), nb), cc);
      const float2 xs = lp_split(x);
      const unsigned long long e = lp_pair(lp_exp2(xs.x), lp_exp2(xs.y));
      s = lp_add2(s, e);
      if constexpr (ENT) u = lp_fma2(e, lp_pair(lp_factor(xs.x), lp_factor(xs.y)), u);
    }
  const float2 s2 = lp_split(s);
  a.s += s2.x + s2.y;
  if constexpr (ENT) {
    const float2 u2 = lp_split(u);
    a.u += u2.x + u2.y;
  }
}

// How many of a group's values are above lt: 16-bit types two to an instruction, whose counts of ones a group's sixteen pairs do not exhaust.
template <typename T, int G>
__device__ __forceinline__ int lp_above(const uint4 (&raw)[G], float lt) {
  int n = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) n += __uint_as_float((&raw[g].x)[j]) > lt;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 one, sum;
    one.x = one.y = from_f32<T>(lt);
    sum.x = sum.y = from_f32<T>(0.f);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = __hadd2(sum, __hgt2(*reinterpret_cast<const T2*>(&(&raw[g].x)[j]), one));
    n = int(to_f32<T>(sum.x) + to_f32<T>(sum.y));
  }
  return n;
}

// How NT threads walk over p[0 .. n): single values up to the first multiple of 16 bytes, vectors by fours, single values behind the last. A warp's four are 128
// vectors in a row (in CTAs of 64 threads: thread, thread + NT ..).
struct LpWalk { int head, nvec, tail; };
template <typename T> __device__ __forceinline__ LpWalk lp_walk(const T* p, int n) {
  const int head = min(n, int((16 - ((uintptr_t)p & 15)) & 15) / int(sizeof(T))), nvec = (n - head) / LpVec<T>::N;
  return {head, nvec, head + nvec * LpVec<T>::N};
}

// Order of logits as whole numbers: NaN above all, -0 as 0; ties by the lower id.
__device__ __forceinline__ uint32_t lp_order(float v) {
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
  return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t id) { return (unsigned long long)lp_order(v) << 32 | uint32_t(~id); }
__device__ __forceinline__ uint32_t lp_id(unsigned long long key) { return ~uint32_t(key); }
__device__ __forceinline__ float lp_of_key(unsigned long long key) {
  const uint32_t o = uint32_t(key >> 32);
  return o == 0xffffffffu ? __uint_as_float(0x7fffffffu) : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ unsigned long long lp_remote(const unsigned long long* p, uint32_t rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lp_cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}

// The largest of a warp's values.
__device__ __forceinline__ float lp_warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
// The parts that the first LANES lanes hold (the others: nothing, {-inf, 0, 0}) as one: to the largest of all at once, then plain sums.
template <bool ENT, int LANES>
__device__ __forceinline__ LpSum lp_warp_sum(LpSum a, float c) {
  const float m = lp_warp_max(a.m), x = (a.m - (m == -INFINITY ? 0.f : m)) * c, f = lp_exp2(x);
  if constexpr (ENT) a.u = f * (a.u + a.s * lp_factor(x));
  a.s *= f;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if constexpr (ENT) a.u += __shfl_xor_sync(0xffffffffu, a.u, o);
  }
  a.m = m;
  return a;
}
// The k-th largest of 64 numbers, by one warp.
__device__ __forceinline__ uint32_t lp_kth(const uint32_t* v, int k) {
  const int lane = threadIdx.x & 31;
  uint32_t a = v[lane], b = v[lane + 32], most = 0;
  if (a < b) { const uint32_t x = a; a = b; b = x; }
  for (int i = 0; i < k; ++i) {
    most = __reduce_max_sync(0xffffffffu, a);
    if (lane == __ffs(__ballot_sync(0xffffffffu, a == most)) - 1) { a = b; b = 0; }
  }
  return most;
}

// out[0 .. k) = the k largest of n distinct keys in order; a key's place is the number of larger ones. All threads of the CTA.
template <int NT>
__device__ __forceinline__ void lp_sort(const unsigned long long* keys, int n, int k, unsigned long long* out) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const unsigned long long key = keys[i];
    int larger = 0;
    for (int j = 0; j < n; ++j) larger += keys[j] > key;
    if (larger < k) out[larger] = key;
  }
  __syncthreads();
}

// The k largest keys of p[0 .. n) (ids from id0 on) into sh.best, one pass a key: for what the shorter way below does not take. (The first pass has no key to stay
// below: that of a NaN at id 0 has all bits set, so no start value is above it.)
template <typename T, int NT>
__device__ __noinline__ void lp_top_by_passes(const T* __restrict__ p, int n, int id0, int k, LpShared<NT>& sh) {
  unsigned long long last = 0;
  for (int i = 0; i < k; ++i) {
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < n; j += NT) {
      const unsigned long long key = lp_key(to_f32<T>(p[j]), id0 + j);
      if ((i == 0 || key < last) && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, best, o);
      best = x > best ? x : best;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.list[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < NT / 32; ++w) best = sh.list[w] > best ? sh.list[w] : best;
    if (threadIdx.x == 0) sh.best[i] = best;
    last = best;
  }
  __syncthreads();
}

// The k largest of p[0 .. n), from what each thread noted on its way: the largest value among its vectors and the group that first had it.
// The k threads with the largest of those values (lowest ids first) have all k of them: a value that is none of these threads' is smaller than
// each of their largest. So only their vectors are looked at again, about k values in all are not below the last of those, and they are ordered.
// For short rows: a CTA of 64 threads.
template <typename T, int NT>
__device__ __forceinline__ void lp_top_of_threads(const T* __restrict__ p, int n, int id0, int k, LpWalk at, float most, int group, LpShared<NT>& sh) {
  constexpr int N = LpVec<T>::N, CAP = LpShared<NT>::kList;
  static_assert(NT == 64, "one thread to each of the 64 groups");
  const uint4* q = reinterpret_cast<const uint4*>(p + at.head);
  // 1. a bound by values alone, so that few threads look up where their largest is: the k-th of the threads'
  const uint32_t own = group < 0 ? 0u : lp_order(most);
  sh.group[threadIdx.x] = own;
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    const uint32_t v = lp_kth(sh.group, k);
    if (threadIdx.x == 0) sh.bound = v;
  }
  __syncthreads();
  // 2. those threads' largest with their ids, and which of them are the k largest
  const uint32_t least = max(uint32_t(sh.bound), 1u);
  unsigned long long mine = 0;
  if (own >= least) {
    // (a group of one vector is a thread's last: there is none behind it)
    uint4 raw[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) raw[x] = __ldg(q + (group + x * NT < at.nvec ? group + x * NT : group));
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const unsigned long long key = lp_key(to_f32<T>(reinterpret_cast<const T*>(&raw[x])[j]), id0 + at.head + (group + x * NT < at.nvec ? group + x * NT : group) * N + j);
        mine = key > mine ? key : mine;
      }
    sh.list[atomicAdd(&sh.n, 1)] = mine;
  }
  __syncthreads();
  const int found = sh.n;
  int larger = NT;
  if (mine) {
    larger = 0;
#pragma unroll 4
    for (int j = 0; j < found; ++j) larger += sh.list[j] > mine;
    if (larger < k) sh.chosen[larger] = threadIdx.x;
  }
  __syncthreads();
  if (threadIdx.x == 0) { sh.n = 0; if (found < k) sh.bound = 0; }
  if (larger == k - 1) sh.bound = mine;
  __syncthreads();
  // 3. the chosen threads' vectors again, dealt to all threads, and the single values at the ends
  const unsigned long long bound = sh.bound;
  const float value = bound ? lp_of_key(bound) : -INFINITY;
  auto offer = [&](float v, int j) {
    if (v >= value) {
      const unsigned long long key = lp_key(v, id0 + j);
      if (key >= bound) {
        const int i = atomicAdd(&sh.n, 1);
        if (i < CAP) sh.list[i] = key;
      }
    }
  };
  const int each = (at.nvec + NT - 1) / NT, all = min(found, k) * each;
  for (int x0 = threadIdx.x; x0 < all; x0 += 4 * NT) {
    uint4 raw[4];
    int i[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int e = x0 + x * NT, b = e / each;
      i[x] = e < all ? sh.chosen[b] + (e - b * each) * NT : at.nvec;
      if (i[x] < at.nvec) raw[x] = __ldg(q + i[x]);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (i[x] < at.nvec) {
#pragma unroll
        for (int j = 0; j < N; ++j) offer(to_f32<T>(reinterpret_cast<const T*>(&raw[x])[j]), at.head + i[x] * N + j);
      }
  }
  if (threadIdx.x < at.head) offer(to_f32<T>(p[threadIdx.x]), threadIdx.x);
  if (threadIdx.x < n - at.tail) offer(to_f32<T>(p[at.tail + threadIdx.x]), at.tail + threadIdx.x);
  __syncthreads();
  const int m = sh.n;
  if (m > CAP || m < min(k, n)) lp_top_by_passes<T, NT>(p, n, id0, k, sh);      // large values close together in few threads, or NaN
  else lp_sort<NT>(sh.list, m, k, sh.best);
}

// The same for long rows, from the largest value of each segment of 2^SEG vectors. The k segments with the largest of those (the first ones among equals) have all k of them:
// whatever stands in another segment comes behind the largest of each of these. They are read again as whole lines (what 20 threads had seen, a sector
// here and there, was a third of a row of 16 bits: 3000 x 151936 with 20 alternatives 239 us, now 168).
template <typename T, int NT, int SEG>
__device__ __forceinline__ void lp_top_of_segments(const T* __restrict__ p, int n, int id0, int k, LpWalk at, LpShared<NT>& sh) {
  constexpr int N = LpVec<T>::N, CAP = LpShared<NT>::kList, EACH = NT / 64;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, segments = (at.nvec + (1 << SEG) - 1) >> SEG;
  const uint4* q = reinterpret_cast<const uint4*>(p + at.head);
  if (segments < k || segments > LpShared<NT>::kSegments) { lp_top_by_passes<T, NT>(p, n, id0, k, sh); return; }
  // 1. a bound, the k-th of 64 groups of segments
  uint32_t own = 0;
  for (int i = threadIdx.x; i < segments; i += NT) own = max(own, lp_order(sh.segment[i]));
#pragma unroll
  for (int o = 1; o < EACH; o *= 2) own = max(own, __shfl_xor_sync(0xffffffffu, own, o));
  if (lane % EACH == 0) sh.group[threadIdx.x / EACH] = own;
  if (threadIdx.x == 0) sh.n = sh.more = 0;
  __syncthreads();
  if (w == 0) {
    const uint32_t v = lp_kth(sh.group, k);
    if (lane == 0) sh.bound = v;
  }
  __syncthreads();
  // 2. the segments not below it, in order: the first k are chosen
  const uint32_t least = uint32_t(sh.bound);
  for (int i = threadIdx.x; i < segments; i += NT) {
    const uint32_t v = lp_order(sh.segment[i]);
    if (v >= least) {
      const int at_list = atomicAdd(&sh.n, 1);
      if (at_list < CAP) sh.list[at_list] = (unsigned long long)v << 32 | uint32_t(~i);
    }
  }
  __syncthreads();
  const int found = sh.n;
  if (found > CAP) { lp_top_by_passes<T, NT>(p, n, id0, k, sh); return; }
  for (int i = threadIdx.x; i < found; i += NT) {
    const unsigned long long key = sh.list[i];
    int larger = 0;
#pragma unroll 4
    for (int j = 0; j < found; ++j) larger += sh.list[j] > key;
    if (larger < k) sh.chosen[larger] = int(~uint32_t(key));
  }
  __syncthreads();
  const float value = sh.segment[sh.chosen[k - 1]];
  // 3. their values that are not below the last one's largest, of those equal to it no more than k a segment, a warp a segment
  auto offer = [&](float v, int j) {
    const int i = atomicAdd(&sh.more, 1);
    if (i < CAP) sh.list[i] = lp_key(v, id0 + j);
  };
  for (int b = w; b < k; b += NT / 32) {
    const int i0 = (sh.chosen[b] << SEG) + lane;
    constexpr int P = 1 << (SEG - 5);
    uint4 raw[P];
#pragma unroll
    for (int g = 0; g < P; ++g) raw[g] = __ldg(q + (i0 + g * 32 < at.nvec ? i0 + g * 32 : 0));
    int seen = 0;                                                        // equal ones in the pieces before
#pragma unroll
    for (int g = 0; g < P; ++g) {
      const int i = i0 + g * 32;
      const uint4 one[1] = {raw[g]};
      const float largest = i < at.nvec ? lp_largest<T, 1>(one) : -INFINITY;
      if (!__any_sync(0xffffffffu, i < at.nvec && largest >= value)) continue;        // most pieces of a segment, which has one alternative or two
      int equal = 0;
      if (i < at.nvec && largest >= value) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float v = to_f32<T>(reinterpret_cast<const T*>(&raw[g])[j]);
          if (v > value) offer(v, at.head + i * N + j);
          equal += v == value;
        }
      }
      if (!__any_sync(0xffffffffu, equal)) continue;
      int before = equal;                                                // equal ones in the lanes up to this one
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
      }
      const int all = __shfl_sync(0xffffffffu, before, 31);
      before += seen - equal;
      seen += all;
      if (equal && before < k) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (to_f32<T>(reinterpret_cast<const T*>(&raw[g])[j]) == value && before++ < k) offer(value, at.head + i * N + j);
      }
    }
  }
  if (threadIdx.x < at.head && to_f32<T>(p[threadIdx.x]) >= value) offer(to_f32<T>(p[threadIdx.x]), threadIdx.x);
  if (threadIdx.x < n - at.tail && to_f32<T>(p[at.tail + threadIdx.x]) >= value) offer(to_f32<T>(p[at.tail + threadIdx.x]), at.tail + threadIdx.x);
  __syncthreads();
  const int m = sh.more;
  if (m > CAP || m < k) lp_top_by_passes<T, NT>(p, n, id0, k, sh);       // more than a thousand large values in a few segments
  else lp_sort<NT>(sh.list, m, k, sh.best);
}

// A row by a cluster of CTAs (of one, where there are rows enough), a slice each.
// NT: 64 threads a CTA for short rows, 256 for long ones; SEG: 0 without alternatives, else 5 or 7, the segments whose largest values are noted (64 threads: theirs).
template <typename T, bool ENT, int NT, int SEG>
__global__ void __launch_bounds__(NT, (sizeof(T) == 4 ? 1024 : 1280) / NT)
lp_rows_kernel(const T* __restrict__ logits, long long rs, int V, int slice, const long long* __restrict__ tokens, float inv_t, int top, float* __restrict__ lp,
               float* __restrict__ ent, long long* __restrict__ rank, long long* __restrict__ top_ids, float* __restrict__ top_lp,
               float4* __restrict__ stats) {
  constexpr bool TOP = SEG != 0;
  __shared__ typename std::conditional<TOP, LpShared<NT>, LpSums<NT>>::type sh;
  const uint32_t parts = lp_cluster_size(), part = cluster_ctarank();
  const long long row = blockIdx.x / parts;
  const long long t = tokens ? tokens[row] : 0;
  if (t < 0 || t >= V) {                                                // all CTAs of the cluster go
    if (part == 0 && threadIdx.x == 0) {
      if (lp) lp[row] = 0.f;
      if (ENT) ent[row] = 0.f;
      if (rank) rank[row] = 0;
      if (stats) stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (part == 0)
      for (int i = threadIdx.x; i < top; i += NT) { top_ids[row * top + i] = -1; top_lp[row * top + i] = 0.f; }
    return;
  }
  const int id0 = part * slice, n = max(0, min(slice, V - id0));
  const T* p = logits + row * rs + id0;
  const float c = inv_t * kLog2e, lt = to_f32<T>(logits[row * rs + t]);
  LpSum a{-INFINITY, 0.f, 0.f};
  int above = 0, group = -1;
  float most = -INFINITY;
  const LpWalk at = lp_walk<T>(p, n);
  auto single = [&](int j) {
    const float v[1] = {to_f32<T>(p[j])};
    lp_join<ENT>(a, v, v[0], c);
    above += v[0] > lt;
  };
  const uint4* q = reinterpret_cast<const uint4*>(p + at.head);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto vectors = [&](auto& raw, int i) {
    constexpr int G = sizeof(raw) / 16;
    float m;
    if constexpr (TOP && NT > 64) {
      auto note = [&](float v, int first) {                                // the largest of the warp's vectors from `first` on
        const float s = lp_warp_max(v);
        const int segment = first >> SEG;
        if (lane == 0 && first < at.nvec && segment < LpShared<NT>::kSegments) sh.segment[segment] = s;
      };
      if constexpr (SEG == 7) {
        m = lp_largest<T, G>(raw);
        note(m, i - lane);
      } else {
        float each[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint4 one[1] = {raw[g]};
          each[g] = lp_largest<T, 1>(one);
          m = g ? fmaxf(m, each[g]) : each[0];
        }
#pragma unroll
        for (int g = 0; g < G; ++g) note(each[g], i - lane + g * 32);
      }
    } else {
      m = lp_largest<T, G>(raw);
    }
    lp_join_vectors<T, ENT, G>(a, raw, m, c);
    if (rank && m > lt) above += lp_above<T, G>(raw, lt);
    if constexpr (TOP && NT == 64)
      if (i < at.nvec && (m > most || group < 0)) { most = m; group = i; }      // (a warp's last lanes may have no vector: what they would note lies behind the row)
  };
  if (threadIdx.x < at.head) single(threadIdx.x);
  constexpr int NEXT = NT == 64 ? NT : 32;                                // from one of a thread's four vectors to the next
  int i = NT == 64 ? threadIdx.x : w * 128 + lane;
  for (; i - lane + 31 + 3 * NEXT < at.nvec; i += 4 * NT) {
    const uint4 raw[4] = {__ldg(q + i), __ldg(q + i + NEXT), __ldg(q + i + 2 * NEXT), __ldg(q + i + 3 * NEXT)};
    vectors(raw, i);
  }
  // a warp's last vectors, all of them under way at once: what lies behind the row's end counts as minus infinities
  constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  if (i - lane + NEXT < at.nvec) {
    uint4 raw[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) raw[g] = i + g * NEXT < at.nvec ? __ldg(q + i + g * NEXT) : make_uint4(none, none, none, none);
    vectors(raw, i);
  } else if (i - lane < at.nvec) {
    const uint4 raw[1] = {i < at.nvec ? __ldg(q + i) : make_uint4(none, none, none, none)};
    vectors(raw, i);
  }
  if (threadIdx.x < n - at.tail) single(at.tail + threadIdx.x);
  // the CTA's threads: a warp each, then the first warp for all of them (no other needs what comes out)
  a = lp_warp_sum<ENT, 32>(a, c);
  above = __reduce_add_sync(0xffffffffu, above);
  if (lane == 0) { sh.red[0][w] = a.m; sh.red[1][w] = a.s; sh.red[2][w] = a.u; sh.redi[w] = above; }
  const bool no_number = __syncthreads_or(a.s != a.s);                    // a NaN or plus infinity, which the maxima on the way do not count
  if (w == 0) {
    constexpr int W = NT / 32;
    a = lane < W ? LpSum{sh.red[0][lane], sh.red[1][lane], sh.red[2][lane]} : LpSum{-INFINITY, 0.f, 0.f};
    a = lp_warp_sum<ENT, W>(a, c);
    a = {a.m, __shfl_sync(0xffffffffu, a.s, 0), __shfl_sync(0xffffffffu, a.u, 0)};
    above = __reduce_add_sync(0xffffffffu, lane < W ? sh.redi[lane] : 0);
  }
  if constexpr (TOP) {
    const int k = min(top, n);
    if (k > 0) {
      if (no_number) lp_top_by_passes<T, NT>(p, n, id0, k, sh);
      else if constexpr (NT == 64) lp_top_of_threads<T, NT>(p, n, id0, k, at, most, group, sh);
      else lp_top_of_segments<T, NT, SEG>(p, n, id0, k, at, sh);
    }
  }
  // the cluster's CTAs
  if (parts > 1) {
    if (threadIdx.x == 0) sh.sums = make_float4(a.m, a.s, a.u, __int_as_float(above));
    __syncthreads();
    cluster_sync_all();
    if (part == 0) {
      LpSum b{-INFINITY, 0.f, 0.f};
      int more = 0;
      if (uint32_t(lane) < parts) {
        const unsigned long long *s0 = reinterpret_cast<const unsigned long long*>(&sh.sums), lo = lp_remote(s0, lane), hi = lp_remote(s0 + 1, lane);
        b = {__uint_as_float(uint32_t(lo)), __uint_as_float(uint32_t(lo >> 32)), __uint_as_float(uint32_t(hi))};
        more = int(uint32_t(hi >> 32));
      }
      b = lp_warp_sum<ENT, kLpMaxCluster>(b, c);
      a = {b.m, __shfl_sync(0xffffffffu, b.s, 0), __shfl_sync(0xffffffffu, b.u, 0)};
      above = __reduce_add_sync(0xffffffffu, more);
      if constexpr (TOP) {
        for (int e = threadIdx.x; e < int(parts) * top; e += NT) {       // a slice has top alternatives, a short last one fewer: keys of zero, below all
          const int x = e / top, j = e - x * top;
          sh.list[e] = j < min(top, max(0, min(slice, V - x * slice))) ? lp_remote(sh.best + j, x) : 0;
        }
        __syncthreads();
        lp_sort<NT>(sh.list, parts * top, top, sh.best);
      }
    }
  }
  if (part == 0) {
    const float ls = logf(a.s), H = ENT ? ls - kLn2 * a.u / a.s : 0.f;
    if (threadIdx.x == 0) {
      if (lp) lp[row] = (lt - a.m) * inv_t - ls;
      if (ENT) ent[row] = H;
      if (rank) rank[row] = 1 + above;
      if (stats) stats[row] = make_float4(a.m, 1.f / a.s, ls, H);
    }
    if constexpr (TOP) {
      if (int(threadIdx.x) < top) {
        const unsigned long long key = sh.best[threadIdx.x];
        top_ids[row * top + threadIdx.x] = lp_id(key);
        top_lp[row * top + threadIdx.x] = (lp_of_key(key) - a.m) * inv_t - ls;
      }
    }
  }
  if (parts > 1) {                                                       // nobody leaves while its memory is read
    __syncthreads();
    cluster_sync_all();
  }
}

// A thread has kGradSteps times 32 bytes of a row: 4096 x 151936 of 16 bits with entropies 385 us (one 438, two 410, eight 382; by CTAs that go over a whole row,
// 16 bytes a load, 411), 1000 x 151936 of 32 bits 190 (187, 189, 192; 213).
constexpr int kGradSteps = 4;
template <typename T, bool HASH>
__global__ void __launch_bounds__(kLpThreads)
lp_rows_grad_kernel(const T* __restrict__ logits, long long rs, int V, const long long* __restrict__ tokens, float inv_t, const float4* __restrict__ stats,
                    const float* __restrict__ g, const float* __restrict__ h, T* __restrict__ out, long long os) {
  constexpr int N = 32 / sizeof(T);
  const long long row = blockIdx.x;
  const T* p = logits + row * rs;
  T* o = out + row * os;
  const int head = min(V, int((32 - ((uintptr_t)p & 31)) & 31) / int(sizeof(T))), nvec = (V - head) / N;
  const bool same = (((uintptr_t)p ^ (uintptr_t)o) & 31) == 0;          // both have their multiples of 32 bytes at the same elements
  const int i0 = blockIdx.y * (kGradSteps * kLpThreads) + threadIdx.x;
  const long long t = tokens ? tokens[row] : -1;
  const bool skip = tokens && (t < 0 || t >= V);
  const float c = inv_t * kLog2e;
  const LpGrad r = lp_grad_of(stats[row], g ? g[row] : 0.f, HASH && h ? h[row] : 0.f, inv_t, t, 1.f);
  auto single = [&](int j) { o[j] = from_f32<T>(skip ? 0.f : lp_grad_at(to_f32<T>(p[j]), r, c) + (j == r.t ? r.g : 0.f)); };
  const unsigned long long nm = lp_pair(-r.m, -r.m), cc = lp_pair(c, c), A = lp_pair(r.A, r.A), B = lp_pair(r.B, r.B);
#pragma unroll
  for (int x = 0; x < kGradSteps; ++x) {
    const int i = i0 + x * kLpThreads;
    if (i >= nvec) break;
    uint32_t w[8];
    if (skip) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = 0;
    } else {
      asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]),
                   "=r"(w[7]) : "l"(p + head + (long long)i * N));
      const long long at = r.t - head - (long long)i * N;               // the token's place among these
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        const float2 v = sizeof(T) == 4 ? make_float2(__uint_as_float(w[j & 7]), __uint_as_float(w[(j + 1) & 7])) : lp_word<T>(w[(j / 2) & 7]);
        const unsigned long long y = lp_mul2(lp_add2(lp_pair(v.x, v.y), nm), cc);
        const float2 ys = lp_split(y);
        const unsigned long long e = lp_pair(lp_exp2(ys.x), lp_exp2(ys.y));
        float2 d = lp_split(lp_mul2(e, HASH ? lp_fma2(B, lp_pair(lp_factor(ys.x), lp_factor(ys.y)), A) : A));
        if (at == j) d.x += r.g;
        if (at == j + 1) d.y += r.g;
        if constexpr (sizeof(T) == 4) { w[j] = __float_as_uint(d.x); w[j + 1] = __float_as_uint(d.y); }
        else {
          alignas(4) T q[2] = {from_f32<T>(d.x), from_f32<T>(d.y)};
          w[j / 2] = *reinterpret_cast<uint32_t*>(q);
        }
      }
    }
    T* to = o + head + (long long)i * N;
    if (same) {
      asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" :: "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]),
                   "l"(to) : "memory");
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) to[j] = reinterpret_cast<const T*>(w)[j];
    }
  }
  if (blockIdx.y == 0) {                                                 // the row's unaligned ends
    if (threadIdx.x < head) single(threadIdx.x);
    const int tail = head + nvec * N + threadIdx.x;
    if (tail < V) single(tail);
  }
}

// ---- logits that are not stored ----
// part [n][rows] = (m, s, u) of n parts of each row, lt [rows] its token's logit. 8 rows a CTA, 32 threads a row (32 rows a CTA and 8 threads a row took
// 41 us of 2048 x 594 parts, the loads' latency).
__global__ void __launch_bounds__(256)
lp_finish_kernel(const float4* __restrict__ part, int n, long long rows, int V, const int* __restrict__ active, const int* __restrict__ from,
                 const long long* __restrict__ tokens, const float* __restrict__ lt, float inv_t, float* __restrict__ lp, float* __restrict__ ent,
                 float4* __restrict__ stats) {
  __shared__ float4 red[32][8];
  const int r = threadIdx.x & 7, slice = threadIdx.x >> 3;
  const float c = inv_t * kLog2e;
  LpSum a{-INFINITY, 0.f, 0.f};
  const long long live = active ? *active : rows;
  if (blockIdx.x * 8ll >= live) return;
  if (const long long row = blockIdx.x * 8ll + r; row < live) {
    for (int i0 = slice; i0 < n; i0 += 32 * 8) {
      float4 x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = i0 + j * 32 < n ? __ldg(part + (long long)(i0 + j * 32) * rows + row) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) a = lp_both<true>(a, {x[j].x, x[j].y, x[j].z}, c);
    }
  }
  red[slice][r] = make_float4(a.m, a.s, a.u, 0.f);
  __syncthreads();
  const float4 x = red[threadIdx.x & 31][threadIdx.x >> 5];              // a warp to each row
  a = {x.x, x.y, x.z};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = lp_both<true>(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)}, c);
  const long long row = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if ((threadIdx.x & 31) || row >= live) return;
  const long long t = tokens ? tokens[row] : 0, to = from ? from[row] : row;
  const bool skip = t < 0 || t >= V;
  const float ls = logf(a.s), H = ls - kLn2 * a.u / a.s;
  if (lp) lp[to] = skip ? 0.f : (lt[row] - a.m) * inv_t - ls;
  if (ent) ent[to] = skip ? 0.f : H;
  if (stats) stats[to] = make_float4(a.m, 1.f / a.s, ls, H);
}

// A power of two that brings the largest gradient of a logit to 2^13 .. 2^14, so that fp16 holds the small ones too, and its reciprocal.
// |dl| <= (|g| + |h| (log V + 1)) / T.
__global__ void __launch_bounds__(256)
lp_scale_kernel(const float* __restrict__ g, const float* __restrict__ h, const long long* __restrict__ tokens, long long rows, int V, float inv_t,
                float log_v, float* __restrict__ scale) {
  __shared__ float red[32];
  float m = 0.f;
  for (long long i = threadIdx.x; i < rows; i += 256)
    if (!tokens || (tokens[i] >= 0 && tokens[i] < V)) m = fmaxf(m, ((g ? fabsf(g[i]) : 0.f) + (h ? fabsf(h[i]) : 0.f) * (log_v + 1.f)) * inv_t);
  m = block_max(m, red);
  if (threadIdx.x) return;
  const int e = m > 0.f && m < INFINITY ? min(max(14 - (ilogbf(m) + 1), -100), 100) : 0;
  scale[0] = ldexpf(1.f, e);
  scale[1] = ldexpf(1.f, -e);
}

// The rows whose tokens are not passed over, in order: from[i] is the i-th of them, place[t] where row t went (-1: passed over), mine[i] its token, *active how
// many (at least one: of tokens that are all passed over the first one stands for itself, as a token of -1). Rows that are passed over get their zeros here. One CTA.
__global__ void __launch_bounds__(1024)
lp_active_kernel(const long long* __restrict__ tokens, int rows, int V, int* __restrict__ from, int* __restrict__ place, long long* __restrict__ mine,
                 int* __restrict__ active, float* __restrict__ lp, float* __restrict__ ent) {
  __shared__ int warps[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int base = 0;
  for (int r0 = 0; r0 < rows; r0 += 4096) {
    long long t[4];
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + threadIdx.x * 4 + j;
      t[j] = r < rows ? tokens[r] : -1;
      n += t[j] >= 0 && t[j] < V;
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) warps[w] = sum;
    __syncthreads();
    int own = lane < w ? warps[lane] : 0;
    const int before = __reduce_add_sync(0xffffffffu, own), all = __reduce_add_sync(0xffffffffu, warps[lane]);
    int at = base + before + sum - n;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + threadIdx.x * 4 + j;
      if (r >= rows) break;
      if (t[j] >= 0 && t[j] < V) {
        from[at] = r;
        mine[at] = t[j];
        place[r] = at++;
      } else {
        place[r] = -1;
        if (lp) lp[r] = 0.f;
        if (ent) ent[r] = 0.f;
      }
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *active = base > 0 ? base : 1;
    if (base == 0) { from[0] = 0; mine[0] = -1; }
  }
}

// Those rows of x, and zeros up to the next multiple of 256 rows: what stands in one k-block or tile with them. (The row that stands for itself is zeros,
// too.)
__global__ void __launch_bounds__(128)
lp_gather_kernel(const uint4* __restrict__ x, long long rs, int vecs, int rows, const int* __restrict__ from, const long long* __restrict__ mine,
                 const int* __restrict__ active, uint4* __restrict__ out) {
  const int r = blockIdx.x, live = *active;
  if (r >= min(rows, (live + 255) / 256 * 256)) return;
  const bool has = r < live && mine[r] >= 0;
  const uint4* p = x + (has ? from[r] : 0) * rs;
  for (int i = threadIdx.x; i < vecs; i += 128) out[(long long)r * vecs + i] = has ? __ldg(p + i) : make_uint4(0, 0, 0, 0);
}

// y[t] = x[place[t]] * scale[1], zeros for rows that were passed over.
template <typename TI, typename T>
__global__ void __launch_bounds__(256)
lp_return_kernel(const TI* __restrict__ x, T* __restrict__ y, int K, const int* __restrict__ place, const float* __restrict__ scale) {
  const int at = place[blockIdx.x];
  const float f = scale ? scale[1] : 1.f;
  for (int k = threadIdx.x * 4; k < K; k += 1024) {                      // K is a multiple of 8
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = at < 0 ? 0.f : to_f32<TI>(x[(long long)at * K + k + j]) * f;
    alignas(8) T r[4] = {from_f32<T>(v[0]), from_f32<T>(v[1]), from_f32<T>(v[2]), from_f32<T>(v[3])};
    *reinterpret_cast<uint2*>(y + (long long)blockIdx.x * K + k) = *reinterpret_cast<uint2*>(r);
  }
}

// y = x * scale[1] in the type of the gradients.
template <typename T>
__global__ void __launch_bounds__(256) lp_cast_kernel(const float* __restrict__ x, T* __restrict__ y, long long n, const float* __restrict__ scale) {
  const float f = scale ? scale[1] : 1.f;
  const long long i = (blockIdx.x * 256ll + threadIdx.x) * 4;
  if (i + 4 <= n) {
    const float4 v = *reinterpret_cast<const float4*>(x + i);
    alignas(8) T r[4] = {from_f32<T>(v.x * f), from_f32<T>(v.y * f), from_f32<T>(v.z * f), from_f32<T>(v.w * f)};
    *reinterpret_cast<uint2*>(y + i) = *reinterpret_cast<uint2*>(r);
  } else {
    for (long long j = i; j < n; ++j) y[j] = from_f32<T>(x[j] * f);
  }
}

}  // namespace b200
using namespace b200;

#define LP_TYPES(dtype, ...)                                                        \
  if (dtype == B200_DT_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }               \
  else if (dtype == B200_DT_FP16) { using T = __half; __VA_ARGS__; }                 \
  else if (dtype == B200_DT_FP32) { using T = float; __VA_ARGS__; }                  \
  else return B200_ERR_UNSUPPORTED;
#define LP_TYPES16(dtype, ...)                                                      \
  if (dtype == B200_DT_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }               \
  else if (dtype == B200_DT_FP16) { using T = __half; __VA_ARGS__; }                 \
  else return B200_ERR_UNSUPPORTED;

static bool lp_bad(long long rows, int V) { return rows < 0 || rows > 0x7fffffffll || V <= 0; }

// CTAs of a row: where rows are few, a cluster of up to eight, as long as each has 32 KB or more and the SMs are not all busy.
static int lp_parts(long long rows, long long bytes) {
  int parts = 1;
  while (parts < kLpMaxCluster && rows * parts * 2 <= 2 * kNumSMs && bytes / (parts * 2) >= 32768) parts *= 2;
  return parts;
}
constexpr long long kLpSmallRow = 32768;
static int lp_slice(int V, int parts) { return ((V + parts - 1) / parts + 31) / 32 * 32; }

template <typename T, bool ENT, int NT, int SEG>
static cudaError_t lp_rows_launch(int parts, const void* logits, long long rs, long long rows, int V, const long long* tokens, float inv_t, int top, float* lp, float* ent,
                                  long long* rank, long long* top_ids, float* top_lp, void* stats, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(rows * parts)); cfg.blockDim = dim3(NT); cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = parts > 1;
  return cudaLaunchKernelEx(&cfg, lp_rows_kernel<T, ENT, NT, SEG>, (const T*)logits, rs, V, parts > 1 ? lp_slice(V, parts) : V, tokens, inv_t, top, lp, ent, rank, top_ids,
                            top_lp, (float4*)stats);
}

B200_API int b200_token_logprobs(const void* logits, long long rs, long long rows, int V, const long long* tokens, float inv_t, int top, float* lp,
                                 float* ent, long long* rank, long long* top_ids, float* top_lp, void* stats, int dtype, void* stream) {
  if (lp_bad(rows, V) || top < 0 || top > kLpMaxTop || top > V) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  const long long bytes = (long long)V * (dtype == B200_DT_FP32 ? 4 : 2);
  const int parts = lp_parts(rows, bytes);
  // Short rows take CTAs of two warps: what a row costs beside its logits (its token, the meeting of its threads) is then one of many on an SM
  // (20000 x 6400 in bf16: 147 us with 256 threads a row, 95 with 64; 51 by now).
  const bool small = parts == 1 && bytes <= kLpSmallRow;
  // A warp notes the largest value of the 128 vectors that it reads at a time where rows have 256 KB or more and reading a segment again for each alternative is a
  // sixteenth of one at most, else of 32: one maximum of a warp instead of four is what rows of 16 bits with entropies and ranks wait for (3000 x 151936 with
  // five alternatives 191 us and 203, with 20 of them 231 and 215; 3000 x 131080 with four 169 and 178, 2000 x 65600 80 and 74).
  const bool wide = (parts > 1 ? lp_slice(V, parts) : V) * (bytes / V) / 16 >= max(2048 * top, 128 * 128);
#define LP_ROWS(ENT, NT, SEG) B200_CHECK((lp_rows_launch<T, ENT, NT, SEG>(parts, logits, rs, rows, V, tokens, inv_t, top, lp, ent, rank, top_ids, top_lp, stats, st)))
  LP_TYPES(dtype, {
    if (small) { if (ent) LP_ROWS(true, 64, 5); else LP_ROWS(false, 64, 5); }
    else if (!top) { if (ent) LP_ROWS(true, 256, 0); else LP_ROWS(false, 256, 0); }
    else if (wide) { if (ent) LP_ROWS(true, 256, 7); else LP_ROWS(false, 256, 7); }
    else { if (ent) LP_ROWS(true, 256, 5); else LP_ROWS(false, 256, 5); }
  });
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_token_logprobs_grad(const void* logits, long long rs, long long rows, int V, const long long* tokens, float inv_t, const void* stats,
                                      const float* g, const float* h, void* out, long long os, int dtype, void* stream) {
  if (lp_bad(rows, V)) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  const long long vecs = ((long long)V * (dtype == B200_DT_FP32 ? 4 : 2)) / 32;
  const long long steps = (vecs + kGradSteps * kLpThreads - 1) / (kGradSteps * kLpThreads);
  if (steps > 65535) return B200_ERR_TOO_LARGE;
  const dim3 grid((unsigned)rows, (unsigned)(steps > 0 ? steps : 1));
  LP_TYPES(dtype, {
    if (h) lp_rows_grad_kernel<T, true><<<grid, kLpThreads, 0, st>>>((const T*)logits, rs, V, tokens, inv_t, (const float4*)stats, g, h, (T*)out, os);
    else lp_rows_grad_kernel<T, false><<<grid, kLpThreads, 0, st>>>((const T*)logits, rs, V, tokens, inv_t, (const float4*)stats, g, h, (T*)out, os);
  });
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_finish(const void* part, int parts, long long rows, int V, const int* active, const int* from, const long long* tokens, const float* lt,
                                 float inv_t, float* lp, float* ent, void* stats, void* stream) {
  if (lp_bad(rows, V) || parts < 1) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  lp_finish_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, (cudaStream_t)stream>>>((const float4*)part, parts, rows, V, active, from, tokens, lt, inv_t, lp, ent,
                                                                                (float4*)stats);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_active(const long long* tokens, const void* x, long long x_rs, int rows, int K, int V, int* from, int* place, long long* mine, int* active,
                                 float* lp, float* ent, void* out, void* stream) {
  if (rows <= 0 || V <= 0 || K <= 0 || K % 8) return B200_ERR_BAD_SHAPE;
  if (((uintptr_t)x | (uintptr_t)out) & 15 || x_rs % 8) return B200_ERR_BAD_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  if (tokens) lp_active_kernel<<<1, 1024, 0, st>>>(tokens, rows, V, from, place, mine, active, lp, ent);      // null: the maps are there already
  lp_gather_kernel<<<rows, 128, 0, st>>>((const uint4*)x, x_rs / 8, K / 8, rows, from, mine, active, (uint4*)out);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_return(const void* x, int x_dtype, void* y, int rows, int K, const int* place, const float* scale, int dtype, void* stream) {
  if (rows <= 0 || K <= 0 || K % 8) return B200_ERR_BAD_SHAPE;
  if (((uintptr_t)x | (uintptr_t)y) & 15) return B200_ERR_BAD_ALIGN;
  if (x_dtype != dtype && x_dtype != B200_DT_FP32) return B200_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  LP_TYPES16(dtype, {
    if (x_dtype == B200_DT_FP32) lp_return_kernel<float, T><<<rows, 256, 0, st>>>((const float*)x, (T*)y, K, place, scale);
    else lp_return_kernel<T, T><<<rows, 256, 0, st>>>((const T*)x, (T*)y, K, place, scale);
  });
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_scale(const float* g, const float* h, const long long* tokens, long long rows, float inv_t, int V, float* scale, void* stream) {
  if (lp_bad(rows, V)) return B200_ERR_BAD_SHAPE;
  lp_scale_kernel<<<1, 256, 0, (cudaStream_t)stream>>>(g, h, tokens, rows, V, inv_t, logf((float)V), scale);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_cast(const float* x, void* y, long long n, const float* scale, int dtype, void* stream) {
  if (n < 0) return B200_ERR_BAD_SHAPE;
  if ((uintptr_t)x % 16 || (uintptr_t)y % 8) return B200_ERR_BAD_ALIGN;
  if (n == 0) return 0;
  LP_TYPES16(dtype, lp_cast_kernel<T><<<(unsigned)((n + 1023) / 1024), 256, 0, (cudaStream_t)stream>>>(x, (T*)y, n, scale));
  B200_LAUNCH_CHECK();
  return 0;
}
