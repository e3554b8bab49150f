// An embedding lookup y[t] = s W[id_t] (+ P[t mod period]) and its gradient by sorted tokens:
//     dW[v] = s * sum over t with id_t = v of dy[t]
// dense, a row of zeros where a token does not occur; every sum in 32 bits, in an order that the ids alone decide: by t within a tile of sorted pairs, then the tiles' sums in order (atomics into the
// table would add in the order in which they arrive). Tokens outside 0 .. V - 1 and the padding token have no gradient.
//
//   embed_lookup the rows of W, eight values of 16 bits or four of 32 at a time, two such pieces a thread under way; bound by HBM (with a CTA a token 16384 rows of
//                64 values took 21 us, the CTAs' launches). A token outside the table gives zeros
//   embed_sort   (token, place) pairs by token, places of a token in order: a radix sort by one cluster of eight CTAs, which hold the counts of
//                a digit in shared memory and read each other's totals there. T ids make 8 T bytes a pass: the sort is bound by its steps'
//                latencies (16384 ids in two passes 19 us, 4096 13), and stands beside the next kernel
//   embed_fill   zeros, the bulk of what is written for a large vocabulary (V D against T D): bound by HBM (151936 x 4096 of 16 bits 164 us, 7.5 TB/s)
//   embed_sum    a CTA takes L sorted pairs and a slice of the columns, reads their rows of dy once, and writes each token's sum. A token whose
//                pairs lie in several CTAs leaves a partial sum in each (16384 x 4096 of 16 bits 26 us)
//   embed_join   adds the partial sums of such a token, in order (8 us)
// Together, captured: 16384 tokens into 151936 x 4096 in bf16 224 us, 4096 into 30522 x 768 in fp32 27; the lookup of 16384 rows of 4096 in bf16 42 us (6.3 TB/s).
// The order has its price where little is written: the lookup and the gradient of 1024 tokens into 6400 x 512 in bf16 take 20 us in a graph (zeros and atomics 10), of 64 tokens into
// 1000 x 64 in fp32 13.6 (3.6), of 4096 into 6400 x 512 in bf16 24 (17): four launches that wait for one another, the sort's steps 7 to 13 us of it by themselves. Outside a graph the two are alike.
#include "common.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kSortCtas = 8, kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortBins = 1024, kSortBits = 10, kSortHeld = 4;
constexpr int kSortSmem = (kSortWarps + 3) * kSortBins * 4;

__device__ __forceinline__ uint32_t es_remote(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)));
  return v;
}

// Exclusive prefix sums of n <= 1024 numbers in shared memory, in place, by the whole CTA.
__device__ __forceinline__ void es_scan(uint32_t* a, int n, uint32_t* warp_total) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  uint32_t own = t < n ? a[t] : 0, sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) warp_total[w] = sum;
  __syncthreads();
  if (w == 0) {
    uint32_t x = warp_total[lane], s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_total[lane] = s - x;
  }
  __syncthreads();
  if (t < n) a[t] = warp_total[w] + sum - own;
  __syncthreads();
}

// ids [T] -> pairs (token, place), ascending by token, then place; ids without a gradient have token V and come last. `a` and `b` hold T
// pairs each; the last of `passes` passes over `bits` bits writes `a`.
__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads)
embed_sort_kernel(const long long* __restrict__ ids, uint2* __restrict__ a, uint2* __restrict__ b, int T, int V, long long pad, int bits,
                  int passes) {
  pdl_launch_dependents();
  extern __shared__ uint32_t sm[];
  uint32_t* count = sm;                                     // [warps][bins]: pairs of the warp with a digit, then the places before them
  uint32_t* total = sm + kSortWarps * kSortBins;            // [bins]: pairs of this CTA with a digit
  uint32_t* start = total + kSortBins;                      // [bins]: where this CTA's pairs with a digit begin
  uint32_t* warp_total = start + kSortBins;
  const uint32_t rank = cluster_ctarank();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, bins = 1 << bits;
  const long long per_warp = ((T + kSortCtas * kSortWarps - 1) / (kSortCtas * kSortWarps) + 31) / 32 * 32ll;
  const long long lo = min((long long)T, (rank * kSortWarps + w) * per_warp), hi = min((long long)T, lo + per_warp);
  uint32_t* mine = count + w * bins;

  const int steps = int((hi - lo + 31) / 32);
  for (int pass = 0; pass < passes; ++pass) {
    const uint2* src = (passes - pass) & 1 ? b : a;         // what this pass reads (the first one reads ids)
    uint2* dst = (passes - pass) & 1 ? a : b;
    const int shift = pass * bits;
    auto pair = [&](long long i) -> uint2 {
      if (pass == 0) {
        const long long id = ids[i];
        return make_uint2(id >= 0 && id < V && id != pad ? uint32_t(id) : uint32_t(V), uint32_t(i));
      }
      return __ldcg(src + i);                               // written by other SMs in the pass before
    };
    uint2 held[kSortHeld];                                  // a warp's first pairs stay where both walks over them find them
#pragma unroll
    for (int x = 0; x < kSortHeld; ++x) held[x] = lo + x * 32 + lane < hi ? pair(lo + x * 32 + lane) : make_uint2(0, 0);
    auto at = [&](int x) -> uint2 {                         // the lane's pair of step x
      uint2 p = make_uint2(0, 0);
#pragma unroll
      for (int y = 0; y < kSortHeld; ++y)
        if (x == y) p = held[y];
      if (x >= kSortHeld && lo + x * 32ll + lane < hi) p = pair(lo + x * 32ll + lane);
      return p;
    };
    for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) count[i] = 0;
    __syncthreads();
    for (int x = 0; x < steps; ++x) {
      const bool has = lo + x * 32ll + lane < hi;
      const uint32_t d = has ? (at(x).x >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (has && lane == __ffs(same) - 1) mine[d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int x = 0; x < kSortWarps; ++x) {
        const uint32_t c = count[x * bins + d];
        count[x * bins + d] = sum;
        sum += c;
      }
      total[d] = sum;
    }
    cluster_sync_all();
    uint32_t before = 0;
    if (threadIdx.x < bins) {
      uint32_t all = 0, c[kSortCtas];
#pragma unroll
      for (uint32_t r = 0; r < kSortCtas; ++r) c[r] = es_remote(total + threadIdx.x, r);
#pragma unroll
      for (uint32_t r = 0; r < kSortCtas; ++r) {
        if (r < rank) before += c[r];
        all += c[r];
      }
      start[threadIdx.x] = all;
    }
    __syncthreads();
    es_scan(start, bins, warp_total);
    if (threadIdx.x < bins) start[threadIdx.x] += before;
    __syncthreads();
    for (int x = 0; x < steps; ++x) {
      const bool has = lo + x * 32ll + lane < hi;
      const uint2 p = at(x);
      const uint32_t d = has ? (p.x >> shift) & (bins - 1) : 0xffffffffu;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (has) dst[start[d] + mine[d] + __popc(same & ((1u << lane) - 1))] = p;
      __syncwarp();
      if (has && lane == __ffs(same) - 1) mine[d] += __popc(same);
      __syncwarp();
    }
    cluster_sync_all();                                     // the pass is written, and nobody reads this CTA's totals any more
  }
}

// n times 32 bytes of zeros, then the last `rest` bytes; one store a thread, since CTAs that go on write at 6.0 to 6.2 TB/s (16 or 32 bytes a store, by TMA the
// same), stores of 32 bytes by as many CTAs as there are at 7.5 (151936 x 4096 of 16 bits: 208 us and 166). Stands beside the sort: its last CTA waits for
// it, so that what follows finds both done.
__global__ void __launch_bounds__(256) embed_fill_kernel(uint8_t* __restrict__ out, long long n, int rest) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) asm volatile("st.global.v8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"l"(out + i * 32), "r"(0) : "memory");
  if (blockIdx.x == gridDim.x - 1) {
    if (threadIdx.x < rest) out[n * 32 + threadIdx.x] = 0;
    pdl_wait();
  }
}

template <typename TO, int N>
__device__ __forceinline__ void es_write(TO* __restrict__ p, const float (&acc)[N], float scale) {
  alignas(16) TO raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i) raw[i] = from_f32<TO>(acc[i] * scale);
  if constexpr (N * sizeof(TO) >= 16) {
#pragma unroll
    for (int i = 0; i < N; i += 16 / sizeof(TO)) *reinterpret_cast<uint4*>(p + i) = *reinterpret_cast<uint4*>(raw + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = raw[i];
  }
}

// Pairs [L tile, L (tile + 1)) of the sorted ones (L a multiple of 32), N columns a thread. `part` [tiles][2][D]: sums of a token that began before the tile, and of
// one that begins in it and goes on behind it. A lane holds one of 32 pairs, so that rows are asked for without waiting for their places.
constexpr int kSumAhead = 8;            // rows under way at a time
template <typename TI, typename TO, int N>
__global__ void __launch_bounds__(128)
embed_sum_kernel(const uint2* __restrict__ pairs, const TI* __restrict__ dy, long long rs, TO* __restrict__ out, float* __restrict__ part, int T,
                 int V, int D, int L, float scale) {
  pdl_launch_dependents();
  pdl_wait();
  const int tile = blockIdx.x, col = (blockIdx.y * blockDim.x + threadIdx.x) * N, lane = threadIdx.x & 31;
  const int lo = tile * L, hi = min(T, lo + L);
  const bool has = col < D;
  uint32_t token = pairs[lo].x;
  if (token >= uint32_t(V)) return;
  const uint32_t before = lo > 0 ? pairs[lo - 1].x : 0xffffffffu, behind = hi < T ? pairs[hi].x : 0xffffffffu;
  bool inside = token != before;        // the token's pairs begin in this tile
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  auto done = [&](bool goes_on) {
    if (!has) return;
    if (inside && !goes_on) { es_write<TO, N>(out + (long long)token * D + col, acc, scale); return; }
    float* p = part + ((long long)tile * 2 + inside) * D + col;
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = acc[i];
  };
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const uint2 mine = i0 + lane < hi ? pairs[i0 + lane] : make_uint2(V, 0);
#pragma unroll
    for (int b = 0; b < 32; b += kSumAhead) {
      alignas(16) TI raw[kSumAhead][N];
      uint32_t tok[kSumAhead];
#pragma unroll
      for (int j = 0; j < kSumAhead; ++j) {
        tok[j] = __shfl_sync(0xffffffffu, mine.x, b + j);
        const uint32_t place = __shfl_sync(0xffffffffu, mine.y, b + j);
        const TI* src = dy + (long long)place * rs + col;
        if (has && tok[j] < uint32_t(V)) {
          if constexpr (N * sizeof(TI) == 16) *reinterpret_cast<uint4*>(raw[j]) = __ldg(reinterpret_cast<const uint4*>(src));
          else
#pragma unroll
            for (int i = 0; i < N; ++i) raw[j][i] = src[i];
        }
      }
#pragma unroll
      for (int j = 0; j < kSumAhead; ++j) {
        if (tok[j] >= uint32_t(V)) break;
        if (tok[j] != token) {
          done(false);
          token = tok[j];
          inside = true;
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += to_f32<TI>(raw[j][i]);
      }
    }
  }
  done(token == behind);
}

template <typename TO, int N>
__global__ void __launch_bounds__(256)
embed_join_kernel(const uint2* __restrict__ pairs, TO* __restrict__ out, const float* __restrict__ part, int T, int V, int D, int L, float scale) {
  pdl_wait();
  const int tile = blockIdx.x, tiles = gridDim.x, lo = tile * L, hi = lo + L;
  if (hi >= T) return;
  const uint32_t token = pairs[hi].x;
  if (token >= uint32_t(V) || pairs[hi - 1].x != token || (pairs[lo].x == token && lo > 0 && pairs[lo - 1].x == token)) return;
  int more = 0;                         // tiles behind this one that begin with the token
  for (int n = blockDim.x; n == blockDim.x;) {
    const long long at = tile + 1ll + more + threadIdx.x;
    n = __syncthreads_count(at < tiles && pairs[at * L].x == token);
    more += n;
  }
  const int col = (blockIdx.y * blockDim.x + threadIdx.x) * N;
  if (col >= D) return;
  float acc[N];
  const float* p = part + ((long long)tile * 2 + 1) * D + col;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = p[i];
  p += D;                               // the next tile's first
#pragma unroll 8
  for (int j = 0; j < more; ++j, p += 2ll * D) {
    if constexpr (N == 4) {
      const float4 v = *reinterpret_cast<const float4*>(p);
      acc[0] += v.x; acc[1] += v.y; acc[2] += v.z; acc[3] += v.w;
    } else {
      acc[0] += p[0];
    }
  }
  TO* o = out + (long long)token * D + col;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = from_f32<TO>(acc[i] * scale);
}

// Quotients of numbers below 2^31 by d: (i + i m / 2^32) / 2^s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1 (a remainder by the period for every piece is what
// rows with positions wait for: 4096 of 4096 in bf16 10.1 us).
struct EsDiv { uint32_t m, s; };
static EsDiv es_div(uint32_t d) {
  uint32_t s = 0;
  while (s < 31 && (1u << s) < d) ++s;
  return {uint32_t(((1ull << s) - d << 32) / d) + 1, s};
}
__device__ __forceinline__ uint32_t es_over(uint32_t i, EsDiv d) { return (i + __umulhi(i, d.m)) >> d.s; }

// Piece i of T tokens' `each` pieces: token i / each. Two pieces a thread, both under way (in graphs 8 rows of 1024 in bf16 1.6 us, with four pieces 1.8, with one 1.6; 4096
// rows 3.2, 3.1 and 3.5; 16384 of 4096 42.5, 43.4 and 53).
template <typename T>
__global__ void __launch_bounds__(256)
embed_lookup_kernel(const long long* __restrict__ ids, const T* __restrict__ table, const T* __restrict__ pos, T* __restrict__ out, unsigned n, unsigned each,
                    long long V, unsigned period, EsDiv by_period, float scale) {
  constexpr int N = 16 / sizeof(T), U = 2;
  unsigned t[U], at[U];
  long long id[U];
  uint4 raw[U], p[U];
#pragma unroll
  for (int x = 0; x < U; ++x) {
    const unsigned i = blockIdx.x * 512u + x * 256u + threadIdx.x;
    t[x] = i / each;
    at[x] = i - t[x] * each;
    id[x] = i < n ? ids[t[x]] : -1;
    if (i >= n) t[x] = 0xffffffffu;
  }
#pragma unroll
  for (int x = 0; x < U; ++x) {
    raw[x] = id[x] >= 0 && id[x] < V ? __ldg(reinterpret_cast<const uint4*>(table) + id[x] * each + at[x]) : make_uint4(0, 0, 0, 0);
    if (pos && t[x] != 0xffffffffu) p[x] = __ldg(reinterpret_cast<const uint4*>(pos) + (long long)(t[x] - es_over(t[x], by_period) * period) * each + at[x]);
  }
#pragma unroll
  for (int x = 0; x < U; ++x) {
    if (t[x] == 0xffffffffu) continue;
    alignas(16) T o[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float v = to_f32<T>(reinterpret_cast<const T*>(&raw[x])[j]) * scale;
      if (pos) v += to_f32<T>(reinterpret_cast<const T*>(&p[x])[j]);
      o[j] = from_f32<T>(v);
    }
    *(reinterpret_cast<uint4*>(out) + (long long)t[x] * each + at[x]) = *reinterpret_cast<uint4*>(o);
  }
}

static int es_tile(long long T) {       // pairs of a CTA: 32, and more from 2^15 tokens on, so that partial sums stay a small part of the work (8 at 4096
  long long L = 32;                     // tokens of 768 columns: sums 11 -> 8 us, joins 5 -> 12)
  while (L * 1024 < T) L *= 2;
  return int(L);
}
static int es_bits(int V) {
  int n = 1;
  while (n < 31 && (1u << n) <= unsigned(V)) ++n;
  return n;
}

}  // namespace b200
using namespace b200;

B200_API int b200_embedding_lookup(const long long* ids, const void* table, const void* pos_table, void* out, long long T, int V, int D, int period, float scale,
                                   int dtype, void* stream) {
  const int N = dtype == B200_DT_FP32 ? 4 : 8;
  if (T < 0 || V <= 0 || D <= 0 || D % N || (pos_table && period <= 0)) return B200_ERR_BAD_SHAPE;
  if (((uintptr_t)table | (uintptr_t)out | (uintptr_t)pos_table) & 15) return B200_ERR_BAD_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned each = unsigned(D / N);
  // pieces are counted in 32 bits: more tokens go in several launches, each with whole periods of positions
  long long most = 0x7fff0000ll / each;
  if (pos_table) most = most / period * period;
  if (most < 1) return B200_ERR_TOO_LARGE;
  const EsDiv by_period = es_div(pos_table ? unsigned(period) : 1);
  for (long long t = 0; t < T; t += most) {
    const unsigned n = unsigned((T - t < most ? T - t : most) * each), grid = (n + 511) / 512;
#define ES_LOOKUP(TT) embed_lookup_kernel<TT><<<grid, 256, 0, st>>>(ids + t, (const TT*)table, (const TT*)pos_table, (TT*)out + t * D, n, each, V, unsigned(period), by_period, scale)
    if (dtype == B200_DT_FP32) ES_LOOKUP(float);
    else if (dtype == B200_DT_BF16) ES_LOOKUP(__nv_bfloat16);
    else if (dtype == B200_DT_FP16) ES_LOOKUP(__half);
    else return B200_ERR_UNSUPPORTED;
  }
  B200_LAUNCH_CHECK();
  return 0;
}

// The same without the table's number of rows: every id that is not below zero is taken for one of them.
B200_API int b200_embedding_fwd(const long long* ids, const void* table, const void* pos_table, void* out, long long T, int D, int period, float scale, int dtype,
                                void* stream) {
  if (T <= 0) return B200_ERR_BAD_SHAPE;
  return b200_embedding_lookup(ids, table, pos_table, out, T, 0x7fffffff, D, period > 0 ? period : 1, scale, dtype, stream);
}

B200_API long long b200_embedding_grad_workspace(long long T, int D) {
  if (T <= 0 || D <= 0) return 16;
  const long long tiles = ceil_div64(T, es_tile(T));
  return 2 * ((T * 8 + 15) / 16 * 16) + tiles * 2 * D * 4;
}

// A launch that may begin while the one before ends: each of these kernels waits for that one before it reads or writes (embed_fill, which has nothing to
// wait for, at its end).
template <typename... K, typename... A>
static cudaError_t es_next(cudaStream_t st, dim3 grid, int threads, void (*kernel)(K...), A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(args)...);
}

template <typename TI, typename TO, int N>
static cudaError_t es_sum(const uint2* a, const void* dy, long long rs, void* out, float* part, int T, int V, int D, int L, float scale, cudaStream_t st) {
  const int lanes = (D + N - 1) / N, threads = lanes >= 128 ? 128 : (lanes + 31) / 32 * 32;
  const dim3 grid((T + L - 1) / L, (lanes + threads - 1) / threads);
  return es_next(st, grid, threads, embed_sum_kernel<TI, TO, N>, a, (const TI*)dy, rs, (TO*)out, part, T, V, D, L, scale);
}

B200_API int b200_embedding_grad(const long long* ids, const void* dy, long long rs, void* out, long long T, int V, int D, float scale,
                                 long long padding, int dtype, int out_dtype, void* workspace, void* stream) {
  if (T < 0 || V <= 0 || D <= 0 || V == 0x7fffffff) return B200_ERR_BAD_SHAPE;
  if (T > 0x3fffffff) return B200_ERR_TOO_LARGE;
  if ((uintptr_t)out % 32 || (uintptr_t)workspace % 16) return B200_ERR_BAD_ALIGN;
  if ((long long)V * D > (1ll << 42)) return B200_ERR_TOO_LARGE;
  if (out_dtype != dtype && out_dtype != B200_DT_FP32) return B200_ERR_UNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  const int es = dtype == B200_DT_FP32 ? 4 : 2, os = out_dtype == B200_DT_FP32 ? 4 : 2;
  const long long bytes = (long long)V * D * os, n32 = bytes / 32;
  uint2* a = (uint2*)workspace;
  uint2* b = (uint2*)((char*)workspace + (T * 8 + 15) / 16 * 16);
  float* part = (float*)((char*)workspace + 2 * ((T * 8 + 15) / 16 * 16));
  if (T > 0) {
    const int all = es_bits(V), passes = (all + kSortBits - 1) / kSortBits, bits = (all + passes - 1) / passes;
    B200_CHECK(cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSmem));
    embed_sort_kernel<<<kSortCtas, kSortThreads, kSortSmem, st>>>(ids, a, b, int(T), V, padding, bits, passes);
    B200_LAUNCH_CHECK();
  }
  {
    const unsigned grid = unsigned((n32 + 256) / 256);                   // at least one, and the last one has room for the rest
    if (T > 0) B200_CHECK(es_next(st, dim3(grid), 256, embed_fill_kernel, (uint8_t*)out, n32, int(bytes - n32 * 32)));
    else embed_fill_kernel<<<grid, 256, 0, st>>>((uint8_t*)out, n32, int(bytes - n32 * 32));
    B200_LAUNCH_CHECK();
  }
  if (T == 0) return 0;
  const int L = es_tile(T);
  const int V16 = 16 / es;
  const bool vec = D % V16 == 0 && (rs * es) % 16 == 0 && (uintptr_t)dy % 16 == 0;
#define ES_SUM(TI, TO) B200_CHECK((vec ? es_sum<TI, TO, 16 / sizeof(TI)>(a, dy, rs, out, part, int(T), V, D, L, scale, st) : es_sum<TI, TO, 1>(a, dy, rs, out, part, int(T), V, D, L, scale, st)))
  if (dtype == B200_DT_FP32) ES_SUM(float, float);
  else if (dtype == B200_DT_BF16 && out_dtype == B200_DT_BF16) ES_SUM(__nv_bfloat16, __nv_bfloat16);
  else if (dtype == B200_DT_BF16) ES_SUM(__nv_bfloat16, float);
  else if (dtype == B200_DT_FP16 && out_dtype == B200_DT_FP16) ES_SUM(__half, __half);
  else if (dtype == B200_DT_FP16) ES_SUM(__half, float);
  else return B200_ERR_UNSUPPORTED;
  B200_LAUNCH_CHECK();
  const int n = D % 4 == 0 ? 4 : 1, threads = D / n >= 256 ? 256 : (D / n + 31) / 32 * 32;
  const dim3 grid(unsigned((T + L - 1) / L), unsigned((D / n + threads - 1) / threads));
#define ES_JOIN(TO) es_next(st, grid, threads, n == 4 ? embed_join_kernel<TO, 4> : embed_join_kernel<TO, 1>, (const uint2*)a, (TO*)out, (const float*)part, int(T), V, D, L, scale)
  if (out_dtype == B200_DT_FP32) B200_CHECK(ES_JOIN(float));
  else if (out_dtype == B200_DT_BF16) B200_CHECK(ES_JOIN(__nv_bfloat16));
  else B200_CHECK(ES_JOIN(__half));
  return 0;
}
