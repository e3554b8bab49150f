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
//   lp_rows        logits [B, V] -> lp, H, rank, alternatives, and (m, 1 / s, log s, H) for the backward pass; a CTA a row
//   lp_rows_grad   logits, (m, 1 / s, log s, H), g, h -> dl, in one pass
// and for logits x w^T that are never there as a whole, a chunk of the vocabulary at a time (products by gemm_tcgen05.cu):
//   lp_chunk       a chunk's logits (fp32) join m, s, u and l_t of their rows
//   lp_finish      lp, H and what the backward pass needs
//   lp_chunk_grad  a chunk's logits, computed again, -> dl in 16 bits, the operand of the products dl w and dl^T x
// Rows of logits are bound by HBM; a 16-bit logit has eight operations beside its exponential.
#include "common.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kLpThreads = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LpSum { float m, s, u; };

__device__ __forceinline__ float lp_exp2(float x) { return exp2f(x); }
// x where it is a factor beside 2^x: below -200 that is zero, and zero times minus infinity would not be.
__device__ __forceinline__ float lp_factor(float x) { return fmaxf(x, -200.f); }

// What lies in two parts of a row as if it were one. c = log2(e) / T.
template <bool ENT>
__device__ __forceinline__ LpSum lp_both(LpSum a, LpSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.u + b.u};               // nothing yet (or a NaN in s)
  const float xa = (a.m - m) * c, xb = (b.m - m) * c, fa = lp_exp2(xa), fb = lp_exp2(xb);
  LpSum r{m, a.s * fa + b.s * fb, 0.f};
  if constexpr (ENT) r.u = fa * (a.u + a.s * lp_factor(xa)) + fb * (b.u + b.s * lp_factor(xb));
  return r;
}

template <bool ENT>
__device__ __forceinline__ LpSum lp_block(LpSum a, float c, float* red) {      // red: 96 floats
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = lp_both<ENT>(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)}, c);
  __syncthreads();
  if (lane == 0) { red[w] = a.m; red[32 + w] = a.s; red[64 + w] = a.u; }
  __syncthreads();
  a = lane < nw ? LpSum{red[lane], red[32 + lane], red[64 + lane]} : LpSum{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = lp_both<ENT>(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.u, o)}, c);
  return a;
}

__device__ __forceinline__ int lp_block_count(int v, int* red) {               // red: 32 ints
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0);
}

// n values join the sums: the largest first, so that a group rescales at most once.
template <bool ENT, int N>
__device__ __forceinline__ void lp_join(LpSum& a, const float (&v)[N], float c) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  if (m > a.m) {
    const float x = (a.m - m) * c, f = lp_exp2(x);
    if constexpr (ENT) a.u = f * (a.u + a.s * lp_factor(x));
    a.s *= f;
    a.m = m;
  }
  const float base = a.m == -INFINITY ? 0.f : a.m;                    // minus infinities alone: their weights are zeros
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float x = (v[i] - base) * c, e = lp_exp2(x);
    a.s += e;
    if constexpr (ENT) a.u = fmaf(e, lp_factor(x), a.u);
  }
}

// f(index of the first, values) for groups of N neighbours of p[0 .. n) and f1 for single ones at its unaligned ends, over the CTA's threads.
template <typename T, typename F, typename F1>
__device__ __forceinline__ void lp_walk(const T* __restrict__ p, int n, F f, F1 f1) {
  constexpr int V = 16 / sizeof(T), G = 4, N = V * G;
  const int head = min(n, int((16 - ((uintptr_t)p & 15)) & 15) / int(sizeof(T)));
  if (threadIdx.x < head) f1(threadIdx.x, to_f32<T>(p[threadIdx.x]));
  const int nvec = (n - head) / V;
  const uint4* q = reinterpret_cast<const uint4*>(p + head);
  int i = threadIdx.x;
  for (; i + (G - 1) * blockDim.x < nvec; i += G * blockDim.x) {
    uint4 raw[G];
#pragma unroll
    for (int g = 0; g < G; ++g) raw[g] = __ldg(q + i + g * blockDim.x);
    float v[N];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < V; ++j) v[g * V + j] = to_f32<T>(reinterpret_cast<const T*>(&raw[g])[j]);
    f(v);
  }
  for (; i < nvec; i += blockDim.x) {
    const uint4 raw = __ldg(q + i);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f32<T>(reinterpret_cast<const T*>(&raw)[j]);
    f(v);
  }
  for (int j = head + nvec * V + threadIdx.x; j < n; j += blockDim.x) f1(j, to_f32<T>(p[j]));
}

// Order of logits as whole numbers: NaN above all, -0 as 0; ties by the lower id.
__device__ __forceinline__ unsigned long long lp_key(float v, uint32_t id) {
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);
  const uint32_t o = v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (unsigned long long)o << 32 | uint32_t(~id);
}

template <typename T, bool ENT>
__global__ void __launch_bounds__(kLpThreads)
lp_rows_kernel(const T* __restrict__ logits, long long rs, int V, const long long* __restrict__ tokens, float inv_t, int top, float* __restrict__ lp,
               float* __restrict__ ent, long long* __restrict__ rank, long long* __restrict__ top_ids, float* __restrict__ top_lp,
               float4* __restrict__ stats) {
  __shared__ float red[96];
  __shared__ int redi[32];
  __shared__ unsigned long long redk[32];
  const long long row = blockIdx.x;
  const long long t = tokens ? tokens[row] : 0;
  if (t < 0 || t >= V) {
    if (threadIdx.x == 0) {
      if (lp) lp[row] = 0.f;
      if (ENT) ent[row] = 0.f;
      if (rank) rank[row] = 0;
      if (stats) stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i = threadIdx.x; i < top; i += blockDim.x) { top_ids[row * top + i] = -1; top_lp[row * top + i] = 0.f; }
    return;
  }
  const T* p = logits + row * rs;
  const float c = inv_t * kLog2e, lt = to_f32<T>(p[t]);
  LpSum a{-INFINITY, 0.f, 0.f};
  int above = 0;
  lp_walk<T>(p, V, [&](const auto& v) {
    lp_join<ENT>(a, v, c);
    if (rank) {
#pragma unroll
      for (int i = 0; i < int(sizeof(v) / 4); ++i) above += v[i] > lt;
    }
  }, [&](int, float x) {
    const float v[1] = {x};
    lp_join<ENT>(a, v, c);
    above += x > lt;
  });
  a = lp_block<ENT>(a, c, red);
  if (rank) above = lp_block_count(above, redi);
  const float ls = logf(a.s);
  const float H = ENT ? ls - kLn2 * a.u / a.s : 0.f;
  if (threadIdx.x == 0) {
    if (lp) lp[row] = (lt - a.m) * inv_t - ls;
    if (ENT) ent[row] = H;
    if (rank) rank[row] = 1 + above;
    if (stats) stats[row] = make_float4(a.m, 1.f / a.s, ls, H);
  }
  unsigned long long last = ~0ull;                                     // above every key: a NaN's has ids below 2^31
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < V; j += blockDim.x) {
      const unsigned long long key = lp_key(to_f32<T>(p[j]), j);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, best, o);
      best = x > best ? x : best;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) redk[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int w = 0; w < kLpThreads / 32; ++w) best = redk[w] > best ? redk[w] : best;
    last = best;
    if (threadIdx.x == 0) {
      const int id = int(~uint32_t(best));
      top_ids[row * top + k] = id;
      top_lp[row * top + k] = (to_f32<T>(p[id]) - a.m) * inv_t - ls;
    }
  }
}

// dl_j = 2^x_j (A + B x_j) + [j = t] g / T with A = -(g + h (H - log s)) / T, B = -h log(2) / T, both with 1 / s in them.
struct LpGrad { float m, A, B, g; long long t; };
__device__ __forceinline__ LpGrad lp_grad_of(float4 st, float g, float h, float inv_t, long long t, float scale) {
  return {st.x, -(g + h * (st.w - st.z)) * inv_t * st.y * scale, -h * kLn2 * inv_t * st.y * scale, g * inv_t * scale, t};
}
__device__ __forceinline__ float lp_grad_at(float l, const LpGrad& q, float c) {
  const float x = (l - q.m) * c;
  return lp_exp2(x) * fmaf(q.B, lp_factor(x), q.A);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads)
lp_rows_grad_kernel(const T* __restrict__ logits, long long rs, int V, const long long* __restrict__ tokens, float inv_t, const float4* __restrict__ stats,
                    const float* __restrict__ g, const float* __restrict__ h, T* __restrict__ out, long long os) {
  constexpr int N = 16 / sizeof(T);
  const long long row = blockIdx.x;
  const long long t = tokens ? tokens[row] : 0;
  const bool skip = t < 0 || t >= V;
  const T* p = logits + row * rs;
  T* o = out + row * os;
  const float c = inv_t * kLog2e;
  const LpGrad q = lp_grad_of(stats[row], g ? g[row] : 0.f, h ? h[row] : 0.f, inv_t, tokens ? t : -1, 1.f);
  const bool same = (((uintptr_t)p ^ (uintptr_t)o) & 15) == 0;          // both aligned at the same elements
  const int head = min(V, int((16 - ((uintptr_t)p & 15)) & 15) / int(sizeof(T)));
  const int nvec = (V - head) / N;
  auto one = [&](int j) { o[j] = from_f32<T>(skip ? 0.f : lp_grad_at(to_f32<T>(p[j]), q, c) + (j == q.t ? q.g : 0.f)); };
  if (threadIdx.x < head) one(threadIdx.x);
  for (int i = threadIdx.x; i < nvec; i += blockDim.x) {
    const int j0 = head + i * N;
    alignas(16) T in[N];
    alignas(16) T r[N];
    if (!skip) *reinterpret_cast<uint4*>(in) = __ldg(reinterpret_cast<const uint4*>(p + j0));
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = from_f32<T>(skip ? 0.f : lp_grad_at(to_f32<T>(in[j]), q, c) + (j0 + j == q.t ? q.g : 0.f));
    if (same) *reinterpret_cast<uint4*>(o + j0) = *reinterpret_cast<uint4*>(r);
    else
#pragma unroll
      for (int j = 0; j < N; ++j) o[j0 + j] = r[j];
  }
  for (int j = head + nvec * N + threadIdx.x; j < V; j += blockDim.x) one(j);
}

// ---- logits a chunk of the vocabulary at a time ----
// run [rows] = (m, s, u, l_t) of what came before columns c0 .. c0 + C of the vocabulary; the first chunk makes it.
template <bool ENT>
__global__ void __launch_bounds__(256)
lp_chunk_kernel(const float* __restrict__ lg, long long rs, int C, int c0, const long long* __restrict__ tokens, float inv_t, float4* __restrict__ run) {
  __shared__ float red[96];
  const long long row = blockIdx.x;
  const float c = inv_t * kLog2e;
  const float* p = lg + row * rs;
  LpSum a{-INFINITY, 0.f, 0.f};
  lp_walk<float>(p, C, [&](const auto& v) { lp_join<ENT>(a, v, c); }, [&](int, float x) { const float v[1] = {x}; lp_join<ENT>(a, v, c); });
  a = lp_block<ENT>(a, c, red);
  if (threadIdx.x == 0) {
    float4 r = c0 == 0 ? make_float4(-INFINITY, 0.f, 0.f, 0.f) : run[row];
    const LpSum b = lp_both<ENT>({r.x, r.y, r.z}, a, c);
    const long long t = tokens ? tokens[row] - c0 : -1;
    run[row] = make_float4(b.m, b.s, b.u, t >= 0 && t < C ? p[t] : r.w);
  }
}

__global__ void __launch_bounds__(256)
lp_finish_kernel(const float4* __restrict__ run, long long rows, int V, const long long* __restrict__ tokens, float inv_t, float* __restrict__ lp,
                 float* __restrict__ ent, float4* __restrict__ stats) {
  const long long row = blockIdx.x * 256ll + threadIdx.x;
  if (row >= rows) return;
  const long long t = tokens ? tokens[row] : 0;
  const bool skip = t < 0 || t >= V;
  const float4 r = run[row];
  const float ls = logf(r.y), H = ls - kLn2 * r.z / r.y;
  if (lp) lp[row] = skip ? 0.f : (r.w - r.x) * inv_t - ls;
  if (ent) ent[row] = skip ? 0.f : H;
  if (stats) stats[row] = make_float4(r.x, 1.f / r.y, ls, H);
}

// A power of two that brings the largest gradient of a logit to 2^13 .. 2^14, so that fp16 holds the small ones too, and its reciprocal.
// |dl| <= (|g| + |h| (log V + 1)) / T.
__global__ void __launch_bounds__(256)
lp_scale_kernel(const float* __restrict__ g, const float* __restrict__ h, long long rows, float inv_t, float log_v, float* __restrict__ scale) {
  __shared__ float red[32];
  float m = 0.f;
  for (long long i = threadIdx.x; i < rows; i += 256) m = fmaxf(m, ((g ? fabsf(g[i]) : 0.f) + (h ? fabsf(h[i]) : 0.f) * (log_v + 1.f)) * inv_t);
  m = block_max(m, red);
  if (threadIdx.x) return;
  const int e = m > 0.f && m < INFINITY ? min(max(14 - (ilogbf(m) + 1), -100), 100) : 0;
  scale[0] = ldexpf(1.f, e);
  scale[1] = ldexpf(1.f, -e);
}

template <typename T>
__global__ void __launch_bounds__(256)
lp_chunk_grad_kernel(const float* __restrict__ lg, long long rs, int C, int c0, int V, const long long* __restrict__ tokens, float inv_t,
                     const float4* __restrict__ stats, const float* __restrict__ g, const float* __restrict__ h, const float* __restrict__ scale,
                     T* __restrict__ out, long long os) {
  const long long row = blockIdx.x;
  const long long t = tokens ? tokens[row] : 0;
  const bool skip = t < 0 || t >= V;
  const float* p = lg + row * rs;
  T* o = out + row * os;
  const float c = inv_t * kLog2e;
  const LpGrad q = lp_grad_of(stats[row], g ? g[row] : 0.f, h ? h[row] : 0.f, inv_t, tokens ? t - c0 : -1, scale ? scale[0] : 1.f);
  for (int j0 = threadIdx.x * 4; j0 < C; j0 += blockDim.x * 4) {        // rows of both are padded to whole groups of four
    const float4 in = *reinterpret_cast<const float4*>(p + j0);
    const float v[4] = {in.x, in.y, in.z, in.w};
    alignas(8) T r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = from_f32<T>(skip || j0 + j >= C ? 0.f : lp_grad_at(v[j], q, c) + (j0 + j == q.t ? q.g : 0.f));
    *reinterpret_cast<uint2*>(o + j0) = *reinterpret_cast<uint2*>(r);
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

B200_API int b200_token_logprobs(const void* logits, long long rs, long long rows, int V, const long long* tokens, float inv_t, int top, float* lp,
                                 float* ent, long long* rank, long long* top_ids, float* top_lp, void* stats, int dtype, void* stream) {
  if (lp_bad(rows, V) || top < 0 || top > 32 || top > V) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  LP_TYPES(dtype, {
    if (ent) lp_rows_kernel<T, true><<<(unsigned)rows, kLpThreads, 0, st>>>((const T*)logits, rs, V, tokens, inv_t, top, lp, ent, rank, top_ids, top_lp, (float4*)stats);
    else lp_rows_kernel<T, false><<<(unsigned)rows, kLpThreads, 0, st>>>((const T*)logits, rs, V, tokens, inv_t, top, lp, ent, rank, top_ids, top_lp, (float4*)stats);
  });
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_token_logprobs_grad(const void* logits, long long rs, long long rows, int V, const long long* tokens, float inv_t, const void* stats,
                                      const float* g, const float* h, void* out, long long os, int dtype, void* stream) {
  if (lp_bad(rows, V)) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  LP_TYPES(dtype, lp_rows_grad_kernel<T><<<(unsigned)rows, kLpThreads, 0, st>>>((const T*)logits, rs, V, tokens, inv_t, (const float4*)stats, g, h,
                                                                             (T*)out, os));
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_chunk(const float* lg, long long rs, long long rows, int C, int c0, const long long* tokens, float inv_t, void* run, int entropy,
                                void* stream) {
  if (lp_bad(rows, C) || c0 < 0) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (entropy) lp_chunk_kernel<true><<<(unsigned)rows, 256, 0, st>>>(lg, rs, C, c0, tokens, inv_t, (float4*)run);
  else lp_chunk_kernel<false><<<(unsigned)rows, 256, 0, st>>>(lg, rs, C, c0, tokens, inv_t, (float4*)run);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_finish(const void* run, long long rows, int V, const long long* tokens, float inv_t, float* lp, float* ent, void* stats,
                                 void* stream) {
  if (lp_bad(rows, V)) return B200_ERR_BAD_SHAPE;
  if (rows == 0) return 0;
  lp_finish_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, (cudaStream_t)stream>>>((const float4*)run, rows, V, tokens, inv_t, lp, ent, (float4*)stats);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_scale(const float* g, const float* h, long long rows, float inv_t, int V, float* scale, void* stream) {
  if (lp_bad(rows, V)) return B200_ERR_BAD_SHAPE;
  lp_scale_kernel<<<1, 256, 0, (cudaStream_t)stream>>>(g, h, rows, inv_t, logf((float)V), scale);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_logprob_chunk_grad(const float* lg, long long rs, long long rows, int C, int c0, int V, const long long* tokens, float inv_t,
                                     const void* stats, const float* g, const float* h, const float* scale, void* out, long long os, int dtype, void* stream) {
  if (lp_bad(rows, C) || c0 < 0 || rs < (C + 3) / 4 * 4 || os < (C + 3) / 4 * 4) return B200_ERR_BAD_SHAPE;
  if (rs % 4 || os % 4 || (uintptr_t)lg % 16 || (uintptr_t)out % 8) return B200_ERR_BAD_ALIGN;
  if (rows == 0) return 0;
  LP_TYPES16(dtype, lp_chunk_grad_kernel<T><<<(unsigned)rows, 256, 0, (cudaStream_t)stream>>>(lg, rs, C, c0, V, tokens, inv_t, (const float4*)stats, g, h,
                                                                                          scale, (T*)out, os));
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
