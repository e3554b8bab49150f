// The arithmetic that the kernels of log probabilities share (logprobs.cu, and the epilogues of gemm_tcgen05.cu).
#pragma once
#include "common.cuh"

namespace b200 {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What is kept of the logits seen so far: the largest, m, and with x = (l - m) log2(e) / T the sums s = sum 2^x and u = sum 2^x x.
struct LpSum { float m, s, u; };

// 2^x to 2^-22 relative; zero below 2^-126 (a weight that adds nothing to a sum of at least 1).
__device__ __forceinline__ float lp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x where it is a factor beside 2^x: below -200 that is zero, and zero times minus infinity would not be.
__device__ __forceinline__ float lp_factor(float x) { return fmaxf(x, -200.f); }

// Two numbers of 32 bits to an instruction.
__device__ __forceinline__ unsigned long long lp_pair(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 lp_split(unsigned long long a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ unsigned long long lp_add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long lp_mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long lp_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

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

// n values, of which m is the largest, join the sums: rescaled at most once for all of them.
template <bool ENT, int N>
__device__ __forceinline__ void lp_join(LpSum& a, const float (&v)[N], float m, float c) {
  if (m > a.m) {
    const float x = (a.m - m) * c, f = lp_exp2(x);
    if constexpr (ENT) a.u = f * (a.u + a.s * lp_factor(x));
    a.s *= f;
    a.m = m;
  }
  const float base = a.m == -INFINITY ? 0.f : a.m;                    // minus infinities alone: their weights are zeros
  if constexpr (N % 2 == 0) {
    const unsigned long long nb = lp_pair(-base, -base), cc = lp_pair(c, c);
    unsigned long long s = 0, u = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const unsigned long long x = lp_mul2(lp_add2(lp_pair(v[i], v[i + 1]), nb), cc);
      const float2 xs = lp_split(x);
      const unsigned long long e = lp_pair(lp_exp2(xs.x), lp_exp2(xs.y));
      s = lp_add2(s, e);
      if constexpr (ENT) u = lp_fma2(e, lp_pair(lp_factor(xs.x), lp_factor(xs.y)), u);
    }
    const float2 s2 = lp_split(s), u2 = lp_split(u);
    a.s += s2.x + s2.y;
    if constexpr (ENT) a.u += u2.x + u2.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = (v[i] - base) * c, e = lp_exp2(x);
      a.s += e;
      if constexpr (ENT) a.u = fmaf(e, lp_factor(x), a.u);
    }
  }
}
template <bool ENT, int N>
__device__ __forceinline__ void lp_join(LpSum& a, const float (&v)[N], float c) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  lp_join<ENT>(a, v, m, c);
}

// dl_j = 2^x_j (A + B x_j) + [j = t] g / T with A = -(g + h (H - log s)) / T, B = -h log(2) / T, both with 1 / s in them.
// st = (m, 1 / s, log s, H) of the row.
struct LpGrad { float m, A, B, g; long long t; };
__device__ __forceinline__ LpGrad lp_grad_of(float4 st, float g, float h, float inv_t, long long t, float scale) {
  return {st.x, -(g + h * (st.w - st.z)) * inv_t * st.y * scale, -h * kLn2 * inv_t * st.y * scale, g * inv_t * scale, t};
}
__device__ __forceinline__ float lp_grad_at(float l, const LpGrad& q, float c) {
  const float x = (l - q.m) * c;
  return lp_exp2(x) * fmaf(q.B, lp_factor(x), q.A);
}

}  // namespace b200
