// Rules on a batch of logits: penalties for repeated tokens, biases, temperature and a grammar's mask, in one pass.
//
// Batch row b follows the rules in row slot[b] of the tables of a LogitState. With l a logit in 32 bits, c(v) how often v stands in the
// row's output and seen(v) whether it stands in its prompt or output:
//   y = l;  seen: y < 0 ? y r : y / r;  c > 0: y -= f c, y -= p;  y += bias(v);  y /= T;  not allowed: -inf
// in this order, each step rounded once to 32 bits. A masked place is minus infinity whatever stood there, NaN included.
//   b200_process_logits    y, fp32
//   b200_greedy_tokens     the best token of each row, the lowest of equals; a NaN is above all (as in torch.argmax)
//
// A CTA owns a slice of a row's vocabulary: it counts the row's history in shared memory (integer atomics: any order, one result), looks up
// which bias (if any) a token has, and streams its logits past these tables. Nothing of a call is kept for the next one.
#include "common.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kLgThreads = 256, kLgSlice = 4096;
constexpr uint32_t kLgSeen = 0x80000000u;      // a token's word: seen at all | how often in the output

struct LogitRules {
  const int* slot;                              // [B] row of the tables; one outside of them has no rules
  int rows;
  const int *tokens, *length, *prompt_length;   // [rows, width]; the first prompt_length of length tokens are the prompt
  int width;
  const float *repetition, *presence, *frequency, *temperature;
  const int *bias_ids, *bias_length;            // [rows, bias_width]; of entries with one id the last one counts
  const float* bias_values;
  int bias_width;
  const int* mask;                              // [rows, words] bit v % 32 of word v / 32: v is allowed; null: no masks
  const unsigned char* masked;                  // [rows]
  int words;
};

struct RowRules {
  float r, f, p, T;
  int s;
  bool rules, counts, masked;
  int n_hist, n_prompt, n_bias;
};

__device__ __forceinline__ RowRules row_rules(const LogitRules& L, int b) {
  RowRules R = {1.f, 0.f, 0.f, 1.f, 0, false, false, false, 0, 0, 0};
  R.s = L.slot ? L.slot[b] : b;
  if ((unsigned)R.s >= (unsigned)L.rows) return R;
  R.rules = true;
  R.r = L.repetition[R.s]; R.f = L.frequency[R.s]; R.p = L.presence[R.s]; R.T = L.temperature[R.s];
  R.counts = R.r != 1.f || R.f != 0.f || R.p != 0.f;
  R.n_hist = R.counts ? min(max(L.length[R.s], 0), L.width) : 0;
  R.n_prompt = L.prompt_length[R.s];
  R.n_bias = L.bias_width > 0 ? min(max(L.bias_length[R.s], 0), L.bias_width) : 0;
  R.masked = L.mask != nullptr && L.masked[R.s] != 0;
  return R;
}

// one logit; word: the token's count and flag, bias: whether it has one
__device__ __forceinline__ float apply_rules(float y, const RowRules& R, uint32_t word, bool has_bias, float bias) {
  if (word & kLgSeen) y = y < 0.f ? __fmul_rn(y, R.r) : __fdiv_rn(y, R.r);
  const uint32_t c = word & ~kLgSeen;
  if (c) {
    y = __fsub_rn(y, __fmul_rn(R.f, (float)c));
    y = __fsub_rn(y, R.p);
  }
  if (has_bias) y = __fadd_rn(y, bias);
  return R.T != 1.f ? __fdiv_rn(y, R.T) : y;
}

// orders floats as unsigned numbers, NaN above all; the lower index wins among equals
__device__ __forceinline__ unsigned long long rank_of(float y, int v) {
  uint32_t u = __float_as_uint(y == 0.f ? 0.f : y);          // -0 and +0 are equals
  u = y != y ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return ((unsigned long long)u << 32) | (uint32_t)~(uint32_t)v;
}

template <typename T, bool GREEDY>
__global__ void __launch_bounds__(kLgThreads)
logits_kernel(const T* __restrict__ x, long long ldx, int V, const LogitRules L, float* __restrict__ out, long long ldo,
              unsigned long long* __restrict__ best) {
  __shared__ uint32_t word[kLgSlice];
  __shared__ int which[kLgSlice];
  __shared__ unsigned long long red[kLgThreads / 32];
  const int b = blockIdx.y, v0 = blockIdx.x * kLgSlice, nv = min(kLgSlice, V - v0), tid = threadIdx.x;
  const RowRules R = row_rules(L, b);
  const bool tables = R.n_hist > 0 || R.n_bias > 0;
  if (tables) {
    for (int i = tid; i < kLgSlice; i += kLgThreads) { word[i] = 0; which[i] = 0; }
    __syncthreads();
    const int* hist = L.tokens + (long long)R.s * L.width;
    for (int i = tid; i < R.n_hist; i += kLgThreads) {
      const int v = hist[i] - v0;
      if ((unsigned)v < (unsigned)nv) {
        atomicOr(&word[v], kLgSeen);
        if (i >= R.n_prompt) atomicAdd(&word[v], 1u);
      }
    }
    const int* ids = L.bias_ids + (long long)R.s * L.bias_width;
    for (int i = tid; i < R.n_bias; i += kLgThreads) {
      const int v = ids[i] - v0;
      if ((unsigned)v < (unsigned)nv) atomicMax(&which[v], i + 1);
    }
    __syncthreads();
  }
  const T* xr = x + (long long)b * ldx + v0;
  const float* values = L.bias_values + (long long)R.s * L.bias_width;
  const int* mask = R.masked ? L.mask + (long long)R.s * L.words + (v0 >> 5) : nullptr;
  unsigned long long mine = 0;
  for (int i = tid; i < nv; i += kLgThreads) {
    float y = to_f32<T>(xr[i]);
    const int w = tables ? which[i] : 0;
    y = apply_rules(y, R, tables ? word[i] : 0u, w > 0, w > 0 ? values[w - 1] : 0.f);
    if (mask && !((mask[i >> 5] >> (i & 31)) & 1)) y = -INFINITY;
    if (GREEDY) mine = max(mine, rank_of(y, v0 + i));
    else out[(long long)b * ldo + v0 + i] = y;
  }
  if (GREEDY) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((tid & 31) == 0) red[tid >> 5] = mine;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kLgThreads / 32; ++w) mine = max(mine, red[w]);
      best[(long long)b * gridDim.x + blockIdx.x] = mine;
    }
  }
}

__global__ void __launch_bounds__(32) greedy_pick_kernel(const unsigned long long* __restrict__ best, int parts, long long* __restrict__ ids) {
  unsigned long long m = 0;
  for (int i = threadIdx.x; i < parts; i += 32) m = max(m, best[(long long)blockIdx.x * parts + i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (threadIdx.x == 0) ids[blockIdx.x] = (long long)(uint32_t)~(uint32_t)m;
}

// tokens that have come: behind the history of their rows. A full row keeps what it has
__global__ void append_tokens_kernel(int* __restrict__ tokens, int rows, int width, int* __restrict__ length, const int* __restrict__ slot,
                                     const long long* __restrict__ ids, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int s = slot ? slot[i] : i;
  if ((unsigned)s >= (unsigned)rows) return;
  const int at = length[s];
  if ((unsigned)at >= (unsigned)width) return;
  tokens[(long long)s * width + at] = (int)ids[i];
  length[s] = at + 1;
}

}  // namespace b200
using namespace b200;

static int logit_rules(const b200_logit_rules* a, const int* slot, LogitRules& L) {
  if (!a || a->rows < 0 || a->width < 0 || a->bias_width < 0 || a->words < 0) return B200_ERR_BAD_SHAPE;
  L = {slot, a->rows, a->tokens, a->length, a->prompt_length, a->width, a->repetition, a->presence, a->frequency, a->temperature,
       a->bias_ids, a->bias_length, a->bias_values, a->bias_width, a->mask, a->masked, a->words};
  return 0;
}

B200_API long long b200_greedy_workspace(int B, int V) { return B < 1 || V < 1 ? 0 : (long long)B * ceil_div(V, kLgSlice) * 8; }

B200_API int b200_process_logits(const void* x, long long ldx, int B, int V, const int* slot, const b200_logit_rules* rules, float* out, long long ldo, int dtype,
                                 void* stream) {
  LogitRules L;
  if (int rc = logit_rules(rules, slot, L)) return rc;
  if (B < 0 || V < 1 || B > 65535 || (L.mask && (long long)L.words * 32 < V)) return B200_ERR_BAD_SHAPE;
  if (B == 0) return 0;
  const dim3 grid(ceil_div(V, kLgSlice), B);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == B200_DT_FP32) logits_kernel<float, false><<<grid, kLgThreads, 0, st>>>((const float*)x, ldx, V, L, out, ldo, nullptr);
  else if (dtype == B200_DT_BF16) logits_kernel<__nv_bfloat16, false><<<grid, kLgThreads, 0, st>>>((const __nv_bfloat16*)x, ldx, V, L, out, ldo, nullptr);
  else if (dtype == B200_DT_FP16) logits_kernel<__half, false><<<grid, kLgThreads, 0, st>>>((const __half*)x, ldx, V, L, out, ldo, nullptr);
  else return B200_ERR_UNSUPPORTED;
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_greedy_tokens(const void* x, long long ldx, int B, int V, const int* slot, const b200_logit_rules* rules, void* workspace, long long* ids, int dtype,
                                void* stream) {
  LogitRules L;
  if (int rc = logit_rules(rules, slot, L)) return rc;
  if (B < 0 || V < 1 || B > 65535 || (L.mask && (long long)L.words * 32 < V)) return B200_ERR_BAD_SHAPE;
  if (B == 0) return 0;
  const dim3 grid(ceil_div(V, kLgSlice), B);
  cudaStream_t st = (cudaStream_t)stream;
  unsigned long long* best = (unsigned long long*)workspace;
  if (dtype == B200_DT_FP32) logits_kernel<float, true><<<grid, kLgThreads, 0, st>>>((const float*)x, ldx, V, L, nullptr, 0, best);
  else if (dtype == B200_DT_BF16) logits_kernel<__nv_bfloat16, true><<<grid, kLgThreads, 0, st>>>((const __nv_bfloat16*)x, ldx, V, L, nullptr, 0, best);
  else if (dtype == B200_DT_FP16) logits_kernel<__half, true><<<grid, kLgThreads, 0, st>>>((const __half*)x, ldx, V, L, nullptr, 0, best);
  else return B200_ERR_UNSUPPORTED;
  greedy_pick_kernel<<<B, 32, 0, st>>>(best, grid.x, ids);
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_append_tokens(int* tokens, int rows, int width, int* length, const int* slot, const long long* ids, int n, void* stream) {
  if (n < 0 || rows < 0 || width < 0) return B200_ERR_BAD_SHAPE;
  if (n == 0) return 0;
  append_tokens_kernel<<<ceil_div(n, 128), 128, 0, (cudaStream_t)stream>>>(tokens, rows, width, length, slot, ids, n);
  B200_LAUNCH_CHECK();
  return 0;
}
