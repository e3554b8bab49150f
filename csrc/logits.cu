// Rules on a batch of logits: penalties for repeated tokens, biases, temperature and a grammar's mask, in one pass.
//
// Batch row b follows the rules in row slot[b] of the tables of a LogitState. With l a logit in 32 bits, c(v) how often v stands in the
// row's output and seen(v) whether it stands in its prompt or output:
//   y = l;  seen: y < 0 ? y r : y / r;  c > 0: y -= f c, y -= p;  y += bias(v);  y /= T;  not allowed: -inf
// in this order, each step rounded once to 32 bits. So r scales what the model says and not the bias (where a bias is added first, r scales it too). A masked place is minus infinity whatever stood there, NaN included.
//   b200_process_logits    y, fp32
//   b200_greedy_tokens     the best token of each row, the lowest of equals; a NaN is above all (as in torch.argmax)
//
// Two kernels. One, a CTA to a row, counts the row's history and notes its biases in a hash table in shared memory (integer atomics: any order, one
// result) and settles the few logits that these say something of, each by one thread. The other streams all of the logits past temperature and mask, as many
// loads under way as registers hold. Where logits are written elsewhere the stream goes first, and what is settled is written over it; where they stay in their
// place, or only the best is asked for, the settling kernel goes first and leaves a bitmap of what the stream is to pass over. Either way the second starts while the
// first ends. Nothing of a call is kept for the next one.
//
// Bound: memory. 128 x 151936 in 32 bits, histories of up to 6000 tokens, 300 biases, half of the rows masked (158 MB): 24 us; here 47 (52 with the settling
// first), 27 of them the stream (5.8 TB/s) and the rest the settling, of which a little is beside it: 3 us of table, 5 to 11 of tokens entered, 6 of single logits, 4800 of a
// row, which lie in half of the memory of its 152 000. A stream of four CTAs to an SM that go on from tile to tile leaves room for the settling kernel beside it, but
// each slows the other: 60 to 74 us. One
// kernel with the counts of a slice in shared memory is kept waiting by its own steps (rules, history, counts, logits): 100 us in slices of 4096
// tokens (which small batches keep, see kLmSlices), 69 to 78 in slices of 20480 with the history counted once for clusters of 2 to 8 CTAs (8 rows: 8.8 and
// 6.5 us; by these two kernels 9.7, by the one of small batches 7.2). The rules applied in the stream, from records in token order, took 64: almost every warp
// had a lane with one.
#include "common.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kLgThreads = 256, kLgQuads = 2;                      // streaming kernel: twice four logits to a thread
constexpr int kLgTokens = kLgThreads * kLgQuads * 4;
constexpr int kLsThreads = 1024, kLsEarly = 6;                     // settling kernel; tokens that a thread asks for before it knows how many there are
constexpr int kLsSlots = 16384;                                    // of its table, at most
constexpr int kLgVocab = 1 << 19;                                  // its bitmap has room for so many tokens
// a token's word: whether it stands in the prompt | its last bias, counted from 1 | how often it stands in the output
constexpr uint32_t kLgSeen = 0x80000000u, kLgCount = 0xfffffu, kLsFree = 0xffffffffu;
constexpr int kLgBias = 20;

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
  float r, f, p, T, inv_T;
  int n_hist, n_prompt, n_bias;
  bool masked;
};

// the rules of table row s: one round of loads
__device__ __forceinline__ RowRules row_rules(const LogitRules& L, int s) {
  RowRules R;
  R.r = L.repetition[s]; R.f = L.frequency[s]; R.p = L.presence[s]; R.T = L.temperature[s];
  const int length = L.length[s];
  R.n_prompt = L.prompt_length[s];
  R.n_bias = L.bias_width > 0 ? min(max(L.bias_length[s], 0), L.bias_width) : 0;
  R.masked = L.mask != nullptr && L.masked[s] != 0;
  R.n_hist = R.r != 1.f || R.f != 0.f || R.p != 0.f ? min(max(length, 0), L.width) : 0;
  R.inv_T = __frcp_rn(R.T);
  return R;
}

// y / d: the product with 1 / d, corrected once by what is left of y (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990), which leaves no more than a division's rounding but in the last of the smallest numbers. The product may pass the largest number where the quotient
// does not: that one goes by halves, which are exact there. An infinite half has nothing left over.
__device__ __forceinline__ float quotient(float y, float d, float inv) {
  const float q = __fmul_rn(y, inv);
  if (fabsf(q) < INFINITY) return __fmaf_rn(__fmaf_rn(-q, d, y), inv, q);
  const float h = __fmul_rn(0.5f, y), p = __fmul_rn(h, inv);
  return fabsf(p) < INFINITY ? __fmul_rn(2.f, __fmaf_rn(__fmaf_rn(-p, d, h), inv, p)) : p;
}
// four at once, two to an instruction
__device__ __forceinline__ void over_temperature(float (&y)[4], float T, float inv_T) {
  const float size = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
  if (__fmul_rn(size, inv_T) < INFINITY) {
    const float2 inv = make_float2(inv_T, inv_T), t = make_float2(T, T);
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float2 v = make_float2(y[e], y[e + 1]), q = __fmul2_rn(v, inv), n = make_float2(-q.x, -q.y);
      const float2 c = __ffma2_rn(__ffma2_rn(n, t, v), inv, q);
      y[e] = c.x; y[e + 1] = c.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = quotient(y[e], T, inv_T);
  }
}
// one logit that the table knows something of (word: what), temperature and all
__device__ __forceinline__ float apply_word(float y, const RowRules& R, uint32_t word, const float* __restrict__ values) {
  const uint32_t c = word & kLgCount, b = (word & ~kLgSeen) >> kLgBias;
  if (c || (word & kLgSeen)) y = y < 0.f ? __fmul_rn(y, R.r) : quotient(y, R.r, __frcp_rn(R.r));
  if (c) {
    y = __fsub_rn(y, __fmul_rn(R.f, (float)c));
    y = __fsub_rn(y, R.p);
  }
  if (b) y = __fadd_rn(y, values[b - 1]);
  return quotient(y, R.T, R.inv_T);
}

// orders floats as unsigned numbers, NaN above all
__device__ __forceinline__ uint32_t order_of(float y) {
  const uint32_t u = __float_as_uint(y == 0.f ? 0.f : y);    // -0 and +0 are equals
  return y != y ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// four logits as they lie in memory
template <typename T> struct Quad;
template <> struct Quad<float> { float4 v; __device__ __forceinline__ float at(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; } };
template <typename T> struct Quad {
  uint2 v;
  __device__ __forceinline__ float at(int i) const {
    const uint32_t w = i < 2 ? v.x : v.y;
    const unsigned short h = (unsigned short)(i & 1 ? w >> 16 : w);
    return to_f32<T>(*reinterpret_cast<const T*>(&h));
  }
};
template <typename T> __device__ __forceinline__ Quad<T> load_quad(const T* x, int left, bool whole) {
  union { Quad<T> q; T e[4]; } u;
  if (whole && left >= 4) return *reinterpret_cast<const Quad<T>*>(x);
#pragma unroll
  for (int i = 0; i < 4; ++i) u.e[i] = i < left ? x[i] : from_f32<T>(0.f);
  return u.q;
}

// the largest of numbers; NaN if one of them is
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ unsigned long long rank_of(float y, int v) { return ((unsigned long long)order_of(y) << 32) | (uint32_t)~(uint32_t)v; }      // of equals the lowest

// what a stream that comes second needs of a batch row's rules
struct __align__(16) RowPlan { float T, inv_T; int mask_row, settled; };      // mask_row: -1 for none; settled: the bitmap has bits

// LAST: it goes over what the streaming kernel left, and sees to the mask. Otherwise it comes first and says what is settled; x and out may then be the same
template <typename T, bool GREEDY, bool LAST>
__global__ void __launch_bounds__(kLsThreads, 1)
logits_settle_kernel(const T* x, long long ldx, int V, const LogitRules L, float* out, long long ldo, RowPlan* __restrict__ plan, uint32_t* __restrict__ bitmap,
                     unsigned long long* __restrict__ best, int parts, int most_slots) {
  extern __shared__ __align__(16) uint32_t smem_ls[];         // bitmap, keys, words, places of the tokens found
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, bit_words = LAST ? 0 : (V + 127) / 128 * 4;
  uint32_t *bits = smem_ls, *keys = bits + bit_words;
  __shared__ unsigned long long red[kLsThreads / 32];
  __shared__ int n_found;
  if (!LAST) pdl_launch_dependents();
  const int row = L.slot ? L.slot[b] : b;
  const bool ruled = (unsigned)row < (unsigned)L.rows;
  // What the row's history and biases are is asked for together with how long they are: a table's row may be read to its end
  RowRules R = {1.f, 0.f, 0.f, 1.f, 1.f, 0, 0, 0, false};
  const long long r0 = ruled ? row : 0;
  const int *hist = L.tokens + r0 * L.width, *ids = L.bias_ids + r0 * L.bias_width;
  int early[kLsEarly], early_bias[2] = {-1, -1};
  if (ruled) {
#pragma unroll
    for (int i = 0; i < kLsEarly; ++i) early[i] = tid + i * kLsThreads < L.width ? hist[tid + i * kLsThreads] : -1;
#pragma unroll
    for (int i = 0; i < 2; ++i)                               // no row has more than 2047
      if (tid + i * kLsThreads < L.bias_width) early_bias[i] = ids[tid + i * kLsThreads];
    R = row_rules(L, row);
  }
  const bool tables = R.n_hist > 0 || R.n_bias > 0;
  if (!LAST && tid == 0) plan[b] = {R.T, R.inv_T, R.masked ? row : -1, tables ? 1 : 0};
  unsigned long long mine = 0;
  if (tables) {
    const int* mask = (GREEDY || LAST) && R.masked ? L.mask + r0 * L.words : nullptr;      // else the stream sees to it
    const float* values = L.bias_values + r0 * L.bias_width;
    const T* xr = x + (long long)b * ldx;
    int slots = min(1024, most_slots);                        // twice the tokens, if that is not too many
    while (slots < most_slots && slots < 2 * (R.n_hist + R.n_bias)) slots *= 2;
    uint32_t* word = keys + slots;
    uint16_t* found = reinterpret_cast<uint16_t*>(word + slots);
    // up to three quarters of its slots the table is one of hashes; a longer history goes by parts of the vocabulary, a slot for each token
    const bool hashed = R.n_hist + R.n_bias <= slots / 4 * 3;
    bool waited = !LAST;
    const int turns = hashed ? 1 : (V + slots - 1) / slots;
    for (int i = tid; i < bit_words / 4; i += kLsThreads) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0, 0, 0, 0);
    for (int turn = 0; turn < turns; ++turn) {
      __syncthreads();                                        // the last turn's words have been read
      if (tid == 0) n_found = 0;
      for (int i = tid; i < slots / 4; i += kLsThreads) {
        reinterpret_cast<uint4*>(keys)[i] = make_uint4(kLsFree, kLsFree, kLsFree, kLsFree);
        reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
      // the slot of token v, -1: not a token, or not this turn's. made: this thread is the first that asked for it
      auto slot_of = [&](int v, bool& made) {
        made = false;
        if ((unsigned)v >= (unsigned)V) return -1;
        if (!hashed) {
          if (v / slots != turn) return -1;
          made = keys[v % slots] == kLsFree && atomicCAS(keys + v % slots, kLsFree, (uint32_t)v) == kLsFree;
          return v % slots;
        }
        uint32_t h = __umulhi((uint32_t)v * 2654435769u, (uint32_t)slots);      // 2^32 / golden ratio
        while (true) {                                        // there are more slots than tokens: it ends
          uint32_t k = *(volatile uint32_t*)(keys + h);
          if (k == kLsFree) {
            k = atomicCAS(keys + h, kLsFree, (uint32_t)v);
            made = k == kLsFree;
          }
          if (made || k == (uint32_t)v) return (int)h;
          h = h + 1 == (uint32_t)slots ? 0u : h + 1;
        }
      };
      // The words of this thread's tokens; each step is done for all of them before the next, so that their waits are one
      int at[kLsEarly + 2];
      uint32_t made = 0;
      bool m;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        at[kLsEarly + i] = -1;
        if (tid + i * kLsThreads < R.n_bias && (at[kLsEarly + i] = slot_of(early_bias[i], m)) >= 0) {
          // while the words hold nothing else: the last bias of a token is the largest
          atomicMax(word + at[kLsEarly + i], (uint32_t)(tid + i * kLsThreads + 1) << kLgBias);
          if (m) made |= 1u << (kLsEarly + i);
        }
      }
      if (R.n_bias > 0) __syncthreads();
      auto count = [&](int i, int w) {
        if (i < R.n_prompt) atomicOr(word + w, kLgSeen);
        else atomicAdd(word + w, 1u);
      };
#pragma unroll
      for (int i = 0; i < kLsEarly; ++i) {
        at[i] = -1;
        if (tid + i * kLsThreads < R.n_hist && (at[i] = slot_of(early[i], m)) >= 0) {
          count(tid + i * kLsThreads, at[i]);
          if (m) made |= 1u << i;
        }
      }
      for (int i = tid + kLsEarly * kLsThreads; i < R.n_hist; i += kLsThreads) {
        const int w = slot_of(hist[i], m);
        if (w >= 0) {
          count(i, w);
          if (m) found[atomicAdd(&n_found, 1)] = (uint16_t)w;
        }
      }
      // the slots that were made, side by side: few threads have many, and most of a warp would wait for the rules of one lane
      int before = __popc(made);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
      }
      int base = 0;
      if (lane == 31 && before > 0) base = atomicAdd(&n_found, before);
      base = __shfl_sync(0xffffffffu, base, 31) + before - __popc(made);
#pragma unroll
      for (int i = 0; i < kLsEarly + 2; ++i)
        if (made >> i & 1) found[base++] = (uint16_t)at[i];
      __syncthreads();
      const int n = n_found;
      constexpr int kAtOnce = 4;                              // loads of so many tokens are under way: the logits that stream past them are as well
      for (int i0 = tid; i0 < n; i0 += kAtOnce * kLsThreads) {
        int v[kAtOnce];
        uint32_t w[kAtOnce], ok[kAtOnce];
        T l[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          if (i0 + i * kLsThreads >= n) break;
          const int at = found[i0 + i * kLsThreads];
          v[i] = (int)keys[at];
          w[i] = word[at];
          l[i] = xr[v[i]];
          if (mask) ok[i] = (uint32_t)mask[v[i] >> 5];
        }
        if (!waited) pdl_wait();                              // these logits are read; what goes over them is written
        waited = true;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          if (i0 + i * kLsThreads >= n) break;
          float y = apply_word(to_f32<T>(l[i]), R, w[i], values);
          if (mask && !(ok[i] >> (v[i] & 31) & 1)) y = -INFINITY;
          if (!LAST) atomicOr(bits + (v[i] >> 5), 1u << (v[i] & 31));
          if (GREEDY) mine = max(mine, rank_of(y, v[i]));
          else out[(long long)b * ldo + v[i]] = y;
        }
      }
    }
    if (!LAST) __syncthreads();
    for (int i = tid; i < bit_words / 4; i += kLsThreads) reinterpret_cast<uint4*>(bitmap)[(long long)b * (bit_words / 4) + i] = reinterpret_cast<const uint4*>(bits)[i];
  }
  if (LAST) pdl_wait();                                       // threads that had nothing to write too: the call ends with its stream
  if (GREEDY) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((tid & 31) == 0) red[tid >> 5] = mine;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kLsThreads / 32; ++w) mine = max(mine, red[w]);
      best[(long long)b * (parts + 1) + parts] = mine;
    }
  }
}

// FIRST: nothing is settled yet
template <typename T, bool GREEDY, bool FIRST>
__global__ void __launch_bounds__(kLgThreads)
logits_stream_kernel(const T* x, long long ldx, int V, const LogitRules L, float* out, long long ldo, const RowPlan* plan, const uint32_t* bitmap, unsigned long long* __restrict__ best, int parts) {
  __shared__ uint32_t red[2][kLgThreads / 32];
  const int b = blockIdx.y, tid = threadIdx.x, v0 = blockIdx.x * kLgTokens + tid * 4;
  const T* xr = x + (long long)b * ldx;
  const bool whole_in = (reinterpret_cast<uintptr_t>(xr) & (4 * sizeof(T) - 1)) == 0;
  Quad<T> q[kLgQuads];
#pragma unroll
  for (int i = 0; i < kLgQuads; ++i) q[i] = load_quad<T>(xr + v0 + i * (kLgThreads * 4), V - v0 - i * (kLgThreads * 4), whole_in);
  if (GREEDY || FIRST) pdl_launch_dependents();
  RowPlan P = {1.f, 1.f, -1, 0};
  if (FIRST) {
    const int row = L.slot ? L.slot[b] : b;
    if ((unsigned)row < (unsigned)L.rows) {
      P.T = L.temperature[row];
      P.inv_T = __frcp_rn(P.T);
      if (L.mask && L.masked[row]) P.mask_row = row;
    }
  } else {
    pdl_wait();
    P = plan[b];
  }
  const uint32_t* known = bitmap + (long long)b * ((V + 127) / 128 * 4);
  uint32_t have[kLgQuads], allow[kLgQuads];
#pragma unroll
  for (int i = 0; i < kLgQuads; ++i) {
    const int v = v0 + i * (kLgThreads * 4);
    have[i] = !FIRST && P.settled && v < V ? known[v >> 5] >> (v & 31) & 15u : 0u;
    allow[i] = P.mask_row >= 0 && v < V ? (uint32_t)L.mask[(long long)P.mask_row * L.words + (v >> 5)] >> (v & 31) & 15u : 15u;
  }
#pragma unroll
  for (int i = 0; i < kLgQuads; ++i)
    if (!GREEDY) have[i] &= allow[i];                         // what is settled and masked is masked
  float* yr = GREEDY ? nullptr : out + (long long)b * ldo;
  const bool whole_out = !GREEDY && (reinterpret_cast<uintptr_t>(yr) & 15) == 0;
  float ys[GREEDY ? kLgQuads : 1][4];
  float most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kLgQuads; ++i) {
    const int v = v0 + i * (kLgThreads * 4), left = V - v;
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = q[i].at(e);
    if (P.T != 1.f) over_temperature(y, P.T, P.inv_T);
    if (P.mask_row >= 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!(allow[i] >> e & 1)) y[e] = -INFINITY;
    }
    if (GREEDY) {
      const uint32_t out_of_it = left >= 4 ? have[i] : have[i] | (left > 0 ? 0xfu << left : 0xfu);
      if (out_of_it) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (out_of_it >> e & 1) y[e] = -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) ys[GREEDY ? i : 0][e] = y[e];
      most = max_or_nan(most, max_or_nan(max_or_nan(y[0], y[1]), max_or_nan(y[2], y[3])));
    } else if (whole_out && left >= 4 && have[i] == 0) {
      *reinterpret_cast<float4*>(yr + v) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left && !(have[i] >> e & 1)) yr[v + e] = y[e];
    }
  }
  if (GREEDY) {
    const int warp = tid >> 5, lane = tid & 31;
    const uint32_t top = order_of(most), warp_top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[0][warp] = warp_top;
    __syncthreads();
    uint32_t all_top = 0;
#pragma unroll
    for (int w = 0; w < kLgThreads / 32; ++w) all_top = max(all_top, red[0][w]);
    unsigned at = 0xffffffffu;
    if (top == all_top) {                                     // the first of this thread's largest
#pragma unroll
      for (int i = kLgQuads - 1; i >= 0; --i)
#pragma unroll
        for (int e = 3; e >= 0; --e)
          if (order_of(ys[GREEDY ? i : 0][e]) == all_top) at = v0 + i * (kLgThreads * 4) + e;
    }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) red[1][warp] = at;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kLgThreads / 32; ++w) at = min(at, red[1][w]);
      best[(long long)b * (parts + 1) + blockIdx.x] = ((unsigned long long)all_top << 32) | (uint32_t)~at;
    }
  }
}

// Small batches: one kernel, a CTA for a slice of kLmTokens tokens of a row, its counts and biases in shared memory. Every slice goes through the whole history.
constexpr int kLmTokens = 4096, kLmSlices = 800;
template <typename T, bool GREEDY>
__global__ void __launch_bounds__(256)
logits_small_kernel(const T* x, long long ldx, int V, const LogitRules L, float* out, long long ldo, unsigned long long* __restrict__ best) {
  __shared__ uint32_t word[kLmTokens];
  __shared__ unsigned long long red[8];
  const int b = blockIdx.y, v0 = blockIdx.x * kLmTokens, nv = min(kLmTokens, V - v0), tid = threadIdx.x;
  const T* xr = x + (long long)b * ldx + v0;
  constexpr int kEach = kLmTokens / 256;
  T l[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (tid + i * 256 < nv) l[i] = xr[tid + i * 256];
  for (int i = tid; i < kLmTokens; i += 256) word[i] = 0;
  const int row = L.slot ? L.slot[b] : b;
  RowRules R = {1.f, 0.f, 0.f, 1.f, 1.f, 0, 0, 0, false};
  const long long r0 = (unsigned)row < (unsigned)L.rows ? row : 0;
  if ((unsigned)row < (unsigned)L.rows) R = row_rules(L, row);
  const float* values = L.bias_values + r0 * L.bias_width;
  const int* mask = R.masked ? L.mask + r0 * L.words + (v0 >> 5) : nullptr;
  if (R.n_hist > 0 || R.n_bias > 0) {
    __syncthreads();
    if (R.n_bias > 0) {                                       // while the words hold nothing else: the last bias of a token is the largest
      const int* ids = L.bias_ids + r0 * L.bias_width;
      for (int i = tid; i < R.n_bias; i += 256) {
        const int v = ids[i] - v0;
        if ((unsigned)v < (unsigned)nv) atomicMax(word + v, (uint32_t)(i + 1) << kLgBias);
      }
      __syncthreads();
    }
    const int* hist = L.tokens + r0 * L.width;
#pragma unroll 4
    for (int i = tid; i < R.n_hist; i += 256) {
      const int v = hist[i] - v0;
      if ((unsigned)v >= (unsigned)nv) continue;
      if (i < R.n_prompt) atomicOr(word + v, kLgSeen);
      else atomicAdd(word + v, 1u);
    }
  }
  __syncthreads();
  unsigned long long mine = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = tid + i * 256;
    if (at >= nv) break;
    float y = to_f32<T>(l[i]);
    const uint32_t w = word[at];
    y = w ? apply_word(y, R, w, values) : quotient(y, R.T, R.inv_T);
    if (mask && !(mask[at >> 5] >> (at & 31) & 1)) y = -INFINITY;
    if (GREEDY) mine = max(mine, rank_of(y, v0 + at));
    else out[(long long)b * ldo + v0 + at] = y;
  }
  if (GREEDY) {
    pdl_launch_dependents();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if ((tid & 31) == 0) red[tid >> 5] = mine;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < 8; ++w) mine = max(mine, red[w]);
      best[(long long)b * gridDim.x + blockIdx.x] = mine;
    }
  }
}

// The best token of each of a few rows: a cluster to a row, a CTA for an eighth of it, whose counts and biases are in shared memory as above. One launch instead of two,
// which is what a call of few rows waits for: 1 row of 151936, history of 900: 7.7 -> 8.9 us on the device, 14.4 -> 12.4 a call; vocabularies of 6400 5.5 -> 4.3 on the
// device, 8 rows of 32768 7.8 -> 5.7. 16 rows of 151936 10.7 -> 16.1: no more than eight.
constexpr int kLbCtas = 8, kLbThreads = 1024, kLbEach = 20, kLbRows = 8, kLbVocab = kLbCtas * (kLbThreads * kLbEach - 128);
template <typename T>
__global__ void __cluster_dims__(kLbCtas, 1, 1) __launch_bounds__(kLbThreads, 1)
logits_best_kernel(const T* x, long long ldx, int V, const LogitRules L, int per, long long* __restrict__ ids) {
  extern __shared__ __align__(16) uint32_t word_lb[];         // [per]
  __shared__ unsigned long long red[kLbThreads / 32], of_cta;
  const int b = blockIdx.y, v0 = blockIdx.x * per, nv = min(per, V - v0), tid = threadIdx.x;
  const T* xr = x + (long long)b * ldx + v0;
  T l[kLbEach];
#pragma unroll
  for (int i = 0; i < kLbEach; ++i)
    if (tid + i * kLbThreads < nv) l[i] = xr[tid + i * kLbThreads];
  const int row = L.slot ? L.slot[b] : b;
  RowRules R = {1.f, 0.f, 0.f, 1.f, 1.f, 0, 0, 0, false};
  const long long r0 = (unsigned)row < (unsigned)L.rows ? row : 0;
  if ((unsigned)row < (unsigned)L.rows) R = row_rules(L, row);
  const float* values = L.bias_values + r0 * L.bias_width;
  const int* mask = R.masked ? L.mask + r0 * L.words + (v0 >> 5) : nullptr;
  const bool tables = R.n_hist > 0 || R.n_bias > 0;
  if (tables) {
    for (int i = tid; i < per / 4; i += kLbThreads) reinterpret_cast<uint4*>(word_lb)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (R.n_bias > 0) {                                       // while the words hold nothing else: the last bias of a token is the largest
      const int* ids_b = L.bias_ids + r0 * L.bias_width;
      for (int i = tid; i < R.n_bias; i += kLbThreads) {
        const int v = ids_b[i] - v0;
        if (v >= 0 && v < nv) atomicMax(word_lb + v, (uint32_t)(i + 1) << kLgBias);
      }
      __syncthreads();
    }
    const int* hist = L.tokens + r0 * L.width;
#pragma unroll 4
    for (int i = tid; i < R.n_hist; i += kLbThreads) {
      const int v = hist[i] - v0;
      if (v < 0 || v >= nv) continue;
      if (i < R.n_prompt) atomicOr(word_lb + v, kLgSeen);
      else atomicAdd(word_lb + v, 1u);
    }
    __syncthreads();
  }
  unsigned long long mine = 0;
#pragma unroll
  for (int i = 0; i < kLbEach; ++i) {
    const int at = tid + i * kLbThreads;
    if (at >= nv) break;
    float y = to_f32<T>(l[i]);
    const uint32_t w = tables ? word_lb[at] : 0u;
    y = w ? apply_word(y, R, w, values) : quotient(y, R.T, R.inv_T);
    if (mask && !(mask[at >> 5] >> (at & 31) & 1)) y = -INFINITY;
    mine = max(mine, rank_of(y, v0 + at));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  if ((tid & 31) == 0) red[tid >> 5] = mine;
  __syncthreads();
  if (tid < 32) {
    mine = red[tid];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if (tid == 0) of_cta = mine;
  }
  cluster_sync_all();
  if (blockIdx.x == 0 && tid < 32) {
    unsigned long long r = 0;
    if (tid < kLbCtas) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(r) : "r"(mapa_shared(smem_u32(&of_cta), tid)) : "memory");
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) r = max(r, __shfl_xor_sync(0xffffffffu, r, o));
    if (tid == 0) ids[b] = (long long)(uint32_t)~(uint32_t)r;
  }
  cluster_sync_all();                                         // its shared memory has been read by the first
}

// the best of a row's CTAs: a warp to a row
__global__ void __launch_bounds__(128) greedy_pick_kernel(const unsigned long long* best, int parts, long long* __restrict__ ids, int B) {
  pdl_wait();
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= B) return;
  unsigned long long m = 0;
  for (int i = lane; i < parts; i += 32) m = max(m, best[(long long)b * parts + i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) ids[b] = (long long)(uint32_t)~(uint32_t)m;
}

// tokens that have come: behind the history of their rows; one that 32 bits do not hold is none of the vocabulary, and -1. A full row keeps what it has
__global__ void append_tokens_kernel(int* __restrict__ tokens, int rows, int width, int* __restrict__ length, const int* __restrict__ slot,
                                     const long long* __restrict__ ids, int n) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int s = slot ? slot[i] : i;
  if ((unsigned)s >= (unsigned)rows) return;
  const int at = length[s];
  if ((unsigned)at >= (unsigned)width) return;
  const long long id = ids[i];
  tokens[(long long)s * width + at] = id == (int)id ? (int)id : -1;
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

static int bitmap_words(int V) { return (V + 127) / 128 * 4; }
// the workspace: a plan for each row, a bitmap, for the greedy form the best of each of a row's CTAs and of its settled logits
static long long work_bytes(int B, int V, bool greedy) {
  return (long long)B * (sizeof(RowPlan) + bitmap_words(V) * 4ll + (greedy ? (ceil_div(V, kLgTokens) + 1) * 8ll : 0));
}

// whether a call is one kernel's: the greedy form's for few rows; the one of small batches (with one that picks, for the greedy form)
static bool few_rows(int B, int V) { return B <= kLbRows && V <= kLbVocab; }
static bool small_batch(int B, int V) { return (long long)B * ceil_div(V, kLmTokens) <= kLmSlices; }

template <typename T, bool GREEDY>
static int launch_logits_as(const void* x, long long ldx, int B, int V, const LogitRules& L, float* out, long long ldo, void* work, long long* ids, cudaStream_t st) {
  RowPlan* plan = (RowPlan*)work;
  uint32_t* bitmap = (uint32_t*)(plan + B);
  unsigned long long* best = GREEDY ? (unsigned long long*)(bitmap + (long long)B * bitmap_words(V)) : nullptr;
  const int parts = ceil_div(V, kLgTokens), slices = ceil_div(V, kLmTokens);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Up to so many slices one kernel is faster: 8 x 151936, histories of 1500: 7.2 us on the device against 9.6 (and a launch less for the host), 16 rows 8.2
  // against 11.1, 24 rows (912 slices) 12.4 against 13.8, but greedy 17.3 against 15.9; 48 rows 20.6 against 18.5, 128 with all rules 100 against 52
  if (GREEDY && few_rows(B, V)) {
    const int per = (ceil_div(V, kLbCtas) + 127) / 128 * 128;
    auto kern = logits_best_kernel<T>;
    // per call: the attribute belongs to the current device, and a process may use several
    if (per * 4 > 48 * 1024) B200_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, per * 4));
    kern<<<dim3(kLbCtas, B), kLbThreads, per * 4, st>>>((const T*)x, ldx, V, L, per, ids);
    B200_LAUNCH_CHECK();
    return 0;
  }
  if (small_batch(B, V)) {
    logits_small_kernel<T, GREEDY><<<dim3(slices, B), 256, 0, st>>>((const T*)x, ldx, V, L, out, ldo, best);
    B200_LAUNCH_CHECK();
    if (!GREEDY) return 0;
    cfg.gridDim = dim3(ceil_div(B, 4)); cfg.blockDim = dim3(128); cfg.stream = st;
    return (int)cudaLaunchKernelEx(&cfg, greedy_pick_kernel, (const unsigned long long*)best, slices, ids, B);
  }
  int slots = 256;                                            // no larger than twice what a row may hold
  while (slots < kLsSlots && slots / 2 < L.width + L.bias_width) slots *= 2;
  if (!GREEDY && x != out) {
    logits_stream_kernel<T, GREEDY, !GREEDY><<<dim3(parts, B), kLgThreads, 0, st>>>((const T*)x, ldx, V, L, out, ldo, nullptr, nullptr, nullptr, parts);
    B200_LAUNCH_CHECK();
    const size_t smem = (size_t)slots * 10;
    auto settle = logits_settle_kernel<T, GREEDY, !GREEDY>;
    // per call: the attribute belongs to the current device, and a process may use several
    if (smem > 48 * 1024) B200_CHECK(cudaFuncSetAttribute(settle, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cfg.gridDim = dim3(B); cfg.blockDim = dim3(kLsThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    return (int)cudaLaunchKernelEx(&cfg, settle, (const T*)x, ldx, V, L, out, ldo, (RowPlan*)nullptr, (uint32_t*)nullptr, (unsigned long long*)nullptr, parts, slots);
  }
  const size_t smem = (size_t)slots * 10 + bitmap_words(V) * 4;      // 224 KB at most
  auto settle = logits_settle_kernel<T, GREEDY, false>;
  // per call: the attribute belongs to the current device, and a process may use several
  if (smem > 48 * 1024) B200_CHECK(cudaFuncSetAttribute(settle, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  settle<<<B, kLsThreads, smem, st>>>((const T*)x, ldx, V, L, out, ldo, plan, bitmap, best, parts, slots);
  B200_LAUNCH_CHECK();
  cfg.gridDim = dim3(parts, B); cfg.blockDim = dim3(kLgThreads); cfg.stream = st;
  B200_CHECK(cudaLaunchKernelEx(&cfg, logits_stream_kernel<T, GREEDY, false>, (const T*)x, ldx, V, L, out, ldo, (const RowPlan*)plan, (const uint32_t*)bitmap, best, parts));
  if (!GREEDY) return 0;
  cfg.gridDim = dim3(ceil_div(B, 4)); cfg.blockDim = dim3(128);
  return (int)cudaLaunchKernelEx(&cfg, greedy_pick_kernel, (const unsigned long long*)best, parts + 1, ids, B);
}

template <bool GREEDY>
static int launch_logits(const void* x, long long ldx, int B, int V, const int* slot, const b200_logit_rules* rules, float* out, long long ldo,
                         void* work, long long* ids, int dtype, void* stream) {
  LogitRules L;
  if (int rc = logit_rules(rules, slot, L)) return rc;
  if (B < 0 || V < 1 || L.width > (int)kLgCount || L.bias_width >= 1 << (31 - kLgBias) || (L.mask && (long long)L.words * 32 < V)) return B200_ERR_BAD_SHAPE;
  if (V > kLgVocab || B > 65535) return B200_ERR_TOO_LARGE;
  if (B == 0) return 0;
  if (reinterpret_cast<uintptr_t>(work) & 15) return B200_ERR_BAD_ALIGN;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == B200_DT_FP32) return launch_logits_as<float, GREEDY>(x, ldx, B, V, L, out, ldo, work, ids, st);
  if (dtype == B200_DT_BF16) return launch_logits_as<__nv_bfloat16, GREEDY>(x, ldx, B, V, L, out, ldo, work, ids, st);
  if (dtype == B200_DT_FP16) return launch_logits_as<__half, GREEDY>(x, ldx, B, V, L, out, ldo, work, ids, st);
  return B200_ERR_UNSUPPORTED;
}

B200_API long long b200_logits_workspace(int B, int V, int greedy) { return B < 1 || V < 1 ? 0 : work_bytes(B, V, greedy != 0); }

B200_API int b200_logits_launches(int B, int V, int greedy) { return B < 1 || V < 1 ? 0 : greedy && few_rows(B, V) ? 1 : (small_batch(B, V) ? 1 : 2) + (greedy != 0); }

B200_API int b200_process_logits(const void* x, long long ldx, int B, int V, const int* slot, const b200_logit_rules* rules, void* workspace, float* out, long long ldo,
                                 int dtype, void* stream) {
  return launch_logits<false>(x, ldx, B, V, slot, rules, out, ldo, workspace, nullptr, dtype, stream);
}

B200_API int b200_greedy_tokens(const void* x, long long ldx, int B, int V, const int* slot, const b200_logit_rules* rules, void* workspace, long long* ids, int dtype,
                                void* stream) {
  return launch_logits<true>(x, ldx, B, V, slot, rules, nullptr, 0, workspace, ids, dtype, stream);
}

B200_API int b200_append_tokens(int* tokens, int rows, int width, int* length, const int* slot, const long long* ids, int n, void* stream) {
  if (n < 0 || rows < 0 || width < 0) return B200_ERR_BAD_SHAPE;
  if (n == 0) return 0;
  append_tokens_kernel<<<ceil_div(n, 128), 128, 0, (cudaStream_t)stream>>>(tokens, rows, width, length, slot, ids, n);
  B200_LAUNCH_CHECK();
  return 0;
}
