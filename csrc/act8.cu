// Activations in 8 bits: what a layer keeps between its forward and its backward pass, at half of 16 bits' room or a quarter of 32's.
//
// 32 neighbours of a row share a power of two 2^e, the least under which all of them are below 127.5; a value is then a whole number of
// it, rounded to the nearest (ties to even):
//     e = min { e : max |x| 2^-e < 127.5 },  q = rint(x 2^-e),  x' = q 2^e,  |x' - x| <= 2^(e - 1) <= max |x| / 127
// (the quotient by a power of two is exact, so the same x gives the same q everywhere). Infinities and NaN do not count for e; they are
// kept as q = -128 and come back as NaN, and leave their neighbours alone. e is held as the byte e + 127, and no larger than that 127 * 2^e is
// still a number of the type (9 in fp16, 121 otherwise), where the largest values are cut to it.
//
//   pack8        q and e of x, or of x + add rounded to the type (what a residual stream's next norm would read)
//   unpack8      x' in the type asked for
//   swiglu8_fwd  y = silu(g) u of a row [g | u], and g and u in 8 bits, in one pass
//   swiglu8_bwd  dg = dy u s(g) (1 + g (1 - s(g))), du = dy silu(g) at the g and u that were kept
//
// All four are bound by HBM: every byte is read or written once. A thread has eight neighbours, four threads a block of 32, whose largest
// they find by two shuffles.
#include "common.cuh"
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kA8Threads = 256;

// Eight neighbours as fp32, by accesses of W bytes; what is not inside the row counts as zeros.
template <typename T, int W>
__device__ __forceinline__ void a8_load(const T* __restrict__ p, int inside, float (&v)[8]) {
  constexpr int N = W / sizeof(T);
  if (inside >= 8) {
    alignas(16) T raw[8];
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      if constexpr (W == 16) *reinterpret_cast<uint4*>(raw + i) = __ldg(reinterpret_cast<const uint4*>(p + i));
      else if constexpr (W == 8) *reinterpret_cast<uint2*>(raw + i) = __ldg(reinterpret_cast<const uint2*>(p + i));
      else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(raw + i) = __ldg(reinterpret_cast<const uint32_t*>(p + i));
      else raw[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < inside ? to_f32<T>(p[i]) : 0.f;
  }
}

template <typename T, int W>
__device__ __forceinline__ void a8_store(T* __restrict__ p, int inside, const float (&v)[8]) {
  constexpr int N = W / sizeof(T);
  alignas(16) T raw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) raw[i] = from_f32<T>(v[i]);
  if (inside >= 8) {
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      if constexpr (W == 16) *reinterpret_cast<uint4*>(p + i) = *reinterpret_cast<uint4*>(raw + i);
      else if constexpr (W == 8) *reinterpret_cast<uint2*>(p + i) = *reinterpret_cast<uint2*>(raw + i);
      else if constexpr (W == 4) *reinterpret_cast<uint32_t*>(p + i) = *reinterpret_cast<uint32_t*>(raw + i);
      else p[i] = raw[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < inside) p[i] = raw[i];
  }
}

// The largest byte e + 127 of a type.
template <typename T> __device__ __forceinline__ constexpr int a8_top() { return 121 + 127; }
template <> __device__ __forceinline__ constexpr int a8_top<__half>() { return 9 + 127; }

// Eight values of a block whose other 24 are with the three neighbouring lanes: their q as eight bytes, and the block's byte of e.
// All lanes of the warp call it.
template <int TOP>
__device__ __forceinline__ uint2 a8_encode(const float (&v)[8], int& eb) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __float_as_uint(v[i]) & 0x7fffffffu;
    most = max(most, a < 0x7f800000u ? a : 0u);
  }
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  // max = 2^(E - 127) * 1.f: 128 * 2^-1 * 1.f is below 127.5 unless the first seven bits of f are all ones
  eb = min(max(int(most >> 23) - 6 + ((most & 0x7f0000u) == 0x7f0000u), 0), TOP);
  const float inv = __uint_as_float(uint32_t(254 - eb) << 23);
  int q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool finite = (__float_as_uint(v[i]) & 0x7fffffffu) < 0x7f800000u;
    q[i] = finite ? min(max(__float2int_rn(v[i] * inv), -127), 127) : -128;
  }
  uint2 r;
  r.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  r.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return r;
}

__device__ __forceinline__ void a8_decode(uint2 r, int eb, float (&v)[8]) {
  const float scale = __uint_as_float(eb > 0 ? uint32_t(eb) << 23 : 0x00400000u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = (i < 4 ? r.x : r.y) ^ 0x80808080u;           // q + 128, into the low byte of 2^23: its difference to 2^23 + 128 is q
    const float q = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + (i & 3))) - 8388736.f;
    v[i] = q == -128.f ? __uint_as_float(0x7fffffffu) : q * scale;
  }
}

// Where a thread's eight values are: row, first column and the block's number in the row. `n` threads have some; the rest of the last warp
// goes along with row -1.
struct A8At { long long row; int col, blk; };
__device__ __forceinline__ A8At a8_at(unsigned n, unsigned per_row) {
  const unsigned i = blockIdx.x * kA8Threads + threadIdx.x;
  if (i >= n) return {-1, 0, 0};
  const unsigned row = i / per_row, at = i - row * per_row;
  return {row, int(at * 8), int(at >> 2)};
}

template <typename T, int W, bool ADD>
__global__ void __launch_bounds__(kA8Threads)
pack8_kernel(const T* __restrict__ x, long long x_rs, const T* __restrict__ add, long long add_rs, uint8_t* __restrict__ q,
             uint8_t* __restrict__ e, unsigned n, int D, int nb) {
  const A8At at = a8_at(n, nb * 4);
  const int inside = at.row < 0 ? 0 : D - at.col;
  float v[8];
  a8_load<T, W>(x + max(at.row, 0ll) * x_rs + at.col, inside, v);
  if constexpr (ADD) {
    float a[8];
    a8_load<T, W>(add + max(at.row, 0ll) * add_rs + at.col, inside, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(from_f32<T>(v[i] + a[i]));      // the stream is rounded where a model adds it
  }
  int eb;
  const uint2 r = a8_encode<a8_top<T>()>(v, eb);
  if (at.row < 0) return;
  *reinterpret_cast<uint2*>(q + (at.row * nb * 32 + at.col)) = r;
  if ((threadIdx.x & 3) == 0) e[at.row * nb + at.blk] = uint8_t(eb);
}

template <typename T, int W>
__global__ void __launch_bounds__(kA8Threads)
unpack8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, T* __restrict__ y, unsigned n, int D, int nb) {
  const A8At at = a8_at(n, nb * 4);
  if (at.row < 0 || at.col >= D) return;
  float v[8];
  a8_decode(__ldg(reinterpret_cast<const uint2*>(q + (at.row * nb * 32 + at.col))), e[at.row * nb + at.blk], v);
  a8_store<T, W>(y + at.row * D + at.col, D - at.col, v);
}

// 1 / (1 + e^-g): rounded to about the last bit in fp32, by the fast exponential and reciprocal where 16 bits are kept.
template <typename T> __device__ __forceinline__ float a8_sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }
template <> __device__ __forceinline__ float a8_sigmoid<float>(float g) { return 1.f / (1.f + expf(-g)); }

template <typename T, int W>
__global__ void __launch_bounds__(kA8Threads)
swiglu8_fwd_kernel(const T* __restrict__ gu, long long rs, T* __restrict__ y, uint8_t* __restrict__ q, uint8_t* __restrict__ e, unsigned n,
                   int F, int nb) {
  const A8At at = a8_at(n, nb * 4);
  const int inside = at.row < 0 ? 0 : F - at.col;
  float g[8], u[8], o[8];
  const T* row = gu + max(at.row, 0ll) * rs + at.col;
  a8_load<T, W>(row, inside, g);
  a8_load<T, W>(row + F, inside, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = g[i] * a8_sigmoid<T>(g[i]) * u[i];
  if (inside > 0) a8_store<T, W>(y + at.row * F + at.col, inside, o);
  if (q == nullptr) return;                                        // nobody asks for a gradient
  int ge, ue;
  const uint2 gq = a8_encode<a8_top<T>()>(g, ge), uq = a8_encode<a8_top<T>()>(u, ue);
  if (at.row < 0) return;
  uint8_t* qr = q + (at.row * 2 * nb * 32 + at.col);
  *reinterpret_cast<uint2*>(qr) = gq;
  *reinterpret_cast<uint2*>(qr + nb * 32) = uq;
  if ((threadIdx.x & 3) == 0) {
    e[at.row * 2 * nb + at.blk] = uint8_t(ge);
    e[at.row * 2 * nb + nb + at.blk] = uint8_t(ue);
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(kA8Threads)
swiglu8_bwd_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, T* __restrict__ dgu, unsigned n,
                   int F, int nb) {
  const A8At at = a8_at(n, nb * 4);
  if (at.row < 0 || at.col >= F) return;
  const int inside = F - at.col;
  float d[8], g[8], u[8];
  const uint8_t* qr = q + (at.row * 2 * nb * 32 + at.col);
  const uint2 gq = __ldg(reinterpret_cast<const uint2*>(qr)), uq = __ldg(reinterpret_cast<const uint2*>(qr + nb * 32));
  const int ge = e[at.row * 2 * nb + at.blk], ue = e[at.row * 2 * nb + nb + at.blk];
  a8_load<T, W>(dy + at.row * F + at.col, inside, d);
  a8_decode(gq, ge, g);
  a8_decode(uq, ue, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float s = a8_sigmoid<T>(g[i]), ds = d[i] * s, gi = g[i];
    g[i] = ds * u[i] * (1.f + gi * (1.f - s));
    u[i] = ds * gi;
  }
  T* o = dgu + at.row * 2 * F + at.col;
  a8_store<T, W>(o, inside, g);
  a8_store<T, W>(o + F, inside, u);
}

// The widest access, up to 16 bytes, that all of these addresses and strides (in bytes) allow.
static int a8_width(std::initializer_list<unsigned long long> all, int es) {
  unsigned long long m = 16;
  for (unsigned long long a : all) m |= a;
  const int w = int(m & -m);
  return w > 16 ? 16 : (w < es ? es : w);
}

// Calls f(first row, rows) for pieces of the rows whose threads a 32-bit number counts.
template <typename F> static void a8_pieces(long long rows, int nb, F f) {
  const long long most = ((1ll << 31) - kA8Threads) / (4ll * nb);
  for (long long r = 0; r < rows; r += most) f(r, rows - r < most ? rows - r : most);
}
static unsigned a8_grid(unsigned n) { return (n + kA8Threads - 1) / kA8Threads; }

}  // namespace b200
using namespace b200;

#define A8_WIDTHS(T, width, ...)                                                    \
  switch (width) {                                                                  \
    case 16: { constexpr int W = 16; __VA_ARGS__; } break;                           \
    case 8: { constexpr int W = 8; __VA_ARGS__; } break;                             \
    case 4: { constexpr int W = 4; __VA_ARGS__; } break;                             \
    default: { constexpr int W = sizeof(T); __VA_ARGS__; } break;                    \
  }
#define A8_TYPES(dtype, ...)                                                        \
  if (dtype == B200_DT_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }               \
  else if (dtype == B200_DT_FP16) { using T = __half; __VA_ARGS__; }                 \
  else if (dtype == B200_DT_FP32) { using T = float; __VA_ARGS__; }                  \
  else return B200_ERR_UNSUPPORTED;

static bool a8_bad(long long rows, int D) { return rows < 0 || D <= 0 || D > (1 << 28); }
static unsigned long long a8_addr(const void* p) { return (unsigned long long)p; }

B200_API int b200_pack8(const void* x, long long x_rs, const void* add, long long add_rs, void* q, void* e, long long rows, int D, int dtype,
                        void* stream) {
  if (a8_bad(rows, D)) return B200_ERR_BAD_SHAPE;
  if (a8_addr(q) % 8) return B200_ERR_BAD_ALIGN;
  const int nb = (D + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = add ? a8_width({a8_addr(x), a8_addr(add), (unsigned long long)x_rs * es, (unsigned long long)add_rs * es}, es)
                        : a8_width({a8_addr(x), (unsigned long long)x_rs * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 4);
    const T* xr = (const T*)x + r * x_rs;
    uint8_t *qr = (uint8_t*)q + r * nb * 32, *er = (uint8_t*)e + r * nb;
    if (add) pack8_kernel<T, W, true><<<a8_grid(n), kA8Threads, 0, st>>>(xr, x_rs, (const T*)add + r * add_rs, add_rs, qr, er, n, D, nb);
    else pack8_kernel<T, W, false><<<a8_grid(n), kA8Threads, 0, st>>>(xr, x_rs, nullptr, 0, qr, er, n, D, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_unpack8(const void* q, const void* e, void* y, long long rows, int D, int dtype, void* stream) {
  if (a8_bad(rows, D)) return B200_ERR_BAD_SHAPE;
  if (a8_addr(q) % 8) return B200_ERR_BAD_ALIGN;
  const int nb = (D + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = a8_width({a8_addr(y), (unsigned long long)D * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 4);
    unpack8_kernel<T, W><<<a8_grid(n), kA8Threads, 0, st>>>((const uint8_t*)q + r * nb * 32, (const uint8_t*)e + r * nb, (T*)y + r * D, n, D, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_swiglu8_fwd(const void* gu, long long rs, void* y, void* q, void* e, long long rows, int F, int dtype, void* stream) {
  if (a8_bad(rows, F)) return B200_ERR_BAD_SHAPE;
  if (a8_addr(q) % 8) return B200_ERR_BAD_ALIGN;
  const int nb = (F + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = a8_width({a8_addr(gu), a8_addr(y), (unsigned long long)rs * es, (unsigned long long)F * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 4);
    swiglu8_fwd_kernel<T, W><<<a8_grid(n), kA8Threads, 0, st>>>((const T*)gu + r * rs, rs, (T*)y + r * F, q ? (uint8_t*)q + r * 2 * nb * 32 : nullptr,
                                                                q ? (uint8_t*)e + r * 2 * nb : nullptr, n, F, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_swiglu8_bwd(const void* dy, const void* q, const void* e, void* dgu, long long rows, int F, int dtype, void* stream) {
  if (a8_bad(rows, F)) return B200_ERR_BAD_SHAPE;
  if (a8_addr(q) % 8) return B200_ERR_BAD_ALIGN;
  const int nb = (F + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = a8_width({a8_addr(dy), a8_addr(dgu), (unsigned long long)F * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 4);
    swiglu8_bwd_kernel<T, W><<<a8_grid(n), kA8Threads, 0, st>>>((const T*)dy + r * F, (const uint8_t*)q + r * 2 * nb * 32,
                                                                (const uint8_t*)e + r * 2 * nb, (T*)dgu + r * 2 * F, n, F, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}
