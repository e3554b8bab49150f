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
// All four are bound by HBM: every byte is read or written once. A thread has sixteen neighbours, two threads a block of 32.
// In bf16: 16384 x 4096, two added, are packed in 47 us and unpacked in 31 (7.2 and 6.6 TB/s); a gated unit of 8192 x 12288 takes 117 us and 129 (6.9 and 6.3 TB/s).
#include "common.cuh"
#include <initializer_list>
#include <type_traits>
#include "../include/b200_ops.h"

namespace b200 {

constexpr int kA8Threads = 256, kA8Each = 16;      // values of a thread: half a block

// Sixteen neighbours as they lie in memory, two of 16 bits to a word, by accesses of W bytes; what is not inside the row counts as zeros.
template <typename T> struct A8Raw { uint32_t w[kA8Each * sizeof(T) / 4]; };

template <typename T, int W>
__device__ __forceinline__ void a8_load(const T* __restrict__ p, int inside, A8Raw<T>& r) {
  constexpr int N = kA8Each * sizeof(T) / 4;
  if (inside >= kA8Each) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
    if constexpr (W == 32) {
#pragma unroll
      for (int i = 0; i < N; i += 8)
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]),
                     "=r"(r.w[i + 4]), "=r"(r.w[i + 5]), "=r"(r.w[i + 6]), "=r"(r.w[i + 7]) : "l"(q + i));
    } else if constexpr (W == 16) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(q + i));
        r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
      }
    } else if constexpr (W == 8) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(q + i));
        r.w[i] = v.x; r.w[i + 1] = v.y;
      }
    } else if constexpr (W == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) r.w[i] = __ldg(q + i);
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < N; ++i) r.w[i] = h[2 * i] | uint32_t(h[2 * i + 1]) << 16;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 4) r.w[i] = i < inside ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
      else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
        r.w[i] = (2 * i < inside ? h[2 * i] : 0u) | (2 * i + 1 < inside ? uint32_t(h[2 * i + 1]) << 16 : 0u);
      }
    }
  }
}

template <typename T, int W>
__device__ __forceinline__ void a8_store(T* __restrict__ p, int inside, const A8Raw<T>& r) {
  constexpr int N = kA8Each * sizeof(T) / 4;
  if (inside >= kA8Each) {
    uint32_t* q = reinterpret_cast<uint32_t*>(p);
    if constexpr (W == 32) {
#pragma unroll
      for (int i = 0; i < N; i += 8)
        asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" :: "r"(r.w[i]), "r"(r.w[i + 1]), "r"(r.w[i + 2]), "r"(r.w[i + 3]),
                     "r"(r.w[i + 4]), "r"(r.w[i + 5]), "r"(r.w[i + 6]), "r"(r.w[i + 7]), "l"(q + i) : "memory");
    } else if constexpr (W == 16) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<uint4*>(q + i) = make_uint4(r.w[i], r.w[i + 1], r.w[i + 2], r.w[i + 3]);
    } else if constexpr (W == 8) {
#pragma unroll
      for (int i = 0; i < N; i += 2) *reinterpret_cast<uint2*>(q + i) = make_uint2(r.w[i], r.w[i + 1]);
    } else if constexpr (W == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) q[i] = r.w[i];
    } else {
      uint16_t* h = reinterpret_cast<uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < N; ++i) { h[2 * i] = uint16_t(r.w[i]); h[2 * i + 1] = uint16_t(r.w[i] >> 16); }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (sizeof(T) == 4) { if (i < inside) reinterpret_cast<uint32_t*>(p)[i] = r.w[i]; }
      else {
        uint16_t* h = reinterpret_cast<uint16_t*>(p);
        if (2 * i < inside) h[2 * i] = uint16_t(r.w[i]);
        if (2 * i + 1 < inside) h[2 * i + 1] = uint16_t(r.w[i] >> 16);
      }
    }
  }
}

template <typename T> __device__ __forceinline__ float a8_at(const A8Raw<T>& r, int i);
template <> __device__ __forceinline__ float a8_at<float>(const A8Raw<float>& r, int i) { return __uint_as_float(r.w[i]); }
template <> __device__ __forceinline__ float a8_at<__nv_bfloat16>(const A8Raw<__nv_bfloat16>& r, int i) {
  return __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
}
template <> __device__ __forceinline__ float a8_at<__half>(const A8Raw<__half>& r, int i) {
  return __half2float(__ushort_as_half(uint16_t(i & 1 ? r.w[i / 2] >> 16 : r.w[i / 2])));
}
// values 2 i and 2 i + 1, rounded
template <typename T> __device__ __forceinline__ void a8_set(A8Raw<T>& r, int i, float a, float b);
template <> __device__ __forceinline__ void a8_set<float>(A8Raw<float>& r, int i, float a, float b) { r.w[2 * i] = __float_as_uint(a); r.w[2 * i + 1] = __float_as_uint(b); }
template <> __device__ __forceinline__ void a8_set<__nv_bfloat16>(A8Raw<__nv_bfloat16>& r, int i, float a, float b) { r.w[i] = pack_bf16x2(a, b); }
template <> __device__ __forceinline__ void a8_set<__half>(A8Raw<__half>& r, int i, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  r.w[i] = *reinterpret_cast<const uint32_t*>(&h);
}
// r + a, rounded to the type: the stream is rounded where a model adds it. (A sum of two 16-bit numbers that 32 bits do not hold lies too close to the
// larger one for the order of roundings to matter, so the packed sum has the bits of one in 32 bits.)
template <typename T> __device__ __forceinline__ void a8_add(A8Raw<T>& r, const A8Raw<T>& a) {
#pragma unroll
  for (int i = 0; i < int(sizeof(r.w) / 4); ++i) {
    if constexpr (sizeof(T) == 4) r.w[i] = __float_as_uint(__uint_as_float(r.w[i]) + __uint_as_float(a.w[i]));
    else if constexpr (std::is_same<T, __half>::value) {
      const __half2 s = __hadd2(*reinterpret_cast<const __half2*>(&r.w[i]), *reinterpret_cast<const __half2*>(&a.w[i]));
      r.w[i] = *reinterpret_cast<const uint32_t*>(&s);
    } else {
      const __nv_bfloat162 s = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&r.w[i]), *reinterpret_cast<const __nv_bfloat162*>(&a.w[i]));
      r.w[i] = *reinterpret_cast<const uint32_t*>(&s);
    }
  }
}

// The largest byte e + 127 of a type.
template <typename T> __device__ __forceinline__ constexpr int a8_top() { return std::is_same<T, __half>::value ? 9 + 127 : 121 + 127; }

// The power of two of a block, of which this thread has half and the neighbouring lane the other: its byte, 2^-e, and whether all values are finite
// and no e was cut. All lanes of the warp call it.
struct A8Scale { int eb; float inv; bool plain; };
template <typename T>
__device__ __forceinline__ A8Scale a8_scale(const A8Raw<T>& r) {
  constexpr int TOP = a8_top<T>();
  uint32_t most = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < kA8Each; ++i) most = max(most, r.w[i] & 0x7fffffffu);
  } else {
#pragma unroll
    for (int i = 0; i < kA8Each / 2; ++i) most = __vmaxu2(most, r.w[i] & 0x7fff7fffu);
    most = max(most & 0xffffu, most >> 16);
  }
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  A8Scale s;
  if constexpr (std::is_same<T, __half>::value) {
    s.plain = most < 0x7c00u;
    most = __float_as_uint(__half2float(__ushort_as_half(uint16_t(most))));
  } else {
    if constexpr (sizeof(T) == 2) most <<= 16;
    s.plain = most < 0x7f800000u;
  }
  // max = 2^(E - 127) * 1.f: 128 * 2^-1 * 1.f is below 127.5 unless the first seven bits of f are all ones
  s.eb = int(most >> 23) - 6 + ((most & 0x7f0000u) == 0x7f0000u);
  s.plain = s.plain && s.eb <= TOP;
  if (!s.plain) {
    uint32_t fin = 0;                                            // the largest finite magnitude
#pragma unroll
    for (int i = 0; i < kA8Each; ++i) {
      const uint32_t a = __float_as_uint(a8_at<T>(r, i)) & 0x7fffffffu;
      fin = max(fin, a < 0x7f800000u ? a : 0u);
    }
    fin = max(fin, __shfl_xor_sync(3u << (threadIdx.x & 30), fin, 1));      // both lanes of a block come here
    s.eb = min(int(fin >> 23) - 6 + ((fin & 0x7f0000u) == 0x7f0000u), TOP);
  }
  s.eb = max(s.eb, 0);
  s.inv = __uint_as_float(uint32_t(254 - s.eb) << 23);
  return s;
}
// Four values as bytes. Plain ones: q is the low byte of x 2^-e + 1.5 (2^23), one operation that rounds as rint does (with conversions, tests
// for infinities and bounds for each value pack8 took 84 us of 16384 x 4096 + 16384 x 4096, bound by its instructions; now 46).
template <bool PLAIN>
__device__ __forceinline__ uint32_t a8_bytes(float a, float b, float c, float d, float inv) {
  auto q = [&](float v) -> uint32_t {
    if constexpr (PLAIN) return __float_as_uint(fmaf(v, inv, 12582912.f));
    else return uint32_t((__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u ? min(max(__float2int_rn(v * inv), -127), 127) : -128);
  };
  return __byte_perm(__byte_perm(q(a), q(b), 0x0040), __byte_perm(q(c), q(d), 0x0040), 0x5410);
}
template <typename T, bool PLAIN>
__device__ __forceinline__ uint4 a8_encode(const A8Raw<T>& r, float inv) {
  uint4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    (&o.x)[i] = a8_bytes<PLAIN>(a8_at<T>(r, 4 * i), a8_at<T>(r, 4 * i + 1), a8_at<T>(r, 4 * i + 2), a8_at<T>(r, 4 * i + 3), inv);
  return o;
}

// q + 128 as the low byte of 2^23 is a number whose difference to 2^23 + 128 is q: times 2^e, one operation without a rounding.
__device__ __forceinline__ void a8_decode(uint4 r, int eb, float (&v)[kA8Each]) {
  const uint32_t w[4] = {r.x ^ 0x80808080u, r.y ^ 0x80808080u, r.z ^ 0x80808080u, r.w ^ 0x80808080u};
  uint32_t zero = 0;                                             // bit 7 of a word's lowest byte that is zero (q = -128)
#pragma unroll
  for (int i = 0; i < 4; ++i) zero |= (w[i] - 0x01010101u) & ~w[i] & 0x80808080u;
  const float scale = __uint_as_float(eb > 0 ? uint32_t(eb) << 23 : 0x00400000u);
  if (!zero && eb <= 127 + 100) {
    const float off = -8388736.f * scale;
#pragma unroll
    for (int i = 0; i < kA8Each; ++i) v[i] = fmaf(__uint_as_float(__byte_perm(w[i / 4], 0x4b000000u, 0x7440 + (i & 3))), scale, off);
  } else {
#pragma unroll
    for (int i = 0; i < kA8Each; ++i) {
      const float q = __uint_as_float(__byte_perm(w[i / 4], 0x4b000000u, 0x7440 + (i & 3))) - 8388736.f;
      v[i] = q == -128.f ? __uint_as_float(0x7fffffffu) : q * scale;
    }
  }
}

// Where a thread's sixteen values are: row, first column and the block's number in the row. `n` threads have some; the rest of the last warp
// goes along with row -1.
struct A8At { long long row; int col, blk; };
__device__ __forceinline__ A8At a8_at(unsigned n, unsigned per_row) {
  const unsigned i = blockIdx.x * kA8Threads + threadIdx.x;
  if (i >= n) return {-1, 0, 0};
  const unsigned row = i / per_row, at = i - row * per_row;
  return {row, int(at * kA8Each), int(at >> 1)};
}

template <typename T, int W, bool ADD>
__global__ void __launch_bounds__(kA8Threads)
pack8_kernel(const T* __restrict__ x, long long x_rs, const T* __restrict__ add, long long add_rs, uint8_t* __restrict__ q,
             uint8_t* __restrict__ e, unsigned n, int D, int nb) {
  const A8At at = a8_at(n, nb * 2);
  const int inside = at.row < 0 ? 0 : D - at.col;
  A8Raw<T> v, a;
  a8_load<T, W>(x + max(at.row, 0ll) * x_rs + at.col, inside, v);
  if constexpr (ADD) {
    a8_load<T, W>(add + max(at.row, 0ll) * add_rs + at.col, inside, a);
    a8_add<T>(v, a);
  }
  const A8Scale s = a8_scale<T>(v);
  if (at.row < 0) return;
  *reinterpret_cast<uint4*>(q + (at.row * nb * 32 + at.col)) = s.plain ? a8_encode<T, true>(v, s.inv) : a8_encode<T, false>(v, s.inv);
  if ((threadIdx.x & 1) == 0) e[at.row * nb + at.blk] = uint8_t(s.eb);
}

template <typename T, int W>
__global__ void __launch_bounds__(kA8Threads)
unpack8_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, T* __restrict__ y, unsigned n, int D, int nb) {
  const A8At at = a8_at(n, nb * 2);
  if (at.row < 0 || at.col >= D) return;
  float v[kA8Each];
  a8_decode(__ldg(reinterpret_cast<const uint4*>(q + (at.row * nb * 32 + at.col))), e[at.row * nb + at.blk], v);
  A8Raw<T> o;
#pragma unroll
  for (int i = 0; i < kA8Each / 2; ++i) a8_set<T>(o, i, v[2 * i], v[2 * i + 1]);
  a8_store<T, W>(y + at.row * D + at.col, D - at.col, o);
}

// 1 / (1 + e^-g): rounded to about the last bit in fp32, by the fast exponential and reciprocal where 16 bits are kept.
template <typename T> __device__ __forceinline__ float a8_sigmoid(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }
template <> __device__ __forceinline__ float a8_sigmoid<float>(float g) { return 1.f / (1.f + expf(-g)); }

// Four columns at a time from here on: what a value needs is unpacked once and nothing of sixteen values but the operands and results is held.
template <typename T, bool PLAIN>
__device__ __forceinline__ void swiglu8_row(const A8Raw<T>& g, const A8Raw<T>& u, float gi, float ui, A8Raw<T>& o, uint4& gq, uint4& uq) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a[4], b[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = a8_at<T>(g, 4 * i + j);
      b[j] = a8_at<T>(u, 4 * i + j);
      y[j] = a[j] * a8_sigmoid<T>(a[j]) * b[j];
    }
    a8_set<T>(o, 2 * i, y[0], y[1]);
    a8_set<T>(o, 2 * i + 1, y[2], y[3]);
    (&gq.x)[i] = a8_bytes<PLAIN>(a[0], a[1], a[2], a[3], gi);
    (&uq.x)[i] = a8_bytes<PLAIN>(b[0], b[1], b[2], b[3], ui);
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(kA8Threads)
swiglu8_fwd_kernel(const T* __restrict__ gu, long long rs, T* __restrict__ y, uint8_t* __restrict__ q, uint8_t* __restrict__ e, unsigned n,
                   int F, int nb) {
  const A8At at = a8_at(n, nb * 2);
  const int inside = at.row < 0 ? 0 : F - at.col;
  A8Raw<T> g, u, o;
  const T* row = gu + max(at.row, 0ll) * rs + at.col;
  a8_load<T, W>(row, inside, g);
  a8_load<T, W>(row + F, inside, u);
  uint4 gq, uq;
  const A8Scale gs = a8_scale<T>(g), us = a8_scale<T>(u);
  if (gs.plain && us.plain) swiglu8_row<T, true>(g, u, gs.inv, us.inv, o, gq, uq);
  else swiglu8_row<T, false>(g, u, gs.inv, us.inv, o, gq, uq);
  if (inside > 0) a8_store<T, W>(y + at.row * F + at.col, inside, o);
  if (q == nullptr || at.row < 0) return;                          // nobody asks for a gradient
  uint8_t* qr = q + (at.row * 2 * nb * 32 + at.col);
  *reinterpret_cast<uint4*>(qr) = gq;
  *reinterpret_cast<uint4*>(qr + nb * 32) = uq;
  if ((threadIdx.x & 1) == 0) {
    e[at.row * 2 * nb + at.blk] = uint8_t(gs.eb);
    e[at.row * 2 * nb + nb + at.blk] = uint8_t(us.eb);
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(kA8Threads)
swiglu8_bwd_kernel(const T* __restrict__ dy, const uint8_t* __restrict__ q, const uint8_t* __restrict__ e, T* __restrict__ dgu, unsigned n,
                   int F, int nb) {
  const A8At at = a8_at(n, nb * 2);
  if (at.row < 0 || at.col >= F) return;
  const int inside = F - at.col;
  A8Raw<T> d, dg, du;
  float g[kA8Each], u[kA8Each];
  const uint8_t* qr = q + (at.row * 2 * nb * 32 + at.col);
  const uint4 gq = __ldg(reinterpret_cast<const uint4*>(qr)), uq = __ldg(reinterpret_cast<const uint4*>(qr + nb * 32));
  const int ge = e[at.row * 2 * nb + at.blk], ue = e[at.row * 2 * nb + nb + at.blk];
  a8_load<T, W>(dy + at.row * F + at.col, inside, d);
  a8_decode(gq, ge, g);
  a8_decode(uq, ue, u);
#pragma unroll
  for (int i = 0; i < kA8Each; ++i) {
    const float s = a8_sigmoid<T>(g[i]), ds = a8_at<T>(d, i) * s, gi = g[i];
    g[i] = ds * u[i] * fmaf(gi, 1.f - s, 1.f);
    u[i] = ds * gi;
  }
#pragma unroll
  for (int i = 0; i < kA8Each / 2; ++i) {
    a8_set<T>(dg, i, g[2 * i], g[2 * i + 1]);
    a8_set<T>(du, i, u[2 * i], u[2 * i + 1]);
  }
  T* o = dgu + at.row * 2 * F + at.col;
  a8_store<T, W>(o, inside, dg);
  a8_store<T, W>(o + F, inside, du);
}

// The widest access, up to 32 bytes, that all of these addresses and strides (in bytes) allow.
static int a8_width(std::initializer_list<unsigned long long> all, int es) {
  unsigned long long m = 32;
  for (unsigned long long a : all) m |= a;
  const int w = int(m & -m);
  return w < es ? es : w;
}

// Calls f(first row, rows) for pieces of the rows whose threads a 32-bit number counts.
template <typename F> static void a8_pieces(long long rows, int nb, F f) {
  const long long most = ((1ll << 31) - kA8Threads) / (2ll * nb);
  for (long long r = 0; r < rows; r += most) f(r, rows - r < most ? rows - r : most);
}
static unsigned a8_grid(unsigned n) { return (n + kA8Threads - 1) / kA8Threads; }

}  // namespace b200
using namespace b200;

#define A8_WIDTHS(T, width, ...)                                                    \
  switch (width) {                                                                  \
    case 32: { constexpr int W = 32; __VA_ARGS__; } break;                           \
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
  if (a8_addr(q) % 16) return B200_ERR_BAD_ALIGN;
  const int nb = (D + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = add ? a8_width({a8_addr(x), a8_addr(add), (unsigned long long)x_rs * es, (unsigned long long)add_rs * es}, es)
                        : a8_width({a8_addr(x), (unsigned long long)x_rs * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 2);
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
  if (a8_addr(q) % 16) return B200_ERR_BAD_ALIGN;
  const int nb = (D + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = a8_width({a8_addr(y), (unsigned long long)D * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 2);
    unpack8_kernel<T, W><<<a8_grid(n), kA8Threads, 0, st>>>((const uint8_t*)q + r * nb * 32, (const uint8_t*)e + r * nb, (T*)y + r * D, n, D, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_swiglu8_fwd(const void* gu, long long rs, void* y, void* q, void* e, long long rows, int F, int dtype, void* stream) {
  if (a8_bad(rows, F)) return B200_ERR_BAD_SHAPE;
  if (a8_addr(q) % 16) return B200_ERR_BAD_ALIGN;
  const int nb = (F + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = a8_width({a8_addr(gu), a8_addr(y), (unsigned long long)rs * es, (unsigned long long)F * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 2);
    swiglu8_fwd_kernel<T, W><<<a8_grid(n), kA8Threads, 0, st>>>((const T*)gu + r * rs, rs, (T*)y + r * F, q ? (uint8_t*)q + r * 2 * nb * 32 : nullptr,
                                                                q ? (uint8_t*)e + r * 2 * nb : nullptr, n, F, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}

B200_API int b200_swiglu8_bwd(const void* dy, const void* q, const void* e, void* dgu, long long rows, int F, int dtype, void* stream) {
  if (a8_bad(rows, F)) return B200_ERR_BAD_SHAPE;
  if (a8_addr(q) % 16) return B200_ERR_BAD_ALIGN;
  const int nb = (F + 31) / 32, es = dtype == B200_DT_FP32 ? 4 : 2;
  const int width = a8_width({a8_addr(dy), a8_addr(dgu), (unsigned long long)F * es}, es);
  cudaStream_t st = (cudaStream_t)stream;
  A8_TYPES(dtype, A8_WIDTHS(T, width, a8_pieces(rows, nb, [&](long long r, long long m) {
    const unsigned n = unsigned(m * nb * 2);
    swiglu8_bwd_kernel<T, W><<<a8_grid(n), kA8Threads, 0, st>>>((const T*)dy + r * F, (const uint8_t*)q + r * 2 * nb * 32,
                                                                (const uint8_t*)e + r * 2 * nb, (T*)dgu + r * 2 * F, n, F, nb);
  })));
  B200_LAUNCH_CHECK();
  return 0;
}
