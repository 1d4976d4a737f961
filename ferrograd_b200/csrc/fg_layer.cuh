// The linear layer with a fused epilogue, its gradient and dropout: element
// types, activations, the counter-based dropout mask and the epilogue that
// every kernel of the layer applies (fg_layer.cu, fg_layer_gemm.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fg_internal.h"

namespace fg {
namespace layer {

// ---- element types: f32, bf16 and f16 in memory, f32 in registers ---------
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&p);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  __half2 p = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t *>(&p);
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t u, __half) {
  return __half22float2(*reinterpret_cast<__half2 *>(&u));
}

// T itself where it is a 16-bit type (what the pair functions above take).
template <typename T>
struct Half16 {
  using type = T;
};
template <>
struct Half16<float> {
  using type = __half;
};

// Eight consecutive elements in 16-byte accesses (the address is aligned).
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = unpack2(w[i], T{});
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<float>(const float *p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4 *>(p)[0];
  const float4 b = reinterpret_cast<const float4 *>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
// The same in two steps, so that a loop can ask for its next elements before
// it computes with the present ones.
template <typename T>
struct Raw8 {
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++)
      q[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) {
      const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (sizeof(T) == 4) {
          v[4 * i + j] = __uint_as_float(w[j]);
        } else {
          const float2 f = unpack2(w[j], typename Half16<T>::type{});
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  uint4 u;
  u.x = pack2(v[0], v[1], T{});
  u.y = pack2(v[2], v[3], T{});
  u.z = pack2(v[4], v[5], T{});
  u.w = pack2(v[6], v[7], T{});
  *reinterpret_cast<uint4 *>(p) = u;
}
template <>
__device__ __forceinline__ void store8<float>(float *p, const float (&v)[8]) {
  reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Eight consecutive elements from any address.  16-bit types come as 4-byte words,
// shifted together where the address is odd among them; the words then reach
// one element to either side, so an address nearer than that to the ends of the
// array [lo, hi) is read element by element.
template <typename T>
__device__ __forceinline__ void load8_off(const T *p, const T *lo, const T *hi, float (&v)[8]) {
  if (sizeof(T) == 2 && p - 1 >= lo && p + 9 <= hi) {
    const bool odd = (reinterpret_cast<uintptr_t>(p) & 2) != 0;
    const uint32_t *w = reinterpret_cast<const uint32_t *>(p - odd);
    uint32_t t[5];
#pragma unroll
    for (int i = 0; i < 4; i++) t[i] = w[i];
    t[4] = odd ? w[4] : 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t u = odd ? __funnelshift_r(t[i], t[i + 1], 16) : t[i];
      const float2 f = unpack2(u, typename Half16<T>::type{});
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32<T>(p[i]);
  }
}

// ---- activations ------------------------------------------------------------
// ReLU is the framework's (0 < z) ? z : 0, so a NaN gives 0.  The others pass
// NaN on and take their limits (0 and z) far from 0: the formulas' products
// of 0 and infinity are kept out by bounding z from below where exp(-z) would
// overflow, and from both sides where a slope multiplies z by a vanishing
// factor.
__device__ __forceinline__ float bound_below(float z, float lo) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(lo));
  return r;
}
__device__ __forceinline__ float bound_both(float z, float lim) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(-lim));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(lim));
  return r;
}

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

// The f32 forms use CUDA's functions; GELU's Phi from erfc keeps the left
// tail's digits.  The 16-bit forms end in a rounding to 8 or 11 bits, so they
// use the hardware's approximate exp2 and reciprocal (2 units of f32) and, for
// Phi, the tail's exponential times a polynomial:
//   Phi(-x) = exp(-x^2 / 2) (c1 t + ... + c6 t^6), t = 1 / (1 + 0.312 x), x >= 0,
// whose coefficients make the largest error of exp(x^2 / 2) Phi(-x) least (a linear
// program over 0 <= x <= 34, weighted by 1 / (2 Phi(-x)) up to 8).  It is off by 2^-15
// of Phi(-x) at most, in the tail as well, and by 1.2e-6 absolutely; the output's
// rounding is 2^-12 or more.  These forms are what lets an epilogue of GELU and
// dropout hide behind a 4096-deep bf16 product (erfcf and full divisions take about
// 90 instructions an element, these 27).
template <bool FAST>
struct Math;
template <>
struct Math<false> {
  static __device__ __forceinline__ float phi(float z) {
    return 0.5f * erfcf(z * -0.70710678118654752f);
  }
  static __device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }
  static __device__ __forceinline__ float gelu_slope(float z) {
    return fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), phi(z));
  }
};
template <>
struct Math<true> {
  static __device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  static __device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  // The factors of Phi(-x): exp(-x^2 / 2), and the polynomial without its first t.
  static __device__ __forceinline__ float bell(float x) {
    return ex2(x * x * -0.72134752044448170f);
  }
  static __device__ __forceinline__ float tail(float t) {
    float p = -0.0696624592f;
    p = fmaf(p, t, 0.163576886f);
    p = fmaf(p, t, 0.0322565362f);
    p = fmaf(p, t, 0.126467645f);
    p = fmaf(p, t, 0.12282186f);
    return fmaf(p, t, 0.124538451f);
  }
  static __device__ __forceinline__ float phi(float z) {
    const float x = fabsf(z);
    const float t = rcp(fmaf(0.312f, x, 1.0f));
    const float h = bell(x) * (t * tail(t));  // Phi(-|z|)
    return z > 0.0f ? 1.0f - h : h;
  }
  static __device__ __forceinline__ float logistic(float z) {
    return rcp(1.0f + ex2(z * -1.4426950408889634f));
  }
  // Phi(z) + z phi(z) from one exponential: with x = |z| and s = Phi(-x) - x
  // phi(x), it is s to the left of 0 and 1 - s to the right.
  static __device__ __forceinline__ float gelu_slope(float z) {
    const float x = fabsf(z);
    const float t = rcp(fmaf(0.312f, x, 1.0f));
    const float s = bell(x) * fmaf(t, tail(t), x * -0.3989422804014327f);
    return z > 0.0f ? 1.0f - s : s;
  }
};

// v = act(v), elementwise.
template <bool FAST>
__device__ __forceinline__ void act8(float (&v)[8], int act) {
  using F = Math<FAST>;
  switch (act) {
    case FG_ACT_RELU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float &x = v[i];
        x = 0.0f < x ? x : 0.0f;
      }
      break;
    case FG_ACT_GELU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float &x = v[i];
        x = bound_below(x, -32.0f);
        x *= F::phi(x);
      }
      break;
    case FG_ACT_GELU_TANH:  // (1 + tanh u) / 2 = logistic(2u)
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float &x = v[i];
        x = bound_below(x, -32.0f);
        x *= F::logistic(x * fmaf(2.0f * kGeluC * kGeluB, x * x, 2.0f * kGeluC));
      }
      break;
    case FG_ACT_SILU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        float &x = v[i];
        x = bound_below(x, -128.0f);
        x *= F::logistic(x);
      }
      break;
    default:
      break;
  }
}

// v *= act'(z), elementwise.  Beyond |z| = 32 (GELU) or 104 (SiLU) the slopes
// are 0 or 1 to every bit of f32.  ReLU's slope selects: where z <= 0 the
// result is 0 whatever v is.
template <bool FAST>
__device__ __forceinline__ void slope8(float (&v)[8], const float (&z)[8], int act) {
  using F = Math<FAST>;
  switch (act) {
    case FG_ACT_RELU:
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = 0.0f < z[i] ? v[i] : 0.0f;
      break;
    case FG_ACT_GELU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float b = bound_both(z[i], 32.0f);
        v[i] *= F::gelu_slope(b);
      }
      break;
    case FG_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float b = bound_both(z[i], 32.0f);
        const float q = b * b;
        const float g = F::logistic(b * fmaf(2.0f * kGeluC * kGeluB, q, 2.0f * kGeluC));
        v[i] *= fmaf(b * g * (1.0f - g), fmaf(6.0f * kGeluC * kGeluB, q, 2.0f * kGeluC), g);
      }
      break;
    case FG_ACT_SILU:
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float b = bound_both(z[i], 128.0f);
        const float g = F::logistic(b);
        v[i] *= g * fmaf(b, 1.0f - g, 1.0f);
      }
      break;
    default:
      break;
  }
}

// ---- dropout: Philox4x32-10 --------------------------------------------------
// J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011: ten rounds of two 32 x 32 -> 64 bit products.  One
// block of 128 bits serves eight neighbouring columns of a row, 16 bits each,
// so the mask depends on (seed, offset, row, column) alone: not on the type,
// the strides, or which kernel asks for it.
struct DropParams {
  int on;                 // the threshold t is not 0
  int some;               // t < 65536: something is kept
  uint32_t threshold_hi;  // t << 16 (some)
  float scale;            // 65536 / (65536 - t)
  uint32_t c2, c3;        // offset
  uint32_t k0[10], k1[10];  // the rounds' keys: seed + round * (0x9E3779B9, 0xBB67AE85)
};

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, const DropParams &d) {
  uint32_t c2 = d.c2, c3 = d.c3;
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ d.k0[r];
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ d.k1[r];
    c3 = (uint32_t)p0;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Applies dropout to the eight columns col .. col+7 (col a multiple of 8) of
// a row.  A dropped element is exactly 0, whatever it was (NaN included).
__device__ __forceinline__ void drop8(const DropParams &d, uint32_t row, uint32_t col,
                                      float (&v)[8]) {
  if (!d.some) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.0f;
    return;
  }
  const uint4 r = philox(col >> 3, row, d);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  // r16 >= t, with r16 in the upper half of a word and anything below it
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = (w[i] << 16) >= d.threshold_hi ? v[2 * i] * d.scale : 0.0f;
    v[2 * i + 1] = w[i] >= d.threshold_hi ? v[2 * i + 1] * d.scale : 0.0f;
  }
}

// ---- the epilogue ------------------------------------------------------------
struct Epilogue {
  int act;
  DropParams drop;
  const void *bias;      // [N] or null
  const void *residual;  // [M, N], pitch ldr, or null
  void *pre;             // [M, N], pitch ldp, or null: z before the activation
  void *out;             // [M, N], pitch ldo
  int64_t ldr, ldp, ldo;
  int M, N;
  int vec;  // every array's rows start on 16-byte boundaries: 16-byte accesses
  float scale = 1.0f;  // of the sums, before the bias (a gradient's products)
};

// v = scale v + bias for the columns col .. col+7 (those beyond N get no bias).
template <typename T>
__device__ __forceinline__ void affine8(const Epilogue &e, int col, float (&v)[8]) {
  if (e.scale != 1.0f) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= e.scale;
  }
  if (!e.bias) return;
  const T *b = static_cast<const T *>(e.bias) + col;
  if (e.vec && col + 8 <= e.N) {
    float t[8];
    load8<T>(b, t);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (col + i < e.N) v[i] += to_f32<T>(b[i]);
  }
}

// Columns c .. c+7 of a lane's row in a swizzled block of 16-byte chunks.
template <typename T, typename Chunk>
__device__ __forceinline__ void store8_smem(Chunk chunk, int c, const float (&v)[8]) {
  if (sizeof(T) == 2) {
    store8<T>(reinterpret_cast<T *>(chunk(c / 8)), v);
  } else {
    *reinterpret_cast<float4 *>(chunk(c / 4)) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(chunk(c / 4 + 1)) = make_float4(v[4], v[5], v[6], v[7]);
  }
}
template <typename T, typename Chunk>
__device__ __forceinline__ void load8_smem(Chunk chunk, int c, float (&v)[8]) {
  if (sizeof(T) == 2) {
    load8<T>(reinterpret_cast<const T *>(chunk(c / 8)), v);
  } else {
    const float4 a = *reinterpret_cast<const float4 *>(chunk(c / 4));
    const float4 b = *reinterpret_cast<const float4 *>(chunk(c / 4 + 1));
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

// z (f32 sums, without the bias) for the columns col .. col+7 of a row -> out
// (and pre).  Everything is f32 until the one rounding of each store; the
// activation sees the unrounded z.
template <typename T>
__device__ __forceinline__ void epilogue8(const Epilogue &e, int row, int col, float (&v)[8]) {
  const int n = min(8, e.N - col);
  const bool vec = e.vec && n == 8;
  auto put = [&](void *base, int64_t ld) {
    T *t = static_cast<T *>(base) + (int64_t)row * ld + col;
    if (vec) {
      store8<T>(t, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) t[i] = from_f32<T>(v[i]);
    }
  };
  affine8<T>(e, col, v);
  if (e.pre) put(e.pre, e.ldp);
  act8<sizeof(T) == 2>(v, e.act);
  if (e.drop.on) drop8(e.drop, row, col, v);
  if (e.residual) {
    const T *r = static_cast<const T *>(e.residual) + (int64_t)row * e.ldr + col;
    if (vec) {
      float t[8];
      load8<T>(r, t);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += t[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) v[i] += to_f32<T>(r[i]);
    }
  }
  put(e.out, e.ldo);
}

// A warp's R x C elements (R * C = 256, C = 2^lc) between global memory, neighbouring
// lanes on neighbouring columns, and a slab of R rows of C + 4 floats in shared
// memory, from which a lane takes eight columns of a row: for rows off 16-byte
// boundaries, whose eight columns a lane would otherwise touch one by one, 32
// sectors a time.  All lanes take part.
template <typename T>
__device__ __forceinline__ void slab_fetch(float *slab, int lc, const T *g, int64_t rs, int64_t cs,
                                           int row0, int col0, int M, int N) {
  const int lane = threadIdx.x & 31;
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int x = i * 32 + lane, r = x >> lc, c = x & ((1 << lc) - 1);
    t[i] = row0 + r < M && col0 + c < N ? to_f32<T>(g[(row0 + r) * rs + (col0 + c) * cs]) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int x = i * 32 + lane;
    slab[(x >> lc) * ((1 << lc) + 4) + (x & ((1 << lc) - 1))] = t[i];
  }
  __syncwarp();
}
template <typename T>
__device__ __forceinline__ void slab_flush(const float *slab, int lc, T *g, int64_t ld, int row0,
                                           int col0, int M, int N) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int x = i * 32 + lane, r = x >> lc, c = x & ((1 << lc) - 1);
    if (row0 + r < M && col0 + c < N)
      g[(int64_t)(row0 + r) * ld + col0 + c] = from_f32<T>(slab[r * ((1 << lc) + 4) + c]);
  }
  __syncwarp();
}

// epilogue8 for such rows: lane (r, c) of the R x C elements at (row0, col0).
template <typename T>
__device__ __forceinline__ void epilogue_slab(const Epilogue &e, float *slab, int lc, int row0,
                                              int col0, int r, int c, float (&v)[8]) {
  float *mine = slab + r * ((1 << lc) + 4) + c;
  auto put = [&] {
    __syncwarp();
    reinterpret_cast<float4 *>(mine)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(mine)[1] = make_float4(v[4], v[5], v[6], v[7]);
  };
  affine8<T>(e, col0 + c, v);
  if (e.pre) {
    put();
    slab_flush<T>(slab, lc, static_cast<T *>(e.pre), e.ldp, row0, col0, e.M, e.N);
  }
  act8<sizeof(T) == 2>(v, e.act);
  if (e.drop.on) drop8(e.drop, row0 + r, col0 + c, v);
  if (e.residual) {
    __syncwarp();
    slab_fetch<T>(slab, lc, static_cast<const T *>(e.residual), e.ldr, 1, row0, col0, e.M, e.N);
    float t[8];
    load8<float>(mine, t);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += t[i];
  }
  put();
  slab_flush<T>(slab, lc, static_cast<T *>(e.out), e.ldo, row0, col0, e.M, e.N);
}

// epilogue8 for one element (of a product with scale 1).
template <typename T>
__device__ __forceinline__ void epilogue1(const Epilogue &e, int row, int col, float z) {
  if (e.bias) z += to_f32<T>(static_cast<const T *>(e.bias)[col]);
  if (e.pre) static_cast<T *>(e.pre)[(int64_t)row * e.ldp + col] = from_f32<T>(z);
  float v[8] = {z, z, z, z, z, z, z, z};
  if (e.act) {
    act8<sizeof(T) == 2>(v, e.act);
    z = v[0];
  }
  if (e.drop.on) {
    drop8(e.drop, row, col & ~7, v);
    const int i = col & 7;
    z = v[0];
#pragma unroll
    for (int k = 1; k < 8; k++)
      if (i == k) z = v[k];
  }
  if (e.residual)
    z += to_f32<T>(static_cast<const T *>(e.residual)[(int64_t)row * e.ldr + col]);
  static_cast<T *>(e.out)[(int64_t)row * e.ldo + col] = from_f32<T>(z);
}

// Walks a rows x groups array from a thread's first piece in equal steps, with
// a division at the start only: (row, group) of the next piece.
struct Walk {
  int64_t row, rows, step_row;
  int group, groups, step_group;
  __device__ Walk(int64_t rows_, int groups_, int64_t at, int64_t step)
      : rows(rows_), groups(groups_) {
    if (at < 0x7fffffff && step < 0x7fffffff) {
      row = (uint32_t)at / (uint32_t)groups;
      step_row = (uint32_t)step / (uint32_t)groups;
    } else {
      row = at / groups;
      step_row = step / groups;
    }
    group = (int)(at - row * groups);
    step_group = (int)(step - step_row * groups);
  }
  __device__ bool inside() const { return row < rows; }
  __device__ void next() {
    row += step_row;
    group += step_group;
    if (group >= groups) {
      group -= groups;
      row++;
    }
  }
};

// Launches a kernel whose blocks begin with grid_wait() (fg_ptx.cuh), so that
// it may start while the stream's previous kernel ends.  Its inputs may then
// still be written while it runs, so none of it reads through the path for data
// that is constant over a kernel's life (no __ldg, no __restrict__: such loads
// may also be moved above the wait).
template <typename... P, typename... A>
int launch_early(void (*kern)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...));
  count_launch();
  return FG_OK;
}

// A matrix operand: element (r, c) at ptr[r * row + c * col].
struct Mat {
  const void *ptr;
  int64_t row, col;
};

// A product's operand as the tensor-core kernel reads it: 16-bit elements
// [planes][outer][pitch], `inner` of each row in use.  K-major: outer = rows,
// inner = k; MN-major: outer = k, inner = rows.
struct Operand {
  const void *ptr;   // null until a staged operand is placed in the workspace
  int64_t inner, outer, pitch;
  int planes, mn_major;
  size_t staged_at;
};
// One copy into such a layout (k_stage); `at`, dst: its place in the workspace.
struct StageJob {
  const void *src;
  void *dst;
  int64_t so, si;  // source strides of the outer and inner index
  int64_t outer, inner, pitch;
  size_t at;
  int vec;
};
struct StageJobs {
  StageJob job[3];
  int n;
};
// Describes rows x k elements of m in place, or adds a staging job and grows
// *ws by its bytes.
Operand resolve_operand(int dtype, const Mat &m, int64_t rows, int64_t k, StageJobs *jobs,
                        size_t *ws);
void place_operand(Operand *o, void *ws);
void place_jobs(StageJobs *jobs, void *ws);
int run_stage(int dtype, const StageJobs &jobs, cudaStream_t st);

// A product of rows and columns e.M, e.N over K with its epilogue.
struct Product {
  Operand a, b;
  int K;
  Epilogue e;
};
int run_tensor_product(int dtype, const Product &x, cudaStream_t st);
int run_tensor_products(int dtype, const Product &x, const Product &y, cudaStream_t st);

// An f32 value as the sum of three bf16 values, each rest exact, such that the six
// products of two values' parts add up to what f32 arithmetic gives beyond its
// range too:
//  * An infinity is (+-1, 0, +-inf).  Against a finite value only its last part
//    meets the other's first, so the sum is +-inf, or NaN for 0; against another
//    infinity 1 meets inf twice.  (inf in front would meet rests of either sign:
//    inf - inf.)
//  * From 4 upwards the parts are cut, not rounded, and so have the value's sign.
//    Below, a part may be rounded up and leave a rest of the other sign, 2^-7 at
//    most: the 64 products of a chain with such rests stay below 2^127.  (With
//    every part rounded, 1e21 * 1e21 came out as -inf.)
// What six products leave out of one is at most 2^-24 of it, and 2^-21 where both
// values are cut.  Below 2^-110 the rests run out of bf16's exponents: the last
// bits are lost.
__device__ __forceinline__ void split3(float v, float &a, float &b, float &c) {
  const uint32_t top = 0xffff0000u;
  const bool cut = fabsf(v) >= 4.0f;
  a = cut ? __uint_as_float(__float_as_uint(v) & top) : __bfloat162float(__float2bfloat16_rn(v));
  const float r = v - a;
  b = cut ? __uint_as_float(__float_as_uint(r) & top) : __bfloat162float(__float2bfloat16_rn(r));
  c = r - b;
  if (!isfinite(v)) {
    a = isinf(v) ? copysignf(1.0f, v) : v;
    b = 0.0f;
    c = isinf(v) ? v : 0.0f;
  }
}

}  // namespace layer
}  // namespace fg
