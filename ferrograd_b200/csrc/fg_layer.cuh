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

// ---- activations ------------------------------------------------------------
// ReLU is the framework's (0 < z) ? z : 0, so a NaN gives 0.  The others pass
// NaN on and take their limits (0 and z) far from 0: the formulas' products
// of 0 and infinity are kept out by bounding z from below where exp(-z) would
// overflow, and from both sides where a slope multiplies z by a vanishing
// factor.
__device__ __forceinline__ float bound_below(float z, float lo) { return z < lo ? lo : z; }
__device__ __forceinline__ float bound_both(float z, float lim) {
  return z < -lim ? -lim : (z > lim ? lim : z);
}

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case FG_ACT_RELU:
      return 0.0f < z ? z : 0.0f;
    case FG_ACT_GELU: {  // z * Phi(z); Phi from erfc keeps the left tail's digits
      const float b = bound_below(z, -16.0f);
      return b * (0.5f * erfcf(b * -0.70710678118654752f));
    }
    case FG_ACT_GELU_TANH: {
      // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u))
      const float b = bound_below(z, -16.0f);
      const float u = kGeluC * (b + kGeluB * b * b * b);
      return b / (1.0f + expf(-2.0f * u));
    }
    case FG_ACT_SILU: {
      const float b = bound_below(z, -128.0f);
      return b / (1.0f + expf(-b));
    }
    default:
      return z;
  }
}

// d act / dz.  Beyond |z| = 16 (GELU) or 104 (SiLU) the slopes are 0 or 1 to
// every bit of f32.
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case FG_ACT_RELU:
      return 0.0f < z ? 1.0f : 0.0f;
    case FG_ACT_GELU: {
      const float b = bound_both(z, 16.0f);
      return 0.5f * erfcf(b * -0.70710678118654752f) +
             b * (0.3989422804014327f * expf(-0.5f * b * b));
    }
    case FG_ACT_GELU_TANH: {
      const float b = bound_both(z, 16.0f);
      const float g = 1.0f / (1.0f + expf(-2.0f * kGeluC * (b + kGeluB * b * b * b)));
      return g + b * g * (1.0f - g) * (2.0f * kGeluC * (1.0f + 3.0f * kGeluB * b * b));
    }
    case FG_ACT_SILU: {
      const float b = bound_both(z, 128.0f);
      const float s = 1.0f / (1.0f + expf(-b));
      return s * (1.0f + b * (1.0f - s));
    }
    default:
      return 1.0f;
  }
}

// ---- dropout: Philox4x32-10 --------------------------------------------------
// J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011: ten rounds of two 32 x 32 -> 64 bit products.  One
// block of 128 bits serves eight neighbouring columns of a row, 16 bits each,
// so the mask depends on (seed, offset, row, column) alone: not on the type,
// the strides, or which kernel asks for it.
struct DropParams {
  uint32_t threshold;  // keep where the 16 bits are >= threshold; 0: dropout is off
  float scale;         // 65536 / (65536 - threshold), 0 where everything is dropped
  uint32_t k0, k1;     // seed
  uint32_t c2, c3;     // offset
};

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3,
                                        uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; r++) {
    const uint32_t h0 = __umulhi(0xD2511F53u, c0), l0 = 0xD2511F53u * c0;
    const uint32_t h1 = __umulhi(0xCD9E8D57u, c2), l1 = 0xCD9E8D57u * c2;
    c0 = h1 ^ c1 ^ k0;
    c1 = l1;
    c2 = h0 ^ c3 ^ k1;
    c3 = l0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Applies dropout to the eight columns col .. col+7 (col a multiple of 8) of
// a row.  A dropped element is exactly 0, whatever it was (NaN included).
__device__ __forceinline__ void drop8(const DropParams &d, uint32_t row, uint32_t col,
                                      float (&v)[8]) {
  const uint4 r = philox(col >> 3, row, d.c2, d.c3, d.k0, d.k1);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = (w[i] & 0xffffu) >= d.threshold ? v[2 * i] * d.scale : 0.0f;
    v[2 * i + 1] = (w[i] >> 16) >= d.threshold ? v[2 * i + 1] * d.scale : 0.0f;
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
};

// z (f32 sums, without the bias) for the columns col .. col+7 of a row ->
// out (and pre).  Everything is f32 until the one rounding of each store; the
// activation sees the unrounded z.
template <typename T>
__device__ __forceinline__ void epilogue8(const Epilogue &e, int row, int col, float (&v)[8]) {
  const bool whole = col + 8 <= e.N;
  const int n = whole ? 8 : e.N - col;
  const bool vec = e.vec && whole;
  if (e.bias) {
    const T *b = static_cast<const T *>(e.bias) + col;
    if (vec) {
      float t[8];
      load8<T>(b, t);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += t[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) v[i] += to_f32<T>(b[i]);
    }
  }
  if (e.pre) {
    T *p = static_cast<T *>(e.pre) + (int64_t)row * e.ldp + col;
    if (vec) {
      store8<T>(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (i < n) p[i] = from_f32<T>(v[i]);
    }
  }
  if (e.act != FG_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = act_value(v[i], e.act);
  }
  if (e.drop.threshold) drop8(e.drop, row, col, v);
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
  T *o = static_cast<T *>(e.out) + (int64_t)row * e.ldo + col;
  if (vec) {
    store8<T>(o, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < n) o[i] = from_f32<T>(v[i]);
  }
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

// How the tensor-core kernel cuts a product up (fg_layer_gemm.cu).
struct Form {
  bool pair;
  int bm, bn, split;
};
Form pick_form(int M, int N, int K, int planes, int sms);
int run_tensor_product(int dtype, const Operand &a, const Operand &b, int K, const Epilogue &e,
                       cudaStream_t st);

// An f32 value as the sum of three bf16 values, each rest exact (an infinity
// is its own first part; a value that would round up to infinity is cut).
__device__ __forceinline__ void split3(float v, float &a, float &b, float &c) {
  a = __bfloat162float(__float2bfloat16_rn(v));
  if (isinf(a) && !isinf(v)) a = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  const float r = isinf(v) ? 0.0f : v - a;
  b = __bfloat162float(__float2bfloat16_rn(r));
  c = r - b;
}

}  // namespace layer
}  // namespace fg
