// The linear layer with a fused epilogue, its gradient and dropout.
//
//   z = x w^T + bias;  out = residual + D(act(z))            fg_linear
//   dz = D(dy) act'(z);  dx = dz w;  dw = dz^T x;  db = sum dz  fg_linear_grad
//   out = residual + D(x)                                    fg_dropout
//
// D is dropout by a counter-based generator (fg_layer.cuh): the mask is
// computed where it is used, forwards and backwards, and never stored.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fg_internal.h"
#include "fg_layer.cuh"
#include "fg_ptx.cuh"

namespace fg {
namespace layer {

using ptx::grid_launch_next;
using ptx::grid_wait;

// ---------------------------------------------------------------------------
// Sums over nothing (K = 0, or a gradient's N = 0): all are 0 and the epilogue remains.
// Bound by the output's writes; a thread has eight columns of a row a step.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) k_linear_empty(const Epilogue e) {
  grid_wait();
  grid_launch_next();
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (Walk at(e.M, (e.N + 7) / 8, first, step); at.inside(); at.next()) {
    float v[8] = {};
    epilogue8<T>(e, (int)at.row, at.group * 8, v);
  }
}

// ---------------------------------------------------------------------------
// Up to 8 rows of x: C = x w^T with w's rows contiguous, in f32 on the CUDA
// cores.  The weight is read once, a warp one or two of its rows at a time, each
// lane 16 bytes of a row; what bounds it is that stream, so a lane asks for the
// next four steps before it multiplies.  The warp's sums meet by shuffles in a
// fixed order.  (A tensor-core tile of so few rows first fills and drains
// accumulators, and joins its k-ranges across CTAs: 1 x 4096 x 4096 bf16, the
// weight from HBM, 12.5 us against 8.7 us here, 3.9 TB/s: 33 MB are too few for
// the copy rate.)  VEC: every row starts on a 16-byte boundary; without it
// elements are read one by one, still in neighbouring lanes.
// ---------------------------------------------------------------------------
constexpr int kRowsMax = 8;

// For MR rows of x: the weight's rows a warp takes, and the steps it has in
// flight.  One 16-bit row of 4096 by itself is 1 x 4096 x 4096 from HBM in 8.7 us, two
// together 12.3; f32 rows by two take 26 us for four rows of x, one by one 38.
template <typename T, int MR>
struct RowsShape {
  static constexpr int rows = sizeof(T) == 2 ? 1 : 2;
  static constexpr int steps = MR <= 4 ? 4 : 2;
};

// Rows up to which it is used instead of the tensor cores' few-row tiles.  In f32 8,
// as those have to split the weight into planes first (8 x 4096 -> 4096 32 us against 62;
// off 16-byte rows 50, 68), in 16 bits 2 (10.2, 12.4; off 16-byte rows, where the
// tiles need a copy of the weight, 22.4, 28.3 -- but 46, 28.5 for three).  Measured at
// 4096 x 4096.  A small layer gains more (2 x 256 -> 256 1.8, 4.5); a long row into few
// outputs loses, as its warps are few: 2 x 8192 -> 128 bf16 12.9, 7.8; 8 in f32 51, 22.
static int rows_limit(int dtype) { return dtype == FG_F32 ? kRowsMax : 2; }

// What a lane reads at once: 16 bytes, or one element.
template <typename T, bool VEC>
struct RawOf {
  using type = uint4;
};
template <>
struct RawOf<float, false> {
  using type = uint32_t;
};
template <>
struct RawOf<__nv_bfloat16, false> {
  using type = uint16_t;
};
template <>
struct RawOf<__half, false> {
  using type = uint16_t;
};
template <typename T>
__device__ __forceinline__ void unraw(const uint4 &r, float (&v)[16 / sizeof(T)]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (sizeof(T) == 4) {
      v[i] = __uint_as_float(w[i]);
    } else {
      const float2 f = unpack2(w[i], typename Half16<T>::type{});
      v[2 * i % (16 / sizeof(T))] = f.x;
      v[(2 * i + 1) % (16 / sizeof(T))] = f.y;
    }
  }
}
template <typename T, typename R>
__device__ __forceinline__ void unraw(const R &r, float (&v)[1]) {
  v[0] = to_f32<T>(*reinterpret_cast<const T *>(&r));
}

template <typename T, int MR, bool VEC>
__global__ void __launch_bounds__(256)
    k_linear_rows(const T *x, int64_t xr, const T *w, int64_t wr, int K,
                  const Epilogue e) {
  constexpr int V = VEC ? 16 / sizeof(T) : 1;  // elements a lane reads at once
  constexpr int R = RowsShape<T, MR>::rows, U = RowsShape<T, MR>::steps;
  const int lane = threadIdx.x & 31;
  const int n0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * R;
  grid_wait();
  grid_launch_next();
  if (n0 >= e.N) return;
  const T *wp[R];
#pragma unroll
  for (int c = 0; c < R; c++) wp[c] = w + min(n0 + c, e.N - 1) * wr;
  float acc[MR][R] = {};
  using Raw = typename RawOf<T, VEC>::type;
  // The weight passes once and x is read by every warp: the one leaves L1 first.
  // (8 x 4096 -> 4096 f32 32 us, with ordinary loads 42; 2 rows in bf16 10.3, 12.4.)
  auto read = [](const T *p) { return *reinterpret_cast<const Raw *>(p); };
  auto pass = [](const T *p) { return __ldcs(reinterpret_cast<const Raw *>(p)); };
  auto step = [&](int64_t k, const Raw(&rw)[R]) {
    float b[R][V];
#pragma unroll
    for (int c = 0; c < R; c++) unraw<T>(rw[c], b[c]);
    Raw rx[MR];
#pragma unroll
    for (int m = 0; m < MR; m++) rx[m] = read(x + min(m, e.M - 1) * xr + k);
#pragma unroll
    for (int m = 0; m < MR; m++) {
      float t[V];
      unraw<T>(rx[m], t);
#pragma unroll
      for (int i = 0; i < V; i++)
#pragma unroll
        for (int c = 0; c < R; c++) acc[m][c] = fmaf(t[i], b[c][i], acc[m][c]);
    }
  };
  constexpr int S = 32 * V;  // elements of a row in one step of the warp
  int64_t k = lane * V;
  for (; k + (U - 1) * S + V <= K; k += U * S) {
    Raw r[U][R];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int c = 0; c < R; c++) r[u][c] = pass(wp[c] + k + u * S);
#pragma unroll
    for (int u = 0; u < U; u++) step(k + u * S, r[u]);
  }
  for (; k + V <= K; k += S) {
    Raw r[R];
#pragma unroll
    for (int c = 0; c < R; c++) r[c] = pass(wp[c] + k);
    step(k, r);
  }
  if (VEC && k < K)  // the row's last elements, fewer than V (one lane has them)
    for (; k < K; k++)
#pragma unroll
      for (int m = 0; m < MR; m++) {
        const float t = to_f32<T>(x[min(m, e.M - 1) * xr + k]);
#pragma unroll
        for (int c = 0; c < R; c++) acc[m][c] = fmaf(t, to_f32<T>(wp[c][k]), acc[m][c]);
      }
#pragma unroll
  for (int m = 0; m < MR; m++)
#pragma unroll
    for (int c = 0; c < R; c++) {
      float s = acc[m][c];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == m * R + c && m < e.M && n0 + c < e.N) epilogue1<T>(e, m, n0 + c, s);
    }
}

template <typename T>
static int run_rows(const fg_linear_args *g, const Epilogue &e, bool vec, cudaStream_t st) {
  const T *x = static_cast<const T *>(g->x), *w = static_cast<const T *>(g->w);
  auto go = [&](auto kern) {
    const int per = 8 * RowsShape<T, 1>::rows;  // the same for every MR
    const unsigned grid = (unsigned)((g->N + (int64_t)per - 1) / per);
    return launch_early(kern, dim3(grid), 256, st, x, g->x_row, w, g->w_row, g->K, e);
  };
  if (g->M == 1) return vec ? go(k_linear_rows<T, 1, true>) : go(k_linear_rows<T, 1, false>);
  if constexpr (sizeof(T) == 4) {  // 16-bit types end at two rows (rows_limit)
    if (g->M > 4) return vec ? go(k_linear_rows<T, 8, true>) : go(k_linear_rows<T, 8, false>);
    if (g->M > 2) return vec ? go(k_linear_rows<T, 4, true>) : go(k_linear_rows<T, 4, false>);
  }
  return vec ? go(k_linear_rows<T, 2, true>) : go(k_linear_rows<T, 2, false>);
}

// ---------------------------------------------------------------------------
// dz = D(dy) * act'(pre), and the column sums of dz over this block's rows
// (f32, one row of `part` a block; k_bias_grad adds them up).
// dz may be null (only the sums are wanted).  What it writes is dz * unit / scale
// (DzScale): without dropout's scale the 16-bit types hold dy itself where no
// slope multiplies it, and f16 does not overflow.
// It reads dy and pre once and writes dz once: 1.6 GB at 16384 x 16384 bf16, GELU,
// 246 us at the copy rate, measured 305 us, with dropout 400: the slope's exponential
// and the conversions are 37 instructions an element, the mask's 5 more, and the issue
// slots, 74% of them taken, bound it, not HBM.  A thread keeps its eight columns down
// the rows, so the column sums need no exchange until the end, and asks for the next
// rows before it computes.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void store_dz(void *dz, int64_t at, int64_t, const float (&v)[8]) {
  store8<T>(static_cast<T *>(dz) + at, v);
}
// f32: three bf16 planes, as the products read them
template <>
__device__ __forceinline__ void store_dz<float>(void *dz, int64_t at, int64_t plane,
                                                const float (&v)[8]) {
  float p[3][8];
#pragma unroll
  for (int i = 0; i < 8; i++) split3(v[i], p[0][i], p[1][i], p[2][i]);
#pragma unroll
  for (int k = 0; k < 3; k++) store8(static_cast<__nv_bfloat16 *>(dz) + k * plane + at, p[k]);
}
// How dz is scaled where it is stored, and what its sums are multiplied by.
struct DzScale {
  float unit, after;
};
// TX: groups of eight columns across a block, 32 or 4 (small matrices); 256 /
// TX rows down it.  Where one block has all rows of its columns it writes db
// itself.
template <typename T, int TX>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2)
    k_layer_dz(const T *dy, int64_t yr, int64_t yc, const T *pre,
               int64_t ldp, int act, const DropParams drop, const DzScale by, void *dz,
               int64_t ldz, float *part, T *db, int M, int N, int rows, int vec) {
  constexpr int TY = 256 / TX;
  __shared__ float red[TY][TX * 8];
  constexpr int U = 2;  // rows in flight, and as many again asked for
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int col = blockIdx.x * (TX * 8) + tx * 8;
  const int r0 = blockIdx.y * rows, r1 = r0 + min(rows, M - r0);  // (r0 + rows may pass 2^31)
  float sum[8] = {};
  grid_wait();
  grid_launch_next();
  auto one = [&](int r, float(&v)[8], const float(&z)[8]) {
    if (drop.on) {  // whose scale is by.unit
      drop8(drop, r, col, v);
    } else if (by.unit != 1.0f) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= by.unit;
    }
    slope8<sizeof(T) == 2>(v, z, act);
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] += v[i];
    // ldz is a multiple of 8 and the rest of a row's last group is 0
    if (dz) store_dz<T>(dz, r * ldz + col, (int64_t)M * ldz, v);
  };
  if (vec && col + 8 <= N) {
    Raw8<T> y[U], p[U], yn[U], pn[U];
    auto ask = [&](int r, Raw8<T>(&a)[U], Raw8<T>(&b)[U]) {
#pragma unroll
      for (int u = 0; u < U; u++)
        if (r + TY * u < r1) {
          a[u].load(dy + (r + TY * u) * yr + col);
          if (act != FG_ACT_NONE) b[u].load(pre + (r + TY * u) * ldp + col);
        }
    };
    ask(r0 + ty, y, p);
    for (int r = r0 + ty; r < r1; r += TY * U) {
      ask(r + TY * U, yn, pn);
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (r + TY * u < r1) {
          float v[8], z[8];
          y[u].get(v);
          p[u].get(z);
          one(r + TY * u, v, z);
        }
        y[u] = yn[u];
        p[u] = pn[u];
      }
    }
  } else if (col < N) {
    for (int r = r0 + ty; r < r1; r += TY) {
      float v[8], z[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        v[i] = col + i < N ? to_f32<T>(dy[r * yr + (col + i) * yc]) : 0.0f;
        z[i] = act != FG_ACT_NONE && col + i < N ? to_f32<T>(pre[r * ldp + col + i]) : 0.0f;
      }
      one(r, v, z);
    }
  }
  if (!db) return;
#pragma unroll
  for (int i = 0; i < 8; i++) red[ty][tx * 8 + i] = sum[i];
  __syncthreads();
  // a tree of TY terms, eight at a time
  constexpr int C = TX * 8;
  auto eight = [&](int r, int col8) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = red[r + i][col8];
    return ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  };
  static_assert(TY * C == 8 * 256, "every thread has eight terms of a column");
  float s = eight(threadIdx.x / C * 8, threadIdx.x % C);
  if (TY > 8) {
    __syncthreads();
    red[threadIdx.x / C][threadIdx.x % C] = s;
    __syncthreads();
    if (threadIdx.x < C) s = eight(0, threadIdx.x);
  }
  const int c = blockIdx.x * C + threadIdx.x;
  if (threadIdx.x < C && c < N) {
    s *= by.after;
    if (gridDim.y == 1)
      db[c] = from_f32<T>(s);
    else
      part[(size_t)blockIdx.y * N + c] = s;
  }
}

// db = the blocks' sums, in a fixed order: 32 columns a block, a column's sums dealt
// to 32 threads, each of which carries the rounding of its additions along (W.
// Kahan, "Further remarks on reducing truncation errors", 1965), and joined as a
// tree.  Latency of a few reads.
template <typename T>
__global__ void __launch_bounds__(1024)
    k_bias_grad(const float *part, int chunks, int N, T *db) {
  __shared__ float red[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + x;
  grid_wait();
  grid_launch_next();
  float s = 0.0f, lost = 0.0f;
  if (c < N) {
#pragma unroll 4
    for (int i = y; i < chunks; i += 32) {
      const float v = part[(size_t)i * N + c] - lost, t = s + v;
      lost = isfinite(t) ? (t - s) - v : 0.0f;
      s = t;
    }
  }
  red[y][x] = s;
#pragma unroll
  for (int half = 16; half > 0; half /= 2) {
    __syncthreads();
    if (y < half) red[y][x] += red[y + half][x];
  }
  if (y == 0 && c < N) db[c] = from_f32<T>(red[0][x]);
}

// ---------------------------------------------------------------------------
// out = residual + D(x): eight columns of a row a step, one Philox call for them.
// Bound by HBM, with the issue slots close behind: 16384 x 16384 bf16 with a
// residual in 266 us, 6.1 TB/s or 0.93 of a copy's rate (an addition of the two
// arrays alone takes 236 us).  Rows off 16-byte boundaries go element by element: 4001 x
// 4097 bf16 39 us, 4001 x 4096 17.  A thread asks for all its groups before it draws.
// ---------------------------------------------------------------------------
// Groups of eight columns a thread takes, 256 groups apart.
template <typename T>
struct DropGroups {
  static constexpr int value = sizeof(T) == 2 ? 4 : 2;
};

// A group of n <= 8 columns, element by element.
template <typename T>
__device__ __forceinline__ void drop_tail(const T *x, const T *residual, T *out,
                                          const DropParams &drop, int64_t row, int col, int n) {
  float v[8], t[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    v[i] = i < n ? to_f32<T>(x[i]) : 0.0f;
    t[i] = residual && i < n ? to_f32<T>(residual[i]) : 0.0f;
  }
  if (drop.on) drop8(drop, (uint32_t)row, col, v);
#pragma unroll
  for (int i = 0; i < 8; i++)
    if (i < n) out[i] = from_f32<T>(residual ? v[i] + t[i] : v[i]);
}

template <typename T>
__global__ void __launch_bounds__(256, 4)
    k_dropout(const T *x, int64_t ldx, const T *residual, int64_t ldr, T *out, int64_t ldo,
              const DropParams drop, int64_t rows, int cols, int vec) {
  constexpr int U = DropGroups<T>::value;
  Walk at(rows, (cols + 7) / 8, (int64_t)blockIdx.x * (256 * U) + threadIdx.x, 256);
  grid_wait();
  grid_launch_next();
  Raw8<T> a[U], b[U];
  int64_t row[U];
  int col[U];
#pragma unroll
  for (int u = 0; u < U; u++, at.next()) {  // every load first
    row[u] = at.row;
    col[u] = at.group * 8;
    if (vec && at.inside() && col[u] + 8 <= cols) {
      a[u].load(x + row[u] * ldx + col[u]);
      if (residual) b[u].load(residual + row[u] * ldr + col[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (row[u] >= rows) return;
    T *o = out + row[u] * ldo + col[u];
    if (vec && col[u] + 8 <= cols) {
      float v[8], t[8];
      a[u].get(v);
      if (drop.on) drop8(drop, (uint32_t)row[u], col[u], v);
      if (residual) {
        b[u].get(t);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += t[i];
      }
      store8<T>(o, v);
    } else {
      drop_tail(x + row[u] * ldx + col[u], residual ? residual + row[u] * ldr + col[u] : nullptr, o,
                drop, row[u], col[u], min(8, cols - col[u]));
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static int elem_size(int dtype) {
  return dtype == FG_F32 ? 4 : dtype == FG_BF16 || dtype == FG_F16 ? 2 : 0;
}

static int make_drop(const char *who, const fg_dropout_spec *s, DropParams *d) {
  *d = DropParams{};
  if (!s) return FG_OK;
  FG_REQUIRE(s->p >= 0.0 && s->p <= 1.0, "%s: dropout probability %g is not in [0, 1]", who, s->p);
  const uint32_t t = (uint32_t)floor(s->p * 65536.0 + 0.5);
  d->on = t > 0;
  d->some = t < 65536;
  d->threshold_hi = t << 16;
  d->scale = d->some ? (float)(65536.0 / (65536 - t)) : 0.0f;
  for (uint32_t r = 0; r < 10; r++) {
    d->k0[r] = (uint32_t)s->seed + r * 0x9E3779B9u;
    d->k1[r] = (uint32_t)(s->seed >> 32) + r * 0xBB67AE85u;
  }
  d->c2 = (uint32_t)s->offset;
  d->c3 = (uint32_t)(s->offset >> 32);
  return FG_OK;
}

// Rows that start on 16-byte boundaries (or an absent array).
static bool rows16(const void *p, int64_t ld, int es) {
  return !p || ((uintptr_t)p % 16 == 0 && ld * es % 16 == 0);
}

// Every address is a multiple of the element's size (an odd one would be a
// misaligned access on the device).
template <typename... P>
static bool whole(int es, const P *...p) {
  return (((uintptr_t)p % es == 0) && ...);
}

// A rows x cols array's bytes [lo, hi), strides of either sign included.
struct Span {
  uintptr_t lo, hi;
};
static Span span(const void *p, int64_t rows, int64_t cols, int64_t rs, int64_t cs, int es) {
  int64_t lo = 0, hi = 0;
  if (rows > 0 && cols > 0) {
    (rs < 0 ? lo : hi) += (rows - 1) * rs;
    (cs < 0 ? lo : hi) += (cols - 1) * cs;
    hi += 1;
  }
  return {(uintptr_t)p + lo * es, (uintptr_t)p + hi * es};
}
// Whether a written array may share bytes with another.  Two column ranges of
// one pitched buffer (equal pitch, disjoint columns) do not.
static bool overlap(const void *w, int64_t rows, int64_t cols, int64_t ld, const void *q,
                    int64_t qrows, int64_t qcols, int64_t qrs, int64_t qcs, int es) {
  if (!w || !q || rows <= 0 || cols <= 0 || qrows <= 0 || qcols <= 0) return false;
  const Span a = span(w, rows, cols, ld, 1, es), b = span(q, qrows, qcols, qrs, qcs, es);
  if (a.lo >= b.hi || b.lo >= a.hi) return false;
  if (ld == qrs && qcs == 1 && ld > 0) {
    const int64_t pitch = ld * es;
    int64_t d = (int64_t)((uintptr_t)q - (uintptr_t)w) % pitch;
    if (d < 0) d += pitch;
    if (d >= cols * es && d + qcols * es <= pitch) return false;
  }
  return true;
}

static int run_empty_product(int dtype, const Epilogue &e, cudaStream_t st) {
  const int64_t blocks = ((int64_t)e.M * ((e.N + 7LL) / 8) + 255) / 256;
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
  if (dtype == FG_F32) return launch_early(k_linear_empty<float>, grid, 256, st, e);
  if (dtype == FG_BF16) return launch_early(k_linear_empty<__nv_bfloat16>, grid, 256, st, e);
  return launch_early(k_linear_empty<__half>, grid, 256, st, e);
}

static int check_common(const char *who, int dtype, int M, int N, int K, int act) {
  FG_REQUIRE(elem_size(dtype) > 0, "%s: dtype %d is not f32, bf16 or f16", who, dtype);
  const int most = 0x7fffff00;  // tile and column arithmetic stays within an int
  FG_REQUIRE(M >= 0 && N >= 0 && K >= 0 && M <= most && N <= most && K <= most,
             "%s: M, N, K must lie in [0, %d] (got %d, %d, %d)", who, most, M, N, K);
  FG_REQUIRE(act >= FG_ACT_NONE && act <= FG_ACT_SILU, "%s: unknown activation %d", who, act);
  return FG_OK;
}

// Where a forward product reads its operands, and the workspace that takes.
struct LinearPlan {
  bool rows, vec;  // k_linear_rows, with 16-byte reads
  Operand x, w;
  StageJobs jobs;
  size_t bytes;
};
static LinearPlan plan_linear(const fg_linear_args *g) {
  LinearPlan p{};
  if (g->M == 0 || g->N == 0 || g->K == 0) return p;
  const int es = elem_size(g->dtype);
  p.vec = rows16(g->x, g->M == 1 ? 0 : g->x_row, es) && rows16(g->w, g->w_row, es);
  p.rows = g->M <= rows_limit(g->dtype) && (g->x_col == 1 || g->K == 1) &&
           (g->w_col == 1 || g->K == 1);
  if (p.rows) return p;
  p.x = resolve_operand(g->dtype, {g->x, g->x_row, g->x_col}, g->M, g->K, &p.jobs, &p.bytes);
  p.w = resolve_operand(g->dtype, {g->w, g->w_row, g->w_col}, g->N, g->K, &p.jobs, &p.bytes);
  return p;
}

static int check_linear(const fg_linear_args *g, DropParams *drop) {
  const char *who = "fg_linear";
  FG_REQUIRE(g, "%s: null arguments", who);
  int rc = check_common(who, g->dtype, g->M, g->N, g->K, g->act);
  if (rc) return rc;
  if ((rc = make_drop(who, &g->drop, drop))) return rc;
  if (g->M == 0 || g->N == 0) return FG_OK;
  const int es = elem_size(g->dtype);
  FG_REQUIRE(g->out && (g->K == 0 || (g->x && g->w)), "%s: null operand", who);
  FG_REQUIRE(whole(es, g->x, g->w, g->bias, g->residual, g->pre, g->out),
             "%s: an address is not a multiple of the element's size", who);
  FG_REQUIRE(g->ld_out >= g->N && (!g->pre || g->ld_pre >= g->N), "%s: output pitch too small",
             who);
  for (int i = 0; i < 2; i++) {
    const void *w = i ? g->pre : g->out;
    const int64_t ld = i ? g->ld_pre : g->ld_out;
    FG_REQUIRE(!overlap(w, g->M, g->N, ld, g->x, g->M, g->K, g->x_row, g->x_col, es) &&
                   !overlap(w, g->M, g->N, ld, g->w, g->N, g->K, g->w_row, g->w_col, es) &&
                   !overlap(w, g->M, g->N, ld, g->bias, 1, g->N, g->N, 1, es),
               "%s: %s overlaps an operand", who, i ? "pre" : "out");
    const bool same = !i && g->residual == g->out && g->ld_residual == g->ld_out;
    FG_REQUIRE(same || !overlap(w, g->M, g->N, ld, g->residual, g->M, g->N, g->ld_residual, 1, es),
               "%s: %s overlaps the residual (only out may, and only be all of it)", who,
               i ? "pre" : "out");
  }
  FG_REQUIRE(!overlap(g->out, g->M, g->N, g->ld_out, g->pre, g->M, g->N, g->ld_pre, 1, es),
             "%s: out overlaps pre", who);
  return FG_OK;
}

static int linear(const fg_linear_args *g, cudaStream_t st) {
  Epilogue e{};
  int rc = check_linear(g, &e.drop);
  if (rc || g->M == 0 || g->N == 0) return rc;
  LinearPlan p = plan_linear(g);
  FG_REQUIRE(g->workspace_bytes >= p.bytes && (p.bytes == 0 || g->workspace),
             "fg_linear: %zu bytes of workspace needed, got %zu", p.bytes, g->workspace_bytes);
  FG_REQUIRE(p.bytes == 0 || whole(256, g->workspace),
             "fg_linear: the workspace is not on a 256-byte boundary");
  const int es = elem_size(g->dtype);
  e.act = g->act;
  e.bias = g->bias;
  e.residual = g->residual;
  e.pre = g->pre;
  e.out = g->out;
  e.ldr = g->ld_residual;
  e.ldp = g->ld_pre;
  e.ldo = g->ld_out;
  e.M = g->M;
  e.N = g->N;
  e.vec = rows16(e.bias, 0, es) && rows16(e.residual, e.ldr, es) && rows16(e.pre, e.ldp, es) &&
          rows16(e.out, e.ldo, es);
  if (g->K == 0) return run_empty_product(g->dtype, e, st);
  if (p.rows) {
    switch (g->dtype) {
      case FG_F32:
        return run_rows<float>(g, e, p.vec, st);
      case FG_BF16:
        return run_rows<__nv_bfloat16>(g, e, p.vec, st);
      default:
        return run_rows<__half>(g, e, p.vec, st);
    }
  }
  place_operand(&p.x, g->workspace);
  place_operand(&p.w, g->workspace);
  place_jobs(&p.jobs, g->workspace);
  if ((rc = run_stage(g->dtype, p.jobs, st))) return rc;
  return run_tensor_product(g->dtype, {p.x, p.w, g->K, e}, st);
}

// How k_layer_dz is cut: blocks of 256 columns for large arrays, of 32 columns x 64
// rows for small ones; rows a block such that there are several waves of blocks and
// a thread adds no more than 16 rows one after another for an f32 sum (64 for a
// 16-bit one), and one block for all rows where eight passes do (then it writes db
// itself and a launch is saved).  f32 db is off by 2^-23 of random sums' norm then;
// with 128 chains added in turn it was 2^-22.
struct DzShape {
  int vec, tx, rows, chunks;
};
static DzShape dz_shape(const fg_linear_grad_args *g) {
  DzShape d{};
  const int es = elem_size(g->dtype);
  d.vec = g->dy_col == 1 && rows16(g->dy, g->dy_row, es) &&
          (g->act == FG_ACT_NONE || rows16(g->pre, g->ld_pre, es));
  d.tx = (int64_t)g->M * g->N >= (4 << 20) ? 32 : 4;
  const int64_t strips = (g->N + 8LL * d.tx - 1) / (8 * d.tx), down = 256 / d.tx;
  const int64_t blocks = d.tx == 32 ? 4096 : 592;
  int64_t chunks = g->M <= 8 * down ? 1 : strips >= blocks ? 1 : blocks / strips;
  if (chunks > 128) chunks = 128;
  const int64_t deep = down * (es == 4 ? 16 : 64);
  if (g->M > 8 * down && chunks < (g->M + deep - 1) / deep) chunks = (g->M + deep - 1) / deep;
  if (chunks > 65535) chunks = 65535;  // of a grid's y
  const int64_t rows = ((g->M + chunks - 1) / chunks + down - 1) / down * down;
  d.rows = (int)(rows < 0x7fffff00 ? rows : 0x7fffff00);
  d.chunks = (int)((g->M + (int64_t)d.rows - 1) / d.rows);
  return d;
}

// dz is written (in a 16-bit type, or as the three planes of f32) where a
// product reads it and it differs from dy; x and w are read in place or staged.
struct GradPlan {
  bool dx, dw, make_dz;
  DzShape shape;
  int64_t ldz;
  size_t dz_off, part_off, bytes;
  Operand z_dx, z_dw, w, x;
  StageJobs jobs;
};
static GradPlan plan_grad(const fg_linear_grad_args *g) {
  GradPlan p{};
  p.dx = g->dx && g->K > 0;
  p.dw = g->dw && g->K > 0;
  p.make_dz = (p.dx || p.dw) && (g->dtype == FG_F32 || g->act != FG_ACT_NONE || g->drop.p > 0.0);
  p.shape = dz_shape(g);
  p.ldz = (g->N + 7LL) / 8 * 8;
  auto take = [&](size_t n) {
    const size_t o = (p.bytes + 255) / 256 * 256;
    p.bytes = o + n;
    return o;
  };
  const int planes = g->dtype == FG_F32 ? 3 : 1;
  p.dz_off = take(p.make_dz ? (size_t)planes * g->M * p.ldz * 2 : 0);
  p.part_off = take(g->db && p.shape.chunks > 1 ? (size_t)p.shape.chunks * g->N * 4 : 0);
  if (p.make_dz) {
    p.z_dx.staged_at = p.dz_off;
    p.z_dx.planes = planes;
    p.z_dx.inner = g->N, p.z_dx.outer = g->M, p.z_dx.pitch = p.ldz;
    p.z_dw = p.z_dx;  // read along its rows for dx, across them for dw
    p.z_dw.mn_major = 1;
  } else {
    if (p.dx)
      p.z_dx = resolve_operand(g->dtype, {g->dy, g->dy_row, g->dy_col}, g->M, g->N, &p.jobs,
                               &p.bytes);
    if (p.dx && !p.z_dx.ptr) {  // staged once for both
      p.z_dw = p.z_dx;
      p.z_dw.mn_major = !p.z_dx.mn_major;
    } else if (p.dw) {
      p.z_dw = resolve_operand(g->dtype, {g->dy, g->dy_col, g->dy_row}, g->N, g->M, &p.jobs,
                               &p.bytes);
    }
  }
  if (p.dx)
    p.w = resolve_operand(g->dtype, {g->w, g->w_col, g->w_row}, g->K, g->N, &p.jobs, &p.bytes);
  if (p.dw)
    p.x = resolve_operand(g->dtype, {g->x, g->x_col, g->x_row}, g->K, g->M, &p.jobs, &p.bytes);
  return p;
}

template <typename T>
static int run_dz(const fg_linear_grad_args *g, const GradPlan &p, const DropParams &drop,
                  const DzScale &by, cudaStream_t st) {
  char *ws = static_cast<char *>(g->workspace);
  const DzShape &d = p.shape;
  float *part = g->db && d.chunks > 1 ? reinterpret_cast<float *>(ws + p.part_off) : nullptr;
  const dim3 grid((unsigned)((g->N + 8LL * d.tx - 1) / (8 * d.tx)), d.chunks);
  int rc = launch_early(d.tx == 32 ? k_layer_dz<T, 32> : k_layer_dz<T, 4>, grid, 256, st,
                        static_cast<const T *>(g->dy), g->dy_row, g->dy_col,
                        static_cast<const T *>(g->pre), g->ld_pre, g->act, drop, by,
                        p.make_dz ? ws + p.dz_off : nullptr, p.ldz, part, static_cast<T *>(g->db),
                        g->M, g->N, d.rows, d.vec);
  if (rc || !part) return rc;
  return launch_early(k_bias_grad<T>, dim3((unsigned)((g->N + 31LL) / 32)), 1024, st, part,
                      d.chunks, g->N, static_cast<T *>(g->db));
}

static int check_grad(const fg_linear_grad_args *g, DropParams *drop) {
  const char *who = "fg_linear_grad";
  FG_REQUIRE(g, "%s: null arguments", who);
  int rc = check_common(who, g->dtype, g->M, g->N, g->K, g->act);
  if (rc) return rc;
  if ((rc = make_drop(who, &g->drop, drop))) return rc;
  const bool rows = g->M > 0 && g->N > 0;
  FG_REQUIRE(!rows || g->dy, "%s: null dy", who);
  FG_REQUIRE(!rows || g->act == FG_ACT_NONE || (g->pre && g->ld_pre >= g->N),
             "%s: the activation's slope needs the pre-activations", who);
  FG_REQUIRE(!(g->dx && rows && g->K > 0) || g->w, "%s: dx needs w", who);
  FG_REQUIRE(!(g->dw && rows && g->K > 0) || g->x, "%s: dw needs x", who);
  FG_REQUIRE((!g->dx || g->ld_dx >= g->K) && (!g->dw || g->ld_dw >= g->K),
             "%s: output pitch too small", who);
  const int es = elem_size(g->dtype);
  FG_REQUIRE(whole(es, g->dy, g->x, g->w, g->act ? g->pre : nullptr, g->dx,
                   g->dx ? g->dx_residual : nullptr, g->dw, g->db),
             "%s: an address is not a multiple of the element's size", who);
  struct Out {
    const char *name;
    const void *p;
    int64_t rows, cols, ld;
  } outs[3] = {{"dx", g->dx, g->M, g->K, g->ld_dx},
               {"dw", g->dw, g->N, g->K, g->ld_dw},
               {"db", g->db, 1, g->N, g->N}};
  for (int i = 0; i < 3; i++) {
    const Out &o = outs[i];
    FG_REQUIRE(
        !overlap(o.p, o.rows, o.cols, o.ld, g->x, g->M, g->K, g->x_row, g->x_col, es) &&
            !overlap(o.p, o.rows, o.cols, o.ld, g->w, g->N, g->K, g->w_row, g->w_col, es) &&
            !overlap(o.p, o.rows, o.cols, o.ld, g->dy, g->M, g->N, g->dy_row, g->dy_col, es) &&
            !overlap(o.p, o.rows, o.cols, o.ld, g->act ? g->pre : nullptr, g->M, g->N, g->ld_pre,
                     1, es),
        "%s: %s overlaps an operand", who, o.name);
    const bool same = i == 0 && g->dx_residual == g->dx && g->ld_dx_residual == g->ld_dx;
    FG_REQUIRE(same || !overlap(o.p, o.rows, o.cols, o.ld, g->dx ? g->dx_residual : nullptr, g->M,
                                g->K, g->ld_dx_residual, 1, es),
               "%s: %s overlaps dx_residual (only dx may, and only be all of it)", who, o.name);
    for (int j = i + 1; j < 3; j++)
      FG_REQUIRE(!overlap(o.p, o.rows, o.cols, o.ld, outs[j].p, outs[j].rows, outs[j].cols,
                          outs[j].ld, 1, es),
                 "%s: %s overlaps %s", who, o.name, outs[j].name);
  }
  return FG_OK;
}

static int zero_rows(void *p, int64_t ld, int64_t rows, int64_t cols, int es, cudaStream_t st) {
  if (!p || rows == 0 || cols == 0) return FG_OK;
  FG_CUDA_TRY(cudaMemset2DAsync(p, ld * es, 0, cols * es, rows, st));
  return FG_OK;
}

static int linear_grad(const fg_linear_grad_args *g, cudaStream_t st) {
  DropParams drop;
  int rc = check_grad(g, &drop);
  if (rc) return rc;
  const int es = elem_size(g->dtype);
  if (g->M == 0 || g->N == 0) {  // sums over nothing
    if (g->dx && g->M > 0 && g->K > 0) {
      Epilogue e{};
      e.out = g->dx, e.ldo = g->ld_dx;
      e.residual = g->dx_residual, e.ldr = g->ld_dx_residual;
      e.M = g->M, e.N = g->K;
      e.vec = rows16(e.out, e.ldo, es) && rows16(e.residual, e.ldr, es);
      if ((rc = run_empty_product(g->dtype, e, st))) return rc;
    }
    if ((rc = zero_rows(g->dw, g->ld_dw, g->N, g->K, es, st))) return rc;
    return zero_rows(g->db, g->N, 1, g->N, es, st);
  }
  GradPlan p = plan_grad(g);
  FG_REQUIRE(g->workspace_bytes >= p.bytes && (p.bytes == 0 || g->workspace),
             "fg_linear_grad: %zu bytes of workspace needed, got %zu", p.bytes,
             g->workspace_bytes);
  FG_REQUIRE(p.bytes == 0 || whole(256, g->workspace),
             "fg_linear_grad: the workspace is not on a 256-byte boundary");
  place_operand(&p.z_dx, g->workspace);
  place_operand(&p.z_dw, g->workspace);
  place_operand(&p.w, g->workspace);
  place_operand(&p.x, g->workspace);
  place_jobs(&p.jobs, g->workspace);
  if ((rc = run_stage(g->dtype, p.jobs, st))) return rc;
  // Dropout's scale multiplies the sums, and GELU's and SiLU's slopes, which reach
  // 1.13, act on halves in f16: the stored dz is finite where dy is.  (A half
  // costs values below 2^-13 a bit.)
  const bool steep = g->act != FG_ACT_NONE && g->act != FG_ACT_RELU;
  const float unit = g->dtype == FG_F16 && steep ? 0.5f : 1.0f;
  const DzScale by{unit, (drop.on && drop.some ? drop.scale : 1.0f) / unit};
  drop.scale = unit;
  if (p.make_dz || g->db) {
    switch (g->dtype) {
      case FG_F32:
        rc = run_dz<float>(g, p, drop, by, st);
        break;
      case FG_BF16:
        rc = run_dz<__nv_bfloat16>(g, p, drop, by, st);
        break;
      default:
        rc = run_dz<__half>(g, p, drop, by, st);
    }
    if (rc) return rc;
  }
  Product dx{p.z_dx, p.w, g->N, {}}, dw{p.z_dw, p.x, g->M, {}};
  dx.e.scale = dw.e.scale = p.make_dz ? by.after : 1.0f;
  // dx[m, k] = sum_n dz(m, n) w(n, k)
  dx.e.out = g->dx;
  dx.e.ldo = g->ld_dx;
  dx.e.residual = g->dx_residual;
  dx.e.ldr = g->ld_dx_residual;
  dx.e.M = g->M;
  dx.e.N = g->K;
  dx.e.vec = rows16(g->dx, g->ld_dx, es) && rows16(g->dx_residual, g->ld_dx_residual, es);
  // dw[n, k] = sum_m dz(m, n) x(m, k)
  dw.e.out = g->dw;
  dw.e.ldo = g->ld_dw;
  dw.e.M = g->N;
  dw.e.N = g->K;
  dw.e.vec = rows16(g->dw, g->ld_dw, es);
  if (p.dx && p.dw) return run_tensor_products(g->dtype, dx, dw, st);
  if (p.dx) return run_tensor_product(g->dtype, dx, st);
  if (p.dw) return run_tensor_product(g->dtype, dw, st);
  return FG_OK;
}

static int dropout(int dtype, int64_t rows, int64_t cols, const void *x, int64_t ldx,
                   const void *residual, int64_t ldr, void *out, int64_t ldo,
                   const fg_dropout_spec *spec, cudaStream_t st) {
  const char *who = "fg_dropout";
  const int es = elem_size(dtype);
  FG_REQUIRE(es > 0, "%s: dtype %d is not f32, bf16 or f16", who, dtype);
  FG_REQUIRE(rows >= 0 && cols >= 0 && rows <= 0x7fffffffLL && cols <= 0x7ffffff0LL,
             "%s: %lld x %lld is out of range", who, (long long)rows, (long long)cols);
  DropParams d;
  int rc = make_drop(who, spec, &d);
  if (rc) return rc;
  if (rows == 0 || cols == 0) return FG_OK;
  FG_REQUIRE(x && out, "%s: null operand", who);
  FG_REQUIRE(whole(es, x, residual, out), "%s: an address is not a multiple of the element's size",
             who);
  FG_REQUIRE(ldo >= cols || rows == 1, "%s: output pitch too small", who);
  FG_REQUIRE((x == out && ldx == ldo) || !overlap(out, rows, cols, ldo, x, rows, cols, ldx, 1, es),
             "%s: out overlaps x (it may only be all of it)", who);
  FG_REQUIRE((residual == out && ldr == ldo) ||
                 !overlap(out, rows, cols, ldo, residual, rows, cols, ldr, 1, es),
             "%s: out overlaps the residual (it may only be all of it)", who);
  const int vec = rows16(x, ldx, es) && rows16(residual, ldr, es) && rows16(out, ldo, es);
  const int64_t groups = rows * ((cols + 7) / 8);
  const int64_t per = 256 * (es == 2 ? DropGroups<__half>::value : DropGroups<float>::value);
  const int64_t blocks = (groups + per - 1) / per;
  FG_REQUIRE(blocks <= 0x7fffffffLL, "%s: %lld x %lld is out of range", who, (long long)rows,
             (long long)cols);
  const dim3 grid((unsigned)blocks);
  auto go = [&](auto kern, auto type) {
    using T = decltype(type);
    return launch_early(kern, grid, 256, st, static_cast<const T *>(x), ldx,
                        static_cast<const T *>(residual), ldr, static_cast<T *>(out), ldo, d, rows,
                        (int)cols, vec);
  };
  if (dtype == FG_F32) return go(k_dropout<float>, float{});
  if (dtype == FG_BF16) return go(k_dropout<__nv_bfloat16>, __nv_bfloat16{});
  return go(k_dropout<__half>, __half{});
}

}  // namespace layer
}  // namespace fg

extern "C" int fg_linear(const fg_linear_args *args, void *stream) {
  return fg::layer::linear(args, (cudaStream_t)stream);
}

extern "C" int fg_linear_workspace(const fg_linear_args *args, size_t *bytes) {
  FG_REQUIRE(args && bytes, "fg_linear_workspace: null argument");
  *bytes = 0;
  fg::layer::DropParams d;
  int rc = fg::layer::check_linear(args, &d);
  if (rc) return rc;
  *bytes = fg::layer::plan_linear(args).bytes;
  return FG_OK;
}

extern "C" int fg_linear_grad_workspace(const fg_linear_grad_args *args, size_t *bytes) {
  FG_REQUIRE(args && bytes, "fg_linear_grad_workspace: null argument");
  *bytes = 0;
  fg::layer::DropParams d;
  int rc = fg::layer::check_grad(args, &d);
  if (rc) return rc;
  if (args->M > 0 && args->N > 0) *bytes = fg::layer::plan_grad(args).bytes;
  return FG_OK;
}

extern "C" int fg_linear_grad(const fg_linear_grad_args *args, void *stream) {
  return fg::layer::linear_grad(args, (cudaStream_t)stream);
}

extern "C" int fg_dropout(int dtype, size_t rows, size_t cols, const void *d_x, int64_t ldx,
                          const void *d_residual, int64_t ldr, void *d_out, int64_t ldo,
                          const fg_dropout_spec *drop, void *stream) {
  FG_REQUIRE(rows <= 0x7fffffffu && cols <= 0x7ffffff0u, "fg_dropout: %zu x %zu is out of range",
             rows, cols);
  return fg::layer::dropout(dtype, (int64_t)rows, (int64_t)cols, d_x, ldx, d_residual, ldr, d_out,
                            ldo, drop, (cudaStream_t)stream);
}
