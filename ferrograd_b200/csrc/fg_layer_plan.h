// How a product of the layer's tensor-core kernel is cut up and laid out in
// shared memory (host code without CUDA, so that it can be swept over every
// shape on the CPU).
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>

namespace fg {
namespace layer {

constexpr int kMaxStages = 16;
// k-blocks of one accumulation chain.  The tensor cores cut the sum at each
// addition, so a chain drifts towards 0: measured on products of one sign, by
// 2^-15.3 of the sum over 4096 terms and 2^-13.3 over 16384.  A rounding to f16 is off
// by 2^-12.3 on average, to bf16 by 2^-9.3: the longer chain does not show in bf16,
// in f16 it makes the whole error 12% larger and the shorter one 1%.  f32 takes 64
// terms.
inline int chain_blocks(int planes, bool bf16) { return planes == 3 ? 2 : bf16 ? 256 : 64; }
constexpr size_t kSharedMax = 227 * 1024;  // what a CTA may ask for

constexpr int kSlabPitch = 20;   // floats; of a warp's 32 x 16 slab (pair)
constexpr int kSplitSlab = 384;  // floats; 8 x 36, 16 x 20 or 32 x 12 (split)

// Warps of a block (Block in fg_layer_gemm.cu).
constexpr int block_first_epi(int cg) { return cg == 2 ? 4 : 2; }
constexpr int block_epi_warps(int cg, bool run) { return cg == 1 ? 4 : run ? 8 : 16; }
constexpr int block_warps(int cg, bool run) {
  return cg == 1 ? 12 : block_first_epi(cg) + block_epi_warps(cg, run);
}

struct Form {
  bool pair;
  int bm, bn, split;
  double cost;  // estimated, in microseconds
};
// A product's rows, columns and depth.
struct Extent {
  int M, N, K;
};
inline int k_blocks(int K, int planes) {
  const int bk = planes == 3 ? 32 : 64;
  return (int)((K + (int64_t)bk - 1) / bk);
}
inline double mma_steps(int K, int planes) { return K / 16.0 * (planes == 3 ? 6.0 : 1.0); }

// Shared memory a CTA must ask for so that the CTAs that fit on an SM never
// need more than its 512 TMEM columns between them: an allocation that had to
// wait while its cluster's other CTAs hold theirs could wait for ever.
inline size_t tmem_share(int cols) { return (size_t)cols / 128 * 47 * 1024; }

// Shared memory of a split CTA's ring: with more CTAs than SMs two fit an SM, so
// that one computes while the other joins; less the joined sums.
inline size_t split_ring(int64_t ctas, int sms, int M, int bn, int split) {
  const size_t cap = (ctas > sms ? 92 : 190) * 1024;
  return split > 1 ? cap - (size_t)(M < 128 ? M : 128) * bn * 4 : cap;
}

// What a launch's shared memory depends on (vec: the outputs' rows start on
// 16-byte boundaries, so that the split form needs no slabs).
struct SharedShape {
  int planes, cg, bn;
  bool run, io;
  int M, a_rows, b_rows, nk, split;
  bool vec;
};
struct SharedPlan {
  int stages;
  int join_at, slab_at;  // split: offsets from the ring
  size_t bytes;
};

// Lays out a product's shared memory: its stages, as many as ring_cap holds
// and the rest leaves room for, and what follows the ring.
inline SharedPlan lay_out(const SharedShape &s, size_t ring_cap) {
  const int bk = s.planes == 3 ? 32 : 64;
  const size_t stage = (size_t)s.planes * (s.a_rows + s.b_rows) * bk * 2;
  // past the ring: the pair's blocks or slabs, or what an MMA of 128 rows reads
  // beyond an A tile of fewer (it lands in unused accumulator rows)
  const size_t tail =
      s.cg == 2 ? (size_t)block_epi_warps(s.cg, s.run) * (s.io ? 4096 : 32 * kSlabPitch * 4)
                : (size_t)128 * bk * 2;
  int64_t stages = (int64_t)(ring_cap / stage);
  if (stages > kMaxStages) stages = kMaxStages;
  if (s.cg == 1) {
    const int64_t per = ((int64_t)s.nk + s.split - 1) / s.split;
    if (stages > per) stages = per;
  }
  const int64_t least = s.planes == 3 ? 2 : 1;  // an f32 chain holds two k-blocks at once
  if (stages < least) stages = least;
  SharedPlan p{};
  for (;; stages--) {
    size_t bytes = stages * stage + tail;
    if (s.cg == 1) {
      const size_t sums = (size_t)((s.M < 128 ? s.M + 7 : 128) & ~7) * s.bn * 4;
      if (bytes < sums) bytes = sums;
      p.join_at = (int)((bytes + 127) & ~(size_t)127);
      if (s.split > 1) bytes = p.join_at + sums;
      p.slab_at = (int)((bytes + 127) & ~(size_t)127);
      if (!s.vec) bytes = p.slab_at + (size_t)block_warps(s.cg, s.run) * kSplitSlab * 4;
    }
    p.stages = (int)stages;
    p.bytes = bytes + 2048;  // barriers, alignment
    if (p.bytes <= kSharedMax || stages == least) break;
  }
  const size_t share = tmem_share(2 * s.bn);
  if (p.bytes < share) p.bytes = share;
  return p;
}

// The form with the least estimated time, in microseconds.  Fitted on one B200
// to every form of 17 shapes from 24 x 64 x 2048 to 2048 x 2048 x 2048 in 16 bits
// and f32: an MMA step (16 deep) costs a pair 0.07 and a lone CTA 0.038 at either
// width; around them a pair spends 6.8, a lone CTA 1.8 and for 128 rows another
// 1.9 (64 wide) or 3.4; joining a cluster's sums costs 0.7 and for 128 rows
// another 1.1 or 3.1.  64-wide CTAs run two to an SM and hide each other's fixed
// part.  It picks the fastest form or one within 10% of it on all 17, operands in L2 (24 x
// 8192 x 2048 f16: 64 wide, k over 8 CTAs, 10.2 against 22.7 unsplit and 42.4 by pairs;
// 1024 x 4096 x 4096 bf16: pairs, 27.6 against 35.1 and 48.3).
inline Form pick_form(const Extent &e, int planes, int chain, int sms) {
  const double steps = mma_steps(e.K, planes);
  const double pairs = ceil(e.M / 256.0) * ceil(e.N / 256.0);
  Form best{true, 256, 256, 1, ceil(pairs / (sms / 2)) * steps * 0.07 + 6.8};
  const int nk = k_blocks(e.K, planes);
  const double rows = e.M < 128 ? e.M / 128.0 : 1.0;
  for (int bn = 64; bn <= 128; bn *= 2)
    // (128-wide CTAs take one chain of 16-bit products, and run one to an SM, so
    // that not enough clusters of 8 fit)
    for (int split = 1; split <= (bn == 64 ? 8 : 4) && split <= nk; split *= 2) {
      if (bn == 128 && (planes == 3 || nk > (int64_t)chain * split)) continue;
      const double ctas = ceil(e.M / 128.0) * ceil((double)e.N / bn) * split;
      if (ctas > 1e8) continue;
      const double fixed = 1.8 + rows * (bn == 64 ? 1.9 : 3.4);
      const double join = split > 1 ? 0.7 + rows * (bn == 64 ? 1.1 : 3.1) : 0.0;
      const double per_sm =
          split > 1 || bn == 128 ? ceil(ctas / sms) : ctas > sms ? ctas / sms : 1.0;
      const double turns = bn == 64 ? ceil(ctas / (2.0 * sms)) : per_sm;
      const double c = 1.5 + join + turns * fixed + per_sm * steps / split * 0.038;
      if (c < best.cost) best = Form{false, 128, bn, split, c};
    }
  return best;
}

// Two independent products (a gradient's dx and dw) as 64-wide split tiles in one
// launch, with one split for both, as far as both have k-blocks and the CTAs one
// turn: whether that is possible, and cheaper than a launch for each in its own form.
// The longer product's CTAs bound it, or the SMs' share of all.  Of 31 gradients
// timed both ways (16-bit and f32, 64 to 16384 rows, widths 64 to 8192) the estimates'
// difference is within 5 us of the measured one for 25, and the slower way is picked for
// three, by 1 to 4 us of 22 to 29.  256 x 784 -> 128 f32 takes 15.0 us in one launch and 21.0
// in two, 512 x 1024 -> 1024 bf16 16.2 and 20.7; 8192 x 128 -> 128 bf16 34.7 and 21.5, 16384 x
// 128 -> 64 f32 260 and 58: its dw, deep and of two tiles, is split no further than dx allows.
inline bool joint_form(const Extent &x, const Extent &y, int planes, int chain, int sms, Form *f) {
  auto tiles_of = [](const Extent &e) {
    return (e.M + (int64_t)127) / 128 * ((e.N + (int64_t)63) / 64);
  };
  const int64_t tx = tiles_of(x), ty = tiles_of(y), tiles = tx + ty;
  const int nkx = k_blocks(x.K, planes), nky = k_blocks(y.K, planes);
  if (tiles > 2 * sms) return false;
  int split = 1;
  while (split < 8 && 2 * split <= nkx && 2 * split <= nky && tiles * 2 * split <= sms) split *= 2;
  if (planes == 1 && (nkx > chain * split || nky > chain * split)) return false;
  const double cx = mma_steps(x.K, planes) / split * 0.038;
  const double cy = mma_steps(y.K, planes) / split * 0.038;
  const double share = (double)split * (tx * cx + ty * cy) / sms;
  const double longer = cx > cy ? cx : cy;
  const int m = x.M > y.M ? x.M : y.M;
  const double rows = m < 128 ? m / 128.0 : 1.0;
  const double cost = 1.5 + (split > 1 ? 0.7 + rows * 1.1 : 0.0) + 1.8 + rows * 1.9 +
                      (longer > share ? longer : share);
  *f = Form{false, 128, 64, split, cost};
  return cost < pick_form(x, planes, chain, sms).cost + pick_form(y, planes, chain, sms).cost;
}

}  // namespace layer
}  // namespace fg
