// The layer's matrix products on the sm_100a tensor cores (tcgen05 + TMEM,
// operands by TMA):  C[m, n] = sum_k A(m, k) B(n, k), then the epilogue of
// fg_layer.cuh in the same kernel.
//
// 16-bit operands are read in place where TMA can describe them (one stride
// 1, the other and the base on 16-byte boundaries); others are first copied to
// an aligned layout (k_stage).  f32 operands are split into three bf16 planes,
// x = x0 + x1 + x2 with each rest exact, and a product runs as the six bf16
// products whose size is at least 2^-16 of the largest; what is dropped is
// 2^-24 of a product at most, or 2^-21 of one of large values (split3).
//
// The tensor cores truncate each addition to their f32 accumulator, so a long
// chain drifts towards 0.  A chain is therefore cut after `chain` k-blocks and
// the epilogue warps add the chains' sums, rounded to nearest, in registers
// while the next chain runs in the other TMEM buffer.  For f32 a chain is 64
// deep and adds its five small products first, so that only four additions
// meet a large accumulator.
//
// Two forms, chosen by pick_form:
//  pair   two CTAs (cta_group::2) on a 256 x 256 tile, persistent.  Each loads
//         128 rows of A and half of B, so an SM reads 64 bytes of shared
//         memory a cycle for its MMAs where a lone 128 x 256 CTA reads 96.
//  split  one CTA a 128 x BN tile, with k split over a cluster of up to 8 CTAs
//         that add their sums through distributed shared memory in rank order:
//         for few rows or few tiles.
//
// Large products are bound by the tensor cores, and those by power: 8192 x 4096 x
// 8192 bf16 without an epilogue takes 344 us, 1600 TFLOP/s (96% of cycles with an MMA),
// with GELU, dropout and pre 375 us, 1470 (90%); 16384 x 4096 x 16384 with them 1.5 ms
// in short runs, 1.77 ms, 1240 TFLOP/s, in long ones.  Operands of either order feed the
// MMAs alike (the gradient's dx and dw of the first, the latter MN-major twice, 334 us).
// f32: 8192 x 4096 x 4096 in 1.32 ms, six products of it 1250 TFLOP/s.  Small ones are
// bound by latencies: 24 x 8192 x 2048 f16 takes 11 us with the weight in L2 (14 from
// HBM), of which the cluster's join and the epilogue are 3.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <math.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "fg_internal.h"
#include "fg_layer.cuh"
#include "fg_layer_plan.h"
#include "fg_ptx.cuh"

namespace fg {
namespace layer {

using namespace fg::ptx;

using True = std::true_type;
using False = std::false_type;

constexpr unsigned kErrLayer = 5u << 16;  // device error word: role 5

// How an operand's tile lies in shared memory.  K-major: rows of BK elements
// (128- or 64-byte swizzle, 8-row atoms); MN-major: chunks of 64 rows, each BK
// k-rows of 128 bytes (128-byte swizzle, 8-k-row atoms).
struct OperandLayout {
  int mn_major;
  int rows;  // rows loaded a CTA (a multiple of 16; of 64 when MN-major)
};

struct ProductArgs {
  int M, N, nk;      // nk: k-blocks
  int chain;         // k-blocks of one accumulation chain
  int stages, split, group;
  int join_at;       // split: offsets from the ring of the joined sums
  int slab_at;       // and of the warps' slabs
  int bf16;
  OperandLayout a, b;
  unsigned int *err;
};

template <int PLANES>
struct Depth {
  static constexpr int BK = PLANES == 3 ? 32 : 64;
};

template <int PLANES>
__device__ __forceinline__ uint64_t desc_base(bool mn_major) {
  constexpr int BK = Depth<PLANES>::BK;
  return mn_major ? smem_desc(0, BK * 128, 1024, kLayoutSw128)
                  : smem_desc(0, 16, 8 * BK * 2, BK == 64 ? kLayoutSw128 : kLayoutSw64);
}

// Tile index -> (m block, n block), row blocks fastest in groups of `group`
// rows, so that the tiles in flight share panels of both operands in L2.
__device__ __forceinline__ void tile_at(int tile, int num_m, int num_n, int group, int &mb,
                                        int &nb) {
  const int per = group * num_n;
  const int g = tile / per;
  const int first = g * group;
  const int gm = min(group, num_m - first);
  const int r = tile - g * per;
  mb = first + r % gm;
  nb = r / gm;
}

constexpr int kBlockCols = 32;  // IO: a warp's block
constexpr int kSlabCols = 16;   // a warp's 32 x 16 slab (pair)

// The block of each form.  RUN: the epilogue warps keep the running sums of the
// chains in registers; without it a product is one chain and they read the
// accumulator where they need it, which leaves registers for twice the warps.
// split: four warps drain the accumulator, and all join in the epilogue, which
// six left waiting on its latencies (5200 cycles for a plain 128 x 64 tile).
template <int CG, bool RUN>
struct Block {
  static constexpr int first_epi = block_first_epi(CG);
  static constexpr int epi_warps = block_epi_warps(CG, RUN);
  static constexpr int warps = block_warps(CG, RUN);
  static constexpr int threads = 32 * warps;
};

// Case `at` of a switch: v = run[at .. at + 15].  The moves' texts differ, or the
// compiler joins the cases into one read of an indexed array in memory.
#define FG_TAKE16(at)                                                                       \
  case at:                                                                                  \
    for (int j = 0; j < 16; j++)                                                            \
      asm volatile("mov.f32 %0, %1; // " #at : "=f"(v[j / 8][j % 8]) : "f"(run[(at) % COLS + j])); \
    break;

// Tensor maps of a call: the operands, and where IO is set the output, the
// pre-activations and the residual.
struct Maps {
  CUtensorMap a, b, out, pre, residual;
};

// What a launch computes: one product, or two (split form) of which the first
// takes the first `ctas` CTAs.
struct Problem {
  Maps maps;
  ProductArgs g;
  Epilogue e;
};
template <bool TWO>
struct Problems {
  Problem at[TWO ? 2 : 1];
  int ctas;
};

// IO (pair form): out, pre and the residual pass through shared memory by TMA.
// At 64 bytes of operands in and 64 out a cycle, the MMAs of 16-bit operands
// leave next to nothing of shared memory's 128, and a warp's 16-byte global
// accesses to 32 rows cost it 32 passes; a TMA block costs 8 to write and 8 to
// read.  It needs rows on 16-byte boundaries that end on one.
template <typename T, int PLANES, int CG, int BN, bool RUN, bool IO, bool TWO>
__global__ void __launch_bounds__(Block<CG, RUN>::threads, CG == 1 && !RUN ? 2 : 1)
    k_layer_product(const __grid_constant__ Problems<TWO> ps) {
  const bool other = TWO && blockIdx.x >= ps.ctas;
  const Problem &pr = ps.at[TWO && other ? 1 : 0];
  const int block_id = TWO && other ? blockIdx.x - ps.ctas : blockIdx.x;
  const Maps &maps = pr.maps;
  const ProductArgs &g = pr.g;
  const Epilogue &e = pr.e;
  const CUtensorMap &tma = maps.a, &tmb = maps.b;
  constexpr int BK = Depth<PLANES>::BK;
  constexpr int kFirstEpi = Block<CG, RUN>::first_epi;  // first epilogue warp
  constexpr int kEpiWarps = Block<CG, RUN>::epi_warps;
  constexpr int COLS = BN * 4 / kEpiWarps;     // accumulator columns of an epilogue thread
  constexpr int BM = 128 * CG;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem);
  uint64_t *empty = full + kMaxStages;
  uint64_t *tmem_full = empty + kMaxStages;
  uint64_t *tmem_empty = tmem_full + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tmem_empty + 2);
  uint64_t *res_full = tmem_empty + 4;  // IO: a warp's block of the residual has landed
  uint8_t *ring = smem + 1024;
  // split: a CTA's sums go where its ring was, [BN / 4][row] of float4; each
  // rank's share of the columns, BN / split, is then copied to that rank's
  // `joined`, [source rank][BN / split / 4][row], completing on `join_bar`
  uint64_t *join_bar = tmem_empty + 4;
  float4 *sums = reinterpret_cast<float4 *>(ring);
  float4 *joined = reinterpret_cast<float4 *>(ring + (g.split > 1 ? g.join_at : 0));
  const uint32_t a_bytes = g.a.rows * (BK * 2), b_bytes = g.b.rows * (BK * 2);
  const uint32_t stage_bytes = PLANES * (a_bytes + b_bytes);

  // (the shuffle tells the compiler that a warp's index is the same in all its
  // lanes, and so the branches and operands that follow from it)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? block_id & 1 : block_id % g.split;  // in the cluster
  const bool leader = CG == 1 || rank == 0;
  const int num_m = (g.M + BM - 1) / BM, num_n = (g.N + BN - 1) / BN;
  const int S = g.stages;

  // This CTA's work: whole tiles (pair), or one tile's share of k (split).
  const int first = CG == 2 ? block_id / 2 : block_id / g.split;
  const int step = CG == 2 ? gridDim.x / 2 : num_m * num_n;
  const int k0 = CG == 2 ? 0 : (int)((long long)g.nk * rank / g.split);
  const int k1 = CG == 2 ? g.nk : (int)((long long)g.nk * (rank + 1) / g.split);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < S; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&tmem_full[i], 1);
      mbar_init(&tmem_empty[i], CG * kEpiWarps);  // one arrival a warp, from both CTAs
    }
    if (IO)
      for (int i = 0; i < kEpiWarps; i++) mbar_init(&res_full[i], 1);
    if (CG == 1) mbar_init(join_bar, 1);
    fence_mbar_init();
    prefetch_tmap(&tma);
    prefetch_tmap(&tmb);
  }
  if (warp == 1) tmem_alloc_cg<CG>(tmem_slot, 2 * BN);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync_all();  // the peer's barriers and TMEM are ready
  if (CG == 1 && g.split > 1) cluster_arrive();  // waited for before the first copy to a peer
  tc_fence_after();
  grid_wait();  // everything above overlaps the previous kernel's end
  if (CG == 1) grid_launch_next();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  // Pair with running sums: 384 threads x 168 registers at launch, of which the epilogue takes
  // 256 x 216 and the others keep 128 x 64.
  if (warp < kFirstEpi) {
    if (CG == 2 && RUN) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // Both loops below run in whole warps and are instantiated for each pair of
    // layouts.  After a wait that gave up they run on with everything switched
    // off, so that no branch of theirs hangs on a barrier's answer.
    const uint32_t on = 1;
    bool alive = true;
    const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), ring0 = smem_u32(ring);
    auto produce = [&](auto a_layout, auto b_layout) {
      // ---------------- TMA producer ----------------
      const uint32_t bars = CG == 2 ? map_to_rank(full0, 0) : full0;
      int s = 0, it = 0, last = 0;
      uint32_t phase = 0, go = on;
      for (int tile = first; tile < num_m * num_n; tile += step) {
        int mb, nb;
        tile_at(tile, num_m, num_n, g.group, mb, nb);
        const int m0 = mb * BM + (CG == 2 ? 128 * (int)rank : 0);
        const int n0 = nb * BN + (CG == 2 ? (BN / 2) * (int)rank : 0);
        for (int kb = k0; kb < k1; kb++, it++) {
          if (it >= S && alive &&
              !mbar_wait_suspended(empty0 + 8 * s, phase ^ 1, g.err, kErrLayer | 1))
            alive = false, go = 0, last = it;
          if (leader) mbar_expect_tx(go, full0 + 8 * s, CG * stage_bytes);
          uint32_t dst = ring0 + s * stage_bytes;
          const uint32_t bar = bars + 8 * s;
          auto load = [&](const CUtensorMap *map, auto layout, int rows, int r0, uint32_t bytes) {
            constexpr bool mn = decltype(layout)::value;
#pragma unroll
            for (int p = 0; p < PLANES; p++) {
#pragma unroll
              for (int c = 0; c < (mn ? 2 : 1); c++) {  // 128 rows at most
                if (mn && 64 * c >= rows) break;
                const int x = mn ? r0 + 64 * c : kb * BK, y = mn ? kb * BK : r0;
                if (PLANES == 1)
                  tma_load_2d_cg<CG>(go, dst + c * (BK * 128), map, bar, x, y);
                else
                  tma_load_3d_cg<CG>(go, dst + c * (BK * 128), map, bar, x, y, p);
              }
              dst += bytes;
            }
          };
          load(&tma, a_layout, g.a.rows, m0, a_bytes);
          load(&tmb, b_layout, g.b.rows, n0, b_bytes);
          if (++s == S) s = 0, phase ^= 1;
        }
      }
      // After a wait that gave up, loads in flight land before the CTA may
      // end: the leader sees them on its barriers; the peer, whose loads
      // complete on the leader's, lets a millisecond pass.
      if (!alive && leader)
        for (int i = last - S < 0 ? 0 : last - S; i < last; i++)
          mbar_wait(&full[i % S], (i / S) & 1, nullptr, 0);
      else if (!alive)
        for (const long long t0 = clock64(); clock64() - t0 < 2000000;) __nanosleep(1000);
    };
    auto multiply = [&](auto a_layout, auto b_layout) {
      constexpr bool a_mn = decltype(a_layout)::value, b_mn = decltype(b_layout)::value;
      // ---------------- MMA issuer ----------------
      const uint32_t idesc = idesc_f16(BM, BN, g.bf16, a_mn, b_mn);
      // a descriptor holds the 18 low bits of an address (those above name the
      // CTA within its cluster)
      const uint64_t da0 = desc_base<PLANES>(a_mn) + ((ring0 & 0x3ffffu) >> 4);
      const uint64_t db0 =
          desc_base<PLANES>(b_mn) + (((ring0 & 0x3ffffu) + PLANES * a_bytes) >> 4);
      // 16 elements further in k: 32 bytes inside a swizzled row, or 16 k-rows
      constexpr int a_step = (a_mn ? 2048 : 32) >> 4, b_step = (b_mn ? 2048 : 32) >> 4;
      const uint32_t tmem_full0 = smem_u32(tmem_full), tmem_empty0 = smem_u32(tmem_empty);
      int s = 0, local = 0;
      uint32_t phase = 0, go = on;
      for (int tile = first; tile < num_m * num_n; tile += step)
        for (int c0 = k0; c0 < k1; c0 += g.chain, local++) {
          const int c1 = min(c0 + g.chain, k1);
          const int buf = local & 1;
          if (local >= 2 && alive &&
              !mbar_wait_suspended(tmem_empty0 + 8 * buf, ((local >> 1) - 1) & 1, g.err,
                                   kErrLayer | 2))
            alive = false, go = 0;
          tc_fence_after();
          const uint32_t d = tmem_base + buf * BN;
          uint32_t acc = 0;
          const int s_first = s;
          auto products = [&](int st, int pa, int pb) {
            const uint64_t da = da0 + ((st * stage_bytes + pa * a_bytes) >> 4);
            const uint64_t db = db0 + ((st * stage_bytes + pb * b_bytes) >> 4);
            mma_f16_steps<CG, BK / 16, a_step, b_step>(go, d, da, db, idesc, acc);
            acc = 1;
          };
          for (int kb = c0; kb < c1; kb++) {
            if (alive && !mbar_wait_suspended(full0 + 8 * s, phase, g.err, kErrLayer | 3))
              alive = false, go = 0;
            tc_fence_after();
            if (PLANES == 1) {
              products(s, 0, 0);
              mma_commit_cg<CG>(go, empty0 + 8 * s);
            } else {  // the small products of the whole chain first
              products(s, 2, 0);
              products(s, 0, 2);
              products(s, 1, 1);
              products(s, 1, 0);
              products(s, 0, 1);
            }
            if (++s == S) s = 0, phase ^= 1;
          }
          if (PLANES == 3) {
            int t = s_first;
            for (int kb = c0; kb < c1; kb++) {
              products(t, 0, 0);
              mma_commit_cg<CG>(go, empty0 + 8 * t);
              if (++t == S) t = 0;
            }
          }
          mma_commit_cg<CG>(go, tmem_full0 + 8 * buf);
        }
    };
    auto by_layout = [&](auto role) {
      if (g.a.mn_major)
        g.b.mn_major ? role(True{}, True{}) : role(True{}, False{});
      else
        g.b.mn_major ? role(False{}, True{}) : role(False{}, False{});
    };
    if (warp == 0)
      by_layout(produce);
    else if (warp == 1 && leader)
      by_layout(multiply);
  } else if (warp < kFirstEpi + kEpiWarps) {
    if (CG == 2 && RUN) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ---------------- epilogue ----------------
    const int q = warp & 3;  // the TMEM lanes this warp may read
    const int part = (warp - kFirstEpi) / 4;  // its columns: COLS of the tile's BN
    const uint32_t t_addr = tmem_base + ((uint32_t)(32 * q) << 16) + part * COLS;
    const uint32_t lead_empty0 = CG == 2 ? map_to_rank(smem_u32(&tmem_empty[0]), 0) : 0;
    int local = 0;
    bool dead = false;  // a wait gave up: touch nothing more, but keep every barrier
    auto release = [&](int buf) {  // this warp has read its part of a TMEM buffer
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2)
          mbar_arrive_cluster(lead_empty0 + buf * 8);
        else
          mbar_arrive_local(&tmem_empty[buf]);
      }
    };
    auto arrived = [&](int chain_no) {  // a chain's sums are in its buffer
      // One lane of four warps polls, and they sleep at a barrier: sixteen
      // polling warps cost the MMAs 4% through the shared memory they share.
      if (q == (kFirstEpi & 3) && lane == 0 && !dead)
        dead = !mbar_wait_suspended(smem_u32(&tmem_full[chain_no & 1]), (chain_no >> 1) & 1, g.err,
                                    kErrLayer | 4);
      __syncwarp();
      dead = named_bar_or(1 + part, 128, dead);
      tc_fence_after();
      return !dead;
    };
    // 16 columns of a pair's tile through the warp's slab, so that lanes hold
    // eight neighbouring columns (rows off 16-byte boundaries)
    float *slab = reinterpret_cast<float *>(ring + S * stage_bytes) +
                  (warp - kFirstEpi) * (32 * kSlabPitch);
    auto finish16 = [&](int row0, int col0) {
      __syncwarp();
#pragma unroll 1
      for (int p = 0; p < 2; p++) {
        float v[8];
        load8<float>(slab + (p * 16 + lane / 2) * kSlabPitch + (lane & 1) * 8, v);
        epilogue_slab<T>(e, slab + p * 16 * kSlabPitch, 4, row0 + 16 * p, col0, lane / 2,
                         (lane & 1) * 8, v);
      }
    };
    // IO: this warp's block of 32 rows x 32 columns in shared memory (swizzled
    // rows of 64 or 128 bytes; a lane holds a row).  Out and pre leave through
    // it, the residual arrives in it; the previous use is over once its store
    // has read it.
    // 16-bit types have a second block for pre, and one pass fills both; f32
    // writes pre and then out through the one that fits.
    constexpr int BC = kBlockCols, kRow = BC * sizeof(T);
    constexpr bool kTwo = sizeof(T) == 2;
    uint8_t *block = ring + S * stage_bytes + (warp - kFirstEpi) * ((kTwo ? 64 : 32) * kRow);
    uint64_t *res_bar = &res_full[warp - kFirstEpi];
    uint32_t res_phase = 0;
    auto chunk = [&](int j) {
      const int x = kRow == 128 ? lane & 7 : (lane >> 1) & 3;
      return block + lane * kRow + ((j ^ x) << 4);
    };
    auto pre_chunk = [&](int j) { return chunk(j) + (kTwo ? 32 * kRow : 0); };
    auto block_free = [&] {
      if (lane == 0) bulk_wait_read();
      __syncwarp();
    };
    auto block_store = [&](const CUtensorMap *map, const uint8_t *from, int row0, int col) {
      if (lane == 0) {
        tma_store_2d(map, from, col, row0);
        bulk_commit();
      }
    };
    auto residual_load = [&](int row0, int col) {
      block_free();
      if (lane == 0) {
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(res_bar, 32 * kRow);
        tma_load_2d(block, &maps.residual, res_bar, col, row0);
      }
    };
    // One block: sums(c, v) gives the sums of columns col + c .. col + c + 15.
    auto finish_block = [&](int row0, int col, bool loaded,
                            auto sums) __attribute__((always_inline)) {
      const int row = row0 + lane;
      if (!kTwo && e.pre) {
        block_free();
#pragma unroll 1
        for (int c = 0; c < BC; c += 16) {
          float v[2][8];
          sums(c, false, v);
#pragma unroll
          for (int p = 0; p < 2; p++) {
            affine8<T>(e, col + c + 8 * p, v[p]);
            store8_smem<T>(pre_chunk, c + 8 * p, v[p]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        block_store(&maps.pre, block, row0, col);
      }
      if (e.residual) {
        if (!loaded) residual_load(row0, col);
        if (lane == 0 && !dead)
          dead = !mbar_wait_suspended(smem_u32(res_bar), res_phase, g.err, kErrLayer | 5);
        dead = __any_sync(0xffffffffu, dead);
        res_phase ^= 1;
      } else {
        block_free();
      }
#pragma unroll 1
      for (int c = 0; c < BC; c += 16) {
        float v[2][8];
        sums(c, true, v);
#pragma unroll
        for (int p = 0; p < 2; p++) {
          affine8<T>(e, col + c + 8 * p, v[p]);
          if (kTwo && e.pre) store8_smem<T>(pre_chunk, c + 8 * p, v[p]);
          act8<sizeof(T) == 2>(v[p], e.act);
          if (e.drop.on) drop8(e.drop, row, col + c + 8 * p, v[p]);
          if (e.residual) {
            float t[8];
            load8_smem<T>(chunk, c + 8 * p, t);
#pragma unroll
            for (int i = 0; i < 8; i++) v[p][i] += t[i];
          }
          store8_smem<T>(chunk, c + 8 * p, v[p]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (kTwo && e.pre) block_store(&maps.pre, block + 32 * kRow, row0, col);
      block_store(&maps.out, block, row0, col);
    };
    // split: sends each rank its share of this CTA's sums
    auto share = [&](int pitch) {
      if (g.split == 1) return;
      fence_proxy_async_smem();
      __syncwarp();
      cluster_wait();  // the peers have started: their barriers are set up
      if (!named_bar_or(1, 128, dead) && warp == kFirstEpi && lane < g.split) {
        const uint32_t bytes = BN / g.split / 4 * pitch * 16;
        if (lane == 0) mbar_arrive_expect_tx(join_bar, g.split * bytes);
        bulk_copy_to_cta(map_to_rank(smem_u32(joined) + rank * bytes, lane),
                         smem_u32(sums) + lane * bytes, bytes,
                         map_to_rank(smem_u32(join_bar), lane));
      }
    };
    for (int tile = first; tile < num_m * num_n; tile += step) {
      int mb, nb;
      tile_at(tile, num_m, num_n, g.group, mb, nb);
      const int row0 = mb * BM + 128 * (int)rank + 32 * q;  // of a pair
      const int col0 = nb * BN + part * COLS;
      const bool inside = row0 < g.M && col0 < g.N;
      if constexpr (!RUN && IO) {
        const int buf = local & 1;
        const bool early = inside && e.residual;
        if (early) residual_load(row0, col0);
        if (arrived(local++)) {
#pragma unroll 1
          for (int b = 0; b < COLS; b += BC) {
            const bool some = inside && col0 + b < g.N;
            if (some)
              finish_block(row0, col0 + b, early && b == 0, [&](int c, bool last, float(&v)[2][8]) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(t_addr + buf * BN + b + c, r);
                tmem_ld_wait();
                if (last && b + c + 16 >= COLS) release(buf);
#pragma unroll
                for (int j = 0; j < 16; j++) v[j / 8][j % 8] = __uint_as_float(r[j]);
              });
            else if (b + BC >= COLS)
              release(buf);
          }
        }
        continue;
      }
      if constexpr (!RUN && CG == 1) {
        const int pitch = (min(128, g.M - mb * BM) + 7) & ~7, row = 32 * q + lane;
        if (arrived(local++)) {
#pragma unroll 1
          for (int c = 0; c < COLS; c += 16) {
            uint32_t r[16];
            tmem_ld_32x32b_x16(t_addr + c, r);
            tmem_ld_wait();
            if (row < pitch) {
#pragma unroll
              for (int j = 0; j < 16; j += 4)
                sums[(c + j) / 4 * pitch + row] =
                    make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]),
                                __uint_as_float(r[j + 2]), __uint_as_float(r[j + 3]));
            }
          }
        }
        share(pitch);
        continue;
      }
      if constexpr (!RUN) {
        const int buf = local & 1;
        if (arrived(local++)) {
#pragma unroll 1
          for (int c = 0; c < COLS; c += kSlabCols) {
            uint32_t r[16];
            tmem_ld_32x32b_x16(t_addr + buf * BN + c, r);
            tmem_ld_wait();
            if (c + kSlabCols >= COLS) release(buf);
            if (row0 >= g.M || col0 + c >= g.N) continue;
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kSlabCols; j += 4)
              *reinterpret_cast<uint4 *>(slab + lane * kSlabPitch + j) =
                  make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
            finish16(row0, col0 + c);
          }
        }
        continue;
      }
      if constexpr (RUN) {
        float run[COLS];
#pragma unroll
        for (int j = 0; j < COLS; j++) run[j] = 0.0f;
        for (int c0 = k0; c0 < k1; c0 += g.chain, local++) {
          if (arrived(local)) {
#pragma unroll
            for (int c = 0; c < COLS; c += 32) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(t_addr + (local & 1) * BN + c, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; j++) run[c + j] += __uint_as_float(r[j]);
            }
            release(local & 1);
          }
        }
        if (IO) {
          if (dead || !inside) continue;
#pragma unroll 1
          for (int b = 0; b < COLS; b += BC) {
            if (col0 + b >= g.N) break;
            finish_block(row0, col0 + b, false, [&](int c, bool, float(&v)[2][8])
                                                    __attribute__((always_inline)) {
              switch (b + c) {
                FG_TAKE16(0)
                FG_TAKE16(16)
                FG_TAKE16(32)
                FG_TAKE16(48)
                FG_TAKE16(64)
                FG_TAKE16(80)
                FG_TAKE16(96)
                FG_TAKE16(112)
              }
            });
          }
        } else if (CG == 2) {
          if (dead || row0 >= g.M) continue;
#pragma unroll 1
          for (int c = 0; c < COLS / kSlabCols; c++) {
            if (col0 + c * kSlabCols >= g.N) break;
            __syncwarp();
#pragma unroll
            for (int cc = 0; cc < COLS / kSlabCols; cc++)
              if (cc == c) {
#pragma unroll
                for (int j = 0; j < kSlabCols; j += 4)
                  *reinterpret_cast<float4 *>(slab + lane * kSlabPitch + j) =
                      make_float4(run[cc * kSlabCols + j], run[cc * kSlabCols + j + 1],
                                  run[cc * kSlabCols + j + 2], run[cc * kSlabCols + j + 3]);
              }
            finish16(row0, col0 + c * kSlabCols);
          }
        } else {
          const int pitch = (min(128, g.M - mb * BM) + 7) & ~7;  // rows, a multiple of 8
          const int row = 32 * q + lane;
          if (!dead && row < pitch) {
#pragma unroll
            for (int j = 0; j < COLS; j += 4)
              sums[j / 4 * pitch + row] = make_float4(run[j], run[j + 1], run[j + 2], run[j + 3]);
          }
          share(pitch);
        }
      }
    }
  }

  if (CG == 1) {
    __syncwarp();
    if (g.split > 1) {
      if (warp < kFirstEpi || warp >= kFirstEpi + kEpiWarps) cluster_wait();
      mbar_wait(join_bar, 0, g.err, kErrLayer | 6);
      __syncwarp();
      cluster_arrive();  // (every copy into this CTA is done; waited for at the end)
    } else {
      __syncthreads();
    }
    // add this rank's columns in rank order and apply the epilogue
    int mb, nb;
    tile_at(first, num_m, num_n, g.group, mb, nb);
    const int rows = min(128, g.M - mb * BM), pitch = (rows + 7) & ~7;
    // a warp takes a power of two, gw <= 4, groups of eight columns of 32 / gw
    // rows at a time: eight lanes read 128 neighbouring bytes, gw lanes write a
    // row's
    const int own = BN / g.split, lgroups = 31 - __clz(own / 8);
    const int lgw = min(lgroups, 2), lrw = 5 - lgw, lacross = lgroups - lgw;
    const int r_in = lane & ((1 << lrw) - 1), c_in = (lane >> lrw) * 8;
    const int pieces = ((rows + (1 << lrw) - 1) >> lrw) << lacross;
    const int col0 = nb * BN + (int)rank * own;
    float *slab = reinterpret_cast<float *>(ring + g.slab_at) + warp * kSplitSlab;
    for (int t = warp; t < pieces; t += Block<CG, RUN>::warps) {
      const int r0 = (t >> lacross) << lrw;
      const int c0 = (t & ((1 << lacross) - 1)) << (lgw + 3);
      const int r = r0 + r_in, col = col0 + c0 + c_in;
      const float4 *x = joined + (c0 + c_in) / 4 * pitch + (r < rows ? r : 0);
      float v[8] = {};
#pragma unroll 4
      for (int k = 0; k < g.split; k++, x += own / 4 * pitch) {  // the ranks' sums, in order
        const float4 lo = x[0], hi = x[pitch];
        v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
        v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
      }
      if (!e.vec)
        epilogue_slab<T>(e, slab, lgw + 3, mb * BM + r0, col0 + c0, r_in, c_in, v);
      else if (r < rows && col < g.N)
        epilogue8<T>(e, mb * BM + r, col, v);
    }
  }
  if (IO && warp >= kFirstEpi && lane == 0) bulk_wait_read();
  tc_fence_before();
  __syncthreads();
  // no CTA leaves while another may still reach its memory
  if (CG == 2) cluster_sync_all();
  if (CG == 1 && g.split > 1) cluster_wait();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_cg<CG>(tmem_base, 2 * BN);
  }
}

// ---------------------------------------------------------------------------
// Operands TMA cannot read in place: copied to [plane][outer][pitch] with
// the contiguous direction innermost; f32 as three bf16 planes.  Bound by HBM and,
// where a row starts off a 16-byte boundary, by its narrower reads: 8192 x 4096 and
// 4096 x 4096 f32 are split in 77 us (0.5 GB, 6.5 TB/s).
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void stage_store(uint4 *dst, int64_t plane16, const float (&v)[8]) {
  if (sizeof(T) == 2) {
    store8<T>(reinterpret_cast<T *>(dst), v);
  } else {
    float p[3][8];
#pragma unroll
    for (int j = 0; j < 8; j++) split3(v[j], p[0][j], p[1][j], p[2][j]);
#pragma unroll
    for (int k = 0; k < 3; k++)
      store8<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16 *>(dst + k * plane16), p[k]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) k_stage(const StageJobs jobs) {
  const StageJob &j = jobs.job[blockIdx.y];
  const int groups = (int)(j.pitch / 8);
  const int64_t plane = groups * j.outer;
  const T *src = static_cast<const T *>(j.src);
  uint4 *dst = static_cast<uint4 *>(j.dst);
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  grid_wait();
  grid_launch_next();
  for (Walk at(j.outer, groups, first, step); at.inside(); at.next()) {
    const int64_t x = (int64_t)at.group * 8;
    float v[8];
    if (j.vec && x + 8 <= j.inner) {
      load8<T>(src + at.row * j.so + x, v);
    } else if (j.si == 1 && x + 8 <= j.inner) {
      load8_off<T>(src + at.row * j.so + x, src, src + (j.outer - 1) * j.so + j.inner, v);
    } else {
#pragma unroll
      for (int k = 0; k < 8; k++)
        v[k] = x + k < j.inner ? to_f32<T>(src[at.row * j.so + (x + k) * j.si]) : 0.0f;
    }
    stage_store<T>(dst + at.row * groups + at.group, plane, v);
  }
}

int run_stage(int dtype, const StageJobs &jobs, cudaStream_t st) {
  if (jobs.n == 0) return FG_OK;
  int64_t most = 0;
  for (int i = 0; i < jobs.n; i++) {
    const int64_t all = jobs.job[i].pitch / 8 * jobs.job[i].outer;
    if (all > most) most = all;
  }
  const int64_t want = (most + 255) / 256;
  const dim3 grid((unsigned)(want < 148 * 8 ? want : 148 * 8), jobs.n);
  if (dtype == FG_F32) return launch_early(k_stage<float>, grid, 256, st, jobs);
  if (dtype == FG_BF16) return launch_early(k_stage<__nv_bfloat16>, grid, 256, st, jobs);
  return launch_early(k_stage<__half>, grid, 256, st, jobs);
}

Operand resolve_operand(int dtype, const Mat &m, int64_t rows, int64_t k, StageJobs *jobs,
                        size_t *ws) {
  Operand o{};
  o.planes = dtype == FG_F32 ? 3 : 1;
  const bool base = (uintptr_t)m.ptr % 16 == 0;
  // (rows that overlap or repeat are copied: a tensor map's may not)
  auto pitch_ok = [](int64_t ld, int64_t outer, int64_t inner) {
    return outer == 1 || (ld >= inner && ld % 8 == 0);
  };
  if (dtype != FG_F32 && base && (m.col == 1 || k == 1) && pitch_ok(m.row, rows, k)) {
    o.ptr = m.ptr;
    o.inner = k, o.outer = rows;
    o.pitch = rows == 1 ? (k + 7) / 8 * 8 : m.row;
    return o;
  }
  if (dtype != FG_F32 && base && (m.row == 1 || rows == 1) && pitch_ok(m.col, k, rows)) {
    o.ptr = m.ptr;
    o.mn_major = 1;
    o.inner = rows, o.outer = k;
    o.pitch = k == 1 ? (rows + 7) / 8 * 8 : m.col;
    return o;
  }
  // staged with the source's contiguous direction innermost
  StageJob j{};
  o.mn_major = m.col != 1 && m.row == 1;
  o.inner = o.mn_major ? rows : k;
  o.outer = o.mn_major ? k : rows;
  o.pitch = (o.inner + 7) / 8 * 8;
  o.staged_at = (*ws + 255) / 256 * 256;
  *ws = o.staged_at + (size_t)o.planes * o.outer * o.pitch * 2;
  j.src = m.ptr;
  j.so = o.mn_major ? m.col : m.row;
  j.si = o.mn_major ? m.row : m.col;
  j.outer = o.outer, j.inner = o.inner, j.pitch = o.pitch;
  const int es = dtype == FG_F32 ? 4 : 2;
  j.vec = j.si == 1 && base && (j.so * es) % 16 == 0;
  j.at = o.staged_at;
  jobs->job[jobs->n++] = j;
  return o;
}

void place_operand(Operand *o, void *ws) {
  if (!o->ptr) o->ptr = static_cast<char *>(ws) + o->staged_at;
}
void place_jobs(StageJobs *jobs, void *ws) {
  for (int i = 0; i < jobs->n; i++) jobs->job[i].dst = static_cast<char *>(ws) + jobs->job[i].at;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void *ptr = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)ptr;
  });
  return fn;
}

// [planes][outer][pitch] of 16-bit elements, or [outer][pitch]; one box is box_rows K-major rows
// of BK elements, or BK k-rows of 64 MN-major elements.
static int make_map(CUtensorMap *map, const Operand &o, int bk, int box_rows, bool bf16) {
  auto fn = encode_fn();
  if (!fn) return set_error(FG_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t pitch = (cuuint64_t)o.pitch * 2;
  const cuuint64_t dims[3] = {(cuuint64_t)o.inner, (cuuint64_t)o.outer, (cuuint64_t)o.planes};
  const cuuint64_t strides[2] = {pitch, pitch * (cuuint64_t)o.outer};
  const cuuint32_t box[3] = {(cuuint32_t)(o.mn_major ? 64 : bk),
                             (cuuint32_t)(o.mn_major ? bk : box_rows), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(
      map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
      o.planes == 1 ? 2 : 3, const_cast<void *>(o.ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
      o.mn_major || bk == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(FG_ERR_CUDA,
                     "cuTensorMapEncodeTiled failed (%d): inner=%lld outer=%lld pitch=%lld", (int)r,
                     (long long)o.inner, (long long)o.outer, (long long)o.pitch);
  return FG_OK;
}

// [M, N] with pitch ld, in blocks of 32 x 32 (rows of 64 or 128 bytes, swizzled).
template <typename T>
static int make_io_map(CUtensorMap *map, const void *ptr, int M, int N, int64_t ld) {
  auto fn = encode_fn();
  if (!fn) return set_error(FG_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * sizeof(T)};
  const cuuint32_t box[2] = {kBlockCols, 32};
  const cuuint32_t estr[2] = {1, 1};
  // 16-bit types are only moved, so either 16-bit map type serves
  const CUresult r =
      fn(map, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
         2, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         sizeof(T) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(FG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): %d x %d, pitch %lld", (int)r,
                     M, N, (long long)ld);
  return FG_OK;
}

template <typename T, int PLANES, int CG, int BN, bool RUN, bool IO, bool TWO>
static int launch(Problems<TWO> &ps, int ctas, size_t ring_cap, cudaStream_t st) {
  auto kern = k_layer_product<T, PLANES, CG, BN, RUN, IO, TWO>;
  size_t bytes = 0;
  for (Problem &pr : ps.at) {
    ProductArgs &g = pr.g;
    const SharedPlan p = lay_out({PLANES, CG, BN, RUN, IO, g.M, g.a.rows, g.b.rows, g.nk, g.split,
                                  pr.e.vec != 0},
                                 ring_cap);
    g.stages = p.stages;
    g.join_at = p.join_at;
    g.slab_at = p.slab_at;
    if (bytes < p.bytes) bytes = p.bytes;
  }
  static std::atomic<bool> attr_done[64];  // (callers on several threads)
  int dev = 0;
  FG_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    FG_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)kSharedMax));
    if (dev >= 0 && dev < 64) attr_done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(Block<CG, RUN>::threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG == 2 ? 2 : ps.at[0].g.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ps));
  count_launch();
  return FG_OK;
}

static int64_t tiles_of(const Epilogue &e, int bm, int bn) {
  return (e.M + (int64_t)bm - 1) / bm * ((e.N + (int64_t)bn - 1) / bn);
}

template <typename T, int PLANES>
static int run_form(const Form &f, Problems<false> &ps, int sms, cudaStream_t st) {
  Maps &maps = ps.at[0].maps;
  const ProductArgs &g = ps.at[0].g;
  const Epilogue &e = ps.at[0].e;
  const int64_t tiles = tiles_of(e, f.bm, f.bn);
  if (f.pair) {
    const int pairs = sms / 2;
    const int ctas = 2 * (int)(tiles < pairs ? tiles : pairs);
    // 16-bit: five stages of 32 KB (a sixth gains nothing) beside sixteen
    // warps' two blocks of 2 KB; f32: four of 48 KB beside eight of 4 KB
    constexpr bool kLong = PLANES == 3;
    const size_t ring = (kLong ? 192 : 160) * 1024;
    // (a tensor map's rows may not repeat, and a TMA store fills up a row's last 16
    // bytes: beyond N it would write zeros over what lies there.  8192 x 4096 -> 8190
    // bf16 in rows of 8192 takes 358 us through slabs, 8192 columns by TMA 348.)
    if (e.vec && (int64_t)e.N * sizeof(T) % 16 == 0 && (!e.residual || e.ldr >= e.N)) {
      int rc = make_io_map<T>(&maps.out, e.out, e.M, e.N, e.ldo);
      if (!rc && e.pre) rc = make_io_map<T>(&maps.pre, e.pre, e.M, e.N, e.ldp);
      if (!rc && e.residual) rc = make_io_map<T>(&maps.residual, e.residual, e.M, e.N, e.ldr);
      if (rc) return rc;
      if (g.chain >= g.nk) return launch<T, PLANES, 2, 256, kLong, true, false>(ps, ctas, ring, st);
      return launch<T, PLANES, 2, 256, true, true, false>(ps, ctas, 192 * 1024, st);
    }
    if (g.chain >= g.nk) return launch<T, PLANES, 2, 256, kLong, false, false>(ps, ctas, ring, st);
    return launch<T, PLANES, 2, 256, true, false, false>(ps, ctas, 192 * 1024, st);
  }
  const int64_t ctas = tiles * f.split;
  const size_t ring = split_ring(ctas, sms, g.M, f.bn, f.split);
  // one chain needs no running sums, except f32's, which are many
  if (PLANES == 3 || (int64_t)g.chain * g.split < g.nk)
    return launch<T, PLANES, 1, 64, true, false, false>(ps, (int)ctas, ring, st);
  if constexpr (PLANES == 1) {
    if (f.bn == 128) return launch<T, 1, 1, 128, false, false, false>(ps, (int)ctas, ring, st);
    return launch<T, 1, 1, 64, false, false, false>(ps, (int)ctas, ring, st);
  }
}

// Two products whose tiles do not fill the SMs by themselves, in one launch of
// 64-wide split tiles with the same split.
template <typename T, int PLANES>
static int run_two(Problems<true> &ps, int64_t ctas, int sms, cudaStream_t st) {
  const int m = ps.at[0].g.M > ps.at[1].g.M ? ps.at[0].g.M : ps.at[1].g.M;
  const size_t ring = split_ring(ctas, sms, m, 64, ps.at[0].g.split);
  return launch<T, PLANES, 1, 64, PLANES == 3, false, true>(ps, (int)ctas, ring, st);
}

static int make_problem(Problem *pr, int dtype, const Operand &a, const Operand &b, int K,
                        const Epilogue &e, const Form &f, unsigned int *err) {
  const int planes = dtype == FG_F32 ? 3 : 1, bk = planes == 3 ? 32 : 64;
  const bool bf16 = dtype != FG_F16;
  ProductArgs &g = pr->g;
  g.M = e.M;
  g.N = e.N;
  g.nk = k_blocks(K, planes);
  g.chain = chain_blocks(planes, bf16);
  g.split = f.split;
  g.group = f.pair ? 16 : 8;
  g.bf16 = bf16;
  g.err = err;
  const int unit_a = a.mn_major ? 64 : 16;
  g.a.mn_major = a.mn_major;
  g.a.rows = f.pair || e.M >= 128 ? 128 : (e.M + unit_a - 1) / unit_a * unit_a;
  g.b.mn_major = b.mn_major;
  g.b.rows = f.pair ? 128 : f.bn;
  pr->e = e;
  int rc = make_map(&pr->maps.a, a, bk, g.a.rows, bf16);
  return rc ? rc : make_map(&pr->maps.b, b, bk, g.b.rows, bf16);
}

int run_tensor_product(int dtype, const Product &x, cudaStream_t st) {
  DevCtx *ctx = ctx_current();
  if (!ctx) return set_error(FG_ERR_CUDA, "no CUDA device context");
  const int sms = ctx->num_sms ? ctx->num_sms : 148;
  const int planes = dtype == FG_F32 ? 3 : 1;
  const Form f =
      pick_form({x.e.M, x.e.N, x.K}, planes, chain_blocks(planes, dtype != FG_F16), sms);
  Problems<false> ps = {};
  int rc = make_problem(&ps.at[0], dtype, x.a, x.b, x.K, x.e, f, ctx->d_err);
  if (rc) return rc;
  switch (dtype) {
    case FG_F32:
      return run_form<float, 3>(f, ps, sms, st);
    case FG_BF16:
      return run_form<__nv_bfloat16, 1>(f, ps, sms, st);
    default:
      return run_form<__half, 1>(f, ps, sms, st);
  }
}

// Two independent products, in one launch where that is cheaper.
int run_tensor_products(int dtype, const Product &x, const Product &y, cudaStream_t st) {
  DevCtx *ctx = ctx_current();
  if (!ctx) return set_error(FG_ERR_CUDA, "no CUDA device context");
  const int sms = ctx->num_sms ? ctx->num_sms : 148;
  const int planes = dtype == FG_F32 ? 3 : 1;
  Form f;
  if (!joint_form({x.e.M, x.e.N, x.K}, {y.e.M, y.e.N, y.K}, planes,
                  chain_blocks(planes, dtype != FG_F16), sms, &f)) {
    int rc = run_tensor_product(dtype, x, st);
    return rc ? rc : run_tensor_product(dtype, y, st);
  }
  const int64_t tx = tiles_of(x.e, 128, 64) * f.split, ctas = tx + tiles_of(y.e, 128, 64) * f.split;
  Problems<true> ps = {};
  ps.ctas = (int)tx;
  int rc = make_problem(&ps.at[0], dtype, x.a, x.b, x.K, x.e, f, ctx->d_err);
  if (rc) return rc;
  if ((rc = make_problem(&ps.at[1], dtype, y.a, y.b, y.K, y.e, f, ctx->d_err))) return rc;
  switch (dtype) {
    case FG_F32:
      return run_two<float, 3>(ps, ctas, sms, st);
    case FG_BF16:
      return run_two<__nv_bfloat16, 1>(ps, ctas, sms, st);
    default:
      return run_two<__half, 1>(ps, ctas, sms, st);
  }
}

}  // namespace layer
}  // namespace fg
