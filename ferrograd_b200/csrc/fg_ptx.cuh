// Thin inline-PTX wrappers for sm_100a: mbarriers (with bounded waits), TMA
// tile loads (plain, this CTA only), tcgen05 TMEM allocation, MMA,
// commit and TMEM loads.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace fg {
namespace ptx {

// Bounded waits give up after this many SM clock cycles (~1 s at 1.9 GHz),
// set the kernel's error word and let the CTA wind down.
constexpr long long kWaitLimitCycles = 2000000000LL;

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count)
               : "memory");
}

__device__ __forceinline__ void fence_mbar_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Wait for the phase with the given parity to complete; false (and the error
// word set to `code`) if it did not within kWaitLimitCycles.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, unsigned int *err,
                                          unsigned int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() - t0 > kWaitLimitCycles) {
      if (err) atomicOr(err, code);
      return false;
    }
  }
  return true;
}

// mbar_wait whose polls may each suspend the thread for up to a millisecond,
// on a barrier given by its shared-memory address.
__device__ __forceinline__ bool mbar_try_suspended(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_suspended(uint32_t bar, uint32_t parity,
                                                    unsigned int *err, unsigned int code) {
  if (mbar_try_suspended(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_suspended(bar, parity)) {
    if (clock64() - t0 > kWaitLimitCycles) {
      if (err) atomicOr(err, code);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void prefetch_tmap(const CUtensorMap *m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)m) : "memory");
}

// 2-D tiled TMA load into this CTA's shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_2d(void *smem_dst, const CUtensorMap *map, uint64_t *bar,
                                            int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(smem_dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

// Orders this thread's earlier generic-proxy shared-memory accesses before
// later async-proxy (TMA) writes to the same shared memory.
__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// 3-D tiled TMA load into this CTA's shared memory, completing on `bar`.
__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *map, uint64_t *bar,
                                            int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// 2-D tiled TMA store from this CTA's shared memory, tracked by the thread's bulk
// groups.  Rows outside the tensor are not written; of a row, whole 16-byte pieces
// are: where it ends inside one, the rest is set to 0.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, const void *smem_src, int x,
                                             int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::
                   "l"((uint64_t)map),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() {
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Every store of this thread's committed groups has read its shared memory.
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

// Named barrier over `threads` threads; true if any of them passed true.
__device__ __forceinline__ bool named_bar_or(uint32_t id, uint32_t threads, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred.aligned q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

// ---- tcgen05 -------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t *slot_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(slot_smem)),
               "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// D[tmem] (+)= A[smem desc] * B[smem desc], kind::tf32, one CTA.
__device__ __forceinline__ void mma_tf32(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                         uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on `bar` once every tcgen05 op this thread issued so far completes.
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

// 32 lanes x 32 consecutive 32-bit columns: thread i gets row (lane base+i).
__device__ __forceinline__ void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptor (tcgen05 "matrix descriptor"):
//   [0,14) start address >> 4, [16,30) leading-dimension byte offset >> 4,
//   [32,46) stride-dimension byte offset >> 4, [46,48) version = 1,
//   [49,52) base offset = 0, [52] LBO mode = 0, [61,64) layout type.
// Layout types used here:
//   kLayoutSw128       (2): 128-byte swizzle of 16-byte chunks, 8-row atoms
//                           (K-major operands)
//   kLayoutSw128Base32 (1): 128-byte swizzle of 32-byte chunks, 4-row atoms --
//                           the only layout tcgen05 accepts for MN-major
//                           32-bit (tf32) operands
constexpr uint32_t kLayoutSw128 = 2;
constexpr uint32_t kLayoutSw128Base32 = 1;
//   kLayoutSw64        (4): 64-byte swizzle of 16-byte chunks, 8-row atoms of
//                           64-byte rows (K-major operands with 16-deep k-blocks)
constexpr uint32_t kLayoutSw64 = 4;
//   kLayoutSw32        (6): 32-byte swizzle of 16-byte chunks, 8-row atoms of
//                           32-byte rows (K-major operands with 8-deep k-blocks)
constexpr uint32_t kLayoutSw32 = 6;

__device__ __forceinline__ uint64_t smem_desc(uint32_t saddr, uint32_t lbo_bytes,
                                              uint32_t sbo_bytes, uint32_t layout) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo_bytes >> 4) & 0x3FFFu) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)(layout & 7u) << 61;
  return d;
}

// Instruction descriptor for kind::tf32 with fp32 accumulation:
//   [4,6) D format (1 = F32), [7,10) A format (2 = TF32), [10,13) B format,
//   [15] A MN-major, [16] B MN-major, [17,23) N >> 3, [24,29) M >> 4.
__host__ __device__ constexpr uint32_t idesc_tf32(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (2u << 7) | (2u << 10) | ((a_mn ? 1u : 0u) << 15) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// ---- 16-bit operands, CTA pairs and clusters --------------------------------
// Instruction descriptor for kind::f16 with fp32 accumulation: as idesc_tf32
// with formats 0 = F16, 1 = BF16 (A and B always alike).
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, bool bf16, bool a_mn, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
         ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// The instructions below are for a warp that passes through them whole: one
// elected lane (the same each time) runs them if `on`, the same in all lanes,
// is not 0.  Elected and predicated in one piece, not branched around by the
// caller, so that their operands stay in the warp's uniform registers: a loop
// in a branch of one lane took 600 cycles a step, mostly to move them.

// D[tmem] (+)= A * B, kind::f16, one CTA or a CTA pair (issued by its leader):
// STEPS k-steps of 16, the descriptors A_STEP and B_STEP apart; the first adds
// to D if accumulate.
template <int CG, int STEPS, int A_STEP, int B_STEP>
__device__ __forceinline__ void mma_f16_steps(uint32_t on, uint32_t d_tmem, uint64_t adesc,
                                              uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  static_assert(STEPS == 2 || STEPS == 4, "two or four steps");
#define FG_MMA(cg, a, b, p) \
  "@q tcgen05.mma.cta_group::" cg ".kind::f16 [%0], " a ", " b ", %3, " p ";\n\t"
#define FG_MMA_STEPS(cg)                                                                          \
  asm volatile(                                                                                   \
      "{\n\t.reg .pred p, q, e, t;\n\t.reg .b64 a, b;\n\t"                                        \
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"              \
      "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t" FG_MMA(cg, "%1", "%2", "p")         \
      "add.s64 a, %1, %6;\n\tadd.s64 b, %2, %7;\n\t" FG_MMA(cg, "a", "b", "t")                    \
      "}" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on),            \
      "n"(A_STEP), "n"(B_STEP)                                                                    \
      : "memory")
#pragma unroll
  for (int k = 0; k < STEPS; k += 2) {
    if (CG == 1)
      FG_MMA_STEPS("1");
    else
      FG_MMA_STEPS("2");
    adesc += 2 * A_STEP;
    bdesc += 2 * B_STEP;
    accumulate = 1;
  }
#undef FG_MMA_STEPS
#undef FG_MMA
}

// Arrive, once every tcgen05 op this thread issued so far completes, on the
// barrier at this shared-memory address, for a pair in both its CTAs.
template <int CG>
__device__ __forceinline__ void mma_commit_cg(uint32_t on, uint32_t bar) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
            bar),
        "r"(on)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster"
        ".b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"((uint16_t)3), "r"(on)
        : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t on, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
      "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes), "r"(on)
      : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc_cg(uint32_t *slot_smem, uint32_t ncols) {
  if (CG == 1) {
    tmem_alloc(slot_smem, ncols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(slot_smem)),
                 "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_cg(uint32_t taddr, uint32_t ncols) {
  if (CG == 1)
    tmem_dealloc(taddr, ncols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}

// The shared::cluster address of this CTA's shared-memory address in CTA `rank`.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  return a;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile(
      "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
          : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Copies bytes (a multiple of 16) of this CTA's shared memory into a CTA of the
// cluster, completing on a barrier there; both addresses shared::cluster.
__device__ __forceinline__ void bulk_copy_to_cta(uint32_t dst_cluster, uint32_t src, uint32_t bytes,
                                                 uint32_t bar_cluster) {
  asm volatile(
      "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes "
      "[%0], [%1], %2, [%3];" ::
          "r"(dst_cluster),
      "r"(src), "r"(bytes), "r"(bar_cluster)
      : "memory");
}
// Programmatic dependent launch: wait for the stream's previous kernel (and
// its memory) / let the next kernel start its prologue.
__device__ __forceinline__ void grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void grid_launch_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// Arrive on a barrier given by its shared::cluster address.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive_local(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Tiled TMA loads into this CTA's own shared memory.  Of a pair's, the bytes
// complete on a barrier given by its shared::cluster address (the leader's).
template <int CG>
__device__ __forceinline__ void tma_load_2d_cg(uint32_t on, uint32_t smem_dst,
                                               const CUtensorMap *map, uint32_t bar, int x, int y) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(smem_dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar), "r"(on)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
        "@q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier"
        "::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(smem_dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar), "r"(on)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_load_3d_cg(uint32_t on, uint32_t smem_dst,
                                               const CUtensorMap *map, uint32_t bar, int x, int y,
                                               int z) {
  if (CG == 1)
    asm volatile(
        "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %6, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(smem_dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(on)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q, e;\n\tsetp.ne.b32 e, %6, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\tand.pred q, q, e;\n\t"
        "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier"
        "::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::"r"(smem_dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(on)
        : "memory");
}

}  // namespace ptx
}  // namespace fg
