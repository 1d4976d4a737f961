// Sweeps the shared-memory layout of the layer's products over every form,
// row count and alignment; prints the shapes that ask for more than a CTA can
// have or whose regions overlap.
#include <stdio.h>

#include "fg_layer_plan.h"

using namespace fg::layer;

static long tried = 0, bad = 0;

static void check(const SharedShape &s, size_t ring) {
  const SharedPlan p = lay_out(s, ring);
  const int bk = s.planes == 3 ? 32 : 64;
  const size_t stages = (size_t)p.stages * s.planes * (s.a_rows + s.b_rows) * bk * 2;
  const size_t sums = (size_t)((s.M < 128 ? s.M + 7 : 128) & ~7) * s.bn * 4;
  bool ok = p.bytes <= kSharedMax && p.stages >= (s.planes == 3 ? 2 : 1) && p.stages <= kMaxStages;
  if (s.cg == 1) {
    // header (1024, aligned), ring with the rows an MMA reads past it or the
    // CTA's sums, joined sums, slabs
    ok = ok && (size_t)p.join_at >= stages + 128 * bk * 2 && (size_t)p.join_at >= sums;
    ok = ok && (size_t)p.slab_at >= p.join_at + (s.split > 1 ? sums : 0);
    const size_t slabs = s.vec ? 0 : (size_t)block_warps(1, s.run) * kSplitSlab * 4;
    ok = ok && p.bytes >= 2048 + p.slab_at + slabs;
  } else {
    const size_t warp = s.io ? 4096 : 32 * kSlabPitch * 4;
    ok = ok && p.bytes >= 2048 + stages + block_epi_warps(2, s.run) * warp;
  }
  tried++;
  if (!ok && bad++ < 20)
    printf("planes %d cg %d bn %d run %d io %d M %d a %d b %d nk %d split %d vec %d: %zu bytes\n",
           s.planes, s.cg, s.bn, s.run, s.io, s.M, s.a_rows, s.b_rows, s.nk, s.split, s.vec,
           p.bytes);
}

int main() {
  const int depths[] = {1, 2, 3, 5, 8, 16, 31, 64, 128, 300, 5000};
  for (int planes = 1; planes <= 3; planes += 2)
    for (int nk : depths)
      for (int vec = 0; vec < 2; vec++) {
        for (int run = 0; run < 2; run++) {
          const size_t ring = (planes == 3 || run ? 192 : 160) * 1024;
          check({planes, 2, 256, run || planes == 3, vec != 0, 1000, 128, 128, nk, 1, vec != 0},
                ring);
        }
        for (int M = 1; M <= 130; M++)
          for (int unit = 16; unit <= 64; unit += 48)
            for (int bn = 64; bn <= (planes == 1 ? 128 : 64); bn *= 2)
              for (int split = 1; split <= (bn == 64 ? 8 : 4) && split <= nk; split *= 2)
                for (int many = 0; many < 2; many++)
                  for (int run = planes == 3; run < (bn == 64 ? 2 : 1); run++) {
                    const int rows = M >= 128 ? 128 : (M + unit - 1) / unit * unit;
                    const size_t ring = split_ring(many ? 149 : 148, 148, M, bn, split);
                    check({planes, 1, bn, run != 0, false, M, rows, bn, nk, split, vec != 0}, ring);
                    // beside a second product of more rows
                    check({planes, 1, bn, run != 0, false, M, rows, bn, nk, split, vec != 0},
                          split_ring(many ? 149 : 148, 148, 128, bn, split));
                  }
      }
  printf("%ld shapes, %ld bad\n", tried, bad);
  return bad != 0;
}
