// Reads lines "planes chain M K N" and prints, for the gradient of M x K -> N, 1 where
// dx and dw go out in one launch, else 0.
#include <stdio.h>

#include "fg_layer_plan.h"

using namespace fg::layer;

int main() {
  int planes, chain, M, K, N;
  while (scanf("%d %d %d %d %d", &planes, &chain, &M, &K, &N) == 5) {
    Form f;
    printf("%d\n", joint_form({M, K, N}, {N, K, M}, planes, chain, 148, &f) ? 1 : 0);
  }
  return 0;
}
