// The 8-bit products' plans (csrc/lrq_fp8plan.h), compiled by the host's own compiler: "rows cols depth nn" a line in, "mt nb
// splits steps" out.
#include <cstdio>

#include "../triton-kernel-test_amd/csrc/lrq_fp8plan.h"

int main() {
  long long rows, cols, depth;
  int nn;
  while (std::scanf("%lld %lld %lld %d", &rows, &cols, &depth, &nn) == 4) {
    const lrq::Plan8 p = lrq::plan8(rows, cols, depth, nn != 0);
    std::printf("%d %d %d %d\n", p.mt, p.nb, p.splits, p.steps);
  }
}
