// Prints the kernels that layers_plan.h picks. stdin, a query a line:
//   product <rows> <ni> <nc> <bf16>  ->  fused|stream|tiles p q splits blocks per split
//   outer <rows> <n> <k>             ->  p q splits tokens per split
//   grids <rows> <n> <k>             ->  workgroups of the quantisation of dy with the copies of dy and x, of
//                                        y, of dx and of dw (0: not in tiles)
//   backward <rows> <n> <k> <bf16>   ->  1 where both products run in one launch
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "layers_plan.h"

int main() {
  char what[16];
  unsigned a, b, c, d;
  while (std::scanf("%15s %u %u %u", what, &a, &b, &c) == 4) {
    if (!std::strcmp(what, "outer")) {
      const nkplan::OuterPlan o = nkplan::outer_plan(a, b, c);
      std::printf("%u %u %u %u\n", o.p, o.q, o.splits, o.split_rows);
      continue;
    }
    if (!std::strcmp(what, "grids")) {
      using namespace nkplan;
      auto product = [&](unsigned ni, unsigned nc) -> unsigned long long {
        const ProductPlan p = product_plan(a, ni, nc, true);
        return p.form == kTiles ? tile_groups(ni, p.p, a, p.q, p.splits) : 0ull;
      };
      const OuterPlan o = outer_plan(a, b, c);
      std::printf("%llu %llu %llu %llu\n", 0ull + quant_groups(a, b) + copy_groups(a, up(b, 8)) + copy_groups(a, up(c, 8)),
                  product(b, c), product(c, b), 0ull + tile_groups(c, o.p, b, o.q, o.splits));
      continue;
    }
    if (std::scanf("%u", &d) != 1) return 1;
    if (!std::strcmp(what, "backward")) {
      std::printf("%d\n", nkplan::backward_in_one(nkplan::product_plan(a, c, b, d != 0), nkplan::outer_plan(a, b, c)));
      continue;
    }
    const nkplan::ProductPlan p = nkplan::product_plan(a, b, c, d != 0);
    static const char* const forms[] = {"fused", "stream", "tiles"};
    std::printf("%s %u %u %u %u\n", forms[p.form], p.p, p.q, p.splits, p.split_blocks);
  }
  return 0;
}
