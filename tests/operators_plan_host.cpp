// Answers queries about csrc/layers/layers_plan.h on standard input, a line each.
#include <cstdio>
#include <cstring>

#include "layers_plan.h"

int main() {
  char what[32];
  while (std::scanf("%31s", what) == 1) {
    unsigned a, b, c, d, e;
    if (!std::strcmp(what, "norm") && std::scanf("%u %u", &a, &b) == 2) {
      const nkplan::NormPlan p = nkplan::norm_plan(a, b), g = nkplan::norm_gradients_plan(a, b);
      std::printf("%u %u %u %u %u %u\n", p.waves, p.chunks, p.rows, p.threads, p.groups, g.groups);
    } else if (!std::strcmp(what, "adapters") && std::scanf("%u %u %u %u %u", &a, &b, &c, &d, &e) == 5) {
      const nkplan::AdapterPlan p = nkplan::adapter_plan(a, b, c, d, e);
      std::printf("%u %u %u %u %u %u %u\n", nkplan::adapter_tile(a, b), nkplan::adapter_ranks(c), p.tiles, p.splits,
                  p.split_blocks, p.wide, p.fused ? 1u : 0u);
    } else if (!std::strcmp(what, "once") && std::scanf("%u %u %u %u", &a, &b, &c, &d) == 4) {
      std::printf("%u\n", nkplan::adapter_once(a, b, c, d) ? 1u : 0u);
    } else if (!std::strcmp(what, "codes") && std::scanf("%u %u %u", &a, &b, &c) == 3) {
      const nkplan::ProductPlan p = nkplan::codes_plan(a, b, c);
      std::printf("%u %u %u\n", static_cast<unsigned>(p.form), p.p, p.q);
    } else if (!std::strcmp(what, "select") && std::scanf("%u %u", &a, &b) == 2) {
      std::printf("%u\n", nkplan::select_groups(a, b));
    } else {
      return 1;
    }
  }
}
