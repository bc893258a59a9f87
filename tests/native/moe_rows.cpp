// Which kernels a call of llmi_hip_moe_matmul_dev or _mlp_dev takes, by the
// rules of csrc/moe_plan.hpp: from lines of
//   matmul <type> <experts> <out> <in> <slots> <per_row>
//   mlp <type> <down's type> <experts> <hidden> <ffn> <tokens> <top_k>
// lines of "few", or of the rows of a group of each product and how slots are
// grouped ("self": every wavefront for itself, "tiles": rows brought into row
// tiles behind the grouping, "rows": rows as they are).
#include <cstdio>
#include <cstring>

#include "../../llm-inference-cpp_amd/csrc/moe_plan.hpp"

using namespace llmi_hip::moe;

namespace {
const char* grouping(std::size_t slots, std::size_t experts, std::size_t rows) {
  return rows > kMostShortRows ? "rows" : self_grouped(slots, experts) ? "self" : "tiles";
}
}  // namespace

int main() {
  char kind[16];
  while (std::scanf("%15s", kind) == 1) {
    if (std::strcmp(kind, "matmul") == 0) {
      Shape s;
      std::size_t slots, per_row;
      if (std::scanf("%d %zu %zu %zu %zu %zu", &s.type, &s.count, &s.out, &s.in, &slots, &per_row) != 6) return 1;
      const std::size_t rows = pick_rows(s, slots, false);
      if (few_matmul(s, slots, per_row)) std::puts("few");
      else std::printf("%zu %s\n", rows, grouping(slots, s.count, rows));
    } else {
      Shape gate, down;
      std::size_t hidden, ffn, tokens, top_k;
      if (std::scanf("%d %d %zu %zu %zu %zu %zu", &gate.type, &down.type, &gate.count, &hidden, &ffn, &tokens, &top_k) != 7) return 1;
      down.count = gate.count;
      gate.out = down.in = ffn;
      gate.in = down.out = hidden;
      const MlpRows rows = pick_mlp_rows(gate, down, tokens * top_k);
      if (few_mlp(tokens, top_k)) std::puts("few");
      else std::printf("%zu %zu %s\n", rows.first, rows.second, grouping(tokens * top_k, gate.count, rows.first));
    }
  }
  return 0;
}
