// Long histories against the limits that a plan is created for
// (csrc/kv8_plan.hpp): a batch within its sequences and tokens makes no more
// work than limits() gives, at the lengths where the size of a piece changes.
#include <cstdio>
#include <vector>

#include "../../llm-inference-cpp_amd/csrc/kv8_plan.hpp"

using namespace llmi_hip::kv8;

int main() {
  for (const std::uint32_t kv : {1u, 2u, 3u, 8u, 9u})
    for (const std::uint32_t dim : {64u, 256u})
      for (const int rows : {1, 8, 20, 64, 65, 66, 72, 100, 127, 128, 129}) {
        // `group` query heads a key/value head, as few tokens as give these rows.
        const int group = rows % 8 == 0 ? 8 : rows % 3 == 0 ? 3 : 1, tokens = rows / group;
        const llmi_kv8_shape sh{kv * static_cast<std::uint32_t>(group), kv, dim, 65536, 64, 2};
        std::vector<std::int32_t> table(64);
        for (int i = 0; i < 64; ++i) table[static_cast<std::size_t>(i)] = i;
        for (const std::size_t target : {kFewTarget, kManyTarget, kUnits})
          for (const std::size_t least : {kFewLeast, kManyLeast})
            for (std::size_t times = 1; times <= 8; ++times) {
              // Positions x heads from this many pieces of `times` x least on to past one more.
              const std::size_t at = target * least * times / kv;
              for (std::size_t len = at > 3 ? at - 3 : 1; len < at + target / kv + 3; len += 1 + (len > at + 4 && len + 8 < at + target / kv ? 5 : 0)) {
                if (len > 3000000 || len < static_cast<std::size_t>(tokens)) continue;
                const std::int32_t slot = 0, count = tokens, start = static_cast<std::int32_t>(len) - tokens;
                Lists l;
                const std::string why = build(sh, 1, &slot, &start, &count, table.data(), 64, 1, static_cast<std::size_t>(tokens), 64, &l);
                const Limits m = limits(sh, 1, static_cast<std::size_t>(tokens));
                if (!why.empty() || l.blocks.size() > m.blocks || l.few.size() > m.few || l.many.size() > m.many || l.parts > m.parts ||
                    l.join.size() > m.join) {
                  std::printf("%u/%u heads of %u, %d tokens after %d positions: %s; few %zu of %zu, many %zu of %zu, parts %zu of %zu, joins %zu of %zu\n",
                              sh.heads, kv, dim, tokens, start, why.c_str(), l.few.size(), m.few, l.many.size(), m.many, l.parts, m.parts, l.join.size(), m.join);
                  return 1;
                }
              }
            }
      }
  std::puts("ok");
  return 0;
}
