// What a captured attention has room for (csrc/kv8_plan.hpp): every batch
// whose sequences have at most as many rows each as the captured batch's.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../llm-inference-cpp_amd/csrc/kv8_plan.hpp"

using namespace llmi_hip::kv8;

int main() {
  const std::vector<std::int32_t> table{0, 1};
  for (std::uint32_t group = 1; group <= 64; ++group)
    for (const std::uint32_t dim : {64u, 256u}) {
      const llmi_kv8_shape sh{2 * group, 2, dim, 4096, 2, 1};
      const auto lists = [&](std::int32_t count) {
        Lists l;
        const std::int32_t slot = 0, start = 900;
        if (!build(sh, 1, &slot, &start, &count, table.data(), 2, 1, 64, 2, &l).empty()) std::abort();
        return l;
      };
      for (std::int32_t count = 1; static_cast<std::uint32_t>(count) * group <= kFewMax; ++count) {
        const std::int32_t room = captured_rows(lists(count), static_cast<int>(dim));
        if (room > few_rows(static_cast<int>(dim)) || room % 4 != 0) return 1;
        for (std::int32_t less = 1; less <= count; ++less)
          if (lists(less).few_rows > room) {
            std::printf("%u heads a key/value head of %u: %d tokens make items of %d rows, captured for %d tokens: %d\n",
                        group, dim, less, lists(less).few_rows, count, room);
            return 1;
          }
      }
    }
  std::puts("ok");
  return 0;
}
