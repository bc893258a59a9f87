// Operands that meet (csrc/moe_plan.hpp: overlap), against every byte of small
// regions, and at the ends of the address space.
#include <cstdio>
#include <vector>

#include "../../llm-inference-cpp_amd/csrc/moe_plan.hpp"

using namespace llmi_hip::moe;

namespace {
int bad = 0;
Region at(std::size_t address, std::size_t rows, std::size_t bytes, std::size_t stride) {
  return {reinterpret_cast<const void*>(address), rows, bytes, stride};
}
void expect(bool want, const Region& a, const Region& b, const char* what) {
  for (int turn = 0; turn < 2; ++turn)
    if (overlap(turn ? b : a, turn ? a : b) != want) {
      std::printf("%s: %p %zu %zu %zu, %p %zu %zu %zu is not %d\n", what, a.at, a.rows, a.bytes, a.stride, b.at, b.rows, b.bytes, b.stride, want);
      ++bad;
    }
}
bool by_bytes(const Region& a, const Region& b) {
  std::vector<bool> taken(512);
  const auto each = [](const Region& r, auto&& fn) {
    for (std::size_t i = 0; i < r.rows; ++i)
      for (std::size_t k = 0; k < r.bytes; ++k) fn(reinterpret_cast<std::uintptr_t>(r.at) + i * r.stride + k);
  };
  bool meets = false;
  each(a, [&](std::size_t p) { taken[p] = true; });
  each(b, [&](std::size_t p) { meets = meets || taken[p]; });
  return meets;
}
}  // namespace

int main() {
  for (std::size_t rows_a : {0, 1, 2, 3, 5})
    for (std::size_t rows_b : {1, 2, 4})
      for (std::size_t bytes_a : {1, 3, 4})
        for (std::size_t bytes_b : {1, 2, 5})
          for (std::size_t gap_a : {0, 1, 2, 7})
            for (std::size_t gap_b : {0, 1, 3, 6})
              for (std::size_t b = 100 - 40; b < 100 + 60; ++b) {
                const Region x = at(100, rows_a, bytes_a, bytes_a + gap_a), y = at(b, rows_b, bytes_b, bytes_b + gap_b);
                expect(by_bytes(x, y), x, y, "small regions");
              }
  // Columns of one array, up to the last row.
  const std::size_t base = std::size_t{1} << 40, rows = std::size_t{1} << 24;
  expect(false, at(base, rows, 256, 512), at(base + 256, rows, 256, 512), "columns");
  expect(true, at(base, rows, 256, 512), at(base + 252, rows, 256, 512), "columns");
  expect(true, at(base, rows, 256, 512), at(base + 256 + (rows - 1) * 512 - 4, 1, 4, 4), "last row");
  expect(false, at(base, rows, 256, 512), at(base + 256 + (rows - 1) * 512, 1, 4, 4), "behind the last row");
  expect(false, at(base, rows, 256, 512), at(base + 256, 2 * rows, 256, 1024), "every second row");
  expect(true, at(base, rows, 256, 512), at(base + 256, rows, 260, 1024), "every second row");
  // Strides that no memory has.
  const float* p = reinterpret_cast<const float*>(base);
  for (std::size_t stride : {SIZE_MAX, SIZE_MAX / 2 + 1, SIZE_MAX / 4 + 1, SIZE_MAX / 4})
    for (std::size_t n : {1, 3}) {
      expect(true, Region::matrix(p, n, 8, stride), Region::whole(p + 7, 4), "long strides");
      expect(false, Region::matrix(p, n, 8, stride), Region::whole(p + 8, 4), "long strides");
      expect(true, Region::matrix(p, n, 8, stride), Region::matrix(p + 4, 5, 8, 100), "long strides");
    }
  if (bad == 0) std::puts("ok");
  return bad != 0;
}
