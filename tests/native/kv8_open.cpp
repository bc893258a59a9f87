// The open-block store of the paged 8-bit key/value cache: random appends
// under one slot, which go on, are taken back (again and again) or begin at
// whole blocks, walked through the work lists (csrc/kv8_plan.hpp).  Where
// Held::serves allows a start inside a block, the rows that the append reads
// from the store are the sequence's own; where it does not, some are not.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "../../llm-inference-cpp_amd/csrc/kv8_plan.hpp"

using namespace llmi_hip::kv8;

int main() {
  std::mt19937 rng(7);
  const auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); };
  const llmi_kv8_shape sh{1, 1, 32, 4096, 1, 1};
  long allowed = 0, refused = 0, twice = 0;
  for (int walk = 0; walk < 3000; ++walk) {
    int store[2][kBlk];            // the write that each row holds, -1: none
    std::vector<int> own(4096, -1);  // the write that each position of the sequence came from, -1: none
    for (auto& half : store) std::fill(half, half + kBlk, -1);
    Held held;
    int length = 0, write = 0, backs = 0;
    for (int step = 0; step < 30; ++step) {
      const int kind = pick(0, 9);
      std::int32_t start = kind < 4 ? length : kind < 8 ? pick(std::max(0, length - 50), length) : 16 * pick(0, length / 16 + 1);
      std::int32_t count = pick(0, 2) == 0 ? pick(1, 70) : pick(1, 6);
      if (start + count > 4000) break;
      // The rows that the append reads from the store, against the sequence's.
      bool right = true;
      for (int p = start / kBlk * kBlk; p < start; ++p)
        right = right && own[static_cast<std::size_t>(p)] >= 0 && store[p / kBlk & 1][p % kBlk] == own[static_cast<std::size_t>(p)];
      if (held.serves(start) != right) {
        std::printf("walk %d step %d: start %d of %d tokens, length %d: allowed %d, rows right %d\n", walk, step, start, count, length,
                    held.serves(start), right);
        return 1;
      }
      if (!right) {
        ++refused;
        continue;
      }
      ++allowed;
      if (start < length && start % kBlk != 0) twice += ++backs > 1;
      if (start >= length) backs = 0;
      const std::int32_t slot = 0, page = 0;
      Lists l;
      if (!build(sh, 1, &slot, &start, &count, &page, 1, 1, 4096, 1, &l).empty()) return 2;
      for (int p = start; p < start + count; ++p) own[static_cast<std::size_t>(p)] = write++;
      std::fill(own.begin() + start + count, own.end(), -1);
      // Blocks in any order; one wavefront does a block and the one at then_pos.
      std::shuffle(l.blocks.begin(), l.blocks.end(), rng);
      for (const BlockItem& it : l.blocks)
        for (const int pos : {it.pos, it.then_pos}) {
          if (pos < 0) continue;
          for (int p = pos; p < std::min(it.start, pos + kBlk); ++p)
            if (store[p / kBlk & 1][p % kBlk] != own[static_cast<std::size_t>(p)]) return 3;
          for (int p = std::max({pos, it.keep, it.start}); p < std::min(it.end, pos + kBlk); ++p)
            store[p / kBlk & 1][p % kBlk] = own[static_cast<std::size_t>(p)];
        }
      held.wrote(start, count);
      length = start + count;
    }
  }
  std::printf("ok: %ld allowed (%ld taken back again), %ld refused\n", allowed, twice, refused);
  return allowed > 1000 && twice > 100 && refused > 100 ? 0 : 4;
}
