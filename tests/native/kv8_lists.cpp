// Walks the work lists of the paged 8-bit key/value cache (csrc/kv8_plan.hpp)
// for random batches: every block of new tokens is written once, inside its
// sequence's table, and no open-block row is replaced before the wavefront
// that needs it has read it.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <utility>

#include "../../llm-inference-cpp_amd/csrc/kv8_plan.hpp"

#define CHECK(c)                                                     \
  do {                                                               \
    if (!(c)) {                                                      \
      std::printf("%s:%d: %s\n", __FILE__, __LINE__, #c);            \
      return 1;                                                      \
    }                                                                \
  } while (0)

using namespace llmi_hip::kv8;

int main() {
  std::mt19937 rng(1);
  const auto pick = [&](int lo, int hi) { return lo + static_cast<int>(rng() % static_cast<unsigned>(hi - lo + 1)); };
  for (int round = 0; round < 3000; ++round) {
    llmi_kv8_shape sh{};
    sh.kv_heads = static_cast<std::uint32_t>(pick(1, 4));
    sh.heads = sh.kv_heads * static_cast<std::uint32_t>(pick(1, 20));
    sh.head_dim = 32u * static_cast<std::uint32_t>(pick(1, 8));
    sh.page_tokens = 16u * static_cast<std::uint32_t>(pick(1, 5));
    const int n = pick(0, 6);
    sh.slots = 6;
    std::vector<std::int32_t> slots, starts, counts;
    std::size_t stride = 1, pages = 1, tokens = 0;
    const int longest = pick(0, 2) == 0 ? 4000 : 120;
    for (int i = 0; i < n; ++i) {
      slots.push_back(i);
      starts.push_back(pick(0, longest));
      counts.push_back(pick(0, 3) == 0 ? pick(0, 300) : pick(0, 5));
      const std::size_t need = (static_cast<std::size_t>(starts.back() + counts.back()) + sh.page_tokens - 1) / sh.page_tokens;
      stride = std::max(stride, need);
      pages += need;
      tokens += static_cast<std::size_t>(counts.back());
    }
    sh.pages = static_cast<std::uint32_t>(pages);
    std::vector<std::int32_t> tables(stride * static_cast<std::size_t>(n), -1);
    std::int32_t next = 0;
    for (int i = 0; i < n; ++i)
      for (std::size_t p = 0; p * sh.page_tokens < static_cast<std::size_t>(starts[static_cast<std::size_t>(i)] + counts[static_cast<std::size_t>(i)]); ++p)
        tables[static_cast<std::size_t>(i) * stride + p] = next++;
    Lists l;
    const std::string why = build(sh, static_cast<std::size_t>(n), slots.data(), starts.data(), counts.data(), tables.data(), stride, 6, 4000, 4000, &l);
    CHECK(why.empty());
    CHECK(l.writable && l.tokens == tokens);
    std::set<std::pair<int, int>> written;  // page, block of it
    std::size_t blocks = 0;
    for (const BlockItem& it : l.blocks) {
      std::size_t of = 0;  // the sequence with these tokens
      while (l.seqs[of].count == 0 || l.seqs[of].row != it.row) ++of;
      const Seq& s = l.seqs[of];
      CHECK(it.start == s.start && it.end == s.start + s.count && it.slot == s.slot);
      const int last = (it.end - 1) / kBlk, per = static_cast<int>(sh.page_tokens) / kBlk;
      CHECK(it.keep == (last - 1) * kBlk);
      for (int k = 0; k < 2; ++k) {
        const int pos = k == 0 ? it.pos : it.then_pos, page = k == 0 ? it.page : it.then_page, block = k == 0 ? it.block : it.then_block;
        if (pos < 0) continue;
        CHECK(pos % kBlk == 0 && pos + kBlk > it.start && pos < it.end);
        CHECK(page == l.table[static_cast<std::size_t>(s.table + pos / kBlk / per)] && block == pos / kBlk % per);
        CHECK(written.insert({page, block}).second);
        ++blocks;
      }
      // A block that reads rows of the store, against every other writer of
      // the same rows (blocks last and last - 1, by parity).
      if (it.pos < s.start)
        for (int b = last - 1; b <= last; ++b)
          if (b > it.pos / kBlk && b % 2 == it.pos / kBlk % 2) CHECK(it.then_pos == b * kBlk);
    }
    std::size_t all = 0;
    for (const Seq& s : l.seqs) {
      if (s.count > 0) all += static_cast<std::size_t>((s.start + s.count - 1) / kBlk - s.start / kBlk + 1);
      for (int i = 0; i < s.count; ++i) CHECK(l.positions.at(static_cast<std::size_t>(s.row + i)) == s.start + i);
    }
    CHECK(blocks == all && l.positions.size() == tokens);
    // Attention: every row and position it may see once, each partial state
    // in slots of its own, and within the limits that a plan is created for.
    const std::size_t group = sh.heads / sh.kv_heads;
    std::vector<std::vector<long>> reach(l.seqs.size());
    for (std::size_t i = 0; i < l.seqs.size(); ++i) reach[i].assign(static_cast<std::size_t>(l.seqs[i].count) * group, 0);
    std::vector<int> slot(l.parts, 0);
    const int few_most = few_rows(static_cast<int>(sh.head_dim));
    const auto walk = [&](const std::vector<AttnItem>& items, int most, bool few) {
      for (const AttnItem& it : items) {
        CHECK(it.rows > 0 && it.rows <= most && it.lo % kTile == 0 && it.lo < it.hi);
        std::size_t of = 0;  // the sequence with these tokens
        while (l.seqs[of].count == 0 || l.seqs[of].row != it.row) ++of;
        const Seq& s = l.seqs[of];
        CHECK(it.start == s.start && it.table == s.table);
        const std::size_t rows = static_cast<std::size_t>(s.count) * group;
        CHECK((rows <= kFewMax) == few && static_cast<std::size_t>(it.row0 + it.rows) <= rows);
        CHECK(it.hi <= s.start + s.count);
        for (int r = it.row0; r < it.row0 + it.rows; ++r) {
          const int own = s.start + r / static_cast<int>(group);  // the row's position
          reach[of][static_cast<std::size_t>(r)] += std::max(0, std::min(it.hi, own + 1) - it.lo);
        }
        if (it.part < 0) continue;
        for (int k = 0; k < most / kSlotRows; ++k) CHECK(++slot.at(static_cast<std::size_t>(it.part + k)) == 1);
        int joins = 0;  // that read this piece, and are of these rows
        for (const JoinItem& j : l.join)
          if (it.part >= j.part && it.part < j.part + j.n * j.step) {
            CHECK(j.row == it.row && j.row0 == it.row0 && j.rows == it.rows && j.rows <= l.join_rows);
            CHECK(j.step == most / kSlotRows && (it.part - j.part) % j.step == 0 && j.n > 1);
            ++joins;
          }
        CHECK(joins == 1);
      }
      return 0;
    };
    CHECK(walk(l.few, few_most, true) == 0 && walk(l.many, kManyRows, false) == 0);
    for (std::size_t i = 0; i < l.seqs.size(); ++i)
      for (std::size_t r = 0; r < reach[i].size(); ++r) CHECK(reach[i][r] == l.seqs[i].start + static_cast<long>(r / group) + 1);
    for (const int n_of : slot) CHECK(n_of == 1);
    const Limits m = limits(sh, static_cast<std::size_t>(n), tokens);
    CHECK(l.blocks.size() <= m.blocks && l.few.size() <= m.few && l.many.size() <= m.many);
    CHECK(l.parts <= m.parts && l.join.size() <= m.join);
  }
  for (std::uint32_t d = 1; d <= 4096; ++d) {
    const Divisor v = divisor(d);
    for (std::uint32_t q = 0; q < 40; ++q)
      for (std::uint32_t x : {q * d, q * d + d - 1, (1u << 27) - 1 - q, ((1u << 27) - 1) / d * d - (q < 1 ? 0 : q * d), static_cast<std::uint32_t>(rng()) >> 5})
        CHECK(x >= (1u << 27) || (std::uint64_t{x} * v.m) >> v.k == x / d);
  }
  std::puts("ok");
  return 0;
}
