// The host side of the paged 8-bit key/value cache (llmi_hip_kv8_*): checks
// of a cache's shape and of a ragged batch, and the work lists that the
// kernels read.  No HIP here: a CPU test builds these lists and walks them.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/llmi_hip.h"

namespace llmi_hip::kv8 {

constexpr int kBlk = LLMI_KV8_BLOCK;  // positions per scale

// One sequence of a batch as the kernels read it: its tokens are rows
// row .. row + count - 1 of q, k and v, at positions start .. start + count - 1;
// its pages are table[table ..].
struct Seq {
  std::int32_t start, count, row, table, slot;
};

// One block that an append writes or a read returns (one wavefront per
// key/value head for its keys and one for its values): positions pos .. of the
// sequence whose tokens are rows row .. (positions start .. end - 1), block
// `block` of page `page`.  then_pos >= 0: the same wavefront goes on with the
// block at then_pos, whose new rows replace rows of the open-block store that
// the first one reads.  keep: rows from this position on go to that store.
struct BlockItem {
  std::int32_t row, start, end, slot, keep;
  std::int32_t pos, page, block;
  std::int32_t then_pos, then_page, then_block;
};

// The rows of a sequence for one key/value head are its tokens' query heads
// of that head: row r is token r / group, head r % group.  Work of the
// attention: up to few_rows(head_dim) rows (`few`: single tokens and drafts)
// or kManyRows rows (`many`: prompts) over positions lo .. hi - 1, lo a
// multiple of a tile.  part >= 0: one of several pieces of these rows'
// history, whose state goes to partial slots part ..
constexpr int kTile = 64;
constexpr int kFewMax = 64;  // most rows of a sequence and key/value head that go as `few` work
constexpr int kManyRows = 128;
constexpr int kSlotRows = 8;  // rows of a partial slot
// 16 rows keep four tiles of accumulators; past 128 dims they are too many registers.
constexpr int few_rows(int dim) { return dim <= 128 ? 16 : 8; }
struct AttnItem {
  std::int32_t row, start, table;  // the sequence's, as in Seq
  std::int32_t row0, rows, lo, hi, part;
};
// The n pieces of rows row0 .. (at most 16 or kManyRows of them): piece c is
// in slots part + c * step ...
struct JoinItem {
  std::int32_t row, row0, rows, part, n, step;
};
// A history is split so that a batch makes about this many units of work
// (item and key/value head), in pieces of at least the second number of
// positions.  Measured with 256 units of `few` work (32/8 heads of 128; one
// unit a compute unit) against 384: 64 users over 120 to 8191 positions 95 us
// against 105, 32 over 2000 23 against 30, 16 drafts of 3 to 6 tokens 30
// against 32; against 128, 4 drafts of 8 tokens over 2000 15 against 18.
// `many` work: 512, the two workgroups that a compute unit holds (up to 128
// dims); its pieces are of that size with the rest in the last one, so that the
// short ones fill what short histories leave (512 units so against 768 in equal
// pieces: 2048 tokens over 6144 435 us against 449, 1000 over 3000 133 against
// 145, 8 prompts of 512 over 2000, 14/2 heads of 64, 86 against 97).
constexpr std::size_t kFewTarget = 256, kFewLeast = 8 * kTile;
constexpr std::size_t kManyTarget = 512, kManyLeast = 4 * kTile;
// Prompts whose pieces would be shorter than kManyShort that way: one unit for
// each compute unit.
constexpr std::size_t kUnits = 256, kManyShort = 4 * kTile;
// Pieces cost their join, 4 us and more: rows are split only if a piece is
// shorter than their history by more than this.  `few`: for 512 = 4 rows x 128
// dims (one user of 32/8 heads of 128 over 1500 positions 8.6 us whole, 11.1
// in pieces; over 3000 12.3 and 9.7; 16 over 3000 18.2 and 21.7), less for
// wider work by the square, since its tiles take longer and its registers
// leave fewer wavefronts to overlap (16 drafts of 3 to 6 tokens 26 us against
// 31 with the same for all widths, 32 users of 8/1 heads of 256 26 against
// 35), for narrower work at most kFewGainMost (16 users over 1000 to 8000
// positions, 9/3 heads of 64, 16 us against 21 without that, one over 5000 9.4
// against 14).  `many`: nothing where whole histories leave compute units
// without work (one prompt of 1024 tokens of 14/2 heads of 64 20.5 us against
// 25), else kManyGain (4 prompts of 512 tokens behind 300, 32/8 heads of 128,
// 53 us against 73; 2 of 500 behind 1000 56 against 70).
constexpr std::size_t kFewGain = 28 * kTile, kFewGainAt = 4 * 128, kFewGainMost = 40 * kTile;
constexpr std::size_t kManyGain = 12 * kTile;

constexpr std::size_t kJoinFill = 2048;  // rows of all heads that fill the chip with a workgroup each
constexpr int kJoinThreads = 256;

// block / d for block < 2^27 (positions below 2^31) and d = the blocks of a
// page, at most 4096: (block * m) >> k with m = 2^k / d + 1, k = 27 + ceil(log2 d):
// m * d exceeds 2^k by at most d <= 2^(k - 27), so the product's excess over
// block / d stays below 1 / d.
struct Divisor {
  std::uint32_t m;
  std::int32_t k;
};
constexpr Divisor divisor(std::uint32_t d) {
  int log = 0;
  while ((1u << log) < d) ++log;
  return {static_cast<std::uint32_t>((std::uint64_t{1} << (27 + log)) / d + 1), 27 + log};
}

// The blocks whose rows a slot of `open` holds: of each parity the last one
// that an append wrote.  An append that starts inside a block reads the rows
// before its start there.
struct Held {
  std::int32_t block[2] = {-1, -1}, rows[2] = {0, 0};
  bool serves(std::int32_t start) const {
    const std::int32_t b = start / kBlk;
    return start % kBlk == 0 || (block[b & 1] == b && rows[b & 1] >= start % kBlk);
  }
  // After an append of `count` > 0 tokens at a start that was served.
  void wrote(std::int32_t start, std::int32_t count) {
    const std::int32_t end = start + count, first = start / kBlk, last = (end - 1) / kBlk;
    const int p = last & 1;
    block[p] = last;
    rows[p] = end - last * kBlk;
    if (first < last) {
      block[1 - p] = last - 1;
      rows[1 - p] = kBlk;
    } else if (block[1 - p] > last) {  // taken back: those positions are no longer the sequence's
      block[1 - p] = -1;
    }
  }
};

struct Lists {
  std::vector<AttnItem> few, many;
  std::vector<JoinItem> join;
  std::int32_t few_rows = 0;  // most rows of a `few` item
  std::int32_t few_seq_rows = 0;  // most rows of a sequence whose work is `few`
  // A workgroup that joins takes join_at rows of an item at a time: one where
  // rows are few (and pieces many), up to as many as its threads hold where
  // they are enough to fill the chip.
  std::int32_t join_rows = 0;  // most rows of a `join` item
  std::int32_t join_at = 1;
  std::size_t parts = 0;       // partial slots of a key/value head
  std::vector<Seq> seqs;
  std::vector<std::int32_t> table;
  std::vector<BlockItem> blocks;       // every block that holds a new token
  std::vector<std::int32_t> positions; // of every token
  std::size_t tokens = 0, longest = 0;
  bool writable = false;
  std::string why_not;  // why the batch cannot be appended
};

inline std::string check_shape(const llmi_kv8_shape* s) {
  if (s == nullptr) return "null shape";
  if (s->heads == 0 || s->kv_heads == 0 || s->heads % s->kv_heads != 0)
    return "heads must be a positive multiple of kv_heads";
  if (s->heads > 4096) return "at most 4096 heads";
  if (s->head_dim < 32 || s->head_dim > 256 || s->head_dim % 32 != 0)
    return "head_dim must be a multiple of 32 from 32 to 256";
  if (s->page_tokens == 0 || s->page_tokens % kBlk != 0 || s->page_tokens > 65536)
    return "page_tokens must be a multiple of 16 up to 65536";
  if (s->pages == 0 || s->pages > 0x7FFFFFFFu) return "pages must be positive and below 2^31";
  if (s->slots == 0 || s->slots > 0x7FFFFFFFu) return "slots must be positive and below 2^31";
  // Sizes and offsets in bytes stay far from 64 bits.
  constexpr std::uint64_t kMost = std::uint64_t{1} << 48;
  const std::uint64_t position = std::uint64_t{s->kv_heads} * s->head_dim;  // at most 2^20
  if (position * s->page_tokens > kMost / s->pages || position * kBlk * 16 > kMost / s->slots)
    return "the cache would be larger than 2^48 bytes";
  return {};
}

// The most that a batch of at most `seqs` sequences and `tokens` tokens makes.
// A kind's positions x heads over its split size are at most its target, so
// are its full pieces x heads; rows that are split have at most twice their
// full pieces; every group of rows adds one item at most.
struct Limits {
  std::size_t blocks, few, many, parts, join;
};
inline Limits limits(const llmi_kv8_shape& sh, std::size_t seqs, std::size_t tokens) {
  const std::size_t busy = std::min(seqs, tokens), group = sh.heads / sh.kv_heads;
  const std::size_t few = kFewTarget / sh.kv_heads;
  const std::size_t many = tokens * group > kFewMax ? kManyTarget / sh.kv_heads : 0;
  const std::size_t rows = static_cast<std::size_t>(few_rows(static_cast<int>(sh.head_dim)));
  return {tokens / kBlk + 2 * busy, few + kFewMax / rows * busy, many + tokens * group / kManyRows + busy,
          2 * few * (rows / kSlotRows) + 2 * many * (kManyRows / kSlotRows), few + many};
}

// The rows of a `few` item that an attention captured with this batch has room
// for: those of any batch whose sequences have no more rows than this one's.
// (Not few_rows: shared out over several items, more rows can make shorter
// items; 20 rows two of 12 and 8, 16 rows one of 16.)
inline std::int32_t captured_rows(const Lists& l, int dim) {
  return std::min((l.few_seq_rows + 3) / 4 * 4, few_rows(dim));
}

// Checks a batch; returns the reason of a refusal.  Fills in the sequences,
// the tables and whether it can be appended.
inline std::string check_batch(const llmi_kv8_shape& sh, std::size_t seqs, const std::int32_t* slots,
                               const std::int32_t* starts, const std::int32_t* counts, const std::int32_t* tables,
                               std::size_t stride, std::size_t max_seqs, std::size_t max_tokens,
                               std::size_t max_pages, Lists* out) {
  Lists& l = *out;
  l = Lists{};
  if (seqs > max_seqs) return "more sequences than the plan was created for";
  if (seqs > 0 && (starts == nullptr || counts == nullptr || tables == nullptr)) return "null array";
  for (std::size_t i = 0; i < seqs; ++i) {
    const std::string of = " of sequence " + std::to_string(i);
    if (starts[i] < 0) return "negative start" + of;
    if (counts[i] < 0) return "negative count" + of;
    const std::int64_t len = std::int64_t{starts[i]} + counts[i];
    // Positions stay below 2^31 - 512, so that a tile's last position fits 32 bits.
    if (len > 0x7FFFFFFF - 512) return "too many positions" + of;
    const std::size_t need = (static_cast<std::size_t>(len) + sh.page_tokens - 1) / sh.page_tokens;
    if (need > stride) return "the page table is too short for the positions" + of;
    if (l.table.size() + need > max_pages) return "more page entries than the plan was created for";
    l.tokens += static_cast<std::size_t>(counts[i]);
    if (l.tokens > max_tokens) return "more tokens than the plan was created for";
    l.longest = std::max(l.longest, static_cast<std::size_t>(len));
    if (slots != nullptr && (slots[i] < 0 || static_cast<std::uint32_t>(slots[i]) >= sh.slots))
      return "slot out of range" + of;
    l.seqs.push_back({starts[i], counts[i], static_cast<std::int32_t>(l.tokens) - counts[i],
                      static_cast<std::int32_t>(l.table.size()), slots != nullptr ? slots[i] : 0});
    for (std::size_t p = 0; p < need; ++p) {
      const std::int32_t page = tables[i * stride + p];
      if (page < 0 || static_cast<std::uint32_t>(page) >= sh.pages) return "page out of range" + of;
      l.table.push_back(page);
    }
  }
  // An append needs a slot of its own for each sequence with new tokens, and
  // pages under them that nothing else in the batch reads or writes.
  l.writable = slots != nullptr || seqs == 0;
  if (!l.writable) l.why_not = "the batch was set without slots";
  if (l.writable) {
    // A bit per page that appears, and that appears again; one per slot in use.
    std::vector<bool> once(sh.pages), again(sh.pages), held(sh.slots);
    for (const std::int32_t p : l.table) {
      if (once[static_cast<std::size_t>(p)]) again[static_cast<std::size_t>(p)] = true;
      once[static_cast<std::size_t>(p)] = true;
    }
    for (const Seq& q : l.seqs) {
      if (q.count == 0) continue;
      const bool taken = held[static_cast<std::size_t>(q.slot)];
      held[static_cast<std::size_t>(q.slot)] = true;
      if (taken) {
        l.writable = false;
        l.why_not = "two sequences with new tokens have the same slot";
        break;
      }
      const std::int32_t page = static_cast<std::int32_t>(sh.page_tokens);
      for (std::int32_t p = q.start / page; p <= (q.start + q.count - 1) / page && l.writable; ++p)
        if (again[static_cast<std::size_t>(l.table[static_cast<std::size_t>(q.table + p)])]) {
          l.writable = false;
          l.why_not = "a page that takes new tokens appears twice in the batch";
        }
      if (!l.writable) break;
    }
  }
  return {};
}

// Checks a batch and builds its lists.
inline std::string build(const llmi_kv8_shape& sh, std::size_t seqs, const std::int32_t* slots,
                         const std::int32_t* starts, const std::int32_t* counts, const std::int32_t* tables,
                         std::size_t stride, std::size_t max_seqs, std::size_t max_tokens, std::size_t max_pages,
                         Lists* out) {
  Lists& l = *out;
  if (std::string why = check_batch(sh, seqs, slots, starts, counts, tables, stride, max_seqs, max_tokens, max_pages, out);
      !why.empty())
    return why;
  for (std::size_t i = 0; i < seqs; ++i) {
    const Seq& q = l.seqs[i];
    if (q.count == 0) continue;
    const std::int32_t first = q.start / kBlk, last = (q.start + q.count - 1) / kBlk;
    // The rows of the last two blocks go to the open-block store, by parity.
    // If the first block has rows in there that one of these would replace,
    // one wavefront does both, in order.
    std::int32_t then = -1;
    if (q.start % kBlk != 0 && last >= first + 2) then = (last - first) % 2 == 0 ? last : last - 1;
    const std::int32_t per = static_cast<std::int32_t>(sh.page_tokens) / kBlk;
    const auto page = [&](std::int32_t b) { return l.table[static_cast<std::size_t>(q.table + b / per)]; };
    for (std::int32_t b = first; b <= last; ++b) {
      if (b == then) continue;
      BlockItem it{q.row, q.start, q.start + q.count, q.slot, (last - 1) * kBlk, b * kBlk, page(b), b % per, -1, 0, 0};
      if (b == first && then >= 0) {
        it.then_pos = then * kBlk;
        it.then_page = page(then);
        it.then_block = then % per;
      }
      l.blocks.push_back(it);
    }
    for (std::int32_t p = q.start; p < q.start + q.count; ++p) l.positions.push_back(p);
  }
  // Attention: rows are split over their history where the batch alone does
  // not make enough work.
  const std::size_t group = sh.heads / sh.kv_heads;
  const auto rows_of = [&](const Seq& q) { return static_cast<std::size_t>(q.count) * group; };
  // Positions that rows row0 .. row0 + n - 1 see: up to the last row's own.
  const auto seen = [&](const Seq& q, std::size_t row0, std::size_t n) {
    return static_cast<std::size_t>(q.start) + (row0 + n - 1) / group + 1;
  };
  // Over all groups of rows of one kind: fn(sequence, first row, rows, positions seen).
  const auto each = [&](bool few, auto&& fn) {
    const std::size_t most = few ? static_cast<std::size_t>(few_rows(static_cast<int>(sh.head_dim))) : kManyRows;
    for (std::size_t i = 0; i < seqs; ++i) {
      const std::size_t rows = rows_of(l.seqs[i]);
      if (rows == 0 || (rows <= kFewMax) != few) continue;
      // Rows of several groups are shared out evenly, in tiles of 4 rows.
      const std::size_t groups = (rows + most - 1) / most;
      const std::size_t even = few ? (rows + 4 * groups - 1) / (4 * groups) * 4 : most;
      for (std::size_t r = 0; r < rows;) {
        const std::size_t n = std::min(even, rows - r);
        fn(i, r, n, seen(l.seqs[i], r, n));
        r += n;
      }
    }
  };
  const auto split_of = [&](bool few) {
    const std::size_t least = few ? kFewLeast : kManyLeast;
    std::size_t reach = 0;  // positions x heads of all groups of rows
    each(few, [&](std::size_t, std::size_t, std::size_t, std::size_t len) { reach += len * sh.kv_heads; });
    std::size_t target = few ? kFewTarget : kManyTarget;
    if (!few && reach < kManyTarget * kManyShort) target = kUnits;
    // (Rounded up throughout: full pieces x heads are at most the target.)
    const std::size_t each_unit = (reach + target - 1) / target;
    return std::max(least, (each_unit + least - 1) / least * least);
  };
  std::size_t whole = 0;  // units of `many` work without pieces
  each(false, [&](std::size_t, std::size_t, std::size_t, std::size_t) { whole += sh.kv_heads; });
  const auto gain = [&](bool few, std::size_t rows) {
    const std::size_t width = sh.head_dim * ((rows + 3) / 4 * 4);
    if (few) return std::min(kFewGainMost, kFewGain * kFewGainAt * kFewGainAt / (width * width));
    return 4 * whole >= 3 * kUnits ? kManyGain : 0;
  };
  const auto lay = [&](bool few, std::size_t split, std::vector<AttnItem>& items) {
    each(few, [&](std::size_t seq, std::size_t r, std::size_t rows, std::size_t len) {
      // `few`: pieces of one size, in whole units of a tile for each wavefront.
      const std::size_t most = len <= split + gain(few, rows) ? 1 : (len + split - 1) / split;
      const std::size_t even = ((len + most - 1) / most + kFewLeast - 1) / kFewLeast * kFewLeast;
      const std::size_t piece = most == 1 ? len : few ? even : split;
      const std::size_t n = (len + piece - 1) / piece;
      const std::size_t slots = few ? few_rows(static_cast<int>(sh.head_dim)) / kSlotRows : kManyRows / kSlotRows;
      const auto i32 = [](std::size_t x) { return static_cast<std::int32_t>(x); };
      const Seq& q = l.seqs[seq];
      for (std::size_t c = 0; c < n; ++c)
        items.push_back({q.row, q.start, q.table, i32(r), i32(rows), i32(c * piece),
                         i32(std::min(len, (c + 1) * piece)), n > 1 ? i32(l.parts + c * slots) : -1});
      if (n == 1) return;
      l.join.push_back({q.row, i32(r), i32(rows), i32(l.parts), i32(n), i32(slots)});
      l.join_rows = std::max(l.join_rows, i32(rows));
      l.parts += n * slots;
    });
  };
  lay(true, split_of(true), l.few);
  lay(false, split_of(false), l.many);
  // The longest first, so that the last to start are short.
  const auto longer = [](const AttnItem& a, const AttnItem& b) { return a.hi - a.lo > b.hi - b.lo; };
  std::stable_sort(l.few.begin(), l.few.end(), longer);
  std::stable_sort(l.many.begin(), l.many.end(), longer);
  // Two `many` units share a compute unit and its matrix cores (up to 128
  // dims).  If all start at once, the second of each is from the other end: a
  // long one with a short one (2048 tokens over 6144, 32/8 heads of 128, 446 us
  // against 458 without, 4 prompts of 512 behind 300 49 against 51; with more
  // units the order above is better: 4 of 900, 24/3 heads of 96, 48 against 54).
  const std::size_t at_once = kUnits / sh.kv_heads;
  if (sh.head_dim <= 128 && l.many.size() > at_once && l.many.size() * sh.kv_heads <= 2 * kUnits)
    std::reverse(l.many.begin() + static_cast<std::ptrdiff_t>(at_once), l.many.end());
  for (const AttnItem& it : l.few) l.few_rows = std::max(l.few_rows, it.rows);
  for (const Seq& q : l.seqs)
    if (rows_of(q) <= kFewMax) l.few_seq_rows = std::max(l.few_seq_rows, static_cast<std::int32_t>(rows_of(q)));
  if (l.join.size() * sh.kv_heads * static_cast<std::size_t>(l.join_rows) > kJoinFill)
    l.join_at = kJoinThreads * 4 / static_cast<std::int32_t>(sh.head_dim);
  return {};
}

}  // namespace llmi_hip::kv8
