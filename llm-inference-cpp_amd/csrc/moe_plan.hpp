// A layer of experts (llmi_hip_moe_*): sizes, limits and checks on the host.
// No HIP here, so that tests on the CPU reach all of it.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <string>

#include "../../include/llmi_hip.h"

namespace llmi_hip::moe {

constexpr std::size_t kMaxExperts = 4096;               // the grouping keeps a counter of each in LDS
constexpr std::size_t kMaxRouted = 1024;                // logits of a token that one wavefront ranks
constexpr std::size_t kMaxTopK = 64;
constexpr std::size_t kMaxSlots = std::size_t{1} << 24;  // rows of all experts together
constexpr std::size_t kMaxInner = std::size_t{1} << 18;  // inputs, and results, of an expert's matrix

constexpr int kTile = 16;                         // outputs and rows of a matrix instruction
constexpr int kStep = 2 * LLMI_BLOCK_SIZE;        // inputs of a step: two blocks
constexpr std::size_t kStepScales = 2 * kTile;    // a tile's scales of a step
// Bytes of a tile's codes of a step, behind which its scales lie.
constexpr std::size_t code_bytes(int type) { return type == LLMI_TYPE_Q4_0 ? 512 : 1024; }
constexpr std::size_t step_bytes(int type) { return code_bytes(type) + kStepScales * sizeof(float); }

// The shape of a set of experts as the device holds it: per expert, tiles of
// 16 outputs; per tile, steps of 64 inputs (outputs and inputs behind the last
// ones have codes and scales of 0).
struct Shape {
  int type = 0;
  std::size_t count = 0, out = 0, in = 0;
  std::size_t blocks() const { return (in + LLMI_BLOCK_SIZE - 1) / LLMI_BLOCK_SIZE; }
  std::size_t steps() const { return (in + kStep - 1) / kStep; }
  std::size_t tiles() const { return (out + kTile - 1) / kTile; }
  std::size_t bytes() const { return count * tiles() * steps() * step_bytes(type); }
};

inline std::string check_shape(const Shape& s) {
  if (s.type != LLMI_TYPE_Q8_0 && s.type != LLMI_TYPE_Q4_0) return "type must be LLMI_TYPE_Q8_0 or LLMI_TYPE_Q4_0";
  if (s.count == 0 || s.count > kMaxExperts) return "1 .. 4096 experts";
  if (s.in == 0 || s.out == 0 || s.in > kMaxInner || s.out > kMaxInner) return "in and out must be 1 .. 2^18";
  return {};
}

// Rows of x that slots come from, per_row of each (any number of them).
inline std::size_t rows_of(std::size_t slots, std::size_t per_row) { return slots == 0 ? 0 : (slots - 1) / per_row + 1; }

// Groups of so many rows of at most: every expert may leave one unfilled.
inline std::size_t most_tiles(std::size_t slots, std::size_t experts, std::size_t rows) {
  return slots / rows + std::min(slots, experts);
}
// Tiles of outputs of a workgroup: of the kernel for short work, of the one for long.
inline std::size_t short_columns(bool gated) { return gated ? 2 : 4; }
inline std::size_t long_columns(bool gated) { return 4 * short_columns(gated); }
// The largest number of slots that goes to the kernel for short work: up to 28
// an expert, or what leaves the one for long work fewer than about 160
// workgroups (tiles of 64 rows, half of one left unfilled by each expert).
// Short and long took, of experts of 2048 x 1024: Q4_0, 57 and 66 us for 24
// slots of each of 64; Q8_0, 80 and 70 for 32; Q4_0, 24 and 45 for 96 of each of 8, 48
// and 47 for 256, 56 and 49 for 350; MLPs of 8: 45 and 75 for 64 of each, 95
// and 87 for 192; Q8_0 896 x 4864: 24 and 27 for 32 of each of 8, 34 and 29 for 64.
inline std::size_t most_short(const Shape& s, bool gated) {
  const std::size_t columns = (s.tiles() + long_columns(gated) - 1) / long_columns(gated);
  const std::size_t room = 160 / columns, left = s.count / 2;
  return std::max(28 * s.count, room > left ? 64 * (room - left) : 0);
}
// Rows of an expert that a workgroup of a grouped product takes: 16, 32 or, of
// long work, 64; 16 up to 48 slots an expert, or where 32 would leave fewer than
// about 400 workgroups.  16 and 32 took, of 8 Q4_0 experts of 2048 x 1024: 15.1
// and 17.2 us for 24 slots of each, 18.0 and 19.2 for 48, 27.1 and 24.1 for 96 (448
// workgroups); of 8 Q8_0 experts of 4864 x 896: 44 and 51 for 64 (280
// workgroups), 70 and 67 for 128 (504).
inline std::size_t pick_rows(const Shape& s, std::size_t slots, bool gated) {
  if (slots > most_short(s, gated)) return 64;
  const std::size_t columns = (s.tiles() + short_columns(gated) - 1) / short_columns(gated);
  return slots <= 48 * s.count || (slots / 32 + s.count / 2) * columns < 400 ? 16 : 32;
}
// Of the two products of an MLP.  The first one writes the row tiles of a short
// second one, whose groups are as large as its own or parts of them.
struct MlpRows {
  std::size_t first, second;
};
inline MlpRows pick_mlp_rows(const Shape& gate, const Shape& down, std::size_t slots) {
  const std::size_t a = pick_rows(gate, slots, true), b = pick_rows(down, slots, false);
  return {a, b <= 32 ? std::min(a, b) : b};
}
constexpr std::size_t kRowTileBytes = 32;  // a group of rows in a list
constexpr std::size_t kLeastRows = 16, kMostShortRows = 32;

// Up to this many slots (a wavefront's lanes) go without a grouping, a
// workgroup for each slot and 32 outputs, of which only those of an expert's
// first slot work.  Products of one or two rows of x, or of up to 16 where the
// workgroups are few (4, 12, 16 and 32 rows of 2 of 8 Q4_0 experts of 2048 x
// 1024: 7.2, 8.2, 9.9 and 14.6 us, grouped 12.3, 13.1, 13.0 and 13.5; 4, 8 and
// 16 rows of 4 of 16 Q8_0 experts of 4096 x 4096: 49, 69 and 90, grouped 51, 64
// and 68).  MLPs of up to 2 tokens (8 of 64 Q4_0 experts 2048 /
// 1024: 28.7 us, grouped 30.9; 4 tokens 59 and 47).
constexpr std::size_t kFewSlots = 64, kFewRows = 16, kFewGroups = 2048, kFewTokens = 2;
inline bool few_matmul(const Shape& s, std::size_t slots, std::size_t per_row) {
  const std::size_t rows = rows_of(slots, per_row);
  return slots <= kFewSlots && (rows <= 2 || (rows <= kFewRows && slots * ((s.tiles() + 1) / 2) <= kFewGroups));
}
inline bool few_mlp(std::size_t tokens, std::size_t top_k) { return tokens * top_k <= kFewSlots && tokens <= kFewTokens; }

// Workgroups that share the inputs of a tile in the second product of few
// tokens, whose sums a launch of its own joins: where the tiles alone would
// leave most of the chip idle.
inline std::size_t few_splits(const Shape& s) { return s.tiles() >= 96 ? 1 : (128 + s.tiles() - 1) / s.tiles(); }
// Blocks of a row between the products of few tokens: whole chunks of four.
inline std::size_t few_blocks(const Shape& s) { return (s.blocks() + 3) / 4 * 4; }

// Places in a call's workspace, each a multiple of 256 bytes.
struct Layout {
  std::size_t bytes = 0;
  std::size_t take(std::size_t n) {
    const std::size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};
// How slots are grouped: up to kOneGroup of them by one workgroup, more by
// grouping_blocks() of them, which count first and then place.  With up to
// kSelfGroup slots of up to kSelfExperts experts, every wavefront that brings
// a row into its row tile finds the place by itself, which spares a launch.
constexpr std::size_t kOneGroup = 4096, kSelfGroup = 2048, kSelfExperts = 256;
inline std::size_t grouping_blocks(std::size_t slots) { return slots <= kOneGroup ? 1 : std::min<std::size_t>((slots + 2047) / 2048, 64); }
inline bool self_grouped(std::size_t slots, std::size_t experts) { return slots <= kSelfGroup && experts <= kSelfExperts; }

// The slots in the order of their experts, and their groups of rows, for the
// two products of an MLP.
struct Grouping {
  std::size_t counts, order, tiles[2], hist;
  void place(Layout* l, std::size_t slots, std::size_t experts) {
    counts = l->take(3 * sizeof(std::int32_t));
    hist = l->take(slots > kOneGroup ? 64 * experts * sizeof(std::int32_t) : 0);
    order = l->take(slots * sizeof(std::int32_t));
    for (std::size_t& t : tiles) t = l->take(most_tiles(slots, experts, kLeastRows) * kRowTileBytes);
  }
};
// Rows in two fp16 parts (4 bytes an element, whole steps) and their factors:
// `rows` rows as they are for the kernel for long work, or row tiles for the
// one for short, whichever is more over all calls of at most so many slots,
// so that a workspace for a number of slots holds every smaller one.
// An MLP's second product for short work has a factor for each block of a row.
struct Parts {
  std::size_t values, factors;
  void place(Layout* l, std::size_t rows, const Shape& s, std::size_t slots, bool gated, bool block_factors = false) {
    const std::size_t small = std::min(slots, most_short(s, gated));
    const std::size_t tiled = std::max(most_tiles(small, s.count, kLeastRows) * kLeastRows,
                                       most_tiles(small, s.count, kMostShortRows) * kMostShortRows);
    const std::size_t n = std::max(rows, tiled);
    values = l->take(n * s.steps() * kStep * 4);
    factors = l->take((block_factors ? std::max(rows, tiled * s.steps() * 2) : n) * sizeof(float));
  }
};
struct MatmulLayout {
  Layout all;
  Grouping group;
  Parts x;
  MatmulLayout(const Shape& s, std::size_t slots, std::size_t per_row) {
    group.place(&all, slots, s.count);
    x.place(&all, rows_of(slots, per_row), s, slots, false);
  }
};
struct MlpLayout {
  Layout all;
  Grouping group;
  Parts x, h_parts;
  std::size_t h, few_factors, sums;  // sums of each slot, or of each split
  MlpLayout(const Shape& gate, const Shape& down, std::size_t tokens, std::size_t top_k) {
    const std::size_t slots = tokens * top_k;
    group.place(&all, slots, gate.count);
    x.place(&all, tokens, gate, slots, true);
    // For long work fp32 rows; of few slots their parts and factors (whole
    // blocks); for short work row tiles (h_parts) alone.
    const std::size_t few = std::min(slots, kFewSlots) * few_blocks(down), many = slots > most_short(down, false) ? slots : 0;
    few_factors = few * 2 * LLMI_BLOCK_SIZE * 2;
    h = all.take(std::max(many * gate.out * sizeof(float), few_factors + few * sizeof(float)));
    h_parts.place(&all, many, down, slots, false, true);
    const std::size_t split = std::min(tokens, kFewTokens) * few_splits(down);
    sums = all.take(std::max(slots, split) * down.out * sizeof(float));
  }
};

// Memory that a call reads or writes: `rows` pieces of `bytes` bytes, `stride`
// bytes apart (at least as long).
struct Region {
  const void* at;
  std::size_t rows, bytes, stride;
  static Region whole(const void* p, std::size_t n) { return {p, 1, n, n}; }
  static Region matrix(const float* p, std::size_t rows, std::size_t width, std::size_t stride) {
    return {p, rows, width * sizeof(float), std::min(stride, SIZE_MAX / sizeof(float)) * sizeof(float)};
  }
};
// Whether two regions have a byte in common.  Spans that are apart settle
// nearly every call; columns of one array, rows between each other's, do not meet.
inline bool overlap(const Region& a, const Region& b) {
  typedef __int128 Wide;  // differences and products of any addresses and strides
  if (a.rows == 0 || b.rows == 0 || a.bytes == 0 || b.bytes == 0) return false;
  if (a.rows > b.rows && a.stride != b.stride) return overlap(b, a);
  const Wide from = static_cast<Wide>(reinterpret_cast<std::uintptr_t>(b.at)) - reinterpret_cast<std::uintptr_t>(a.at);
  const Wide a_end = static_cast<Wide>(a.rows - 1) * a.stride + a.bytes, b_end = from + static_cast<Wide>(b.rows - 1) * b.stride + b.bytes;
  if (from >= a_end || b_end <= 0) return false;
  // Row i of a (at i a.stride) meets row j of b (at from + j b.stride) where
  // j b.stride lies between at - from - b.bytes and at - from + a.bytes, both excluded.
  const auto row_meets = [&](Wide at, Wide first) {
    const Wide below = at - from - static_cast<Wide>(b.bytes), stride = b.stride;
    Wide j = below / stride;
    if (j * stride > below) --j;  // the quotient rounded down
    j = std::max(j + 1, first);
    return j < static_cast<Wide>(b.rows) && j * stride < at - from + static_cast<Wide>(a.bytes);
  };
  // Of equal strides only j - i counts.
  if (a.stride == b.stride) return row_meets(0, -static_cast<Wide>(a.rows - 1));
  for (std::size_t i = 0; i < a.rows; ++i)
    if (row_meets(static_cast<Wide>(i) * a.stride, 0)) return true;
  return false;
}

inline std::string check_matmul(std::size_t slots, std::size_t per_row) {
  if (per_row == 0) return "slots of a row must be at least 1";
  if (slots > kMaxSlots) return "more than 2^24 slots";
  return {};
}
inline std::string check_mlp(const Shape& gate, const Shape& down, std::size_t tokens, std::size_t top_k) {
  if (down.in != gate.out || down.count != gate.count) return "down's inputs and experts must be gate's results and experts";
  if (top_k == 0 || top_k > kMaxTopK) return "top_k must be 1 .. 64";
  if (tokens > kMaxSlots / top_k) return "more than 2^24 slots (tokens x top_k)";
  return {};
}
inline std::string check_route(std::size_t tokens, std::size_t experts, std::size_t top_k, std::size_t stride) {
  if (experts == 0 || experts > kMaxRouted) return "1 .. 1024 experts";
  if (top_k == 0 || top_k > kMaxTopK || top_k > experts) return "top_k must be 1 .. 64 and at most the number of experts";
  if (stride < experts) return "stride shorter than a token's logits";
  if (tokens > kMaxSlots) return "more than 2^24 tokens";
  return {};
}

}  // namespace llmi_hip::moe
