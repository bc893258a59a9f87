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

constexpr int kTile = 16;        // outputs and rows of a matrix instruction
constexpr int kChunkBlocks = 4;  // blocks of 32 weights that one 16-byte load of a lane covers (Q4_0)

// The shape of a set of experts as the device holds it: per expert, tiles of
// 16 outputs; per tile, chunks of 4 blocks (128 inputs; the last one filled
// up with codes and scales of 0).
struct Shape {
  int type = 0;
  std::size_t count = 0, out = 0, in = 0;
  std::size_t blocks() const { return (in + LLMI_BLOCK_SIZE - 1) / LLMI_BLOCK_SIZE; }
  std::size_t chunks() const { return (blocks() + kChunkBlocks - 1) / kChunkBlocks; }
  std::size_t tiles() const { return (out + kTile - 1) / kTile; }
  std::size_t chunk_bytes() const { return type == LLMI_TYPE_Q4_0 ? 1024 : 2048; }
  std::size_t code_bytes() const { return count * tiles() * chunks() * chunk_bytes(); }
  std::size_t scale_floats() const { return count * tiles() * chunks() * kTile * kChunkBlocks; }
};

inline std::string check_shape(const Shape& s) {
  if (s.type != LLMI_TYPE_Q8_0 && s.type != LLMI_TYPE_Q4_0) return "type must be LLMI_TYPE_Q8_0 or LLMI_TYPE_Q4_0";
  if (s.count == 0 || s.count > kMaxExperts) return "1 .. 4096 experts";
  if (s.in == 0 || s.out == 0 || s.in > kMaxInner || s.out > kMaxInner) return "in and out must be 1 .. 2^18";
  return {};
}

// Rows of an expert that a workgroup of the grouped products takes.
constexpr std::size_t kRows = 64;
// Groups of kRows rows of at most: every expert may leave one unfilled.
inline std::size_t most_tiles(std::size_t slots, std::size_t experts) {
  return slots / kRows + std::min(slots, experts);
}

// Up to this many slots (a wavefront's lanes) and tokens (rows of a matrix
// instruction) go without a grouping.
constexpr std::size_t kFewSlots = 64, kFewTokens = 16;
inline bool few_matmul(std::size_t slots) { return slots <= kFewSlots; }
inline bool few_mlp(std::size_t tokens, std::size_t top_k) { return tokens * top_k <= kFewSlots && tokens <= kFewTokens; }

// Places in a call's workspace, each a multiple of 256 bytes.
struct Layout {
  std::size_t bytes = 0;
  std::size_t take(std::size_t n) {
    const std::size_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  }
};
// The slots in the order of their experts, and their groups of rows.
struct Grouping {
  std::size_t counts, order, tiles;
  void place(Layout* l, std::size_t slots, std::size_t experts) {
    counts = l->take(2 * sizeof(std::int32_t));
    order = l->take(slots * sizeof(std::int32_t));
    tiles = l->take(most_tiles(slots, experts) * 4 * sizeof(std::int32_t));
  }
};
// Rows in two fp16 parts (4 bytes an element, whole chunks) and their factors.
struct Parts {
  std::size_t values, factors;
  void place(Layout* l, std::size_t rows, const Shape& s) {
    values = l->take(rows * s.chunks() * kChunkBlocks * LLMI_BLOCK_SIZE * 4);
    factors = l->take(rows * sizeof(float));
  }
};
struct MatmulLayout {
  Layout all;
  Grouping group;
  Parts x;
  MatmulLayout(const Shape& s, std::size_t slots, std::size_t per_row) {
    group.place(&all, slots, s.count);
    x.place(&all, (slots + per_row - 1) / per_row, s);
  }
};
struct MlpLayout {
  Layout all;
  Grouping group;
  Parts x, h_parts;
  std::size_t h, sums;
  MlpLayout(const Shape& gate, const Shape& down, std::size_t tokens, std::size_t top_k) {
    const std::size_t slots = tokens * top_k;
    group.place(&all, slots, gate.count);
    x.place(&all, tokens, gate);
    h = all.take(slots * gate.out * sizeof(float));
    h_parts.place(&all, slots, down);
    sums = all.take(slots * down.out * sizeof(float));
  }
};

inline std::string check_matmul(const Shape& s, std::size_t slots, std::size_t per_row) {
  if (per_row == 0) return "slots of a row must be at least 1";
  if (slots > kMaxSlots) return "more than 2^24 slots";
  (void)s;
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
