// A layer of experts on the device: what its kernels share.
#pragma once

#include "common.hpp"
#include "moe_plan.hpp"

namespace llmi_hip::moe {

// The experts' codes in the order in which the matrix instructions take them.
// Lane l of a wavefront holds output l % 16 of a tile and, of each block, the
// 8 inputs 8 (l / 16) ...  Step ((expert * tiles + tile) * steps + step) takes
// step_bytes(type), so that a tile's steps are one stream:
//   Q4_0  at lane * 8: two dwords, one of each block; its nibbles, from the
//         lowest, are the codes + 8 of inputs 0 2 4 6 1 3 5 7;
//   Q8_0  at lane * 16: codes + 128 of the 8 inputs of the one block, then of
//         the other;
//   behind the codes 32 floats: the scale of output o and block b at 2 o + b.
struct Matrices {
  const std::uint8_t* steps = nullptr;
};

// An entry of a list of groups of rows, the same for all groups of an expert: its
// positions are begin .. begin + slots - 1 of the order, its groups the list's
// group0 .. group0 + groups - 1, each but the last one full.  next0: where the
// second list's groups are as large or smaller, the expert's first one there.
struct RowTile {
  std::int32_t expert, begin, slots, group0, groups, next0, unused[2];
};
static_assert(sizeof(RowTile) == kRowTileBytes);
struct Groups {
  std::int32_t* counts;  // slots that have an expert, row tiles of both lists
  std::int32_t* order;   // slots, those of expert 0 first
  RowTile* tiles[2];     // of rows[0] and rows[1] rows each
  int rows[2];           // powers of two
  std::int32_t* hist;    // [grouping_blocks][expert], of more than kOneGroup slots
};

// Workgroups of a launch, which has to stay below 2^32 threads; the kernels
// go on with further units from there.
constexpr std::size_t kMostGroups = std::size_t{1} << 22;

// Rows in two fp16 parts: x = factor * (high + low), with the row's largest
// |x| between 2^14 and 2^15 times the factor, a power of two.
//   rows as they are: values [row][step][block][high, low][32], factors [row];
//   in row tiles of MT * 16 rows: values [tile][step][16 rows of MT][block]
//     [high, low][lane][8], lane l holding inputs 8 (l / 16) .. of row l % 16,
//     factors [tile][row].
struct SplitRows {
  _Float16* values;
  float* factors;
};
// Where rows come from: slot s has x's row s / per_row, at least 1 (launch_split,
// which takes the rows one after the other, does not look at it).
struct RowSource {
  const float* x;
  std::size_t stride, in, steps;
  std::uint32_t per_row;
};
// Groups the slots, and brings x into the layout that list 0's product takes.
int launch_prepare(const std::int32_t* ids, std::size_t slots, std::size_t experts, const Groups& g, const RowSource& x,
                   const SplitRows& to, hipStream_t s);
// The *live rows of x (at most `rows`) as they are.
int launch_split(const RowSource& x, std::size_t rows, const std::int32_t* live, const SplitRows& to, hipStream_t s);

// y[slot or position] = W_expert x over all row tiles of a list; with `up`,
// silu(gate x) * (up x).  x: in row tiles where the list's have at most
// kMostShortRows rows; else rows as they are, x's row of a position being the
// position (per_row 0) or order[position] / per_row.
struct Product {
  Shape shape;
  Matrices m, up;
  SplitRows x;
  Groups g;
  int list;  // which of its tile lists
  std::size_t slots, per_row;
  bool y_by_position;
  float* y;
  std::size_t y_stride;
  // A gated pair's results in the row tiles of the second list (y NULL), each
  // block of a row with a factor of its own: factors [tile][step][block][row].
  SplitRows h;
  std::size_t h_steps;
  bool block_factors;  // x comes so
};
int launch_product(const Product& p, hipStream_t s);

// Results of a gated pair for the second product of few tokens, in two fp16
// parts, each 32 of a row with a factor of their own: values [slot][block]
// [high, low][32], factors [slot][block], a multiple of 4 blocks.
struct FewParts {
  _Float16* values;
  float* factors;
  int blocks;
};
// A product for at most kFewSlots slots, in one launch: y[slot] = W_expert
// x[slot / per_row], or the gated pair into h.
struct FewProduct {
  Shape shape;
  Matrices m, up;
  const std::int32_t* ids;
  std::size_t slots, per_row;
  const float* x;
  std::size_t x_stride;
  float* y;
  std::size_t y_stride;
  FewParts h;
};
int launch_few(const FewProduct& p, hipStream_t s);
// y[t] = residual[t] + sum over j of weights[t][j] W_expert h[t * top_k + j]
// for at most kFewSlots slots of at most kFewTokens tokens.
struct FewSum {
  Shape shape;
  Matrices m;
  const std::int32_t* ids;
  const float* weights;
  std::size_t tokens, top_k;
  FewParts h;
  const float* residual;
  std::size_t r_stride;
  float* y;
  std::size_t y_stride;
  float* parts;  // few_splits(shape) * tokens * out floats where there are several
};
int launch_few_sum(const FewSum& p, hipStream_t s);

}  // namespace llmi_hip::moe

struct llmi_hip_experts {
  llmi_hip::moe::Shape shape;
  std::uint8_t* steps = nullptr;
  llmi_hip::moe::Matrices view() const { return {steps}; }
  ~llmi_hip_experts() {
    if (steps != nullptr) (void)hipFree(steps);
  }
};
