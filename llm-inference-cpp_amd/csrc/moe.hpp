// A layer of experts on the device: what its kernels share.
#pragma once

#include "common.hpp"
#include "moe_plan.hpp"

namespace llmi_hip::moe {

// One expert's matrices of all tiles: codes in the order in which the matrix
// instructions take them.  Lane l of a wavefront holds output l % 16 of a
// tile and, of each block, the 8 inputs 8 (l / 16) ...:
//   Q4_0  codes[((expert * tiles + tile) * chunks + chunk) * 1024 + lane * 16]:
//         four dwords, one of each block of the chunk; its nibbles, from the
//         lowest, are the codes + 8 of inputs 0 2 4 6 1 3 5 7;
//   Q8_0  the same with 2048 bytes a chunk: 1024 for its first two blocks,
//         1024 for the others; a lane's 16 bytes are codes + 128 of 8 inputs of
//         the one block, then of the other.
//   scales[((expert * tiles + tile) * chunks + chunk) * 64 + output * 4 + block].
struct Matrices {
  const std::uint8_t* codes = nullptr;
  const float* scales = nullptr;
};

// A group of rows of one expert: positions first .. first + rows - 1 of the order.
struct RowTile {
  std::int32_t expert, first, rows, pad;
};
struct Groups {
  std::int32_t* counts;  // slots that have an expert, row tiles
  std::int32_t* order;   // slots, those of expert 0 first
  RowTile* tiles;
};
int launch_group(const std::int32_t* ids, std::size_t slots, std::size_t experts, const Groups& g, hipStream_t s);

// Workgroups of a launch, which has to stay below 2^32 threads; the kernels
// go on with further units from there.
constexpr std::size_t kMostGroups = std::size_t{1} << 22;

// Rows x [rows][in] (stride floats apart) in two fp16 parts: x = factor *
// (high + low), with the row's largest |x| between 2^14 and 2^15 times the
// factor, a power of two.  live: the number of rows in device memory (NULL: all).
struct SplitRows {
  _Float16* values;  // [row][chunks * 4 blocks][high, low][32]
  float* factors;
};
int launch_split(const float* x, std::size_t rows, std::size_t in, std::size_t chunks, std::size_t stride,
                 const std::int32_t* live, const SplitRows& to, hipStream_t s);

// y[slot or position] = W_expert x[row] over all row tiles; with `up`,
// silu(gate x) * (up x).  per_row > 0: x's rows are slot / per_row and y's the
// slots; 0: x's rows are positions of the order.
struct Product {
  Shape shape;
  Matrices m, up;
  SplitRows x;
  Groups g;
  std::size_t slots, per_row;
  bool x_by_position, y_by_position;
  float* y;
  std::size_t y_stride;
};
int launch_product(const Product& p, hipStream_t s);

// The same for at most kFewSlots slots, in one launch: y[slot] = W_expert
// x[slot / per_row] (or the gated pair).
struct FewProduct {
  Shape shape;
  Matrices m, up;
  const std::int32_t* ids;
  std::size_t slots, per_row;
  const float* x;
  std::size_t x_stride;
  float* y;
  std::size_t y_stride;
};
int launch_few(const FewProduct& p, hipStream_t s);
// y[t] = residual[t] + sum over j of weights[t][j] W_expert h[t * top_k + j]
// for at most kFewSlots slots of at most kFewTokens tokens, h's rows side by side.
struct FewSum {
  Shape shape;
  Matrices m;
  const std::int32_t* ids;
  const float* weights;
  std::size_t tokens, top_k;
  const float *h, *residual;
  std::size_t r_stride;
  float* y;
  std::size_t y_stride;
};
int launch_few_sum(const FewSum& p, hipStream_t s);

}  // namespace llmi_hip::moe

struct llmi_hip_experts {
  llmi_hip::moe::Shape shape;
  std::uint8_t* codes = nullptr;
  float* scales = nullptr;
  llmi_hip::moe::Matrices view() const { return {codes, scales}; }
  ~llmi_hip_experts() {
    if (codes != nullptr) (void)hipFree(codes);
    if (scales != nullptr) (void)hipFree(scales);
  }
};
