// The paged 8-bit key/value cache on the device: what its kernels share.
#pragma once

#include "common.hpp"
#include "kv8_plan.hpp"

namespace llmi_hip::kv8 {

// Item counts of the batch that is set, in device memory (launches replayed
// from a graph read them there).
struct Counts {
  std::int32_t blocks, tokens, few, many, join, join_rows, join_at;
};

// A plan's device lists.
struct View {
  const Counts* counts;
  const std::int32_t* positions;
  const std::int32_t* table;
  const BlockItem* blocks;
  const AttnItem* few;
  const AttnItem* many;
  const JoinItem* join;
};

struct Geometry {
  int heads, kv_heads, group, dim, page_blocks;
  Divisor by_page;  // divides a block by page_blocks
};

// Which page of its sequence's table holds a block.
__device__ __forceinline__ int page_of(const Geometry& g, int block) {
  return static_cast<int>((static_cast<std::uint64_t>(static_cast<std::uint32_t>(block)) * g.by_page.m) >> g.by_page.k);
}
// A block of head h in [page][kv head][block], given the page's id and its
// place in the table.  Ids and positions were checked on the host, so the
// index is in range.
__device__ __forceinline__ std::size_t block_at(const Geometry& g, int id, int page, int block, int h) {
  return (static_cast<std::size_t>(id) * g.kv_heads + h) * g.page_blocks + (block - page * g.page_blocks);
}
// Workgroups (of at most 512 threads) of a launch, which has to stay below
// 2^32 threads; every kernel here goes on with further units from there.
constexpr std::size_t kMostGroups = std::size_t{1} << 22;

int launch_attention(const llmi_hip_kv8_plan* p, const llmi_kv8_layer& layer, const float* q, std::size_t q_stride,
                     float scale, float* out, std::size_t out_stride, hipStream_t s, bool captured);

}  // namespace llmi_hip::kv8

struct llmi_hip_kv8_plan {
  llmi_kv8_shape shape{};
  std::size_t max_seqs = 0, max_tokens = 0, max_pages = 0;
  llmi_hip::kv8::Geometry g{};
  // One device allocation, filled by one copy from pinned memory; `copied`
  // marks the copy's end, before which the pinned side is not written again.
  std::uint8_t* dev = nullptr;
  std::uint8_t* pinned = nullptr;
  std::size_t bytes = 0, off_positions = 0, off_table = 0, off_blocks = 0, off_few = 0, off_many = 0, off_join = 0;
  llmi_hip::kv8::Limits most{};
  float* parts = nullptr;  // the attention's partial states (launches of one plan follow each other)
  hipEvent_t copied = nullptr;
  bool set = false;
  llmi_hip::kv8::Lists lists;
  // What captured launches ask of every batch set later: appends were
  // captured, with rotation tables of this many positions; attention was, for
  // `few` items of this many rows, with or without `many` items.
  mutable bool append_captured = false;
  mutable std::size_t captured_positions = SIZE_MAX;
  mutable std::int32_t captured_few = 0x7FFFFFFF;
  mutable bool captured_many = true;
  llmi_hip::kv8::View view() const {
    using namespace llmi_hip::kv8;
    return {reinterpret_cast<const Counts*>(dev), reinterpret_cast<const std::int32_t*>(dev + off_positions),
            reinterpret_cast<const std::int32_t*>(dev + off_table),
            reinterpret_cast<const BlockItem*>(dev + off_blocks), reinterpret_cast<const AttnItem*>(dev + off_few),
            reinterpret_cast<const AttnItem*>(dev + off_many), reinterpret_cast<const JoinItem*>(dev + off_join)};
  }
  ~llmi_hip_kv8_plan();
};
