// The paged 8-bit key/value cache on the device: what its kernels share.
#pragma once

#include "common.hpp"
#include "kv8_plan.hpp"

namespace llmi_hip::kv8 {

// Item counts of the batch that is set, in device memory (launches replayed
// from a graph read them there).
struct Counts {
  std::int32_t append, tokens, seqs, few, many, join;
};

// A plan's device lists.
struct View {
  const Counts* counts;
  const Seq* seqs;
  const std::int32_t* table;
  const AppendItem* append;
  const FewItem* few;
  const ManyItem* many;
  const JoinItem* join;
};

struct Geometry {
  int heads, kv_heads, group, dim, page_blocks;
  std::size_t block_bytes;  // of one head's block of k (or v): 16 * dim
};

// Block `block` of sequence s for head h: its index in [page][kv head][block].
// Page ids and positions were checked on the host, so the index is in range.
__device__ __forceinline__ std::size_t block_index(const Geometry& g, const std::int32_t* __restrict__ table,
                                                   const Seq& s, int block, int h) {
  const int page = block / g.page_blocks;
  const std::size_t id = static_cast<std::size_t>(table[s.table + page]);
  return (id * g.kv_heads + h) * g.page_blocks + (block - page * g.page_blocks);
}

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
  std::size_t bytes = 0, off_seqs = 0, off_table = 0, off_append = 0, off_few = 0, off_many = 0, off_join = 0;
  std::size_t max_append = 0, max_few = 0, max_many = 0, max_join = 0, max_parts = 0;
  // The attention's partial states (launches of one plan follow each other).
  float* parts = nullptr;
  hipEvent_t copied = nullptr;
  bool set = false;
  llmi_hip::kv8::Lists lists;
  // What captured launches ask of every batch set later: appends were
  // captured, with rotation tables of this many positions.
  mutable bool append_captured = false;
  mutable std::size_t captured_positions = SIZE_MAX;
  llmi_hip::kv8::View view() const {
    using namespace llmi_hip::kv8;
    return {reinterpret_cast<const Counts*>(dev), reinterpret_cast<const Seq*>(dev + off_seqs),
            reinterpret_cast<const std::int32_t*>(dev + off_table),
            reinterpret_cast<const AppendItem*>(dev + off_append), reinterpret_cast<const FewItem*>(dev + off_few),
            reinterpret_cast<const ManyItem*>(dev + off_many), reinterpret_cast<const JoinItem*>(dev + off_join)};
  }
  ~llmi_hip_kv8_plan();
};
