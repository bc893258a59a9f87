// What the experts' products of many slots need beforehand: the slots grouped
// by expert, and their rows in two fp16 parts.  Both are short work that no
// matrix waits for, so what counts is the number of launches and of waits in a
// row: one launch up to 4096 slots, where rows go as they are or every
// wavefront finds its place by itself (512 slots of 64 experts with rows of
// 2048: 7.5 us; 1024 slots, 512 rows of 896: 5.4 us), two for more (32768 slots,
// 4096 rows of 2048: 16.1 and 10.3 us, the counts' way through memory in both).
#include "moe_device.hpp"

namespace llmi_hip::moe {
namespace {

// -------------------------------------------------------------------- rows

constexpr int kThreads = 256, kWaves = kThreads / 64;

// A row of x for a wavefront: up to 2048 inputs at a time, all asked for before
// the first is used; a row that is no longer stays in registers.
struct Row {
  static constexpr int kBatch = 4, kInputs = kBatch * 512;
  const float* row;
  int in, lane;
  float v[kBatch][8];
  __device__ __forceinline__ Row(const RowSource& src, std::size_t from, int l)
      : row(src.x + from * src.stride), in(static_cast<int>(src.in)), lane(l) {
    load(0);
  }
  __device__ __forceinline__ void load(int base) {
#pragma unroll
    for (int c = 0; c < kBatch; ++c) {
      const int k = base + c * 512 + lane * 8;
      if (k + 8 <= in) {
        const f4 a = *reinterpret_cast<const f4*>(row + k), b = *reinterpret_cast<const f4*>(row + k + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[c][i] = a[i];
          v[c][4 + i] = b[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = k + i < in ? row[k + i] : 0.0f;
      }
    }
  }
};

// The row in two parts.  The factor is taken from the largest finite |x|: an
// inf or NaN stays one in the high part and shows in its own row alone.
// MT > 0: row r of the row tiles of 16 MT rows; 0: row r as it is.
template <int MT>
__device__ __forceinline__ void store_row(Row& x, const RowSource& src, int r, const SplitRows& to) {
  constexpr int kRows = MT * kTile;
  const int padded = static_cast<int>(src.steps) * kStep;
  std::uint32_t top = 0;
  for (int base = 0; base < x.in; base += Row::kInputs) {
    if (base > 0) x.load(base);
#pragma unroll
    for (int c = 0; c < Row::kBatch; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, finite_bits(x.v[c][i]));
  }
  const Factor f(across(top, Larger{}));
  if (x.lane == 0) to.factors[r] = f.back;
  for (int base = 0; base < padded; base += Row::kInputs) {
    if (x.in > Row::kInputs) x.load(base);
#pragma unroll
    for (int c = 0; c < Row::kBatch; ++c) {
      const int k = base + c * 512 + x.lane * 8;
      if (k >= padded) continue;
      f16x8 high, low;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        _Float16 a, b;
        two_parts(x.v[c][i] * f.up, a, b);
        high[i] = a;
        low[i] = b;
      }
      if constexpr (MT > 0) {
        const std::size_t piece = ((static_cast<std::size_t>(r / kRows) * src.steps + k / kStep) * MT + r % kRows / kTile) * 4 + k % kStep / kBlock * 2;
        f16x8* at = reinterpret_cast<f16x8*>(to.values) + piece * 64 + k % kBlock / 8 * kTile + r % kTile;
        at[0] = high;
        at[64] = low;
      } else {
        _Float16* at = to.values + (static_cast<std::size_t>(r) * padded + k / kBlock * kBlock) * 2 + k % kBlock;
        *reinterpret_cast<f16x8*>(at) = high;
        *reinterpret_cast<f16x8*>(at + kBlock) = low;
      }
    }
  }
}
template <int MT>
__device__ __forceinline__ void split_row(const RowSource& src, std::size_t from, int r, const SplitRows& to, int lane) {
  Row x(src, from, lane);
  store_row<MT>(x, src, r, to);
}
__device__ __forceinline__ std::size_t row_of(const RowSource& src, int slot) { return static_cast<std::uint32_t>(slot) / src.per_row; }

// Rows as they are.  Bound by memory: 32768 rows of 1024 in 47.6 us, 5.6 TB/s.
__global__ void __launch_bounds__(kThreads) split_kernel(RowSource src, int rows, const std::int32_t* __restrict__ live,
                                                         SplitRows to) {
  const int most = min(*live, rows);
  for (int r = blockIdx.x * kWaves + (threadIdx.x >> 6); r < most; r += gridDim.x * kWaves)
    split_row<0>(src, static_cast<std::size_t>(r), r, to, threadIdx.x & 63);
}

// The rows of list 0, into row tiles.
template <int MT>
__global__ void __launch_bounds__(kThreads) split_tiles_kernel(RowSource src, Groups g, SplitRows to) {
  constexpr int kRows = MT * kTile;
  const int most = g.counts[1] * kRows;
  for (int r = blockIdx.x * kWaves + (threadIdx.x >> 6); r < most; r += gridDim.x * kWaves) {
    const RowTile t = g.tiles[0][r / kRows];
    const int at = r - t.group0 * kRows;  // of the expert's rows
    if (at >= t.slots) continue;          // nothing reads its results
    const int pos = t.begin + at;
    split_row<MT>(src, row_of(src, g.order[pos]), r, to, threadIdx.x & 63);
  }
}

// ---------------------------------------------------------------- grouping

constexpr int kGroupThreads = 1024;

// Running sums over the experts: count[e] becomes the place of e's first slot;
// tile(list, index, RowTile) gets every group of rows, by the thread of its
// expert; the totals (slots, groups of both lists) come back in all threads.
template <typename Fn>
__device__ __forceinline__ void lay_ranges(std::int32_t* count, int experts, const Groups& g, std::int32_t (&total)[3], Fn&& tile) {
  __shared__ std::int32_t waves[3][kGroupThreads / 64];
  const int t = threadIdx.x, lane = t & 63, shift0 = __builtin_ctz(g.rows[0]), shift1 = __builtin_ctz(g.rows[1]);
  total[0] = total[1] = total[2] = 0;
  for (int e0 = 0; e0 < experts; e0 += kGroupThreads) {
    const int e = e0 + t;
    const std::int32_t n = e < experts ? count[e] : 0;
    const std::int32_t own[3] = {n, (n + g.rows[0] - 1) >> shift0, (n + g.rows[1] - 1) >> shift1};
    std::int32_t at[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      std::int32_t a = own[i];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const std::int32_t x = __shfl_up(a, o, 64);
        if (lane >= o) a += x;
      }
      if (lane == 63) waves[i][t >> 6] = a;
      at[i] = total[i] + a - own[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int w = 0; w < kGroupThreads / 64; ++w) {
        const std::int32_t x = waves[i][w];
        if (w < t >> 6) at[i] += x;
        total[i] += x;
      }
    if (e < experts) {
      count[e] = at[0];
#pragma unroll
      for (int l = 0; l < 2; ++l)
        for (std::int32_t i = 0; i < own[1 + l]; ++i)
          tile(l, at[1 + l] + i, RowTile{e, at[0], n, at[1 + l], own[1 + l], at[2], {}});
    }
    __syncthreads();
  }
}

// All slots, by one workgroup.  Which place of its expert's range a slot gets
// depends on the order of the counters' increments; no result does, since a
// row's sums are the same at every place of a tile.
__device__ void group_slots(const std::int32_t* __restrict__ ids, int slots, int experts, const Groups& g, std::int32_t* count) {
  const int t = threadIdx.x;
  for (int e = t; e < experts; e += kGroupThreads) count[e] = 0;
  __syncthreads();
  for (int i = t; i < slots; i += kGroupThreads) {
    const std::int32_t e = ids[i];
    if (e >= 0 && e < experts) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  std::int32_t total[3];
  lay_ranges(count, experts, g, total, [&](int l, std::int32_t at, const RowTile& r) { g.tiles[l][at] = r; });
  for (int i = t; i < slots; i += kGroupThreads) {
    const std::int32_t e = ids[i];
    if (e >= 0 && e < experts) g.order[atomicAdd(&count[e], 1)] = i;
  }
  if (t < 3) g.counts[t] = total[t];
}

// The first launch for many slots.  Workgroups below `blocks` group (one: all
// of it; several: each counts its part of the slots), the others bring rows as
// they are into two parts meanwhile.
__global__ void __launch_bounds__(kGroupThreads) prepare_kernel(const std::int32_t* __restrict__ ids, int slots, int experts,
                                                                Groups g, int blocks, RowSource src, int rows, SplitRows to) {
  __shared__ std::int32_t count[kMaxExperts];
  const int t = threadIdx.x, b = blockIdx.x;
  if (b >= blocks) {
    const int waves = (static_cast<int>(gridDim.x) - blocks) * (kGroupThreads / 64);
    for (int r = (b - blocks) * (kGroupThreads / 64) + (t >> 6); r < rows; r += waves)
      split_row<0>(src, static_cast<std::size_t>(r), r, to, t & 63);
    return;
  }
  if (blocks == 1) {
    group_slots(ids, slots, experts, g, count);
    return;
  }
  for (int e = t; e < experts; e += kGroupThreads) count[e] = 0;
  __syncthreads();
  const int each = (slots + blocks - 1) / blocks, end = min((b + 1) * each, slots);
  for (int i = b * each + t; i < end; i += kGroupThreads) {
    const std::int32_t e = ids[i];
    if (e >= 0 && e < experts) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  for (int e = t; e < experts; e += kGroupThreads) g.hist[b * experts + e] = count[e];
}
// The second one, of several parts: every workgroup sums up the counts and
// places its part of the slots.
__global__ void __launch_bounds__(kGroupThreads) place_kernel(const std::int32_t* __restrict__ ids, int slots, int experts,
                                                              Groups g, int blocks) {
  __shared__ std::int32_t count[kMaxExperts];
  const int t = threadIdx.x, b = blockIdx.x;
  for (int e = t; e < experts; e += kGroupThreads) {
    std::int32_t n = 0;
#pragma unroll 8
    for (int i = 0; i < blocks; ++i) n += g.hist[i * experts + e];
    count[e] = n;
  }
  __syncthreads();
  std::int32_t total[3];
  lay_ranges(count, experts, g, total, [&](int l, std::int32_t at, const RowTile& r) {
    if (r.expert % blocks == b) g.tiles[l][at] = r;
  });
  for (int e = t; e < experts; e += kGroupThreads) {
    std::int32_t n = 0;
#pragma unroll 8
    for (int i = 0; i < b; ++i) n += g.hist[i * experts + e];
    count[e] += n;
  }
  __syncthreads();
  const int each = (slots + blocks - 1) / blocks, end = min((b + 1) * each, slots);
  for (int i = b * each + t; i < end; i += kGroupThreads) {
    const std::int32_t e = ids[i];
    if (e >= 0 && e < experts) g.order[atomicAdd(&count[e], 1)] = i;
  }
  if (b == 0 && t < 3) g.counts[t] = total[t];
}

// Up to kSelfGroup slots, a wavefront each: it asks for its row of x, counts
// with its workgroup every expert's slots, and so finds its own place (slots
// keep their order), to which it brings the row; the place in the order and the
// groups of rows that start with its slot it stores for the products.
template <int MT>
__global__ void __launch_bounds__(kThreads) self_kernel(const std::int32_t* __restrict__ ids, int slots, int experts, Groups g,
                                                        RowSource src, SplitRows to) {
  constexpr int kEach = static_cast<int>(kSelfExperts) / 64;
  // Three counts in a word: slots, groups of either list.
  constexpr int kAt1 = 12, kAt2 = 22;
  static_assert(kSelfGroup < (1 << kAt1) && kSelfGroup / kLeastRows + kSelfExperts < (1 << (kAt2 - kAt1)));
  __shared__ std::int32_t count[kSelfExperts];
  __shared__ std::int16_t all[kSelfGroup];  // the slots' experts, -1: none
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int slot = blockIdx.x * kWaves + wave;
  for (int e = t; e < static_cast<int>(kSelfExperts); e += kThreads) count[e] = 0;
  __syncthreads();
  Row x(src, row_of(src, min(slot, slots - 1)), lane);
  for (int i = t; i < slots; i += kThreads) {
    const std::int32_t e = ids[i];
    const bool live = e >= 0 && e < experts;
    all[i] = static_cast<std::int16_t>(live ? e : -1);
    if (live) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  if (slot >= slots) return;
  const auto add = [](std::uint32_t a, std::uint32_t b) { return a + b; };
  const int shift0 = __builtin_ctz(g.rows[0]), shift1 = __builtin_ctz(g.rows[1]);
  std::uint32_t word[kEach], sum = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const std::uint32_t n = static_cast<std::uint32_t>(count[i * 64 + lane]);
    word[i] = n | (n + g.rows[0] - 1) >> shift0 << kAt1 | (n + g.rows[1] - 1) >> shift1 << kAt2;
    sum += word[i];
  }
  const auto part = [](std::uint32_t w, int i) {
    return static_cast<std::int32_t>(i == 0 ? w & ((1u << kAt1) - 1) : i == 1 ? w >> kAt1 & ((1u << (kAt2 - kAt1)) - 1) : w >> kAt2);
  };
  if (slot == 0) {
    sum = across(sum, add);
    if (lane < 3) g.counts[lane] = part(sum, lane);
  }
  const int e = __builtin_amdgcn_readfirstlane(all[slot]);
  if (e < 0) return;
  std::uint32_t before = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (i * 64 + lane < e) before += word[i];
  before = across(before, add);
  int rank = 0;
  for (int c = 0; c <= slot / 64; ++c) {
    const int i = c * 64 + lane;
    rank += __builtin_popcountll(__ballot(i < slot && all[i] == e));
  }
  const int r0 = g.rows[0], r1 = g.rows[1], n = count[e], begin = part(before, 0);
  const int group0 = part(before, 1), group1 = part(before, 2), tile0 = group0 + (rank >> shift0), tile1 = group1 + (rank >> shift1);
  if (lane == 0) {
    g.order[begin + rank] = slot;
    if ((rank & (r0 - 1)) == 0) g.tiles[0][tile0] = RowTile{e, begin, n, group0, (n + r0 - 1) >> shift0, group1, {}};
    if ((rank & (r1 - 1)) == 0) g.tiles[1][tile1] = RowTile{e, begin, n, group1, (n + r1 - 1) >> shift1, group1, {}};
  }
  store_row<MT>(x, src, tile0 * (MT * kTile) + rank % (MT * kTile), to);
}

}  // namespace

int launch_prepare(const std::int32_t* ids, std::size_t slots, std::size_t experts, const Groups& g, const RowSource& x,
                   const SplitRows& to, hipStream_t s) {
  const int n = static_cast<int>(slots), e = static_cast<int>(experts), r0 = g.rows[0];
  const bool tiled = r0 <= static_cast<int>(kMostShortRows);
  const std::size_t tile_rows = most_tiles(slots, experts, static_cast<std::size_t>(r0)) * static_cast<std::size_t>(r0);
  if (tiled && self_grouped(slots, experts)) {
    const unsigned grid = static_cast<unsigned>(ceil_div(slots, kWaves));
    if (r0 == 16) self_kernel<1><<<grid, kThreads, 0, s>>>(ids, n, e, g, x, to);
    else self_kernel<2><<<grid, kThreads, 0, s>>>(ids, n, e, g, x, to);
    LLMI_TRY_HIP(hipGetLastError());
    return LLMI_OK;
  }
  const int blocks = static_cast<int>(grouping_blocks(slots));
  const std::size_t rows = tiled ? 0 : ceil_div(slots, x.per_row);
  const unsigned grid = static_cast<unsigned>(blocks + std::min<std::size_t>(ceil_div(rows, kGroupThreads / 64), 1 << 16));
  prepare_kernel<<<grid, kGroupThreads, 0, s>>>(ids, n, e, g, blocks, x, static_cast<int>(rows), to);
  LLMI_TRY_HIP(hipGetLastError());
  if (blocks > 1) {
    place_kernel<<<static_cast<unsigned>(blocks), kGroupThreads, 0, s>>>(ids, n, e, g, blocks);
    LLMI_TRY_HIP(hipGetLastError());
  }
  if (tiled) {
    const unsigned tile_grid = static_cast<unsigned>(std::min<std::size_t>(ceil_div(tile_rows, kWaves), kMostGroups));
    if (r0 == 16) split_tiles_kernel<1><<<tile_grid, kThreads, 0, s>>>(x, g, to);
    else split_tiles_kernel<2><<<tile_grid, kThreads, 0, s>>>(x, g, to);
    LLMI_TRY_HIP(hipGetLastError());
  }
  return LLMI_OK;
}

int launch_split(const RowSource& x, std::size_t rows, const std::int32_t* live, const SplitRows& to, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(std::min<std::size_t>(ceil_div(rows, kWaves), kMostGroups));
  split_kernel<<<grid, kThreads, 0, s>>>(x, static_cast<int>(rows), live, to);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // namespace llmi_hip::moe
