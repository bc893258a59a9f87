// The experts' products on the matrix cores.
//
// y = sum over blocks b of scale[o][b] * (sum over the block of x * code):
// one fp16 matrix instruction of 16 rows x 16 outputs x 32 inputs sums a
// block.  Codes (-128 .. 127) are exact in fp16; x enters as two fp16 parts,
// high and low, of together 22 bits (a rounding of at most 2^-22 of each
// element, or 2^-39 of its row's largest), so each block takes two
// instructions into one fp32 sum, which is then multiplied by the block's
// fp32 scale and added in fp32.
#include <type_traits>

#include "moe_device.hpp"

namespace llmi_hip::moe {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kRowTiles = static_cast<int>(kRows) / kTile;

// x in two parts: one wavefront a row.  The factor is taken from the largest
// finite |x|: an inf or NaN stays one in the high part and shows in its own
// row alone.
__global__ void __launch_bounds__(kThreads) split_kernel(const float* __restrict__ x, int rows, int in, int chunks,
                                                         std::size_t stride, const std::int32_t* __restrict__ live,
                                                         SplitRows to) {
  const int lane = threadIdx.x & 63;
  const int most = live != nullptr ? min(*live, rows) : rows;
  for (int r = blockIdx.x * kWaves + (threadIdx.x >> 6); r < most; r += gridDim.x * kWaves) {
    const float* row = x + static_cast<std::size_t>(r) * stride;
    const auto load8 = [&](int k, float (&v)[8]) {
      if (k + 8 <= in) {
        const f4 a = *reinterpret_cast<const f4*>(row + k), b = *reinterpret_cast<const f4*>(row + k + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = a[i];
          v[4 + i] = b[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < in ? row[k + i] : 0.0f;
      }
    };
    std::uint32_t top = 0;
    for (int k = lane * 8; k < in; k += 512) {
      float v[8];
      load8(k, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, finite_bits(v[i]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(top), o, 64)));
    const Factor f(top);
    if (lane == 0) to.factors[r] = f.back;
    _Float16* out = to.values + static_cast<std::size_t>(r) * chunks * (kChunkBlocks * kBlock * 2);
    for (int k = lane * 8; k < chunks * kChunkBlocks * kBlock; k += 512) {
      float v[8];
      load8(k, v);
      f16x8 high, low;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        _Float16 a, b;
        two_parts(v[i] * f.up, a, b);
        high[i] = a;
        low[i] = b;
      }
      _Float16* at = out + (k / kBlock) * 2 * kBlock + k % kBlock;
      *reinterpret_cast<f16x8*>(at) = high;
      *reinterpret_cast<f16x8*>(at + kBlock) = low;
    }
  }
}

struct ProductArgs {
  Matrices m, up;
  SplitRows x;
  Groups g;
  float* y;
  std::size_t y_stride;
  int out, tiles, chunks, per_row, x_by_position, y_by_position, columns;  // columns: groups of 16 * kWaves * NT outputs
};

// A workgroup takes 64 rows of one expert and 4 wavefronts' outputs beside
// each other; the rows' parts of a chunk go through LDS.
template <int TYPE, int NT, bool GATED>
__global__ void __launch_bounds__(kThreads) product_kernel(ProductArgs p) {
  __shared__ __attribute__((aligned(16))) f16x8 xs[kRowTiles * kChunkBlocks * 2][64];
  constexpr int kMats = GATED ? 2 : 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int units = p.g.counts[1] * p.columns;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const RowTile rt = p.g.tiles[u / p.columns];
    const int col0 = (u % p.columns) * kWaves * NT + wave * NT;
    // The row that this lane stages: row lane % 16 of each tile of 16, rows
    // past the last one repeating it (their results are not stored).
    const _Float16* src[kRowTiles];
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i) {
      const int pos = rt.first + min(i * kTile + lane % kTile, rt.rows - 1);
      const std::size_t row = p.x_by_position ? static_cast<std::size_t>(pos) : static_cast<std::size_t>(p.g.order[pos] / p.per_row);
      src[i] = p.x.values + row * p.chunks * (kChunkBlocks * kBlock * 2) + lane / kTile * 8;
    }
    f32x4 acc[kMats][NT][kRowTiles] = {};
    for (int c = 0; c < p.chunks; ++c) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int part = wave * 2 + f;  // block, high / low
          xs[i * kChunkBlocks * 2 + part][lane] = *reinterpret_cast<const f16x8*>(src[i] + (c * kChunkBlocks * 2 + part) * kBlock);
        }
      __syncthreads();
      Chunk<TYPE> w[kMats][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const std::size_t at = (static_cast<std::size_t>(rt.expert) * p.tiles + min(col0 + n, p.tiles - 1)) * p.chunks + c;
        w[0][n].load(p.m, at, lane);
        if constexpr (GATED) w[1][n].load(p.up, at, lane);
      }
#pragma unroll
      for (int b = 0; b < kChunkBlocks; ++b)
#pragma unroll
        for (int m = 0; m < kMats; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const f16x8 code = w[m][n].codes(b);
#pragma unroll
            for (int i = 0; i < kRowTiles; ++i) {
              f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
              d = __builtin_amdgcn_mfma_f32_16x16x32_f16(xs[(i * kChunkBlocks + b) * 2][lane], code, d, 0, 0, 0);
              d = __builtin_amdgcn_mfma_f32_16x16x32_f16(xs[(i * kChunkBlocks + b) * 2 + 1][lane], code, d, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[m][n][i][r] = __builtin_fmaf(d[r], w[m][n].s[b], acc[m][n][i][r]);
            }
          }
    }
    // Lane l holds output l % 16 of rows 4 (l / 16) .. + 3.
#pragma unroll
    for (int i = 0; i < kRowTiles; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = i * kTile + lane / kTile * 4 + r;
        if (at >= rt.rows) continue;
        const int pos = rt.first + at, slot = p.g.order[pos];
        const float back = p.x.factors[p.x_by_position ? pos : slot / p.per_row];
        float* to = p.y + static_cast<std::size_t>(p.y_by_position ? pos : slot) * p.y_stride;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int o = (col0 + n) * kTile + lane % kTile;
          float v = acc[0][n][i][r] * back;
          if constexpr (GATED) v = silu(v) * (acc[kMats - 1][n][i][r] * back);
          if (o < p.out) to[o] = v;
        }
      }
  }
}

}  // namespace

int launch_split(const float* x, std::size_t rows, std::size_t in, std::size_t chunks, std::size_t stride,
                 const std::int32_t* live, const SplitRows& to, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(std::min<std::size_t>(ceil_div(rows, kWaves), kMostGroups));
  split_kernel<<<grid, kThreads, 0, s>>>(x, static_cast<int>(rows), static_cast<int>(in), static_cast<int>(chunks), stride, live, to);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

int launch_product(const Product& p, hipStream_t s) {
  const bool gated = p.up.codes != nullptr;
  const int nt = gated ? 1 : 2;
  const std::size_t columns = ceil_div(p.shape.tiles(), static_cast<std::size_t>(kWaves * nt));
  const std::size_t most = most_tiles(p.slots, p.shape.count) * columns;
  LLMI_REQUIRE(most <= 0x7FFFFFFFu, "moe: too many slots and results");
  const unsigned grid = static_cast<unsigned>(std::min<std::size_t>(most, kMostGroups));
  const ProductArgs a{p.m, p.up, p.x, p.g, p.y, p.y_stride, static_cast<int>(p.shape.out), static_cast<int>(p.shape.tiles()),
                      static_cast<int>(p.shape.chunks()), static_cast<int>(p.per_row), p.x_by_position, p.y_by_position,
                      static_cast<int>(columns)};
  if (p.shape.type == LLMI_TYPE_Q4_0) {
    if (gated) product_kernel<LLMI_TYPE_Q4_0, 1, true><<<grid, kThreads, 0, s>>>(a);
    else product_kernel<LLMI_TYPE_Q4_0, 2, false><<<grid, kThreads, 0, s>>>(a);
  } else {
    if (gated) product_kernel<LLMI_TYPE_Q8_0, 1, true><<<grid, kThreads, 0, s>>>(a);
    else product_kernel<LLMI_TYPE_Q8_0, 2, false><<<grid, kThreads, 0, s>>>(a);
  }
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // namespace llmi_hip::moe
