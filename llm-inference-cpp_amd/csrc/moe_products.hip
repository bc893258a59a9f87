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

struct ProductArgs {
  Matrices m, up;
  SplitRows x;
  Groups g;
  float* y;
  std::size_t y_stride;
  int out, tiles, steps, per_row, y_by_position, columns;  // columns: groups of outputs that a workgroup takes
  int first, list;  // unit of the first workgroup; which tile list
  SplitRows h;      // a gated pair's results in row tiles (values NULL: in y)
  int h_steps, h_rows;
};

// 8 results side by side of a gated pair (outputs 8 g .. of block `block`, by
// the lane of the row and g; rows beside each other's lanes write beside each
// other) in the row tiles of the second product, row `row` of tile `tile`.
// Lanes l, l + 16, l + 32, l + 48 hold a row's block and have to be active together.
__device__ __forceinline__ void store_parts(const ProductArgs& p, int tile, int row, int block, int g, const float (&v)[8], bool live) {
  std::uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, finite_bits(v[i]));
  const Factor f(across_rows(top, Larger{}));
  f16x8 high, low;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    _Float16 a, b;
    two_parts(v[i] * f.up, a, b);
    high[i] = a;
    low[i] = b;
  }
  if (!live) return;
  const std::size_t piece = ((static_cast<std::size_t>(tile) * p.h_steps + block / 2) * (p.h_rows / kTile) + row / kTile) * 4 + block % 2 * 2;
  f16x8* const at = reinterpret_cast<f16x8*>(p.h.values) + piece * 64 + g * kTile + row % kTile;
  at[0] = high;
  at[64] = low;
  if (g == 0) p.h.factors[(static_cast<std::size_t>(tile) * p.h_steps * 2 + block) * p.h_rows + row] = f.back;
}

// 16 bytes of each lane, OFFSET behind its own address, into LDS, lane after
// lane from `to` (common to the wavefront).  Nothing waits for it but landed().
// The instruction adds its offset to both addresses; between a write of m0 and
// such a load this family needs one wait state, which nobody inserts in here.
// m0 is named as written, so that no m0 of the compiler's lives across it; that
// it is no register to allocate, as the compiler would warn, is known.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int OFFSET>
__device__ __forceinline__ void to_lds(const std::uint8_t* from, std::uint32_t to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off offset:%2" ::"v"(from), "s"(to - OFFSET), "n"(OFFSET) : "memory", "m0");
}
// The same from an address common to the wavefront and each lane's offset.
__device__ __forceinline__ void to_lds_from(GlobalBytes from, std::uint32_t offset, std::uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(from), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
// All of this wavefront's loads have landed and its reads of LDS are done;
// then those of the workgroup's.
__device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The group of rows and the outputs of a unit.  In the order of units come the
// experts, of each up to 8 groups of rows at a time, of these all columns, and of
// a column those groups: so what runs at a time on an XCD shares weights as well
// as rows in its L2 (group after group, 1024 tokens of 2 of 8 Q8_0 experts of
// 4096 x 8192 took 968 us, this way 875, 64 tokens 267 and 247; experts that fit
// into the L2 take the same).
struct Unit {
  int tile, col, expert, first, rows, next;
};
template <int ROWS>
__device__ __forceinline__ Unit unit_of(const ProductArgs& p, int u) {
  constexpr int kBeside = 8;
  const RowTile t = (p.list == 0 ? p.g.tiles[0] : p.g.tiles[1])[u / p.columns];
  const int groups = __builtin_amdgcn_readfirstlane(t.groups), group0 = __builtin_amdgcn_readfirstlane(t.group0);
  const int begin = __builtin_amdgcn_readfirstlane(t.begin), slots = __builtin_amdgcn_readfirstlane(t.slots);
  std::uint32_t col = u - group0 * p.columns, group = 0;
  if (groups > 1) {
    std::uint32_t first = 0;
    if (groups > kBeside) {
      const std::uint32_t block = col / (kBeside * p.columns);
      first = block * kBeside;
      col -= first * p.columns;
    }
    const std::uint32_t beside = min(kBeside, groups - static_cast<int>(first)), in_block = col;
    col = in_block / beside;
    group = first + in_block - col * beside;
  }
  const int row = static_cast<int>(group) * ROWS;
  return {group0 + static_cast<int>(group), static_cast<int>(col), __builtin_amdgcn_readfirstlane(t.expert), begin + row, min(slots - row, ROWS),
          __builtin_amdgcn_readfirstlane(t.next0) + (row >> __builtin_ctz(p.h_rows))};
}

// fn of 0 .. N - 1 as constants.
template <int N, typename Fn>
__device__ __forceinline__ void each(Fn&& fn) {
  if constexpr (N > 0) {
    each<N - 1>(fn);
    fn(std::integral_constant<int, N - 1>{});
  }
}

// A workgroup takes 16 MT rows of one expert and, with its 4 wavefronts beside
// each other, 64 NT outputs (32 NT of each matrix of a gated pair).  The rows'
// parts go through LDS, 64 inputs at a time in two buffers, filled while the
// other one is used.  A wavefront's weights come through LDS of its own, a step
// (Q8_0) or two (Q4_0) ahead, and are taken into registers in the middle of the
// step before theirs: asked for into registers instead, they were half as long
// on their way or left room for two wavefronts a SIMD (4096 rows against 16
// Q4_0 experts of 896 x 4864: 85 -> 80 us).  Bound by the vector units beside
// the matrix units, and by power: two matrix instructions (32 clocks) have 4
// additions (16), a quarter of a block's 10 conversions and the reads of LDS
// beside them.  32768 rows against Q4_0 pairs of 2048 x 1024: 480 to 550 us by
// the card's clock, 1.0 to 1.1 PFLOP/s of matrix instructions (a large fp16
// library product reaches 1.37); back to 2048: 255 to 290 us.  128 rows a
// workgroup halve the conversions but take the registers of a third wavefront,
// and were no faster; chains of 32 x 32 x 16 instructions, with a quarter of the
// scales' additions hidden, were slower.
template <int TYPE, int MT, int NT, bool GATED>
__global__ void __launch_bounds__(kThreads, 3) long_kernel(ProductArgs p) {
  static_assert(MT == kWaves && NT == 4);
  constexpr int kParts = MT * 4;  // 1 KiB pieces of a buffer: (16 rows, block, high / low)
  constexpr int kCodes = static_cast<int>(code_bytes(TYPE)), kScales = static_cast<int>(kStepScales) * 4;
  // Steps of weights on their way at once, as three workgroups' LDS has room;
  // a wavefront's loads of a step of rows and of weights.
  constexpr int kAhead = TYPE == LLMI_TYPE_Q4_0 ? 2 : 1, kRowLoads = 4, kLoads = TYPE == LLMI_TYPE_Q4_0 ? 4 : 6;
  __shared__ __attribute__((aligned(16))) f16x8 xs[2][kParts][64];
  __shared__ __attribute__((aligned(16))) std::uint8_t ws[kWaves][kAhead][NT * (kCodes + kScales)];  // a wavefront's: codes, then scales
  __shared__ std::int32_t to_row[MT * kTile];  // y's rows, and the factors of x's
  __shared__ float back[MT * kTile];
  constexpr int kCols = GATED ? NT / 2 : NT;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int units = p.g.counts[1 + p.list] * p.columns;
  // Workgroups go to the 8 XCDs in turn: each XCD takes neighbouring units.
  const int per = (units + 7) / 8, b = p.first + static_cast<int>(blockIdx.x), u = b % 8 * per + b / 8;
  if (b / 8 >= per || u >= units) return;
  const Unit unit = unit_of<MT * kTile>(p, u);
  const int expert = unit.expert, first = unit.first, rows = unit.rows, col0 = (unit.col * kWaves + wave) * kCols;
  // Rows past the last one repeat it; their results are not stored.
  const auto x_row = [&](int pos) { return p.per_row == 0 ? pos : p.g.order[pos] / p.per_row; };
  if (threadIdx.x < MT * kTile) {
    const int pos = first + min(static_cast<int>(threadIdx.x), rows - 1);
    to_row[threadIdx.x] = p.y_by_position ? pos : p.g.order[pos];
    back[threadIdx.x] = p.x.factors[x_row(pos)];
  }
  // The rows that this lane brings in: row lane / 4 of the wavefront's tile of
  // 16, so that 4 lanes read 64 bytes beside each other.  In LDS a row's four 16
  // bytes lie side by side, in an order that differs from 4 rows to the next:
  // lanes that read one input group of 16 rows use all banks.
  const std::uint8_t* src = reinterpret_cast<const std::uint8_t*>(p.x.values) +
                            static_cast<std::size_t>(x_row(first + min(wave * kTile + lane / 4, rows - 1))) * p.steps * (kStep * 4) +
                            (lane % 4 ^ (4 - lane / 16) % 4) * 16;
  const int read_at = lane % kTile * 4 + (lane / kTile ^ (4 - lane % kTile / 4) % 4);
  const std::uint32_t lds = static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(&xs[0][0][0]));
  const auto bring = [&](int buf) {  // the next 64 inputs
    const std::uint32_t to = lds + (buf * kParts + wave * 4) * 1024;
    to_lds<0>(src, to);
    to_lds<64>(src, to + 1 * 1024);
    to_lds<128>(src, to + 2 * 1024);
    to_lds<192>(src, to + 3 * 1024);
    src += 256;
  };
  // Weights, two tiles of a matrix at a time: their codes, then their scales.
  GlobalBytes at[NT / 2];
  std::uint32_t apart[NT / 2];  // from the first tile to the second
#pragma unroll
  for (int n = 0; n < NT; n += 2) {
    const int col = min(col0 + n % kCols, p.tiles - 1);
    at[n / 2] = tile_at<TYPE>(n < kCols ? p.m : p.up, static_cast<std::size_t>(expert) * p.tiles + col, p.steps);
    apart[n / 2] = (min(col0 + n % kCols + 1, p.tiles - 1) - col) * static_cast<std::uint32_t>(p.steps) * static_cast<std::uint32_t>(step_bytes(TYPE));
  }
  const std::uint32_t lds_w = static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>(&ws[0][0][0])) + wave * kAhead * NT * (kCodes + kScales);
  const auto bring_weights = [&](int buf, int step) {
    const std::uint32_t to = lds_w + buf * (NT * (kCodes + kScales));
#pragma unroll
    for (int n = 0; n < NT; n += 2) {
      const GlobalBytes from = at[n / 2] + static_cast<std::uint32_t>(step) * static_cast<std::uint32_t>(step_bytes(TYPE));
      if constexpr (TYPE == LLMI_TYPE_Q4_0) {
        to_lds_from(from, lane / 32 * apart[n / 2] + lane % 32 * 16, to + n * kCodes);
      } else {
        to_lds_from(from, lane * 16, to + n * kCodes);
        to_lds_from(from, apart[n / 2] + lane * 16, to + (n + 1) * kCodes);
      }
      if (lane < 16) to_lds_from(from, lane / 8 * apart[n / 2] + kCodes + lane % 8 * 16, to + NT * kCodes + n * kScales);
    }
  };
  std::uint32_t raw[NT][kCodes / 256];
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
  f32x2 scale[2][NT];
  const auto take = [&](int buf, f32x2 (&s)[NT]) {
    const std::uint8_t* const from = &ws[wave][buf][0];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if constexpr (TYPE == LLMI_TYPE_Q4_0) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(from + n * kCodes + lane * 8);
        raw[n][0] = v[0];
        raw[n][1] = v[1];
      } else {
        const u32x4 v = *reinterpret_cast<const u32x4*>(from + n * kCodes + lane * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[n][i] = v[i];
      }
      s[n] = *reinterpret_cast<const f32x2*>(from + NT * kCodes + n * kScales + lane % kTile * 8);
    }
  };
  const auto codes = [&](int n, int block) {
    if constexpr (TYPE == LLMI_TYPE_Q4_0) return codes_q4(raw[n][block]);
    else return codes_q8(raw[n][2 * block], raw[n][2 * block + 1]);
  };
  const int last = p.steps - 1;
  f32x4 acc[NT][MT] = {};
  bring(0);
#pragma unroll
  for (int i = 0; i < kAhead; ++i) bring_weights(i, min(i, last));
  landed();
  take(0, scale[0]);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  bring_weights(0, min(kAhead, last));
  for (int h = 0; h < p.steps; h += 2) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (h + j >= p.steps) break;
      if (h + j < last) bring(1 - j);
      // Two outputs' tiles at a time: their four instructions, beside them the
      // additions of the two before, whose results are there by now.  The
      // regions keep the compiler from holding more operands at once than the
      // registers have room for.
      f16x8 code[NT];
      f16x8 x[2][2];
      f32x4 d[2][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) code[n] = codes(n, 0);
      x[0][0] = xs[j][0][read_at];
      x[0][1] = xs[j][1][read_at];
      constexpr int kPairs = NT / 2, kSteps = 2 * MT * kPairs;
      const auto add = [&](auto step) {
        constexpr int q = decltype(step)::value, i = q / kPairs % MT, n0 = q % kPairs * 2, b2 = q / (kPairs * MT);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[n0 + n][i][r] = __builtin_fmaf(d[q % 2][n][r], scale[j][n0 + n][b2], acc[n0 + n][i][r]);
        // Here, not at the end of the block, where the compiler would put them all.
#pragma unroll
        for (int n = 0; n < 2; ++n) asm volatile("" : "+v"(acc[n0 + n][i]));
      };
      each<kSteps>([&](auto step) {
        constexpr int q = decltype(step)::value, ib = q / kPairs, i = ib % MT, n0 = q % kPairs * 2, b2 = ib / MT;
        // The next step's weights, whose registers are free: this step's second
        // block has become fp16.  Loads come back in order; younger than these
        // weights are the next rows (and, of Q4_0, the weights after them).
        if constexpr (q == kSteps / 2) {
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kRowLoads + (kAhead - 1) * kLoads) : "memory");
          take((j + 1) % kAhead, scale[1 - j]);
        }
        if constexpr (q == kSteps / 2 + 2) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          bring_weights((j + 1) % kAhead, min(h + j + 1 + kAhead, last));
        }
        if constexpr (n0 == 0 && ib + 1 < 2 * MT) {  // the next rows' parts
          x[(ib + 1) % 2][0] = xs[j][(ib + 1) % MT * 4 + (ib + 1) / MT * 2][read_at];
          x[(ib + 1) % 2][1] = xs[j][(ib + 1) % MT * 4 + (ib + 1) / MT * 2 + 1][read_at];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) d[q % 2][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[ib % 2][0], code[n0 + n], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < 2; ++n) d[q % 2][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[ib % 2][1], code[n0 + n], d[q % 2][n], 0, 0, 0);
        if constexpr (q > 0) add(std::integral_constant<int, q - 1>{});
        if constexpr (b2 == 0 && i == MT - 1) {  // the next block's codes
#pragma unroll
          for (int n = 0; n < 2; ++n) code[n0 + n] = codes(n0 + n, 1);
        }
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                              // one matrix instruction,
          __builtin_amdgcn_sched_group_barrier(0x002, b2 == 0 && i == MT - 1 ? 6 : 2, 0);  // vector ones beside it
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      add(std::integral_constant<int, kSteps - 1>{});
      // The next rows have landed (only weights are younger), and all have read these.
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLoads) : "memory");
    }
  }
  landed();  // nothing is on its way into LDS any more
  if constexpr (GATED) {
    if (p.h.values != nullptr) {
      // The wavefront's outputs of a row are one block (kCols is 2).  16 rows at
      // a time go through its part of LDS, from a lane's rows to a lane's outputs.
      constexpr int kStride = kCols * kTile + 4;  // 16-byte rows whose quads meet all banks
      float* const turn = reinterpret_cast<float*>(&xs[0][0][0]) + wave * kTile * kStride;
      const int block = col0 / kCols;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        if (i * kTile >= rows) break;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = lane / kTile * 4 + r;
          const float f = back[i * kTile + row];
#pragma unroll
          for (int n = 0; n < kCols; ++n) {
            const float v = silu(acc[n][i][r] * f) * (acc[kCols + n][i][r] * f);
            turn[row * kStride + n * kTile + lane % kTile] = (col0 + n) * kTile + lane % kTile < p.out ? v : 0.0f;
          }
        }
        wave_sync();
        const f32x4* const at = reinterpret_cast<const f32x4*>(turn + lane % kTile * kStride + lane / kTile * 8);
        const f32x4 a = at[0], b8 = at[1];
        const float v[8] = {a[0], a[1], a[2], a[3], b8[0], b8[1], b8[2], b8[3]};
        const int row = i * kTile + lane % kTile;
        store_parts(p, unit.next + i * kTile / p.h_rows, row % p.h_rows, block, lane / kTile, v, row < rows && block < p.h_steps * 2);
        wave_sync();
      }
      return;
    }
  }
  // Lane l holds output l % 16 of rows 4 (l / 16) .. + 3.
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (i * kTile >= rows) break;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = i * kTile + lane / kTile * 4 + r;
      const float f = back[row];
      if constexpr (GATED) {
        float v[kCols];
#pragma unroll
        for (int n = 0; n < kCols; ++n) v[n] = silu(acc[n][i][r] * f) * (acc[kCols + n][i][r] * f);
        float* const to = p.y + static_cast<std::size_t>(to_row[row]) * p.y_stride;
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
          const int o = (col0 + n) * kTile + lane % kTile;
          if (row < rows && o < p.out) to[o] = v[n];
        }
      } else {
        float* const to = p.y + static_cast<std::size_t>(to_row[row]) * p.y_stride;
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
          const int o = (col0 + n) * kTile + lane % kTile;
          if (row < rows && o < p.out) to[o] = acc[n][i][r] * f;
        }
      }
    }
  }
}

// The same for few rows an expert, or little work: no LDS on the way.  A
// workgroup takes 16 MT rows and 16 NT outputs (8 NT of each matrix of a
// gated pair); its 4 wavefronts share the inputs, each with its own loads of
// rows and weights in flight while it works on those before them, and their
// sums meet in LDS, in their order.  Bound by the weights' way from memory and
// its latency: 512 rows of 64 Q4_0 experts, pairs of 2048 x 1024 40 us at 4.2 TB/s
// of weights, back to 2048 25 us at 3.4, Q8_0 2048 x 1024 28 us at 5.4 (out of the
// last-level cache); vector units issue in 38 % of the clocks, matrix units are
// busy in 17 %.  Wavefronts beside each other that share a ring of 4 steps of
// rows in LDS halve the reads from L2 and were a tenth slower: a CU then has 2 or
// 3 workgroups, where it has 9 of these.
// BLOCKS: every block of a row of x has a factor of its own.
template <int TYPE, int MT, int NT, bool GATED, bool BLOCKS>
__global__ void __launch_bounds__(kThreads, MT == 1 ? 4 : 3) short_kernel(ProductArgs p) {
  constexpr int kCols = GATED ? NT / 2 : NT;
  __shared__ __attribute__((aligned(16))) float meet[kWaves][NT][MT][kTile][kTile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int units = p.g.counts[1 + p.list] * p.columns;
  const int per = (units + 7) / 8, b = p.first + static_cast<int>(blockIdx.x), u = b % 8 * per + b / 8;
  if (b / 8 >= per || u >= units) return;
  const Unit unit = unit_of<MT * kTile>(p, u);
  const int tile = unit.tile, expert = unit.expert, first = unit.first, rows = unit.rows, col0 = unit.col * kCols;
  // This wavefront's steps.
  const int share = (p.steps + kWaves - 1) / kWaves;
  const int h0 = min(wave * share, p.steps), h1 = min(h0 + share, p.steps);
  const std::uint8_t* const src = reinterpret_cast<const std::uint8_t*>(p.x.values) + static_cast<std::size_t>(tile) * p.steps * (MT * 4096);
  GlobalBytes at[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
    at[n] = tile_at<TYPE>(n < kCols ? p.m : p.up, static_cast<std::size_t>(expert) * p.tiles + min(col0 + n % kCols, p.tiles - 1), p.steps);
  struct Stage {
    Weights<TYPE> w[NT];
    f16x8 x[MT][4];              // block, high / low
    f32x4 f[BLOCKS ? MT : 1][2];  // factors of the lane's rows of a result
  };
  LaneAt lane_at(lane);
  std::uint32_t x_at = (lane / kTile * kTile + min(lane % kTile, rows - 1)) * 16;
  const auto ask = [&](Stage& s, int h) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s.w[n].load(at[n], h, lane_at);
    asm volatile("" : "+v"(x_at));
    const GlobalBytes from = (GlobalBytes)src + static_cast<std::size_t>(h) * (MT * 4096);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int f = 0; f < 4; ++f) s.x[i][f] = *(const __attribute__((address_space(1))) f16x8*)(from + (i * 4 + f) * 1024 + x_at);
    if constexpr (BLOCKS) {
      const float* const at_factors = p.x.factors + (static_cast<std::size_t>(tile) * p.steps + h) * (2 * MT * kTile);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int b2 = 0; b2 < 2; ++b2) s.f[i][b2] = *reinterpret_cast<const f32x4*>(at_factors + (b2 * MT + i) * kTile + lane / kTile * 4);
    }
  };
  f32x4 acc[NT][MT] = {};
  const auto work = [&](const Stage& s) {
#pragma unroll
    for (int b2 = 0; b2 < 2; ++b2)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const f16x8 code = s.w[n].codes(b2);
        f32x4 d[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) d[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(s.x[i][2 * b2], code, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) d[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(s.x[i][2 * b2 + 1], code, d[i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // The sum first by its scale, then by the power of two: scale times
            // factor may lie below the normal numbers, where it would lose bits.
            if constexpr (BLOCKS) acc[n][i][r] = __builtin_fmaf(d[i][r] * s.w[n].s[b2], s.f[i][b2][r], acc[n][i][r]);
            else acc[n][i][r] = __builtin_fmaf(d[i][r], s.w[n].s[b2], acc[n][i][r]);
          }
      }
  };
  if (h0 < h1) {
    // One step in flight behind the one that is worked on, by many wavefronts:
    // with two, half as many fit and a kernel takes a tenth longer.
    Stage s0, s1;
    ask(s0, h0);
    for (int h = h0; h < h1; h += 2) {
      ask(s1, min(h + 1, h1 - 1));
      work(s0);
      if (h + 1 >= h1) break;
      ask(s0, min(h + 2, h1 - 1));
      work(s1);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) meet[wave][n][i][lane / kTile * 4 + r][lane % kTile] = acc[n][i][r];
  __syncthreads();
  if constexpr (GATED) {
    if (p.h.values != nullptr) {
      // A wavefront 16 rows, a lane 8 outputs of one (the 32 of kCols 2 are a block).
      if (wave >= MT) return;
      const int row = wave * kTile + lane % kTile, g = lane / kTile, block = col0 / kCols;
      float v[8], u[8] = {};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const f32x4 a = *reinterpret_cast<const f32x4*>(&meet[w][g / 2][wave][lane % kTile][g % 2 * 8 + q * 4]);
          const f32x4 c = *reinterpret_cast<const f32x4*>(&meet[w][kCols + g / 2][wave][lane % kTile][g % 2 * 8 + q * 4]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[q * 4 + i] += a[i];
            u[q * 4 + i] += c[i];
          }
        }
      const bool live = row < rows;
      const float f = live ? p.x.factors[tile * (MT * kTile) + row] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (col0 * kTile + g * 8 + i < p.out) ? silu(v[i] * f) * (u[i] * f) : 0.0f;
      const int to = unit.next + wave * kTile / p.h_rows;
      store_parts(p, to, row % p.h_rows, block, g, v, live);
      // A last step's second block without outputs is 0.
      if (block == p.columns - 1 && block + 1 < p.h_steps * 2) {
        const float none[8] = {};
        store_parts(p, to, row % p.h_rows, block + 1, g, none, live);
      }
      return;
    }
  }
  for (int t = threadIdx.x; t < min(rows, MT * kTile) * (kCols * kTile); t += kThreads) {
    const int row = t / (kCols * kTile), col = t % (kCols * kTile), o = col0 * kTile + col;
    const int n = col / kTile, i = row / kTile;
    if (o >= p.out) continue;
    float v[2] = {0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      v[0] += meet[w][n][i][row % kTile][col % kTile];
      if constexpr (GATED) v[1] += meet[w][kCols + n][i][row % kTile][col % kTile];
    }
    const int pos = first + row;
    if constexpr (!BLOCKS) {
      const float f = p.x.factors[tile * (MT * kTile) + row];
      v[0] *= f;
      v[1] *= f;
    }
    p.y[static_cast<std::size_t>(p.y_by_position ? pos : p.g.order[pos]) * p.y_stride + o] = GATED ? silu(v[0]) * v[1] : v[0];
  }
}

}  // namespace

int launch_product(const Product& p, hipStream_t s) {
  const bool gated = p.up.steps != nullptr;
  constexpr int kNT = 4;
  const int rows = p.g.rows[p.list];
  const std::size_t cols = rows <= static_cast<int>(kMostShortRows) ? short_columns(gated) : long_columns(gated);
  const std::size_t columns = ceil_div(p.shape.tiles(), cols);
  const std::size_t all = ceil_div(most_tiles(p.slots, p.shape.count, static_cast<std::size_t>(rows)) * columns, 8) * 8;
  ProductArgs a{p.m, p.up, p.x, p.g, p.y, p.y_stride, static_cast<int>(p.shape.out), static_cast<int>(p.shape.tiles()),
                static_cast<int>(p.shape.steps()), static_cast<int>(p.per_row), p.y_by_position, static_cast<int>(columns), 0, p.list,
                p.h, static_cast<int>(p.h_steps), p.g.rows[1]};
  for (std::size_t first = 0; first < all; first += kMostGroups) {
    a.first = static_cast<int>(first);
    const unsigned grid = static_cast<unsigned>(std::min(all - first, kMostGroups));
    const auto run = [&](auto type, auto gate) {
      switch (rows) {
        case 16:
          if (!gate && p.block_factors) short_kernel<type, 1, kNT, false, true><<<grid, kThreads, 0, s>>>(a);
          else short_kernel<type, 1, kNT, gate, false><<<grid, kThreads, 0, s>>>(a);
          break;
        case 32:
          if (!gate && p.block_factors) short_kernel<type, 2, kNT, false, true><<<grid, kThreads, 0, s>>>(a);
          else short_kernel<type, 2, kNT, gate, false><<<grid, kThreads, 0, s>>>(a);
          break;
        default: long_kernel<type, 4, kNT, gate><<<grid, kThreads, 0, s>>>(a); break;
      }
    };
    constexpr std::integral_constant<int, LLMI_TYPE_Q4_0> q4{};
    constexpr std::integral_constant<int, LLMI_TYPE_Q8_0> q8{};
    if (p.shape.type == LLMI_TYPE_Q4_0) gated ? run(q4, std::true_type{}) : run(q4, std::false_type{});
    else gated ? run(q8, std::true_type{}) : run(q8, std::false_type{});
  }
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // namespace llmi_hip::moe
