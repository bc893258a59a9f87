// The experts' products for few slots (up to 64): decoding users.
//
// What bounds them is the weights' way from memory and the time until the
// first of them arrives (one token's 2 of 8 Q8_0 experts of 4096 x 8192: 29.8 us
// for the pair of matrices, 5.1 TB/s, 16.1 for the third, 4.7; 8 of 64 Q4_0
// experts of 2048 x 1024: 7.9 and 7.1 us, of which half is latency; one product
// of 2 of 8, 576 x 1536: a launch).  So there is one launch a product (two for an MLP):
// every workgroup finds its expert's slots in the ids by itself, its
// wavefronts share the inputs of one tile of 16 outputs and ask for all of
// their weights at once, and x is brought into its two fp16 parts on the way,
// each chunk of 128 inputs of a row with its own power of two, by the
// wavefront that uses it: no barrier until the wavefronts' sums meet.
#include <type_traits>

#include "moe_device.hpp"

namespace llmi_hip::moe {
namespace {

constexpr int kChunk = 2 * kStep;  // inputs that a wavefront takes at a time
constexpr int kMostRows = 8;  // rows of an expert that a wavefront takes at a time
constexpr int kRowBytes = kChunk * 4 + 16;  // a row of a chunk in LDS, both parts; 16 bytes keep rows off each other's banks

// A wavefront's part of LDS: 2 or kMostRows rows of a chunk in two parts, and what
// each row's sum is multiplied by.
struct WaveLds {
  std::uint8_t* rows;
  float* factors;
};

// Four inputs of each of 2 * PAIRS rows: lanes 0 .. 31 hold row 2p of pair p,
// the others row 2p + 1; lane l inputs 4 (l % 32) .. of the chunk.
// QUADS: rows of a multiple of 4 inputs.
template <int PAIRS, bool QUADS>
struct Rows {
  f32x4 v[PAIRS];
  // Every address is inside the row; what lies behind it is put to 0 when the
  // rows are stored, so that nothing here waits for a load.
  __device__ __forceinline__ void load(int p, const float* row, int chunk, int in, int lane) {
    const int k = chunk * kChunk + lane % 32 * 4;
    if constexpr (QUADS) {
      v[p] = *reinterpret_cast<const f4*>(row + min(k, in - 4));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[p][i] = row[min(k + i, in - 1)];
    }
  }
  __device__ __forceinline__ void store(const WaveLds& to, int chunk, int in, int lane) const {
    const int k = lane % 32 * 4, left = in - chunk * kChunk - k;
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) {
      float x[4];
      std::uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = i < left ? v[p][i] : 0.0f;
        top = max(top, finite_bits(x[i]));
      }
      top = max_of_half(top);
      const Factor f(top);
      f16x4 high, low;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        _Float16 a, b;
        two_parts(x[i] * f.up, a, b);
        high[i] = a;
        low[i] = b;
      }
      const int row = 2 * p + lane / 32;
      std::uint8_t* at = to.rows + row * kRowBytes + k / kBlock * (4 * kBlock) + k % kBlock * 2;
      *reinterpret_cast<f16x4*>(at) = high;
      *reinterpret_cast<f16x4*>(at + 2 * kBlock) = low;
      if (lane % 32 == 0) to.factors[row] = f.back;
    }
  }
};

// Block b of a chunk's rows times one tile's codes: rows 4 (l / 16) .., output
// l % 16.  at: this lane's row and inputs.
__device__ __forceinline__ f32x4 times_codes(const std::uint8_t* at, int b, const f16x8& code) {
  const f16x8 high = *reinterpret_cast<const f16x8*>(at + b * (4 * kBlock));
  const f16x8 low = *reinterpret_cast<const f16x8*>(at + b * (4 * kBlock) + 2 * kBlock);
  f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
  d = __builtin_amdgcn_mfma_f32_16x16x32_f16(high, code, d, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(low, code, d, 0, 0, 0);
}
// Rows past the ROWS that count read the last one: their results mean nothing.
template <int ROWS>
__device__ __forceinline__ const std::uint8_t* lane_row(const std::uint8_t* rows, int lane) {
  return rows + min(lane % kTile, ROWS - 1) * kRowBytes + lane / kTile * 16;
}

// acc += factor * (x W^T) over one chunk, of MATS tiles.
template <int TYPE, int MATS, int ROWS>
__device__ __forceinline__ void add_chunk(f32x4 (&acc)[MATS], const Weights<TYPE> (&w)[MATS][2], const WaveLds& lds, int lane) {
  constexpr int kR = ROWS < 4 ? ROWS : 4;
  const std::uint8_t* const at = lane_row<ROWS>(lds.rows, lane);
  f32x4 sum[MATS] = {};
#pragma unroll
  for (int b = 0; b < 4; ++b)
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
      const f32x4 d = times_codes(at, b, w[m][b / 2].codes(b % 2));
#pragma unroll
      for (int r = 0; r < kR; ++r) sum[m][r] = __builtin_fmaf(d[r], w[m][b / 2].s[b % 2], sum[m][r]);
    }
  const f32x4 f = *reinterpret_cast<const f32x4*>(lds.factors + lane / kTile * 4);
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int r = 0; r < kR; ++r) acc[m][r] = __builtin_fmaf(sum[m][r], f[r], acc[m][r]);
}

struct FewArgs {
  Matrices m, up;
  const std::int32_t* ids;
  const float* x;
  float* y;
  FewParts h;
  std::size_t x_stride, y_stride;
  int slots, per_row, experts, out, in, tiles, pairs, steps, chunks, rows;  // rows: LDS rows of a wavefront
};

// ------------------------------------------------- products of each slot

constexpr int kWaves = 8, kThreads = kWaves * 64;

// One workgroup for each slot and 32 outputs (two tiles); the first slot of
// an expert takes all of its slots, the others leave.  A gated pair's results
// go to p.h in two parts, each 32 of a row with their own power of two.
// 32 outputs, since 16 would have every row brought into its parts twice as
// often (one token of 64 experts 17.7 -> 16.5 us, of 4096 x 8192 58.7 -> 54.7).
template <int TYPE, bool GATED, bool MORE, bool QUADS>
__global__ void __launch_bounds__(kThreads) few_kernel(FewArgs p) {
  extern __shared__ __attribute__((aligned(16))) std::uint8_t lds[];
  constexpr int kMats = GATED ? 4 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = blockIdx.x / p.pairs, pair = blockIdx.x % p.pairs;
  const std::int32_t mine = lane < p.slots ? p.ids[lane] : -1;
  const int expert = __builtin_amdgcn_readlane(mine, slot);
  if (expert < 0 || expert >= p.experts) return;
  std::uint64_t same = __ballot(mine == expert);
  if (__builtin_ctzll(same) != slot) return;
  const std::size_t tile0 = static_cast<std::size_t>(expert) * p.tiles;
  GlobalBytes from[kMats];
#pragma unroll
  for (int m = 0; m < kMats; ++m) from[m] = tile_at<TYPE>(m < 2 ? p.m : p.up, tile0 + min(pair * 2 + m % 2, p.tiles - 1), p.steps);
  const int each = (p.chunks + kWaves - 1) / kWaves;
  const int c0 = min(wave * each, p.chunks), c1 = min(c0 + each, p.chunks);
  const WaveLds w{lds + wave * (p.rows * kRowBytes + 64), reinterpret_cast<float*>(lds + wave * (p.rows * kRowBytes + 64) + p.rows * kRowBytes)};
  float* const meet = reinterpret_cast<float*>(lds);
  LaneAt lane_at(lane);

  while (same != 0) {
    // Up to kMostRows of the expert's slots at a time: lane r holds the r-th.
    const int rows = min(__builtin_popcountll(same), MORE ? kMostRows : 2);
    int row_slot = 0;
    for (int r = 0; r < rows; ++r) {
      const int at = __builtin_ctzll(same);
      same &= same - 1;
      if (lane == r) row_slot = at;
    }
    f32x4 acc[kMats] = {};
    const auto take = [&](auto count) {
      constexpr int kRows = decltype(count)::value, kPairs = (kRows + 1) / 2, kDepth = 2;
      const float* at[kPairs];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int r = min(2 * i + lane / 32, rows - 1);
        at[i] = p.x + static_cast<std::size_t>(__shfl(row_slot, r, 64) / p.per_row) * p.x_stride;
      }
      // Chunks in flight: the ring's places are filled kDepth chunks ahead.
      Weights<TYPE> ring[kDepth][kMats][2];
      Rows<kPairs, QUADS> x[kDepth];
      const auto ask = [&](int i, int c) {
        // The last chunk may have one step only: taken twice, with x 0 behind its end.
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int step = min(2 * c + t, p.steps - 1);
#pragma unroll
          for (int m = 0; m < kMats; ++m) ring[i][m][t].load(from[m], step, lane_at);
        }
#pragma unroll
        for (int j = 0; j < kPairs; ++j) x[i].load(j, at[j], c, p.in, lane);
      };
#pragma unroll
      for (int i = 0; i < kDepth; ++i)
        if (c0 + i < c1) ask(i, c0 + i);
      for (int c = c0; c < c1; c += kDepth)
#pragma unroll
        for (int i = 0; i < kDepth; ++i) {
          if (c + i >= c1) break;
          x[i].store(w, c + i, p.in, lane);
          wave_sync();
          add_chunk<TYPE, kMats, kRows>(acc, ring[i], w, lane);
          wave_sync();
          if (c + i + kDepth < c1) ask(i, c + i + kDepth);
        }
    };
    if (rows == 1) take(std::integral_constant<int, 1>{});
    else if (!MORE || rows == 2) take(std::integral_constant<int, 2>{});
    else if constexpr (MORE) take(std::integral_constant<int, kMostRows>{});

    // The wavefronts' sums meet, in their order.
    __syncthreads();
#pragma unroll
    for (int m = 0; m < kMats; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) meet[((wave * kMats + m) * kTile + lane / kTile * 4 + r) * kTile + lane % kTile] = acc[m][r];
    __syncthreads();
    // 32 threads a row, their outputs side by side.
    const int row = threadIdx.x / 32, col = threadIdx.x % 32, o = pair * 32 + col;
    const int to = __shfl(row_slot, min(row, rows - 1), 64);
    if (row < rows) {
      float v[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kWaves; ++i)
#pragma unroll
        for (int m = 0; m < kMats / 2; ++m) v[m] += meet[((i * kMats + 2 * m + col / kTile) * kTile + row) * kTile + col % kTile];
      if constexpr (GATED) {
        const float h = o < p.out ? silu(v[0]) * v[1] : 0.0f;
        const Factor f(max_of_half(finite_bits(h)));
        _Float16 high, low;
        two_parts(h * f.up, high, low);
        const std::size_t block = static_cast<std::size_t>(to) * p.h.blocks + pair;
        p.h.values[block * 64 + col] = high;
        p.h.values[block * 64 + 32 + col] = low;
        if (col == 0) p.h.factors[block] = f.back;
        // Blocks up to a whole chunk, which the second product reads, are 0.
        if (pair == p.pairs - 1)
          for (std::size_t i = 1; pair + i < static_cast<std::size_t>(p.h.blocks); ++i) {
            reinterpret_cast<std::uint32_t*>(p.h.values)[(block + i) * 32 + col] = 0;
            if (col == 0) p.h.factors[block + i] = 0.0f;
          }
      } else if (o < p.out) {
        p.y[static_cast<std::size_t>(to) * p.y_stride + o] = v[0];
      }
    }
    __syncthreads();
  }
}

// ------------------------------------ the second product and a token's sum

constexpr int kSumWaves = 16, kSumThreads = kSumWaves * 64;
// Of each block of a chunk 16 bytes: the factors of both rows, then what the
// tokens weigh the expert with.
constexpr int kSumRows = 4, kSumFactorBytes = 4 * kSumRows * 4;

struct SumArgs {
  Matrices m;
  const std::int32_t* ids;
  const float *weights, *residual;
  FewParts h;
  float* y;  // or partial sums [split][token][out], without the residual
  std::size_t r_stride, y_stride, split_stride;
  int tokens, top_k, experts, out, tiles, steps, chunks, splits;
};

// One workgroup a tile of 16 outputs (or, where the tiles are too few for the
// chip, a part of its inputs), for both tokens: its wavefronts share the
// chunks of all chosen experts.  Row m of a product is token m, with the
// weight that it gives the expert (0 where it has not chosen it), so the sums
// over inputs and over experts are one.
template <int TYPE, int ROWS>
__global__ void __launch_bounds__(kSumThreads) few_sum_kernel(SumArgs p) {
  static_assert(ROWS <= static_cast<int>(kFewTokens) && kFewTokens == 2);
  extern __shared__ __attribute__((aligned(16))) std::uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % p.tiles, split = blockIdx.x / p.tiles, slots = p.tokens * p.top_k;
  const std::int32_t mine = lane < slots ? p.ids[lane] : -1;
  const float weight = lane < slots ? p.weights[lane] : 0.0f;
  // Bit s: slot s is the first of its expert.
  std::uint64_t firsts = 0;
  for (int s = 0; s < slots; ++s) {
    const int e = __builtin_amdgcn_readlane(mine, s);
    if (e >= 0 && e < p.experts && __builtin_ctzll(__ballot(mine == e)) == s) firsts |= std::uint64_t{1} << s;
  }
  // Units (expert, chunk), in equal shares of the splits and their wavefronts.
  const int units = __builtin_popcountll(firsts) * p.chunks, sharers = p.splits * kSumWaves;
  const int each = (units + sharers - 1) / sharers;
  const int u0 = min((split * kSumWaves + wave) * each, units), u1 = min(u0 + each, units);
  // This wavefront's rows of a chunk, and their factors and weights [block][kSumRows].
  std::uint8_t* const rows_at = lds + wave * (2 * kRowBytes + kSumFactorBytes);
  float* const factors_at = reinterpret_cast<float*>(rows_at + 2 * kRowBytes);
  float* const meet = reinterpret_cast<float*>(lds);
  LaneAt lane_at(lane);
  constexpr int kDepth = TYPE == LLMI_TYPE_Q4_0 ? 4 : 3;
  f32x4 acc = {};
  Weights<TYPE> ring[kDepth][2];
  u32x4 x[kDepth];
  float factor[kDepth], times[kDepth];
  bool live[kDepth];
  // The unit that is asked for next: its number and chunk, its expert (the
  // lowest bit that is left) and this lane's row of it: for the values row
  // lane / 32, 16 bytes of each chunk's 512; for the factors row lane / 4, one
  // of a chunk's four.
  std::uint64_t left = firsts;
  for (int i = u0 / p.chunks; i > 0 && left != 0; --i) left &= left - 1;
  int next = u0, chunk = u0 % p.chunks;
  GlobalBytes w_at = nullptr;
  const _Float16* row = nullptr;
  const float* factor_row = nullptr;
  float row_times = 0.0f;
  bool row_live = false;
  const auto enter = [&] {
    const int s = __builtin_ctzll(left), e = __builtin_amdgcn_readlane(mine, s);
    const std::uint64_t same = __ballot(mine == e);
    w_at = tile_at<TYPE>(p.m, static_cast<std::size_t>(e) * p.tiles + tile, p.steps);
    // The token's slots of this expert, as bits from its first slot on.
    const auto chosen = [&](int t) {
      const std::uint64_t bits = same >> (t * p.top_k);
      return p.top_k < 64 ? bits & ((std::uint64_t{1} << p.top_k) - 1) : bits;
    };
    const auto slot_of = [&](int t, std::uint64_t bits) { return bits != 0 ? t * p.top_k + __builtin_ctzll(bits) : s; };
    const int tv = min(lane / 32, p.tokens - 1), tf = min(min(lane / 4, 1), p.tokens - 1);
    std::uint64_t bits = chosen(tv);
    row_live = bits != 0;
    row = p.h.values + (static_cast<std::size_t>(slot_of(tv, bits)) * p.h.blocks + chunk * 4) * 64 + lane % 32 * 8;
    bits = chosen(tf);
    factor_row = p.h.factors + static_cast<std::size_t>(slot_of(tf, bits)) * p.h.blocks + chunk * 4 + lane % 4;
    row_times = 0.0f;  // of a token that has not chosen it
    while (__any(bits != 0)) {  // an expert chosen twice counts with both weights
      const float one = __shfl(weight, bits != 0 ? slot_of(tf, bits) : 0, 64);
      if (bits != 0) row_times += one;
      bits &= bits - 1;
    }
  };
  if (u0 < u1) enter();
  const auto ask = [&](int i) {
#pragma unroll
    for (int t = 0; t < 2; ++t) ring[i][t].load(w_at, min(2 * chunk + t, p.steps - 1), lane_at);
    x[i] = *reinterpret_cast<const u32x4*>(row);
    live[i] = row_live;
    row += 4 * 64;
    factor[i] = *factor_row;
    times[i] = row_times;
    factor_row += 4;
    if (++next < u1 && ++chunk == p.chunks) {
      chunk = 0;
      left &= left - 1;
      enter();
    }
  };
#pragma unroll
  for (int i = 0; i < kDepth; ++i)
    if (next < u1) ask(i);
  for (int u = u0; u < u1; u += kDepth)
#pragma unroll
    for (int i = 0; i < kDepth; ++i) {
      if (u + i >= u1) break;
      // A row that does not count is 0, whatever stands there.
      *reinterpret_cast<u32x4*>(rows_at + lane / 32 * kRowBytes + lane % 32 * 16) = ROWS == 1 || live[i] ? x[i] : u32x4{0, 0, 0, 0};
      if (lane / 4 < 2) {
        factors_at[lane % 4 * kSumRows + lane / 4] = factor[i];
        factors_at[lane % 4 * kSumRows + 2 + lane / 4] = times[i];
      }
      wave_sync();
      const std::uint8_t* const from = lane_row<ROWS>(rows_at, lane);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 d = times_codes(from, b, ring[i][b / 2].codes(b % 2));
        const f32x4 f = *reinterpret_cast<const f32x4*>(factors_at + b * kSumRows);
#pragma unroll
        for (int r = 0; r < ROWS; ++r)  // the power of two last: with the weight it may lie below the normal numbers
          acc[r] = __builtin_fmaf(d[r] * ring[i][b / 2].s[b % 2] * f[2 + r], f[r], acc[r]);
      }
      wave_sync();
      if (next < u1) ask(i);
    }
  // Lanes 0 .. 15 hold the rows that count.
  __syncthreads();
  if (lane < kTile) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) meet[(wave * ROWS + r) * kTile + lane] = acc[r];
  }
  __syncthreads();
  const int t = threadIdx.x / kTile, o = tile * kTile + threadIdx.x % kTile;
  if (t < p.tokens && o < p.out) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kSumWaves; ++i) v += meet[(i * ROWS + t) * kTile + threadIdx.x % kTile];
    if (p.residual != nullptr) v = p.residual[static_cast<std::size_t>(t) * p.r_stride + o] + v;
    p.y[static_cast<std::size_t>(split) * p.split_stride + static_cast<std::size_t>(t) * p.y_stride + o] = v;
  }
}

// y = residual + the sum of the splits, in their order.
__global__ void __launch_bounds__(256) few_join_kernel(const float* __restrict__ parts, int splits, int tokens, int out,
                                                       const float* residual, std::size_t r_stride, float* y,
                                                       std::size_t y_stride) {
  const int u = blockIdx.x * 256 + threadIdx.x, t = u / out, o = u % out;
  if (t >= tokens) return;
  float v = 0.0f;
  for (int i = 0; i < splits; ++i) v += parts[(static_cast<std::size_t>(i) * tokens + t) * out + o];
  if (residual != nullptr) v = residual[static_cast<std::size_t>(t) * r_stride + o] + v;
  y[static_cast<std::size_t>(t) * y_stride + o] = v;
}

// fn of each flag as a std::bool_constant.
template <typename Fn>
void with_flags(Fn&& fn) {
  fn();
}
template <typename Fn, typename... More>
void with_flags(Fn&& fn, bool flag, More... more) {
  if (flag) with_flags([&](auto... rest) { fn(std::true_type{}, rest...); }, more...);
  else with_flags([&](auto... rest) { fn(std::false_type{}, rest...); }, more...);
}

// LDS of a workgroup: its wavefronts' rows, then their sums of MATS tiles.
std::size_t lds_bytes(int waves, int rows, int extra, int mats) {
  return std::max<std::size_t>(static_cast<std::size_t>(waves) * (rows * kRowBytes + extra),
                               static_cast<std::size_t>(waves) * mats * kTile * kTile * sizeof(float));
}

}  // namespace

int launch_few(const FewProduct& f, hipStream_t s) {
  const Shape& sh = f.shape;
  // An expert has more than two rows only where x has, or where ids repeat.
  const bool more = ceil_div(f.slots, f.per_row) > 2;
  const int rows = more ? kMostRows : 2;
  const std::size_t pairs = ceil_div(sh.tiles(), 2);
  const FewArgs a{f.m, f.up, f.ids, f.x, f.y, f.h, f.x_stride, f.y_stride, static_cast<int>(f.slots), static_cast<int>(f.per_row),
                  static_cast<int>(sh.count), static_cast<int>(sh.out), static_cast<int>(sh.in), static_cast<int>(sh.tiles()),
                  static_cast<int>(pairs), static_cast<int>(sh.steps()), static_cast<int>(ceil_div(sh.steps(), 2)), rows};
  const unsigned grid = static_cast<unsigned>(f.slots * pairs);
  const bool gated = f.up.steps != nullptr;
  LLMI_REQUIRE(!gated || !more, "moe: too many rows of x for a gated pair");
  with_flags([&](auto gate, auto many, auto quads) {
    if constexpr (!(gate && many)) {
      const std::size_t lds = lds_bytes(kWaves, rows, 64, gate ? 4 : 2);
      if (sh.type == LLMI_TYPE_Q4_0) few_kernel<LLMI_TYPE_Q4_0, gate, many, quads><<<grid, kThreads, lds, s>>>(a);
      else few_kernel<LLMI_TYPE_Q8_0, gate, many, quads><<<grid, kThreads, lds, s>>>(a);
    }
  }, gated, more, sh.in % 4 == 0);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

int launch_few_sum(const FewSum& f, hipStream_t s) {
  const Shape& sh = f.shape;
  const std::size_t splits = few_splits(sh);
  const bool joined = splits > 1;
  const SumArgs a{f.m, f.ids, f.weights, joined ? nullptr : f.residual, f.h, joined ? f.parts : f.y, f.r_stride,
                  joined ? sh.out : f.y_stride, f.tokens * sh.out, static_cast<int>(f.tokens), static_cast<int>(f.top_k),
                  static_cast<int>(sh.count), static_cast<int>(sh.out), static_cast<int>(sh.tiles()),
                  static_cast<int>(sh.steps()), static_cast<int>(ceil_div(sh.steps(), 2)), static_cast<int>(splits)};
  const unsigned grid = static_cast<unsigned>(sh.tiles() * splits);
  constexpr std::size_t lds = kSumWaves * (2 * kRowBytes + kSumFactorBytes);  // the sums that meet in it take less
  const auto run = [&](auto count) {
    if (sh.type == LLMI_TYPE_Q4_0) few_sum_kernel<LLMI_TYPE_Q4_0, count><<<grid, kSumThreads, lds, s>>>(a);
    else few_sum_kernel<LLMI_TYPE_Q8_0, count><<<grid, kSumThreads, lds, s>>>(a);
  };
  if (f.tokens == 1) run(std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, 2>{});
  LLMI_TRY_HIP(hipGetLastError());
  if (joined) {
    few_join_kernel<<<static_cast<unsigned>(ceil_div(f.tokens * sh.out, 256)), 256, 0, s>>>(
        f.parts, static_cast<int>(splits), static_cast<int>(f.tokens), static_cast<int>(sh.out), f.residual, f.r_stride, f.y,
        f.y_stride);
    LLMI_TRY_HIP(hipGetLastError());
  }
  return LLMI_OK;
}

}  // namespace llmi_hip::moe
