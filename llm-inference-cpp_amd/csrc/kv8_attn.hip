// Attention over the paged 8-bit key/value cache (llmi_hip_kv8_attention_dev).
#include "kv8.hpp"

namespace llmi_hip::kv8 {
namespace {

constexpr int kThreads = 256, kWaves = 4;

struct AttnArgs {
  View v;
  Geometry g;
  const std::int8_t *k, *val;
  const float* scales;
  const float* q;
  float* out;
  float* parts;  // rows of partial states: o (dim floats each), then (maximum, sum) each
  std::size_t q_stride, out_stride, part_states;  // part_states: float offset of the (maximum, sum) pairs
  float scale;
  int nfew, nmany, njoin;  // -1: from v.counts (a captured launch)
};

// ------------------------------------------------------------- few rows
// Single tokens and drafts: up to 16 rows (tokens x query heads of one
// key/value head) against a range of positions; HBM-bound, so the codes are
// read once, 16 bytes a lane, and go to the matrix cores as they are (8-bit
// products, exact in 32 bits).  For that the fp32 side is put into four signed
// base-256 digits: X = round(x * 2^(30 - e)), X = sum_i 2^(8i) D_i, one matrix
// row per digit, so that row 4h + i of a product is head h's digit i and a
// lane finds the four digits' sums of one head in its four accumulators.
//   scores   S[head][position] = Q K^T   A = digits of q, B = key codes
//   output   O[head][dim]      = W V     A = digits of w, B = value codes
// with w = p * (value scale / the tile's largest) in [0, 1], p the weight
// against the running maximum.  A wavefront takes tiles of 64 positions = 4
// blocks; a workgroup's four wavefronts take a range's tiles in turn and merge.
typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any float

// Maximum over the 16 lanes of a row of lanes, in every lane.
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false)));  // row_ror:8
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xF, 0xF, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xF, 0xF, false)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xF, 0xF, false)));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xF, 0xF, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xF, 0xF, false));
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xF, 0xF, false));
}
// The four signed digits of X (|X| <= 2^30), lowest in the lowest byte.
__device__ __forceinline__ std::uint32_t digits(int x) {
  return (static_cast<std::uint32_t>(x) + 0x00808080u) ^ 0x00808080u;
}
// sum_i 2^(8i) s[i]
__device__ __forceinline__ float undigit(i4 s) {
  float x = static_cast<float>(s[3]);
  x = fmaf(x, 256.0f, static_cast<float>(s[2]));
  x = fmaf(x, 256.0f, static_cast<float>(s[1]));
  return fmaf(x, 256.0f, static_cast<float>(s[0]));
}

// HD: head_dim; MT: tiles of 4 rows (16 digit rows).
template <int HD, int MT>
__global__ void __launch_bounds__(kThreads) attention_few(AttnArgs A) {
  constexpr int kG = HD / 16;            // 16-dim groups of a block
  constexpr int kC = (HD + 63) / 64;     // 64-dim steps of a score product
  constexpr int kRows = 4 * MT;
  constexpr float kLog2e = 1.44269504088896340736f;
  __shared__ union {
    std::uint32_t w[kWaves][4][4][16];   // a tile's weight digits: [block][head of the 4][position]
    float o[kWaves][kRows][HD];          // the wavefronts' outputs, merged at the end
  } sh;
  __shared__ float sh_m[kWaves][kRows], sh_l[kWaves][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo16 = lane & 15, grp = lane >> 4;
  const int nfew = A.nfew >= 0 ? A.nfew : A.v.counts->few;
  const int units = nfew * A.g.kv_heads;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = u / A.g.kv_heads, h = u - item * A.g.kv_heads;
    const FewItem it = A.v.few[item];
    if ((it.rows + 3) / 4 > MT || (MT > 1 && (it.rows + 3) / 4 <= MT / 2)) continue;  // another instance's
    const Seq s = A.v.seqs[it.seq];

    // The digits of q: lane (digit row lo16, dims 16 grp ..) of each 64-dim step.
    i4 qd[MT][kC];
    float m[MT], l[MT], o[MT][kG];
    int qe[MT];  // this lane's score row (head grp of the tile): its exponent
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = 4 * mt + lo16 / 4;
      const bool live = r < it.rows;
      const int row = it.row0 + (live ? r : 0), tok = row / A.g.group;
      const float* qp = A.q + static_cast<std::size_t>(s.row + tok) * A.q_stride +
                        static_cast<std::size_t>(h * A.g.group + (row - tok * A.g.group)) * HD;
      float x[kC][16];
      float top = 0.0f;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const int g = 4 * c + grp;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[c][i] = live && g < kG ? qp[g * 16 + i] : 0.0f;
          top = fmaxf(top, fabsf(x[c][i]));
          bad |= !(fabsf(x[c][i]) < INFINITY);
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      bad = bad || __shfl_xor(bad, 16, 64);
      bad = bad || __shfl_xor(bad, 32, 64);
      int e;
      (void)frexpf(top, &e);  // top < 2^e
      if (bad || !(top > 0.0f)) e = 0;
#pragma unroll
      for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          std::uint32_t d = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int X = bad ? 0 : static_cast<int>(rintf(ldexpf(x[c][4 * j + i], 30 - e)));
            d |= ((digits(X) >> (8 * (lo16 & 3))) & 0xFFu) << (8 * i);
          }
          qd[mt][c][j] = static_cast<int>(d);
        }
      // Lanes 4 hd .. of any group hold head hd's; an inf or NaN in q makes the row's sum NaN.
      qe[mt] = __shfl(e - 30, 4 * grp, 64);
      l[mt] = __shfl(static_cast<int>(bad), 4 * grp, 64) != 0 ? __builtin_nanf("") : 0.0f;
    }

    int limit[MT];  // last position that this lane's row sees, -1 for rows of nobody
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = 4 * mt + grp;
      limit[mt] = r < it.rows ? s.start + (it.row0 + r) / A.g.group : -1;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt] = -INFINITY;
#pragma unroll
      for (int g = 0; g < kG; ++g) o[mt][g] = 0.0f;
    }

    const int last_block = (it.hi - 1) / kBlk;
    for (int base = it.lo + wave * kTile; base < it.hi; base += kWaves * kTile) {
      // This lane's block of the tile; behind the range, the last one again
      // (its positions there are masked), with scales of 0.
      const int block = base / kBlk + grp;
      const std::size_t at = block_index(A.g, A.v.table, s, min(block, last_block), h);
      float2 sc = reinterpret_cast<const float2*>(A.scales)[at];
      if (block > last_block) sc = make_float2(0.0f, 0.0f);
      const std::int8_t* kp = A.k + at * (16 * HD);
      const std::int8_t* vp = A.val + at * (16 * HD) + lo16 * 16;
      // Keys: every lane needs all four blocks, position lo16, dims 16 (4c + grp) ...
      i4 kf[4][kC];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const std::uint64_t p = reinterpret_cast<std::uint64_t>(kp);
        const std::uint32_t plo = __builtin_amdgcn_readlane(static_cast<int>(p), 16 * b);
        const std::uint32_t phi = __builtin_amdgcn_readlane(static_cast<int>(p >> 32), 16 * b);
        const auto* src = reinterpret_cast<const std::int8_t*>((static_cast<std::uint64_t>(phi) << 32) | plo);
#pragma unroll
        for (int c = 0; c < kC; ++c)
          kf[b][c] = *reinterpret_cast<const i4*>(src + min(4 * c + grp, kG - 1) * 256 + lo16 * 16);
      }
      i4 vf[kG];
#pragma unroll
      for (int g = 0; g < kG; ++g) vf[g] = *reinterpret_cast<const i4*>(vp + g * 256);

      float ks[4], vs[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        ks[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc.x), 16 * b));
        vs[b] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc.y), 16 * b));
      }
      // The tile's largest finite value scale; 2^-96 keeps 2^30 / top finite.
      float vf_s[4], top = 0x1p-96f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        vf_s[b] = vs[b] < INFINITY ? vs[b] : 0.0f;
        top = fmaxf(top, vf_s[b]);
      }
      const float to_fix = 0x1p30f / top;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float x[4];
        float mx = m[mt];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          i4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < kC; ++c) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qd[mt][c], kf[b][c], acc, 0, 0, 0);
          x[b] = undigit(acc) * ldexpf(A.scale * kLog2e * ks[b], qe[mt]);
          if (base + b * kBlk + lo16 > limit[mt]) x[b] = -INFINITY;
          mx = fmaxf(mx, x[b]);
        }
        mx = row16_max(mx);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float keep = exp2f(m[mt] - ref);
        m[mt] = mx;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bool seen = base + b * kBlk + lo16 <= limit[mt];
          const float p = exp2f(x[b] - ref);
          // A value scale that is inf or NaN shows in the sum of the rows that see the block.
          if (seen) sum += fmaf(vs[b], 0.0f, p);
          const int w = static_cast<int>(rintf(p * (vf_s[b] * to_fix)));
          sh.w[wave][b][grp][lo16] = digits(w);
        }
        l[mt] = fmaf(l[mt], keep, sum);
        __builtin_amdgcn_wave_barrier();
        // Digit row lo16 (head lo16 / 4, digit lo16 % 4) over this lane group's block.
        i4 wd;
        const std::uint32_t pick = 0x01010101u * (lo16 & 3);
        const auto* src = reinterpret_cast<const uint4*>(&sh.w[wave][grp][lo16 / 4][0]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 d = src[j];
          // Bytes 0-3 of the selector's numbering are the second operand's, 4-7 the first's.
          const std::uint32_t a = __builtin_amdgcn_perm(d.y, d.x, (pick & 0xFFu) | (((pick & 0xFFu) + 4u) << 8));
          const std::uint32_t b2 = __builtin_amdgcn_perm(d.w, d.z, (pick & 0xFFu) | (((pick & 0xFFu) + 4u) << 8));
          wd[j] = static_cast<int>(__builtin_amdgcn_perm(b2, a, 0x05040100u));
        }
        __builtin_amdgcn_wave_barrier();
        const float from_fix = top * 0x1p-30f;
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          i4 acc = {0, 0, 0, 0};
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wd, vf[g], acc, 0, 0, 0);
          o[mt][g] = fmaf(o[mt][g], keep, undigit(acc) * from_fix);
        }
      }
    }

    // Merge the four wavefronts: lane (dim lo16 of each group, head grp).
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const float ls = row16_sum(l[mt]);
      if (lo16 == 0) {
        sh_m[wave][4 * mt + grp] = m[mt];
        sh_l[wave][4 * mt + grp] = ls;
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) sh.o[wave][4 * mt + grp][16 * g + lo16] = o[mt][g];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < it.rows * HD; e += kThreads) {
      const int r = e / HD, d = e - r * HD;
      float top = sh_m[0][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sh_m[w][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, acc = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = exp2f(sh_m[w][r] - ref);
        sum = fmaf(sh_l[w][r], f, sum);
        acc = fmaf(sh.o[w][r][d], f, acc);
      }
      if (it.part >= 0) {
        const std::size_t slot = (static_cast<std::size_t>(it.part) * A.g.kv_heads + h) * kFewRows + r;
        A.parts[slot * HD + d] = acc;
        if (d == 0) *reinterpret_cast<float2*>(A.parts + A.part_states + 2 * slot) = make_float2(top, sum);
      } else {
        const int row = it.row0 + r, tok = row / A.g.group;
        A.out[static_cast<std::size_t>(s.row + tok) * A.out_stride +
              static_cast<std::size_t>(h * A.g.group + (row - tok * A.g.group)) * HD + d] = acc / sum;
      }
    }
    __syncthreads();
  }
}

// Joins the partial states of split rows: one workgroup per row group, head
// and row, in the splits' order.
__global__ void __launch_bounds__(kThreads) attention_join(AttnArgs A) {
  __shared__ float sh_o[kThreads], sh_l[kThreads];
  const int njoin = A.njoin >= 0 ? A.njoin : A.v.counts->join;
  const int dim = A.g.dim;
  const long units = static_cast<long>(njoin) * A.g.kv_heads * kFewRows;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const int r = static_cast<int>(u % kFewRows);
    const int h = static_cast<int>(u / kFewRows % A.g.kv_heads);
    const JoinItem it = A.v.join[u / kFewRows / A.g.kv_heads];
    if (r >= it.rows) continue;
    const auto slot = [&](int c) {
      return (static_cast<std::size_t>(it.part + c * it.step) * A.g.kv_heads + h * it.step) * kFewRows + it.off + r;
    };
    const auto state = [&](int c) { return *reinterpret_cast<const float2*>(A.parts + A.part_states + 2 * slot(c)); };
    float top = -INFINITY;
    for (int c = threadIdx.x & 63; c < it.n; c += 64) top = fmaxf(top, state(c).x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float ref = top == -INFINITY ? 0.0f : top;
    // 64 dims at a time, a quarter of the splits to each wavefront.
    const Seq s = A.v.seqs[it.seq];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int d0 = 0; d0 < dim; d0 += 64) {
      const int d = d0 + lane;
      float sum = 0.0f, acc = 0.0f;
      for (int c = wave; c < it.n; c += kWaves) {
        const float2 ml = state(c);
        const float f = exp2f(ml.x - ref);
        sum = fmaf(ml.y, f, sum);
        if (d < dim) acc = fmaf(A.parts[slot(c) * dim + d], f, acc);
      }
      sh_o[threadIdx.x] = acc;
      sh_l[threadIdx.x] = sum;
      __syncthreads();
      if (wave == 0 && d < dim) {
        for (int w = 1; w < kWaves; ++w) {
          acc += sh_o[64 * w + lane];
          sum += sh_l[64 * w + lane];
        }
        const int row = it.row0 + r, tok = row / A.g.group;
        A.out[static_cast<std::size_t>(s.row + tok) * A.out_stride +
              static_cast<std::size_t>(h * A.g.group + (row - tok * A.g.group)) * dim + d] = acc / sum;
      }
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------ many rows
// Prompts and chunks: 128 rows (tokens x query heads of one key/value head) a
// workgroup, 32 a wavefront, on the 16-bit matrix instructions.  The codes are
// exact in fp16; the fp32 side enters as two fp16 parts (22 bits):
//   S^T[position][row] = K Q^T   A = codes of 32 positions, B = q * 2^s, two parts
//   O^T[dim][row]      = V^T W^T A = codes of 32 dims, B = w, two parts
// A row is a column of both, so its maximum, sum and rescaling are one lane's
// (and its partner's 32 lanes on), and the weights go from the first product's
// accumulators to the second's operand without leaving the registers: a lane
// holds positions 4h .. 4h+3 and 8+4h .. of each 16 (h = lane / 32), and the
// value tile is staged in that order.
// w = p * (value scale / the largest so far) * 2^kWeightBits: block scales
// differ along the sum, so they ride on the weights.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kWeightBits = 14;

// The four signed bytes of w as fp16, exact: 1024 + (byte + 128) is an fp16
// whose low byte is the code plus 128.
__device__ __forceinline__ void halves(std::uint32_t w, std::uint32_t* out) {
  const std::uint32_t u = w ^ 0x80808080u;
  const h2 bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
  const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u));
  const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u));
  out[0] = __builtin_bit_cast(std::uint32_t, static_cast<h2>(a - bias));
  out[1] = __builtin_bit_cast(std::uint32_t, static_cast<h2>(b - bias));
}

template <int HD>
__global__ void __launch_bounds__(kThreads, HD <= 128 ? 2 : 1) attention_many(AttnArgs A) {
  constexpr int kG = HD / 16;
  constexpr int kChunks = 4 * HD;  // 16-byte pieces of a tile's keys (and of its values)
  constexpr int kPer = (kChunks + kThreads - 1) / kThreads;
  constexpr float kLog2e = 1.44269504088896340736f;
  __shared__ uint4 sh_k[2][kG][2][kTile];     // [16-dim group][half of it][position]: 8 fp16
  __shared__ uint4 sh_v[2][kTile / 16][2][HD];  // [block][h][dim]: positions 4h.., 8 + 4h..
  __shared__ float2 sh_s[2][4];
  const int lane = threadIdx.x & 63, col = lane & 31, h2nd = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nmany = A.nmany >= 0 ? A.nmany : A.v.counts->many;
  const int units = nmany * A.g.kv_heads;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = u / A.g.kv_heads, head = u - item * A.g.kv_heads;
    const ManyItem it = A.v.many[item];
    const Seq s = A.v.seqs[it.seq];
    const int r = wave * 32 + col;
    const bool live = r < it.rows;
    const int row = it.row0 + (live ? r : 0), tok = row / A.g.group;
    const int limit = live ? s.start + tok : -1;
    const std::size_t head_off = static_cast<std::size_t>(head * A.g.group + (row - tok * A.g.group)) * HD;

    // q * 2^qs, its largest below 2^14, as two fp16 parts.
    h8 qh[kG], ql[kG];
    int qs;
    {
      const float* qp = A.q + static_cast<std::size_t>(s.row + tok) * A.q_stride + head_off;
      float x[kG][8], top = 0.0f;
#pragma unroll
      for (int g = 0; g < kG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[g][i] = live ? qp[16 * g + 8 * h2nd + i] : 0.0f;
          top = fmaxf(top, fabsf(x[g][i]));
        }
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      int e = 0;
      (void)frexpf(top, &e);
      if (!(top > 0.0f && top < INFINITY)) e = 0;
      qs = 14 - e;
#pragma unroll
      for (int g = 0; g < kG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = ldexpf(x[g][i], qs);
          qh[g][i] = static_cast<_Float16>(y);
          ql[g][i] = static_cast<_Float16>(y - static_cast<float>(qh[g][i]));
        }
    }
    // The wavefront's rows see at most up to `reach`, and all of them up to `all`.
    int reach = limit, all = live ? limit : 0x7FFFFFFF;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      reach = max(reach, __shfl_xor(reach, o, 64));
      all = min(all, __shfl_xor(all, o, 64));
    }
    reach = __builtin_amdgcn_readfirstlane(reach);
    all = __builtin_amdgcn_readfirstlane(all);

    f16v o[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f, vtop = 0x1p-96f;

    const int last_block = (it.hi - 1) / kBlk;
    uint4 kreg[kPer], vreg[kPer];
    float2 sreg = make_float2(0.0f, 0.0f);
    const auto fetch = [&](int base) {
#pragma unroll
      for (int n = 0; n < kPer; ++n) {
        const int c = n * kThreads + threadIdx.x;
        if (kChunks % kThreads != 0 && c >= kChunks) break;
        const int b = c / HD, at_chunk = c - b * HD;
        const std::size_t at = block_index(A.g, A.v.table, s, min(base / kBlk + b, last_block), head);
        kreg[n] = reinterpret_cast<const uint4*>(A.k + at * (16 * HD))[at_chunk];
        vreg[n] = reinterpret_cast<const uint4*>(A.val + at * (16 * HD))[at_chunk];
      }
      if (threadIdx.x < 4) {
        const int b = base / kBlk + static_cast<int>(threadIdx.x);
        sreg = make_float2(0.0f, 0.0f);
        if (b <= last_block)
          sreg = reinterpret_cast<const float2*>(A.scales)[block_index(A.g, A.v.table, s, b, head)];
      }
    };
    const auto stage = [&](int buf) {
#pragma unroll
      for (int n = 0; n < kPer; ++n) {
        const int c = n * kThreads + threadIdx.x;
        if (kChunks % kThreads != 0 && c >= kChunks) break;
        const int b = c / HD, at_chunk = c - b * HD;
        std::uint32_t x[8];
        halves(kreg[n].x, x);
        halves(kreg[n].y, x + 2);
        halves(kreg[n].z, x + 4);
        halves(kreg[n].w, x + 6);
        const int g = at_chunk / 16, p = b * 16 + at_chunk % 16;
        sh_k[buf][g][0][p] = make_uint4(x[0], x[1], x[2], x[3]);
        sh_k[buf][g][1][p] = make_uint4(x[4], x[5], x[6], x[7]);
        halves(vreg[n].x, x);
        halves(vreg[n].y, x + 2);
        halves(vreg[n].z, x + 4);
        halves(vreg[n].w, x + 6);
        sh_v[buf][b][0][at_chunk] = make_uint4(x[0], x[1], x[4], x[5]);
        sh_v[buf][b][1][at_chunk] = make_uint4(x[2], x[3], x[6], x[7]);
      }
      if (threadIdx.x < 4) sh_s[buf][threadIdx.x] = sreg;
    };

    fetch(it.lo);
    stage(0);
    __syncthreads();
    int buf = 0;
    for (int base = it.lo; base < it.hi; base += kTile, buf ^= 1) {
      const bool more = base + kTile < it.hi;
      if (more) fetch(base + kTile);
      if (base <= reach) {
        f16v st[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) st[t][i] = 0.0f;
#pragma unroll
          for (int g = 0; g < kG; ++g) {
            const h8 a = __builtin_bit_cast(h8, sh_k[buf][g][h2nd][32 * t + col]);
            st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[g], st[t], 0, 0, 0);
            st[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[g], st[t], 0, 0, 0);
          }
        }
        // Scores in base-2 units; positions behind a row's own leave nothing.
        float2 sc[4];
        float vf[4], tile_top = vtop;
        bool whole = true;  // every value scale of the tile is finite
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          sc[b] = sh_s[buf][b];
          const bool fin = sc[b].y < INFINITY;
          whole = whole && fin;
          vf[b] = fin ? sc[b].y : 0.0f;
          tile_top = fmaxf(tile_top, vf[b]);
        }
        float mx = m;
        const bool edge = base + kTile - 1 > all;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float f = ldexpf(A.scale * kLog2e * sc[b].x, -qs);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float x = st[b / 2][8 * (b & 1) + i] * f;
            if (edge && base + 16 * b + 8 * (i / 4) + 4 * h2nd + i % 4 > limit) x = -INFINITY;
            st[b / 2][8 * (b & 1) + i] = x;
            mx = fmaxf(mx, x);
          }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float keep = exp2f(m - ref);
        const float rescale = keep * (vtop / tile_top);
        m = mx;
        vtop = tile_top;
        if (__any(rescale != 1.0f)) {
#pragma unroll
          for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= rescale;
        }
        const float to_w = ldexpf(1.0f, kWeightBits) / tile_top;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float fw = vf[b] * to_w;
          h8 wh, wl;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p = exp2f(st[b / 2][8 * (b & 1) + i] - ref);
            sum += p;
            const float w = p * fw;
            wh[i] = static_cast<_Float16>(w);
            wl[i] = static_cast<_Float16>(w - static_cast<float>(wh[i]));
          }
#pragma unroll
          for (int d = 0; d < HD / 32; ++d) {
            const h8 a = __builtin_bit_cast(h8, sh_v[buf][b][h2nd][32 * d + col]);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, wh, o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, wl, o[d], 0, 0, 0);
          }
        }
        if (!whole) {
          // A value scale that is inf or NaN shows in the rows that see a position of its block.
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (base + 16 * b <= limit) sum = fmaf(sc[b].y, 0.0f, sum);
        }
        l = fmaf(l, keep, sum);
      }
      if (more) stage(buf ^ 1);
      __syncthreads();
    }

    l += __shfl_xor(l, 32, 64);
    const float unit = vtop * ldexpf(1.0f, -kWeightBits);
    if (live) {
      float* dst;
      float f;
      if (it.part >= 0) {
        const std::size_t slot =
            (static_cast<std::size_t>(it.part) * A.g.kv_heads + head * kManySlots) * kFewRows + r;
        dst = A.parts + slot * HD;
        f = unit;
        if (h2nd == 0) *reinterpret_cast<float2*>(A.parts + A.part_states + 2 * slot) = make_float2(m, l);
      } else {
        dst = A.out + static_cast<std::size_t>(s.row + tok) * A.out_stride + head_off;
        f = unit / l;
      }
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f4*>(dst + 32 * d + 8 * i + 4 * h2nd) =
              f4{o[d][4 * i] * f, o[d][4 * i + 1] * f, o[d][4 * i + 2] * f, o[d][4 * i + 3] * f};
    }
  }
}

template <int HD>
void launch_few(const AttnArgs& a, unsigned grid, unsigned sizes, hipStream_t s) {
  if (sizes & 1) attention_few<HD, 1><<<grid, kThreads, 0, s>>>(a);
  if (sizes & 2) attention_few<HD, 2><<<grid, kThreads, 0, s>>>(a);
  if (sizes & 4) attention_few<HD, 4><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

int launch_attention(const llmi_hip_kv8_plan* p, const llmi_kv8_layer& layer, const float* q, std::size_t q_stride,
                     float scale, float* out, std::size_t out_stride, hipStream_t s, bool captured) {
  const Lists& l = p->lists;
  AttnArgs a{p->view(), p->g, layer.k, layer.v, layer.scales, q, out, p->parts, q_stride, out_stride,
             p->max_parts * p->g.kv_heads * kFewRows * p->g.dim, scale,
             captured ? -1 : static_cast<int>(l.few.size()), captured ? -1 : static_cast<int>(l.many.size()),
             captured ? -1 : static_cast<int>(l.join.size())};
  const std::size_t heads = static_cast<std::size_t>(p->g.kv_heads);
  const auto grid = [](std::size_t units) {
    return static_cast<unsigned>(std::min<std::size_t>(std::max<std::size_t>(units, 1), 1u << 20));
  };
  unsigned sizes = captured ? 7 : 0;  // which tile counts the batch has
  for (const FewItem& it : l.few) sizes |= it.rows <= 4 ? 1 : it.rows <= 8 ? 2 : 4;
  if (sizes != 0) {
    const unsigned n = grid((captured ? p->max_few : l.few.size()) * heads);
    switch (p->g.dim) {
      case 32: launch_few<32>(a, n, sizes, s); break;
      case 64: launch_few<64>(a, n, sizes, s); break;
      case 96: launch_few<96>(a, n, sizes, s); break;
      case 128: launch_few<128>(a, n, sizes, s); break;
      case 160: launch_few<160>(a, n, sizes, s); break;
      case 192: launch_few<192>(a, n, sizes, s); break;
      case 224: launch_few<224>(a, n, sizes, s); break;
      default: launch_few<256>(a, n, sizes, s); break;
    }
  }
  if (captured || !l.many.empty()) {
    const unsigned n = grid((captured ? p->max_many : l.many.size()) * heads);
    switch (p->g.dim) {
      case 32: attention_many<32><<<n, kThreads, 0, s>>>(a); break;
      case 64: attention_many<64><<<n, kThreads, 0, s>>>(a); break;
      case 96: attention_many<96><<<n, kThreads, 0, s>>>(a); break;
      case 128: attention_many<128><<<n, kThreads, 0, s>>>(a); break;
      case 160: attention_many<160><<<n, kThreads, 0, s>>>(a); break;
      case 192: attention_many<192><<<n, kThreads, 0, s>>>(a); break;
      case 224: attention_many<224><<<n, kThreads, 0, s>>>(a); break;
      default: attention_many<256><<<n, kThreads, 0, s>>>(a); break;
    }
  }
  if (captured || !l.join.empty())
    attention_join<<<grid((captured ? p->max_join : l.join.size()) * heads * kFewRows), kThreads, 0, s>>>(a);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // namespace llmi_hip::kv8
