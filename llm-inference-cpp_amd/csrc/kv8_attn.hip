// Attention over the paged 8-bit key/value cache (llmi_hip_kv8_attention_dev).
#include "kv8.hpp"

namespace llmi_hip::kv8 {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any float
constexpr float kLog2e = 1.44269504088896340736f;

struct AttnArgs {
  View v;
  Geometry g;
  const std::int8_t *k, *val;
  const float* scales;
  const float* q;
  float* out;
  float* parts;  // rows of partial states: o (dim floats each), then (maximum, sum) each
  std::size_t q_stride, out_stride, part_states;  // part_states: where the (maximum, sum) pairs begin, in floats
  float scale;
  int nfew, nmany, njoin;  // -1: from v.counts (a captured launch)
};

// 2^x by the hardware instruction: one rounding; results below 2^-126, which
// no sum here keeps, are 0.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Row r of a work item (row0 being its first): its token and its place in q and out.
struct Row {
  int tok;
  std::size_t off;  // of head_dim floats in the token's row
};
__device__ __forceinline__ Row row_of(const AttnArgs& A, int row0, int head, int r) {
  const int row = row0 + r, tok = row / A.g.group;
  return {tok, static_cast<std::size_t>(head * A.g.group + (row - tok * A.g.group)) * A.g.dim};
}
// Row r of a piece whose state is in slots `part` .. part + step - 1.
__device__ __forceinline__ std::size_t part_row(const AttnArgs& A, int part, int step, int head, int r) {
  return (static_cast<std::size_t>(part) * A.g.kv_heads + static_cast<std::size_t>(head) * step) * kSlotRows + r;
}

// Joins the pieces of split rows: each share's in their order, then the
// shares', so that a batch gives the same bits every time.  A
// workgroup takes `at` rows of one head; a thread four dims of a row over
// every `share`-th piece, eight loads of each kind in flight (what bounds
// this is their latency), with the running maximum; the shares meet in LDS.
__global__ void __launch_bounds__(kJoinThreads) attention_join(AttnArgs A, int join_rows, int join_at) {
  __shared__ float2 sh_state[kJoinThreads];
  __shared__ float4 sh_o[kJoinThreads];
  const int njoin = A.njoin >= 0 ? A.njoin : A.v.counts->join;
  const int at = A.njoin >= 0 ? join_at : A.v.counts->join_at;
  const int chunks = ((A.njoin >= 0 ? join_rows : A.v.counts->join_rows) + at - 1) / at;
  const int quads = A.g.dim / 4, cells = at * quads, share = kJoinThreads / cells;
  const int mine = static_cast<int>(threadIdx.x) % cells, of = static_cast<int>(threadIdx.x) / cells;
  const int units = njoin * A.g.kv_heads * chunks;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = u / (A.g.kv_heads * chunks), rest = u - item * A.g.kv_heads * chunks;
    const int head = rest / chunks, r = (rest - head * chunks) * at + mine / quads, d = 4 * (mine % quads);
    const JoinItem it = A.v.join[item];
    float m = -INFINITY, l = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < it.rows && of < share) {
      for (int c0 = of; c0 < it.n; c0 += 8 * share) {
        float2 st[8];
        float4 o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const std::size_t row = part_row(A, it.part + min(c0 + j * share, it.n - 1) * it.step, it.step, head, r);
          st[j] = *reinterpret_cast<const float2*>(A.parts + A.part_states + 2 * row);
          o[j] = *reinterpret_cast<const float4*>(A.parts + row * A.g.dim + d);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c0 + j * share >= it.n) st[j] = make_float2(-INFINITY, 0.0f);
          top = fmaxf(top, st[j].x);
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        const float keep = exp2_hw(m - ref);
        l *= keep;
        x = make_float4(x.x * keep, x.y * keep, x.z * keep, x.w * keep);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c0 + j * share >= it.n) continue;  // (a repeated piece may hold NaN)
          const float f = exp2_hw(st[j].x - ref);
          l = fmaf(st[j].y, f, l);
          x = make_float4(fmaf(o[j].x, f, x.x), fmaf(o[j].y, f, x.y), fmaf(o[j].z, f, x.z), fmaf(o[j].w, f, x.w));
        }
        m = top;
      }
    }
    sh_state[threadIdx.x] = make_float2(m, l);
    sh_o[threadIdx.x] = x;
    __syncthreads();
    if (of == 0 && r < it.rows) {
      for (int w = 1; w < share; ++w) {
        const float2 s = sh_state[w * cells + mine];
        const float4 o = sh_o[w * cells + mine];
        const float top = fmaxf(m, s.x), ref = top == -INFINITY ? 0.0f : top;
        const float f = exp2_hw(m - ref), g = exp2_hw(s.x - ref);
        l = fmaf(s.y, g, l * f);
        x = make_float4(fmaf(o.x, g, x.x * f), fmaf(o.y, g, x.y * f), fmaf(o.z, g, x.z * f), fmaf(o.w, g, x.w * f));
        m = top;
      }
      const Row w = row_of(A, it.row0, head, r);
      *reinterpret_cast<f4*>(A.out + static_cast<std::size_t>(it.row + w.tok) * A.out_stride + w.off + d) =
          f4{x.x / l, x.y / l, x.z / l, x.w / l};
    }
    __syncthreads();
  }
}

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
// with w = p * value scale, fixed-point against a power of two over the row's
// largest of the tile (so that large values that a row does not see, or gives
// no weight, cost the others no bits), p the weight against the running
// maximum.  A wavefront takes tiles of 64 positions = 4
// blocks; a workgroup's wavefronts take a range's tiles in turn and merge.
// Why digits: the codes need no conversion, so the vector ALUs see only the
// scores (one per position, head and lane group, not one per code), and 31
// fixed-point bits are more than fp32's 24.
// Measured: 64 users of 32/8 heads of 128 over 263k positions 95 us, 5.7 TB/s
// of codes and scales (a large copy moves 4.7, reads and writes together);
// over 4000 positions each 93 us.  One user over 300 positions (9/3 heads of
// 64) 4.5 us, what a launch and its four dependent loads take.  16 drafts of 3
// to 6 tokens (12 to 24 rows a head): 26.7 us with the join for 60 MB, bound by
// the four row tiles' scores and by one workgroup a compute unit (their
// registers).
constexpr int kFewWaves = 8, kFewThreads = 64 * kFewWaves;

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
// sum_i 2^(8i) s[i].  |s[i]| is at most 2^7 * 127 * 256 < 2^22, so pairs fit 32 bits.
__device__ __forceinline__ float undigit(i4 s) {
  return fmaf(static_cast<float>((s[3] << 8) + s[2]), 65536.0f, static_cast<float>((s[1] << 8) + s[0]));
}

// HD: head_dim; MT: tiles of 4 rows (16 digit rows) there is room for.
template <int HD, int MT>
__global__ void __launch_bounds__(kFewThreads) attention_few(AttnArgs A) {
  constexpr int kWaves = kFewWaves, kThreads = kFewThreads;
  constexpr int kG = HD / 16;            // 16-dim groups of a block
  constexpr int kC = (HD + 63) / 64;     // 64-dim steps of a score product
  constexpr int kRows = 4 * MT;
  __shared__ union {
    std::uint32_t w[kWaves][4][4][16];   // a tile's weight digits: [block][head of the 4][position]
    float o[kWaves][kRows][HD + 16];     // (16: a row of lanes writes other banks than the next)
                                         // the wavefronts' outputs, merged at the end
  } sh;
  __shared__ float sh_m[kWaves][kRows], sh_l[kWaves][kRows];
  __shared__ i4 sh_q[MT][kC][64];       // the digits of q as the products take them
  __shared__ int sh_qe[MT][4];          // a row's exponent
  __shared__ float sh_qbad[MT][4];      // NaN for a row with inf or NaN in q, else 0
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lo16 = lane & 15, grp = lane >> 4;
  const int nfew = A.nfew >= 0 ? A.nfew : A.v.counts->few;
  const unsigned units = static_cast<unsigned>(nfew) * A.g.kv_heads;
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = static_cast<int>(u / A.g.kv_heads), h = static_cast<int>(u) - item * A.g.kv_heads;
    const AttnItem it = A.v.few[item];

    const int last_block = (it.hi - 1) / kBlk;
    // This lane's block of a tile is block base / 16 + grp; behind the range,
    // the last one again (its positions there are masked), with scales of 0.
    // Its page id is read a tile ahead.
    const auto page_id = [&](int base) { return A.v.table[it.table + page_of(A.g, min(base / kBlk + grp, last_block))]; };
    int id = page_id(min(it.lo + wave * kTile, it.hi - 1));
    // A tile's keys: every lane needs all four blocks, position lo16, dims
    // 16 (4c + grp) ...  They are asked for as soon as the tile before has
    // used its own, and the values once the scores are made (all together at
    // the tile's start: 64 users of 32/8 heads of 128 over 4000 positions 94 us
    // against 92, one user over 300 positions 5.6 against 4.7).
    std::size_t at = 0;
    float2 sc = make_float2(0.0f, 0.0f);
    i4 kf[4][kC];
    const auto fetch_keys = [&](int base) {
      const int block = min(base / kBlk + grp, last_block);
      at = block_at(A.g, id, page_of(A.g, block), block, h);
      if (base + kWaves * kTile < it.hi) id = page_id(base + kWaves * kTile);
      sc = reinterpret_cast<const float2*>(A.scales)[at];
      const std::uint64_t p = reinterpret_cast<std::uint64_t>(A.k + at * (16 * HD));
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const std::uint32_t plo = __builtin_amdgcn_readlane(static_cast<int>(p), 16 * b);
        const std::uint32_t phi = __builtin_amdgcn_readlane(static_cast<int>(p >> 32), 16 * b);
        const auto* src = reinterpret_cast<const std::int8_t*>((static_cast<std::uint64_t>(phi) << 32) | plo);
#pragma unroll
        for (int c = 0; c < kC; ++c)
          kf[b][c] = *reinterpret_cast<const i4*>(src + min(4 * c + grp, kG - 1) * 256 + lo16 * 16);
      }
    };
    i4 vf[kG];
    const auto fetch_values = [&]() {
      const std::int8_t* vp = A.val + at * (16 * HD) + lo16 * 16;
#pragma unroll
      for (int g = 0; g < kG; ++g) vf[g] = *reinterpret_cast<const i4*>(vp + g * 256);
    };
    // (The first tile's are on their way while q is prepared.)
    if (it.lo + wave * kTile < it.hi) fetch_keys(it.lo + wave * kTile);

    // The digits of q, by one wavefront for each tile of rows: lane (digit row
    // lo16, dims 16 grp ..) of each 64-dim step.
    if (wave < MT) {
      const int r = 4 * wave + lo16 / 4;
      // Rows of nobody repeat the first one; nothing of theirs is kept.
      const Row w = row_of(A, it.row0, h, r < it.rows ? r : 0);
      const float* qp = A.q + static_cast<std::size_t>(it.row + w.tok) * A.q_stride + w.off;
      float x[kC][16];
      float top = 0.0f;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        const int g = 4 * c + grp;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const f4 y = *reinterpret_cast<const f4*>(qp + min(g, kG - 1) * 16 + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[c][i + j] = g < kG ? y[j] : 0.0f;
            top = fmaxf(top, fabsf(x[c][i + j]));
            bad |= !(fabsf(x[c][i + j]) < INFINITY);
          }
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      // (Every lane takes part in an exchange: no short-circuit.)
      bad |= __shfl_xor(static_cast<int>(bad), 16, 64) != 0;
      bad |= __shfl_xor(static_cast<int>(bad), 32, 64) != 0;
      int e;
      (void)frexpf(top, &e);  // top < 2^e
      if (bad || !(top > 0.0f)) e = 0;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        i4 d4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          std::uint32_t d = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int X = bad ? 0 : static_cast<int>(rintf(ldexpf(x[c][4 * j + i], 30 - e)));
            d |= ((digits(X) >> (8 * (lo16 & 3))) & 0xFFu) << (8 * i);
          }
          d4[j] = static_cast<int>(d);
        }
        sh_q[wave][c][lane] = d4;
      }
      if (lane < 16 && (lane & 3) == 0) {
        sh_qe[wave][lane / 4] = e - 30;
        sh_qbad[wave][lane / 4] = bad ? __builtin_nanf("") : 0.0f;
      }
    }
    __syncthreads();
    i4 qd[MT][kC];
    float m[MT], l[MT], o[MT][kG];
    int qe[MT];  // this lane's score row (head grp of the tile)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int c = 0; c < kC; ++c) qd[mt][c] = sh_q[mt][c][lane];
      qe[mt] = sh_qe[mt][grp];
      l[mt] = sh_qbad[mt][grp];
    }

    int limit[MT];  // last position that this lane's row sees, -1 for rows of nobody
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = 4 * mt + grp;
      limit[mt] = r < it.rows ? it.start + (it.row0 + r) / A.g.group : -1;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m[mt] = -INFINITY;
#pragma unroll
      for (int g = 0; g < kG; ++g) o[mt][g] = 0.0f;
    }

    for (int base = it.lo + wave * kTile; base < it.hi; base += kWaves * kTile) {
      if (base / kBlk + grp > last_block) sc = make_float2(0.0f, 0.0f);
      // The blocks' value scales (0 where not finite; NaN then in `odd`), and
      // their mantissas and exponents apart: a weight times a scale is taken in
      // these two steps, so that small scales cost no bits.
      const auto of_block = [](float x, int b) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16 * b)); };
      const float sc_value = sc.y < INFINITY ? sc.y : 0.0f, sc_odd = sc.y * 0.0f;
      const float sc_mant = __builtin_amdgcn_frexp_mantf(sc_value);
      const int sc_exp = __builtin_amdgcn_frexp_expf(sc_value);
      float ks[4], vs[4], vm[4], odd[4];
      int ve[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        ks[b] = of_block(sc.x, b);
        vs[b] = of_block(sc_value, b);
        vm[b] = of_block(sc_mant, b);
        odd[b] = of_block(sc_odd, b);
        ve[b] = __builtin_amdgcn_readlane(sc_exp, 16 * b);
      }
      float x[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          i4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < kC; ++c) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qd[mt][c], kf[b][c], acc, 0, 0, 0);
          x[mt][b] = undigit(acc) * ldexpf(A.scale * kLog2e * ks[b], qe[mt]);
          if (base + b * kBlk + lo16 > limit[mt]) x[mt][b] = -INFINITY;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      fetch_values();
      if (base + kWaves * kTile < it.hi) fetch_keys(base + kWaves * kTile);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float mx = fmaxf(fmaxf(fmaxf(x[mt][0], x[mt][1]), fmaxf(x[mt][2], x[mt][3])), m[mt]);
        mx = row16_max(mx);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        const float keep = exp2_hw(m[mt] - ref);
        m[mt] = mx;
        float sum = 0.0f, w[4], top = 0.0f;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const bool seen = base + b * kBlk + lo16 <= limit[mt];
          const float p = exp2_hw(x[mt][b] - ref);
          // A value scale that is inf or NaN shows in the sum of the rows that see the block.
          if (seen) sum += p + odd[b];
          w[b] = p * vm[b];
          top = fmaxf(top, p * vs[b]);
        }
        // The row's largest is below 2^we (for which a denormal product will do).
        const int we = __builtin_amdgcn_frexp_expf(row16_max(top));
#pragma unroll
        for (int b = 0; b < 4; ++b)
          sh.w[wave][b][grp][lo16] = digits(static_cast<int>(rintf(ldexpf(w[b], 30 - we + ve[b]))));
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
#pragma unroll
        for (int g = 0; g < kG; ++g) {
          i4 acc = {0, 0, 0, 0};
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wd, vf[g], acc, 0, 0, 0);
          o[mt][g] = fmaf(o[mt][g], keep, ldexpf(undigit(acc), we - 30));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // Merge the wavefronts' states: lane (dim lo16 of each group, head grp).
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
    for (int e = threadIdx.x; e < it.rows * (HD / 2); e += kThreads) {
      const int r = e / (HD / 2), d = 2 * (e - r * (HD / 2));
      float top = sh_m[0][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sh_m[w][r]);
      const float ref = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = exp2_hw(sh_m[w][r] - ref);
        sum = fmaf(sh_l[w][r], f, sum);
        x = fmaf(sh.o[w][r][d], f, x);
        y = fmaf(sh.o[w][r][d + 1], f, y);
      }
      if (it.part >= 0) {
        const std::size_t row = part_row(A, it.part, few_rows(HD) / kSlotRows, h, r);
        *reinterpret_cast<float2*>(A.parts + row * HD + d) = make_float2(x, y);
        if (d == 0) *reinterpret_cast<float2*>(A.parts + A.part_states + 2 * row) = make_float2(top, sum);
      } else {
        const Row w = row_of(A, it.row0, h, r);
        float* dst = A.out + static_cast<std::size_t>(it.row + w.tok) * A.out_stride + w.off + d;
        dst[0] = x / sum;
        dst[1] = y / sum;
      }
    }
    __syncthreads();
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
// w = p * value scale * 2^kWeightBits over (to a power of two) the row's
// largest product of the two so far: block scales differ along the sum, so
// they ride on the weights (against the largest scale alone, a block that a row
// does not see, or gives no weight, would take bits from the others).
// Why two parts: one fp16 part of q or w is off by 2^-12, which shows as 1e-4
// of the result; two are off by 2^-22 or less, below fp32's sums.  That is twice the
// formula's products: 2048 tokens over 6144 positions of 32/8 heads of 128
// are 481 GFLOP, 414 us at the 1162 TFLOP/s of a large fp16 library product;
// this kernel takes 408 to 421 by card.  The matrix units are busy 52 %
// of the clocks; what is left are the staging's conversions (38 us without
// them), the wait for a tile's codes (20) and the maximum's dependency.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f16v __attribute__((ext_vector_type(16)));
constexpr int kWeightBits = 8;  // with kSlack: weights stay below 2^14
constexpr float kSlack = 6.0f;

// x of the lane 32 on (or back).
__device__ __forceinline__ float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) != 0 ? r[0] : r[1]);
}

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

constexpr int kAhead = 4;  // operands on their way from LDS

template <int HD>
__global__ void __launch_bounds__(256, HD <= 128 ? 2 : 1) attention_many(AttnArgs A) {

  constexpr int kG = HD / 16;
  constexpr int kPer = (HD + 63) / 64;  // 16-byte pieces a lane has of a block's keys (and of its values)
  __shared__ uint4 sh_k[2][kG][2][kTile];     // [16-dim group][half of it][position]: 8 fp16
  __shared__ uint4 sh_v[2][kTile / 16][2][HD];  // [block][h][dim]: positions 4h.., 8 + 4h..
  __shared__ float4 sh_s[2][4];               // a tile's blocks: see block_terms
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nmany = A.nmany >= 0 ? A.nmany : A.v.counts->many;
  const unsigned units = static_cast<unsigned>(nmany) * A.g.kv_heads;
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    const int item = static_cast<int>(u / A.g.kv_heads), head = static_cast<int>(u) - item * A.g.kv_heads;
    const AttnItem it = A.v.many[item];
    // (Opaque: what is computed from it is not kept in registers around the loop over units.)
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    const int col = lane & 31, h2nd = lane >> 5;
    const int r = wave * 32 + col;
    const bool live = r < it.rows;
    const Row own = row_of(A, it.row0, head, live ? r : 0);
    const int limit = live ? it.start + own.tok : -1;
    // A negative scale goes to q, so that a block's largest score is its largest product.
    const float q_sign = A.scale < 0.0f ? -1.0f : 1.0f, scale = fabsf(A.scale) * kLog2e;

    const int last_block = (it.hi - 1) / kBlk;
    // A wavefront brings one of the tile's four blocks; its page id is read a
    // tile ahead of it (behind the range: the last block again, whose
    // positions there are masked).
    uint4 kreg[kPer], vreg[kPer];
    float2 sreg = make_float2(0.0f, 0.0f);
    bool sreg_live = true;
    // (The index is the wavefront's; kept in a vector register, so that the
    // load is waited for where the id is used and not where it is made.)
    int id = 0;
    const auto lookup = [&](int base) {
      int at = it.table + page_of(A.g, min(base / kBlk + wave, last_block));
      asm volatile("" : "+v"(at));
      id = A.v.table[at];
    };
    const auto fetch = [&](int base) {
      const int want = base / kBlk + wave, block = min(want, last_block);
      const std::size_t at = block_at(A.g, __builtin_amdgcn_readfirstlane(id), page_of(A.g, block), block, head);
      const auto* kp = reinterpret_cast<const uint4*>(A.k + at * (16 * HD));
      const auto* vp = reinterpret_cast<const uint4*>(A.val + at * (16 * HD));
#pragma unroll
      for (int n = 0; n < kPer; ++n) {
        const int c = min(n * 64 + lane, HD - 1);
        kreg[n] = kp[c];
        vreg[n] = vp[c];
      }
      sreg = reinterpret_cast<const float2*>(A.scales)[at];
      sreg_live = want <= last_block;
    };
    // The first tile's codes are on their way while q is prepared.
    lookup(it.lo);
    fetch(it.lo);
    if (it.lo + kTile < it.hi) lookup(it.lo + kTile);

    // q * 2^qs, its largest below 2^14, as two fp16 parts.
    h8 qh[kG], ql[kG];
    int qs;
    {
      const float* qp = A.q + static_cast<std::size_t>(it.row + own.tok) * A.q_stride + own.off;
      float x[kG][8], top = 0.0f;
#pragma unroll
      for (int g = 0; g < kG; ++g)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const f4 y = *reinterpret_cast<const f4*>(qp + 16 * g + 8 * h2nd + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[g][i + j] = y[j] * q_sign;
            top = fmaxf(top, fabsf(y[j]));
          }
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
    // All of the wavefront's rows see positions up to `all`.
    int all = live ? limit : 0x7FFFFFFF;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) all = min(all, __shfl_xor(all, o, 64));
    all = __builtin_amdgcn_readfirstlane(all);

    f16v o[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    // m: what scores are taken against, about kSlack below the largest so far
    // at most; rm: the same for scores plus log2 of the value scale.  Both are
    // whole numbers, so that factors between them are exact.
    float m = -INFINITY, l = 0.0f, rm = -INFINITY;

    // What the products take of the block that `fetch` brought: the key scale
    // times the softmax's, the value scale's exponent (-inf: its codes are 0,
    // or masked), NaN if a scale is not finite, and log2 of the value scale's
    // mantissa (apart from the exponent, next to which it would lose bits).
    const auto block_terms = [&]() {
      const bool fin = sreg.y > 0.0f && sreg.y < INFINITY;
      return sreg_live ? make_float4(scale * sreg.x, fin ? static_cast<float>(__builtin_amdgcn_frexp_expf(sreg.y)) : -INFINITY,
                                     fmaf(sreg.x, 0.0f, sreg.y * 0.0f),
                                     fin ? __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(sreg.y)) : 0.0f)
                       : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
    };
    // Staging in kPieces steps, each four codes of every lane to fp16; every
    // second one stores eight of them: dims 0-7 or 8-15 of a position's keys,
    // positions 0-3, 8-11 or 4-7, 12-15 of a dim's values.
    constexpr int kPieces = 8 * kPer;
    std::uint32_t half[4];
    const auto stage_step = [&](int to, int q) {
      const int n = q / 8, j = q % 4, side = j / 2;
      const bool keys = q % 8 < 4;
      const uint4 u = keys ? kreg[n] : vreg[n];
      const int from = keys ? j : (j % 2) * 2 + side;  // which four of the sixteen
      halves(from == 0 ? u.x : from == 1 ? u.y : from == 2 ? u.z : u.w, half + 2 * (j % 2));
      if (j % 2 == 0) return;
      const int c = n * 64 + lane;
      if (HD % 64 != 0 && c >= HD) return;
      const uint4 out = make_uint4(half[0], half[1], half[2], half[3]);
      if (keys)
        sh_k[to][c / 16][side][16 * wave + c % 16] = out;
      else
        sh_v[to][wave][side][c] = out;
    };
    const auto stage = [&](int to) {
#pragma unroll
      for (int q = 0; q < kPieces; ++q) stage_step(to, q);
      if (lane == 0) sh_s[to][wave] = block_terms();
    };

    stage(0);
    if (it.lo + kTile < it.hi) fetch(it.lo + kTile);
    if (it.lo + 2 * kTile < it.hi) lookup(it.lo + 2 * kTile);
    __syncthreads();
    int buf = 0;
    // Per tile: the score products, with the next tile's staging between
    // them; the tile after that fetched; the weights; the output products,
    // with the next block's weights between them.  The order is fixed by
    // scheduling barriers: kAhead operands are on their way from LDS while
    // the products of earlier ones run.
    for (int base = it.lo; base < it.hi; base += kTile, buf ^= 1) {
      f16v st[2];
      float4 term[4];
      const f16v zero = {};

      h8 kf[kAhead];
      const auto key = [&](int n) { return __builtin_bit_cast(h8, sh_k[buf][n / 2][h2nd][32 * (n & 1) + col]); };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) kf[n] = key(n);
      constexpr int kSteps = 2 * kG, kEach = (kPieces + kSteps - 1) / kSteps;
#pragma unroll
      for (int n = 0; n < kSteps; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        f16v& s = st[n & 1];
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n % kAhead], qh[n / 2], n < 2 ? zero : s, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        // (Behind the last tile the pieces are the one before's, and go to the buffer that is free.)
#pragma unroll
        for (int q = n * kEach; q < (n + 1) * kEach && q < kPieces; ++q) stage_step(buf ^ 1, q);
        if (n == kSteps - 2) {
#pragma unroll
          for (int b = 0; b < 4; ++b) term[b] = sh_s[buf][b];
        }
        __builtin_amdgcn_sched_barrier(0);
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[n % kAhead], ql[n / 2], s, 0, 0, 0);
        if (n + kAhead < kSteps) kf[n % kAhead] = key(n + kAhead);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (lane == 0) sh_s[buf ^ 1][wave] = block_terms();
      if (base + 2 * kTile < it.hi) fetch(base + 2 * kTile);
      if (base + 3 * kTile < it.hi) lookup(base + 3 * kTile);
      // Per block: scores are f times the products (f is positive: where
      // the scale is 0 the products are, and a masked -inf stays -inf).
      float f[4], ratio[4], bad = 0.0f;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f[b] = fmaxf(ldexpf(term[b].x, -qs), 0x1p-126f);
        bad += term[b].z;
      }
      // Positions behind a row's own leave nothing.
      if (base + kTile - 1 > all) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (base + 16 * b + 8 * (i / 4) + 4 * h2nd + i % 4 > limit) st[b / 2][8 * (b & 1) + i] = -INFINITY;
      }
      float mx = -INFINITY, rx = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, st[b / 2][8 * (b & 1) + i]);
        mx = fmaxf(mx, top * f[b]);
        rx = fmaxf(rx, fmaf(top, f[b], term[b].y));
      }
      mx = fmaxf(mx, other_half(mx));
      rx = fmaxf(rx, other_half(rx));
      // The sums are rescaled where one of the two has grown by more than
      // kSlack (weights may be up to 2^kSlack before that).
      const bool grown = mx > m + kSlack, risen = rx > rm + kSlack;
      if (__any(grown || risen)) {
        const float now = grown ? rintf(mx) : m, r_now = risen ? rintf(rx) : rm;
        l *= now == -INFINITY ? 0.0f : exp2_hw(m - now);
        const float rescale = r_now == -INFINITY ? 0.0f : exp2_hw(rm - r_now);
        m = now;
        rm = r_now;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[d][i] *= rescale;
      }
      // Weights carry 2^ratio, the value scale against rm.  One below 2^-60
      // counts as that; a scale of 0 has codes of 0.
      const float base_m = m == -INFINITY ? 0.0f : m, base_r = base_m - (rm == -INFINITY ? 0.0f : rm);
#pragma unroll
      for (int b = 0; b < 4; ++b) ratio[b] = term[b].y == -INFINITY ? 0.0f : fmaxf(term[b].y + base_r + term[b].w, -60.0f);
      const float ref = static_cast<float>(kWeightBits) - base_m;
      float off[4], part[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        off[b] = ratio[b] + ref;
        part[b] = 0.0f;
      }
      // Weights i and i + 1 of block b, in their two fp16 parts.
      std::uint32_t wh[2][4], wl[2][4];
      const auto weigh = [&](int b, int i) {
        const float w0 = exp2_hw(fmaf(st[b / 2][8 * (b & 1) + i], f[b], off[b]));
        const float w1 = exp2_hw(fmaf(st[b / 2][8 * (b & 1) + i + 1], f[b], off[b]));
        part[b] += w0;
        part[b] += w1;
        const h2 hi = {static_cast<_Float16>(w0), static_cast<_Float16>(w1)};
        const std::uint32_t hi_bits = __builtin_bit_cast(std::uint32_t, hi);
        std::uint32_t lo;  // fp16(w - hi), each half in one instruction
        asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(hi_bits), "v"(w0));
        asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(hi_bits), "v"(w1));
        wh[b & 1][i / 2] = hi_bits;
        wl[b & 1][i / 2] = lo;
      };
      const auto both = [&](const std::uint32_t (&w)[4]) {
        return __builtin_bit_cast(h8, make_uint4(w[0], w[1], w[2], w[3]));
      };
      constexpr int kD = HD / 32;
      h8 vfr[kAhead];
      const auto value = [&](int n) { return __builtin_bit_cast(h8, sh_v[buf][n / kD][h2nd][32 * (n % kD) + col]); };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) vfr[n] = value(n);
#pragma unroll
      for (int i = 0; i < 8; i += 2) weigh(0, i);
#pragma unroll
      for (int n = 0; n < 4 * kD; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        const int b = n / kD, d = n % kD;
        // Pairs of the next block's weights that this step computes.
        const int i0 = d * 4 / kD, i1 = (d + 1) * 4 / kD;
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vfr[n % kAhead], both(wh[b & 1]), o[d], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = i0; i < (i0 + i1 + 1) / 2; ++i)
          if (b < 3) weigh(b + 1, 2 * i);
        __builtin_amdgcn_sched_barrier(0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vfr[n % kAhead], both(wl[b & 1]), o[d], 0, 0, 0);
        if (n + kAhead < 4 * kD) vfr[n % kAhead] = value(n + kAhead);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = (i0 + i1 + 1) / 2; i < i1; ++i)
          if (b < 3) weigh(b + 1, 2 * i);
      }
      __builtin_amdgcn_sched_barrier(0);
      float sum = 0.0f;
#pragma unroll
      for (int b = 0; b < 4; ++b) sum = fmaf(part[b], exp2_hw(-ratio[b]) * (1.0f / (1 << kWeightBits)), sum);
      if (bad != bad) {
        // A scale that is inf or NaN shows in the rows that see a position of its block.
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (base + 16 * b <= limit) sum += sh_s[buf][b].z;
      }
      l += sum;
      __syncthreads();
    }

    l += __shfl_xor(l, 32, 64);
    // What the output's sums are to be multiplied with is 2^unit.
    const int unit = static_cast<int>(fminf(fmaxf(rm - m, -1000.0f), 1000.0f)) - kWeightBits;
    const float any_value = rm == -INFINITY ? 0.0f : 1.0f;
    int end_lane = threadIdx.x & 63;
    asm volatile("" : "+v"(end_lane));
    const int end_h = end_lane >> 5, end_r = wave * 32 + (end_lane & 31);
    const Row mine = row_of(A, it.row0, head, live ? end_r : 0);
    if (live && it.part >= 0) {
      const std::size_t part = part_row(A, it.part, kManyRows / kSlotRows, head, end_r);
      if (end_h == 0) *reinterpret_cast<float2*>(A.parts + A.part_states + 2 * part) = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(A.parts + part * HD + 32 * d + 8 * i + 4 * end_h) =
              make_float4(ldexpf(o[d][4 * i] * any_value, unit), ldexpf(o[d][4 * i + 1] * any_value, unit),
                          ldexpf(o[d][4 * i + 2] * any_value, unit), ldexpf(o[d][4 * i + 3] * any_value, unit));
    } else if (live) {
      float* dst = A.out + static_cast<std::size_t>(it.row + mine.tok) * A.out_stride + mine.off;
      const float f = any_value / l;
#pragma unroll
      for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f4*>(dst + 32 * d + 8 * i + 4 * end_h) =
              f4{ldexpf(o[d][4 * i] * f, unit), ldexpf(o[d][4 * i + 1] * f, unit), ldexpf(o[d][4 * i + 2] * f, unit),
                 ldexpf(o[d][4 * i + 3] * f, unit)};
    }
  }
}

template <int HD>
void launch(const AttnArgs& a, unsigned few, unsigned many, int rows, hipStream_t s) {
  if (few > 0) {
    if (rows <= 4)
      attention_few<HD, 1><<<few, kFewThreads, 0, s>>>(a);
    else if (rows <= 8)
      attention_few<HD, 2><<<few, kFewThreads, 0, s>>>(a);
    else if constexpr (few_rows(HD) > 8) {
      if (rows <= 12)
        attention_few<HD, 3><<<few, kFewThreads, 0, s>>>(a);
      else
        attention_few<HD, 4><<<few, kFewThreads, 0, s>>>(a);
    }
  }
  if (many > 0) attention_many<HD><<<many, 256, 0, s>>>(a);
}

}  // namespace

int launch_attention(const llmi_hip_kv8_plan* p, const llmi_kv8_layer& layer, const float* q, std::size_t q_stride,
                     float scale, float* out, std::size_t out_stride, hipStream_t s, bool captured) {
  const Lists& l = p->lists;
  const std::size_t heads = static_cast<std::size_t>(p->g.kv_heads);
  const std::size_t part_rows = p->most.parts * static_cast<std::size_t>(p->g.kv_heads) * kSlotRows;
  AttnArgs a{p->view(), p->g, layer.k, layer.v, layer.scales, q, out, p->parts, q_stride, out_stride,
             part_rows * static_cast<std::size_t>(p->g.dim), scale, captured ? -1 : static_cast<int>(l.few.size()),
             captured ? -1 : static_cast<int>(l.many.size()),
             captured ? -1 : static_cast<int>(l.join.size())};
  // A captured launch has the kernels that the batch needs (an empty one:
  // every kind), each with room for any batch that the plan takes, but no more
  // workgroups than fill the chip several times (each takes further units in
  // turn).  Batches of other kinds are refused from then on.
  const bool any = captured && l.tokens == 0;
  const bool has_few = any || !l.few.empty(), has_many = any || !l.many.empty();
  const int most_rows = few_rows(p->g.dim);
  const int rows = any ? most_rows : captured ? captured_rows(l, p->g.dim) : l.few_rows;
  if (captured) {
    p->captured_few = std::min(p->captured_few, has_few ? rows : 0);
    p->captured_many = p->captured_many && has_many;
  }
  const auto grid = [&](bool has, std::size_t items, std::size_t most) {
    if (!has) return 0u;
    const std::size_t units = (captured ? most : items) * heads;
    return static_cast<unsigned>(std::min<std::size_t>(units, captured ? 4096 : kMostGroups));
  };
  const unsigned few = grid(has_few, l.few.size(), p->most.few), many = grid(has_many, l.many.size(), p->most.many);
  switch (p->g.dim) {
    case 32: launch<32>(a, few, many, rows, s); break;
    case 64: launch<64>(a, few, many, rows, s); break;
    case 96: launch<96>(a, few, many, rows, s); break;
    case 128: launch<128>(a, few, many, rows, s); break;
    case 160: launch<160>(a, few, many, rows, s); break;
    case 192: launch<192>(a, few, many, rows, s); break;
    case 224: launch<224>(a, few, many, rows, s); break;
    default: launch<256>(a, few, many, rows, s); break;
  }
  if (captured || !l.join.empty()) {
    const std::size_t chunks = (l.join_rows + l.join_at - 1) / l.join_at;
    const std::size_t units = captured ? 4096 : l.join.size() * heads * chunks;
    attention_join<<<static_cast<unsigned>(units), kJoinThreads, 0, s>>>(a, l.join_rows, l.join_at);
  }
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // namespace llmi_hip::kv8
