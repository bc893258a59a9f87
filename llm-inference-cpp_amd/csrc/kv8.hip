// The paged 8-bit key/value cache (llmi_hip_kv8_*): plans, append, read.
#include <cstring>
#include <memory>
#include <new>

#include "kv8.hpp"

namespace llmi_hip::kv8 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// Dword-aligned vectors: rows may start at any float.
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void load8(const float* __restrict__ p, float* x) {
  const f4 a = *reinterpret_cast<const f4*>(p), b = *reinterpret_cast<const f4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = a[i];
    x[4 + i] = b[i];
  }
}
__device__ __forceinline__ void store8(float* p, const float* x) {
  *reinterpret_cast<f4*>(p) = f4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f4*>(p + 4) = f4{x[4], x[5], x[6], x[7]};
}

// |x| as an unsigned integer orders like the value, with inf and NaN above
// every finite one, so that the largest of a block shows them.
__device__ __forceinline__ std::uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ std::uint32_t wave_umax(std::uint32_t v) {
  const auto ror = [](std::uint32_t x, auto ctrl) {  // within the 16 lanes of a row
    return static_cast<std::uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x120 + decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v = max(v, ror(v, std::integral_constant<int, 8>{}));
  v = max(v, ror(v, std::integral_constant<int, 4>{}));
  v = max(v, ror(v, std::integral_constant<int, 2>{}));
  v = max(v, ror(v, std::integral_constant<int, 1>{}));
  const auto row = [&](int lane) { return static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)); };
  return max(max(row(0), row(16)), max(row(32), row(48)));
}
// A block's scale, float(amax / 127) with one rounding (NaN and inf stay what
// they are), and what its codes are computed with.
struct Scale {
  float s, inverse;
  bool usable, plain;  // finite and not 0; 1 / s is a normal number too
  __device__ __forceinline__ explicit Scale(std::uint32_t amax)
      : s(static_cast<float>(static_cast<double>(__uint_as_float(amax)) / 127.0)),
        inverse(1.0f / s),
        usable(s > 0.0f && amax < 0x7F800000u),
        plain(s >= 0x1p-120f) {}
};
// The nearest integer to x / s, ties to even.  |x / s| is below 128, so the
// fp32 product with 1 / s is within 2^-15 of it and decides unless it comes
// that near to a border.  There the 64-bit quotient does: a quotient of two
// fp32 numbers is either a tie, which 64 bits hold exactly, or at least 2^-26
// of itself away from one.
__device__ __forceinline__ int code_of(float x, const Scale& s) {
  if (!s.usable) return 0;
  const float t = x * s.inverse;
  float r = rintf(t);
  if (!(fabsf(t - r) < 0.4999f) || !s.plain)
    r = static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(s.s)));
  return static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
}
// Byte j of a dword of codes.
__device__ __forceinline__ float code_value(std::uint32_t four, int j) {
  return static_cast<float>(static_cast<std::int32_t>(four << (24 - 8 * j)) >> 24);
}

// Lanes that share a row of a head: each holds dims 8c .. 8c+7 and their
// rotation partners DIM/2 + 8c ..; a power of two, so that sums over the row
// are exchanges between neighbours.
constexpr int lanes_per_row(int dim) { return dim <= 32 ? 2 : dim <= 64 ? 4 : dim <= 128 ? 8 : 16; }

// Norm and rotation of a row in 64 bits, rounded once: k's codes sit next to
// rounding borders, and one rounding makes them independent of the order of
// the norm's sum.  The 64-bit arithmetic is nearly hidden behind the loads (14k
// tokens of 32/8 heads of 128 with the norm's weights 157 us, without them 145).
// w, co, si: this lane's 16 (dims 8c .. and partners) and 8 + 8 numbers.
template <int DIM>
__device__ __forceinline__ void norm_rotate(float (&x)[16], bool live, bool norm, const float (&w)[16], float eps,
                                            bool turn, const float (&co)[8], const float (&si)[8]) {
  double r = 1.0;
  if (norm) {
    double ss = 0.0;
    if (live) {
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fma(static_cast<double>(x[i]), static_cast<double>(x[i]), ss);
    }
#pragma unroll
    for (int o = 1; o < lanes_per_row(DIM); o <<= 1) ss += __shfl_xor(ss, o, 64);
    r = 1.0 / sqrt(ss / DIM + static_cast<double>(eps));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double a = x[i], b = x[8 + i];
    if (norm) {
      a = a * r * static_cast<double>(w[i]);
      b = b * r * static_cast<double>(w[8 + i]);
    }
    if (turn) {
      const double c = co[i], s = si[i];
      const double t = fma(a, c, -(b * s));
      b = fma(b, c, a * s);
      a = t;
    }
    x[i] = static_cast<float>(a);
    x[8 + i] = static_cast<float>(b);
  }
}

struct AppendArgs {
  View v;
  Geometry g;
  llmi_kv8_layer layer;
  const float *q, *k, *val, *q_norm, *k_norm, *cos_t, *sin_t;
  float* q_out;
  std::size_t q_stride, k_stride, v_stride, q_out_stride;
  float eps;
  int nblocks, ntokens;  // -1: from v.counts (a captured launch)
  int q_each;            // head groups of a token that one wavefront takes
};

// A block as one wavefront sees it.
struct Block {
  int pos;
  std::size_t at;  // in [page][kv head][block]
};
__device__ __forceinline__ Block block_of(const Geometry& g, const BlockItem& it, int h, bool then) {
  const std::size_t page = then ? it.then_page : it.page;
  return {then ? it.then_pos : it.pos, (page * g.kv_heads + h) * g.page_blocks + (then ? it.then_block : it.block)};
}
__device__ __forceinline__ float* open_rows(const AppendArgs& A, const BlockItem& it, int dim, int h, int pos,
                                            int which) {
  return A.layer.open +
         ((((static_cast<std::size_t>(it.slot) * A.g.kv_heads + h) * 2 + (pos / kBlk & 1)) * 2 + which) * kBlk) * dim;
}

// Four codes of x / scale in a dword.
__device__ __forceinline__ std::uint32_t codes4(const float* x, const Scale& s) {
  std::uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= (static_cast<std::uint32_t>(code_of(x[j], s)) & 0xFFu) << (8 * j);
  return w;
}

// Keys of one block and head: lanes take (position, 8 dims and partners).
template <int DIM>
__device__ void append_keys(const AppendArgs& A, const BlockItem& it, int h, const Block& b, int lane) {
  constexpr int kLpr = lanes_per_row(DIM), kRows = 64 / kLpr, kPasses = (kBlk + kRows - 1) / kRows, kHalf = DIM / 2;
  const int c = lane % kLpr;
  float* open = open_rows(A, it, DIM, h, b.pos, 0);
  float x[kPasses][16];
  const bool chunk = DIM / 16 == kLpr || c < DIM / 16;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int tok = p * kRows + lane / kLpr, pos = b.pos + tok;
    const bool in = chunk && tok < kBlk;
    const float* src = pos < it.start ? open + tok * DIM
                                      : A.k + static_cast<std::size_t>(it.row + (pos - it.start)) * A.k_stride +
                                            static_cast<std::size_t>(h) * DIM;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[p][i] = 0.0f;
    if (in && pos < it.end) {
      load8(src + 8 * c, x[p]);
      load8(src + kHalf + 8 * c, x[p] + 8);
    }
  }
  // (Every lane loads: one without a row of its own the first token's.)
  float w[16] = {}, co[kPasses][8] = {}, si[kPasses][8] = {};
  const int c_in = chunk ? c : 0;
  if (A.k_norm != nullptr) {
    load8(A.k_norm + 8 * c_in, w);
    load8(A.k_norm + kHalf + 8 * c_in, w + 8);
  }
  if (A.cos_t != nullptr) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int pos = b.pos + p * kRows + lane / kLpr;
      const std::size_t at =
          static_cast<std::size_t>(pos >= it.start && pos < it.end ? pos : it.start) * kHalf + 8 * c_in;
      load8(A.cos_t + at, co[p]);
      load8(A.sin_t + at, si[p]);
    }
  }
  std::uint32_t amax = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int tok = p * kRows + lane / kLpr, pos = b.pos + tok;
    const bool fresh = chunk && tok < kBlk && pos >= it.start && pos < it.end;
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[p][i];
    norm_rotate<DIM>(y, fresh, A.k_norm != nullptr, w, A.eps, A.cos_t != nullptr, co[p], si[p]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (fresh) x[p][i] = y[i];
      amax = max(amax, abs_bits(x[p][i]));
    }
  }
  const Scale scale(wave_umax(amax));
  std::int8_t* dst = A.layer.k + b.at * (kBlk * DIM);
  if (lane == 0) A.layer.scales[2 * b.at] = scale.s;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int tok = p * kRows + lane / kLpr, pos = b.pos + tok;
    if (!chunk || tok >= kBlk) continue;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int d = side * kHalf + 8 * c;
      *reinterpret_cast<uint2*>(dst + (d / 16) * 256 + tok * 16 + d % 16) =
          make_uint2(codes4(&x[p][8 * side], scale), codes4(&x[p][8 * side + 4], scale));
    }
    if (pos >= it.keep && pos >= it.start && pos < it.end) {
      store8(open + tok * DIM + 8 * c, x[p]);
      store8(open + tok * DIM + kHalf + 8 * c, x[p] + 8);
    }
  }
}

// Dims that a lane has side by side where it takes whole dims (values, and
// both in read_kernel).
constexpr int dims_per_lane(int dim) { return dim % 256 == 0 ? 4 : dim % 128 == 0 ? 2 : 1; }
template <int N>
__device__ __forceinline__ void loadn(const float* p, float* x) {
  typedef float v __attribute__((ext_vector_type(N), aligned(4)));
  const v a = *reinterpret_cast<const v*>(p);
  if constexpr (N == 1) {
    x[0] = *p;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = a[i];
  }
}
template <int N>
__device__ __forceinline__ void storen(float* p, const float* x) {
  if constexpr (N == 1) {
    *p = x[0];
  } else {
    typedef float v __attribute__((ext_vector_type(N), aligned(4)));
    v a;
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = x[i];
    *reinterpret_cast<v*>(p) = a;
  }
}

// Values of one block and head: lanes take whole dims, so that a lane's 16
// codes are the 16 neighbouring bytes of its dim.
template <int DIM>
__device__ void append_values(const AppendArgs& A, const BlockItem& it, int h, const Block& b, int lane) {
  constexpr int kN = dims_per_lane(DIM), kGroups = (DIM + 64 * kN - 1) / (64 * kN);
  float* open = open_rows(A, it, DIM, h, b.pos, 1);
  float x[kGroups][kBlk][kN];
  std::uint32_t amax = 0;
#pragma unroll
  for (int n = 0; n < kGroups; ++n) {
    const int d = (n * 64 + lane) * kN;
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const int pos = b.pos + t;
#pragma unroll
      for (int i = 0; i < kN; ++i) x[n][t][i] = 0.0f;
      if (d < DIM && pos < it.end)
        loadn<kN>((pos < it.start ? open + t * DIM
                                  : A.val + static_cast<std::size_t>(it.row + (pos - it.start)) * A.v_stride +
                                        static_cast<std::size_t>(h) * DIM) +
                      d,
                  x[n][t]);
    }
  }
#pragma unroll
  for (int n = 0; n < kGroups; ++n)
#pragma unroll
    for (int t = 0; t < kBlk; ++t)
#pragma unroll
      for (int i = 0; i < kN; ++i) amax = max(amax, abs_bits(x[n][t][i]));
  const Scale scale(wave_umax(amax));
  std::int8_t* dst = A.layer.v + b.at * (kBlk * DIM);
  if (lane == 0) A.layer.scales[2 * b.at + 1] = scale.s;
#pragma unroll
  for (int n = 0; n < kGroups; ++n) {
    const int d = (n * 64 + lane) * kN;
    if (d >= DIM) continue;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      std::uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y[4] = {x[n][4 * j][i], x[n][4 * j + 1][i], x[n][4 * j + 2][i], x[n][4 * j + 3][i]};
        w[j] = codes4(y, scale);
      }
      *reinterpret_cast<uint4*>(dst + (d + i) * kBlk) = make_uint4(w[0], w[1], w[2], w[3]);
    }
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const int pos = b.pos + t;
      if (pos >= it.keep && pos >= it.start && pos < it.end) storen<kN>(open + t * DIM + d, x[n][t]);
    }
  }
}

// Units of work, one wavefront each: blocks' keys and values (item, head, k /
// v), then tokens' q (64 / lanes_per_row heads at a time, q_each times).  HBM
// bounds it: 14279 tokens of 32/8 heads of 128 with norms move 0.64 GB in 152
// us, 4.2 TB/s (a large copy: 4.7); a launch of its own for q took as long,
// and so did fewer registers.  One token: 4.5 us, the launch, its item, its
// rows and the stores.
template <int DIM>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs A) {
  constexpr int kLpr = lanes_per_row(DIM), kRows = 64 / kLpr, kHalf = DIM / 2;
  const int lane = threadIdx.x & 63;
  const int nblocks = A.nblocks >= 0 ? A.nblocks : A.v.counts->blocks;
  const int ntokens = A.ntokens >= 0 ? A.ntokens : A.v.counts->tokens;
  const unsigned kv_units = 2u * nblocks * A.g.kv_heads;
  const unsigned per_token = (A.g.heads + kRows * A.q_each - 1) / (kRows * A.q_each);
  const unsigned units = kv_units + (A.q != nullptr ? ntokens * per_token : 0u);
  for (unsigned u = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < units;
       u += gridDim.x * kWaves) {
    if (u < kv_units) {
      const unsigned pair = u >> 1, item = pair / A.g.kv_heads;
      const int h = static_cast<int>(pair - item * A.g.kv_heads);
      const BlockItem it = A.v.blocks[item];
      for (int then = 0; then < (it.then_pos >= 0 ? 2 : 1); ++then) {
        const Block b = block_of(A.g, it, h, then != 0);
        if ((u & 1) == 0)
          append_keys<DIM>(A, it, h, b, lane);
        else
          append_values<DIM>(A, it, h, b, lane);
      }
      continue;
    }
    const unsigned t = (u - kv_units) / per_token, part = u - kv_units - t * per_token;
    const int c = lane % kLpr;
    const bool chunk = DIM / 16 == kLpr || c < DIM / 16;
    float w[16] = {}, co[8] = {}, si[8] = {};
    if (A.q_norm != nullptr && chunk) {
      load8(A.q_norm + 8 * c, w);
      load8(A.q_norm + kHalf + 8 * c, w + 8);
    }
    if (A.cos_t != nullptr && chunk) {
      const std::size_t at = static_cast<std::size_t>(A.v.positions[t]) * kHalf + 8 * c;
      load8(A.cos_t + at, co);
      load8(A.sin_t + at, si);
    }
    for (int e = 0; e < A.q_each; ++e) {
      const int head = (static_cast<int>(part) * A.q_each + e) * kRows + lane / kLpr;
      const bool live = chunk && head < A.g.heads;
      float x[16] = {};
      const std::size_t off = static_cast<std::size_t>(head) * DIM + 8 * c;
      if (live) {
        const float* src = A.q + t * A.q_stride + off;
        load8(src, x);
        load8(src + kHalf, x + 8);
      }
      norm_rotate<DIM>(x, live, A.q_norm != nullptr, w, A.eps, A.cos_t != nullptr, co, si);
      if (live) {
        float* dst = A.q_out + t * A.q_out_stride + off;
        store8(dst, x);
        store8(dst + kHalf, x + 8);
      }
    }
  }
}

struct ReadArgs {
  View v;
  Geometry g;
  llmi_kv8_layer layer;
  float *k, *val;
  std::size_t k_stride, v_stride;
  int nblocks;
};

// One wavefront per block, head and k / v.  Keys: a lane four dims of a
// position; values: whole dims, as they are stored.  Either way a store
// instruction writes whole rows side by side.  HBM-bound, four fifths of it
// the fp32 rows: 40k positions of 8 heads of 128 in 92 us, 4.4 TB/s (152 us
// with 64-byte stores and the values' codes a byte at a time).
template <int DIM>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs A) {
  const int lane = threadIdx.x & 63;
  const int nblocks = A.nblocks >= 0 ? A.nblocks : A.v.counts->blocks;
  const unsigned units = 2u * nblocks * A.g.kv_heads;
  for (unsigned u = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < units;
       u += gridDim.x * kWaves) {
    const unsigned pair = u >> 1, item = pair / A.g.kv_heads;
    const int h = static_cast<int>(pair - item * A.g.kv_heads);
    const bool keys = (u & 1) == 0;
    float* out = keys ? A.k : A.val;
    if (out == nullptr) continue;
    const std::size_t stride = keys ? A.k_stride : A.v_stride;
    const BlockItem it = A.v.blocks[item];
    for (int then = 0; then < (it.then_pos >= 0 ? 2 : 1); ++then) {
      const Block b = block_of(A.g, it, h, then != 0);
      const float scale = A.layer.scales[2 * b.at + (keys ? 0 : 1)];
      const int lo = max(it.start - b.pos, 0), hi = min(it.end - b.pos, kBlk);  // rows of the block
      float* rows = out + (static_cast<std::int64_t>(it.row) + b.pos - it.start) * static_cast<std::int64_t>(stride) +
                    static_cast<std::int64_t>(h) * DIM;
      if (keys) {
        const std::int8_t* src = A.layer.k + b.at * (kBlk * DIM);
#pragma unroll
        for (int n = 0; n < DIM / 16; ++n) {
          const int e = n * 64 + lane, r = e / (DIM / 4), d = 4 * (e % (DIM / 4));
          if (r < lo || r >= hi) continue;
          const std::uint32_t c = *reinterpret_cast<const std::uint32_t*>(src + (d / 16) * 256 + r * 16 + d % 16);
          const float x[4] = {code_value(c, 0) * scale, code_value(c, 1) * scale, code_value(c, 2) * scale,
                              code_value(c, 3) * scale};
          storen<4>(rows + static_cast<std::int64_t>(r) * static_cast<std::int64_t>(stride) + d, x);
        }
      } else {
        constexpr int kN = dims_per_lane(DIM);
        const std::int8_t* src = A.layer.v + b.at * (kBlk * DIM);
#pragma unroll
        for (int n = 0; n < (DIM + 64 * kN - 1) / (64 * kN); ++n) {
          const int d = (n * 64 + lane) * kN;
          if (d >= DIM) continue;
          uint4 c[kN];
#pragma unroll
          for (int i = 0; i < kN; ++i) c[i] = *reinterpret_cast<const uint4*>(src + (d + i) * kBlk);
#pragma unroll
          for (int r = 0; r < kBlk; ++r) {
            if (r < lo || r >= hi) continue;
            float x[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) {
              const std::uint32_t four = r < 4 ? c[i].x : r < 8 ? c[i].y : r < 12 ? c[i].z : c[i].w;
              x[i] = code_value(four, r % 4) * scale;
            }
            storen<kN>(rows + static_cast<std::int64_t>(r) * static_cast<std::int64_t>(stride) + d, x);
          }
        }
      }
    }
  }
}

bool capturing(hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(s, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

// Workgroups for `units` wavefronts of work; a captured launch, which has
// room for any batch that its plan takes, fills the chip a few times and
// goes on from there.
unsigned grid_for(std::size_t units, bool captured) {
  return static_cast<unsigned>(std::min<std::size_t>(std::max<std::size_t>(ceil_div(units, kWaves), 1), captured ? 8192 : kMostGroups));
}

// fn(std::integral_constant<int, head_dim>) for the plan's head size.
template <typename Fn>
void with_dim(int dim, Fn&& fn) {
  switch (dim) {
    case 32: fn(std::integral_constant<int, 32>{}); break;
    case 64: fn(std::integral_constant<int, 64>{}); break;
    case 96: fn(std::integral_constant<int, 96>{}); break;
    case 128: fn(std::integral_constant<int, 128>{}); break;
    case 160: fn(std::integral_constant<int, 160>{}); break;
    case 192: fn(std::integral_constant<int, 192>{}); break;
    case 224: fn(std::integral_constant<int, 224>{}); break;
    default: fn(std::integral_constant<int, 256>{}); break;
  }
}

std::string check_layer(const llmi_kv8_layer* l, bool open) {
  if (l == nullptr) return "null layer";
  if (l->k == nullptr || l->v == nullptr || l->scales == nullptr || (open && l->open == nullptr))
    return "null pointer in the layer";
  const auto bits = reinterpret_cast<std::uintptr_t>(l->k) | reinterpret_cast<std::uintptr_t>(l->v) |
                    reinterpret_cast<std::uintptr_t>(l->scales) | reinterpret_cast<std::uintptr_t>(l->open);
  if (bits % 16 != 0) return "the layer's pointers must be 16-byte aligned";
  return {};
}

int require_set(const llmi_hip_kv8_plan* p, const char* what) {
  LLMI_REQUIRE(p != nullptr, std::string(what) + ": null plan");
  if (!p->set) return fail(LLMI_ERR_STATE, std::string(what) + ": no batch set (llmi_hip_kv8_plan_set)");
  return LLMI_OK;
}

}  // namespace
}  // namespace llmi_hip::kv8

using namespace llmi_hip;
using namespace llmi_hip::kv8;

llmi_hip_kv8_plan::~llmi_hip_kv8_plan() {
  if (copied != nullptr) (void)hipEventDestroy(copied);
  if (dev != nullptr) (void)hipFree(dev);
  if (parts != nullptr) (void)hipFree(parts);
  if (pinned != nullptr) (void)hipHostFree(pinned);
}

extern "C" {

int llmi_hip_kv8_sizes(const llmi_kv8_shape* shape, size_t* code_bytes, size_t* scale_floats, size_t* open_floats) {
  const std::string why = check_shape(shape);
  LLMI_REQUIRE(why.empty(), "kv8_sizes: " + why);
  const std::size_t head_pages = static_cast<std::size_t>(shape->pages) * shape->kv_heads;
  if (code_bytes != nullptr) *code_bytes = head_pages * shape->page_tokens * shape->head_dim;
  if (scale_floats != nullptr) *scale_floats = head_pages * (shape->page_tokens / kBlk) * 2;
  if (open_floats != nullptr)
    *open_floats = static_cast<std::size_t>(shape->slots) * shape->kv_heads * 4 * kBlk * shape->head_dim;
  return LLMI_OK;
}

int llmi_hip_kv8_check(const llmi_kv8_shape* shape, size_t seqs, const int32_t* slots, const int32_t* starts,
                       const int32_t* counts, const int32_t* tables, size_t table_stride) {
  std::string why = check_shape(shape);
  if (why.empty()) {
    try {
      Lists l;
      why = check_batch(*shape, seqs, slots, starts, counts, tables, table_stride, 0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFFF, &l);
      if (why.empty() && !l.writable) why = l.why_not;
    } catch (const std::bad_alloc&) {
      why = "out of host memory";
    }
  }
  LLMI_REQUIRE(why.empty(), "kv8_check: " + why);
  return LLMI_OK;
}

int llmi_hip_kv8_plan_create(const llmi_kv8_shape* shape, size_t max_seqs, size_t max_tokens, size_t max_pages,
                             llmi_hip_kv8_plan** plan) {
  LLMI_REQUIRE_INIT();
  LLMI_REQUIRE(plan != nullptr, "kv8_plan_create: null out-pointer");
  *plan = nullptr;
  const std::string why = check_shape(shape);
  LLMI_REQUIRE(why.empty(), "kv8_plan_create: " + why);
  LLMI_REQUIRE(max_seqs > 0 && max_seqs <= (1u << 20), "kv8_plan_create: max_seqs must be 1 .. 2^20");
  LLMI_REQUIRE(max_tokens > 0 && max_tokens <= (1u << 24), "kv8_plan_create: max_tokens must be 1 .. 2^24");
  if (max_pages == 0) max_pages = shape->pages;
  LLMI_REQUIRE(max_pages <= (1u << 30), "kv8_plan_create: max_pages must be at most 2^30");
  std::unique_ptr<llmi_hip_kv8_plan> p(new (std::nothrow) llmi_hip_kv8_plan);
  if (p == nullptr) return fail(LLMI_ERR_HIP, "kv8_plan_create: out of host memory");
  p->shape = *shape;
  p->max_seqs = max_seqs;
  p->max_tokens = max_tokens;
  p->max_pages = max_pages;
  p->g.heads = static_cast<int>(shape->heads);
  p->g.kv_heads = static_cast<int>(shape->kv_heads);
  p->g.group = p->g.heads / p->g.kv_heads;
  p->g.dim = static_cast<int>(shape->head_dim);
  p->g.page_blocks = static_cast<int>(shape->page_tokens) / kBlk;
  p->g.by_page = divisor(static_cast<std::uint32_t>(p->g.page_blocks));
  p->most = limits(*shape, max_seqs, max_tokens);
  // Kernels count rows of a key/value head and units of work (item and head) in 32 bits.
  LLMI_REQUIRE(max_tokens * (shape->heads / shape->kv_heads) <= (std::size_t{1} << 30),
               "kv8_plan_create: more than 2^30 rows (tokens x heads / kv_heads)");
  LLMI_REQUIRE(std::max({2 * p->most.blocks, p->most.few, p->most.many}) * shape->kv_heads <= 0x7FFFFFFFu,
               "kv8_plan_create: too many sequences and tokens for the heads");
  const auto take = [&](std::size_t bytes) {
    const std::size_t at = p->bytes;
    p->bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  (void)take(sizeof(Counts));
  p->off_positions = take(max_tokens * sizeof(std::int32_t));
  p->off_blocks = take(p->most.blocks * sizeof(BlockItem));
  p->off_few = take(p->most.few * sizeof(AttnItem));
  p->off_many = take(p->most.many * sizeof(AttnItem));
  p->off_join = take(p->most.join * sizeof(JoinItem));
  p->off_table = take(max_pages * sizeof(std::int32_t));
  LLMI_TRY_HIP(hipMalloc(reinterpret_cast<void**>(&p->dev), p->bytes));
  LLMI_TRY_HIP(hipHostMalloc(reinterpret_cast<void**>(&p->pinned), p->bytes, hipHostMallocDefault));
  const std::size_t rows = p->most.parts * shape->kv_heads * kSlotRows;
  LLMI_TRY_HIP(hipMalloc(reinterpret_cast<void**>(&p->parts), (rows + 1) * (shape->head_dim + 2) * sizeof(float)));
  LLMI_TRY_HIP(hipEventCreateWithFlags(&p->copied, hipEventDisableTiming));
  *plan = p.release();
  return LLMI_OK;
}

int llmi_hip_kv8_plan_set(llmi_hip_kv8_plan* p, size_t seqs, const int32_t* slots, const int32_t* starts,
                          const int32_t* counts, const int32_t* tables, size_t table_stride, void* stream) {
  LLMI_REQUIRE_INIT();
  LLMI_REQUIRE(p != nullptr, "kv8_plan_set: null plan");
  hipStream_t s = pick(stream);
  if (capturing(s)) return fail(LLMI_ERR_STATE, "kv8_plan_set: the stream is capturing a graph");
  try {
    Lists l;
    const std::string why = build(p->shape, seqs, slots, starts, counts, tables, table_stride, p->max_seqs,
                                  p->max_tokens, p->max_pages, &l);
    LLMI_REQUIRE(why.empty(), "kv8_plan_set: " + why);
    LLMI_REQUIRE(l.blocks.size() <= p->most.blocks && l.few.size() <= p->most.few &&
                     l.many.size() <= p->most.many && l.parts <= p->most.parts && l.join.size() <= p->most.join,
                 "kv8_plan_set: more work than the plan was created for");
    LLMI_REQUIRE(l.few_rows <= p->captured_few && (l.many.empty() || p->captured_many),
                 "kv8_plan_set: more tokens of a sequence than an attention of this plan was captured for");
    if (p->append_captured) {
      LLMI_REQUIRE(l.writable, "kv8_plan_set: an append of this plan was captured, and " + l.why_not);
      LLMI_REQUIRE(l.longest <= p->captured_positions,
                   "kv8_plan_set: more positions than the rotation tables of a captured append have");
    }
    LLMI_TRY_HIP(hipEventSynchronize(p->copied));
    const Counts c{static_cast<std::int32_t>(l.blocks.size()), static_cast<std::int32_t>(l.tokens),
                   static_cast<std::int32_t>(l.few.size()),
                   static_cast<std::int32_t>(l.many.size()), static_cast<std::int32_t>(l.join.size()),
                   l.join_rows, l.join_at};
    const auto put = [&](std::size_t at, const auto& v) {
      if (!v.empty()) std::memcpy(p->pinned + at, v.data(), v.size() * sizeof(v[0]));
    };
    std::memcpy(p->pinned, &c, sizeof c);
    put(p->off_positions, l.positions);
    put(p->off_blocks, l.blocks);
    put(p->off_few, l.few);
    put(p->off_many, l.many);
    put(p->off_join, l.join);
    put(p->off_table, l.table);
    const std::size_t used = p->off_table + l.table.size() * sizeof(std::int32_t);
    p->set = false;
    LLMI_TRY_HIP(hipMemcpyAsync(p->dev, p->pinned, used, hipMemcpyHostToDevice, s));
    LLMI_TRY_HIP(hipEventRecord(p->copied, s));
    p->lists = std::move(l);
    p->set = true;
  } catch (const std::bad_alloc&) {
    return fail(LLMI_ERR_HIP, "kv8_plan_set: out of host memory");
  }
  return LLMI_OK;
}

int llmi_hip_kv8_plan_free(llmi_hip_kv8_plan* p) {
  if (p == nullptr) return LLMI_OK;
  // Launches that use the plan may be queued on any stream.
  (void)hipDeviceSynchronize();
  delete p;
  return LLMI_OK;
}

int llmi_hip_kv8_append_dev(const llmi_hip_kv8_plan* p, const llmi_kv8_layer* layer, const float* q, size_t q_stride,
                            const float* k, size_t k_stride, const float* v, size_t v_stride, const float* q_norm,
                            const float* k_norm, float eps, const float* cos_t, const float* sin_t, size_t positions,
                            float* q_out, size_t q_out_stride, void* stream) {
  LLMI_REQUIRE_INIT();
  if (int rc = require_set(p, "kv8_append")) return rc;
  if (!p->lists.writable) return fail(LLMI_ERR_STATE, "kv8_append: " + p->lists.why_not);
  const std::string why = check_layer(layer, true);
  LLMI_REQUIRE(why.empty(), "kv8_append: " + why);
  const Geometry& g = p->g;
  const std::size_t qrow = static_cast<std::size_t>(g.heads) * g.dim, krow = static_cast<std::size_t>(g.kv_heads) * g.dim;
  LLMI_REQUIRE(k != nullptr && v != nullptr, "kv8_append: null k or v");
  LLMI_REQUIRE(k_stride >= krow && v_stride >= krow, "kv8_append: k_stride or v_stride shorter than a row");
  if (q != nullptr) {
    LLMI_REQUIRE(q_out != nullptr, "kv8_append: q without q_out");
    LLMI_REQUIRE(q_stride >= qrow && q_out_stride >= qrow, "kv8_append: q_stride or q_out_stride shorter than a row");
    LLMI_REQUIRE(q != q_out || q_stride == q_out_stride, "kv8_append: q in place needs equal strides");
  }
  LLMI_REQUIRE((q_norm != nullptr) == (k_norm != nullptr), "kv8_append: q_norm and k_norm go together");
  LLMI_REQUIRE(q_norm == nullptr || eps >= 0.0f, "kv8_append: eps must not be negative");
  LLMI_REQUIRE((cos_t != nullptr) == (sin_t != nullptr), "kv8_append: cos_t and sin_t go together");
  const bool captured = capturing(pick(stream));
  LLMI_REQUIRE(cos_t == nullptr || positions >= p->lists.longest,
               "kv8_append: the rotation tables have fewer positions than the batch");
  if (p->lists.tokens == 0 && !captured) return LLMI_OK;
  std::size_t blocks = p->lists.blocks.size(), tokens = p->lists.tokens;
  if (captured) {
    p->append_captured = true;
    if (cos_t != nullptr) p->captured_positions = std::min(p->captured_positions, positions);
    blocks = p->most.blocks;
    tokens = p->max_tokens;
  }
  // A wavefront takes one group of a token's heads; all of them, with the
  // norm's and the rotation's factors loaded once, where the groups would be
  // more than the chip holds wavefronts (8 of 4 SIMDs of 256 compute units).
  const std::size_t rows = 64 / static_cast<std::size_t>(lanes_per_row(g.dim));
  const std::size_t groups = ceil_div(static_cast<std::size_t>(g.heads), rows);
  const std::size_t each = tokens * groups > 8192 ? groups : 1;
  const std::size_t units = 2 * blocks * g.kv_heads + (q != nullptr ? tokens * ceil_div(groups, each) : 0);
  LLMI_REQUIRE(units <= 0x7FFFFFFFu, "kv8_append: too many tokens and heads");
  const AppendArgs a{p->view(), g, *layer, q, k, v, q_norm, k_norm, cos_t, sin_t, q_out, q_stride, k_stride, v_stride,
                     q_out_stride, eps, captured ? -1 : static_cast<int>(blocks),
                     captured ? -1 : static_cast<int>(tokens), static_cast<int>(each)};
  hipStream_t s = pick(stream);
  with_dim(g.dim, [&](auto dim) { append_kernel<dim><<<grid_for(units, captured), kThreads, 0, s>>>(a); });
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

int llmi_hip_kv8_attention_dev(const llmi_hip_kv8_plan* p, const llmi_kv8_layer* layer, const float* q,
                               size_t q_stride, float scale, float* out, size_t out_stride, void* stream) {
  LLMI_REQUIRE_INIT();
  if (int rc = require_set(p, "kv8_attention")) return rc;
  const std::string why = check_layer(layer, false);
  LLMI_REQUIRE(why.empty(), "kv8_attention: " + why);
  const std::size_t row = static_cast<std::size_t>(p->g.heads) * p->g.dim;
  LLMI_REQUIRE(q != nullptr && out != nullptr, "kv8_attention: null q or out");
  LLMI_REQUIRE(q_stride >= row && out_stride >= row, "kv8_attention: q_stride or out_stride shorter than a row");
  LLMI_REQUIRE(q != out || q_stride == out_stride, "kv8_attention: q in place needs equal strides");
  LLMI_REQUIRE(scale - scale == 0.0f, "kv8_attention: scale must be finite");
  const bool captured = capturing(pick(stream));
  if (p->lists.tokens == 0 && !captured) return LLMI_OK;
  return launch_attention(p, *layer, q, q_stride, scale, out, out_stride, pick(stream), captured);
}

int llmi_hip_kv8_read_dev(const llmi_hip_kv8_plan* p, const llmi_kv8_layer* layer, float* k, size_t k_stride, float* v,
                          size_t v_stride, void* stream) {
  LLMI_REQUIRE_INIT();
  if (int rc = require_set(p, "kv8_read")) return rc;
  const std::string why = check_layer(layer, false);
  LLMI_REQUIRE(why.empty(), "kv8_read: " + why);
  const std::size_t row = static_cast<std::size_t>(p->g.kv_heads) * p->g.dim;
  LLMI_REQUIRE((k == nullptr || k_stride >= row) && (v == nullptr || v_stride >= row),
               "kv8_read: k_stride or v_stride shorter than a row");
  const bool captured = capturing(pick(stream));
  if ((k == nullptr && v == nullptr) || (p->lists.tokens == 0 && !captured)) return LLMI_OK;
  const std::size_t blocks = captured ? p->most.blocks : p->lists.blocks.size();
  const ReadArgs a{p->view(), p->g, *layer, k, v, k_stride, v_stride, captured ? -1 : static_cast<int>(blocks)};
  hipStream_t s = pick(stream);
  with_dim(p->g.dim, [&](auto dim) {
    read_kernel<dim><<<grid_for(2 * blocks * p->g.kv_heads, captured), kThreads, 0, s>>>(a);
  });
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // extern "C"
