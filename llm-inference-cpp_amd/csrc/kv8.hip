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
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<std::uint32_t>(__shfl_xor(static_cast<int>(v), o, 64)));
  return v;
}
// float(amax / 127) with one rounding; NaN and inf stay what they are.
__device__ __forceinline__ float block_scale(std::uint32_t amax) {
  return static_cast<float>(static_cast<double>(__uint_as_float(amax)) / 127.0);
}
// The nearest integer to x / scale, ties to even.  The quotient of two fp32
// numbers is either a tie, which 64 bits hold exactly, or at least 2^-26 of
// itself away from one: the 64-bit quotient rounds like the exact one.
__device__ __forceinline__ int code_of(float x, float scale, bool finite) {
  if (!finite) return 0;
  const double r = rint(static_cast<double>(x) / static_cast<double>(scale));
  return static_cast<int>(fmin(fmax(r, -127.0), 127.0));
}
__device__ __forceinline__ bool usable(float scale) { return scale > 0.0f && abs_bits(scale) < 0x7F800000u; }

// What a lane holds of one row of a head: dims 8c .. 8c+7 (a) and their
// rotation partners dim/2 + 8c ... (b).  `lpr` neighbouring lanes (a power
// of two, at least dim / 16) share a row.
// Norm and rotation in 64 bits, rounded once.
__device__ __forceinline__ void norm_rotate(float* a, float* b, bool live, int lpr, int c, int dim,
                                            const float* __restrict__ w, float eps, const float* __restrict__ cos_r,
                                            const float* __restrict__ sin_r) {
  double ss = 0.0;
  if (w != nullptr) {
    if (live) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss = fma(static_cast<double>(a[i]), static_cast<double>(a[i]), ss);
        ss = fma(static_cast<double>(b[i]), static_cast<double>(b[i]), ss);
      }
    }
    for (int o = 1; o < lpr; o <<= 1) ss += __shfl_xor(ss, o, 64);
  }
  if (!live) return;
  double r = 1.0;
  float wa[8], wb[8];
  if (w != nullptr) {
    r = 1.0 / sqrt(ss / dim + static_cast<double>(eps));
    load8(w + 8 * c, wa);
    load8(w + dim / 2 + 8 * c, wb);
  }
  float co[8], si[8];
  if (cos_r != nullptr) {
    load8(cos_r + 8 * c, co);
    load8(sin_r + 8 * c, si);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    double x = a[i], y = b[i];
    if (w != nullptr) {
      x = x * r * static_cast<double>(wa[i]);
      y = y * r * static_cast<double>(wb[i]);
    }
    if (cos_r != nullptr) {
      const double cc = co[i], sn = si[i];
      const double t = fma(x, cc, -(y * sn));
      y = fma(y, cc, x * sn);
      x = t;
    }
    a[i] = static_cast<float>(x);
    b[i] = static_cast<float>(y);
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
  int nappend, ntokens;  // -1: from v.counts (a captured launch)
};

__device__ __forceinline__ float* open_rows(const AppendArgs& A, const Seq& s, int h, int block, int which) {
  return A.layer.open + ((((static_cast<std::size_t>(s.slot) * A.g.kv_heads + h) * 2 + (block & 1)) * 2 + which) * 16) *
                            static_cast<std::size_t>(A.g.dim);
}

// Keys of one block and head: lanes take (position, 8-dim pair chunk).
template <int LPR>
__device__ void append_keys(const AppendArgs& A, const Seq& s, int h, int block, int last, int lane) {
  constexpr int kRows = 64 / LPR, kPasses = LPR < 4 ? 1 : LPR / 4;
  const int dim = A.g.dim, half = dim / 2, c = lane % LPR;
  float* open = open_rows(A, s, h, block, 0);
  float x[kPasses][16];
  std::uint32_t amax = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int tok = p * kRows + lane / LPR, pos = block * kBlk + tok;
    const bool chunk = c < dim / 16 && tok < kBlk;
    const bool fresh = chunk && pos >= s.start && pos < s.start + s.count;
    const bool held = chunk && pos < s.start;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[p][i] = 0.0f;
    if (fresh) {
      const float* src = A.k + static_cast<std::size_t>(s.row + (pos - s.start)) * A.k_stride +
                         static_cast<std::size_t>(h) * dim;
      load8(src + 8 * c, x[p]);
      load8(src + half + 8 * c, x[p] + 8);
    } else if (held) {
      load8(open + tok * dim + 8 * c, x[p]);
      load8(open + tok * dim + half + 8 * c, x[p] + 8);
    }
    const std::size_t t = static_cast<std::size_t>(fresh ? pos : 0) * half;
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[p][i];
    norm_rotate(y, y + 8, fresh, LPR, c, dim, A.k_norm, A.eps, A.cos_t != nullptr ? A.cos_t + t : nullptr,
                A.cos_t != nullptr ? A.sin_t + t : nullptr);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[p][i] = y[i];
      amax = max(amax, abs_bits(y[i]));
    }
  }
  amax = wave_umax(amax);
  const float scale = block_scale(amax);
  const bool ok = usable(scale);
  const std::size_t at = block_index(A.g, A.v.table, s, block, h);
  std::int8_t* dst = A.layer.k + at * A.g.block_bytes;
  if (lane == 0) A.layer.scales[2 * at] = scale;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int tok = p * kRows + lane / LPR, pos = block * kBlk + tok;
    if (c >= dim / 16 || tok >= kBlk) continue;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const int d = side * half + 8 * c;
      std::uint32_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[i] |= (static_cast<std::uint32_t>(code_of(x[p][8 * side + 4 * i + j], scale, ok)) & 0xFFu) << (8 * j);
      }
      *reinterpret_cast<uint2*>(dst + (d / 16) * 256 + tok * 16 + d % 16) = make_uint2(w[0], w[1]);
    }
    if (block >= last - 1 && pos >= s.start && pos < s.start + s.count) {
      store8(open + tok * dim + 8 * c, x[p]);
      store8(open + tok * dim + half + 8 * c, x[p] + 8);
    }
  }
}

// Values of one block and head: lanes take whole dims, so that a lane's 16
// codes are the 16 neighbouring bytes of its dim.
template <int LPR>
__device__ void append_values(const AppendArgs& A, const Seq& s, int h, int block, int last, int lane) {
  constexpr int kGroups = LPR < 4 ? 1 : LPR / 4;  // of 64 dims
  const int dim = A.g.dim;
  float* open = open_rows(A, s, h, block, 1);
  float x[kGroups][16];
  std::uint32_t amax = 0;
#pragma unroll
  for (int n = 0; n < kGroups; ++n) {
    const int d = n * 64 + lane;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const int pos = block * kBlk + t;
      x[n][t] = 0.0f;
      if (d < dim) {
        if (pos < s.start)
          x[n][t] = open[t * dim + d];
        else if (pos < s.start + s.count)
          x[n][t] = A.val[static_cast<std::size_t>(s.row + (pos - s.start)) * A.v_stride +
                          static_cast<std::size_t>(h) * dim + d];
      }
      amax = max(amax, abs_bits(x[n][t]));
    }
  }
  amax = wave_umax(amax);
  const float scale = block_scale(amax);
  const bool ok = usable(scale);
  const std::size_t at = block_index(A.g, A.v.table, s, block, h);
  std::int8_t* dst = A.layer.v + at * A.g.block_bytes;
  if (lane == 0) A.layer.scales[2 * at + 1] = scale;
#pragma unroll
  for (int n = 0; n < kGroups; ++n) {
    const int d = n * 64 + lane;
    if (d >= dim) continue;
    std::uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[i] |= (static_cast<std::uint32_t>(code_of(x[n][4 * i + j], scale, ok)) & 0xFFu) << (8 * j);
    }
    *reinterpret_cast<uint4*>(dst + d * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    if (block >= last - 1) {
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const int pos = block * kBlk + t;
        if (pos >= s.start && pos < s.start + s.count) open[t * dim + d] = x[n][t];
      }
    }
  }
}

// One wavefront per unit of work: the blocks' keys and values first (item,
// head, k / v), then q (64 / LPR rows of a token and head each).
template <int LPR>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs A) {
  const int lane = threadIdx.x & 63;
  const int nappend = A.nappend >= 0 ? A.nappend : A.v.counts->append;
  const int ntokens = A.ntokens >= 0 ? A.ntokens : A.v.counts->tokens;
  const long kv_units = 2L * nappend * A.g.kv_heads;
  const long q_rows = A.q != nullptr ? static_cast<long>(ntokens) * A.g.heads : 0;
  const long units = kv_units + (q_rows + 64 / LPR - 1) / (64 / LPR);
  for (long u = static_cast<long>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < units;
       u += static_cast<long>(gridDim.x) * kWaves) {
    if (u < kv_units) {
      const int which = u & 1;
      const int h = static_cast<int>((u >> 1) % A.g.kv_heads);
      const AppendItem it = A.v.append[(u >> 1) / A.g.kv_heads];
      const Seq s = A.v.seqs[it.seq];
      const int last = (s.start + s.count - 1) / kBlk;
      for (int block = it.block; block >= 0; block = block == it.block ? it.then : -1) {
        if (which == 0)
          append_keys<LPR>(A, s, h, block, last, lane);
        else
          append_values<LPR>(A, s, h, block, last, lane);
      }
      continue;
    }
    const long r = (u - kv_units) * (64 / LPR) + lane / LPR;
    const int c = lane % LPR, dim = A.g.dim, half = dim / 2;
    const bool live = r < q_rows && c < dim / 16;
    const long t = live ? r / A.g.heads : 0, h = live ? r % A.g.heads : 0;
    int pos = 0;
    if (A.cos_t != nullptr && live) {
      // The token's sequence: the last one that starts at or before row t.
      int lo = 0, hi = A.v.counts->seqs - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (A.v.seqs[mid].row <= t)
          lo = mid;
        else
          hi = mid - 1;
      }
      pos = A.v.seqs[lo].start + static_cast<int>(t) - A.v.seqs[lo].row;
    }
    float a[8] = {}, b[8] = {};
    if (live) {
      const float* src = A.q + static_cast<std::size_t>(t) * A.q_stride + static_cast<std::size_t>(h) * dim;
      load8(src + 8 * c, a);
      load8(src + half + 8 * c, b);
    }
    const std::size_t at = static_cast<std::size_t>(pos) * half;
    norm_rotate(a, b, live, LPR, c, dim, A.q_norm, A.eps, A.cos_t != nullptr ? A.cos_t + at : nullptr,
                A.cos_t != nullptr ? A.sin_t + at : nullptr);
    if (live) {
      float* dst = A.q_out + static_cast<std::size_t>(t) * A.q_out_stride + static_cast<std::size_t>(h) * dim;
      store8(dst + 8 * c, a);
      store8(dst + half + 8 * c, b);
    }
  }
}

struct ReadArgs {
  View v;
  Geometry g;
  llmi_kv8_layer layer;
  float *k, *val;
  std::size_t k_stride, v_stride;
  int nappend;
};

// One wavefront per block, head and k / v: 16 dims of 16 positions at a time,
// lane (position, 4 dims).
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs A) {
  const int lane = threadIdx.x & 63;
  const int nitems = A.nappend >= 0 ? A.nappend : A.v.counts->append;
  const long units = 2L * nitems * A.g.kv_heads;
  const int tok = lane >> 2, d4 = (lane & 3) * 4;
  for (long u = static_cast<long>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); u < units;
       u += static_cast<long>(gridDim.x) * kWaves) {
    const int which = u & 1;
    float* out = which == 0 ? A.k : A.val;
    if (out == nullptr) continue;
    const std::size_t stride = which == 0 ? A.k_stride : A.v_stride;
    const int h = static_cast<int>((u >> 1) % A.g.kv_heads);
    const AppendItem it = A.v.append[(u >> 1) / A.g.kv_heads];
    const Seq s = A.v.seqs[it.seq];
    for (int block = it.block; block >= 0; block = block == it.block ? it.then : -1) {
      const int pos = block * kBlk + tok;
      const std::size_t at = block_index(A.g, A.v.table, s, block, h);
      const std::int8_t* src = (which == 0 ? A.layer.k : A.layer.v) + at * A.g.block_bytes;
      const float scale = A.layer.scales[2 * at + which];
      if (pos < s.start || pos >= s.start + s.count) continue;
      float* row = out + static_cast<std::size_t>(s.row + (pos - s.start)) * stride +
                   static_cast<std::size_t>(h) * A.g.dim + d4;
      for (int g = 0; g < A.g.dim / 16; ++g) {
        std::int8_t c[4];
        if (which == 0) {
          __builtin_memcpy(c, src + g * 256 + tok * 16 + d4, 4);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) c[j] = src[g * 256 + (d4 + j) * 16 + tok];
        }
        *reinterpret_cast<f4*>(row + g * 16) =
            f4{static_cast<float>(c[0]) * scale, static_cast<float>(c[1]) * scale, static_cast<float>(c[2]) * scale,
               static_cast<float>(c[3]) * scale};
      }
    }
  }
}

bool capturing(hipStream_t s) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(s, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

unsigned grid_for(std::size_t units) {
  return static_cast<unsigned>(std::min<std::size_t>(std::max<std::size_t>(ceil_div(units, kWaves), 1), 1u << 20));
}

int lanes_per_row(int dim) { return dim <= 32 ? 2 : dim <= 64 ? 4 : dim <= 128 ? 8 : 16; }

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
      why = build(*shape, seqs, slots, starts, counts, tables, table_stride, 0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFFF, &l);
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
  p->g.block_bytes = static_cast<std::size_t>(kBlk) * shape->head_dim;
  p->g.by_page = divisor(static_cast<std::uint32_t>(p->g.page_blocks));
  p->most = limits(*shape, max_seqs, max_tokens);
  // Kernels count units of work (item and key/value head) in 32 bits.
  LLMI_REQUIRE(std::max({2 * p->most.append, p->most.few, p->most.many}) * shape->kv_heads <= 0x7FFFFFFFu,
               "kv8_plan_create: too many sequences and tokens for the heads");
  const auto take = [&](std::size_t bytes) {
    const std::size_t at = p->bytes;
    p->bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  (void)take(sizeof(Counts));
  p->off_seqs = take(max_seqs * sizeof(Seq));
  p->off_append = take(p->most.append * sizeof(AppendItem));
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
    LLMI_REQUIRE(l.append.size() <= p->most.append && l.few.size() <= p->most.few &&
                     l.many.size() <= p->most.many && l.parts <= p->most.parts && l.join.size() <= p->most.join,
                 "kv8_plan_set: more work than the plan was created for");
    if (p->append_captured) {
      LLMI_REQUIRE(l.writable, "kv8_plan_set: an append of this plan was captured, and " + l.why_not);
      LLMI_REQUIRE(l.longest <= p->captured_positions,
                   "kv8_plan_set: more positions than the rotation tables of a captured append have");
    }
    LLMI_TRY_HIP(hipEventSynchronize(p->copied));
    const Counts c{static_cast<std::int32_t>(l.append.size()), static_cast<std::int32_t>(l.tokens),
                   static_cast<std::int32_t>(l.seqs.size()), static_cast<std::int32_t>(l.few.size()),
                   static_cast<std::int32_t>(l.many.size()), static_cast<std::int32_t>(l.join.size())};
    const auto put = [&](std::size_t at, const auto& v) {
      if (!v.empty()) std::memcpy(p->pinned + at, v.data(), v.size() * sizeof(v[0]));
    };
    std::memcpy(p->pinned, &c, sizeof c);
    put(p->off_seqs, l.seqs);
    put(p->off_append, l.append);
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
  const int lpr = lanes_per_row(g.dim);
  AppendArgs a{p->view(), g, *layer, q, k, v, q_norm, k_norm, cos_t, sin_t, q_out, q_stride, k_stride, v_stride,
               q_out_stride, eps, static_cast<int>(p->lists.append.size()), static_cast<int>(p->lists.tokens)};
  std::size_t blocks = p->lists.append.size(), tokens = p->lists.tokens;
  if (captured) {
    p->append_captured = true;
    if (cos_t != nullptr) p->captured_positions = std::min(p->captured_positions, positions);
    a.nappend = a.ntokens = -1;
    blocks = p->most.append;
    tokens = p->max_tokens;
  }
  const std::size_t units = 2 * blocks * g.kv_heads + (q != nullptr ? ceil_div(tokens * g.heads * lpr, 64) : 0);
  const unsigned grid = grid_for(units);
  hipStream_t s = pick(stream);
  if (lpr == 2)
    append_kernel<2><<<grid, kThreads, 0, s>>>(a);
  else if (lpr == 4)
    append_kernel<4><<<grid, kThreads, 0, s>>>(a);
  else if (lpr == 8)
    append_kernel<8><<<grid, kThreads, 0, s>>>(a);
  else
    append_kernel<16><<<grid, kThreads, 0, s>>>(a);
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
  ReadArgs a{p->view(), p->g, *layer, k, v, k_stride, v_stride, static_cast<int>(p->lists.append.size())};
  std::size_t blocks = p->lists.append.size();
  if (captured) {
    a.nappend = -1;
    blocks = p->most.append;
  }
  read_kernel<<<grid_for(2 * blocks * p->g.kv_heads), kThreads, 0, pick(stream)>>>(a);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // extern "C"
