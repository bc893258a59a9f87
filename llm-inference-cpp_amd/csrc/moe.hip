// A layer of experts: the router, the experts' device layout, the sum of a
// token's experts, and the entry points.  Products of few slots are in
// moe_few.hip, the others in moe_products.hip, what these need before them
// (grouping, rows in two parts) in moe_prepare.hip.
#include <initializer_list>
#include <memory>
#include <new>

#include "moe_device.hpp"

namespace llmi_hip::moe {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// ------------------------------------------------------------------ router

// A logit as an unsigned integer of the same order, 0 for what is never
// chosen (-inf, NaN); +0 and -0 are equal.
__device__ __forceinline__ std::uint32_t rank_bits(float l) {
  if (!(l > -__builtin_inff())) return 0;
  const std::uint32_t b = __float_as_uint(l + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// One wavefront a token; lane l holds logits l, l + 64, ...  Every round takes
// the largest rank of all lanes, and of the logits that have it the first: the
// lowest place of a lane's, then the lowest lane.  The rounds are bound by their
// chains of rotations and ballots (8192 tokens, 8 of 128 experts: 5.8 us, memory
// alone 1; with exchanges through LDS in place of the rotations 12.4; 8 of 256
// 7.3, of 512 and 1024, which share a variant, 14.9 and 17.5); one to 64 tokens
// take a launch, 4.5 us.
template <int N>
__global__ void __launch_bounds__(kThreads) route_kernel(const float* __restrict__ logits, std::size_t stride,
                                                         std::size_t tokens, int experts, int top_k, int renormalise,
                                                         float scale, std::int32_t* __restrict__ ids,
                                                         float* __restrict__ weights) {
  const int lane = threadIdx.x & 63;
  for (std::size_t t = blockIdx.x * static_cast<std::size_t>(kWaves) + (threadIdx.x >> 6); t < tokens;
       t += static_cast<std::size_t>(gridDim.x) * kWaves) {
    std::uint32_t rank[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = lane + 64 * i;
      rank[i] = e < experts ? rank_bits(logits[t * stride + e]) : 0;
    }
    const auto most = [&] {
      std::uint32_t r = rank[0];
#pragma unroll
      for (int i = 1; i < N; ++i) r = max(r, rank[i]);
      return across(r, Larger{});
    };
    const auto logit = [](std::uint32_t r) { return __uint_as_float(r & 0x80000000u ? r & 0x7FFFFFFFu : ~r); };
    std::uint32_t best = most();
    const float top = logit(best);
    // exp(l - max); equal ones (both +inf among them) give 1.
    const auto weight = [&](std::uint32_t r) {
      const float l = logit(r);
      return l == top ? 1.0f : expf(l - top);
    };
    float total = 0.0f;
    if (!renormalise) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (rank[i] != 0) total += weight(rank[i]);
      total = __uint_as_float(across(__float_as_uint(total), [](std::uint32_t a, std::uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
      }));
    }
    // Choice j is kept by lane j (top_k <= 64).
    std::uint32_t mine = 0;
    int id = -1;
    for (int j = 0; j < top_k && best != 0; ++j) {
      bool found = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const std::uint64_t has = __ballot(rank[i] == best);
        if (found || has == 0) continue;
        found = true;
        const int first = __builtin_ctzll(has);
        if (lane == j) {
          mine = best;
          id = first + 64 * i;
        }
        if (lane == first) rank[i] = 0;
      }
      best = most();
    }
    const float w = id >= 0 ? weight(mine) : 0.0f;
    if (renormalise)  // lanes hold the choices: their sum, like that of all
      total = __uint_as_float(across(__float_as_uint(w), [](std::uint32_t a, std::uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
      }));
    if (lane < top_k) {
      ids[t * top_k + lane] = id;
      weights[t * top_k + lane] = id >= 0 ? scale * (w / total) : 0.0f;
    }
  }
}

// ------------------------------------------------------------------ layout

// The reference's planar codes of one or more experts -> the tiles' order, a
// thread for each lane of each step.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) lay_out(const std::uint8_t* __restrict__ data,
                                                    const float* __restrict__ scales, std::size_t count, int out, int in,
                                                    std::uint8_t* __restrict__ to) {
  const int blocks = (in + kBlock - 1) / kBlock, steps = (in + kStep - 1) / kStep;
  const int tiles = (out + kTile - 1) / kTile;
  const std::size_t row_bytes = TYPE == LLMI_TYPE_Q4_0 ? (in + 1) / 2 : in;
  const std::size_t units = count * tiles * steps * 64;
  for (std::size_t u = blockIdx.x * static_cast<std::size_t>(kThreads) + threadIdx.x; u < units;
       u += static_cast<std::size_t>(gridDim.x) * kThreads) {
    const int lane = static_cast<int>(u % 64);
    const std::size_t c = u / 64;  // (expert * tiles + tile) * steps + step
    const int step = static_cast<int>(c % steps), tile = static_cast<int>(c / steps % tiles);
    const std::size_t expert = c / steps / tiles;
    const int o = tile * kTile + lane % kTile;
    const std::uint8_t* row = data + (expert * out + static_cast<std::size_t>(o)) * row_bytes;
    std::uint32_t words[TYPE == LLMI_TYPE_Q4_0 ? 2 : 4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int k0 = step * kStep + b * kBlock + 8 * (lane / kTile);
      std::uint32_t code[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = k0 + i;
        const bool live = o < out && k < in;
        if constexpr (TYPE == LLMI_TYPE_Q4_0)
          code[i] = live ? (row[k / 2] >> (k % 2 * 4)) & 15u : 8u;
        else
          code[i] = live ? (row[k] ^ 0x80u) : 0x80u;
      }
      if constexpr (TYPE == LLMI_TYPE_Q4_0) {
        words[b] = code[0] | code[2] << 4 | code[4] << 8 | code[6] << 12 | code[1] << 16 | code[3] << 20 |
                   code[5] << 24 | code[7] << 28;
      } else {
        words[2 * b] = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        words[2 * b + 1] = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
      }
    }
    std::uint8_t* const at = to + c * step_bytes(TYPE);
    if constexpr (TYPE == LLMI_TYPE_Q4_0) *reinterpret_cast<uint2*>(at + lane * 8) = uint2{words[0], words[1]};
    else *reinterpret_cast<uint4*>(at + lane * 16) = uint4{words[0], words[1], words[2], words[3]};
    if (lane < static_cast<int>(kStepScales)) {  // output lane / 2, block lane % 2
      const int so = tile * kTile + lane / 2, sb = step * 2 + lane % 2;
      reinterpret_cast<float*>(at + code_bytes(TYPE))[lane] = so < out && sb < blocks ? scales[(expert * out + static_cast<std::size_t>(so)) * blocks + sb] : 0.0f;
    }
  }
}

unsigned grid_for(std::size_t units, std::size_t each) {
  return static_cast<unsigned>(std::min<std::size_t>(std::max<std::size_t>(ceil_div(units, each), 1), kMostGroups));
}

int launch_lay_out(const std::uint8_t* data, const float* scales, const Shape& s, std::uint8_t* to, hipStream_t st) {
  const unsigned grid = grid_for(s.count * s.tiles() * s.steps() * 64, kThreads);
  const int out = static_cast<int>(s.out), in = static_cast<int>(s.in);
  if (s.type == LLMI_TYPE_Q4_0)
    lay_out<LLMI_TYPE_Q4_0><<<grid, kThreads, 0, st>>>(data, scales, s.count, out, in, to);
  else
    lay_out<LLMI_TYPE_Q8_0><<<grid, kThreads, 0, st>>>(data, scales, s.count, out, in, to);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

int new_experts(const Shape& s, std::unique_ptr<llmi_hip_experts>* to) {
  to->reset(new (std::nothrow) llmi_hip_experts);
  if (*to == nullptr) return fail(LLMI_ERR_HIP, "experts: out of host memory");
  (*to)->shape = s;
  LLMI_TRY_HIP(hipMalloc(reinterpret_cast<void**>(&(*to)->steps), s.bytes()));
  return LLMI_OK;
}

// ------------------------------------------------------- a token's sum

// y[t] = residual[t] + sum over j of weights[t][j] * sums[t * top_k + j], in
// the order of j; 4 results a thread.  Bound by memory: 4096 tokens of 8 experts
// and 2048 results 57 us, 5.3 TB/s (choice after choice 63); 64 tokens 4.9 us, a
// launch and two loads in a row.
__global__ void __launch_bounds__(kThreads) sum_kernel(const float* __restrict__ sums,
                                                       const std::int32_t* __restrict__ ids,
                                                       const float* __restrict__ weights, std::size_t tokens, int top_k,
                                                       int experts, int width, const float* residual,
                                                       std::size_t r_stride, float* y, std::size_t y_stride) {
  const std::size_t quads = (static_cast<std::size_t>(width) + 3) / 4;
  const std::size_t units = tokens * quads;
  for (std::size_t u = blockIdx.x * static_cast<std::size_t>(kThreads) + threadIdx.x; u < units;
       u += static_cast<std::size_t>(gridDim.x) * kThreads) {
    const std::size_t t = u / quads;
    const int o = static_cast<int>(u % quads) * 4;
    const bool whole = o + 4 <= width;
    const auto load = [&](const float* p) {
      if (whole) return *reinterpret_cast<const f4*>(p);
      f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int i = 0; i < width - o; ++i) v[i] = p[i];
      return v;
    };
    f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    // Several choices at a time, all asked for before one is looked at; the row
    // of a choice that has no expert is there, but means nothing.
    constexpr int kAtOnce = 8;
    for (int j0 = 0; j0 < top_k; j0 += kAtOnce) {
      std::int32_t e[kAtOnce];
      float w[kAtOnce];
      f4 v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (j0 + i >= top_k) break;
        const std::size_t slot = t * top_k + j0 + i;
        e[i] = ids[slot];
        w[i] = weights[slot];
        v[i] = load(sums + slot * width + o);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (j0 + i >= top_k) break;
        if (e[i] < 0 || e[i] >= experts) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(w[i], v[i][c], acc[c]);
      }
    }
    if (residual != nullptr) {
      const f4 r = load(residual + t * r_stride + o);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = r[i] + acc[i];
    }
    float* to = y + t * y_stride + o;
    if (whole)
      *reinterpret_cast<f4*>(to) = acc;
    else
      for (int i = 0; i < width - o; ++i) to[i] = acc[i];
  }
}

std::string check_workspace(const void* work, std::size_t bytes, std::size_t need) {
  if (work == nullptr) return "null workspace";
  if (reinterpret_cast<std::uintptr_t>(work) % 16 != 0) return "the workspace must be 16-byte aligned";
  if (bytes < need) return "workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed";
  return {};
}
// Whether a region that the call writes meets any of the others.
std::string check_apart(const char* name, const Region& written, std::initializer_list<Region> others) {
  for (const Region& r : others)
    if (overlap(written, r)) return std::string(name) + " overlaps another operand";
  return {};
}
Groups groups_at(std::uint8_t* work, const Grouping& g, std::size_t rows0, std::size_t rows1) {
  return {reinterpret_cast<std::int32_t*>(work + g.counts),
          reinterpret_cast<std::int32_t*>(work + g.order),
          {reinterpret_cast<RowTile*>(work + g.tiles[0]), reinterpret_cast<RowTile*>(work + g.tiles[1])},
          {static_cast<int>(rows0), static_cast<int>(rows1)},
          reinterpret_cast<std::int32_t*>(work + g.hist)};
}
SplitRows parts_at(std::uint8_t* work, const Parts& p) {
  return {reinterpret_cast<_Float16*>(work + p.values), reinterpret_cast<float*>(work + p.factors)};
}

}  // namespace

}  // namespace llmi_hip::moe

using namespace llmi_hip;
using namespace llmi_hip::moe;

extern "C" {

int llmi_hip_moe_route_dev(const float* logits, size_t stride, size_t tokens, size_t experts, size_t top_k,
                           int renormalise, float scale, int32_t* ids, float* weights, void* stream) {
  LLMI_REQUIRE_INIT();
  const std::string why = check_route(tokens, experts, top_k, stride);
  LLMI_REQUIRE(why.empty(), "moe_route: " + why);
  LLMI_REQUIRE(scale - scale == 0.0f, "moe_route: scale must be finite");
  if (tokens == 0) return LLMI_OK;
  LLMI_REQUIRE(logits != nullptr && ids != nullptr && weights != nullptr, "moe_route: null pointer");
  const Region r_logits = Region::matrix(logits, tokens, experts, stride), r_ids = Region::whole(ids, tokens * top_k * sizeof(*ids)),
               r_weights = Region::whole(weights, tokens * top_k * sizeof(*weights));
  std::string meets = check_apart("ids", r_ids, {r_logits, r_weights});
  if (meets.empty()) meets = check_apart("weights", r_weights, {r_logits});
  LLMI_REQUIRE(meets.empty(), "moe_route: " + meets);
  hipStream_t s = pick(stream);
  const unsigned grid = grid_for(tokens, kWaves);
  const int e = static_cast<int>(experts), k = static_cast<int>(top_k);
  const auto run = [&](auto n) {
    route_kernel<n><<<grid, kThreads, 0, s>>>(logits, stride, tokens, e, k, renormalise, scale, ids, weights);
  };
  if (experts <= 64) run(std::integral_constant<int, 1>{});
  else if (experts <= 128) run(std::integral_constant<int, 2>{});
  else if (experts <= 256) run(std::integral_constant<int, 4>{});
  else run(std::integral_constant<int, 16>{});
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

int llmi_hip_experts_upload_dev(const uint8_t* data, const float* scales, size_t count, size_t out, size_t in, int type,
                                llmi_hip_experts** experts) {
  LLMI_REQUIRE_INIT();
  LLMI_REQUIRE(experts != nullptr, "experts_upload: null out-pointer");
  *experts = nullptr;
  Shape s;
  s.type = type;
  s.count = count;
  s.out = out;
  s.in = in;
  const std::string why = check_shape(s);
  LLMI_REQUIRE(why.empty(), "experts_upload: " + why);
  LLMI_REQUIRE(data != nullptr && scales != nullptr, "experts_upload: null pointer");
  std::unique_ptr<llmi_hip_experts> e;
  if (int rc = new_experts(s, &e)) return rc;
  if (int rc = launch_lay_out(data, scales, s, e->steps, library_stream())) return rc;
  LLMI_TRY_HIP(hipStreamSynchronize(library_stream()));
  *experts = e.release();
  return LLMI_OK;
}

int llmi_hip_experts_create(const llmi_hip_weight* const* weights, size_t count, llmi_hip_experts** experts) {
  LLMI_REQUIRE_INIT();
  LLMI_REQUIRE(experts != nullptr, "experts_create: null out-pointer");
  *experts = nullptr;
  LLMI_REQUIRE(weights != nullptr && count > 0 && weights[0] != nullptr, "experts_create: null weight");
  Shape s;
  s.type = weights[0]->m.type;
  s.count = count;
  s.out = weights[0]->m.out;
  s.in = weights[0]->m.in;
  const std::string why = check_shape(s);
  LLMI_REQUIRE(why.empty(), "experts_create: " + why);
  for (size_t i = 1; i < count; ++i) {
    LLMI_REQUIRE(weights[i] != nullptr, "experts_create: null weight");
    const DeviceMatrix& m = weights[i]->m;
    LLMI_REQUIRE(m.type == s.type && m.out == s.out && m.in == s.in, "experts_create: weights of different types or shapes");
  }
  std::unique_ptr<llmi_hip_experts> e;
  if (int rc = new_experts(s, &e)) return rc;
  // One expert after the other through its planar form.
  const std::size_t nd = s.out * row_bytes(s.in, s.type), at_scales = (nd + 255) / 256 * 256;
  std::uint8_t* planar = nullptr;
  LLMI_TRY_HIP(hipMalloc(reinterpret_cast<void**>(&planar), at_scales + s.out * s.blocks() * sizeof(float)));
  float* planar_scales = reinterpret_cast<float*>(planar + at_scales);
  Shape one = s;
  one.count = 1;
  int rc = LLMI_OK;
  for (size_t i = 0; i < count && rc == LLMI_OK; ++i) {
    rc = launch_relayout_to_planar(weights[i]->m, planar, planar_scales, library_stream());
    if (rc == LLMI_OK)
      rc = launch_lay_out(planar, planar_scales, one, e->steps + i * one.bytes(), library_stream());
  }
  const hipError_t end = hipStreamSynchronize(library_stream());
  (void)hipFree(planar);
  if (rc != LLMI_OK) return rc;
  LLMI_TRY_HIP(end);
  *experts = e.release();
  return LLMI_OK;
}

int llmi_hip_experts_free(llmi_hip_experts* experts) {
  if (experts == nullptr) return LLMI_OK;
  (void)hipDeviceSynchronize();  // launches that use them may be queued on any stream
  delete experts;
  return LLMI_OK;
}

int llmi_hip_moe_matmul_bytes(const llmi_hip_experts* experts, size_t slots, size_t per_row, size_t* bytes) {
  LLMI_REQUIRE(experts != nullptr && bytes != nullptr, "moe_matmul_bytes: null pointer");
  const std::string why = check_matmul(slots, per_row);
  LLMI_REQUIRE(why.empty(), "moe_matmul_bytes: " + why);
  *bytes = MatmulLayout(experts->shape, slots, per_row).all.bytes;
  return LLMI_OK;
}

int llmi_hip_moe_matmul_dev(const llmi_hip_experts* experts, const int32_t* ids, size_t slots, size_t per_row,
                            const float* x, size_t x_stride, float* y, size_t y_stride, void* work, size_t work_bytes,
                            void* stream) {
  LLMI_REQUIRE_INIT();
  LLMI_REQUIRE(experts != nullptr, "moe_matmul: null experts");
  const Shape& sh = experts->shape;
  std::string why = check_matmul(slots, per_row);
  LLMI_REQUIRE(why.empty(), "moe_matmul: " + why);
  LLMI_REQUIRE(x_stride >= sh.in && y_stride >= sh.out, "moe_matmul: x_stride or y_stride shorter than a row");
  if (slots == 0) return LLMI_OK;
  LLMI_REQUIRE(ids != nullptr && x != nullptr && y != nullptr, "moe_matmul: null pointer");
  LLMI_REQUIRE(x != y, "moe_matmul: y must not be x");
  const MatmulLayout l(sh, slots, per_row);
  why = check_workspace(work, work_bytes, l.all.bytes);
  LLMI_REQUIRE(why.empty(), "moe_matmul: " + why);
  const Region r_ids = Region::whole(ids, slots * sizeof(*ids)), r_x = Region::matrix(x, rows_of(slots, per_row), sh.in, x_stride),
               r_y = Region::matrix(y, slots, sh.out, y_stride);
  why = check_apart("y", r_y, {r_ids, r_x});
  if (why.empty()) why = check_apart("the workspace", Region::whole(work, l.all.bytes), {r_ids, r_x, r_y});
  LLMI_REQUIRE(why.empty(), "moe_matmul: " + why);
  hipStream_t s = pick(stream);
  per_row = std::min(per_row, slots);  // more than all slots mean the same row; the kernels have 32 bits for it
  if (few_matmul(sh, slots, per_row))
    return launch_few(FewProduct{sh, experts->view(), {}, ids, slots, per_row, x, x_stride, y, y_stride, {}}, s);
  auto* w = static_cast<std::uint8_t*>(work);
  const std::size_t rows = pick_rows(sh, slots, false);
  const Groups g = groups_at(w, l.group, rows, rows);
  const SplitRows xs = parts_at(w, l.x);
  const RowSource src{x, x_stride, sh.in, sh.steps(), static_cast<std::uint32_t>(per_row)};
  if (int rc = launch_prepare(ids, slots, sh.count, g, src, xs, s)) return rc;
  return launch_product(Product{sh, experts->view(), {}, xs, g, 0, slots, per_row, false, y, y_stride, {}, 0, false}, s);
}

int llmi_hip_moe_mlp_bytes(const llmi_hip_experts* gate, const llmi_hip_experts* down, size_t tokens, size_t top_k,
                           size_t* bytes) {
  LLMI_REQUIRE(gate != nullptr && down != nullptr && bytes != nullptr, "moe_mlp_bytes: null pointer");
  const std::string why = check_mlp(gate->shape, down->shape, tokens, top_k);
  LLMI_REQUIRE(why.empty(), "moe_mlp_bytes: " + why);
  *bytes = MlpLayout(gate->shape, down->shape, tokens, top_k).all.bytes;
  return LLMI_OK;
}

int llmi_hip_moe_mlp_dev(const llmi_hip_experts* gate, const llmi_hip_experts* up, const llmi_hip_experts* down,
                         const int32_t* ids, const float* weights, size_t tokens, size_t top_k, const float* x,
                         size_t x_stride, const float* residual, size_t residual_stride, float* y, size_t y_stride,
                         void* work, size_t work_bytes, void* stream) {
  LLMI_REQUIRE_INIT();
  LLMI_REQUIRE(gate != nullptr && up != nullptr && down != nullptr, "moe_mlp: null experts");
  const Shape &gs = gate->shape, &us = up->shape, &ds = down->shape;
  LLMI_REQUIRE(gs.type == us.type && gs.count == us.count && gs.out == us.out && gs.in == us.in,
               "moe_mlp: gate and up of different types or shapes");
  std::string why = check_mlp(gs, ds, tokens, top_k);
  LLMI_REQUIRE(why.empty(), "moe_mlp: " + why);
  LLMI_REQUIRE(x_stride >= gs.in && y_stride >= ds.out, "moe_mlp: x_stride or y_stride shorter than a row");
  LLMI_REQUIRE(residual == nullptr || residual_stride >= ds.out, "moe_mlp: residual_stride shorter than a row");
  LLMI_REQUIRE(residual != y || residual == nullptr || residual_stride == y_stride, "moe_mlp: residual in place needs equal strides");
  if (tokens == 0) return LLMI_OK;
  LLMI_REQUIRE(ids != nullptr && weights != nullptr && x != nullptr && y != nullptr, "moe_mlp: null pointer");
  const MlpLayout l(gs, ds, tokens, top_k);
  why = check_workspace(work, work_bytes, l.all.bytes);
  LLMI_REQUIRE(why.empty(), "moe_mlp: " + why);
  const std::size_t slots = tokens * top_k;
  // x may lie anywhere beside y: no launch that writes y reads it.
  const Region r_ids = Region::whole(ids, slots * sizeof(*ids)), r_weights = Region::whole(weights, slots * sizeof(*weights)),
               r_x = Region::matrix(x, tokens, gs.in, x_stride), r_y = Region::matrix(y, tokens, ds.out, y_stride),
               r_residual = Region::matrix(residual, residual == nullptr ? 0 : tokens, ds.out, residual_stride);
  why = check_apart("y", r_y, {r_ids, r_weights});
  if (why.empty() && residual != y) why = check_apart("y", r_y, {r_residual});
  if (why.empty()) why = check_apart("the workspace", Region::whole(work, l.all.bytes), {r_ids, r_weights, r_x, r_y, r_residual});
  LLMI_REQUIRE(why.empty(), "moe_mlp: " + why);
  hipStream_t s = pick(stream);
  auto* w = static_cast<std::uint8_t*>(work);
  const MlpRows rows = pick_mlp_rows(gs, ds, slots);
  const Groups g = groups_at(w, l.group, rows.first, rows.second);
  const SplitRows xs = parts_at(w, l.x), hs = parts_at(w, l.h_parts);
  auto* h = reinterpret_cast<float*>(w + l.h);
  auto* sums = reinterpret_cast<float*>(w + l.sums);
  if (few_mlp(tokens, top_k)) {
    const FewParts parts{reinterpret_cast<_Float16*>(w + l.h), reinterpret_cast<float*>(w + l.h + l.few_factors),
                         static_cast<int>(few_blocks(ds))};
    if (int rc = launch_few(FewProduct{gs, gate->view(), up->view(), ids, slots, top_k, x, x_stride, nullptr, 0, parts}, s)) return rc;
    return launch_few_sum(FewSum{ds, down->view(), ids, weights, tokens, top_k, parts, residual, residual_stride, y, y_stride, sums}, s);
  }
  const RowSource src{x, x_stride, gs.in, gs.steps(), static_cast<std::uint32_t>(top_k)}, h_src{h, ds.in, ds.in, ds.steps(), 0};
  if (int rc = launch_prepare(ids, slots, gs.count, g, src, xs, s)) return rc;
  // The results between the products: for short work in its row tiles at once,
  // else as fp32 rows, whose parts need each whole row's largest.
  const bool tiled = g.rows[1] <= static_cast<int>(kMostShortRows);
  Product first{gs, gate->view(), up->view(), xs, g, 0, slots, top_k, true, h, gs.out, {}, 0, false};
  if (tiled) {
    first.y = nullptr;
    first.h = hs;
    first.h_steps = ds.steps();
  }
  if (int rc = launch_product(first, s)) return rc;
  if (!tiled)
    if (int rc = launch_split(h_src, slots, g.counts, hs, s)) return rc;
  if (int rc = launch_product(Product{ds, down->view(), {}, hs, g, 1, slots, 0, false, sums, ds.out, {}, 0, tiled}, s)) return rc;
  sum_kernel<<<grid_for(tokens * ceil_div(ds.out, 4), kThreads), kThreads, 0, s>>>(
      sums, ids, weights, tokens, static_cast<int>(top_k), static_cast<int>(ds.count), static_cast<int>(ds.out), residual,
      residual_stride, y, y_stride);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // extern "C"
