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
  std::size_t q_stride, out_stride;
  float scale;
  int ntokens;
};

__device__ __forceinline__ float wave_maxf(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_sumf(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One wavefront per token and head; 64 positions at a time, one pass with the
// running maximum and sum.
__global__ void __launch_bounds__(kThreads) attention_simple(AttnArgs A) {
  __shared__ float q_s[kWaves][256];
  __shared__ float p_s[kWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int dim = A.g.dim;
  const int ntokens = A.ntokens >= 0 ? A.ntokens : A.v.counts->tokens;
  const long rows = static_cast<long>(ntokens) * A.g.heads;
  for (long r = static_cast<long>(blockIdx.x) * kWaves + wave; r < rows; r += static_cast<long>(gridDim.x) * kWaves) {
    const long t = r / A.g.heads;
    const int h = static_cast<int>(r % A.g.heads), kvh = h / A.g.group;
    int lo = 0, hi = A.v.counts->seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (A.v.seqs[mid].row <= t)
        lo = mid;
      else
        hi = mid - 1;
    }
    const Seq s = A.v.seqs[lo];
    const int npos = s.start + static_cast<int>(t) - s.row + 1;
    for (int d = lane; d < dim; d += 64) q_s[wave][d] = A.q[t * A.q_stride + static_cast<std::size_t>(h) * dim + d];
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, l = 0.0f, o[4] = {};
    for (int base = 0; base < npos; base += 64) {
      const int pos = base + lane, block = pos / kBlk;
      float sc = -INFINITY, vs = 0.0f;
      std::size_t at = 0;
      if (pos < npos) {
        at = block_index(A.g, A.v.table, s, block, kvh);
        const std::int8_t* kp = A.k + at * A.g.block_bytes + (pos % kBlk) * 16;
        float acc = 0.0f;
        for (int g = 0; g < dim / 16; ++g)
          for (int j = 0; j < 16; ++j) acc = fmaf(q_s[wave][g * 16 + j], static_cast<float>(kp[g * 256 + j]), acc);
        sc = acc * A.scales[2 * at] * A.scale;
        vs = A.scales[2 * at + 1];
      }
      const float mx = fmaxf(m, wave_maxf(sc));
      const float keep = expf(m - mx);
      const float p = pos < npos ? expf(sc - mx) : 0.0f;
      l = l * keep + wave_sumf(p);
      m = mx;
      p_s[wave][lane] = pos < npos ? p * vs : 0.0f;
      __builtin_amdgcn_wave_barrier();
      const int nhere = min(64, npos - base);
      for (int n = 0; n * 64 < dim; ++n) {
        const int d = n * 64 + lane;
        float acc = 0.0f;
        for (int b = 0; b * kBlk < nhere; ++b) {
          const std::size_t bi = block_index(A.g, A.v.table, s, base / kBlk + b, kvh);
          if (d < dim) {
            const std::int8_t* vp = A.val + bi * A.g.block_bytes + d * 16;
            for (int j = 0; j < kBlk && b * kBlk + j < nhere; ++j)
              acc = fmaf(p_s[wave][b * kBlk + j], static_cast<float>(vp[j]), acc);
          }
        }
        o[n] = o[n] * keep + acc;
      }
      __builtin_amdgcn_wave_barrier();
    }
    for (int n = 0; n * 64 < dim; ++n) {
      const int d = n * 64 + lane;
      if (d < dim) A.out[t * A.out_stride + static_cast<std::size_t>(h) * dim + d] = o[n] / l;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

}  // namespace

int launch_attention(const llmi_hip_kv8_plan* p, const llmi_kv8_layer& layer, const float* q, std::size_t q_stride,
                     float scale, float* out, std::size_t out_stride, hipStream_t s, bool captured) {
  AttnArgs a{p->view(), p->g, layer.k, layer.v, layer.scales, q, out, q_stride, out_stride, scale,
             captured ? -1 : static_cast<int>(p->lists.tokens)};
  const std::size_t rows = (captured ? p->max_tokens : p->lists.tokens) * static_cast<std::size_t>(p->g.heads);
  attention_simple<<<static_cast<unsigned>(std::min<std::size_t>(ceil_div(rows, kWaves), 1u << 20)), kThreads, 0, s>>>(a);
  LLMI_TRY_HIP(hipGetLastError());
  return LLMI_OK;
}

}  // namespace llmi_hip::kv8
