// Device code that the experts' product kernels share: codes to fp16, a
// lane's weights of a chunk, and rows in two fp16 parts.
#pragma once

#include <type_traits>

#include "moe.hpp"

namespace llmi_hip::moe {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));  // rows may start at any float
typedef std::uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A constant in a vector register: v_and_or_b32 takes one scalar operand only.
__device__ __forceinline__ std::uint32_t magic() {
  std::uint32_t m;
  asm("v_mov_b32 %0, 0x64006400" : "=v"(m));
  return m;
}
__device__ __forceinline__ f16x2 as_f16(std::uint32_t v) { return __builtin_bit_cast(f16x2, v); }

// Eight 4-bit codes of a dword: nibbles moved into fp16 mantissas give 1024 +
// n or 1024 + 16 n, from which n - 8 is exact in one operation.
__device__ __forceinline__ f16x8 codes_q4(std::uint32_t w) {
  const f16x2 one = {static_cast<_Float16>(-1032.0f), static_cast<_Float16>(-1032.0f)};
  const f16x2 by = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
  const f16x2 off = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
  const std::uint32_t v = w >> 8, k = magic();
  const f16x2 a = as_f16((w & 0x000F000Fu) | k) + one;
  const f16x2 b = __builtin_elementwise_fma(as_f16((w & 0x00F000F0u) | k), by, off);
  const f16x2 c = as_f16((v & 0x000F000Fu) | k) + one;
  const f16x2 d = __builtin_elementwise_fma(as_f16((v & 0x00F000F0u) | k), by, off);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// Eight codes + 128 of two dwords, likewise.
__device__ __forceinline__ f16x8 codes_q8(std::uint32_t lo, std::uint32_t hi) {
  const f16x2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  const auto two = [&](std::uint32_t w, std::uint32_t sel) {
    return as_f16(__builtin_amdgcn_perm(0x64646464u, w, sel)) + off;
  };
  const f16x2 a = two(lo, 0x04010400u), b = two(lo, 0x04030402u), c = two(hi, 0x04010400u), d = two(hi, 0x04030402u);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

typedef const __attribute__((address_space(1))) std::uint8_t* GlobalBytes;

// A lane's offsets, opaque at each use: addresses stay a scalar base and a
// 32-bit offset (hoisted out of a loop, the compiler would make them 64 bits).
struct LaneAt {
  std::uint32_t by8, by16, scale;
  __device__ __forceinline__ explicit LaneAt(int lane)
      : by8(static_cast<std::uint32_t>(lane) * 8), by16(static_cast<std::uint32_t>(lane) * 16),
        scale(static_cast<std::uint32_t>(lane % kTile) * 8) {}
  __device__ __forceinline__ void here() { asm volatile("" : "+v"(by8), "+v"(by16), "+v"(scale)); }
};

// Where the steps of an expert's tile are; tile: expert * tiles + tile.
template <int TYPE>
__device__ __forceinline__ GlobalBytes tile_at(const Matrices& m, std::size_t tile, int steps) {
  return (GlobalBytes)m.steps + tile * steps * step_bytes(TYPE);
}

// A lane's weights of one tile and step.
template <int TYPE>
struct Weights {
  typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  std::uint32_t c[TYPE == LLMI_TYPE_Q4_0 ? 2 : 4];
  float s[2];
  // Step `step` of a tile whose steps are at `from`, common to the wavefront.
  __device__ __forceinline__ void load(GlobalBytes from, int step, LaneAt& lane) {
    lane.here();
    const std::uint32_t code_at = TYPE == LLMI_TYPE_Q4_0 ? lane.by8 : lane.by16;
    const GlobalBytes at = from + static_cast<std::uint32_t>(step) * static_cast<std::uint32_t>(step_bytes(TYPE));  // at most 2^12 steps
    if constexpr (TYPE == LLMI_TYPE_Q4_0) {
      const u32x2 v = *(const __attribute__((address_space(1))) u32x2*)(at + code_at);
      c[0] = v[0];
      c[1] = v[1];
    } else {
      const u32x4 v = *(const __attribute__((address_space(1))) u32x4*)(at + code_at);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = v[i];
    }
    const f32x2 v = *(const __attribute__((address_space(1))) f32x2*)(at + code_bytes(TYPE) + lane.scale);
    s[0] = v[0];
    s[1] = v[1];
  }
  __device__ __forceinline__ f16x8 codes(int b) const {
    if constexpr (TYPE == LLMI_TYPE_Q4_0) return codes_q4(c[b]);
    else return codes_q8(c[2 * b], c[2 * b + 1]);
  }
};

// Orders the lanes' LDS exchange of one wavefront for the compiler.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// |x| as an unsigned integer, 0 for inf and NaN: the largest finite one.
__device__ __forceinline__ std::uint32_t finite_bits(float x) {
  const std::uint32_t b = __float_as_uint(x) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? b : 0;
}
// The power of two that brings a largest |x| of these bits to 2^14 .. 2^15,
// and its inverse; the exponent is held at -112 or more, so that both are
// normal numbers.
struct Factor {
  float up, back;
  __device__ __forceinline__ explicit Factor(std::uint32_t top) {
    const int e = max(static_cast<int>(top >> 23) - 127, -112);
    up = __uint_as_float(static_cast<std::uint32_t>(127 + 14 - e) << 23);
    back = __uint_as_float(static_cast<std::uint32_t>(127 - 14 + e) << 23);
  }
};
// high + low = a up to 2^-22 of it (2^-25 below 2^-3); inf and NaN stay in
// the high part.
__device__ __forceinline__ void two_parts(float a, _Float16& high, _Float16& low) {
  high = static_cast<_Float16>(a);
  low = fabsf(a) < __builtin_inff() ? static_cast<_Float16>(a - static_cast<float>(high)) : static_cast<_Float16>(0.0f);
}

// fn over a 32-bit value of 16 lanes (a row of them), in all: rotations.
template <typename Fn>
__device__ __forceinline__ std::uint32_t across_row(std::uint32_t v, Fn&& fn) {
  const auto ror = [](std::uint32_t x, auto by) {
    return static_cast<std::uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x120 + decltype(by)::value, 0xF, 0xF, false));
  };
  v = fn(v, ror(v, std::integral_constant<int, 8>{}));
  v = fn(v, ror(v, std::integral_constant<int, 4>{}));
  v = fn(v, ror(v, std::integral_constant<int, 2>{}));
  return fn(v, ror(v, std::integral_constant<int, 1>{}));
}
// Of lanes l, l + 16, l + 32 and l + 48: exchanges of sixteens and of halves.
template <typename Fn>
__device__ __forceinline__ std::uint32_t across_rows(std::uint32_t v, Fn&& fn) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = fn(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fn(b[0], b[1]);
}
// Of all 64 lanes.
template <typename Fn>
__device__ __forceinline__ std::uint32_t across(std::uint32_t v, Fn&& fn) {
  return across_rows(across_row(v, fn), fn);
}
struct Larger {
  __device__ __forceinline__ std::uint32_t operator()(std::uint32_t a, std::uint32_t b) const { return max(a, b); }
};
// The largest of 32 lanes: 16, then an exchange of the two sixteens.
__device__ __forceinline__ std::uint32_t max_of_half(std::uint32_t v) {
  v = across_row(v, Larger{});
  const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(both[0], both[1]);
}

// g / (1 + exp(-g)) to a few units of the last place, without the branches of
// expf and of an IEEE quotient (they were a seventh of the vector work of a
// prompt's gated product): exp(-g) = 2^t with t = -g log2(e) in two parts, the
// hardware's 2^t and reciprocal (1 unit each), the reciprocal refined once.
// Beyond +-150 the exponential is inf or 0 either way; NaN stays one.  Gates
// below about -87, whose 1 + exp(-g) passes fp32, give 0 (silu is -2^-120 there).
__device__ __forceinline__ float silu(float g) {
  const float c = fminf(fmaxf(g, -150.0f), 150.0f);
  constexpr float kLog2e = 0x1.715476p+0f, kRest = 0x1.4ae0bep-26f, kLn2 = 0x1.62e43p-1f;
  const float t = -c * kLog2e;
  const float rest = __builtin_fmaf(-c, kLog2e, -t) - c * kRest;
  float e = __builtin_amdgcn_exp2f(t);
  e *= __builtin_fmaf(rest, kLn2, 1.0f);
  const float d = 1.0f + e;
  float r = __builtin_amdgcn_rcpf(d);
  const float refined = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
  r = d < 0x1p126f ? refined : r;  // of an inf, or where the refinement's product would be one
  return g * r;
}

}  // namespace llmi_hip::moe
