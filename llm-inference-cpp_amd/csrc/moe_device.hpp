// Device code that the experts' product kernels share: codes to fp16, a
// lane's weights of a chunk, and rows in two fp16 parts.
#pragma once

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

// A lane's weights of one tile and step.
template <int TYPE>
struct Weights {
  typedef std::uint32_t u32x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  std::uint32_t c[TYPE == LLMI_TYPE_Q4_0 ? 2 : 4];
  float s[2];
  // at: (expert * tiles + tile) * steps + step, common to the wavefront.
  __device__ __forceinline__ void load(const Matrices& m, std::size_t at, LaneAt& lane) {
    lane.here();
    const std::uint32_t code_at = TYPE == LLMI_TYPE_Q4_0 ? lane.by8 : lane.by16, scale_at = lane.scale;
    if constexpr (TYPE == LLMI_TYPE_Q4_0) {
      const u32x2 v = *(const __attribute__((address_space(1))) u32x2*)((GlobalBytes)m.codes + at * 512 + code_at);
      c[0] = v[0];
      c[1] = v[1];
    } else {
      const u32x4 v = *(const __attribute__((address_space(1))) u32x4*)((GlobalBytes)m.codes + at * 1024 + code_at);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = v[i];
    }
    const f32x2 v = *(const __attribute__((address_space(1))) f32x2*)((GlobalBytes)(m.scales + at * kStepScales) + scale_at);
    s[0] = v[0];
    s[1] = v[1];
  }
  // For the compiler: the loads are complete.
  __device__ __forceinline__ void here() {
#pragma unroll
    for (std::uint32_t& v : c) asm volatile("" : "+v"(v));
#pragma unroll
    for (float& v : s) asm volatile("" : "+v"(v));
  }
  __device__ __forceinline__ f16x8 codes(int b) const {
    if constexpr (TYPE == LLMI_TYPE_Q4_0) return codes_q4(c[b]);
    else return codes_q8(c[2 * b], c[2 * b + 1]);
  }
};

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

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

}  // namespace llmi_hip::moe
