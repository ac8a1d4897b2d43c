// A key/value cache held in 4 or 8 bits: its layout, and the arithmetic that the kernels over it share.
//
// A head row of D values (64 or 128) is cut into groups of 32. A group has one bfloat16 scale s and codes c,
// stored as c + 8 (4 bits, the even column in the low half of a byte) or c + 128 (8 bits), and stands for c * s.
// s has at most four significant bits beside 4-bit codes (|c| <= 7) and is a power of two beside 8-bit codes
// (|c| <= 127), so c * s has at most seven and is exact in bfloat16 (and so is 136 * s, which the conversion subtracts): the tensor cores multiply the cached values
// themselves, nothing is rounded between the cache and the product, and no scale has to be carried past it.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace ctdk {
namespace kvq {

constexpr int kGroup = 32;
constexpr int kCapacityStep = 64;        // positions: the kernels load whole tiles of up to 64
constexpr float kMost = 0x1p100f;        // a magnitude from here on makes its group NaN (sums with the biases below stay finite)

struct Cache {
  const uint8_t* codes[2];               // keys, values: [B, Hk, capacity, D * bits / 8]
  const __nv_bfloat16* scales[2];        // [B, Hk, capacity, D / 32]
  int64_t capacity;
  int B, Hk;
};

#ifdef __CUDACC__

// Bits of a scale that stands for NaN: larger than any that is written (below 2^98), in either sign.
__device__ __forceinline__ bool is_nan_scale(uint32_t bits) { return (bits & 0x7fffu) >= 0x7080u; }

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// x * s + c on two bfloat16 values, one rounding.
__device__ __forceinline__ uint32_t hfma2_bf16(uint32_t x, uint32_t s, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(s), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t hmul2_bf16(uint32_t x, uint32_t s) { return hfma2_bf16(x, s, 0x80008000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 4 bits: the codes at bits 4k and 4k + 16 of w, times the scales s2, as two bfloat16 values. The nibble under the
// exponent of 128 is the number 128 + u; (128 + u) * s - 136 * s is rounded once and exact. b2 = bias4(s2).
__device__ __forceinline__ uint32_t bias4(uint32_t s2) { return hmul2_bf16(s2, 0xc308c308u); }   // -136 * s
template <int K>
__device__ __forceinline__ uint32_t value4(uint32_t w, uint32_t s2, uint32_t b2) {
  return hfma2_bf16(((w >> (4 * K)) & 0x000f000fu) | 0x43004300u, s2, b2);
}
// 8 bits: byte K of w, as the fp32 number 2^23 + u.
template <int K>
__device__ __forceinline__ float magic8(uint32_t w) {
  return __uint_as_float(prmt(w, 0x4b000000u, 0x7650u + K));
}
// (2^23 + u) * s - (2^23 + 128) * s, exact, for two codes with scales s0, s1 and biases b = -(2^23 + 128) * s.
__device__ __forceinline__ uint32_t values8(float f0, float f1, float s0, float s1, float b0, float b1) {
  float x, y;
  ffma2(x, y, f0, f1, s0, s1, b0, b1);
  return pack_bf16(x, y);
}
__device__ __forceinline__ float bias8(float s) { return s * -8388736.0f; }

#endif  // __CUDACC__

}  // namespace kvq
}  // namespace ctdk
