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

// x / n for x >= 0, n > 0: 64-bit divisions are a hundred instructions, and the numbers are small as a rule.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t n) {
  if (((x | n) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(n);
  return x / n;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ void unpack_f16(uint32_t w, float& lo, float& hi) {
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.f32.f16 %0, a;\n cvt.f32.f16 %1, b;\n}" : "=f"(lo), "=f"(hi) : "r"(w));
}
// Eight neighbouring values, 16-byte aligned, as floats.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// x * s + c on two bfloat16 (fp16) values, one rounding.
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t x, uint32_t s, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(s), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t x, uint32_t s) { return fma_bf16x2(x, s, 0x80008000u); }
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t x, uint32_t s, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(s), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t x, uint32_t c) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(c));
  return d;
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t x, uint32_t s) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(s));
  return d;
}
#endif  // __CUDACC__

// Every conversion below is exact, one operation behind the extraction of the bits.
// Bit patterns that the conversions need, as values that the compiler does not know: with two constants known in one
// operation it spends a second one on it.
struct Patterns {
  uint32_t x43, x3f;                     // bfloat16 128, 1 / 2
  uint32_t up0, up4, less;               // fp16 2^15, 2^11; minus the codes' bias, times 2^-9
};
inline Patterns patterns(int bits) { return {0x43004300u, 0x3f003f00u, 0x78007800u, 0x68006800u, bits == 4 ? 0xa400a400u : 0xb400b400u}; }

#ifdef __CUDACC__
// Stored codes u as fp16 numbers: the bits alone are the subnormal numbers u * 2^-24, or u * 2^-20 where they lie four places higher.
// 4-bit codes: of w's nibbles, pair i of out holds i and i + 4; pairs 1 and 3 are the ones times 2^-20.
__device__ __forceinline__ void codes4_f16(uint32_t w, uint32_t (&out)[4]) {
  const uint32_t v = w >> 8;
  out[0] = w & 0x000f000fu;
  out[1] = w & 0x00f000f0u;
  out[2] = v & 0x000f000fu;
  out[3] = v & 0x00f000f0u;
}
// 8-bit codes: bytes 0, 1 and 2, 3.
__device__ __forceinline__ void codes8_f16(uint32_t w, uint32_t (&out)[2]) {
  out[0] = prmt(w, 0, 0x4140);
  out[1] = prmt(w, 0, 0x4342);
}
// The same numbers without the bias, times 2^-9: (u - 8) * 2^-9, (u - 128) * 2^-9.
__device__ __forceinline__ void unbias4_f16(uint32_t (&x)[4], const Patterns& c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fma_f16x2(x[i], i & 1 ? c.up4 : c.up0, c.less);
}
__device__ __forceinline__ void unbias8_f16(uint32_t (&x)[2], const Patterns& c) {
#pragma unroll
  for (int i = 0; i < 2; ++i) x[i] = fma_f16x2(x[i], c.up0, c.less);
}
// Codes times their scales as bfloat16 numbers: the bits go under the exponent of a power of two.
// 4 bits: nibble i of both halves of w, the halves' scales in s2.
__device__ __forceinline__ uint32_t bias4(uint32_t s2) { return mul_bf16x2(s2, 0xc308c308u); }   // -136 s
__device__ __forceinline__ void values4_bf16(uint32_t w, uint32_t s2, uint32_t b2, const Patterns& c, uint32_t (&out)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = fma_bf16x2(((w >> (4 * i)) & 0x000f000fu) | c.x43, s2, b2);   // (128 + u) s - 136 s
}
// 8 bits: byte i of both halves of w. The mantissa takes seven bits; the eighth moves the exponent of a half.
struct Scale8 {
  uint32_t s, b, t;                      // s, -384 s, 256 s
};
__device__ __forceinline__ Scale8 scale8(uint32_t s2) { return {s2, mul_bf16x2(s2, 0xc3c0c3c0u), mul_bf16x2(s2, 0x43804380u)}; }
__device__ __forceinline__ void values8_bf16(uint32_t w, const Scale8& s, const Patterns& c, uint32_t (&out)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = w >> (8 * i);
    const uint32_t low = fma_bf16x2((v & 0x007f007fu) | c.x43, s.s, s.b);   // (128 + u mod 128) s - 384 s
    out[i] = fma_bf16x2((v & 0x00800080u) | c.x3f, s.t, low);               // + 128 s or 256 s
  }
}

#endif  // __CUDACC__

}  // namespace kvq
}  // namespace ctdk
