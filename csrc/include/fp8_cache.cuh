// A cache of keys or values in 8 bits: e4m3 codes [blocks][kv_heads][block_size][128] and one scale byte per token and head
// [blocks][kv_heads][block_size].  A byte b scales the head's 128 codes by 2^(b - 127), 255 stands for NaN.
//
// The scale is a power of two, the smallest with which no entry exceeds 448, the largest e4m3 number (not below 2^-126).  e4m3 is a
// floating type: another scale would round no entry closer, except those below 2^-14 of the head's largest, which a power of two moves
// into the subnormals one binade earlier.  In return the byte costs 1 / 128 of the codes (an fp32 scale 4 / 128), a code times its
// scale is exact in bf16, and a product over keys takes the scale in as an addition to its exponent.
#pragma once

#include <cuda_fp8.h>

#include "ptx.cuh"

namespace forge {

constexpr int kFp8D = 128;                 // entries of a head
constexpr uint32_t kScaleNan = 255;
constexpr uint32_t kCodesNan = 0x7F7F7F7Fu;

// |x| as an unsigned number: ordered like the values, infinities above them and NaN above those, so that a maximum keeps NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Scale byte of a head whose largest entry has these absolute bits.  448 = 1.75 2^8: the exponent less 8, one more where the mantissa is above 1.75.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t amax) {
  if (amax >= 0x7F800000u) return kScaleNan;
  const int b = static_cast<int>((amax + 0x1FFFFFu) >> 23) - 8;
  return static_cast<uint32_t>(b < 1 ? 1 : b);
}
// 2^(127 - b): what entries are multiplied by before they are rounded (b = 1 .. 247).
__device__ __forceinline__ float fp8_inverse_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }
// 2^(b - 127), NaN for 255.
__device__ __forceinline__ float fp8_scale(uint32_t b) {
  return b == kScaleNan ? __uint_as_float(0x7FC00000u) : b == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(b << 23);
}

// Four entries -> four codes, rounded to nearest even.
__device__ __forceinline__ uint32_t fp8_pack(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Two codes (bits 0..15) -> two halves, exact.
__device__ __forceinline__ uint32_t fp8_to_half2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(codes)));
  return h;
}
// Four codes -> the halves of bits 0..15 and of bits 16..31.
__device__ __forceinline__ void fp8x4_to_half2(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n"
      : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float2 fp8_to_float2(uint32_t codes) {
  const uint32_t h = fp8_to_half2(codes & 0xFFFFu);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace forge
