// A cache of keys or values in 8 bits: e4m3 codes [blocks][kv_heads][block_size][128] and one scale byte per token and head
// [blocks][kv_heads][block_size].  A byte b scales the head's 128 codes by 2^(b - 127), 255 stands for NaN.
//
// The scale is a power of two, the smallest with which no entry exceeds 448, the largest e4m3 number (not below 2^-126).  e4m3 is a
// floating type: a finer scale has no smaller bound on an entry's relative error (2^-4), although it may hold a single entry closer, the head's
// largest above all; only entries below 2^-14 of the largest come among the subnormals one binade earlier.  In return the byte costs
// 1 / 128 of the codes (an fp32 scale 4 / 128), a product over keys takes the scale in as an addition to its exponent, and a code times
// its scale is exact in bf16 from byte 3 on (below that, products under 2^-133 are rounded) and finite (see fp8_quantise).
#pragma once

#include <cuda_fp8.h>

#include "ptx.cuh"

namespace forge {

constexpr int kFp8D = 128;                 // entries of a head
constexpr uint32_t kScaleNan = 255;
constexpr uint32_t kScaleTop = 247;        // of heads whose largest entry is above 448 2^119: 2^120
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

// ---- a head in eight lanes: lane j has entries 8j .. (x) and 64 + 8j .. (y), the pairs that the rotation mixes ----

// Eight consecutive bf16 values; kVec: one 16-byte access.
template <bool kVec>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p) {
  if constexpr (kVec) return *reinterpret_cast<const uint4*>(p);
  const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
  return make_uint4(s[0] | static_cast<uint32_t>(s[1]) << 16, s[2] | static_cast<uint32_t>(s[3]) << 16, s[4] | static_cast<uint32_t>(s[5]) << 16,
                    s[6] | static_cast<uint32_t>(s[7]) << 16);
}
__device__ __forceinline__ void unpack8(uint4 r, float v[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
  }
}
__device__ __forceinline__ uint4 pack8(const float v[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
// The larger one, NaN if one is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// A lane's norm weights of query or key heads (null: no norm).
struct Fp8Weights {
  float lo[8], hi[8];
  template <bool kVec>
  __device__ __forceinline__ void load(const __nv_bfloat16* w, int j) {
    if (w == nullptr) return;
    unpack8(load8<kVec>(w + 8 * j), lo);
    unpack8(load8<kVec>(w + 64 + 8 * j), hi);
  }
};

// RMS norm, if any, and rotation by the angles whose cos and sin stand at cs and cs + 64 (null: none), in fp32.  octet: the head's lanes.
__device__ __forceinline__ void fp8_norm_rotate(float (&x)[8], float (&y)[8], const Fp8Weights& w, bool norm, float eps, const float* cs, unsigned octet) {
  if (norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(octet, ss, o);
    const float inv = rsqrtf(ss * (1.f / kFp8D) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = x[i] * inv * w.lo[i];
      y[i] = y[i] * inv * w.hi[i];
    }
  }
  if (cs != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 c = *reinterpret_cast<const float4*>(cs + i), s = *reinterpret_cast<const float4*>(cs + 64 + i);
      rotate_pair(x[i], y[i], c.x, s.x);
      rotate_pair(x[i + 1], y[i + 1], c.y, s.y);
      rotate_pair(x[i + 2], y[i + 2], c.z, s.z);
      rotate_pair(x[i + 3], y[i + 3], c.w, s.w);
    }
  }
}

// Of four codes those of 256 become 240, the number before it (0x78, 0x77): under the scale 2^120 256 would be infinite.
__device__ __forceinline__ uint32_t fp8_keep_finite(uint32_t codes) { return (codes & 0x80808080u) | __vminu4(codes & 0x7F7F7F7Fu, 0x77777777u); }

// Codes of a head (code[0]: of x, code[1]: of y); its scale byte.  A finite head stays finite: entries from 248 2^120 on, which are nearer to 256 than to
// 240, are held as 240 2^120, off by no more than half a step's 2^-4 all the same.
__device__ __forceinline__ uint32_t fp8_quantise(const float (&x)[8], const float (&y)[8], unsigned octet, uint2 (&code)[2]) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max_or_nan(amax, max_or_nan(fabsf(x[i]), fabsf(y[i])));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = max_or_nan(amax, __shfl_xor_sync(octet, amax, o));
  const uint32_t b = fp8_scale_byte(abs_bits(amax));
  code[0] = code[1] = make_uint2(kCodesNan, kCodesNan);
  if (b != kScaleNan) {
    const float m = fp8_inverse_scale(b);
    code[0] = make_uint2(fp8_pack(x[0] * m, x[1] * m, x[2] * m, x[3] * m), fp8_pack(x[4] * m, x[5] * m, x[6] * m, x[7] * m));
    code[1] = make_uint2(fp8_pack(y[0] * m, y[1] * m, y[2] * m, y[3] * m), fp8_pack(y[4] * m, y[5] * m, y[6] * m, y[7] * m));
    if (b == kScaleTop) {
#pragma unroll
      for (int i = 0; i < 2; ++i) code[i] = make_uint2(fp8_keep_finite(code[i].x), fp8_keep_finite(code[i].y));
    }
  }
  return b;
}

}  // namespace forge
