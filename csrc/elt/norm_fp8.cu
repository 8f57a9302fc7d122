// RMS norm with the residual's addition and an output in 8 bits: what a projection with block-scaled fp8 weights takes in.
//
//   s = x + r, rounded to bf16 and stored in r;   y = s w / sqrt(mean(s^2) + eps), in fp32
//   per 128 entries:  scale = max|y| / 448 (1 where all are zero),  codes = e4m3(y / scale)
//
// The root is a factor of every entry and of the largest one, so the codes do not depend on it: with t = s w they are e4m3(t m), m = 448 / max|t|, and
// scale = 1 / (m sqrt(mean(s^2) + eps)).  Entries therefore go from load to store in one pass and no row waits for its sum; only
// the scales, one for 128 entries, are written after it.  One CTA per row, a thread has eight entries, 16 threads a group of 128.
// Bound by memory: 7 bytes per entry with a residual, 3 without, where a norm and a quantiser of their own move 10 (6) and need two
// launches.  The norm is not rounded before it is quantised.  No counterpart in the reference.
#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"
#include "../include/scalar.cuh"

namespace forge {

constexpr int kNormFp8Threads = 1024;

struct NormFp8 {
  const __nv_bfloat16* x;
  __nv_bfloat16* residual;                              // null: none
  const __nv_bfloat16* w;
  uint8_t* codes;
  float* scales;
  int scale_ld, H;
  float eps;
};

// kVectors of eight entries per thread.
template <bool kAdd, int kVectors>
__global__ void __launch_bounds__(kNormFp8Threads) rms_norm_fp8_kernel(const NormFp8 a) {
  __shared__ float red[kNormFp8Threads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t row = blockIdx.x;
  const int nvec = a.H >> 3, warps = blockDim.x >> 5;
  float m[kVectors], ss = 0.f;                          // m: 0 for a group of zeros
#pragma unroll
  for (int c = 0; c < kVectors; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    m[c] = 0.f;
    if (c * static_cast<int>(blockDim.x) >= nvec) break;             // uniform: the shuffles below take whole warps
    float t[8], amax = 0.f;
    if (i < nvec) {
      const size_t at = row * a.H + 8 * i;
      const uint4 xv = *reinterpret_cast<const uint4*>(a.x + at), wv = *reinterpret_cast<const uint4*>(a.w + 8 * i);
      uint32_t s[4] = {xv.x, xv.y, xv.z, xv.w};
      const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
      if constexpr (kAdd) {
        const uint4 rv = *reinterpret_cast<const uint4*>(a.residual + at);
        const uint32_t r[4] = {rv.x, rv.y, rv.z, rv.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = pack_bf16x2(bf16_lo(s[e]) + bf16_lo(r[e]), bf16_hi(s[e]) + bf16_hi(r[e]));
        *reinterpret_cast<uint4*>(a.residual + at) = make_uint4(s[0], s[1], s[2], s[3]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = bf16_lo(s[e]), hi = bf16_hi(s[e]);
        ss = fmaf(lo, lo, fmaf(hi, hi, ss));
        t[2 * e] = lo * bf16_lo(w[e]);
        t[2 * e + 1] = hi * bf16_hi(w[e]);
        amax = fmaxf(amax, fmaxf(fabsf(t[2 * e]), fabsf(t[2 * e + 1])));
      }
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (i >= nvec) continue;
    const float mul = fminf(448.f / amax, 0x1p126f);    // (infinite for zeros and for what is next to them)
    *reinterpret_cast<uint2*>(a.codes + row * a.H + 8 * i) =
        make_uint2(fp8_pack(t[0] * mul, t[1] * mul, t[2] * mul, t[3] * mul), fp8_pack(t[4] * mul, t[5] * mul, t[6] * mul, t[7] * mul));
    m[c] = amax == 0.f ? 0.f : mul;
  }
  ss = warp_sum_f(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  if (threadIdx.x & 15) return;
  ss = 0.f;
  for (int i = 0; i < warps; ++i) ss += red[i];
  const float inv = rsqrtf(ss / static_cast<float>(a.H) + a.eps);
#pragma unroll
  for (int c = 0; c < kVectors; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (i < nvec) a.scales[static_cast<size_t>(i >> 4) * a.scale_ld + row] = m[c] != 0.f ? inv / m[c] : inv == inv ? 1.f : inv;   // (NaN in the row)
  }
}

template <int kVectors>
static cudaError_t launch_rows(const NormFp8& a, int rows, cudaStream_t stream) {
  const int threads = ((a.H / 8 + kVectors - 1) / kVectors + 31) / 32 * 32;
  return launch_kernel(a.residual != nullptr ? rms_norm_fp8_kernel<true, kVectors> : rms_norm_fp8_kernel<false, kVectors>, dim3(rows), dim3(threads), 0,
                       stream, 0, a);
}

// x, residual [rows][H] bf16 (residual may be null), w [H], codes [rows][H], scales [H / 128][scale_ld >= rows].
extern "C" int forge_rms_norm_fp8(const void* x, void* residual, const void* w, void* codes, float* scales, int scale_ld, int rows, int H,
                                  float eps, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (H < 128 || H % 128 != 0 || H > 2 * kNormFp8Threads * 8 || scale_ld < rows) return -1;
  const NormFp8 a{static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(residual), static_cast<const __nv_bfloat16*>(w),
                  static_cast<uint8_t*>(codes), scales, scale_ld, H, eps};
  return (H <= kNormFp8Threads * 8 ? launch_rows<1>(a, rows, stream) : launch_rows<2>(a, rows, stream)) == cudaSuccess ? 0 : -2;
}

}  // namespace forge
