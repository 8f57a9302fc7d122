// RMS norm with the residual's addition and an output in 8 bits: what a projection with block-scaled fp8 weights takes in.
//
//   s = x + r, rounded to bf16 and stored in r;   y = s w / sqrt(mean(s^2) + eps), in fp32
//   per 128 entries:  scale = max|y| / 448 (1 where all are zero),  codes = e4m3(y / scale)
//
// One CTA per row, the row in registers between the passes; 16 threads have a group of 128 entries.  Bound by memory: 7 bytes per
// entry with a residual, 3 without, where a norm and a quantiser of their own move 10 (6) and need two launches.  The norm is not rounded before
// it is quantised.  No counterpart in the reference.
#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"
#include "../include/scalar.cuh"

namespace forge {

constexpr int kNormFp8Chunks = 4, kNormFp8Threads = 512;

template <bool kAdd>
__global__ void __launch_bounds__(kNormFp8Threads) rms_norm_fp8_kernel(const __nv_bfloat16* __restrict__ x, __nv_bfloat16* __restrict__ residual,
                                                                       const __nv_bfloat16* __restrict__ w, uint8_t* __restrict__ codes,
                                                                       float* __restrict__ scales, int scale_ld, int H, float eps) {
  __shared__ float red[kNormFp8Threads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t row = blockIdx.x;
  const int nvec = H >> 3, warps = blockDim.x >> 5;
  float v[kNormFp8Chunks][8];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < kNormFp8Chunks; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (i >= nvec) continue;
    load_n<8>(x + row * H + 8 * i, v[c]);
    if constexpr (kAdd) {
      float r[8];
      load_n<8>(residual + row * H + 8 * i, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = __bfloat162float(__float2bfloat16_rn(v[c][e] + r[e]));
      store_n<8>(residual + row * H + 8 * i, v[c]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[c][e], v[c][e], ss);
  }
  ss = warp_sum_f(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < warps; ++i) ss += red[i];
  const float inv = rsqrtf(ss / static_cast<float>(H) + eps);
#pragma unroll
  for (int c = 0; c < kNormFp8Chunks; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (c * static_cast<int>(blockDim.x) >= nvec) break;              // uniform: the shuffles below take whole warps
    float y[8], wv[8], amax = 0.f;
    if (i < nvec) {
      load_n<8>(w + 8 * i, wv);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = v[c][e] * inv * wv[e];
        amax = fmaxf(amax, fabsf(y[e]));
      }
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (i >= nvec) continue;
    const float s = amax > 0.f ? amax / 448.f : 1.f;
    *reinterpret_cast<uint2*>(codes + row * H + 8 * i) =
        make_uint2(fp8_pack(y[0] / s, y[1] / s, y[2] / s, y[3] / s), fp8_pack(y[4] / s, y[5] / s, y[6] / s, y[7] / s));
    if ((i & 15) == 0) scales[static_cast<size_t>(i >> 4) * scale_ld + row] = s;
  }
}

// x, residual [rows][H] bf16 (residual may be null), w [H], codes [rows][H], scales [H / 128][scale_ld >= rows].
extern "C" int forge_rms_norm_fp8(const void* x, void* residual, const void* w, void* codes, float* scales, int scale_ld, int rows, int H,
                                  float eps, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (H < 128 || H % 128 != 0 || H > kNormFp8Chunks * kNormFp8Threads * 8 || scale_ld < rows) return -1;
  int threads = ((H >> 3) + 31) / 32 * 32;
  if (threads > kNormFp8Threads) threads = kNormFp8Threads;
  return launch_kernel(residual != nullptr ? rms_norm_fp8_kernel<true> : rms_norm_fp8_kernel<false>, dim3(rows), dim3(threads), 0, stream, 0,
                       static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(residual), static_cast<const __nv_bfloat16*>(w),
                       static_cast<uint8_t*>(codes), scales, scale_ld, H, eps) == cudaSuccess ? 0 : -2;
}

}  // namespace forge
