// RMS norm with the residual's addition and an output in 8 bits: what a projection with block-scaled fp8 weights takes in.
//
//   s = x + r, rounded to bf16 and stored in r;   y = s w / sqrt(mean(s^2) + eps), in fp32
//   per 128 entries:  scale = max|y| / 448 (1 where all are zero),  codes = e4m3(y / scale)
//
// Few rows: one CTA per row, a thread has eight entries (16 threads a group of 128).  Many rows: one warp per row, all of its loads under
// way at once and no barrier; the row stays in registers as the bf16 it is held in.  Bound by memory: 7 bytes per entry with a residual, 3
// without, where a norm and a quantiser of their own move 10 (6) and need two launches.  The norm is not rounded before it is
// quantised.  No counterpart in the reference.
#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"
#include "../include/scalar.cuh"

namespace forge {

constexpr int kNormFp8Threads = 512;

struct NormFp8 {
  const __nv_bfloat16* x;
  __nv_bfloat16* residual;                              // null: none
  const __nv_bfloat16* w;
  uint8_t* codes;
  float* scales;
  int scale_ld, rows, H;
  float eps;
};

// Eight entries of the stream as four pairs of bf16: x, or x + r rounded and stored; adds their squares.
template <bool kAdd>
__device__ __forceinline__ uint4 norm_fp8_take(uint4 v, uint4 r, __nv_bfloat16* to, float& ss) {
  uint32_t s[4] = {v.x, v.y, v.z, v.w};
  if constexpr (kAdd) {
    const uint32_t b[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = pack_bf16x2(bf16_lo(s[i]) + bf16_lo(b[i]), bf16_hi(s[i]) + bf16_hi(b[i]));
    *reinterpret_cast<uint4*>(to) = make_uint4(s[0], s[1], s[2], s[3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) ss = fmaf(bf16_lo(s[i]), bf16_lo(s[i]), fmaf(bf16_hi(s[i]), bf16_hi(s[i]), ss));
  return make_uint4(s[0], s[1], s[2], s[3]);
}

// Vector i of a row (entries 8 i ..) normed and quantised; 16 neighbouring lanes have a group and come here together.  `in`: there is such a vector.
__device__ __forceinline__ void norm_fp8_put(const NormFp8& a, size_t row, int i, bool in, uint4 s, float inv) {
  float y[8], amax = 0.f;
  if (in) {
    const uint4 wv = *reinterpret_cast<const uint4*>(a.w + 8 * i);
    const uint32_t v[4] = {s.x, s.y, s.z, s.w}, w[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[2 * e] = bf16_lo(v[e]) * inv * bf16_lo(w[e]);
      y[2 * e + 1] = bf16_hi(v[e]) * inv * bf16_hi(w[e]);
      amax = fmaxf(amax, fmaxf(fabsf(y[2 * e]), fabsf(y[2 * e + 1])));
    }
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (!in) return;
  const float scale = amax > 0.f ? amax / 448.f : 1.f, m = 1.f / scale;
  *reinterpret_cast<uint2*>(a.codes + row * a.H + 8 * i) =
      make_uint2(fp8_pack(y[0] * m, y[1] * m, y[2] * m, y[3] * m), fp8_pack(y[4] * m, y[5] * m, y[6] * m, y[7] * m));
  if ((i & 15) == 0) a.scales[static_cast<size_t>(i >> 4) * a.scale_ld + row] = scale;
}

// One CTA per row; kVectors of eight entries per thread.
template <bool kAdd, int kVectors>
__global__ void __launch_bounds__(kNormFp8Threads) rms_norm_fp8_kernel(const NormFp8 a) {
  __shared__ float red[kNormFp8Threads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t row = blockIdx.x;
  const int nvec = a.H >> 3, warps = blockDim.x >> 5;
  uint4 s[kVectors];
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < kVectors; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (i >= nvec) continue;
    const size_t at = row * a.H + 8 * i;
    s[c] = norm_fp8_take<kAdd>(*reinterpret_cast<const uint4*>(a.x + at), kAdd ? *reinterpret_cast<const uint4*>(a.residual + at) : make_uint4(0, 0, 0, 0),
                               a.residual + at, ss);
  }
  ss = warp_sum_f(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < warps; ++i) ss += red[i];
  const float inv = rsqrtf(ss / static_cast<float>(a.H) + a.eps);
#pragma unroll
  for (int c = 0; c < kVectors; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (c * static_cast<int>(blockDim.x) < nvec) norm_fp8_put(a, row, i, i < nvec, s[c], inv);           // (uniform: whole warps)
  }
}

// One warp per row; kVectors of eight entries per lane.
template <bool kAdd, int kVectors>
__global__ void __launch_bounds__(128) rms_norm_fp8_warp_kernel(const NormFp8 a) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, nvec = a.H >> 3;
  const size_t row = static_cast<size_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<size_t>(a.rows)) return;
  uint4 s[kVectors], r[kAdd ? kVectors : 1];
#pragma unroll
  for (int c = 0; c < kVectors; ++c) {
    const int i = lane + 32 * c;
    if (i >= nvec) continue;
    s[c] = *reinterpret_cast<const uint4*>(a.x + row * a.H + 8 * i);
    if constexpr (kAdd) r[c] = *reinterpret_cast<const uint4*>(a.residual + row * a.H + 8 * i);
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < kVectors; ++c) {
    const int i = lane + 32 * c;
    if (i < nvec) s[c] = norm_fp8_take<kAdd>(s[c], r[kAdd ? c : 0], a.residual + row * a.H + 8 * i, ss);
  }
  const float inv = rsqrtf(warp_sum_f(ss) / static_cast<float>(a.H) + a.eps);
#pragma unroll
  for (int c = 0; c < kVectors; ++c)
    if (32 * c < nvec) norm_fp8_put(a, row, lane + 32 * c, lane + 32 * c < nvec, s[c], inv);
}

template <int kVectors>
static cudaError_t launch_rows(const NormFp8& a, cudaStream_t stream) {
  int threads = ((a.H >> 3) + 31) / 32 * 32;
  if (threads > kNormFp8Threads) threads = kNormFp8Threads;
  return launch_kernel(a.residual != nullptr ? rms_norm_fp8_kernel<true, kVectors> : rms_norm_fp8_kernel<false, kVectors>, dim3(a.rows), dim3(threads), 0,
                       stream, 0, a);
}
template <int kVectors>
static cudaError_t launch_warps(const NormFp8& a, cudaStream_t stream) {
  return launch_kernel(a.residual != nullptr ? rms_norm_fp8_warp_kernel<true, kVectors> : rms_norm_fp8_warp_kernel<false, kVectors>, dim3((a.rows + 3) / 4),
                       dim3(128), 0, stream, 0, a);
}

// x, residual [rows][H] bf16 (residual may be null), w [H], codes [rows][H], scales [H / 128][scale_ld >= rows].
extern "C" int forge_rms_norm_fp8(const void* x, void* residual, const void* w, void* codes, float* scales, int scale_ld, int rows, int H,
                                  float eps, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (H < 128 || H % 128 != 0 || H > 4 * kNormFp8Threads * 8 || scale_ld < rows) return -1;
  const NormFp8 a{static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(residual), static_cast<const __nv_bfloat16*>(w),
                  static_cast<uint8_t*>(codes), scales, scale_ld, rows, H, eps};
  cudaError_t e;
  if (rows < 8 * device_sm_count() || H > 5120) e = H <= kNormFp8Threads * 8 ? launch_rows<1>(a, stream) : launch_rows<4>(a, stream);
  else if (H <= 1024) e = launch_warps<4>(a, stream);
  else if (H <= 2048) e = launch_warps<8>(a, stream);
  else if (H <= 2560) e = launch_warps<10>(a, stream);
  else if (H <= 4096) e = launch_warps<16>(a, stream);
  else e = launch_warps<20>(a, stream);
  return e == cudaSuccess ? 0 : -2;
}

}  // namespace forge
