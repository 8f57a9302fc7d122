// Attention of one new token per sequence over a paged 8-bit cache (include/fp8_cache.cuh).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m),   c = scale log2(e),   m = max_j c q.k_j
//
// A CTA per sequence and query head; its warps take the tokens in turn and their sums are joined at the end.
#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"

namespace forge {

__global__ void __launch_bounds__(128) decode_fp8_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_codes,
                                                         const uint8_t* __restrict__ k_scales, const uint8_t* __restrict__ v_codes,
                                                         const uint8_t* __restrict__ v_scales, const int* __restrict__ block_tables,
                                                         const int* __restrict__ lens, __nv_bfloat16* __restrict__ out, int nq, int nkv,
                                                         int block_size, int table_width, int num_blocks, float scale_log2, unsigned* status) {
  __shared__ float s_o[4][kFp8D], s_m[4], s_l[4];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / (nq / nkv), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int len = lens[b];
  if (len > table_width * block_size) {
    if (threadIdx.x == 0) set_status(status, kStatusBadIndex);
    len = table_width * block_size;
  }
  const __nv_bfloat16* qp = q + (static_cast<size_t>(b) * nq + h) * kFp8D + 4 * lane;
  const float qv[4] = {__bfloat162float(qp[0]), __bfloat162float(qp[1]), __bfloat162float(qp[2]), __bfloat162float(qp[3])};
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int t = warp; t < len; t += 4) {
    int blk = block_tables[static_cast<size_t>(b) * table_width + t / block_size];
    if (blk < 0 || blk >= num_blocks) {
      set_status(status, kStatusBadIndex);
      blk = 0;
    }
    const size_t row = (static_cast<size_t>(blk) * nkv + kvh) * block_size + t % block_size;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(k_codes + row * kFp8D + 4 * lane), vw = *reinterpret_cast<const uint32_t*>(v_codes + row * kFp8D + 4 * lane);
    const float2 k0 = fp8_to_float2(kw), k1 = fp8_to_float2(kw >> 16), v0 = fp8_to_float2(vw), v1 = fp8_to_float2(vw >> 16);
    float d = qv[0] * k0.x + qv[1] * k0.y + qv[2] * k1.x + qv[3] * k1.y;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) d += __shfl_xor_sync(0xffffffffu, d, i);
    const float s = d * fp8_scale(k_scales[row]) * scale_log2;
    const float m_new = fmaxf(m, s), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - m_use), p = exp2f(s - m_use), pv = p * fp8_scale(v_scales[row]);
    l = l * alpha + p;
    o[0] = o[0] * alpha + pv * v0.x;
    o[1] = o[1] * alpha + pv * v0.y;
    o[2] = o[2] * alpha + pv * v1.x;
    o[3] = o[3] * alpha + pv * v1.y;
    m = m_new;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s_o[warp][4 * lane + e] = o[e];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < 4; ++w) {
    const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - M);
    L += s_l[w] * f;
    O += s_o[w][threadIdx.x] * f;
  }
  out[(static_cast<size_t>(b) * nq + h) * kFp8D + threadIdx.x] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
}

// q [B, nq, 128], out [B, nq * 128] bf16; a length of zero gives a row of zeros.
extern "C" int forge_decode_fp8(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                const int* block_tables, const int* lens, void* out, int B, int nq, int nkv, int block_size, int table_width,
                                int num_blocks, float scale, unsigned* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (B > 65535 || nkv < 1 || nq % nkv != 0) return -1;
  return launch_kernel(decode_fp8_kernel, dim3(nq, B), dim3(128), 0, stream, 0, static_cast<const __nv_bfloat16*>(q),
                       static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(k_scales), static_cast<const uint8_t*>(v_codes),
                       static_cast<const uint8_t*>(v_scales), block_tables, lens, static_cast<__nv_bfloat16*>(out), nq, nkv, block_size, table_width,
                       num_blocks, scale * 1.4426950408889634f, status) == cudaSuccess ? 0 : -2;
}

}  // namespace forge
