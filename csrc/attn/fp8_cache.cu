// Writing and reading an 8-bit KV cache (layout and scales: include/fp8_cache.cuh).
//
//   store    split of the packed qkv row, per-head RMS norm of q and k, rotation, quantisation of k and v into the paged cache.
//            What the bf16 cache's kernel does (elt/elementwise.cu), but everything between the projection and the one rounding of a
//            result stays in fp32.
//   expand   pages of sequences in order as bf16 pages, for attention of prompts: exact, so a prompt attends to the same
//            values whether its prefix was cached or written a moment ago.
//
// No counterpart in the reference, whose cache has the model's type.
#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"

namespace forge {

// Eight consecutive bf16 values; kVec: one 16-byte access.
template <bool kVec>
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float v[8]) {
  if constexpr (kVec) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_lo(w[i]);
      v[2 * i + 1] = bf16_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
  }
}

struct Fp8Store {
  const __nv_bfloat16* qkv;
  long long ld;
  const __nv_bfloat16 *qw, *kw;             // norm weights, null: no norm
  float eps;
  const float* rope;                        // null: no rotation
  int rope_rows;
  const int *positions, *slots;
  __nv_bfloat16* q_out;
  uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  int T, nq, nkv, block_size;
  long long num_slots;
  int heads_per_warp;
  unsigned* status;
};

// Eight lanes per head, lane j of them has entries 8j.. and 64 + 8j.., the pairs that the rotation mixes; a warp works on four heads
// of a token at a time, `heads_per_warp` in all, so that position, slot and angles are fetched once.  Bound by memory: qkv read once,
// q and the codes written once.
template <bool kVec>
__global__ void __launch_bounds__(128) fp8_store_kernel(const Fp8Store a) {
  pdl_launch_dependents();
  pdl_wait();
  const int heads = a.nq + 2 * a.nkv, groups = (heads + a.heads_per_warp - 1) / a.heads_per_warp;
  const long long wid = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (wid >= static_cast<long long>(a.T) * groups) return;
  const int lane = threadIdx.x & 31, j = lane & 7, sub = lane >> 3;
  const int t = static_cast<int>(wid / groups);
  const int h_begin = static_cast<int>(wid % groups) * a.heads_per_warp, h_end = min(h_begin + a.heads_per_warp, heads);
  float c[8], s[8];
  if (a.rope != nullptr) {
    const float* cs = a.rope + static_cast<size_t>(min(max(a.positions[t], 0), a.rope_rows - 1)) * kFp8D;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(cs + 8 * j + i);
      *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(cs + 64 + 8 * j + i);
    }
  }
  const long long slot = a.slots[t];
  const bool slot_ok = slot >= 0 && slot < a.num_slots;
  if (slot >= a.num_slots && lane == 0) set_status(a.status, kStatusBadIndex);

  for (int h0 = h_begin; h0 < h_end; h0 += 4) {
    const int h = h0 + sub;
    const bool live = h < h_end, is_q = h < a.nq, is_k = !is_q && h < a.nq + a.nkv;
    const __nv_bfloat16* src = a.qkv + static_cast<size_t>(t) * a.ld + static_cast<size_t>(live ? h : h_begin) * kFp8D;
    float lo[8], hi[8];
    load8<kVec>(src + 8 * j, lo);
    load8<kVec>(src + 64 + 8 * j, hi);
    const __nv_bfloat16* w = is_q ? a.qw : is_k ? a.kw : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = add_squares(lo[i], hi[i], ss);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w != nullptr) {
      const float inv = rsqrtf(ss / static_cast<float>(kFp8D) + a.eps);
      float wl[8], wh[8];
      load8<kVec>(w + 8 * j, wl);
      load8<kVec>(w + 64 + 8 * j, wh);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = lo[i] * inv * wl[i];
        hi[i] = hi[i] * inv * wh[i];
      }
    }
    if (a.rope != nullptr && (is_q || is_k)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) rotate_pair(lo[i], hi[i], c[i], s[i]);
    }
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, max(abs_bits(lo[i]), abs_bits(hi[i])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live) continue;
    if (is_q) {
      __nv_bfloat16* dst = a.q_out + (static_cast<size_t>(t) * a.nq + h) * kFp8D + 8 * j;
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(lo[4], lo[5]), pack_bf16x2(lo[6], lo[7]));
      *reinterpret_cast<uint4*>(dst + 64) = make_uint4(pack_bf16x2(hi[0], hi[1]), pack_bf16x2(hi[2], hi[3]), pack_bf16x2(hi[4], hi[5]), pack_bf16x2(hi[6], hi[7]));
      continue;
    }
    if (!slot_ok) continue;
    const int kvh = is_k ? h - a.nq : h - a.nq - a.nkv;
    const size_t row = (static_cast<size_t>(slot / a.block_size) * a.nkv + kvh) * a.block_size + slot % a.block_size;
    const uint32_t b = fp8_scale_byte(amax);
    uint2 code[2] = {make_uint2(kCodesNan, kCodesNan), make_uint2(kCodesNan, kCodesNan)};
    if (b != kScaleNan) {
      const float m = fp8_inverse_scale(b);
      code[0] = make_uint2(fp8_pack(lo[0] * m, lo[1] * m, lo[2] * m, lo[3] * m), fp8_pack(lo[4] * m, lo[5] * m, lo[6] * m, lo[7] * m));
      code[1] = make_uint2(fp8_pack(hi[0] * m, hi[1] * m, hi[2] * m, hi[3] * m), fp8_pack(hi[4] * m, hi[5] * m, hi[6] * m, hi[7] * m));
    }
    uint8_t* dst = (is_k ? a.k_codes : a.v_codes) + row * kFp8D + 8 * j;
    *reinterpret_cast<uint2*>(dst) = code[0];
    *reinterpret_cast<uint2*>(dst + 64) = code[1];
    if (j == 0) (is_k ? a.k_scales : a.v_scales)[row] = static_cast<uint8_t>(b);
  }
}

// qkv [T, (nq + 2 nkv) * 128] with rows ld apart; rope fp32 [rope_rows][128] = cos, sin; slot < 0 is passed over, slot >= num_slots too and
// reported.  The slots of a call are distinct.
extern "C" int forge_fp8_store(const void* qkv, long long ld, const void* qw, const void* kw, float eps, const float* rope, int rope_rows,
                               const int* positions, const int* slots, void* q_out, void* k_codes, void* k_scales, void* v_codes, void* v_scales,
                               int T, int nq, int nkv, int block_size, long long num_slots, unsigned* status, cudaStream_t stream) {
  if (T <= 0) return 0;
  Fp8Store a;
  a.qkv = static_cast<const __nv_bfloat16*>(qkv); a.ld = ld;
  a.qw = static_cast<const __nv_bfloat16*>(qw); a.kw = static_cast<const __nv_bfloat16*>(kw); a.eps = eps;
  a.rope = rope; a.rope_rows = rope_rows; a.positions = positions; a.slots = slots;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.k_codes = static_cast<uint8_t*>(k_codes); a.k_scales = static_cast<uint8_t*>(k_scales);
  a.v_codes = static_cast<uint8_t*>(v_codes); a.v_scales = static_cast<uint8_t*>(v_scales);
  a.T = T; a.nq = nq; a.nkv = nkv; a.block_size = block_size; a.num_slots = num_slots; a.status = status;
  a.heads_per_warp = T >= 4096 ? 16 : T >= 512 ? 8 : 4;
  const int groups = (nq + 2 * nkv + a.heads_per_warp - 1) / a.heads_per_warp;
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(T) * groups + 3) / 4));
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = ld % 8 == 0 && aligned(qkv) && aligned(qw) && aligned(kw);
  return launch_kernel(vec ? fp8_store_kernel<true> : fp8_store_kernel<false>, grid, dim3(128), 0, stream, 0, a) == cudaSuccess ? 0 : -2;
}

// ---------------------------------------------------------------------------------------------------------
// Pages of sequences, in order, as bf16.  A CTA takes `rows` token rows of one page of one head of K or V.
// ---------------------------------------------------------------------------------------------------------
constexpr int kExpandThreads = 256;

__global__ void __launch_bounds__(kExpandThreads) fp8_expand_kernel(
    const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ k_scales, const uint8_t* __restrict__ v_codes,
    const uint8_t* __restrict__ v_scales, const int* __restrict__ block_tables, const int* __restrict__ lens, int table_width, int num_blocks,
    int nkv, int block_size, int rows, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ tables,
    int capacity, unsigned* status) {
  __shared__ int red[kExpandThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.y, page = blockIdx.x;
  const int parts = block_size / rows, z = blockIdx.z;
  const int part = z % parts, kvh = z / parts % nkv, is_v = z / parts / nkv;
  const int cap = table_width * block_size;
  const bool first_cta = z == 0;
  int len = lens[seq];
  if (len > cap) {
    if (first_cta && page == 0 && threadIdx.x == 0) set_status(status, kStatusBadIndex);
    len = cap;
  }
  const int need = (max(len, 0) + block_size - 1) / block_size;
  if (page >= need) {
    if (first_cta && threadIdx.x == 0) tables[static_cast<size_t>(seq) * table_width + page] = -1;
    return;
  }
  int before = 0;                                       // pages of the sequences before this one
  for (int i = threadIdx.x; i < seq; i += kExpandThreads) before += (min(max(lens[i], 0), cap) + block_size - 1) / block_size;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int i = 0; i < kExpandThreads / 32; ++i) before += red[i];
  const int to = before + page;
  if (to >= capacity) {
    if (first_cta && threadIdx.x == 0) {
      set_status(status, kStatusBadIndex);
      tables[static_cast<size_t>(seq) * table_width + page] = -1;
    }
    return;
  }
  int blk = block_tables[static_cast<size_t>(seq) * table_width + page];
  if (blk < 0 || blk >= num_blocks) {
    if (first_cta && threadIdx.x == 0) set_status(status, kStatusBadIndex);
    blk = 0;
  }
  if (first_cta && threadIdx.x == 0) tables[static_cast<size_t>(seq) * table_width + page] = to;
  const size_t row0 = (static_cast<size_t>(blk) * nkv + kvh) * block_size + part * rows;
  const size_t out0 = (static_cast<size_t>(to) * nkv + kvh) * block_size + part * rows;
  const int live = min(len - page * block_size - part * rows, rows);
  const uint8_t* codes = (is_v ? v_codes : k_codes) + row0 * kFp8D;
  const uint8_t* scales = (is_v ? v_scales : k_scales) + row0;
  __nv_bfloat16* out = (is_v ? v_out : k_out) + out0 * kFp8D;
  for (int i = threadIdx.x; i < rows * 8; i += kExpandThreads) {                // 16 codes each
    const int r = i >> 3;
    uint32_t o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (r < live) {
      const uint4 raw = *reinterpret_cast<const uint4*>(codes + i * 16);
      const float m = fp8_scale(scales[r]);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 f = fp8_to_float2(w[e >> 1] >> (16 * (e & 1)));
        o[e] = pack_bf16x2(f.x * m, f.y * m);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(out + i * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// k_out, v_out [capacity][nkv][block_size][128]; tables [num_seqs][table_width] gets the page numbers in them, -1 behind a sequence's last.
// A sequence's pages follow one another, and the sequences too; entries behind a sequence's last token are zero.
extern "C" int forge_fp8_expand(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const int* block_tables,
                                const int* lens, int num_seqs, int table_width, int num_blocks, int nkv, int block_size, void* k_out, void* v_out,
                                int* tables, int capacity, unsigned* status, cudaStream_t stream) {
  if (num_seqs <= 0 || table_width <= 0) return 0;
  if (block_size < 1 || num_seqs > 65535) return -1;
  const int rows = block_size % 64 == 0 ? 64 : block_size;
  const long long z = 2ll * nkv * (block_size / rows);
  if (z > 65535) return -1;
  const dim3 grid(static_cast<unsigned>(table_width), static_cast<unsigned>(num_seqs), static_cast<unsigned>(z));
  return launch_kernel(fp8_expand_kernel, grid, dim3(kExpandThreads), 0, stream, 0, static_cast<const uint8_t*>(k_codes),
                       static_cast<const uint8_t*>(k_scales), static_cast<const uint8_t*>(v_codes), static_cast<const uint8_t*>(v_scales), block_tables,
                       lens, table_width, num_blocks, nkv, block_size, rows, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out),
                       tables, capacity, status) == cudaSuccess ? 0 : -2;
}

}  // namespace forge
