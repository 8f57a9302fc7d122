// Writing and reading an 8-bit KV cache (layout and scales: include/fp8_cache.cuh).
//
//   store    split of the packed qkv row, per-head RMS norm of q and k, rotation, quantisation of k and v into the paged cache.
//            What the bf16 cache's kernel does (elt/elementwise.cu), but everything between the projection and the one rounding of a
//            result stays in fp32.
//   expand   pages of sequences in order as bf16 pages, for attention of prompts: exact, so a prompt attends to the same
//            values whether its prefix was cached or written a moment ago.
//
// No counterpart in the reference, whose cache has the model's type.
#include <algorithm>

#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"

namespace forge {

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
// The larger one, NaN if one is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
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
  unsigned* status;
};

// Eight lanes per head, lane j of them has entries 8j.. and 64 + 8j.., the pairs that the rotation mixes; a warp works on kSets sets of
// four heads of a token, all of whose loads are under way at once.  Norm weight and rotation make one linear map of a pair, computed once for
// all query heads and once for all key heads of a token; the root follows it, for keys in the factor that brings entries to codes.
// Bound by memory: qkv read once, q and the codes written once.
template <bool kVec, int kSets>
__global__ void __launch_bounds__(128) fp8_store_kernel(const Fp8Store a) {
  pdl_launch_dependents();
  pdl_wait();
  const int heads = a.nq + 2 * a.nkv, groups = (heads + 4 * kSets - 1) / (4 * kSets);
  const long long wid = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (wid >= static_cast<long long>(a.T) * groups) return;
  const int lane = threadIdx.x & 31, j = lane & 7, sub = lane >> 3;
  const unsigned octet = 0xFFu << (8 * sub);             // the lanes of a head; the four heads of a set may be of different kinds
  const int t = static_cast<int>(wid / groups), h0 = static_cast<int>(wid - static_cast<long long>(t) * groups) * 4 * kSets + sub;
  uint4 raw[kSets][2];
#pragma unroll
  for (int k = 0; k < kSets; ++k) {
    const __nv_bfloat16* src = a.qkv + static_cast<size_t>(t) * a.ld + static_cast<size_t>(min(h0 + 4 * k, heads - 1)) * kFp8D + 8 * j;
    raw[k][0] = load8<kVec>(src);
    raw[k][1] = load8<kVec>(src + 64);
  }
  const long long slot = a.slots[t];
  const bool slot_ok = slot >= 0 && slot < a.num_slots;
  if (slot >= a.num_slots && lane == 0) set_status(a.status, kStatusBadIndex);
  const long long block = slot / a.block_size;
  const size_t row0 = static_cast<size_t>(block) * a.nkv * a.block_size + (slot - block * a.block_size);        // of KV head 0
  const float* cs = a.rope == nullptr ? nullptr : a.rope + static_cast<size_t>(min(max(a.positions[t], 0), a.rope_rows - 1)) * kFp8D + 8 * j;

  float xx[8], xy[8], yx[8], yy[8];                      // x' = x xx - y xy,  y' = y yy + x yx
  int kind = -1;                                         // 0: for query heads, 1: for key heads
#pragma unroll
  for (int k = 0; k < kSets; ++k) {
    const int h = h0 + 4 * k;
    if (h >= heads) break;
    const bool is_q = h < a.nq, is_v = h >= a.nq + a.nkv;
    float x[8], y[8], inv = 1.f;
    unpack8(raw[k][0], x);
    unpack8(raw[k][1], y);
    if (!is_v) {
      const __nv_bfloat16* w = is_q ? a.qw : a.kw;
      if (kind != (is_q ? 0 : 1)) {
        kind = is_q ? 0 : 1;
#pragma unroll
        for (int i = 0; i < 8; ++i) xx[i] = yy[i] = 1.f;
        if (w != nullptr) {
          unpack8(load8<kVec>(w + 8 * j), xx);
          unpack8(load8<kVec>(w + 64 + 8 * j), yy);
        }
        if (cs != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 c = *reinterpret_cast<const float4*>(cs + i), s = *reinterpret_cast<const float4*>(cs + 64 + i);
            const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              yx[i + e] = xx[i + e] * sv[e];
              xy[i + e] = yy[i + e] * sv[e];
              xx[i + e] *= cv[e];
              yy[i + e] *= cv[e];
            }
          }
        }
      }
      if (w != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) ss += __shfl_xor_sync(octet, ss, o);
        inv = rsqrtf(ss * (1.f / kFp8D) + a.eps);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x[i] * xx[i], v = y[i] * yy[i];
        if (cs != nullptr) {
          const float x0 = x[i];
          x[i] = fmaf(-y[i], xy[i], u);
          y[i] = fmaf(x0, yx[i], v);
        } else {
          x[i] = u;
          y[i] = v;
        }
      }
    }
    if (is_q) {
      __nv_bfloat16* dst = a.q_out + (static_cast<size_t>(t) * a.nq + h) * kFp8D + 8 * j;
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(x[0] * inv, x[1] * inv), pack_bf16x2(x[2] * inv, x[3] * inv), pack_bf16x2(x[4] * inv, x[5] * inv),
                                                  pack_bf16x2(x[6] * inv, x[7] * inv));
      *reinterpret_cast<uint4*>(dst + 64) = make_uint4(pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv),
                                                       pack_bf16x2(y[4] * inv, y[5] * inv), pack_bf16x2(y[6] * inv, y[7] * inv));
      continue;
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_or_nan(amax, max_or_nan(fabsf(x[i]), fabsf(y[i])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max_or_nan(amax, __shfl_xor_sync(octet, amax, o));
    if (!slot_ok) continue;
    const size_t row = row0 + static_cast<size_t>(is_v ? h - a.nq - a.nkv : h - a.nq) * a.block_size;
    const uint32_t b = fp8_scale_byte(abs_bits(amax * inv));
    uint2 code[2] = {make_uint2(kCodesNan, kCodesNan), make_uint2(kCodesNan, kCodesNan)};
    if (b != kScaleNan) {
      const float m = fp8_inverse_scale(b) * inv;
      code[0] = make_uint2(fp8_pack(x[0] * m, x[1] * m, x[2] * m, x[3] * m), fp8_pack(x[4] * m, x[5] * m, x[6] * m, x[7] * m));
      code[1] = make_uint2(fp8_pack(y[0] * m, y[1] * m, y[2] * m, y[3] * m), fp8_pack(y[4] * m, y[5] * m, y[6] * m, y[7] * m));
    }
    uint8_t* dst = (is_v ? a.v_codes : a.k_codes) + row * kFp8D + 8 * j;
    *reinterpret_cast<uint2*>(dst) = code[0];
    *reinterpret_cast<uint2*>(dst + 64) = code[1];
    if (j == 0) (is_v ? a.v_scales : a.k_scales)[row] = static_cast<uint8_t>(b);
  }
}

template <bool kVec, int kSets>
static int launch_store(const Fp8Store& a, cudaStream_t stream) {
  const int groups = (a.nq + 2 * a.nkv + 4 * kSets - 1) / (4 * kSets);
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.T) * groups + 3) / 4));
  return launch_kernel(fp8_store_kernel<kVec, kSets>, grid, dim3(128), 0, stream, 0, a) == cudaSuccess ? 0 : -2;
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
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = ld % 8 == 0 && aligned(qkv) && aligned(qw) && aligned(kw);
  if (!vec) return launch_store<false, 1>(a, stream);
  return T < 512 ? launch_store<true, 1>(a, stream) : T < 2048 ? launch_store<true, 2>(a, stream) : launch_store<true, 4>(a, stream);
}

// ---------------------------------------------------------------------------------------------------------
// Pages of sequences, in order, as bf16.  A CTA takes `rows` token rows of one page of one head of K or V.  Lengths, table entry and, once the
// latter is there, the codes are asked for one after the other; where the page goes is found out meanwhile.  Bound by memory.
// ---------------------------------------------------------------------------------------------------------
constexpr int kExpandThreads = 256, kExpandLoads = 4;

__global__ void __launch_bounds__(kExpandThreads) fp8_expand_kernel(
    const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ k_scales, const uint8_t* __restrict__ v_codes,
    const uint8_t* __restrict__ v_scales, const int* __restrict__ block_tables, const int* __restrict__ lens, int table_width, int num_blocks,
    int nkv, int block_size, int rows, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out, int* __restrict__ tables,
    int capacity, unsigned* status) {
  __shared__ int red[kExpandThreads / 32];
  const int seq = blockIdx.y, page = blockIdx.x;
  const int parts = block_size / rows, z = blockIdx.z;
  const int part = z % parts, kvh = z / parts % nkv, is_v = z / parts / nkv;
  const int cap = table_width * block_size;
  const bool scribe = z == 0 && threadIdx.x == 0;       // writes the page's table entry
  pdl_launch_dependents();
  pdl_wait();
  int len = lens[seq];
  int blk = block_tables[static_cast<size_t>(seq) * table_width + page];
  int before = 0;                                       // pages of the sequences before this one
  for (int i = threadIdx.x; i < seq; i += kExpandThreads) before += (min(max(lens[i], 0), cap) + block_size - 1) / block_size;
  if (len > cap) {
    if (scribe && page == 0) set_status(status, kStatusBadIndex);
    len = cap;
  }
  int* entry = tables + static_cast<size_t>(seq) * table_width + page;
  if (page * block_size >= len) {
    if (scribe) *entry = -1;
    return;
  }
  if (blk < 0 || blk >= num_blocks) {
    if (scribe) set_status(status, kStatusBadIndex);
    blk = 0;
  }
  const size_t row0 = (static_cast<size_t>(blk) * nkv + kvh) * block_size + part * rows;
  const int live = min(len - page * block_size - part * rows, rows);
  const uint8_t* codes = (is_v ? v_codes : k_codes) + row0 * kFp8D;
  const uint8_t* scales = (is_v ? v_scales : k_scales) + row0;
  uint4 raw[kExpandLoads];
  uint32_t scale[kExpandLoads];
  const auto fetch = [&](int i0) {                      // 16 codes each; zeros behind the last token
#pragma unroll
    for (int k = 0; k < kExpandLoads; ++k) {
      const int i = i0 + k * kExpandThreads;
      const bool in = i >> 3 < live;
      raw[k] = in ? *reinterpret_cast<const uint4*>(codes + static_cast<size_t>(i) * 16) : make_uint4(0, 0, 0, 0);
      scale[k] = in ? scales[i >> 3] : 0u;
    }
  };
  fetch(threadIdx.x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int i = 0; i < kExpandThreads / 32; ++i) before += red[i];
  const int to = before + page;
  if (to >= capacity) {
    if (scribe) {
      set_status(status, kStatusBadIndex);
      *entry = -1;
    }
    return;
  }
  if (scribe) *entry = to;
  __nv_bfloat16* out = (is_v ? v_out : k_out) + ((static_cast<size_t>(to) * nkv + kvh) * block_size + part * rows) * kFp8D;
  for (int i0 = threadIdx.x; i0 < rows * 8; i0 += kExpandLoads * kExpandThreads) {
    if (i0 != threadIdx.x) fetch(i0);
#pragma unroll
    for (int k = 0; k < kExpandLoads; ++k) {
      const int i = i0 + k * kExpandThreads;
      if (i >= rows * 8) break;
      const float m = fp8_scale(scale[k]);
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
      uint32_t o[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = fp8_to_float2(w[e]), g = fp8_to_float2(w[e] >> 16);
        o[2 * e] = pack_bf16x2(f.x * m, f.y * m);
        o[2 * e + 1] = pack_bf16x2(g.x * m, g.y * m);
      }
      uint4* dst = reinterpret_cast<uint4*>(out + static_cast<size_t>(i) * 16);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

// k_out, v_out [capacity][nkv][block_size][128]; tables [num_seqs][table_width] gets the page numbers in them, -1 behind a sequence's last.
// A sequence's pages follow one another, and the sequences too; entries behind a sequence's last token are zero.
extern "C" int forge_fp8_expand(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const int* block_tables,
                                const int* lens, int num_seqs, int table_width, int num_blocks, int nkv, int block_size, void* k_out, void* v_out,
                                int* tables, int capacity, unsigned* status, cudaStream_t stream) {
  if (num_seqs <= 0 || table_width <= 0) return 0;
  if (block_size < 1 || num_seqs > 65535) return -1;
  // a CTA's rows: a page's, or a part of them where there are few pages
  int rows = std::min(block_size, 32 * kExpandLoads);
  while (rows > 32 && 2ll * capacity * nkv * (block_size / rows) < 4 * device_sm_count()) rows /= 2;
  const long long z = 2ll * nkv * (block_size / rows);
  if (z > 65535) return -1;
  const dim3 grid(static_cast<unsigned>(table_width), static_cast<unsigned>(num_seqs), static_cast<unsigned>(z));
  return launch_kernel(fp8_expand_kernel, grid, dim3(kExpandThreads), 0, stream, 0, static_cast<const uint8_t*>(k_codes),
                       static_cast<const uint8_t*>(k_scales), static_cast<const uint8_t*>(v_codes), static_cast<const uint8_t*>(v_scales), block_tables,
                       lens, table_width, num_blocks, nkv, block_size, rows, static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out),
                       tables, capacity, status) == cudaSuccess ? 0 : -2;
}

}  // namespace forge
