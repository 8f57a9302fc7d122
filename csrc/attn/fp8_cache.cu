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
#include <type_traits>

#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/ptx.cuh"

namespace forge {

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
  int T, nq, nkv, block_size, num_slots;
  unsigned* status;
};

// Eight lanes per head, lane j of them has entries 8j.. and 64 + 8j.., the pairs that the rotation mixes; a warp has a set of four heads.
enum { kStoreQ = 0, kStoreK = 1, kStoreV = 2 };
__device__ __forceinline__ int fp8_store_kind(const Fp8Store& a, int h) { return h < a.nq ? kStoreQ : h < a.nq + a.nkv ? kStoreK : kStoreV; }

// raw: the head's entries; cs: cos and sin of the token at 8j and 64 + 8j, null: no rotation; row0: the slot's row of KV head 0.
template <int kKind>
__device__ __forceinline__ void fp8_store_head(const Fp8Store& a, int t, int h, const uint4* raw, const Fp8Weights& w, const float* cs, bool slot_ok,
                                               size_t row0, int lane) {
  const int j = lane & 7;
  const unsigned octet = 0xFFu << (lane & 24);           // the lanes of a head; the four heads of a set may be of different kinds
  float x[8], y[8];
  unpack8(raw[0], x);
  unpack8(raw[1], y);
  if constexpr (kKind != kStoreV) fp8_norm_rotate(x, y, w, (kKind == kStoreQ ? a.qw : a.kw) != nullptr, a.eps, cs, octet);
  if constexpr (kKind == kStoreQ) {
    __nv_bfloat16* dst = a.q_out + (static_cast<size_t>(t) * a.nq + h) * kFp8D + 8 * j;
    *reinterpret_cast<uint4*>(dst) = pack8(x);
    *reinterpret_cast<uint4*>(dst + 64) = pack8(y);
  } else {
    uint2 code[2];
    const uint32_t b = fp8_quantise(x, y, octet, code);
    if (!slot_ok) return;
    const size_t row = row0 + static_cast<size_t>(kKind == kStoreV ? h - a.nq - a.nkv : h - a.nq) * a.block_size;
    uint8_t* dst = (kKind == kStoreV ? a.v_codes : a.k_codes) + row * kFp8D + 8 * j;
    *reinterpret_cast<uint2*>(dst) = code[0];
    *reinterpret_cast<uint2*>(dst + 64) = code[1];
    if (j == 0) (kKind == kStoreV ? a.v_scales : a.k_scales)[row] = static_cast<uint8_t>(b);
  }
}
// Any head, weights included.
template <bool kVec>
__device__ __forceinline__ void fp8_store_any(const Fp8Store& a, int t, int h, const uint4* raw, const float* cs, bool slot_ok, size_t row0, int lane) {
  Fp8Weights w;
  const int kind = fp8_store_kind(a, h);
  if (kind == kStoreQ) {
    w.load<kVec>(a.qw, lane & 7);
    fp8_store_head<kStoreQ>(a, t, h, raw, w, cs, slot_ok, row0, lane);
  } else if (kind == kStoreK) {
    w.load<kVec>(a.kw, lane & 7);
    fp8_store_head<kStoreK>(a, t, h, raw, w, cs, slot_ok, row0, lane);
  } else {
    fp8_store_head<kStoreV>(a, t, h, raw, w, cs, slot_ok, row0, lane);
  }
}

// The slot's row of KV head 0; false: no such slot, or none.
__device__ __forceinline__ bool fp8_slot_row(const Fp8Store& a, int slot, size_t& row0) {
  const int block = slot / a.block_size;
  row0 = static_cast<size_t>(block) * a.nkv * a.block_size + (slot - block * a.block_size);
  return slot >= 0 && slot < a.num_slots;
}
__device__ __forceinline__ int fp8_angle_row(const Fp8Store& a, int position) { return min(max(position, 0), a.rope_rows - 1); }

// Few tokens, or rows that are not aligned: a warp per set of heads.
template <bool kVec>
__global__ void __launch_bounds__(128) fp8_store_kernel(const Fp8Store a) {
  pdl_launch_dependents();
  pdl_wait();
  const int heads = a.nq + 2 * a.nkv, sets = (heads + 3) / 4;
  const long long wid = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (wid >= static_cast<long long>(a.T) * sets) return;
  const int lane = threadIdx.x & 31, j = lane & 7;
  const int t = static_cast<int>(wid / sets), h = static_cast<int>(wid - static_cast<long long>(t) * sets) * 4 + (lane >> 3);
  const __nv_bfloat16* src = a.qkv + static_cast<size_t>(t) * a.ld + static_cast<size_t>(min(h, heads - 1)) * kFp8D + 8 * j;
  const uint4 raw[2] = {load8<kVec>(src), load8<kVec>(src + 64)};
  const int slot = a.slots[t];
  if (slot >= a.num_slots && lane == 0) set_status(a.status, kStatusBadIndex);
  size_t row0;
  const bool slot_ok = fp8_slot_row(a, slot, row0);
  const float* cs = a.rope == nullptr ? nullptr : a.rope + static_cast<size_t>(fp8_angle_row(a, a.positions[t])) * kFp8D + 8 * j;
  if (h < heads) fp8_store_any<kVec>(a, t, h, raw, cs, slot_ok, row0, lane);
}

// Many tokens: a loading warp brings whole rows of the projection and their angles into a ring by bulk copies, the others take sets of heads
// from it, so that memory is asked ahead of the arithmetic whatever that takes.  Persistent, two CTAs per SM; shared memory is asked for
// so that no third fits beside them: of equal shares none may wait for a CTA that another SM would have had room for.
constexpr int kStoreRingTokens = 2048, kStoreRingSets = 8;         // from which on
constexpr int kStoreWarps = 12, kStoreCtasPerSm = 2, kStoreSmem = 108 * 1024, kStoreMaxStages = 8;

__global__ void __launch_bounds__(32 * (kStoreWarps + 1), kStoreCtasPerSm) fp8_store_ring_kernel(const Fp8Store a, int stages) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kStoreMaxStages], empty[kStoreMaxStages];
  __shared__ int s_slot[kStoreMaxStages];
  const int heads = a.nq + 2 * a.nkv, sets = (heads + 3) / 4, row_bytes = heads * kFp8D * 2, stage_bytes = row_bytes + kFp8D * 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, consumers = (blockDim.x >> 5) - 1;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], consumers);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  int s = 0, phase = 0;
  const auto next = [&] {
    if (++s == stages) {
      s = 0;
      phase ^= 1;
    }
  };
  if (warp == consumers) {
    bool ok = true;
    int issued = 0;                                      // rows that may be on their way, at most as many as there are stages
    for (int t0 = blockIdx.x; t0 < a.T && ok; t0 += 32 * gridDim.x) {             // slots and positions of 32 tokens at a time
      const int mine = t0 + lane * gridDim.x;
      const int slot = mine < a.T ? a.slots[mine] : -1, at = mine < a.T && a.rope != nullptr ? fp8_angle_row(a, a.positions[mine]) : 0;
      if (slot >= a.num_slots) set_status(a.status, kStatusBadIndex);
      for (int i = 0; i < 32 && ok; ++i) {
        const int t = t0 + i * gridDim.x, to = __shfl_sync(0xffffffffu, slot, i), angle = __shfl_sync(0xffffffffu, at, i);
        if (t >= a.T) break;
        if (lane == 0) {
          ok = mbar_wait_parked(&empty[s], phase ^ 1, a.status);
          if (ok) {
            uint8_t* stage = smem + s * stage_bytes;
            s_slot[s] = to;
            mbar_expect_tx(&full[s], a.rope != nullptr ? stage_bytes : row_bytes);
            bulk_load(stage, a.qkv + static_cast<size_t>(t) * a.ld, row_bytes, &full[s]);
            if (a.rope != nullptr) bulk_load(stage + row_bytes, a.rope + static_cast<size_t>(angle) * kFp8D, kFp8D * 4, &full[s]);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        issued = min(issued + 1, stages);
        next();
      }
    }
    // none may be on its way to a CTA that has left because a wait had run out
    for (int i = 1; i <= issued && lane == 0; ++i) {
      const int at = s - i;
      if (!mbar_wait_parked(&full[at < 0 ? at + stages : at], at < 0 ? phase ^ 1 : phase, a.status)) break;
    }
    return;
  }
  const int j = lane & 7;
  const auto walk = [&](auto&& take) {                   // take(token, stage, angles, slot's row, whether there is one)
    for (int t = blockIdx.x; t < a.T; t += gridDim.x, next()) {
      if (!mbar_wait(&full[s], phase, a.status)) return;
      const uint8_t* stage = smem + s * stage_bytes;
      size_t row0;
      const bool slot_ok = fp8_slot_row(a, s_slot[s], row0);
      take(t, stage, a.rope == nullptr ? nullptr : reinterpret_cast<const float*>(stage + row_bytes) + 8 * j, row0, slot_ok);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
  };
  // one set to a warp, of four heads of one kind: weights and kind are found out once
  const int h = 4 * warp + (lane >> 3), kind = fp8_store_kind(a, min(h, heads - 1));
  const auto same = [&](auto k) {
    Fp8Weights w;
    if (k.value != kStoreV) w.load<true>(k.value == kStoreQ ? a.qw : a.kw, j);
    walk([&](int t, const uint8_t* stage, const float* cs, size_t row0, bool slot_ok) {
      const uint4* src = reinterpret_cast<const uint4*>(stage + h * kFp8D * 2) + j;
      const uint4 raw[2] = {src[0], src[8]};
      fp8_store_head<k.value>(a, t, h, raw, w, cs, slot_ok, row0, lane);
    });
  };
  const int first = __shfl_sync(0xffffffffu, kind, 0);   // (by all lanes, whatever their head)
  if (sets <= consumers && __all_sync(0xffffffffu, h < heads && kind == first)) {
    if (kind == kStoreQ) same(std::integral_constant<int, kStoreQ>{});
    else if (kind == kStoreK) same(std::integral_constant<int, kStoreK>{});
    else same(std::integral_constant<int, kStoreV>{});
    return;
  }
  walk([&](int t, const uint8_t* stage, const float* cs, size_t row0, bool slot_ok) {
    for (int set = warp; set < sets; set += consumers) {
      const int head = 4 * set + (lane >> 3);
      if (head < heads) {
        const uint4* src = reinterpret_cast<const uint4*>(stage + head * kFp8D * 2) + j;
        const uint4 raw[2] = {src[0], src[8]};
        fp8_store_any<true>(a, t, head, raw, cs, slot_ok, row0, lane);
      }
    }
  });
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
  a.T = T; a.nq = nq; a.nkv = nkv; a.block_size = block_size; a.num_slots = static_cast<int>(num_slots); a.status = status;
  const auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = ld % 8 == 0 && aligned(qkv) && aligned(qw) && aligned(kw);
  const int heads = nq + 2 * nkv, sets = (heads + 3) / 4, stage = heads * kFp8D * 2 + kFp8D * 4;
  const int stages = std::min(kStoreMaxStages, kStoreSmem / stage);
  // Measured, a warp per set / ring, us: 32 + 16 heads, 1024 tokens 6.2 / 6.1, 2048: 12.8 / 10.5, 4001: 23.8 / 18.7, 8192: 45 / 35; 16 + 16 heads, 1024:
  // 4.8 / 5.1, 2048: 7.8 / 8.1, 4001: 16.4 / 15.0; 64 + 16 heads (two sets to a warp), 1024: 9.7 / 11.3, 2048: 20.2 / 20.9, 4001: 39 / 36; 8 + 2 heads
  // (three warps at work), 4001: 6.8 / 16.1.  One number for all: at 2048 tokens it gains with 32 + 16 heads and loses 3 to 4 % with the other two.
  if (vec && stages >= 3 && T >= kStoreRingTokens && sets >= kStoreRingSets) {
    FORGE_ENSURE_DYN_SMEM(fp8_store_ring_kernel, kStoreSmem);
    const int ctas = std::min(T, kStoreCtasPerSm * device_sm_count());
    return launch_kernel(fp8_store_ring_kernel, dim3(ctas), dim3(32 * (std::min(sets, kStoreWarps) + 1)), kStoreSmem, stream, 0, a, stages) == cudaSuccess
               ? 0 : -2;
  }
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(T) * sets + 3) / 4));
  return launch_kernel(vec ? fp8_store_kernel<true> : fp8_store_kernel<false>, grid, dim3(128), 0, stream, 0, a) == cudaSuccess ? 0 : -2;
}

// ---------------------------------------------------------------------------------------------------------
// Pages of sequences, in order, as bf16.  A CTA takes `rows` token rows of one page of one head of K or V.  Lengths, table entry and, once the
// latter is there, the codes are asked for one after the other; where the page goes is found out meanwhile.  Bound by memory.
// A CTA may be there while the kernel before still writes the cache, so nothing that is read here may pass for constant over the kernel's life
// (no __restrict__): the loads stay behind the wait.
// ---------------------------------------------------------------------------------------------------------
constexpr int kExpandThreads = 128, kExpandLoads = 8;           // 28 x 100 .. 1024 in pages of 256 / of 64: 256 threads 19.6 / 25.3 us, 128 17.9 / 16.3, 64 18.6 / 17.4

struct Fp8Expand {
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int *block_tables, *lens;
  int table_width, num_blocks, nkv, block_size;
  int rows;                                             // of a CTA: at most kExpandLoads * kExpandThreads / 16
  __nv_bfloat16 *k_out, *v_out;
  int* tables;
  int capacity;
  unsigned* status;
};

__global__ void __launch_bounds__(kExpandThreads) fp8_expand_kernel(const Fp8Expand a) {
  __shared__ int red[kExpandThreads / 32];
  const int seq = blockIdx.y, page = blockIdx.x, block_size = a.block_size, rows = a.rows;
  const int parts = block_size / rows, z = blockIdx.z;
  const int part = z % parts, kvh = z / parts % a.nkv, is_v = z / parts / a.nkv;
  const int cap = a.table_width * block_size;
  const bool scribe = z == 0 && threadIdx.x == 0;       // writes the page's table entry
  pdl_launch_dependents();
  pdl_wait();
  int len = a.lens[seq];
  int blk = a.block_tables[static_cast<size_t>(seq) * a.table_width + page];
  int before = 0;                                       // pages of the sequences before this one
  for (int i = threadIdx.x; i < seq; i += kExpandThreads) before += (min(max(a.lens[i], 0), cap) + block_size - 1) / block_size;
  if (len > cap) {
    if (scribe && page == 0) set_status(a.status, kStatusBadIndex);
    len = cap;
  }
  int* entry = a.tables + static_cast<size_t>(seq) * a.table_width + page;
  if (page * block_size >= len) {
    if (scribe) *entry = -1;
    return;
  }
  if (blk < 0 || blk >= a.num_blocks) {
    if (scribe) set_status(a.status, kStatusBadIndex);
    blk = 0;
  }
  const size_t row0 = (static_cast<size_t>(blk) * a.nkv + kvh) * block_size + part * rows;
  const int live = min(len - page * block_size - part * rows, rows);
  const uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + row0 * kFp8D;
  const uint8_t* scales = (is_v ? a.v_scales : a.k_scales) + row0;
  uint2 raw[kExpandLoads];                              // 8 codes each; zeros behind the last token
  uint32_t scale[kExpandLoads];
#pragma unroll
  for (int k = 0; k < kExpandLoads; ++k) {
    const int i = threadIdx.x + k * kExpandThreads;
    const bool in = i >> 4 < live;
    raw[k] = in ? *reinterpret_cast<const uint2*>(codes + static_cast<size_t>(i) * 8) : make_uint2(0, 0);
    scale[k] = in ? scales[i >> 4] : 0u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int i = 0; i < kExpandThreads / 32; ++i) before += red[i];
  const int to = before + page;
  if (to >= a.capacity) {
    if (scribe) {
      set_status(a.status, kStatusBadIndex);
      *entry = -1;
    }
    return;
  }
  if (scribe) *entry = to;
  __nv_bfloat16* out = (is_v ? a.v_out : a.k_out) + ((static_cast<size_t>(to) * a.nkv + kvh) * block_size + part * rows) * kFp8D;
#pragma unroll
  for (int k = 0; k < kExpandLoads; ++k) {
    const int i = threadIdx.x + k * kExpandThreads;
    if (i >= rows * 16) break;
    const float m = fp8_scale(scale[k]);
    const float2 f0 = fp8_to_float2(raw[k].x), f1 = fp8_to_float2(raw[k].x >> 16), f2 = fp8_to_float2(raw[k].y), f3 = fp8_to_float2(raw[k].y >> 16);
    *reinterpret_cast<uint4*>(out + static_cast<size_t>(i) * 8) =
        make_uint4(pack_bf16x2(f0.x * m, f0.y * m), pack_bf16x2(f1.x * m, f1.y * m), pack_bf16x2(f2.x * m, f2.y * m), pack_bf16x2(f3.x * m, f3.y * m));
  }
}

// k_out, v_out [capacity][nkv][block_size][128]; tables [num_seqs][table_width] gets the page numbers in them, -1 behind a sequence's last.
// A sequence's pages follow one another, and the sequences too; entries behind a sequence's last token are zero.
extern "C" int forge_fp8_expand(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const int* block_tables,
                                const int* lens, int num_seqs, int table_width, int num_blocks, int nkv, int block_size, void* k_out, void* v_out,
                                int* tables, int capacity, unsigned* status, cudaStream_t stream) {
  if (num_seqs <= 0 || table_width <= 0) return 0;
  if (block_size < 1 || num_seqs > 65535) return -1;
  // a CTA's rows: 64, or 32 where there are few pages (64 / 32, us: 1 x 100 tokens 1.97 / 1.69, 1 x 700 2.28 / 2.57, 1 x 2000 3.88 / 3.34: two of the
  // three gain more than the other loses)
  int rows = std::min(block_size, kExpandLoads * kExpandThreads / 16);
  while (rows > 32 && 2ll * capacity * nkv * (block_size / rows) < 4 * device_sm_count()) rows /= 2;
  const long long z = 2ll * nkv * (block_size / rows);
  if (z > 65535) return -1;
  const dim3 grid(static_cast<unsigned>(table_width), static_cast<unsigned>(num_seqs), static_cast<unsigned>(z));
  const Fp8Expand a{static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(k_scales), static_cast<const uint8_t*>(v_codes),
                    static_cast<const uint8_t*>(v_scales), block_tables, lens, table_width, num_blocks, nkv, block_size, rows,
                    static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), tables, capacity, status};
  return launch_kernel(fp8_expand_kernel, grid, dim3(kExpandThreads), 0, stream, 0, a) == cudaSuccess ? 0 : -2;
}

}  // namespace forge
