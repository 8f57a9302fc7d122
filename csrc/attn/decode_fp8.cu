// Attention of one new token per sequence over a paged 8-bit cache (include/fp8_cache.cuh).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m),   c = scale log2(e),   m = max_j c q.k_j
//
// Work and its split.  An item is a sequence and a KV head with up to eight of its query heads (larger groups take several).  The
// tiles of 64 tokens of all items, in order, are dealt out equally to three CTAs per SM: CTA i of C takes tiles [N i / C, N (i + 1) / C), so
// short and long contexts, few and many sequences fill the GPU alike.  An item inside one CTA is finished there; the parts of one that
// is cut are joined by a second kernel.  Lengths are read on the device, so the launch fits a CUDA graph whatever they become.
//
// A tile.  One warp loads (2-D TMA boxes of 128-byte rows with the 128-byte swizzle; scale bytes by bulk copies; a ring of three stages that
// never drains across items), four take 16 tokens of it each, with maximum, sum and results of their own until the item's end:
//   S^T [16 tokens x 8 heads] = K Q^T,   O^T [128 dims x 8 heads] += V^T P^T,   mma.sync m16n8k16, fp16 operands, fp32 sums.
// Codes of e4m3 are exact in fp16.  Which entries of K stand at which place of the inner dimension is free as long as Q's stand there too, and so is the
// order of the rows of O^T: a lane takes 32 consecutive entries of a key and 16 of a value with 16-byte reads that touch every
// bank once, and converts them in place; V^T needs no transposing load, two tokens' bytes are interleaved instead.
//   Queries are brought to [2^14, 2^15) by a power of two per head, which keeps every bit of their bf16 down to 2^-31 of the largest entry.
//   A value's scale 2^e goes into its weight's exponent: w_j = 2^(c q.k_j + e_j - u + 7), u a maximum of its own, and the weight into fp16 with 11 bits
//   (half a step 2^-11, against 2^-8 of the bf16 result): a value that counts is never lost beside one with a larger scale that does not.  The
//   sum of the p_j is kept in fp32 and without that rounding.  m and u move only when they are exceeded by 8, so w_j <= 2^15 and products are
//   rescaled rarely.
//
// What is behind a sequence's last token never counts: its scores, weights and value bytes are replaced, whatever they are.
// Bound by memory: 258 bytes per key and KV head.
#include <algorithm>

#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/mma_sync.cuh"
#include "../include/ptx.cuh"

namespace forge {

constexpr int kF8Tile = 64;                            // tokens
constexpr int kF8Half = kF8Tile * kFp8D;               // bytes of K or V codes of a tile
constexpr int kF8Stages = 3;
constexpr int kF8CtasPerSm = 3;
constexpr int kF8Threads = 160;                        // four consumer warps and a producer
constexpr int kF8Seqs = 512;                           // sequences of a launch
constexpr int kF8Heads = 8;                            // query heads of an item
constexpr float kF8Rise = 8.f;                         // how far a score may exceed the maximum in use
constexpr float kF8Top = 7.f;                          // weights are at most 2^(7 + 8)

struct Fp8Decode {
  const __nv_bfloat16* q;
  const uint8_t *k_scales, *v_scales;
  const int *block_tables, *lens;
  __nv_bfloat16* out;
  float *part_o, *part_ml;                             // [2 CTAs][G][128], [2 CTAs][G][2]: of a CTA the part that continues an item, then the one that is cut
  int* tiles_before;                                   // [B + 1], for the joining kernel
  int B, nq, nkv, group, G, slices, block_size, table_width, num_blocks;
  float scale_log2;
  unsigned* status;
};

// The CTAs that get tiles: all, or as many as there are tiles.
__device__ __forceinline__ int f8_workers(int tiles) { return min(static_cast<int>(gridDim.x), tiles); }
__device__ __forceinline__ int f8_share(int tiles, int workers, int i) { return static_cast<int>(static_cast<long long>(tiles) * i / workers); }
// The worker that has tile t.
__device__ __forceinline__ int f8_owner(int tiles, int workers, int t) {
  return static_cast<int>((static_cast<long long>(t + 1) * workers - 1) / tiles);
}
// The last sequence with before[s] * items <= t.
__device__ __forceinline__ int f8_sequence(const int* before, int B, int items, int t) {
  int lo = 0, hi = B;                                  // before[lo] * items <= t < before[hi] * items
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] * items <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t f8_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float f8_max_over_tokens(float x) {           // lanes with the same l % 4
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float f8_sum_over_tokens(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}

constexpr int f8_smem(int G) {
  return 1024 + kF8Stages * (2 * kF8Half + 2 * kF8Tile) + 4 * G * kFp8D * 4 + 4 * 3 * G * 4 + (kF8Seqs + 1) * 4 + kF8Seqs * 4 + 2 * kF8Stages * 8 + 64;
}

__global__ void __launch_bounds__(kF8Threads, kF8CtasPerSm)
decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Fp8Decode a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_scales = smem + kF8Stages * 2 * kF8Half;                    // [stage][K, V][64]
  float* s_acc = reinterpret_cast<float*>(s_scales + kF8Stages * 2 * kF8Tile);      // [warp][G][128]
  float* s_m = s_acc + 4 * a.G * kFp8D;                                  // [warp][G]
  float* s_l = s_m + 4 * a.G;                                            // [warp][G]
  float* s_u = s_l + 4 * a.G;                                            // [warp][G]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(s_u + 4 * a.G);
  uint64_t* empty_bar = full_bar + kF8Stages;
  int* s_before = reinterpret_cast<int*>(empty_bar + kF8Stages);         // [B + 1] tiles of the sequences before
  int* s_len = s_before + kF8Seqs + 1;                                   // [B]
  __shared__ int s_warp[kF8Threads / 32];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    for (int s = 0; s < kF8Stages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 4);
    }
    fence_mbar_init();
  }
  pdl_wait();                                          // q, the cache and the step buffer come from predecessors

  // tiles of every sequence, and of those before it; four sequences per thread
  {
    constexpr int kPer = (kF8Seqs + kF8Threads - 1) / kF8Threads;
    const int cap = a.table_width * a.block_size;
    int n[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = threadIdx.x * kPer + e;
      int len = b < a.B ? a.lens[b] : 0;
      if (len > cap) {                                 // a corrupted length: clamped and reported
        set_status(a.status, kStatusBadIndex);
        len = cap;
      }
      len = max(len, 0);
      if (b < a.B) s_len[b] = len;
      n[e] = (len + kF8Tile - 1) / kF8Tile;
      sum += n[e];
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    if (lane == 31) s_warp[warp] = before;
    before -= sum;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before += s_warp[w];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = threadIdx.x * kPer + e;
      if (b <= a.B) s_before[b] = before;
      before += n[e];
    }
    __syncthreads();
  }
  const int items = a.nkv * a.slices, tiles = s_before[a.B] * items, workers = f8_workers(tiles);
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b <= a.B; b += kF8Threads) a.tiles_before[b] = s_before[b];
  const bool busy = static_cast<int>(blockIdx.x) < workers;
  const int t_begin = busy ? f8_share(tiles, workers, blockIdx.x) : 0, t_end = busy ? f8_share(tiles, workers, blockIdx.x + 1) : 0;

  if (warp == 4) {
    // ------------------------------------------------------------------ producer
    if (lane != 0 || t_begin >= t_end) return;
    int seq = f8_sequence(s_before, a.B, items, t_begin);
    int n = s_before[seq + 1] - s_before[seq];
    int item = (t_begin - s_before[seq] * items) / n, j = (t_begin - s_before[seq] * items) % n;
    const int rows = min(a.block_size, kF8Tile);
    for (int t = t_begin, use = 0; t < t_end; ++t, ++use) {
      const int s = use % kF8Stages, kvh = item / a.slices, left = s_len[seq] - j * kF8Tile;
      const int pages = min((left + rows - 1) / rows, kF8Tile / rows);
      const int* table = a.block_tables + static_cast<size_t>(seq) * a.table_width;
      if (!mbar_wait_parked(&empty_bar[s], ((use / kF8Stages) & 1) ^ 1, a.status)) return;
      mbar_expect_tx(&full_bar[s], pages * rows * 2 * (kFp8D + 1));
      uint8_t* stage = smem + s * 2 * kF8Half;
      uint8_t* scales = s_scales + s * 2 * kF8Tile;
      for (int p = 0; p < pages; ++p) {
        const int tok = j * kF8Tile + p * rows;
        int blk = table[tok / a.block_size];
        if (blk < 0 || blk >= a.num_blocks) {
          set_status(a.status, kStatusBadIndex);
          blk = 0;
        }
        const int row = (blk * a.nkv + kvh) * a.block_size + tok % a.block_size;
        tma_load_2d(stage + p * rows * kFp8D, &tm_k, &full_bar[s], 0, row);
        tma_load_2d(stage + kF8Half + p * rows * kFp8D, &tm_v, &full_bar[s], 0, row);
        bulk_load(scales + p * rows, a.k_scales + row, rows, &full_bar[s]);
        bulk_load(scales + kF8Tile + p * rows, a.v_scales + row, rows, &full_bar[s]);
      }
      if (++j == n) {
        j = 0;
        if (++item == items) {
          item = 0;
          do ++seq;
          while (seq < a.B && s_before[seq + 1] == s_before[seq]);
          if (seq < a.B) n = s_before[seq + 1] - s_before[seq];
        }
      }
    }
    return;
  }

  // -------------------------------------------------------------------- consumers (warps 0..3): 16 tokens of every tile each
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)    // rows without tokens: zeros
    if (s_len[b] == 0)
      for (int i = threadIdx.x; i < a.nq * kFp8D; i += 128) a.out[static_cast<size_t>(b) * a.nq * kFp8D + i] = __float2bfloat16_rn(0.f);
  const int g = lane >> 2, quad = lane & 3;            // S^T: rows g and g + 8, heads 2 quad and 2 quad + 1
  const int r0 = warp * 16;
  bool ok = true;                                      // once a wait has run out none is made any more, but every barrier still is
  int use = 0;
  for (int t = t_begin; t < t_end;) {
    const int seq = f8_sequence(s_before, a.B, items, t);
    const int n = s_before[seq + 1] - s_before[seq], first = t - s_before[seq] * items, item = first / n, j0 = first - item * n;
    const int count = min(n - j0, t_end - t), len = s_len[seq];
    const int head0 = (item / a.slices) * a.group + (item % a.slices) * a.G, heads = min(a.G, a.group - (item % a.slices) * a.G);
    // ---- queries: 32 consecutive entries of head g, as fp16 of a power of two
    uint32_t qh[16];
    float qf[2];                                         // of heads 2 quad, 2 quad + 1: back to scores in base 2
    {
      float x[32];
      uint32_t top = 0;
      const __nv_bfloat16* src = a.q + (static_cast<size_t>(seq) * a.nq + head0 + g) * kFp8D + 32 * quad;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 r = g < heads ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[8 * i + 2 * e] = bf16_lo(w[e]);
          x[8 * i + 2 * e + 1] = bf16_hi(w[e]);
        }
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) top = max(top, abs_bits(x[i]));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float up = __uint_as_float(min(268u - (top >> 23), 254u) << 23);       // 2^14 / 2^exponent, at most 2^127
#pragma unroll
      for (int i = 0; i < 16; ++i) qh[i] = f8_half2(x[2 * i] * up, x[2 * i + 1] * up);
      qf[0] = a.scale_log2 / __shfl_sync(0xffffffffu, up, 8 * quad);
      qf[1] = a.scale_log2 / __shfl_sync(0xffffffffu, up, 8 * quad + 4);
    }
    float m[2] = {-INFINITY, -INFINITY}, u[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    float o[8][4];                                       // [i][0], [i][1]: dim 16 g + 2 i of heads 2 quad, 2 quad + 1; [2], [3]: the dim after it
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    for (int i = 0; i < count; ++i, ++use) {
      const int s = use % kF8Stages, valid = len - (j0 + i) * kF8Tile;
      ok = ok && mbar_wait(&full_bar[s], (use / kF8Stages) & 1, a.status);
      if (r0 < valid) {
        const uint8_t* Ks = smem + s * 2 * kF8Half + r0 * kFp8D;
        const uint8_t* Vs = Ks + kF8Half;
        const uint8_t* sc = s_scales + s * 2 * kF8Tile + r0;
        const bool whole = r0 + 16 <= valid, in0 = r0 + g < valid, in1 = r0 + g + 8 < valid;
        // ---- scores
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = ((2 * quad + h) ^ g) << 4;
          const uint4 ka = *reinterpret_cast<const uint4*>(Ks + g * kFp8D + at), kb = *reinterpret_cast<const uint4*>(Ks + (g + 8) * kFp8D + at);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t f[4] = {fp8_to_half2(wa[e] & 0xFFFFu), fp8_to_half2(wb[e] & 0xFFFFu), fp8_to_half2(wa[e] >> 16), fp8_to_half2(wb[e] >> 16)};
            mma16816_f16(c[e & 1], f, qh[8 * h + 2 * e], qh[8 * h + 2 * e + 1]);
          }
        }
        const float k0 = fp8_scale(sc[g]), k1 = fp8_scale(sc[g + 8]);
        const uint32_t b0 = sc[kF8Tile + g], b1 = sc[kF8Tile + g + 8];
        float e0 = b0 == kScaleNan ? __uint_as_float(0x7FC00000u) : static_cast<float>(static_cast<int>(b0) - 127);
        float e1 = b1 == kScaleNan ? __uint_as_float(0x7FC00000u) : static_cast<float>(static_cast<int>(b1) - 127);
        float x[4] = {(c[0][0] + c[1][0]) * qf[0] * k0, (c[0][1] + c[1][1]) * qf[1] * k0, (c[0][2] + c[1][2]) * qf[0] * k1, (c[0][3] + c[1][3]) * qf[1] * k1};
        if (!whole) {
          if (!in0) x[0] = x[1] = -INFINITY, e0 = 0.f;
          if (!in1) x[2] = x[3] = -INFINITY, e1 = 0.f;
        }
        float y[4] = {x[0] + e0, x[1] + e0, x[2] + e1, x[3] + e1};
        // ---- maxima
        const float x0 = fmaxf(x[0], x[2]), x1 = fmaxf(x[1], x[3]), y0 = fmaxf(y[0], y[2]), y1 = fmaxf(y[1], y[3]);
        if (__any_sync(0xffffffffu, x0 > m[0] + kF8Rise || x1 > m[1] + kF8Rise || y0 > u[0] + kF8Rise || y1 > u[1] + kF8Rise)) {
          const float tops[4] = {f8_max_over_tokens(x0), f8_max_over_tokens(x1), f8_max_over_tokens(y0), f8_max_over_tokens(y1)};
#pragma unroll
          for (int h = 0; h < 2; ++h) {                  // each head decides by itself, so its bits do not depend on the others
            if (tops[h] > m[h] + kF8Rise) {
              l[h] *= ex2_approx(m[h] - tops[h]);        // 0 at first
              m[h] = tops[h];
            }
            if (tops[2 + h] > u[h] + kF8Rise) {
              const float down = ex2_approx(u[h] - tops[2 + h]);
#pragma unroll
              for (int d = 0; d < 8; ++d) {
                o[d][h] *= down;
                o[d][2 + h] *= down;
              }
              u[h] = tops[2 + h];
            }
          }
        }
        // ---- weights; without a finite score so far (NaN) any reference does
        const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
        l[0] += ex2_approx(x[0] - m0) + ex2_approx(x[2] - m0);           // -inf -> 0
        l[1] += ex2_approx(x[1] - m1) + ex2_approx(x[3] - m1);
        const float u0 = (u[0] == -INFINITY ? 0.f : u[0]) - kF8Top, u1 = (u[1] == -INFINITY ? 0.f : u[1]) - kF8Top;
        const uint32_t p0 = transpose8x8(f8_half2(ex2_approx(y[0] - u0), ex2_approx(y[1] - u1)));
        const uint32_t p1 = transpose8x8(f8_half2(ex2_approx(y[2] - u0), ex2_approx(y[3] - u1)));
        // ---- values: tokens 2 quad, 2 quad + 1 and eight further on, dims 16 g ..
        uint4 v[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int tok = 2 * quad + (h & 1) + 8 * (h >> 1);
          v[h] = *reinterpret_cast<const uint4*>(Vs + tok * kFp8D + ((g ^ (tok & 7)) << 4));
          if (!whole && r0 + tok >= valid) v[h] = make_uint4(0, 0, 0, 0);
        }
        const uint32_t w[4][4] = {{v[0].x, v[0].y, v[0].z, v[0].w}, {v[1].x, v[1].y, v[1].z, v[1].w}, {v[2].x, v[2].y, v[2].z, v[2].w}, {v[3].x, v[3].y, v[3].z, v[3].w}};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t lo = __byte_perm(w[0][e], w[1][e], h ? 0x7362 : 0x5140), hi = __byte_perm(w[2][e], w[3][e], h ? 0x7362 : 0x5140);
            const uint32_t f[4] = {fp8_to_half2(lo & 0xFFFFu), fp8_to_half2(lo >> 16), fp8_to_half2(hi & 0xFFFFu), fp8_to_half2(hi >> 16)};
            mma16816_f16(o[2 * e + h], f, p0, p1);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
    }
    // ---- join the warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] = f8_sum_over_tokens(l[h]);
      const int head = 2 * quad + h;
      if (head < heads) {
        float* dst = s_acc + (warp * a.G + head) * kFp8D + 16 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(o[2 * i][h], o[2 * i][2 + h], o[2 * i + 1][h], o[2 * i + 1][2 + h]);
        if (g == 0) {
          s_m[warp * a.G + head] = m[h];
          s_l[warp * a.G + head] = l[h];
          s_u[warp * a.G + head] = u[h];
        }
      }
    }
    named_barrier_sync(1, 128);
    const bool complete = count == n;
    const int d = threadIdx.x, slot = 2 * blockIdx.x + (j0 == 0 ? 1 : 0);
    for (int h = 0; h < heads; ++h) {
      float M = -INFINITY, U = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        M = fmaxf(M, s_m[w * a.G + h]);
        U = fmaxf(U, s_u[w * a.G + h]);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {                      // (a warp without a maximum has zeros, or NaN)
        const float mw = s_m[w * a.G + h], uw = s_u[w * a.G + h];
        L = fmaf(s_l[w * a.G + h], mw == -INFINITY ? 0.f : exp2f(mw - M), L);
        O = fmaf(s_acc[(w * a.G + h) * kFp8D + d], uw == -INFINITY ? 0.f : exp2f(uw - U), O);
      }
      const float y = L == 0.f ? 0.f : O / L * exp2f(U - M - kF8Top);
      if (complete) {
        a.out[(static_cast<size_t>(seq) * a.nq + head0 + h) * kFp8D + d] = __float2bfloat16_rn(y);
      } else {
        const size_t p = static_cast<size_t>(slot) * a.G + h;
        a.part_o[p * kFp8D + d] = y;
        if (d == 0) {
          a.part_ml[2 * p] = M;
          a.part_ml[2 * p + 1] = L;
        }
      }
    }
    named_barrier_sync(1, 128);                          // the joining area is the next item's
    t += count;
  }
}

// Joins the parts of items that were cut.  CTA i looks at the cut before worker i; the item's first cut does the work, one or more warps
// per head taking its parts in turn.
constexpr int kF8JoinWarps = 8;

__global__ void __launch_bounds__(32 * kF8JoinWarps) decode_fp8_join_kernel(const Fp8Decode a) {
  __shared__ float4 s_o[kF8JoinWarps][32];
  __shared__ float s_l[kF8JoinWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int items = a.nkv * a.slices, tiles = a.tiles_before[a.B] * items, workers = f8_workers(tiles), cut = blockIdx.x;
  if (cut < 1 || cut >= workers) return;
  const int t = f8_share(tiles, workers, cut), seq = f8_sequence(a.tiles_before, a.B, items, t);
  const int n = a.tiles_before[seq + 1] - a.tiles_before[seq], first = t - a.tiles_before[seq] * items, item = first / n, begin = t - (first - item * n);
  if (begin == t || f8_owner(tiles, workers, begin) != cut - 1) return;
  const int parts = f8_owner(tiles, workers, begin + n - 1) - cut + 2;   // of workers cut - 1 (its second slot), cut, ... (their first)
  const int slice = item % a.slices, heads = min(a.G, a.group - slice * a.G), head0 = (item / a.slices) * a.group + slice * a.G;
  const int per_head = a.G <= 1 ? 8 : a.G <= 2 ? 4 : a.G <= 4 ? 2 : 1;   // warps
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = warp / per_head, sub = warp % per_head;
  auto slot = [&](int i) { return static_cast<size_t>(i == 0 ? 2 * (cut - 1) + 1 : 2 * (cut + i - 1)) * a.G + head; };
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  if (head < heads) {
    for (int i = lane; i < parts; i += 32) M = fmaxf(M, a.part_ml[2 * slot(i)]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
#pragma unroll 4
    for (int i = sub; i < parts; i += per_head) {
      const size_t p = slot(i);
      const float mi = a.part_ml[2 * p], f = (mi == -INFINITY ? 0.f : exp2f(mi - M)) * a.part_ml[2 * p + 1];
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + p * kFp8D + 4 * lane);
      L += f;
      O.x = fmaf(f, v.x, O.x);
      O.y = fmaf(f, v.y, O.y);
      O.z = fmaf(f, v.z, O.z);
      O.w = fmaf(f, v.w, O.w);
    }
  }
  s_o[warp][lane] = O;
  if (lane == 0) s_l[warp] = L;
  __syncthreads();
  if (head >= heads || sub != 0) return;
  for (int i = 1; i < per_head; ++i) {
    const float4 v = s_o[warp + i][lane];
    O.x += v.x; O.y += v.y; O.z += v.z; O.w += v.w;
    L += s_l[warp + i];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2*>(a.out + (static_cast<size_t>(seq) * a.nq + head0 + head) * kFp8D + 4 * lane) =
      make_uint2(pack_bf16x2(O.x * inv, O.y * inv), pack_bf16x2(O.z * inv, O.w * inv));
}

extern "C" int forge_make_tmap_2d(CUtensorMap* tm, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, int elem_bytes);

// Grid and scratch of a launch of up to 512 sequences; G: query heads of an item.
struct F8Grid {
  int slices, G, ctas;
};
static F8Grid f8_grid(int B, int nq, int nkv, int block_size, int table_width) {
  F8Grid z;
  const int group = nq / nkv;
  z.slices = (group + kF8Heads - 1) / kF8Heads;
  z.G = (group + z.slices - 1) / z.slices;
  const long long most = static_cast<long long>(std::min(B, kF8Seqs)) * nkv * z.slices *
                         ((static_cast<long long>(table_width) * block_size + kF8Tile - 1) / kF8Tile);
  z.ctas = static_cast<int>(std::max(1ll, std::min<long long>(most, static_cast<long long>(kF8CtasPerSm) * device_sm_count())));
  return z;
}

extern "C" long long forge_decode_fp8_scratch_floats(int B, int nq, int nkv, int block_size, int table_width) {
  const F8Grid z = f8_grid(B, nq, nkv, block_size, table_width);
  return 2ll * z.ctas * z.G * (kFp8D + 2) + kF8Seqs + 1;
}

// q [B, nq, 128], out [B, nq * 128] bf16; a length of zero or less gives a row of zeros.  scratch: forge_decode_fp8_scratch_floats, 16-byte aligned.
extern "C" int forge_decode_fp8(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                const int* block_tables, const int* lens, void* out, float* scratch, int B, int nq, int nkv, int block_size,
                                int table_width, int num_blocks, float scale, unsigned* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (nkv < 1 || nq % nkv != 0 || block_size < 16 || (block_size & (block_size - 1))) return -1;
  const F8Grid z = f8_grid(B, nq, nkv, block_size, table_width);
  const long long tiles = (static_cast<long long>(table_width) * block_size + kF8Tile - 1) / kF8Tile;
  if (std::min(B, kF8Seqs) * tiles * nkv * z.slices > INT32_MAX) return -1;
  CUtensorMap tm_k, tm_v;
  const uint64_t rows = static_cast<uint64_t>(num_blocks) * nkv * block_size;
  const uint32_t box = static_cast<uint32_t>(std::min(block_size, kF8Tile));
  if (forge_make_tmap_2d(&tm_k, k_codes, rows, kFp8D, kFp8D, box, 1) != 0 || forge_make_tmap_2d(&tm_v, v_codes, rows, kFp8D, kFp8D, box, 1) != 0) return -2;
  FORGE_ENSURE_DYN_SMEM(decode_fp8_kernel, f8_smem(kF8Heads));
  static_assert(kF8CtasPerSm * (f8_smem(kF8Heads) + 1024) <= 228 * 1024, "CTAs per SM");
  for (int b0 = 0; b0 < B; b0 += kF8Seqs) {
    Fp8Decode a;
    a.q = static_cast<const __nv_bfloat16*>(q) + static_cast<size_t>(b0) * nq * kFp8D;
    a.k_scales = static_cast<const uint8_t*>(k_scales); a.v_scales = static_cast<const uint8_t*>(v_scales);
    a.block_tables = block_tables + static_cast<size_t>(b0) * table_width; a.lens = lens + b0;
    a.out = static_cast<__nv_bfloat16*>(out) + static_cast<size_t>(b0) * nq * kFp8D;
    a.part_o = scratch;
    a.part_ml = scratch + static_cast<size_t>(2) * z.ctas * z.G * kFp8D;
    a.tiles_before = reinterpret_cast<int*>(a.part_ml + static_cast<size_t>(2) * z.ctas * z.G * 2);
    a.B = std::min(B - b0, kF8Seqs); a.nq = nq; a.nkv = nkv; a.group = nq / nkv; a.G = z.G; a.slices = z.slices;
    a.block_size = block_size; a.table_width = table_width; a.num_blocks = num_blocks;
    a.scale_log2 = scale * 1.4426950408889634f; a.status = status;
    if (launch_kernel(decode_fp8_kernel, dim3(z.ctas), dim3(kF8Threads), f8_smem(z.G), stream, 0, tm_k, tm_v, a) != cudaSuccess) return -5;
    if (launch_kernel(decode_fp8_join_kernel, dim3(z.ctas), dim3(32 * kF8JoinWarps), 0, stream, 0, a) != cudaSuccess) return -5;
  }
  return 0;
}

}  // namespace forge
