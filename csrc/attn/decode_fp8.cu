// Attention of one new token per sequence over a paged 8-bit cache (include/fp8_cache.cuh).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c q.k_j - m),   c = scale log2(e),   m = max_j c q.k_j
//
// An item is a sequence and a KV head with up to eight of its query heads (larger groups take several items).
//
// A tile: 32 tokens for every consumer warp.  One warp loads (2-D TMA boxes of 128-byte rows with the 128-byte swizzle; scale bytes by bulk
// copies; a ring of stages that never drains across items); the others each have a maximum, a sum and results of their own
// until the item's end:
//   S^T [16 tokens x 8 heads] = K Q^T,   O^T [128 dims x 8 heads] += V^T P^T,   mma.sync m16n8k16, fp16 operands, fp32 sums.
// Codes of e4m3 are exact in fp16.  Which entries of K stand at which place of the inner dimension is free as long as Q's stand there too, and so is the
// order of the rows of O^T: a lane takes 32 consecutive entries of a key and 16 of a value with 16-byte reads that touch every
// bank once, and converts them in place; V^T needs no transposing load, two tokens' bytes are interleaved instead.
//   Queries are brought to [2^14, 2^15) by a power of two per head, which keeps every bit of their bf16 down to 2^-31 of the largest entry.
//   A value's scale 2^e goes into its weight's exponent: w_j = 2^(c q.k_j + e_j - u + 7), u a maximum of its own: a value that counts is never lost
//   beside one with a larger scale that does not.  A weight is two halves, its first 11 bits and what is left of it: within 2^-22 of itself, or 2^-31 of
//   the largest (fp16 has no smaller numbers).  With the first half alone results were off by 2^-12 of the mean |value|, where those over a
//   bf16 cache are not.  Of up to four heads columns 4 .. 7 are the same heads once more, with the second halves, and the columns are added up
//   at the item's end; of more heads both halves are multiplied.  The first half alone / columns / both, 32 / 8 heads: 16 x 768 tokens 11.8 / 12.1 /
//   12.6 us, 32 x 768 15.3 / 15.8 / 16.6, 256 x 100 .. 1500 77.1 / 77.2 / 79.2.  The sum of the p_j is kept in fp32.  m and u move only when they are
//   exceeded by 8, so w_j <= 2^15 and products are rescaled rarely.
// What is behind a sequence's last token never counts: its scores, weights and value bytes are replaced, whatever they are.
//
// The split, many items.  The tiles of 64 tokens of all items, in order, are dealt out to four teams per SM, of two consumer warps and a loading one with a
// ring each: an item counts as its tiles and kF8ItemCost more for its beginning and end, and team i of C takes the i-th of C equal shares,
// so short and long contexts, few and many sequences fill the GPU alike.  An item inside one team is finished there; the parts of one that
// is cut are joined by a second kernel, in order, so that the same step gives the same bits; how an item is cut depends on the others, and
// with it the last bits of its sums.  Lengths are read on the device, so the launch fits a CUDA graph whatever they become.
// The four teams of an SM are one CTA: as CTAs of their own, launched beside the end of another kernel (PDL), some SMs took only
// three, and the others ran after all the rest (256 sequences of 100 .. 1500 tokens: 82 us after an idle GPU, 116 in a row).
// The split, few items of moderate length.  A cluster of one to eight CTAs takes an item, each a run of its tiles of 128 tokens, and they join what they
// have through distributed shared memory: one launch, and none of the chain from kernel to kernel.
// From the raw projection (kRaw): the step's norm, rotation and cache write happen here too, one launch less; every CTA of a cluster makes the item's queries
// for itself, and the warp that owns the newest token puts it into its tile and into the cache.
// Bound by memory: 258 bytes per key and KV head; few items by latency (length -> block table -> keys -> scores -> results).
#include <algorithm>

#include "../include/fp8_cache.cuh"
#include "../include/launch.cuh"
#include "../include/mma_sync.cuh"
#include "../include/ptx.cuh"

namespace forge {

constexpr int kF8Seqs = 512;                           // sequences of a launch
constexpr int kF8Heads = 8;                            // query heads of an item
constexpr float kF8Rise = 8.f;                         // how far a score may exceed the maximum in use
constexpr float kF8Top = 7.f;                          // weights are at most 2^(7 + 8)
constexpr float kF8Least = -3.402823466e38f;           // maximum before any score.  Finite, so that a score of -infinity (masked, or beyond 32 bits) has no weight beside it

struct Fp8Decode {
  const __nv_bfloat16* q;                              // null: from the raw projection
  uint8_t *k_codes, *v_codes, *k_scales, *v_scales;
  const int *block_tables, *lens;
  __nv_bfloat16* out;
  float *part_o, *part_ml;                             // [2 teams][G][128], [2 teams][G][2]: of a team the part that continues an item, then the one that is cut
  int4* cuts;                                          // [teams]: what the joining kernel has to do at the cut before a team
  int B, nq, nkv, group, G, slices, block_size, table_width, num_blocks;
  int stages;                                          // clusters: of the ring; one where no CTA has more than a tile
  float scale_log2;
  unsigned* status;
  // the step's raw projection [B][(nq + 2 nkv) * 128]: queries are normed and rotated here, and the newest token (position length - 1) stored
  const __nv_bfloat16 *qkv, *qw, *kw;                  // norm weights may be null
  long long ld_qkv;
  const float* rope;                                   // [rope_rows][128] cos, sin; null: no rotation
  int rope_rows;
  float eps;
};

// ---- from the raw projection: what fp8_store_kernel does, with the same roundings.  Eight lanes to a head.
__device__ __forceinline__ const float* f8_angles(const Fp8Decode& a, int len, int lane) {
  return a.rope == nullptr ? nullptr : a.rope + static_cast<size_t>(min(max(len - 1, 0), a.rope_rows - 1)) * kFp8D + 8 * (lane & 7);
}
// Query heads 4 set .. of an item, bf16 [heads][128] into shared memory.
__device__ __forceinline__ void f8_make_queries(const Fp8Decode& a, int seq, int head0, int heads, int len, int set, __nv_bfloat16* to, int lane) {
  const int j = lane & 7, h = 4 * set + (lane >> 3);
  if (h < heads) {
    const __nv_bfloat16* src = a.qkv + seq * a.ld_qkv + static_cast<size_t>(head0 + h) * kFp8D + 8 * j;
    const uint4 lo = load8<true>(src), hi = load8<true>(src + 64);
    Fp8Weights w;
    w.load<true>(a.qw, j);
    float x[8], y[8];
    unpack8(lo, x);
    unpack8(hi, y);
    fp8_norm_rotate(x, y, w, a.qw != nullptr, a.eps, f8_angles(a, len, lane), 0xFFu << (lane & 24));
    *reinterpret_cast<uint4*>(to + h * kFp8D + 8 * j) = pack8(x);
    *reinterpret_cast<uint4*>(to + h * kFp8D + 64 + 8 * j) = pack8(y);
  }
  __syncwarp();
}
// The newest token of a KV head: codes of its key and its value, 128 bytes each, then their scale bytes.  Lanes 0 .. 7 make the key's, 8 .. 15 the value's.
constexpr int kF8Newest = 2 * kFp8D + 16;
__device__ __forceinline__ void f8_make_newest(const Fp8Decode& a, int seq, int kvh, int len, uint8_t* to, int lane) {
  const int j = lane & 7, is_v = lane >> 3;
  if (is_v < 2) {
    const __nv_bfloat16* src = a.qkv + seq * a.ld_qkv + static_cast<size_t>(a.nq + is_v * a.nkv + kvh) * kFp8D + 8 * j;
    float x[8], y[8];
    unpack8(load8<true>(src), x);
    unpack8(load8<true>(src + 64), y);
    const unsigned octet = 0xFFu << (lane & 24);
    if (!is_v) {
      Fp8Weights w;
      w.load<true>(a.kw, j);
      fp8_norm_rotate(x, y, w, a.kw != nullptr, a.eps, f8_angles(a, len, lane), octet);
    }
    uint2 code[2];
    const uint32_t scale = fp8_quantise(x, y, octet, code);
    *reinterpret_cast<uint2*>(to + is_v * kFp8D + 8 * j) = code[0];
    *reinterpret_cast<uint2*>(to + is_v * kFp8D + 64 + 8 * j) = code[1];
    if (j == 0) to[2 * kFp8D + is_v] = static_cast<uint8_t>(scale);
  }
  __syncwarp();
}
// By the same warp, into its row r of the tile that has just landed, whose place in the cache did not hold the token yet, and into the cache.  No other
// warp reads that row.
__device__ __forceinline__ void f8_put_newest(const Fp8Decode& a, int seq, int kvh, int len, const uint8_t* from, uint8_t* K, uint8_t* V, uint8_t* k_scales,
                                              uint8_t* v_scales, int lane) {
  const int i = lane & 7, is_v = lane >> 3, at = len - 1, r = at & 31;
  if (is_v < 2) {
    const uint4 piece = *reinterpret_cast<const uint4*>(from + is_v * kFp8D + 16 * i);
    const uint8_t scale = from[2 * kFp8D + is_v];
    *reinterpret_cast<uint4*>((is_v ? V : K) + r * kFp8D + ((i ^ (r & 7)) << 4)) = piece;
    if (i == 0) (is_v ? v_scales : k_scales)[r] = scale;
    const int blk = a.block_tables[static_cast<size_t>(seq) * a.table_width + at / a.block_size];
    if (blk >= 0 && blk < a.num_blocks && a.lens[seq] == len) {          // (reported where the tile is loaded, and the length where it was clamped)
      const size_t to = (static_cast<size_t>(blk) * a.nkv + kvh) * a.block_size + at % a.block_size;
      *reinterpret_cast<uint4*>((is_v ? a.v_codes : a.k_codes) + to * kFp8D + 16 * i) = piece;
      if (i == 0) (is_v ? a.v_scales : a.k_scales)[to] = scale;
    }
  }
  fence_proxy_async_smem();                            // a later copy into this stage comes after these writes
  __syncwarp();
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

// The ring of tiles of kWarps consumer warps.
template <int kWarps, int kStages>
struct F8Ring {
  static constexpr int kTile = 32 * kWarps, kHalf = kTile * kFp8D, kBytes = kStages * (2 * kHalf + 2 * kTile);
  uint8_t *codes, *scales;                             // [stage][K, V][tokens][128], [stage][K, V][tokens]
  uint64_t *full, *empty;
  int s = 0, phase = 0, issued = 0;                    // issued: tiles that may be on their way, at most kStages
  __device__ __forceinline__ void next() {
    if (++s == kStages) {
      s = 0;
      phase ^= 1;
    }
  }
  __device__ __forceinline__ void init() {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
  }
  // A warp: tiles [j, j + count) of a sequence with `len` tokens.  `held`: the lane's of 32 table entries from page `from` on.  False: a wait has
  // run out.
  __device__ __forceinline__ bool load(const Fp8Decode& a, const CUtensorMap* tm_k, const CUtensorMap* tm_v, int seq, int kvh, int len, int j, int count,
                                       int from, int held, int lane) {
    const int rows = min(a.block_size, kTile);
    for (const int end = j + count; j < end; ++j) {
      const int tok0 = j * kTile, pages = (min(len - tok0, kTile) + rows - 1) / rows;
      bool ok = true;
      if (lane == 0) {
        ok = mbar_wait_parked(&empty[s], phase ^ 1, a.status);
        if (ok) mbar_expect_tx(&full[s], pages * rows * 2 * (kFp8D + 1));
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
      for (int p = 0; p < pages; ++p) {
        const int tok = tok0 + p * rows, page = tok / a.block_size;
        if (page >= from + 32) {
          from = page;
          held = entry(a, seq, page + lane);
        }
        int blk = __shfl_sync(0xffffffffu, held, page - from);
        if (lane != 0) continue;
        if (blk < 0 || blk >= a.num_blocks) {
          set_status(a.status, kStatusBadIndex);
          blk = 0;
        }
        const int row = (blk * a.nkv + kvh) * a.block_size + tok % a.block_size;
        uint8_t* to = codes + s * 2 * kHalf + p * rows * kFp8D;
        tma_load_2d(to, tm_k, &full[s], 0, row);
        tma_load_2d(to + kHalf, tm_v, &full[s], 0, row);
        uint8_t* sc = scales + s * 2 * kTile + p * rows;
        bulk_load(sc, a.k_scales + row, rows, &full[s]);
        bulk_load(sc + kTile, a.v_scales + row, rows, &full[s]);
      }
      __syncwarp();
      issued = min(issued + 1, kStages);
      next();
    }
    return true;
  }
  // By the loading warp, at its end: waits for the last copies, so that none is on its way to the shared memory of a CTA that has left because a wait
  // had run out.  (Otherwise the consumers wait for them.)
  __device__ __forceinline__ void settle(unsigned* status, int lane) {
    if (lane == 0) {
      bool ok = true;
      for (int i = 1; i <= issued && ok; ++i) {
        const int at = s - i;
        ok = mbar_wait_parked(&full[at < 0 ? at + kStages : at], at < 0 ? phase ^ 1 : phase, status);
      }
    }
    __syncwarp();
  }
  static __device__ __forceinline__ int entry(const Fp8Decode& a, int seq, int page) {
    return page < a.table_width ? a.block_tables[static_cast<size_t>(seq) * a.table_width + page] : -1;
  }
};

// A consumer warp's share of an item.  Lane l = 4 g + quad holds scores of tokens g + 8 i and heads 2 quad, 2 quad + 1, and of the results dims
// 16 g .. 16 g + 15 of these heads.
// kWide: of more than four heads.  Otherwise heads 4 .. 7 are heads 0 .. 3 again, and their results are what the second halves of the weights add.
template <bool kWide>
struct F8State {
  uint32_t qh[16];                                     // 32 consecutive entries of head g, from 32 quad on
  float qf[2];                                         // of heads 2 quad, 2 quad + 1: from products to scores in base 2
  float m[2], u[2], l[2];
  float o[8][4];                                       // [i][0], [i][1]: dim 16 g + 2 i of heads 2 quad, 2 quad + 1; [2], [3]: the dim after it

  __device__ __forceinline__ void begin(const __nv_bfloat16* q_rows, int heads, float scale_log2, int lane) {
    const int g = kWide ? lane >> 2 : (lane >> 2) & 3, quad = lane & 3;
    uint32_t w[16], top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 r = g < heads ? *reinterpret_cast<const uint4*>(q_rows + g * kFp8D + 32 * quad + 8 * i) : make_uint4(0, 0, 0, 0);
      w[4 * i] = r.x; w[4 * i + 1] = r.y; w[4 * i + 2] = r.z; w[4 * i + 3] = r.w;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, max(abs_bits(bf16_lo(w[i])), abs_bits(bf16_hi(w[i]))));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float up = __uint_as_float(min(268u - (top >> 23), 254u) << 23);         // 2^14 / 2^exponent, at most 2^127
#pragma unroll
    for (int i = 0; i < 16; ++i) qh[i] = f8_half2(bf16_lo(w[i]) * up, bf16_hi(w[i]) * up);
    qf[0] = scale_log2 / __shfl_sync(0xffffffffu, up, 8 * quad);
    qf[1] = scale_log2 / __shfl_sync(0xffffffffu, up, 8 * quad + 4);
    m[0] = m[1] = u[0] = u[1] = kF8Least;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  }

  // 32 tokens; of them `valid` (1 or more; kWhole: all) count.  K, V: their rows, of a 1024-byte aligned tile with the 128-byte swizzle.
  __device__ __forceinline__ void take(const uint8_t* K, const uint8_t* V, const uint8_t* k_scales, const uint8_t* v_scales, int valid, int lane) {
    if (valid >= 32) take_tokens<true>(K, V, k_scales, v_scales, 32, lane);
    else take_tokens<false>(K, V, k_scales, v_scales, valid, lane);
  }
  template <bool kWhole>
  __device__ __forceinline__ void take_tokens(const uint8_t* K, const uint8_t* V, const uint8_t* k_scales, const uint8_t* v_scales, int valid, int lane) {
    const int g = lane >> 2, quad = lane & 3;
    // ---- products
    float c[2][2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c[t][0][e] = c[t][1][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* at = K + (16 * t + g) * kFp8D + (((2 * quad + h) ^ g) << 4);
        const uint4 ka = *reinterpret_cast<const uint4*>(at), kb = *reinterpret_cast<const uint4*>(at + 8 * kFp8D);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t f[4];
          fp8x4_to_half2(wa[e], f[0], f[2]);
          fp8x4_to_half2(wb[e], f[1], f[3]);
          mma16816_f16(c[t][e & 1], f, qh[8 * h + 2 * e], qh[8 * h + 2 * e + 1]);
        }
      }
    }
    // ---- scores x and exponents y of the weights, of tokens 8 i + g
    const float ks = fp8_scale(k_scales[lane]);
    const uint32_t vb = v_scales[lane];
    const float vs = vb == kScaleNan ? __uint_as_float(0x7FC00000u) : static_cast<float>(static_cast<int>(vb) - 127);
    float x[4][2], y[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float k = __shfl_sync(0xffffffffu, ks, 8 * i + g), e = __shfl_sync(0xffffffffu, vs, 8 * i + g);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        x[i][h] = (c[i >> 1][0][2 * (i & 1) + h] + c[i >> 1][1][2 * (i & 1) + h]) * qf[h] * k;
        y[i][h] = x[i][h] + e;
      }
    }
    if constexpr (!kWhole) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (8 * i + g >= valid) x[i][0] = x[i][1] = y[i][0] = y[i][1] = -INFINITY;
    }
    // ---- maxima
    float xm[2], ym[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      xm[h] = fmaxf(fmaxf(x[0][h], x[1][h]), fmaxf(x[2][h], x[3][h]));
      ym[h] = fmaxf(fmaxf(y[0][h], y[1][h]), fmaxf(y[2][h], y[3][h]));
    }
    if (__any_sync(0xffffffffu, xm[0] > m[0] + kF8Rise || xm[1] > m[1] + kF8Rise || ym[0] > u[0] + kF8Rise || ym[1] > u[1] + kF8Rise)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {                      // each head decides by itself, so its bits do not depend on the others
        xm[h] = f8_max_over_tokens(xm[h]);
        ym[h] = f8_max_over_tokens(ym[h]);
        if (xm[h] > m[h] + kF8Rise) {
          l[h] *= ex2_approx(m[h] - xm[h]);              // 0 at first
          m[h] = xm[h];
        }
        if (ym[h] > u[h] + kF8Rise) {
          const float down = ex2_approx(u[h] - ym[h]);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[d][h] *= down;
            o[d][2 + h] *= down;
          }
          u[h] = ym[h];
        }
      }
    }
    // ---- weights.  A score that is NaN or +infinity makes the result NaN; where all are -infinity the sums stay zero, and so does the result.
    const float u0 = u[0] - kF8Top, u1 = u[1] - kF8Top;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t p[2], rest[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = 2 * t + k;
        l[0] += ex2_approx(x[i][0] - m[0]);              // -inf -> 0
        l[1] += ex2_approx(x[i][1] - m[1]);
        const float w0 = ex2_approx(y[i][0] - u0), w1 = ex2_approx(y[i][1] - u1);
        const float h0 = __uint_as_float(__float_as_uint(w0) & 0xFFFFE000u), h1 = __uint_as_float(__float_as_uint(w1) & 0xFFFFE000u);     // 11 bits
        const uint32_t whole = f8_half2(h0, h1), left = f8_half2(w0 - h0, w1 - h1);
        p[k] = transpose8x8(kWide || quad < 2 ? whole : left);
        if constexpr (kWide) rest[k] = transpose8x8(left);
      }
      // ---- values: of 16 tokens 2 quad, 2 quad + 1 and eight further on, dims 16 g ..
      uint32_t w[4][4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int tok = 16 * t + 2 * quad + (h & 1) + 8 * (h >> 1);
        uint4 v = *reinterpret_cast<const uint4*>(V + tok * kFp8D + ((g ^ (tok & 7)) << 4));
        if (!kWhole && tok >= valid) v = make_uint4(0, 0, 0, 0);
        w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t f[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          fp8x4_to_half2(__byte_perm(w[0][e], w[1][e], h ? 0x7362 : 0x5140), f[h][0], f[h][1]);
          fp8x4_to_half2(__byte_perm(w[2][e], w[3][e], h ? 0x7362 : 0x5140), f[h][2], f[h][3]);
          mma16816_f16(o[2 * e + h], f[h], p[0], p[1]);
        }
        if constexpr (kWide) {
#pragma unroll
          for (int h = 0; h < 2; ++h) mma16816_f16(o[2 * e + h], f[h], rest[0], rest[1]);
        }
      }
    }
  }

  // To and from a joining area: the same lane of another warp has the same heads and dims.  Afterwards l is the sum over the
  // tokens and not the lane's.
  static constexpr int kOFloats = 32 * 32, kJoinFloats = kOFloats + 6 * 4;
  __device__ __forceinline__ void sum_up() {
    l[0] = f8_sum_over_tokens(l[0]);
    l[1] = f8_sum_over_tokens(l[1]);
  }
  __device__ __forceinline__ void publish(float* area, float* maxima, int lane) const {
#pragma unroll
    for (int i = 0; i < 32; ++i) area[i * 32 + lane] = o[i >> 2][i & 3];
    if (lane < 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        maxima[4 * h + lane] = m[h];
        maxima[4 * (2 + h) + lane] = u[h];
        maxima[4 * (4 + h) + lane] = l[h];
      }
    }
  }
  __device__ __forceinline__ void join(const float* area, const float* maxima, int lane) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {                        // (without a score: zeros)
      const float* other = maxima + (lane & 3);
      const float m2 = other[4 * h], u2 = other[4 * (2 + h)], M = fmaxf(m[h], m2), U = fmaxf(u[h], u2);
      l[h] = l[h] * (m[h] == kF8Least ? 0.f : ex2_approx(m[h] - M)) + other[4 * (4 + h)] * (m2 == kF8Least ? 0.f : ex2_approx(m2 - M));
      const float f = u[h] == kF8Least ? 0.f : ex2_approx(u[h] - U), f2 = u2 == kF8Least ? 0.f : ex2_approx(u2 - U);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float& v = o[k >> 1][2 * (k & 1) + h];
        v = v * f + area[(2 * k + h) * 32 + lane] * f2;
      }
      m[h] = M;
      u[h] = U;
    }
  }
  // o <- results.
  __device__ __forceinline__ void finish() {
    if constexpr (!kWide) {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i >> 2][i & 3] += __shfl_xor_sync(0xffffffffu, o[i >> 2][i & 3], 2);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float f = l[h] == 0.f ? 0.f : 1.f / l[h] * exp2f(u[h] - m[h] - kF8Top);        // (no score: zeros)
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k >> 1][2 * (k & 1) + h] *= f;
    }
  }
  __device__ __forceinline__ void store(__nv_bfloat16* rows, int heads, int lane) const {
    const int g = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (2 * quad + h >= heads) continue;
      uint4* dst = reinterpret_cast<uint4*>(rows + (2 * quad + h) * kFp8D + 16 * g);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        dst[i] = make_uint4(pack_bf16x2(o[4 * i][h], o[4 * i][2 + h]), pack_bf16x2(o[4 * i + 1][h], o[4 * i + 1][2 + h]),
                            pack_bf16x2(o[4 * i + 2][h], o[4 * i + 2][2 + h]), pack_bf16x2(o[4 * i + 3][h], o[4 * i + 3][2 + h]));
    }
  }
  // Results in fp32 [heads][128] with maximum and sum [heads][2].
  __device__ __forceinline__ void store_part(float* rows, float* ml, int heads, int lane) const {
    const int g = lane >> 2, quad = lane & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (2 * quad + h >= heads) continue;
      float4* dst = reinterpret_cast<float4*>(rows + (2 * quad + h) * kFp8D + 16 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = make_float4(o[2 * i][h], o[2 * i][2 + h], o[2 * i + 1][h], o[2 * i + 1][2 + h]);
      if (g == 0) {
        ml[2 * (2 * quad + h)] = m[h];
        ml[2 * (2 * quad + h) + 1] = l[h];
      }
    }
  }
};

// ---------------------------------------------------------------------------------------------------------
// Equal shares
// ---------------------------------------------------------------------------------------------------------
constexpr int kF8Warps = 2, kF8Stages = 3, kF8Teams = 4;
constexpr int kF8TeamWarps = kF8Warps + 1, kF8Threads = 32 * kF8Teams * kF8TeamWarps;
constexpr int kF8ItemCost = 2;                         // tiles (1, 3: 256 x 100 .. 1500 81.8, 76.3 us for 75.7)
constexpr int kF8Share = 4;                            // units to a team at least, or there are fewer teams at work (2, 8: 13 x 200 .. 2000 13.7, 16.7 us for 13.4)
using F8FlatRing = F8Ring<kF8Warps, kF8Stages>;

constexpr int kF8JoinArea = (kF8Warps - 1) * F8State<true>::kJoinFloats;
constexpr int kF8FlatSmem = 1024 + kF8Teams * (F8FlatRing::kBytes + kF8JoinArea * 4 + 2 * kF8Stages * 8) + (kF8Seqs + 1 + kF8Threads / 32) * 4;
static_assert(kF8FlatSmem <= 227 * 1024, "shared memory");

// A place in the list of units: an item is kF8ItemCost units and one for every tile; tile j stands at unit kF8ItemCost + j of its item.
struct F8Place {
  int seq, item, n, j, base;                           // tiles of an item of the sequence; first tile from here on; unit the item begins at
};
__device__ __forceinline__ F8Place f8_place(const int* before, int B, int items, int unit) {
  int lo = 0, hi = B;                                  // before[lo] * items <= unit < before[hi] * items
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (before[mid] * items <= unit) lo = mid;
    else hi = mid;
  }
  F8Place p;
  p.seq = lo;
  const int size = before[lo + 1] - before[lo], at = unit - before[lo] * items;
  p.n = size - kF8ItemCost;
  p.item = at / size;
  p.base = before[lo] * items + p.item * size;
  p.j = max(0, unit - p.base - kF8ItemCost);
  return p;
}

template <bool kWide>
__global__ void __launch_bounds__(kF8Threads, 1)
decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Fp8Decode a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int lane = threadIdx.x & 31, cap = a.table_width * a.block_size;
  const int team = threadIdx.x / (32 * kF8TeamWarps), warp = threadIdx.x / 32 % kF8TeamWarps;            // warps 0 .. kF8Warps - 1: consumers
  uint8_t* scales = smem + kF8Teams * kF8Stages * 2 * F8FlatRing::kHalf;
  float* join = reinterpret_cast<float*>(scales + kF8Teams * kF8Stages * 2 * F8FlatRing::kTile);
  uint64_t* bars = reinterpret_cast<uint64_t*>(join + kF8Teams * kF8JoinArea);
  int* s_before = reinterpret_cast<int*>(bars + kF8Teams * 2 * kF8Stages);         // [B + 1] units of the sequences before, per item
  int* s_warp = s_before + kF8Seqs + 1;
  F8FlatRing ring;
  ring.codes = smem + team * kF8Stages * 2 * F8FlatRing::kHalf;
  ring.scales = scales + team * kF8Stages * 2 * F8FlatRing::kTile;
  ring.full = bars + team * 2 * kF8Stages;
  ring.empty = ring.full + kF8Stages;
  float* s_join = join + team * kF8JoinArea;

  pdl_launch_dependents();
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    ring.init();
    fence_mbar_init();
  }
  pdl_wait();                                          // q, the cache and the step buffer come from predecessors

  {
    constexpr int kPer = (kF8Seqs + kF8Threads - 1) / kF8Threads;
    int n[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = threadIdx.x * kPer + e;
      int len = b < a.B ? a.lens[b] : 0;
      if (len > cap) {                                 // a corrupted length: clamped and reported
        set_status(a.status, kStatusBadIndex);
        len = cap;
      }
      n[e] = len > 0 ? (len + F8FlatRing::kTile - 1) / F8FlatRing::kTile + kF8ItemCost : 0;
      sum += n[e];
    }
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    if (lane == 31) s_warp[threadIdx.x / 32] = before;
    before -= sum;
    __syncthreads();
    for (int w = 0; w < threadIdx.x / 32; ++w) before += s_warp[w];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int b = threadIdx.x * kPer + e;
      if (b <= a.B) s_before[b] = before;
      before += n[e];
    }
    __syncthreads();
  }
  const int items = a.nkv * a.slices, units = s_before[a.B] * items;
  const int me = team * gridDim.x + blockIdx.x, workers = min(static_cast<int>(kF8Teams * gridDim.x), (units + kF8Share - 1) / kF8Share);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)    // rows without tokens: zeros
    if (s_before[b + 1] == s_before[b])
      for (int i = threadIdx.x; i < a.nq * kFp8D / 8; i += kF8Threads)
        reinterpret_cast<uint4*>(a.out + static_cast<size_t>(b) * a.nq * kFp8D)[i] = make_uint4(0, 0, 0, 0);
  if (me >= workers) {
    if (warp == 0 && lane == 0) a.cuts[me] = make_int4(0, 0, 0, 0);
    return;
  }
  const auto share = [&](int i) { return static_cast<int>(static_cast<long long>(units) * i / workers); };
  const int u_begin = share(me), u_end = share(me + 1);
  const F8Place start = f8_place(s_before, a.B, items, u_begin);
  if (warp == 0 && lane == 0) {
    // a cut inside an item, the item's first: its parts are the second slot of the team before and the first slots of this one and those after it
    const auto owner = [&](int unit) { return static_cast<int>((static_cast<long long>(unit + 1) * workers - 1) / units); };
    int parts = 0;
    if (start.j > 0 && owner(start.base + kF8ItemCost) == me - 1) parts = owner(start.base + kF8ItemCost + start.n - 1) - me + 2;
    a.cuts[me] = make_int4(parts, start.seq, start.item, 0);
  }

  // the items of this share, in order; every role walks the same list
  int seq = start.seq, item = start.item, n = start.n, j = start.j, base = start.base;
  bool ok = true;                                      // once a wait has run out none is made any more and no stage given back, but every barrier still is
  using State = F8State<kWide>;
  State st;
  while (base + kF8ItemCost + j < u_end) {
    const int count = min(n - j, u_end - (base + kF8ItemCost + j)), len = min(a.lens[seq], cap);
    const int kvh = item / a.slices, slice = item - kvh * a.slices, head0 = kvh * a.group + slice * a.G, heads = min(a.G, a.group - slice * a.G);
    if (warp == kF8Warps) {
      const int from = j * F8FlatRing::kTile / a.block_size;
      if (ok) ok = ring.load(a, &tm_k, &tm_v, seq, kvh, len, j, count, from, ring.entry(a, seq, from + lane), lane);
    } else {
      st.begin(a.q + (static_cast<size_t>(seq) * a.nq + head0) * kFp8D, heads, a.scale_log2, lane);
      for (int i = 0; i < count; ++i, ring.next()) {
        const int valid = len - (j + i) * F8FlatRing::kTile - 32 * warp;
        ok = ok && mbar_wait_parked(&ring.full[ring.s], ring.phase, a.status);
        if (valid > 0) {
          const uint8_t* K = ring.codes + ring.s * 2 * F8FlatRing::kHalf + 32 * warp * kFp8D;
          const uint8_t* sc = ring.scales + ring.s * 2 * F8FlatRing::kTile + 32 * warp;
          st.take(K, K + F8FlatRing::kHalf, sc, sc + F8FlatRing::kTile, valid, lane);
        }
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(&ring.empty[ring.s]);
      }
      st.sum_up();
      if (warp > 0) st.publish(s_join + (warp - 1) * State::kJoinFloats, s_join + (warp - 1) * State::kJoinFloats + State::kOFloats, lane);
      named_barrier_sync(1 + team, 32 * kF8Warps);
      if (warp == 0) {
#pragma unroll
        for (int w = 1; w < kF8Warps; ++w)
          st.join(s_join + (w - 1) * State::kJoinFloats, s_join + (w - 1) * State::kJoinFloats + State::kOFloats, lane);
      }
      named_barrier_sync(1 + team, 32 * kF8Warps);            // the joining area is the next item's
      if (warp == 0) {
        st.finish();
        if (count == n) {
          st.store(a.out + (static_cast<size_t>(seq) * a.nq + head0) * kFp8D, heads, lane);
        } else {
          const size_t p = static_cast<size_t>(2 * me + (j == 0 ? 1 : 0)) * a.G;
          st.store_part(a.part_o + p * kFp8D, a.part_ml + 2 * p, heads, lane);
        }
      }
    }
    base += n + kF8ItemCost;
    j = 0;
    if (++item == items) {
      item = 0;
      do ++seq;
      while (seq < a.B && s_before[seq + 1] == s_before[seq]);
      if (seq >= a.B) break;
      n = s_before[seq + 1] - s_before[seq] - kF8ItemCost;
    }
  }
  if (warp == kF8Warps) ring.settle(a.status, lane);
}

// Joins the parts of an item that was cut.  A CTA for a cut and a head, its warps take the parts in turn.  Four warps with 32 registers find place beside
// a CTA of the kernel before and are there when it ends (64 x 2304 tokens, 64 / 8 heads: 61.7 us with eight warps, 58.8 with four); items that are cut into
// many parts take eight (1 x 16000, 32 / 8 heads: 15.7, 18.0 with four).
constexpr int kF8JoinWarps = 8;

__global__ void __launch_bounds__(32 * kF8JoinWarps, 8) decode_fp8_join_kernel(const Fp8Decode a) {
  __shared__ float4 s_o[kF8JoinWarps][32];
  __shared__ float2 s_ml[kF8JoinWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int me = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int4 cut = a.cuts[me];
  const int parts = cut.x, kvh = cut.z / a.slices, slice = cut.z - kvh * a.slices;
  if (parts == 0 || head >= min(a.G, a.group - slice * a.G)) return;
  const auto slot = [&](int i) { return static_cast<size_t>(i == 0 ? 2 * (me - 1) + 1 : 2 * (me + i - 1)) * a.G + head; };
  float M = kF8Least, L = 0.f;                           // of the warp's parts
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < parts; i += warps) {
    const size_t p = slot(i);
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * p);
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + p * kFp8D + 4 * lane);
    const float m = fmaxf(M, ml.x);
    const float keep = M == kF8Least ? 0.f : ex2_approx(M - m), f = (ml.x == kF8Least ? 0.f : ex2_approx(ml.x - m)) * ml.y;
    M = m;
    L = L * keep + f;
    O.x = O.x * keep + f * v.x;
    O.y = O.y * keep + f * v.y;
    O.z = O.z * keep + f * v.z;
    O.w = O.w * keep + f * v.w;
  }
  s_o[warp][lane] = O;
  if (lane == 0) s_ml[warp] = make_float2(M, L);
  __syncthreads();
  if (warp != 0) return;
  const int n = min(warps, parts);
  for (int i = 0; i < n; ++i) M = fmaxf(M, s_ml[i].x);
  L = 0.f;
  O = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < n; ++i) {
    const float4 v = s_o[i][lane];
    const float f = s_ml[i].x == kF8Least ? 0.f : ex2_approx(s_ml[i].x - M);
    L += f * s_ml[i].y;
    O.x += f * v.x; O.y += f * v.y; O.z += f * v.z; O.w += f * v.w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int h = kvh * a.group + slice * a.G + head;
  *reinterpret_cast<uint2*>(a.out + (static_cast<size_t>(cut.y) * a.nq + h) * kFp8D + 4 * lane) =
      make_uint2(pack_bf16x2(O.x * inv, O.y * inv), pack_bf16x2(O.z * inv, O.w * inv));
}

// ---------------------------------------------------------------------------------------------------------
// Few items: a cluster of CTAs each
// ---------------------------------------------------------------------------------------------------------
constexpr int kF8CWarps = 4, kF8CStages = 2, kF8CThreads = 32 * (kF8CWarps + 1), kF8CCtasPerSm = 2;
using F8ClusterRing = F8Ring<kF8CWarps, kF8CStages>;
// Little of it, since the products before and after keep weights in the same SMs meanwhile: 84 -> 39 KB for one sequence of 1020 tokens took a layer of
// 4096 x 12288 with 32 / 8 heads from 99.7 to 98.9 us.
constexpr int f8_cluster_smem(int G, int stages) {
  return 1024 + stages * (F8ClusterRing::kBytes / kF8CStages) + kF8Newest + G * (kFp8D + 2) * 4 + 2 * kF8CStages * 8;
}

// Grid (CTAs of an item, items): CTA r of C takes tiles [n r / C, n (r + 1) / C) of its item's n, and its share of the results is what all
// of them left in their shared memory, joined.
template <bool kRaw, bool kWide>
__global__ void __launch_bounds__(kF8CThreads, kF8CCtasPerSm)
decode_fp8_cluster_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Fp8Decode a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cap = a.table_width * a.block_size;
  F8ClusterRing ring;
  ring.codes = smem;
  ring.scales = smem + a.stages * 2 * F8ClusterRing::kHalf;
  uint8_t* newest = ring.scales + a.stages * 2 * F8ClusterRing::kTile;
  float* s_o = reinterpret_cast<float*>(newest + kF8Newest);             // [G][128]
  float* s_ml = s_o + a.G * kFp8D;                                       // [G][2]
  ring.full = reinterpret_cast<uint64_t*>(s_ml + 2 * a.G);
  ring.empty = ring.full + kF8CStages;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    ring.init();
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();

  const int items = a.nkv * a.slices, seq = blockIdx.y / items, item = blockIdx.y - seq * items, rank = blockIdx.x, C = gridDim.x;
  const int kvh = item / a.slices, slice = item - kvh * a.slices, head0 = kvh * a.group + slice * a.G, heads = min(a.G, a.group - slice * a.G);
  __nv_bfloat16* out = a.out + (static_cast<size_t>(seq) * a.nq + head0) * kFp8D;
  int len = a.lens[seq];
  const int held = warp == kF8CWarps ? ring.entry(a, seq, lane) : 0;     // asked for with the length
  if (len > cap) {                                       // a corrupted length: clamped and reported
    if (threadIdx.x == 0) set_status(a.status, kStatusBadIndex);
    len = cap;
  }
  len = max(len, 0);
  const int n = (len + F8ClusterRing::kTile - 1) / F8ClusterRing::kTile, j = n * rank / C, count = n * (rank + 1) / C - j;
  if (warp == kF8CWarps) {
    ring.load(a, &tm_k, &tm_v, seq, kvh, len, j, count, 0, held, lane);
    ring.settle(a.status, lane);
  } else {
    F8State<kWide> st;
    if constexpr (kRaw) {
      __nv_bfloat16* s_q = reinterpret_cast<__nv_bfloat16*>(s_o);        // free until results are there, after the next barrier but one
      if (4 * warp < heads) f8_make_queries(a, seq, head0, heads, len, warp, s_q, lane);
      if (count > 0 && j + count == n && (len - 1) % F8ClusterRing::kTile / 32 == warp) f8_make_newest(a, seq, kvh, len, newest, lane);
      named_barrier_sync(1, 32 * kF8CWarps);
      st.begin(s_q, heads, a.scale_log2, lane);
    } else {
      st.begin(a.q + (static_cast<size_t>(seq) * a.nq + head0) * kFp8D, heads, a.scale_log2, lane);
    }
    bool ok = true;
    for (int i = 0; i < count; ++i, ring.next()) {
      const int valid = len - (j + i) * F8ClusterRing::kTile - 32 * warp;
      ok = ok && mbar_wait_parked(&ring.full[ring.s], ring.phase, a.status);
      if (valid > 0) {
        uint8_t* K = ring.codes + ring.s * 2 * F8ClusterRing::kHalf + 32 * warp * kFp8D;
        uint8_t* sc = ring.scales + ring.s * 2 * F8ClusterRing::kTile + 32 * warp;
        if (kRaw && valid <= 32) f8_put_newest(a, seq, kvh, len, newest, K, K + F8ClusterRing::kHalf, sc, sc + F8ClusterRing::kTile, lane);
        st.take(K, K + F8ClusterRing::kHalf, sc, sc + F8ClusterRing::kTile, valid, lane);
      }
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(&ring.empty[ring.s]);
    }
    st.sum_up();
    // what a warp has takes the place of its own rows of the first stage, which no other reads and into which nothing is loaded any more
    const auto joins = [&](int w, int half) { return reinterpret_cast<float*>(ring.codes + half * F8ClusterRing::kHalf + 32 * w * kFp8D); };
    if (warp > 0) st.publish(joins(warp, 0), joins(warp, 1), lane);
    named_barrier_sync(1, 32 * kF8CWarps);
    if (warp == 0) {
#pragma unroll
      for (int w = 1; w < kF8CWarps; ++w) st.join(joins(w, 0), joins(w, 1), lane);
      st.finish();
      if (C == 1) st.store(out, heads, lane);
      else st.store_part(s_o, s_ml, heads, lane);
    }
  }
  if (C == 1) return;
  __syncwarp();
  cluster_sync();
  const int pieces = heads * (kFp8D / 4);                // four dims of a head each
  for (int i = pieces * rank / C + threadIdx.x; i < pieces * (rank + 1) / C; i += kF8CThreads) {
    const int head = i / (kFp8D / 4);
    float M = kF8Least, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    const uint32_t ml_at = smem_u32(s_ml + 2 * head), o_at = smem_u32(s_o + 4 * i);
    for (int c = 0; c < C; ++c) M = fmaxf(M, ld_dsmem_f2(dsmem_addr(ml_at, c)).x);
    for (int c = 0; c < C; ++c) {
      const float2 ml = ld_dsmem_f2(dsmem_addr(ml_at, c));
      const float4 v = ld_dsmem_f4(dsmem_addr(o_at, c));
      const float f = (ml.x == kF8Least ? 0.f : ex2_approx(ml.x - M)) * ml.y;
      L += f;
      O.x = fmaf(f, v.x, O.x);
      O.y = fmaf(f, v.y, O.y);
      O.z = fmaf(f, v.z, O.z);
      O.w = fmaf(f, v.w, O.w);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<uint2*>(out + 4 * i) = make_uint2(pack_bf16x2(O.x * inv, O.y * inv), pack_bf16x2(O.z * inv, O.w * inv));
  }
  __syncwarp();
  cluster_sync();                                        // nobody's shared memory goes before it has been read
}

extern "C" int forge_make_tmap_2d(CUtensorMap* tm, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows, int elem_bytes);

static bool f8_shape(int nq, int nkv, int block_size) { return nkv >= 1 && nq >= nkv && nq % nkv == 0 && block_size >= 16 && (block_size & (block_size - 1)) == 0; }

// Grid of a launch of up to 512 sequences; G: query heads of an item.
struct F8Grid {
  int slices, G, ctas, teams;
};
static F8Grid f8_grid(int B, int nq, int nkv, int block_size, int table_width) {
  F8Grid z;
  const int group = nq / nkv;
  z.slices = (group + kF8Heads - 1) / kF8Heads;
  z.G = (group + z.slices - 1) / z.slices;
  const long long most = static_cast<long long>(std::min(B, kF8Seqs)) * nkv * z.slices *
                         ((static_cast<long long>(table_width) * block_size + F8FlatRing::kTile - 1) / F8FlatRing::kTile + kF8ItemCost);
  z.ctas = static_cast<int>(std::max(1ll, std::min<long long>(most, device_sm_count())));
  z.teams = z.ctas * kF8Teams;
  return z;
}

// CTAs of an item's cluster, 0: equal shares over the GPU.  mode 1: equal shares, 2: clusters, 0: by size, the longest context being taken to be as
// long as the block table is wide.  That is so where the caller cuts the table to the step; the engine's captured steps have tables of max_model_len
// tokens, whatever the contexts, so with 8 KV heads they take clusters up to 8 sequences at 4096, up to 4 at 8192 and none beyond (16 x 768 tokens, 32 / 8
// heads, in a table of 768 / 4096: 9.3 / 12.1 us; 1 x 1000 in one of 8192 / 32768: 6.0 / 10.1).
// Measured with tables as wide as the longest context and weights of 11 bits (with 22 both are 1 to 3 % slower), equal shares / clusters, us, 32 / 8 heads.
// Clusters of 8: 1 x 700 tokens 9.4 / 6.2, 1 x 6000 12.1 / 10.9, 1 x 9000 12.7 / 13.7, 1 x 16000 14.5 / 21.7, 4 x 6000 15.6 / 13.2, 4 x 9000 17.6 / 17.5.  Of 4: 8 x 200 .. 2000 11.7 / 9.7, 8 x 3000 14.8 / 12.7, 8 x 5000
// 18.2 / 19.0.  Of 2, for which lengths that differ count more: 16 x 768 11.9 / 9.1, 16 x 1500 14.4 / 12.7, 16 x 200 .. 1500 12.2 / 12.0, 13 x 200 .. 2000
// 12.2 / 14.2.  One CTA: 32 x 768 15.4 / 11.5, 32 x 100 .. 768 12.0 / 10.7, 32 x 100 .. 1024 13.4 / 13.2, 32 x 1500 21.9 / 22.4.  More than 256 CTAs: 100 x
// 100 .. 300 16.8 / 18.0.  8 / 1 heads: 32 x 200 .. 2000 (clusters of 8) 13.8 / 7.5, 64 x 100 .. 500 12.2 / 6.3.  Clusters of 8 find no place beside
// each other long before every SM has as many CTAs as fit it: hence two per SM (where one fitted, with a third stage, 32 clusters took 16.1 for
// 7.8) and the bound of 256.  Clusters of 16 were no faster where eight fit (1 x 3001: 7.9), and 11.5 for 6.7 where they did not.
static int f8_cluster(long long items, int table_width, int block_size, int mode) {
  constexpr int kCtas = 256;
  if (mode == 1 || items > 65535) return 0;
  const long long tiles = (static_cast<long long>(table_width) * block_size + F8ClusterRing::kTile - 1) / F8ClusterRing::kTile;
  int c = 8;
  while (c > 1 && (items * c > kCtas || c > tiles)) c /= 2;
  return mode == 2 || (items * c <= kCtas && tiles <= (c >= 4 ? 8 * c : 6 * c + 2)) ? c : 0;
}

// Whether a step should come from the raw projection: one launch less, against every CTA of a cluster making the item's queries.  -1: no such shape.
extern "C" int forge_decode_fp8_qkv_pays(int B, int nq, int nkv, int block_size, int table_width) {
  if (!f8_shape(nq, nkv, block_size)) return -1;
  return B > 0 && f8_cluster(static_cast<long long>(B) * nkv * f8_grid(B, nq, nkv, block_size, table_width).slices, table_width, block_size, 0) > 0;
}

// 0: none needed.
extern "C" long long forge_decode_fp8_scratch_floats(int B, int nq, int nkv, int block_size, int table_width, int mode) {
  if (!f8_shape(nq, nkv, block_size)) return 0;
  const F8Grid z = f8_grid(B, nq, nkv, block_size, table_width);
  if (f8_cluster(static_cast<long long>(B) * nkv * z.slices, table_width, block_size, mode)) return 0;
  return 2ll * z.teams * z.G * (kFp8D + 2) + 4ll * z.teams;
}

static bool f8_maps(const Fp8Decode& a, int tile, CUtensorMap* tm_k, CUtensorMap* tm_v) {
  const uint64_t rows = static_cast<uint64_t>(a.num_blocks) * a.nkv * a.block_size;
  const uint32_t box = static_cast<uint32_t>(std::min(a.block_size, tile));
  return forge_make_tmap_2d(tm_k, a.k_codes, rows, kFp8D, kFp8D, box, 1) == 0 && forge_make_tmap_2d(tm_v, a.v_codes, rows, kFp8D, kFp8D, box, 1) == 0;
}

template <bool kRaw, bool kWide>
static int f8_launch_clusters(Fp8Decode a, int C, cudaStream_t stream) {
  a.stages = static_cast<long long>(a.table_width) * a.block_size <= static_cast<long long>(C) * F8ClusterRing::kTile ? 1 : kF8CStages;
  CUtensorMap tm_k, tm_v;
  if (!f8_maps(a, F8ClusterRing::kTile, &tm_k, &tm_v)) return -2;
  FORGE_ENSURE_DYN_SMEM((decode_fp8_cluster_kernel<kRaw, kWide>), f8_cluster_smem(kF8Heads, kF8CStages));
  return launch_kernel_cluster_x(decode_fp8_cluster_kernel<kRaw, kWide>, dim3(C, static_cast<unsigned>(a.B * a.nkv * a.slices)), dim3(kF8CThreads), f8_cluster_smem(a.G, a.stages),
                                 stream, C, tm_k, tm_v, a) == cudaSuccess ? 0 : -5;
}

static Fp8Decode f8_operands(void* k_codes, void* k_scales, void* v_codes, void* v_scales, const int* block_tables, const int* lens, void* out,
                             const F8Grid& z, int B, int nq, int nkv, int block_size, int table_width, int num_blocks, float scale, unsigned* status) {
  Fp8Decode a = {};
  a.k_codes = static_cast<uint8_t*>(k_codes); a.k_scales = static_cast<uint8_t*>(k_scales);
  a.v_codes = static_cast<uint8_t*>(v_codes); a.v_scales = static_cast<uint8_t*>(v_scales);
  a.block_tables = block_tables; a.lens = lens; a.out = static_cast<__nv_bfloat16*>(out);
  a.B = B; a.nq = nq; a.nkv = nkv; a.group = nq / nkv; a.G = z.G; a.slices = z.slices; a.block_size = block_size; a.table_width = table_width; a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f; a.status = status;
  return a;
}

// q [B, nq, 128], out [B, nq * 128] bf16; a length of zero or less gives a row of zeros.  scratch: forge_decode_fp8_scratch_floats, 16-byte aligned.
extern "C" int forge_decode_fp8(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                                const int* block_tables, const int* lens, void* out, float* scratch, int B, int nq, int nkv, int block_size,
                                int table_width, int num_blocks, float scale, int mode, unsigned* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (!f8_shape(nq, nkv, block_size)) return -1;
  const F8Grid z = f8_grid(B, nq, nkv, block_size, table_width);
  Fp8Decode a = f8_operands(const_cast<void*>(k_codes), const_cast<void*>(k_scales), const_cast<void*>(v_codes), const_cast<void*>(v_scales), block_tables,
                            lens, out, z, B, nq, nkv, block_size, table_width, num_blocks, scale, status);
  a.q = static_cast<const __nv_bfloat16*>(q);
  if (const int C = f8_cluster(static_cast<long long>(B) * nkv * z.slices, table_width, block_size, mode))
    return z.G > 4 ? f8_launch_clusters<false, true>(a, C, stream) : f8_launch_clusters<false, false>(a, C, stream);
  const long long tiles = (static_cast<long long>(table_width) * block_size + F8FlatRing::kTile - 1) / F8FlatRing::kTile;
  if (std::min(B, kF8Seqs) * (tiles + kF8ItemCost) * nkv * z.slices > INT32_MAX) return -1;
  CUtensorMap tm_k, tm_v;
  if (!f8_maps(a, F8FlatRing::kTile, &tm_k, &tm_v)) return -2;
  FORGE_ENSURE_DYN_SMEM(decode_fp8_kernel<true>, kF8FlatSmem);
  FORGE_ENSURE_DYN_SMEM(decode_fp8_kernel<false>, kF8FlatSmem);
  const auto shares = z.G > 4 ? decode_fp8_kernel<true> : decode_fp8_kernel<false>;
  a.cuts = reinterpret_cast<int4*>(scratch);
  a.part_o = scratch + 4ll * z.teams;
  a.part_ml = a.part_o + 2ll * z.teams * z.G * kFp8D;
  for (int left = B; left > 0; left -= kF8Seqs) {
    a.B = std::min(left, kF8Seqs);
    if (launch_kernel(shares, dim3(z.ctas), dim3(kF8Threads), kF8FlatSmem, stream, 0, tm_k, tm_v, a) != cudaSuccess) return -5;
    if (launch_kernel(decode_fp8_join_kernel, dim3(z.teams, z.G), dim3(a.B * nkv * z.slices <= 32 ? 256 : 128), 0, stream, 0, a) != cudaSuccess) return -5;
    a.q += static_cast<size_t>(kF8Seqs) * nq * kFp8D;
    a.block_tables += static_cast<size_t>(kF8Seqs) * table_width;
    a.lens += kF8Seqs;
    a.out += static_cast<size_t>(kF8Seqs) * nq * kFp8D;
  }
  return 0;
}

// The same from the raw projection qkv [B, (nq + 2 nkv) * 128] of the sequences' newest tokens (position length - 1; rows ld apart, 16-byte aligned): queries
// are normed and rotated, and the newest token's keys and values stored, as forge_fp8_store does, bit for bit.  Always by clusters; at most 2^16 items.
extern "C" int forge_decode_fp8_qkv(const void* qkv, long long ld, const void* qw, const void* kw, float eps, const float* rope, int rope_rows,
                                    void* k_codes, void* k_scales, void* v_codes, void* v_scales, const int* block_tables, const int* lens, void* out, int B,
                                    int nq, int nkv, int block_size, int table_width, int num_blocks, float scale, unsigned* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (!f8_shape(nq, nkv, block_size)) return -1;
  const F8Grid z = f8_grid(B, nq, nkv, block_size, table_width);
  const int C = f8_cluster(static_cast<long long>(B) * nkv * z.slices, table_width, block_size, 2);
  if (C == 0) return -1;
  Fp8Decode a = f8_operands(k_codes, k_scales, v_codes, v_scales, block_tables, lens, out, z, B, nq, nkv, block_size, table_width, num_blocks, scale, status);
  a.qkv = static_cast<const __nv_bfloat16*>(qkv); a.ld_qkv = ld;
  a.qw = static_cast<const __nv_bfloat16*>(qw); a.kw = static_cast<const __nv_bfloat16*>(kw);
  a.eps = eps; a.rope = rope; a.rope_rows = rope_rows;
  return z.G > 4 ? f8_launch_clusters<true, true>(a, C, stream) : f8_launch_clusters<true, false>(a, C, stream);
}

}  // namespace forge
