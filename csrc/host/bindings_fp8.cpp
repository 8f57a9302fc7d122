// Bindings of the ops that keep keys, values and normed rows in 8 bits.  As in bindings.cpp every argument is checked here (device, type,
// contiguity, shapes, alignment), so a malformed call raises in Python instead of reaching a kernel.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cstdint>
#include <tuple>

#include "checks.h"

extern "C" {
int forge_fp8_store(const void* qkv, long long ld, const void* qw, const void* kw, float eps, const float* rope, int rope_rows,
                    const int* positions, const int* slots, void* q_out, void* k_codes, void* k_scales, void* v_codes, void* v_scales, int T,
                    int nq, int nkv, int block_size, long long num_slots, unsigned* status, cudaStream_t stream);
int forge_fp8_expand(const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales, const int* block_tables,
                     const int* lens, int num_seqs, int table_width, int num_blocks, int nkv, int block_size, void* k_out, void* v_out,
                     int* tables, int capacity, unsigned* status, cudaStream_t stream);
int forge_decode_fp8(const void* q, const void* k_codes, const void* k_scales, const void* v_codes, const void* v_scales,
                     const int* block_tables, const int* lens, void* out, float* scratch, int B, int nq, int nkv, int block_size, int table_width,
                     int num_blocks, float scale, int mode, unsigned* status, cudaStream_t stream);
int forge_decode_fp8_qkv(const void* qkv, long long ld, const void* qw, const void* kw, float eps, const float* rope, int rope_rows, void* k_codes,
                         void* k_scales, void* v_codes, void* v_scales, const int* block_tables, const int* lens, void* out, int B, int nq, int nkv,
                         int block_size, int table_width, int num_blocks, float scale, unsigned* status, cudaStream_t stream);
int forge_decode_fp8_qkv_pays(int B, int nq, int nkv, int block_size, int table_width);
long long forge_decode_fp8_scratch_floats(int B, int nq, int nkv, int block_size, int table_width, int mode);
int forge_rms_norm_fp8(const void* x, void* residual, const void* w, void* codes, float* scales, int scale_ld, int rows, int H, float eps,
                       cudaStream_t stream);
}

namespace {

constexpr auto BF = at::kBFloat16;
constexpr auto U8 = at::kByte;
constexpr auto E4M3 = at::kFloat8_e4m3fn;

// An uninitialised tensor beside `like`, without the way through the dispatcher: half a microsecond each, of calls of eight.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
void same_device(const Tensor& a, const Tensor& b, const char* what) { TORCH_CHECK(a.device() == b.device(), what, ": tensors on one device expected"); }
void aligned16(const Tensor& t, const char* what) { TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, what, ": 16-byte alignment needed"); }

// One half (keys or values) of a paged 8-bit cache.
struct Half {
  void *codes, *scales;
  int64_t blocks, nkv, block;
};
Half cache_half(const Tensor& codes, const Tensor& scales, const Tensor& with, const char* what) {
  TORCH_CHECK(codes.dim() == 4 && codes.size(3) == 128, what, ": codes must be [blocks, kv_heads, block_size, 128]");
  TORCH_CHECK(scales.dim() == 3 && scales.size(0) == codes.size(0) && scales.size(1) == codes.size(1) && scales.size(2) == codes.size(2), what,
              ": scales must be [blocks, kv_heads, block_size]");
  TORCH_CHECK(codes.size(0) >= 1 && codes.size(1) >= 1, what, ": an empty cache");
  same_device(codes, with, what);
  same_device(scales, with, what);
  Half h{data(codes, E4M3, 1, what), data(scales, U8, 1, what), codes.size(0), codes.size(1), codes.size(2)};
  aligned16(codes, what);
  aligned16(scales, what);
  TORCH_CHECK(h.block >= 16 && (h.block & (h.block - 1)) == 0, what, ": block_size must be a power of two from 16 on");
  TORCH_CHECK(h.blocks * h.nkv * h.block <= INT32_MAX, what, ": more than 2^31 - 1 token rows");
  return h;
}

const void* norm_weight(const OptTensor& w, const Tensor& with, const char* what) {
  if (!w.has_value()) return nullptr;
  TORCH_CHECK(w->numel() == 128, what, ": norm weights have 128 entries");
  same_device(*w, with, what);
  return data(*w, BF, 128, what);
}

// The rotation table, if any.
const float* angles(const OptTensor& rope, const Tensor& with, int& rows, const char* what) {
  rows = 0;
  if (!rope.has_value()) return nullptr;
  TORCH_CHECK(rope->dim() == 2 && rope->size(1) == 128 && rope->size(0) >= 1, what, ": the rotation table must be [positions, 128]");
  same_device(*rope, with, what);
  const float* p = floats(*rope, 128, what);
  aligned16(*rope, what);
  rows = i32(rope->size(0));
  return p;
}

// Returns q [T, nq, 128].
Tensor fp8_store(const Tensor& qkv, const OptTensor& qw, const OptTensor& kw, double eps, const OptTensor& rope, const Tensor& positions,
                 const Tensor& slots, const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales, int64_t nq,
                 const Tensor& status) {
  const Half k = cache_half(k_codes, k_scales, qkv, "fp8_store"), v = cache_half(v_codes, v_scales, qkv, "fp8_store");
  TORCH_CHECK(k_codes.sizes() == v_codes.sizes(), "fp8_store: keys and values of one shape expected");
  TORCH_CHECK(qkv.dim() == 2 && nq >= 1, "fp8_store: qkv must be [T, (nq + 2 nkv) * 128]");
  const int64_t T = qkv.size(0);
  view2(qkv, BF, T, (nq + 2 * k.nkv) * 128, "fp8_store: qkv");
  TORCH_CHECK(T <= 1 || qkv.stride(0) >= qkv.size(1), "fp8_store: rows of qkv overlap");
  int rope_rows;
  const float* rp = angles(rope, qkv, rope_rows, "fp8_store: rotation table");
  same_device(positions, qkv, "fp8_store");
  same_device(slots, qkv, "fp8_store");
  same_device(status, qkv, "fp8_store");
  const c10::cuda::CUDAGuard guard(qkv.device());
  Tensor q = fresh({T, nq, 128}, BF, qkv);
  check_rc(forge_fp8_store(qkv.data_ptr(), T > 1 ? qkv.stride(0) : qkv.size(1), norm_weight(qw, qkv, "fp8_store"), norm_weight(kw, qkv, "fp8_store"),
                           static_cast<float>(eps), rp, rope_rows, ints(positions, T, "fp8_store: positions"), ints(slots, T, "fp8_store: slots"), q.data_ptr(),
                           k.codes, k.scales, v.codes, v.scales, i32(T), i32(nq), i32(k.nkv), i32(k.block), k.blocks * k.block,
                           status_word(status), stream_of(qkv)),
           "forge_fp8_store");
  return q;
}

// Returns (keys, values) [pages, nkv, block_size, 128] and the page numbers [sequences, width].
std::tuple<Tensor, Tensor, Tensor> fp8_expand(const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales,
                                              const Tensor& block_tables, const Tensor& lens, int64_t pages, const Tensor& status) {
  const Half k = cache_half(k_codes, k_scales, k_codes, "fp8_expand"), v = cache_half(v_codes, v_scales, k_codes, "fp8_expand");
  TORCH_CHECK(k_codes.sizes() == v_codes.sizes(), "fp8_expand: keys and values of one shape expected");
  TORCH_CHECK(block_tables.dim() == 2 && pages >= 0, "fp8_expand: tables must be [sequences, width], and the pages not negative");
  for (const Tensor* t : {&block_tables, &lens, &status}) same_device(*t, k_codes, "fp8_expand");
  const int64_t S = block_tables.size(0), W = block_tables.size(1);
  TORCH_CHECK(S <= 65535 && W * k.block <= INT32_MAX, "fp8_expand: too many sequences or too wide a table");
  const int* bt = ints(block_tables, S * W, "fp8_expand: tables");
  const int* ln = ints(lens, S, "fp8_expand: lengths");
  const c10::cuda::CUDAGuard guard(k_codes.device());
  Tensor k_out = fresh({pages, k.nkv, k.block, 128}, BF, k_codes), v_out = fresh({pages, k.nkv, k.block, 128}, BF, k_codes);
  Tensor tables = fresh({S, W}, at::kInt, k_codes);
  check_rc(forge_fp8_expand(k.codes, k.scales, v.codes, v.scales, bt, ln, i32(S), i32(W), i32(k.blocks), i32(k.nkv), i32(k.block), k_out.data_ptr(),
                            v_out.data_ptr(), tables.data_ptr<int>(), i32(pages), status_word(status), stream_of(k_codes)),
           "forge_fp8_expand");
  return {k_out, v_out, tables};
}

// The attention kernels round lengths up to whole tiles of up to 128 tokens in 32 bits.
constexpr int64_t kMostTokens = INT32_MAX - 127;

// Returns [sequences, nq * 128].  mode: 0 by size, 1 equal shares over the GPU, 2 a cluster of CTAs per sequence and KV head.
Tensor decode_fp8(const Tensor& q, const Tensor& k_codes, const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales,
                  const Tensor& block_tables, const Tensor& lens, double scale, const Tensor& status, int64_t mode) {
  const Half k = cache_half(k_codes, k_scales, q, "decode_fp8"), v = cache_half(v_codes, v_scales, q, "decode_fp8");
  TORCH_CHECK(k_codes.sizes() == v_codes.sizes(), "decode_fp8: keys and values of one shape expected");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && block_tables.dim() == 2, "decode_fp8: q must be [sequences, heads, 128], tables [sequences, width]");
  const int64_t B = q.size(0), nq = q.size(1), W = block_tables.size(1);
  TORCH_CHECK(nq >= 1 && nq % k.nkv == 0, "decode_fp8: query heads must be a multiple of the KV heads");
  TORCH_CHECK(block_tables.size(0) >= B, "decode_fp8: a table for every sequence expected");
  TORCH_CHECK(W * k.block <= kMostTokens, "decode_fp8: too wide a table");
  for (const Tensor* t : {&block_tables, &lens, &status}) same_device(*t, q, "decode_fp8");
  const void* qp = data(q, BF, 0, "decode_fp8: q");
  if (B > 0) aligned16(q, "decode_fp8: q");
  const int* bt = ints(block_tables, B * W, "decode_fp8: tables");
  const int* ln = ints(lens, B, "decode_fp8: lengths");
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = fresh({B, nq * 128}, BF, q);
  const int64_t floats = forge_decode_fp8_scratch_floats(i32(B), i32(nq), i32(k.nkv), i32(k.block), i32(W), i32(mode));
  Tensor scratch;
  if (floats > 0) scratch = fresh({floats}, at::kFloat, q);
  check_rc(forge_decode_fp8(qp, k.codes, k.scales, v.codes, v.scales, bt, ln, out.data_ptr(), floats > 0 ? scratch.data_ptr<float>() : nullptr, i32(B), i32(nq),
                            i32(k.nkv), i32(k.block), i32(W), i32(k.blocks), static_cast<float>(scale), i32(mode), status_word(status), stream_of(q)),
           "forge_decode_fp8");
  return out;
}

// From the raw projection qkv [sequences, (nq + 2 nkv) * 128]: norm, rotation and the store of the newest token included.
Tensor decode_fp8_qkv(const Tensor& qkv, const OptTensor& qw, const OptTensor& kw, double eps, const OptTensor& rope, const Tensor& k_codes,
                      const Tensor& k_scales, const Tensor& v_codes, const Tensor& v_scales, const Tensor& block_tables, const Tensor& lens, int64_t nq,
                      double scale, const Tensor& status) {
  const Half k = cache_half(k_codes, k_scales, qkv, "decode_fp8_qkv"), v = cache_half(v_codes, v_scales, qkv, "decode_fp8_qkv");
  TORCH_CHECK(k_codes.sizes() == v_codes.sizes(), "decode_fp8_qkv: keys and values of one shape expected");
  TORCH_CHECK(qkv.dim() == 2 && block_tables.dim() == 2, "decode_fp8_qkv: qkv must be [sequences, (nq + 2 nkv) * 128], tables [sequences, width]");
  const int64_t B = qkv.size(0), W = block_tables.size(1), ld = B > 1 ? qkv.stride(0) : qkv.size(1);
  TORCH_CHECK(nq >= 1 && nq % k.nkv == 0, "decode_fp8_qkv: query heads must be a multiple of the KV heads");
  view2(qkv, BF, B, (nq + 2 * k.nkv) * 128, "decode_fp8_qkv: qkv");
  TORCH_CHECK(ld >= qkv.size(1) && ld % 8 == 0, "decode_fp8_qkv: rows of qkv overlap, or are not aligned to 16 bytes");
  TORCH_CHECK(block_tables.size(0) >= B && W * k.block <= kMostTokens, "decode_fp8_qkv: a table for every sequence expected, not too wide");
  for (const Tensor* t : {&block_tables, &lens, &status}) same_device(*t, qkv, "decode_fp8_qkv");
  if (B > 0) aligned16(qkv, "decode_fp8_qkv: qkv");
  for (const OptTensor* w : {&qw, &kw})
    if (w->has_value()) aligned16(**w, "decode_fp8_qkv: norm weights");
  TORCH_CHECK(B * nq <= 65535, "decode_fp8_qkv: at most 65535 query heads in all: use store and attention");
  int rope_rows;
  const float* rp = angles(rope, qkv, rope_rows, "decode_fp8_qkv: rotation table");
  const int* bt = ints(block_tables, B * W, "decode_fp8_qkv: tables");
  const int* ln = ints(lens, B, "decode_fp8_qkv: lengths");
  const void *qwp = norm_weight(qw, qkv, "decode_fp8_qkv"), *kwp = norm_weight(kw, qkv, "decode_fp8_qkv");
  const c10::cuda::CUDAGuard guard(qkv.device());
  Tensor out = fresh({B, nq * 128}, BF, qkv);
  check_rc(forge_decode_fp8_qkv(qkv.data_ptr(), ld, qwp, kwp, static_cast<float>(eps), rp, rope_rows, k.codes, k.scales, v.codes, v.scales, bt, ln,
                                out.data_ptr(), i32(B), i32(nq), i32(k.nkv), i32(k.block), i32(W), i32(k.blocks), static_cast<float>(scale),
                                status_word(status), stream_of(qkv)),
           "forge_decode_fp8_qkv");
  return out;
}

bool decode_fp8_qkv_pays(int64_t B, int64_t nq, int64_t nkv, int64_t block, int64_t W) {
  const int pays = forge_decode_fp8_qkv_pays(i32(B), i32(nq), i32(nkv), i32(block), i32(W));
  TORCH_CHECK(pays >= 0, "decode_fp8_qkv_pays: query heads must be a multiple of the KV heads, block_size a power of two from 16 on; got ", nq, ", ", nkv, ", ", block);
  return pays != 0;
}

// Returns the codes [rows, H] and their scales [H / 128, rows rounded up to 4].
std::tuple<Tensor, Tensor> rms_norm_fp8(const Tensor& x, const OptTensor& residual, const Tensor& w, double eps) {
  TORCH_CHECK(x.dim() == 2 && x.size(1) >= 128 && x.size(1) % 128 == 0 && x.size(1) <= 16384,
              "rms_norm_fp8: rows must have a multiple of 128 entries, at most 16384");
  const int64_t M = x.size(0), H = x.size(1);
  TORCH_CHECK(w.numel() == H, "rms_norm_fp8: a weight for every column expected");
  void* res = nullptr;
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes(), "rms_norm_fp8: residual of the shape of x expected");
    same_device(*residual, x, "rms_norm_fp8");
    res = data(*residual, BF, 0, "rms_norm_fp8: residual");
    if (M > 0) aligned16(*residual, "rms_norm_fp8: residual");
  }
  same_device(w, x, "rms_norm_fp8");
  const void *xp = data(x, BF, 0, "rms_norm_fp8: x"), *wp = data(w, BF, H, "rms_norm_fp8: weight");
  if (M > 0) aligned16(x, "rms_norm_fp8: x");
  aligned16(w, "rms_norm_fp8: weight");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor codes = fresh({M, H}, E4M3, x), scales = fresh({H / 128, (M + 3) / 4 * 4}, at::kFloat, x);
  check_rc(forge_rms_norm_fp8(xp, res, wp, codes.data_ptr(), scales.data_ptr<float>(), i32(scales.size(1)), i32(M), i32(H), static_cast<float>(eps),
                              stream_of(x)),
           "forge_rms_norm_fp8");
  return {codes, scales};
}

}  // namespace

void register_fp8(pybind11::module& m) {
  m.def("fp8_store", &fp8_store);
  m.def("fp8_expand", &fp8_expand);
  m.def("decode_fp8", &decode_fp8);
  m.def("decode_fp8_qkv", &decode_fp8_qkv);
  m.def("decode_fp8_qkv_pays", &decode_fp8_qkv_pays);
  m.def("rms_norm_fp8", &rms_norm_fp8);
}
