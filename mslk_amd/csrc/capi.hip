// C ABI of the library (declared in include/mslk_amd.h): argument validation, shape-class
// dispatch, error reporting.  No allocation, no synchronisation, no host reads of device memory.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "../../include/mslk_amd.h"
#include "attention.h"
#include "kernels.h"
#include "mx.h"

namespace {

thread_local char g_err[512] = "";

int fail(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return 1;
}

int check_hip(hipError_t e, const char* what) {
  if (e == hipSuccess) return 0;
  return fail("%s: %s", what, hipGetErrorString(e));
}

constexpr int64_t kIntMax = 2147483647;

// Device memory for the padded operand copies (or the fp32 sums of a K split) of mslk_amd_f8f8bf16_rowwise_static_scratch: part of the code object, so
// every GPU the library runs on holds its own copy from module load until the process ends.  In host code the name
// below is only a handle for hipGetSymbolAddress; kernels and copies get the per-device address it returns.
constexpr size_t kScratchBytes = MSLK_AMD_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mutex;
void* g_scratch_ptr[kMaxDevices] = {};

// Address of `scratch` on the current device; looked up once per device, with that device current.
int scratch_of_current_device(void** out) {
  int dev = 0;
  if (int rc = check_hip(hipGetDevice(&dev), "hipGetDevice")) return rc;
  if (dev < 0 || dev >= kMaxDevices) return fail("static scratch: device index %d out of range", dev);
  std::lock_guard<std::mutex> lock(g_scratch_mutex);
  if (g_scratch_ptr[dev] == nullptr) {
    void* ptr = nullptr;
    if (int rc = check_hip(hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)), "hipGetSymbolAddress(scratch)")) return rc;
    if (ptr == nullptr) return fail("static scratch: hipGetSymbolAddress returned a null address");
    g_scratch_ptr[dev] = ptr;
  }
  *out = g_scratch_ptr[dev];
  return 0;
}

}  // namespace

using namespace mslk_amd;

namespace {

// ---------------------------------------------------------------------------------------------------------------------
// attention: checks shared by its entry points
// ---------------------------------------------------------------------------------------------------------------------
constexpr int64_t kMaxTokens = int64_t(1) << 30;

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_heads(const char* op, int dtype, int64_t tokens, int64_t Hq, int64_t Hkv, int64_t D) {
  if (dtype != MSLK_AMD_DTYPE_BF16 && dtype != MSLK_AMD_DTYPE_F16) return fail("%s: bf16 or fp16 expected (dtype code %d)", op, dtype);
  if (tokens < 0 || tokens >= kMaxTokens) return fail("%s: token counts must be in [0, 2^30) (got %lld)", op, (long long)tokens);
  if (Hq <= 0 || Hkv <= 0 || Hq > 65535 || Hq % Hkv != 0)
    return fail("%s: the query heads (%lld, at most 65535) must be a multiple of the KV heads (%lld)", op, (long long)Hq, (long long)Hkv);
  if (D <= 0 || D > kMaxHeadDim || D % 8 != 0) return fail("%s: the head dimension must be a multiple of 8, at most 256 (got %lld)", op, (long long)D);
  return 0;
}
int check_rows(const char* op, const char* what, const mslk_amd_heads* h, HeadRows& out) {
  if (h == nullptr || h->data == nullptr) return fail("%s: null pointer (%s)", op, what);
  // (offsets inside a tile of 64 rows are 32-bit numbers of bytes)
  if (h->token_stride < 0 || h->head_stride < 0 || h->token_stride >= (int64_t(1) << 25)) return fail("%s: stride of %s out of range", op, what);
  if (!aligned(h->data, 16) || h->token_stride % 8 != 0 || h->head_stride % 8 != 0) return fail("%s: rows of %s must begin on 16-byte boundaries", op, what);
  out = HeadRows{(const uint16_t*)h->data, h->token_stride, h->head_stride};
  return 0;
}
int check_cache(const char* op, const mslk_amd_paged_cache* c, int dtype, int64_t sequences, PagedCache& out) {
  if (c == nullptr) return fail("%s: null pointer (cache)", op);
  if (c->dtype != dtype && c->dtype != MSLK_AMD_DTYPE_E4M3FN) return fail("%s: the cache must hold the type of the queries or e4m3 codes (dtype code %d)", op, c->dtype);
  if (sequences < 0 || sequences > 65535) return fail("%s: at most 65535 sequences (got %lld)", op, (long long)sequences);
  if (c->pages < 0 || c->pages > kIntMax || c->page_size <= 0 || c->page_size >= kMaxTokens || c->table_width < 0 || c->table_width >= kMaxTokens)
    return fail("%s: pages, page_size or table_width out of range", op);
  const bool fp8 = c->dtype == MSLK_AMD_DTYPE_E4M3FN;
  if (sequences > 0 && ((c->table_width > 0 && !c->page_table) || !c->kv_lens)) return fail("%s: null pointer (page_table, kv_lens)", op);
  if (c->pages > 0 && (!c->k || !c->v || (fp8 && (!c->k_scale || !c->v_scale)))) return fail("%s: null pointer (cache)", op);
  const uintptr_t row = fp8 ? 8 : 16;
  bool fits = aligned(c->k, row) && aligned(c->v, row);
  for (int i = 0; i < 3; ++i) {
    out.k_stride[i] = c->k_stride[i];
    out.v_stride[i] = c->v_stride[i];
    out.k_scale_stride[i] = c->k_scale_stride[i];
    out.v_scale_stride[i] = c->v_scale_stride[i];
    fits = fits && c->k_stride[i] % 8 == 0 && c->v_stride[i] % 8 == 0;
    // (the kernels count pieces of eight channels, and scales, of a page in 32 bits)
    const int64_t most = int64_t(1) << 32;
    if (c->k_stride[i] < 0 || c->v_stride[i] < 0 || c->k_scale_stride[i] < 0 || c->v_scale_stride[i] < 0 || c->k_stride[i] >= 8 * most ||
        c->v_stride[i] >= 8 * most || c->k_scale_stride[i] >= most || c->v_scale_stride[i] >= most)
      return fail("%s: stride of the cache out of range", op);
  }
  if (!fits) return fail("%s: rows of the cache must begin on %d-byte boundaries", op, (int)row);
  out.k = c->k;
  out.v = c->v;
  out.k_scale = c->k_scale;
  out.v_scale = c->v_scale;
  out.pages = (int)c->pages;
  out.page_size = divider((uint32_t)c->page_size);
  out.table = c->page_table;
  out.table_width = (int)c->table_width;
  out.table_stride = c->table_stride;
  out.lens = c->kv_lens;
  return 0;
}
int check_scale(const char* op, float scale) {   // (the kernels multiply by scale log2(e), which has to be finite too)
  return scale > 0.f && scale <= 2e38f ? 0 : fail("%s: scale must be positive and at most 2e38", op);
}

// ---------------------------------------------------------------------------------------------------------------------
// MXFP4: checks shared by its products
// ---------------------------------------------------------------------------------------------------------------------
int check_mx(const char* op, const void* xq, const void* wq, const void* x_scale, const void* w_scale, const void* y, int y_dtype, int64_t M, int64_t N,
             int64_t K, int gated, int G, const void* workspace, size_t workspace_bytes, size_t wanted) {
  if (M < 0 || N < 0 || K < 0 || G < 0) return fail("%s: negative dimension", op);
  if (K % 32 != 0) return fail("%s: K must be a multiple of 32 (got %lld)", op, (long long)K);
  if (M > kIntMax || N > kIntMax || K >= (int64_t(1) << 24)) return fail("%s: dimension out of range (M, N < 2^31, K < 2^24)", op);
  if (G > (1 << 30)) return fail("%s: at most 2^30 groups (got %d)", op, G);   // (kernels count them in steps of 64)
  if (gated && (N + 256) * K >= (int64_t(1) << 33)) return fail("%s: gated weights of N = %lld, K = %lld are too large (N K < 2^33)", op, (long long)N, (long long)K);
  if (y_dtype != MSLK_AMD_DTYPE_BF16 && y_dtype != MSLK_AMD_DTYPE_F16) return fail("%s: bf16 or fp16 output expected (dtype code %d)", op, y_dtype);
  if (M == 0 || N == 0 || G == 0) return 0;
  if (!y) return fail("%s: null output", op);
  if (!aligned(y, 2)) return fail("%s: the output must be 2-byte aligned", op);
  if (K > 0 && (!xq || !wq || !x_scale || !w_scale)) return fail("%s: null pointer", op);
  if (!aligned(xq, 16) || !aligned(wq, 16)) return fail("%s: codes must be 16-byte aligned", op);
  if (wanted > 0 && (!workspace || workspace_bytes < wanted || !aligned(workspace, 16)))
    return fail("%s: a 16-byte aligned workspace of %zu bytes is wanted", op, wanted);
  return 0;
}

}  // namespace

extern "C" {

const char* mslk_amd_version(void) { return "mslk_amd 0.1 (gfx950)"; }
const char* mslk_amd_last_error(void) { return g_err; }

int mslk_amd_quantize_fp8_row(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_row_stride,
                              void* xq, int64_t K_out, float* scale, const float* scale_ub, void* stream) {
  if (x_dtype < 0 || x_dtype > 2) return fail("quantize_fp8_row: unsupported input dtype code %d", x_dtype);
  if (rows < 0 || K <= 0) return fail("quantize_fp8_row: rows must be >= 0 and K > 0 (got %lld, %lld)", (long long)rows, (long long)K);
  if (K_out < K) return fail("quantize_fp8_row: K_out (%lld) < K (%lld)", (long long)K_out, (long long)K);
  if (rows == 0) return 0;
  if (rows > kIntMax) return fail("quantize_fp8_row: rows (%lld) exceeds 2^31-1", (long long)rows);
  if (!x || !xq || !scale) return fail("quantize_fp8_row: null pointer");
  return check_hip(launch_quantize_fp8_row(x, x_dtype, rows, K, x_row_stride, xq, K_out, scale, scale_ub, nullptr, 0, 1,
                                           0, 0.f, (hipStream_t)stream),
                   "quantize_fp8_row launch");
}

int mslk_amd_quantize_fp8_row_jagged(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_row_stride,
                                     void* xq, int64_t K_out, float* scale, const float* scale_ub,
                                     const void* zero_start_index, int index_dtype, int64_t rows_per_group,
                                     void* stream) {
  if (x_dtype < 0 || x_dtype > 2) return fail("quantize_fp8_row_jagged: unsupported input dtype code %d", x_dtype);
  if (index_dtype != MSLK_AMD_INDEX_I64 && index_dtype != MSLK_AMD_INDEX_I32)
    return fail("quantize_fp8_row_jagged: unsupported index dtype code %d", index_dtype);
  if (rows < 0 || K <= 0) return fail("quantize_fp8_row_jagged: rows must be >= 0 and K > 0 (got %lld, %lld)", (long long)rows, (long long)K);
  if (K_out < K) return fail("quantize_fp8_row_jagged: K_out (%lld) < K (%lld)", (long long)K_out, (long long)K);
  if (rows_per_group <= 0 || rows % rows_per_group != 0)
    return fail("quantize_fp8_row_jagged: rows (%lld) must be a multiple of rows_per_group (%lld)", (long long)rows,
                (long long)rows_per_group);
  if (rows == 0) return 0;
  if (rows > kIntMax) return fail("quantize_fp8_row_jagged: rows (%lld) exceeds 2^31-1", (long long)rows);
  if (!x || !xq || !scale || !zero_start_index) return fail("quantize_fp8_row_jagged: null pointer");
  return check_hip(launch_quantize_fp8_row(x, x_dtype, rows, K, x_row_stride, xq, K_out, scale, scale_ub,
                                           zero_start_index, index_dtype == MSLK_AMD_INDEX_I32, rows_per_group,
                                           0, 0.f, (hipStream_t)stream),
                   "quantize_fp8_row_jagged launch");
}

int mslk_amd_quantize_fp8_row_triton_arithmetic(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t x_row_stride,
                                                void* xq, int64_t K_out, float* scale, const float* scale_ub, float eps,
                                                const void* zero_start_index, int index_dtype, int64_t rows_per_group,
                                                void* stream) {
  const char* op = "quantize_fp8_row_triton_arithmetic";
  if (x_dtype < 0 || x_dtype > 2) return fail("%s: unsupported input dtype code %d", op, x_dtype);
  if (rows < 0 || K <= 0) return fail("%s: rows must be >= 0 and K > 0 (got %lld, %lld)", op, (long long)rows, (long long)K);
  if (K_out < K) return fail("%s: K_out (%lld) < K (%lld)", op, (long long)K_out, (long long)K);
  if (!(eps > 0.f)) return fail("%s: eps must be positive", op);
  if (zero_start_index != nullptr) {
    if (index_dtype != MSLK_AMD_INDEX_I64 && index_dtype != MSLK_AMD_INDEX_I32) return fail("%s: unsupported index dtype code %d", op, index_dtype);
    if (rows_per_group <= 0 || rows % rows_per_group != 0)
      return fail("%s: rows (%lld) must be a multiple of rows_per_group (%lld)", op, (long long)rows, (long long)rows_per_group);
  }
  if (rows == 0) return 0;
  if (rows > kIntMax) return fail("%s: rows (%lld) exceeds 2^31-1", op, (long long)rows);
  if (!x || !xq || !scale) return fail("%s: null pointer", op);
  return check_hip(launch_quantize_fp8_row(x, x_dtype, rows, K, x_row_stride, xq, K_out, scale, scale_ub, zero_start_index,
                                           index_dtype == MSLK_AMD_INDEX_I32, rows_per_group, 1, eps, (hipStream_t)stream),
                   "quantize_fp8_row_triton_arithmetic launch");
}

int mslk_amd_dequantize_fp8_row(const void* xq, const float* scale, int64_t rows, int64_t K, void* out, void* stream) {
  if (rows < 0 || K < 0) return fail("dequantize_fp8_row: negative dimension");
  if (rows == 0 || K == 0) return 0;
  if (!xq || !scale || !out) return fail("dequantize_fp8_row: null pointer");
  return check_hip(launch_dequantize_fp8_row(xq, scale, rows, K, out, (hipStream_t)stream), "dequantize_fp8_row launch");
}

int mslk_amd_silu_mul_quant(const void* x0, const void* x1, int x_dtype, int64_t T, int64_t D, int64_t x0_row_stride,
                            int64_t x1_row_stride, void* out, float* out_scale, const float* scale_ub,
                            const void* valid_token_count, int count_dtype, void* stream) {
  if (x_dtype != MSLK_AMD_DTYPE_BF16 && x_dtype != MSLK_AMD_DTYPE_F16)
    return fail("silu_mul_quant: inputs must be bf16 or fp16 (dtype code %d)", x_dtype);
  if (count_dtype != MSLK_AMD_INDEX_I64 && count_dtype != MSLK_AMD_INDEX_I32)
    return fail("silu_mul_quant: unsupported valid_token_count dtype code %d", count_dtype);
  if (T < 0 || D < 0) return fail("silu_mul_quant: negative dimension");
  if (T > kIntMax || D > kIntMax) return fail("silu_mul_quant: dimension exceeds 2^31-1");
  if (T == 0 || D == 0) return 0;
  if (!x0 || !x1 || !out || !out_scale) return fail("silu_mul_quant: null pointer");
  if (x0_row_stride < D || x1_row_stride < D) return fail("silu_mul_quant: row stride smaller than D");
  FusedQuantArgs p{};
  p.x0 = x0; p.x1 = x1; p.stride0 = x0_row_stride; p.stride1 = x1_row_stride; p.dtype = x_dtype;
  p.out = (uint8_t*)out; p.out_scale = out_scale; p.rows = T; p.D = (int)D; p.scale_ub = scale_ub;
  p.valid_count = valid_token_count; p.valid_is_i64 = count_dtype == MSLK_AMD_INDEX_I64;
  return check_hip(launch_fused_quant(p, kFusedSiluMul, (hipStream_t)stream), "silu_mul_quant launch");
}

int mslk_amd_gather_scale_quant_dense_tokens(const void* x, int x_dtype, int64_t T, int64_t D,
                                             const void* token_indices, int token_dtype,
                                             const void* expert_indices, int expert_dtype, int64_t a,
                                             const void* scores, int score_dtype, int64_t E, int64_t score_stride_t,
                                             int64_t score_stride_e, void* out, float* out_scale,
                                             const float* scale_ub, const void* valid_token_count, int count_dtype,
                                             void* stream) {
  const char* op = "gather_scale_quant_dense_tokens";
  if (x_dtype != MSLK_AMD_DTYPE_BF16 && x_dtype != MSLK_AMD_DTYPE_F16) return fail("%s: x must be bf16 or fp16 (dtype code %d)", op, x_dtype);
  if (score_dtype < 0 || score_dtype > 2) return fail("%s: unsupported scores dtype code %d", op, score_dtype);
  if ((token_dtype | expert_dtype | count_dtype) & ~1) return fail("%s: index dtype codes must be MSLK_AMD_INDEX_I64 or _I32", op);
  if (T < 0 || D < 0 || a < 0 || E < 0) return fail("%s: negative dimension", op);
  if (a > kIntMax || D > kIntMax) return fail("%s: dimension exceeds 2^31-1", op);
  if (a == 0 || D == 0) return 0;
  if (!x || !token_indices || !expert_indices || !scores || !out || !out_scale) return fail("%s: null pointer", op);
  FusedQuantArgs p{};
  p.x0 = x; p.stride0 = D; p.dtype = x_dtype;
  p.out = (uint8_t*)out; p.out_scale = out_scale; p.rows = a; p.D = (int)D; p.scale_ub = scale_ub;
  p.valid_count = valid_token_count; p.valid_is_i64 = count_dtype == MSLK_AMD_INDEX_I64;
  p.token_idx = token_indices; p.token_is_i64 = token_dtype == MSLK_AMD_INDEX_I64;
  p.expert_idx = expert_indices; p.expert_is_i64 = expert_dtype == MSLK_AMD_INDEX_I64;
  p.scores = scores; p.score_dtype = score_dtype; p.stride_t = score_stride_t; p.stride_e = score_stride_e;
  p.T = T; p.E = E;
  return check_hip(launch_fused_quant(p, kFusedGatherScale, (hipStream_t)stream), "gather_scale_quant launch");
}

// K that is not a multiple of 16: the operand rows cannot be fetched by the 16-byte loads of the MFMA kernels.  With a
// workspace the call copies both operands into rows of K rounded up to 16 (zero tail: code 0x00 is +0) and runs the
// ordinary kernels on the copies; without one it falls back to the scalar kernel, which is orders of magnitude slower.
// K a multiple of 16 on a shape with few output tiles and a long K: with a workspace of slices * M * N floats the call
// splits K (gemm_splitk.hip); without one it runs the ordinary kernels.
size_t mslk_amd_f8f8bf16_rowwise_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M > kIntMax || N > kIntMax || K > kIntMax) return 0;
  if (K % 16 != 0) return (size_t)((M + N) * ((K + 15) / 16 * 16));
  const SplitKPlan plan = splitk_plan(M, N, K, device_compute_units());
  return plan.slices > 1 ? (size_t)plan.slices * (size_t)M * (size_t)N * sizeof(float) : 0;
}

static int rowwise_impl(const char* op, int out_f16, int preshuffled, const void* xq, const void* wq, const float* x_scale,
                        const float* w_scale, const void* bias, int bias_dtype, void* y, int64_t M, int64_t N,
                        int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || K < 0) return fail("%s: negative dimension", op);
  if (M > kIntMax || N > kIntMax || K > kIntMax) return fail("%s: dimension exceeds 2^31-1", op);
  if (bias_dtype < 0 || bias_dtype > 2) return fail("%s: bad bias dtype code %d", op, bias_dtype);
  if ((bias_dtype != 0) != (bias != nullptr)) return fail("%s: bias pointer and bias dtype disagree", op);
  hipStream_t s = (hipStream_t)stream;
  if (M == 0 || N == 0) return 0;
  if (!y) return fail("%s: null output", op);
  if (K == 0) return check_hip(launch_fill_zero_bf16((uint16_t*)y, M * N, s), "zero fill");
  if (!xq || !wq || !x_scale || !w_scale) return fail("%s: null pointer", op);
  if (preshuffled && (N % 16 != 0 || K % 64 != 0))
    return fail("%s: pre-shuffled weights need N %% 16 == 0 and K %% 64 == 0 (got N=%lld, K=%lld)", op, (long long)N, (long long)K);
  GemmProblem p{(const uint8_t*)xq, (const uint8_t*)wq, x_scale, w_scale, bias, (uint16_t*)y,
                (int)M, (int)N, (int)K, bias_dtype, out_f16, preshuffled};
  // Operand rows the 16-byte loads cannot fetch (K % 16 != 0, or a base pointer that is not 16-byte aligned) are copied
  // into the workspace when the caller gave one that holds both copies.
  const int64_t Kp = (K + 15) / 16 * 16;
  const bool unfetchable = K % 16 != 0 || reinterpret_cast<uintptr_t>(xq) % 16 != 0 || reinterpret_cast<uintptr_t>(wq) % 16 != 0;
  if (unfetchable && !preshuffled && workspace && workspace_bytes >= (size_t)((M + N) * Kp) &&
      reinterpret_cast<uintptr_t>(workspace) % 16 == 0) {
    if (Kp <= kIntMax) {
      uint8_t* xp = static_cast<uint8_t*>(workspace);
      uint8_t* wp = xp + M * Kp;
      if (int rc = check_hip(launch_pad_rows(p.xq, xp, M, K, Kp, s), "pad rows launch")) return rc;
      if (int rc = check_hip(launch_pad_rows(p.wq, wp, N, K, Kp, s), "pad rows launch")) return rc;
      p.xq = xp;
      p.wq = wp;
      p.K = (int)Kp;
    }
  }
  const bool tiled_ok = dense_tiled_supports(p);
  // Few output tiles and a long K: split K when the caller's workspace holds the fp32 sums of every slice.
  if (!unfetchable && tiled_ok && workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0) {
    const SplitKPlan plan = splitk_plan(M, N, K, device_compute_units());
    if (plan.slices > 1 && workspace_bytes >= (size_t)plan.slices * (size_t)M * (size_t)N * sizeof(float))
      return check_hip(launch_splitk(p, plan, static_cast<float*>(workspace), s), "split-K launch");
  }
  // M <= 64: the weight-streaming kernel, except on wide row-major weights, where short tiles that share their
  // activation rows through LDS win from M = 9 on.  Pre-shuffled weights
  // keep the streaming kernel, whose register-direct weight loads stay ahead up to M = 64.
  const bool wide = !p.w_preshuffled && p.M > 8 && p.N >= kShortTileMinN;
  if (skinny_supports(p) && !(tiled_ok && wide)) return check_hip(launch_skinny(p, s), "skinny launch");
  if (tiled_ok) return check_hip(launch_dense_tiled(p, s), "tiled launch");
  return check_hip(launch_generic(p, s), "generic launch");
}

int mslk_amd_f8f8bf16_rowwise(const void* xq, const void* wq, const float* x_scale, const float* w_scale,
                              const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                              void* workspace, size_t workspace_bytes, void* stream) {
  return rowwise_impl("f8f8bf16_rowwise", 0, 0, xq, wq, x_scale, w_scale, bias, bias_dtype, y, M, N, K, workspace, workspace_bytes, stream);
}

size_t mslk_amd_static_scratch_bytes(void) { return kScratchBytes; }

int mslk_amd_f8f8bf16_rowwise_static_scratch(const void* xq, const void* wq, const float* x_scale, const float* w_scale,
                                             const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                                             void* stream) {
  const char* op = "f8f8bf16_rowwise_static_scratch";
  void* ptr = nullptr;
  size_t bytes = 0;
  const bool unfetchable = K % 16 != 0 || reinterpret_cast<uintptr_t>(xq) % 16 != 0 || reinterpret_cast<uintptr_t>(wq) % 16 != 0;
  if (M > 0 && N > 0 && K > 0 && M <= kIntMax && N <= kIntMax && K <= kIntMax && unfetchable) {
    const int64_t Kp = (K + 15) / 16 * 16;
    const double need = ((double)M + (double)N) * (double)Kp;
    if (need > (double)kScratchBytes)
      return fail("%s: the padded operand copies need (M + N) * round_up(K, 16) = %.0f bytes, the static scratch array holds %zu; "
                  "use mslk_amd_f8f8bf16_rowwise with a workspace", op, need, kScratchBytes);
    if (int rc = scratch_of_current_device(&ptr)) return rc;
    bytes = kScratchBytes;
  } else {
    // a shape the library would split along K: the fp32 sums of the slices go into the array when they fit (otherwise
    // the unsplit kernels run, as without a workspace)
    const size_t need = mslk_amd_f8f8bf16_rowwise_workspace_bytes(M, N, K);
    if (need > 0 && need <= kScratchBytes) {
      if (int rc = scratch_of_current_device(&ptr)) return rc;
      bytes = kScratchBytes;
    }
  }
  return rowwise_impl(op, 0, 0, xq, wq, x_scale, w_scale, bias, bias_dtype, y, M, N, K, ptr, bytes, stream);
}

int mslk_amd_quantize_f8f8bf16_rowwise_supported(int64_t M, int64_t N, int64_t K) {
  return M >= 1 && M <= 4 && N >= 1 && N <= kIntMax && K >= 1024 && K % 128 == 0 && K <= (int64_t(1) << 25);
}

int mslk_amd_quantize_f8f8bf16_rowwise(const void* x, int x_dtype, int64_t x_row_stride, const void* wq, const float* w_scale,
                                       const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                                       void* xq_out, float* x_scale_out, void* stream) {
  const char* op = "quantize_f8f8bf16_rowwise";
  if (x_dtype != MSLK_AMD_DTYPE_BF16) return fail("%s: activations must be bf16 (dtype code %d)", op, x_dtype);
  if (bias_dtype < 0 || bias_dtype > 2) return fail("%s: bad bias dtype code %d", op, bias_dtype);
  if ((bias_dtype != 0) != (bias != nullptr)) return fail("%s: bias pointer and bias dtype disagree", op);
  if (!mslk_amd_quantize_f8f8bf16_rowwise_supported(M, N, K))
    return fail("%s: the one-launch path needs 1 <= M <= 4 and K a multiple of 128, at least 1024 (got M=%lld, N=%lld, K=%lld); "
                "use mslk_amd_quantize_fp8_row followed by mslk_amd_f8f8bf16_rowwise", op, (long long)M, (long long)N, (long long)K);
  if (!x || !wq || !w_scale || !y) return fail("%s: null pointer", op);
  GemmProblem p{nullptr, (const uint8_t*)wq, nullptr, w_scale, bias, (uint16_t*)y, (int)M, (int)N, (int)K, bias_dtype, 0, 0};
  if (!skinny_fused_quant_supports(p, x, x_row_stride) || (xq_out && reinterpret_cast<uintptr_t>(xq_out) % 16 != 0))
    return fail("%s: x, wq and xq_out must be 16-byte aligned and the row stride of x a multiple of 8 elements, at least K", op);
  return check_hip(launch_skinny_fused_quant(p, x, x_row_stride, xq_out, x_scale_out, (hipStream_t)stream), "fused decode launch");
}

int mslk_amd_f8f8f16_rowwise(const void* xq, const void* wq, const float* x_scale, const float* w_scale,
                             const void* bias, int bias_dtype, void* y, int64_t M, int64_t N, int64_t K,
                             void* workspace, size_t workspace_bytes, void* stream) {
  return rowwise_impl("f8f8f16_rowwise", 1, 0, xq, wq, x_scale, w_scale, bias, bias_dtype, y, M, N, K, workspace, workspace_bytes, stream);
}

int mslk_amd_f8f8_rowwise_preshuffle(const void* xq, const void* wq_shuffled, const float* x_scale, const float* w_scale,
                                     const void* bias, int bias_dtype, void* y, int y_dtype, int64_t M, int64_t N,
                                     int64_t K, void* stream) {
  if (y_dtype != MSLK_AMD_DTYPE_BF16 && y_dtype != MSLK_AMD_DTYPE_F16)
    return fail("f8f8_rowwise_preshuffle: output dtype code %d is neither bf16 nor fp16", y_dtype);
  return rowwise_impl(y_dtype == MSLK_AMD_DTYPE_F16 ? "f8f8f16_rowwise_preshuffle" : "f8f8bf16_rowwise_preshuffle",
                      y_dtype == MSLK_AMD_DTYPE_F16, 1, xq, wq_shuffled, x_scale, w_scale, bias, bias_dtype, y, M, N, K, nullptr, 0, stream);
}

int mslk_amd_f8f8_rowwise_preshuffle_workspace(const void* xq, const void* wq_shuffled, const float* x_scale, const float* w_scale,
                                               const void* bias, int bias_dtype, void* y, int y_dtype, int64_t M, int64_t N,
                                               int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (y_dtype != MSLK_AMD_DTYPE_BF16 && y_dtype != MSLK_AMD_DTYPE_F16)
    return fail("f8f8_rowwise_preshuffle: output dtype code %d is neither bf16 nor fp16", y_dtype);
  return rowwise_impl(y_dtype == MSLK_AMD_DTYPE_F16 ? "f8f8f16_rowwise_preshuffle" : "f8f8bf16_rowwise_preshuffle",
                      y_dtype == MSLK_AMD_DTYPE_F16, 1, xq, wq_shuffled, x_scale, w_scale, bias, bias_dtype, y, M, N, K, workspace,
                      workspace_bytes, stream);
}

int mslk_amd_preshuffle_b(const void* wq, void* wq_shuffled, int64_t G, int64_t N, int64_t K, void* stream) {
  if (G < 0 || N < 0 || K < 0) return fail("preshuffle_b: negative dimension");
  if (N % 16 != 0 || K % 64 != 0) return fail("preshuffle_b needs N %% 16 == 0 and K %% 64 == 0, got N=%lld K=%lld", (long long)N, (long long)K);
  if (G == 0 || N == 0 || K == 0) return 0;
  if (!wq || !wq_shuffled) return fail("preshuffle_b: null pointer");
  if (wq == wq_shuffled) return fail("preshuffle_b: the permutation cannot run in place");
  if (reinterpret_cast<uintptr_t>(wq) % 16 || reinterpret_cast<uintptr_t>(wq_shuffled) % 16) return fail("preshuffle_b: pointers must be 16-byte aligned");
  return check_hip(launch_preshuffle_b(wq, wq_shuffled, G, N, K, (hipStream_t)stream), "preshuffle_b launch");
}

int mslk_amd_f8f8bf16_rowwise_grouped(int G, const void* const* xq, const void* const* wq,
                                      const float* const* x_scale, const float* const* w_scale, void* const* y,
                                      const int64_t* M, const int64_t* N, const int64_t* K, void* stream) {
  if (G < 0) return fail("f8f8bf16_rowwise_grouped: negative group count");
  hipStream_t s = (hipStream_t)stream;
  GroupTable tab;
  tab.count = 0;
  tab.total_tiles = 0;
  auto flush = [&]() -> int {
    if (tab.count == 0) return 0;
    int rc = check_hip(launch_grouped_tiled(tab, s), "grouped launch");
    tab.count = 0;
    tab.total_tiles = 0;
    return rc;
  };
  for (int g = 0; g < G; ++g) {
    if (M[g] < 0 || N[g] < 0 || K[g] < 0 || M[g] > kIntMax || N[g] > kIntMax || K[g] > kIntMax)
      return fail("f8f8bf16_rowwise_grouped: bad dimensions in group %d", g);
    if (M[g] == 0 || N[g] == 0) continue;
    if (!y[g]) return fail("f8f8bf16_rowwise_grouped: null output in group %d", g);
    if (K[g] == 0) {
      if (int rc = check_hip(launch_fill_zero_bf16((uint16_t*)y[g], M[g] * N[g], s), "zero fill")) return rc;
      continue;
    }
    if (!xq[g] || !wq[g] || !x_scale[g] || !w_scale[g]) return fail("f8f8bf16_rowwise_grouped: null pointer in group %d", g);
    GemmProblem p{(const uint8_t*)xq[g], (const uint8_t*)wq[g], x_scale[g], w_scale[g], nullptr, (uint16_t*)y[g],
                  (int)M[g], (int)N[g], (int)K[g], 0, 0, 0};
    if (!dense_tiled_supports(p)) {  // odd K or alignment: per-group fallback
      if (int rc = check_hip(launch_generic(p, s), "generic launch")) return rc;
      continue;
    }
    GroupDesc& d = tab.g[tab.count];
    d.xq = p.xq; d.wq = p.wq; d.xs = p.xs; d.ws = p.ws; d.y = p.y;
    d.M = p.M; d.N = p.N; d.K = p.K;
    d.tile_begin = tab.total_tiles;
    const int64_t tiles = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256);
    if (tab.total_tiles + tiles > kIntMax) return fail("f8f8bf16_rowwise_grouped: too many tiles");
    tab.total_tiles += (int)tiles;
    if (++tab.count == kMaxGroupsPerLaunch)
      if (int rc = flush()) return rc;
  }
  return flush();
}

int mslk_amd_f8f8bf16_rowwise_grouped_stacked(const void* xq, const void* wq, const float* x_scale,
                                              const float* w_scale, const int64_t* m_sizes_dev, int G,
                                              int64_t total_M, int64_t N, int64_t K, void* y, void* stream) {
  if (G < 0 || total_M < 0 || N < 0 || K < 0) return fail("f8f8bf16_rowwise_grouped_stacked: negative dimension");
  if (total_M > kIntMax || N > kIntMax || K > kIntMax) return fail("f8f8bf16_rowwise_grouped_stacked: dimension exceeds 2^31-1");
  hipStream_t s = (hipStream_t)stream;
  if (G == 0 || total_M == 0 || N == 0) return 0;
  if (!y) return fail("f8f8bf16_rowwise_grouped_stacked: null output");
  if (K == 0) return check_hip(launch_fill_zero_bf16((uint16_t*)y, total_M * N, s), "zero fill");
  if (!xq || !wq || !x_scale || !w_scale || !m_sizes_dev) return fail("f8f8bf16_rowwise_grouped_stacked: null pointer");
  DeviceGroups p{(const uint8_t*)xq, (const uint8_t*)wq, x_scale, w_scale, nullptr, (uint16_t*)y, m_sizes_dev, G,
                 (int)total_M, (int)N, (int)K, 0, 0};
  return check_hip(launch_device_groups(p, kGroupsSizesM, s), "grouped stacked launch");
}

int mslk_amd_f8f8bf16_rowwise_grouped_mm(const void* xq, const void* wq, const float* x_scale,
                                         const float* w_scale, const int32_t* offsets_dev, int layout, int G,
                                         int64_t M, int64_t N, int64_t K, void* y, void* stream) {
  if (layout < MSLK_AMD_GROUPS_M_OFFSETS || layout > MSLK_AMD_GROUPS_UNIFORM)
    return fail("f8f8bf16_rowwise_grouped_mm: unknown group layout code %d", layout);
  if (G < 0 || M < 0 || N < 0 || K < 0) return fail("f8f8bf16_rowwise_grouped_mm: negative dimension");
  if (M > kIntMax || N > kIntMax || K > kIntMax) return fail("f8f8bf16_rowwise_grouped_mm: dimension exceeds 2^31-1");
  const bool uniform = layout == MSLK_AMD_GROUPS_UNIFORM;
  if (uniform != (offsets_dev == nullptr))
    return fail(uniform ? "f8f8bf16_rowwise_grouped_mm: offsets must be NULL for the uniform layout"
                        : "f8f8bf16_rowwise_grouped_mm: offsets are required for this layout");
  hipStream_t s = (hipStream_t)stream;
  if (G == 0 || M == 0 || N == 0) return 0;
  if (!y) return fail("f8f8bf16_rowwise_grouped_mm: null output");
  const bool stacked_out = layout == MSLK_AMD_GROUPS_K_OFFSETS || uniform;   // y is [G, M, N]
  if (stacked_out && (double)G * (double)M * (double)N > 9.0e18) return fail("f8f8bf16_rowwise_grouped_mm: output too large");
  // K == 0 needs no special case: every tile a group owns is written with the empty sum.
  if ((K > 0 && (!xq || !wq)) || !x_scale || !w_scale) return fail("f8f8bf16_rowwise_grouped_mm: null pointer");
  DeviceGroups p{(const uint8_t*)xq, (const uint8_t*)wq, x_scale, w_scale, nullptr, (uint16_t*)y, offsets_dev, G,
                 (int)M, (int)N, (int)K, 0, 0};
  return check_hip(launch_device_groups(p, layout, s), "grouped_mm launch");
}

int mslk_amd_f8f8bf16_rowwise_grouped_dynamic(const void* xq, const void* wq, const float* x_scale,
                                              const float* w_scale, const int64_t* zero_start_index_M_dev, int G,
                                              int64_t M, int64_t N, int64_t K, void* y, int zeroing_output,
                                              void* stream) {
  if (G < 0 || M < 0 || N < 0 || K < 0) return fail("f8f8bf16_rowwise_grouped_dynamic: negative dimension");
  if (M > kIntMax || N > kIntMax || K > kIntMax) return fail("f8f8bf16_rowwise_grouped_dynamic: dimension exceeds 2^31-1");
  hipStream_t s = (hipStream_t)stream;
  if (G == 0 || M == 0 || N == 0) return 0;
  if (!y) return fail("f8f8bf16_rowwise_grouped_dynamic: null output");
  if ((double)G * (double)M * (double)N > 9.0e18) return fail("f8f8bf16_rowwise_grouped_dynamic: output too large");
  if ((K > 0 && (!xq || !wq)) || !x_scale || !w_scale || !zero_start_index_M_dev)
    return fail("f8f8bf16_rowwise_grouped_dynamic: null pointer");
  if (zeroing_output)
    if (int rc = check_hip(launch_fill_zero_bf16((uint16_t*)y, (int64_t)G * M * N, s), "zero fill")) return rc;
  DeviceGroups p{(const uint8_t*)xq, (const uint8_t*)wq, x_scale, w_scale, nullptr, (uint16_t*)y, zero_start_index_M_dev,
                 G, (int)M, (int)N, (int)K, 0, 0};
  return check_hip(launch_device_groups(p, kGroupsPrepadM, s), "grouped dynamic launch");
}

int mslk_amd_f8f8bf16_rowwise_batched(const void* xq, const void* wq, const float* x_scale, const float* w_scale,
                                      const void* bias, int bias_dtype, int64_t B, int64_t M, int64_t N,
                                      int64_t K, void* y, void* stream) {
  if (B < 0 || M < 0 || N < 0 || K < 0) return fail("f8f8bf16_rowwise_batched: negative dimension");
  if (B > kIntMax || M > kIntMax || N > kIntMax || K > kIntMax) return fail("f8f8bf16_rowwise_batched: dimension exceeds 2^31-1");
  if (bias_dtype < 0 || bias_dtype > 2) return fail("f8f8bf16_rowwise_batched: bad bias dtype code %d", bias_dtype);
  if ((bias_dtype != 0) != (bias != nullptr)) return fail("f8f8bf16_rowwise_batched: bias pointer and bias dtype disagree");
  hipStream_t s = (hipStream_t)stream;
  if (B == 0 || M == 0 || N == 0) return 0;
  if (!y) return fail("f8f8bf16_rowwise_batched: null output");
  if ((double)B * (double)M * (double)N > 9.0e18) return fail("f8f8bf16_rowwise_batched: output too large");
  if ((K > 0 && (!xq || !wq)) || !x_scale || !w_scale) return fail("f8f8bf16_rowwise_batched: null pointer");
  DeviceGroups p{(const uint8_t*)xq, (const uint8_t*)wq, x_scale, w_scale, bias, (uint16_t*)y, nullptr, (int)B,
                 (int)M, (int)N, (int)K, bias_dtype, 0};
  return check_hip(launch_device_groups(p, kGroupsUniform, s), "batched launch");
}

int mslk_amd_append_kv(const mslk_amd_heads* q, const mslk_amd_heads* k, const mslk_amd_heads* v, int dtype, int64_t tokens,
                       int64_t Hq, int64_t Hkv, int64_t D, const mslk_amd_paged_cache* cache, const int32_t* cu_seqlens,
                       int64_t sequences, const float* rotary, int64_t rotary_positions, int64_t rotary_dim, int interleaved,
                       void* q_out, void* stream) {
  const char* op = "append_kv";
  AppendArgs p{};
  if (int rc = check_heads(op, dtype, tokens, Hq, Hkv, D)) return rc;
  if (int rc = check_cache(op, cache, dtype, sequences, p.cache)) return rc;
  if (cu_seqlens == nullptr && sequences != tokens)
    return fail("%s: without cu_seqlens there is one token per sequence (%lld tokens, %lld sequences)", op, (long long)tokens, (long long)sequences);
  if (rotary != nullptr && (rotary_positions < 0 || rotary_dim < 2 || rotary_dim > D || rotary_dim % 2 != 0))
    return fail("%s: rotary_dim must be even and at most the head dimension (got %lld)", op, (long long)rotary_dim);
  if (tokens == 0) return 0;
  if (int rc = check_rows(op, "q", q, p.q)) return rc;
  if (int rc = check_rows(op, "k", k, p.k)) return rc;
  if (int rc = check_rows(op, "v", v, p.v)) return rc;
  if (!q_out || !aligned(q_out, 16)) return fail("%s: q_out must not be null and be 16-byte aligned", op);
  p.q_out = (uint16_t*)q_out;
  p.cu_seqlens = cu_seqlens;
  p.rotary = rotary;
  p.rotary_positions = rotary_positions;
  p.rotary_dim = rotary != nullptr ? (int)rotary_dim : 0;
  p.interleaved = interleaved != 0;
  p.tokens = tokens;
  p.sequences = (int)sequences;
  p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.D = (int)D; p.dtype = dtype;
  p.fp8 = cache->dtype == MSLK_AMD_DTYPE_E4M3FN;
  return check_hip(launch_append_kv(p, (hipStream_t)stream), "append_kv launch");
}

size_t mslk_amd_attention_decode_workspace_bytes(int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D, int64_t table_width, int64_t page_size) {
  if (sequences <= 0 || sequences > 65535 || Hq <= 0 || Hkv <= 0 || Hq > 65535 || Hq % Hkv != 0 || D <= 0 || D > kMaxHeadDim || table_width < 0 ||
      table_width >= kMaxTokens || page_size <= 0 || page_size >= kMaxTokens || table_width * page_size > kMaxTokens)
    return 0;
  return decode_workspace_bytes(sequences, Hq, Hkv, D, table_width * page_size);
}

int mslk_amd_attention_decode(const mslk_amd_heads* q, int dtype, int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D,
                              const mslk_amd_paged_cache* cache, float scale, void* out, float* lse, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* op = "attention_decode";
  DecodeArgs p{};
  if (int rc = check_heads(op, dtype, sequences, Hq, Hkv, D)) return rc;
  if (int rc = check_cache(op, cache, dtype, sequences, p.cache)) return rc;
  if (int rc = check_scale(op, scale)) return rc;
  if (sequences == 0) return 0;
  if (int rc = check_rows(op, "q", q, p.q)) return rc;
  if (!out || !lse || !aligned(out, 16)) return fail("%s: out and lse must not be null and out be 16-byte aligned", op);
  if (cache->table_width * cache->page_size > kMaxTokens)   // (a key's number and a sequence's tiles are counted in 32 bits)
    return fail("%s: the page table must have room for at most 2^30 keys per sequence (%lld pages of %lld)", op, (long long)cache->table_width,
                (long long)cache->page_size);
  const int64_t blocks = sequences * Hkv * ((Hq / Hkv + 15) / 16);
  if (blocks * (cache->table_width * cache->page_size / 32 + 1) >= (int64_t(1) << 31))
    return fail("%s: the page tables have room for too many keys (at most 2^31 tiles of 32, over sequences and KV heads)", op);
  // keys without a page are read from page 0, and what they give is dropped: there has to be one
  if (cache->pages == 0) return fail("%s: the cache must hold at least one page", op);
  const size_t need = mslk_amd_attention_decode_workspace_bytes(sequences, Hq, Hkv, D, cache->table_width, cache->page_size);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail("%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", op, need, workspace ? workspace_bytes : (size_t)0);
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.partial = (float*)workspace;
  p.sequences = (int)sequences;
  p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.D = (int)D; p.dtype = dtype;
  p.fp8 = cache->dtype == MSLK_AMD_DTYPE_E4M3FN;
  p.scale = scale;
  return check_hip(launch_attention_decode(p, (hipStream_t)stream), "attention_decode launch");
}

int mslk_amd_attention_prompt(const mslk_amd_heads* q, const mslk_amd_heads* k, const mslk_amd_heads* v, int dtype, int64_t tokens,
                              int64_t keys, int64_t Hq, int64_t Hkv, int64_t D, const int32_t* cu_seqlens,
                              const int32_t* cu_seqlens_k, int64_t sequences, int causal, float scale, void* out, float* lse,
                              void* stream) {
  const char* op = "attention_prompt";
  PromptArgs p{};
  if (int rc = check_heads(op, dtype, tokens, Hq, Hkv, D)) return rc;
  if (keys < 0 || keys >= kMaxTokens) return fail("%s: token counts must be in [0, 2^30) (got %lld)", op, (long long)keys);
  if (sequences < 0 || sequences >= kMaxTokens) return fail("%s: sequences out of range (got %lld)", op, (long long)sequences);
  if (cu_seqlens_k == nullptr && keys != tokens) return fail("%s: without cu_seqlens_k there are as many keys as queries (%lld, %lld)", op, (long long)keys, (long long)tokens);
  if (int rc = check_scale(op, scale)) return rc;
  if (tokens == 0) return 0;
  if (!cu_seqlens) return fail("%s: null pointer (cu_seqlens)", op);
  if (int rc = check_rows(op, "q", q, p.q)) return rc;
  if (keys > 0) {
    if (int rc = check_rows(op, "k", k, p.k)) return rc;
    if (int rc = check_rows(op, "v", v, p.v)) return rc;
    // (the kernel tells rows behind the last key by their offset; the stride of a single key has no meaning)
    if (keys == 1) p.k.token_stride = p.v.token_stride = D;
    if (p.k.token_stride < D || p.v.token_stride < D) return fail("%s: rows of k and v must not overlap (token strides of at least the head dimension)", op);
  }
  if (!out || !lse || !aligned(out, 16)) return fail("%s: out and lse must not be null and out be 16-byte aligned", op);
  p.out = (uint16_t*)out;
  p.lse = lse;
  p.cu_q = cu_seqlens;
  p.cu_k = cu_seqlens_k != nullptr ? cu_seqlens_k : cu_seqlens;
  p.tokens = tokens;
  p.keys = keys;
  p.sequences = (int)sequences;
  p.Hq = (int)Hq; p.Hkv = (int)Hkv; p.D = (int)D; p.dtype = dtype;
  p.causal = causal != 0;
  p.group = divider((uint32_t)(Hq / Hkv));
  p.scale = scale;
  return check_hip(launch_attention_prompt(p, (hipStream_t)stream), "attention_prompt launch");
}

int mslk_amd_quantize_mxfp4(const void* a, int a_dtype, int64_t rows, int64_t K, int64_t a_row_stride, void* codes, void* scales, void* stream) {
  const char* op = "quantize_mxfp4";
  if (a_dtype < 0 || a_dtype > 2) return fail("%s: unsupported input dtype code %d", op, a_dtype);
  if (rows < 0 || K < 0 || K > kIntMax) return fail("%s: dimension out of range", op);
  if (K % 32 != 0) return fail("%s: K must be a multiple of 32 (got %lld)", op, (long long)K);
  if (a_row_stride < 0) return fail("%s: negative row stride", op);
  if (rows == 0 || K == 0) return 0;
  if (!a || !codes || !scales) return fail("%s: null pointer", op);
  if (!aligned(codes, 4) || !aligned(a, a_dtype == MSLK_AMD_DTYPE_F32 ? 4 : 2)) return fail("%s: misaligned pointer", op);
  return check_hip(launch_quantize_mxfp4(a, a_dtype, rows, K, a_row_stride, codes, scales, (hipStream_t)stream), "quantize_mxfp4 launch");
}

int mslk_amd_dequantize_mxfp4(const void* codes, const void* scales, int64_t rows, int64_t K, void* out, int out_dtype, void* stream) {
  const char* op = "dequantize_mxfp4";
  if (out_dtype < 0 || out_dtype > 2) return fail("%s: unsupported output dtype code %d", op, out_dtype);
  if (rows < 0 || K < 0 || K > kIntMax) return fail("%s: dimension out of range", op);
  if (K % 32 != 0) return fail("%s: K must be a multiple of 32 (got %lld)", op, (long long)K);
  if (rows == 0 || K == 0) return 0;
  if (!codes || !scales || !out) return fail("%s: null pointer", op);
  if (!aligned(codes, 4) || !aligned(out, 16)) return fail("%s: misaligned pointer", op);
  return check_hip(launch_dequantize_mxfp4(codes, scales, rows, K, out, out_dtype, (hipStream_t)stream), "dequantize_mxfp4 launch");
}

size_t mslk_amd_mxfp4_mm_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int aligned) {
  if (M > kIntMax || N > kIntMax || K >= (int64_t(1) << 24)) return 0;
  return mx_workspace_bytes(M, N, K, gated, 1, false, aligned != 0);
}

int mslk_amd_mxfp4_mm(const void* xq, const void* wq, const void* x_scale, const void* w_scale, const void* bias, int bias_dtype, int gated,
                      void* y, int y_dtype, int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = gated ? "mxfp4_gated_mm" : "mxfp4_mm";
  const bool scales_aligned = aligned(x_scale, 16) && aligned(w_scale, 16);
  if (int rc = check_mx(op, xq, wq, x_scale, w_scale, y, y_dtype, M, N, K, gated, 1, workspace, workspace_bytes,
                        mslk_amd_mxfp4_mm_workspace_bytes(M, N, K, gated, scales_aligned)))
    return rc;
  if (bias_dtype < 0 || bias_dtype > 2) return fail("%s: bad bias dtype code %d", op, bias_dtype);
  if ((bias_dtype != 0) != (bias != nullptr)) return fail("%s: bias pointer and bias dtype disagree", op);
  if (gated && bias) return fail("%s: a gated product takes no bias", op);
  if (M == 0 || N == 0) return 0;
  MxProblem p{};
  p.xq = (const uint8_t*)xq; p.wq = (const uint8_t*)wq; p.xs.data = (const uint8_t*)x_scale; p.ws.data = (const uint8_t*)w_scale;
  p.bias = bias; p.bias_dtype = bias_dtype; p.y = (uint16_t*)y; p.out_f16 = y_dtype == MSLK_AMD_DTYPE_F16;
  p.M = (int)M; p.N = (int)N; p.K = (int)K; p.gated = gated != 0;
  return check_hip(launch_mx_mm(p, workspace, scales_aligned, (hipStream_t)stream), op);
}

size_t mslk_amd_mxfp4_grouped_mm_workspace_bytes(int G, int64_t total_M, int64_t N, int64_t K, int gated, int aligned) {
  if (total_M > kIntMax || N > kIntMax || K >= (int64_t(1) << 24) || G <= 0) return 0;
  return mx_workspace_bytes(total_M, N, K, gated, G, true, aligned != 0);
}

int mslk_amd_mxfp4_grouped_mm(const void* xq, const void* wq, const void* x_scale, const void* w_scale, const int64_t* m_sizes_dev, int G, int gated,
                              void* y, int y_dtype, int64_t total_M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "mxfp4_grouped_mm";
  const bool scales_aligned = aligned(x_scale, 16) && aligned(w_scale, 16);
  if (int rc = check_mx(op, xq, wq, x_scale, w_scale, y, y_dtype, total_M, N, K, gated, G, workspace, workspace_bytes,
                        mslk_amd_mxfp4_grouped_mm_workspace_bytes(G, total_M, N, K, gated, scales_aligned)))
    return rc;
  if (total_M == 0 || N == 0 || G == 0) return 0;
  if (!m_sizes_dev) return fail("%s: null pointer", op);
  MxProblem p{};
  p.xq = (const uint8_t*)xq; p.wq = (const uint8_t*)wq; p.xs.data = (const uint8_t*)x_scale; p.ws.data = (const uint8_t*)w_scale;
  p.y = (uint16_t*)y; p.out_f16 = y_dtype == MSLK_AMD_DTYPE_F16;
  p.M = (int)total_M; p.N = (int)N; p.K = (int)K; p.gated = gated != 0; p.G = G; p.m_sizes = m_sizes_dev;
  return check_hip(launch_mx_mm(p, workspace, scales_aligned, (hipStream_t)stream), op);
}

int mslk_amd_debug_cast_e4m3fn(const float* in, int64_t n, void* out, void* stream) {
  if (n < 0) return fail("debug_cast_e4m3fn: negative count");
  if (n == 0) return 0;
  if (!in || !out) return fail("debug_cast_e4m3fn: null pointer");
  return check_hip(launch_cast_e4m3fn(in, n, out, (hipStream_t)stream), "cast launch");
}

const char* mslk_amd_debug_dispatch_name(int64_t M, int64_t N, int64_t K, int bias_dtype, int y_dtype, int preshuffled,
                                         int with_workspace) {
  // Aligned stand-in pointers: the dry run dereferences nothing and launches nothing.
  void* const fake = reinterpret_cast<void*>(uintptr_t(1) << 20);
  thread_local char result[600];
  const size_t wbytes = with_workspace ? mslk_amd_f8f8bf16_rowwise_workspace_bytes(M, N, K) : 0;
  dispatch_probe_begin();
  const int rc = rowwise_impl("debug_dispatch_name", y_dtype == MSLK_AMD_DTYPE_F16, preshuffled, fake, fake, (const float*)fake,
                              (const float*)fake, bias_dtype ? fake : nullptr, bias_dtype, fake, M, N, K, wbytes ? fake : nullptr,
                              wbytes, nullptr);
  const char* text = dispatch_probe_end();
  if (rc != 0) snprintf(result, sizeof(result), "error: %s", g_err);
  else snprintf(result, sizeof(result), "%s", text[0] ? text : "nothing to launch");
  return result;
}

const char* mslk_amd_debug_grouped_dispatch_name(int layout, int G, int64_t M, int64_t N, int64_t K) {
  void* const fake = reinterpret_cast<void*>(uintptr_t(1) << 20);
  const float* const scale = static_cast<const float*>(fake);
  thread_local char result[600];
  dispatch_probe_begin();
  int rc;
  if (layout == 0)
    rc = mslk_amd_f8f8bf16_rowwise_grouped_stacked(fake, fake, scale, scale, static_cast<const int64_t*>(fake), G, M, N, K, fake, nullptr);
  else
    rc = mslk_amd_f8f8bf16_rowwise_grouped_mm(fake, fake, scale, scale, layout == MSLK_AMD_GROUPS_UNIFORM ? nullptr : static_cast<const int32_t*>(fake),
                                              layout, G, M, N, K, fake, nullptr);
  const char* text = dispatch_probe_end();
  if (rc != 0) snprintf(result, sizeof(result), "error: %s", g_err);
  else snprintf(result, sizeof(result), "%s", text[0] ? text : "nothing to launch");
  return result;
}

const char* mslk_amd_debug_grouped_list_dispatch_name(int G, const int64_t* M, const int64_t* N, const int64_t* K) {
  void* const fake = reinterpret_cast<void*>(uintptr_t(1) << 20);
  thread_local char result[600];
  constexpr int kMost = 256;
  if (G > kMost) return "error: more than 256 groups";
  const void* operands[kMost];
  const float* scales[kMost];
  void* outputs[kMost];
  for (int g = 0; g < G; ++g) {
    operands[g] = outputs[g] = fake;
    scales[g] = static_cast<const float*>(fake);
  }
  dispatch_probe_begin();
  const int rc = mslk_amd_f8f8bf16_rowwise_grouped(G, operands, operands, scales, scales, outputs, M, N, K, nullptr);
  const char* text = dispatch_probe_end();
  if (rc != 0) snprintf(result, sizeof(result), "error: %s", g_err);
  else snprintf(result, sizeof(result), "%s", text[0] ? text : "nothing to launch");
  return result;
}

const char* mslk_amd_debug_mxfp4_dispatch_name(int64_t M, int64_t N, int64_t K, int gated, int groups, int aligned_scales) {
  void* const fake = reinterpret_cast<void*>(uintptr_t(1) << 20);
  const void* const scales = static_cast<const char*>(fake) + (aligned_scales ? 0 : 1);
  thread_local char result[600];
  const size_t room = ~size_t(0);
  dispatch_probe_begin();
  const int rc = groups != 0 ? mslk_amd_mxfp4_grouped_mm(fake, fake, scales, scales, static_cast<const int64_t*>(fake), groups, gated, fake, MSLK_AMD_DTYPE_BF16,
                                                         M, N, K, fake, room, nullptr)
                             : mslk_amd_mxfp4_mm(fake, fake, scales, scales, nullptr, 0, gated, fake, MSLK_AMD_DTYPE_BF16, M, N, K, fake, room, nullptr);
  const char* text = dispatch_probe_end();
  if (rc != 0) snprintf(result, sizeof(result), "error: %s", g_err);
  else snprintf(result, sizeof(result), "%s", text[0] ? text : "nothing to launch");
  return result;
}

int mslk_amd_debug_row_walk(int tiles, int wgs, int worker, int pass, int* piece, int* pieces) {
  if (tiles < 0 || tiles > (1 << 28) || wgs <= 0 || wgs > 1024 || worker < 0 || worker >= 2 * wgs || pass < 0 || pass > (1 << 20) || !piece || !pieces) return -2;
  return debug_row_walk(tiles, wgs, worker, pass, piece, pieces);
}

int mslk_amd_debug_stream_read(const void* src, int64_t bytes, int mode, int workgroups, void* sink, void* stream) {
  if (mode < 0 || mode > 2) return fail("debug_stream_read: mode must be 0 (register loads), 1 (LDS DMA loads) or 2 (non-temporal LDS DMA loads)");
  if (bytes < 0 || bytes % (mode == 0 ? 16 : 1024) != 0) return fail("debug_stream_read: bytes must be a non-negative multiple of %d", mode == 0 ? 16 : 1024);
  if (workgroups <= 0 || workgroups > 65536) return fail("debug_stream_read: workgroups must be in 1 .. 65536");
  if (bytes == 0) return 0;
  if (!src || reinterpret_cast<uintptr_t>(src) % 16 != 0) return fail("debug_stream_read: src must be a 16-byte aligned device pointer");
  return check_hip(launch_debug_stream_read(src, bytes, mode, workgroups, sink, (hipStream_t)stream), "stream read launch");
}

int mslk_amd_debug_mfma_loop(const void* operands, int form, int iters, int workgroups, void* sink, void* stream) {
  if (form < 0 || form > 3) return fail("debug_mfma_loop: form must be 0 (16x16x128) or 1 (32x32x64), of e2m1 codes 2 or 3");
  if (iters < 0 || iters > (1 << 20)) return fail("debug_mfma_loop: iters must be in 0 .. 2^20");
  if (workgroups <= 0 || workgroups > 65536) return fail("debug_mfma_loop: workgroups must be in 1 .. 65536");
  if (!operands || reinterpret_cast<uintptr_t>(operands) % 32 != 0) return fail("debug_mfma_loop: operands must be a 32-byte aligned device pointer to 128 KiB");
  return check_hip(launch_debug_mfma_loop(operands, form, iters, workgroups, sink, (hipStream_t)stream), "mfma loop launch");
}

int mslk_amd_debug_tile_streams(const void* x, int64_t x_bytes, const void* w, int64_t w_bytes, int64_t K, int tiles_m, int tiles_n,
                                int which, void* stream) {
  if (which < 1 || which > 3) return fail("debug_tile_streams: which must be 1 (activations), 2 (weights) or 3 (both)");
  if (K < 128 || K % 128 != 0 || K > (1 << 20)) return fail("debug_tile_streams: K must be a multiple of 128 in 128 .. 2^20, got %lld", (long long)K);
  if (tiles_m <= 0 || tiles_n <= 0 || (int64_t)tiles_m * tiles_n > (1 << 20)) return fail("debug_tile_streams: tiles_m * tiles_n must be in 1 .. 2^20");
  if (x_bytes < (int64_t)tiles_m * 128 * K || w_bytes < (int64_t)tiles_n * 64 * K)
    return fail("debug_tile_streams: x must hold tiles_m * 128 rows of K bytes and w tiles_n * 64 rows");
  if (!x || !w || reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(w) % 16 != 0)
    return fail("debug_tile_streams: x and w must be 16-byte aligned device pointers");
  return check_hip(launch_debug_tile_streams(x, w, (int)K, tiles_m, tiles_n, which, (hipStream_t)stream), "tile streams launch");
}

int mslk_amd_debug_gemm_phases(const void* xq, const void* wq, const float* x_scale, const float* w_scale, void* y, int64_t M,
                               int64_t N, int64_t K, uint64_t* stamps, void* stream) {
  if (M <= 0 || N <= 0 || M % 256 != 0 || N % 256 != 0 || M > (1 << 20) || N > (1 << 20))
    return fail("debug_gemm_phases: M and N must be positive multiples of 256 (interior tiles only), got M=%lld N=%lld", (long long)M, (long long)N);
  if (K < 256 || K % 128 != 0 || K > (1 << 24)) return fail("debug_gemm_phases: K must be a multiple of 128, at least 256, got %lld", (long long)K);
  if ((M / 256) * (N / 256) > (1 << 20)) return fail("debug_gemm_phases: more than 2^20 tiles");
  if (!xq || !wq || !x_scale || !w_scale || !y || !stamps) return fail("debug_gemm_phases: null pointer");
  if (reinterpret_cast<uintptr_t>(xq) % 16 || reinterpret_cast<uintptr_t>(wq) % 16 || reinterpret_cast<uintptr_t>(y) % 16 ||
      reinterpret_cast<uintptr_t>(w_scale) % 16 || reinterpret_cast<uintptr_t>(stamps) % 8)
    return fail("debug_gemm_phases: operands, output and w_scale must be 16-byte aligned, stamps 8-byte aligned");
  GemmProblem p{(const uint8_t*)xq, (const uint8_t*)wq, x_scale, w_scale, nullptr, (uint16_t*)y, (int)M, (int)N, (int)K, 0, 0, 0};
  return check_hip(launch_debug_gemm_phases(p, stamps, (hipStream_t)stream), "gemm phases launch");
}

}  // extern "C"
