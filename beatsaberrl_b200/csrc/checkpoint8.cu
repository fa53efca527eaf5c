// C entry points of the operators around activations kept in 8 bits (pack8.cu, norm8.cuh, wgrad8_tc5.cu): argument checks, all on the
// host and ahead of the first launch.
#include "kernels.cuh"
#include "pack8.cuh"

using namespace bsrl;

namespace {
constexpr int64_t kMaxD = ((int64_t)1 << 31) - 64;
constexpr int kMaxSide = 1 << 20;
constexpr int64_t kMaxWeight = (int64_t)1 << 31;       // elements: keeps the numbers of tiles and work items in 32 bits

int refuse(int status, const char* what, const char* why) {
  set_error("%s: %s", what, why);
  return status;
}
bool float_type(int dtype) { return dtype == BSRL_F32 || dtype == BSRL_F16 || dtype == BSRL_BF16; }
int size_of(int dtype) { return dtype == BSRL_F32 ? 4 : 2; }
bool aligned_to(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// a (rows, d) matrix: its type, pitch and first element's alignment; addresses stay within 2^62 bytes
int check_rows(const char* what, const void* p, int dtype, int64_t ld, int64_t rows, int64_t d) {
  if (!float_type(dtype)) return refuse(BSRL_ERR_UNSUPPORTED, what, "elements must be f32, f16 or bf16");
  if (rows < 0 || rows > (int64_t)1 << 40 || d < 1 || d > kMaxD) return refuse(BSRL_ERR_SHAPE, what, "rows must be 0 .. 2^40, the width 1 .. 2^31 - 64");
  if (ld < d || ld > (int64_t)1 << 48 || (rows > 1 && ld > ((int64_t)1 << 60) / rows)) return refuse(BSRL_ERR_SHAPE, what, "a row pitch is smaller than the width, or too large");
  if (!p && rows > 0) return refuse(BSRL_ERR_NULL, what, "NULL operand");
  if (!aligned_to(p, size_of(dtype))) return refuse(BSRL_ERR_ALIGN, what, "an operand is not aligned to its elements");
  return BSRL_OK;
}
int check_kept(const char* what, const uint8_t* codes, const uint8_t* exps, int kind, int64_t rows) {
  if (kind != BSRL_INT8 && kind != BSRL_E4M3) return refuse(BSRL_ERR_UNSUPPORTED, what, "the kind must be BSRL_INT8 or BSRL_E4M3");
  if (rows > 0 && (!codes || !exps)) return refuse(BSRL_ERR_NULL, what, "NULL codes or exps");
  if (!aligned16(codes) || !aligned_to(exps, 4)) return refuse(BSRL_ERR_ALIGN, what, "codes must be 16-byte, exps 4-byte aligned");
  return BSRL_OK;
}
cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

#define CHECK(expr)                 \
  do {                              \
    const int rc__ = (expr);        \
    if (rc__ != BSRL_OK) return rc__; \
  } while (0)
}  // namespace

extern "C" {

int64_t bsrl_pack8_pitch(int64_t d) {
  if (d < 1 || d > kMaxD) {
    set_error("pack8: the width must be 1 .. 2^31 - 64");
    return -1;
  }
  return p8::pitch_of(d);
}

int bsrl_pack8(const void* x, int32_t dtype, int64_t ldx, int64_t rows, int64_t d, int32_t kind, uint8_t* codes, uint8_t* exps, void* stream) {
  CHECK(check_rows("pack8", x, dtype, ldx, rows, d));
  CHECK(check_kept("pack8", codes, exps, kind, rows));
  return rows == 0 ? BSRL_OK : pack8(x, dtype, ldx, rows, d, kind, codes, exps, as_stream(stream));
}

int bsrl_expand8(const uint8_t* codes, const uint8_t* exps, int32_t kind, int64_t rows, int64_t d, void* out, int32_t dtype, int64_t ldo,
                 void* stream) {
  CHECK(check_rows("expand8", out, dtype, ldo, rows, d));
  CHECK(check_kept("expand8", codes, exps, kind, rows));
  return rows == 0 ? BSRL_OK : expand8(codes, exps, kind, rows, d, out, dtype, ldo, as_stream(stream));
}

int bsrl_gelu8(const void* x, int32_t dtype, int64_t ldx, int64_t rows, int64_t d, void* y, int64_t ldy, int32_t kind, uint8_t* codes,
               uint8_t* exps, void* stream) {
  CHECK(check_rows("gelu8", x, dtype, ldx, rows, d));
  CHECK(check_rows("gelu8", y, dtype, ldy, rows, d));
  CHECK(check_kept("gelu8", codes, exps, kind, rows));
  return rows == 0 ? BSRL_OK : gelu8(x, dtype, ldx, rows, d, y, ldy, kind, codes, exps, as_stream(stream));
}

int bsrl_gelu8_bwd(const void* gy, int32_t dtype, int64_t ldgy, const uint8_t* codes, const uint8_t* exps, int32_t kind, int64_t rows, int64_t d,
                   void* gx, int64_t ldgx, void* stream) {
  CHECK(check_rows("gelu8_bwd", gy, dtype, ldgy, rows, d));
  CHECK(check_rows("gelu8_bwd", gx, dtype, ldgx, rows, d));
  CHECK(check_kept("gelu8_bwd", codes, exps, kind, rows));
  return rows == 0 ? BSRL_OK : gelu8_bwd(gy, dtype, ldgy, codes, exps, kind, rows, d, gx, ldgx, as_stream(stream));
}

int bsrl_layernorm8(const void* x, const void* residual, int32_t dtype, int64_t ldx, int64_t ldr, const float* gamma, const float* beta, float eps,
                    int64_t rows, int32_t d, void* z, int64_t ldz, void* y, int32_t y_dtype, int64_t ldy, int32_t kind, uint8_t* codes,
                    uint8_t* exps, float* mean, float* rstd, void* stream) {
  const char* me = "layernorm8";
  CHECK(check_rows(me, x, dtype, ldx, rows, d));
  CHECK(check_rows(me, y, y_dtype, ldy, rows, d));
  if (residual) {
    CHECK(check_rows(me, residual, dtype, ldr, rows, d));
    CHECK(check_rows(me, z, dtype, ldz, rows, d));
  }
  CHECK(check_kept(me, codes, exps, kind, rows));
  if (d > norm8_max_width()) return refuse(BSRL_ERR_SHAPE, me, "rows are at most 8,192 wide");
  if (!norm8_types_ok(dtype, y_dtype)) return refuse(BSRL_ERR_UNSUPPORTED, me, "16-bit rows give results of their own type");
  if (!gamma || (rows > 0 && (!mean || !rstd))) return refuse(BSRL_ERR_NULL, me, "NULL gamma, mean or rstd");
  if (!aligned_to(gamma, 4) || !aligned_to(beta, 4) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return refuse(BSRL_ERR_ALIGN, me, "an fp32 operand is not aligned to its elements");
  if (rows == 0) return BSRL_OK;
  return norm8_fwd(Norm8Args{x, residual, residual ? z : nullptr, y, gamma, beta, codes, exps, mean, rstd, rows, ldx, ldr, ldz, ldy, d, kind, dtype,
                             y_dtype, eps}, as_stream(stream));
}

int64_t bsrl_layernorm8_bwd_workspace_bytes(int64_t rows, int32_t d) {
  if (rows < 0 || d < 1 || d > norm8_max_width()) {
    set_error("layernorm8_bwd: rows must not be negative, the width 1 .. 8,192");
    return -1;
  }
  return norm8_bwd_workspace(rows, d);
}

int bsrl_layernorm8_bwd(const void* gy, int32_t gy_dtype, int64_t ldgy, const void* g_residual, int64_t ldgr, const uint8_t* codes,
                        const uint8_t* exps, int32_t kind, const float* mean, const float* rstd, const float* gamma, int64_t rows, int32_t d,
                        void* gx, int32_t dtype, int64_t ldgx, float* g_gamma, float* g_beta, void* workspace, int64_t workspace_bytes,
                        void* stream) {
  const char* me = "layernorm8_bwd";
  CHECK(check_rows(me, gy, gy_dtype, ldgy, rows, d));
  CHECK(check_rows(me, gx, dtype, ldgx, rows, d));
  if (g_residual) CHECK(check_rows(me, g_residual, dtype, ldgr, rows, d));
  CHECK(check_kept(me, codes, exps, kind, rows));
  if (d > norm8_max_width()) return refuse(BSRL_ERR_SHAPE, me, "rows are at most 8,192 wide");
  if (!norm8_types_ok(dtype, gy_dtype)) return refuse(BSRL_ERR_UNSUPPORTED, me, "16-bit rows take gradients of their own type");
  if (!gamma || (rows > 0 && (!mean || !rstd))) return refuse(BSRL_ERR_NULL, me, "NULL gamma, mean or rstd");
  if (!aligned_to(gamma, 4) || !aligned_to(g_gamma, 4) || !aligned_to(g_beta, 4) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return refuse(BSRL_ERR_ALIGN, me, "an fp32 operand is not aligned to its elements");
  cudaStream_t st = as_stream(stream);
  if (rows == 0) {
    if (g_gamma) BSRL_CUDA_OK(cudaMemsetAsync(g_gamma, 0, (size_t)d * 4, st));
    if (g_beta) BSRL_CUDA_OK(cudaMemsetAsync(g_beta, 0, (size_t)d * 4, st));
    return BSRL_OK;
  }
  const int64_t need = norm8_bwd_workspace(rows, d);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) {
    set_error("%s: workspace of %lld bytes, 16-byte aligned, needed", me, (long long)need);
    return BSRL_ERR_WORKSPACE;
  }
  return norm8_bwd(Norm8BwdArgs{gy, g_residual, gx, gamma, codes, exps, mean, rstd, g_gamma, g_beta, rows, ldgy, ldgr, ldgx, d, kind, dtype, gy_dtype},
                   static_cast<float*>(workspace), st);
}

int64_t bsrl_linear8_wgrad_workspace_bytes(int64_t rows, int32_t n, int32_t k, int32_t aligned) {
  if (rows < 0 || rows > 0x7fffff00 - 1 || n < 1 || k < 1 || n > kMaxSide || k > kMaxSide || (int64_t)n * k > kMaxWeight) {
    set_error("linear8_wgrad: rows must be 0 .. 2^31 - 257, n and k 1 .. 2^20, n k at most 2^31");
    return -1;
  }
  return rows == 0 ? 0 : wgrad8_workspace(rows, n, k, aligned != 0);
}

int bsrl_linear8_wgrad_plan(int64_t rows, int32_t n, int32_t k, int32_t* plan) {
  const char* me = "linear8_wgrad_plan";
  if (rows < 1 || rows > 0x7fffff00 - 1 || n < 1 || k < 1 || n > kMaxSide || k > kMaxSide || (int64_t)n * k > kMaxWeight)
    return refuse(BSRL_ERR_SHAPE, me, "rows must be 1 .. 2^31 - 257, n and k 1 .. 2^20, n k at most 2^31");
  if (!plan) return refuse(BSRL_ERR_NULL, me, "NULL plan");
  int32_t p[3];
  wgrad8_plan(rows, n, k, p);
  for (int i = 0; i < 3; ++i) plan[i] = p[i];
  return BSRL_OK;
}

int bsrl_linear8_wgrad(const void* gy, int32_t gy_dtype, int64_t ldgy, const uint8_t* codes, const uint8_t* exps, int32_t kind, int64_t rows,
                       int32_t n, int32_t k, float* g_weight, float* g_bias, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* me = "linear8_wgrad";
  if (rows < 0 || rows > 0x7fffff00 - 1 || n < 1 || k < 1 || n > kMaxSide || k > kMaxSide || (int64_t)n * k > kMaxWeight)
    return refuse(BSRL_ERR_SHAPE, me, "rows must be 0 .. 2^31 - 257, n and k 1 .. 2^20, n k at most 2^31");
  CHECK(check_rows(me, gy, gy_dtype, ldgy, rows, n));
  CHECK(check_kept(me, codes, exps, kind, rows));
  if (gy_dtype == BSRL_F32) return refuse(BSRL_ERR_UNSUPPORTED, me, "gy must be f16 or bf16");
  if (!g_weight) return refuse(BSRL_ERR_NULL, me, "NULL g_weight");
  if (!aligned_to(g_weight, 4) || !aligned_to(g_bias, 4)) return refuse(BSRL_ERR_ALIGN, me, "an fp32 operand is not aligned to its elements");
  cudaStream_t st = as_stream(stream);
  if (rows == 0) {
    BSRL_CUDA_OK(cudaMemsetAsync(g_weight, 0, (size_t)n * k * 4, st));
    if (g_bias) BSRL_CUDA_OK(cudaMemsetAsync(g_bias, 0, (size_t)n * 4, st));
    return BSRL_OK;
  }
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255)) return refuse(BSRL_ERR_WORKSPACE, me, "a workspace, 256-byte aligned, is needed");
  return wgrad8(gy, gy_dtype, ldgy, codes, exps, kind, rows, n, k, g_weight, k, g_bias, workspace, workspace_bytes, st);
}

}  // extern "C"
