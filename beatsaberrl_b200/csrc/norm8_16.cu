// LayerNorm with its input kept in 8 bits: 16-bit rows (norm8.cuh), and the sum of the blocks' partial parameter gradients.
#include <algorithm>

#include "norm8.cuh"

namespace bsrl {
namespace norm8 {
template <>
int fwd(const FwdArgs<__half, __half>& p, bool aligned, cudaStream_t stream) { return launch_fwd(p, aligned, stream); }
template <>
int fwd(const FwdArgs<__nv_bfloat16, __nv_bfloat16>& p, bool aligned, cudaStream_t stream) { return launch_fwd(p, aligned, stream); }
template <>
int bwd(const BwdArgs<__half, __half>& p, bool aligned, cudaStream_t stream) { return launch_bwd(p, aligned, stream); }
template <>
int bwd(const BwdArgs<__nv_bfloat16, __nv_bfloat16>& p, bool aligned, cudaStream_t stream) { return launch_bwd(p, aligned, stream); }

namespace {
// out = sum over parts (n_parts, cols), in order: a block takes 32 columns, its 32 warps every 32nd part each, then the warps' sums one
// after the other.  The first d columns go to a, the others to b.
__global__ void __launch_bounds__(1024) add_parts_kernel(const float* __restrict__ parts, int n_parts, int d, float* a, float* b) {
  pdl_begin();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane, cols = 2 * d;
  float sum = 0.f;
  if (col < cols) {
#pragma unroll 8
    for (int p = warp; p < n_parts; p += 32) sum += parts[(int64_t)p * cols + col];
  }
  s[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && col < cols) {
#pragma unroll
    for (int w = 1; w < 32; ++w) sum += s[w][lane];
    if (col < d) {
      if (a) a[col] = sum;
    } else if (b) {
      b[col - d] = sum;
    }
  }
}
}  // namespace
}  // namespace norm8

namespace {
using namespace norm8;
// whether every row of every operand starts on a whole piece: 16 bytes, fp32 32
struct Rows {
  const void* base;
  int64_t ld;
  int size;
};
bool on_pieces(int d, std::initializer_list<Rows> all) {
  if (d % 8) return false;
  for (const Rows& r : all)
    if (r.base && (reinterpret_cast<uintptr_t>(r.base) % (8 * r.size) || r.ld % 8)) return false;
  return true;
}
template <typename T, typename TY>
int run_fwd(const Norm8Args& a, cudaStream_t stream) {
  const FwdArgs<T, TY> p{static_cast<const T*>(a.x), static_cast<const T*>(a.residual), static_cast<T*>(a.z), static_cast<TY*>(a.y), a.gamma, a.beta,
                         a.codes, a.exps, a.mean, a.rstd, a.rows, a.ldx, a.ldr, a.ldz, a.ldy, a.d, a.kind, a.eps};
  const bool aligned = on_pieces(a.d, {{a.x, a.ldx, sizeof(T)}, {a.residual, a.ldr, sizeof(T)}, {a.z, a.ldz, sizeof(T)}, {a.y, a.ldy, sizeof(TY)}, {a.gamma, 8, 4}, {a.beta, 8, 4}});
  return fwd<T, TY>(p, aligned, stream);
}
bool bwd_on_pieces(const Norm8BwdArgs& a) {
  const int t = a.dtype == BSRL_F32 ? 4 : 2, ty = a.gy_dtype == BSRL_F32 ? 4 : 2;
  return on_pieces(a.d, {{a.gy, a.ldgy, ty}, {a.g_residual, a.ldgr, t}, {a.gx, a.ldgx, t}, {a.gamma, 8, 4}});
}
template <typename T, typename TY>
int run_bwd(const Norm8BwdArgs& a, bool aligned, float* parts, cudaStream_t stream) {
  const BwdArgs<T, TY> p{static_cast<const TY*>(a.gy), static_cast<const T*>(a.g_residual), static_cast<T*>(a.gx), a.gamma, a.codes, a.exps,
                         a.mean, a.rstd, a.g_gamma, a.g_beta, parts, a.rows, a.ldgy, a.ldgr, a.ldgx, a.d, a.kind};
  return bwd<T, TY>(p, aligned, stream);
}
}  // namespace

bool norm8_types_ok(int dtype, int y_dtype) {
  return dtype == BSRL_F32 ? y_dtype == BSRL_F32 || y_dtype == BSRL_F16 || y_dtype == BSRL_BF16
                           : (dtype == BSRL_F16 || dtype == BSRL_BF16) && y_dtype == dtype;
}
int norm8_max_width() { return kMaxWidth; }

int norm8_fwd(const Norm8Args& a, cudaStream_t stream) {
  if (a.dtype == BSRL_F16) return run_fwd<__half, __half>(a, stream);
  if (a.dtype == BSRL_BF16) return run_fwd<__nv_bfloat16, __nv_bfloat16>(a, stream);
  if (a.y_dtype == BSRL_F16) return run_fwd<float, __half>(a, stream);
  if (a.y_dtype == BSRL_BF16) return run_fwd<float, __nv_bfloat16>(a, stream);
  return run_fwd<float, float>(a, stream);
}

int64_t norm8_bwd_workspace(int64_t rows, int d) {
  int blocks = 0;                                  // the more of aligned and unaligned rows
  for (const bool aligned : {true, false}) blocks = std::max(blocks, blocks_of(shape_of(d, aligned, true), rows, true));
  return blocks > 1 ? (int64_t)blocks * 2 * d * (int64_t)sizeof(float) : 0;
}
int norm8_bwd(const Norm8BwdArgs& a, float* workspace, cudaStream_t stream) {
  const bool aligned = bwd_on_pieces(a);
  const int blocks = blocks_of(shape_of(a.d, aligned, true), a.rows, true);
  float* parts = blocks > 1 && (a.g_gamma || a.g_beta) ? workspace : nullptr;
  int rc;
  if (a.dtype == BSRL_F16) rc = run_bwd<__half, __half>(a, aligned, parts, stream);
  else if (a.dtype == BSRL_BF16) rc = run_bwd<__nv_bfloat16, __nv_bfloat16>(a, aligned, parts, stream);
  else if (a.gy_dtype == BSRL_F16) rc = run_bwd<float, __half>(a, aligned, parts, stream);
  else if (a.gy_dtype == BSRL_BF16) rc = run_bwd<float, __nv_bfloat16>(a, aligned, parts, stream);
  else rc = run_bwd<float, float>(a, aligned, parts, stream);
  if (rc != BSRL_OK || !parts) return rc;
  PdlScope overlap;
  pdl_enable();
  launch_kernel(add_parts_kernel, (unsigned)((2 * a.d + 31) / 32), 1024, 0, stream, static_cast<const float*>(parts), blocks, a.d, a.g_gamma, a.g_beta);
  BSRL_LAUNCH_OK("add_parts_kernel");
  return BSRL_OK;
}

}  // namespace bsrl
