// LayerNorm with its input kept in 8 bits: fp32 rows (norm8.cuh).
#include "norm8.cuh"

namespace bsrl {
namespace norm8 {
template <>
int fwd(const FwdArgs<float, float>& p, bool aligned, cudaStream_t stream) { return launch_fwd(p, aligned, stream); }
template <>
int fwd(const FwdArgs<float, __half>& p, bool aligned, cudaStream_t stream) { return launch_fwd(p, aligned, stream); }
template <>
int fwd(const FwdArgs<float, __nv_bfloat16>& p, bool aligned, cudaStream_t stream) { return launch_fwd(p, aligned, stream); }
template <>
int bwd(const BwdArgs<float, float>& p, bool aligned, cudaStream_t stream) { return launch_bwd(p, aligned, stream); }
template <>
int bwd(const BwdArgs<float, __half>& p, bool aligned, cudaStream_t stream) { return launch_bwd(p, aligned, stream); }
template <>
int bwd(const BwdArgs<float, __nv_bfloat16>& p, bool aligned, cudaStream_t stream) { return launch_bwd(p, aligned, stream); }
}  // namespace norm8
}  // namespace bsrl
