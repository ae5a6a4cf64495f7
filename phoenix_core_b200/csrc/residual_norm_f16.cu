#include "residual_norm.cuh"

namespace pcb {
int norm_fwd_f16(const RNParams& p, cudaStream_t stream) { return fwd_typed<__half, 8>(p, stream); }
int norm_bwd_f16(const RNParams& p, const RNPlan& plan, cudaStream_t stream) { return bwd_typed<__half, 8>(p, plan, stream); }
}  // namespace pcb
