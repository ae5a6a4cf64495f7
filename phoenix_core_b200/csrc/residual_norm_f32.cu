#include "residual_norm.cuh"

namespace pcb {
int norm_fwd_f32(const RNParams& p, cudaStream_t stream) { return fwd_typed<float, 4>(p, stream); }
int norm_bwd_f32(const RNParams& p, const RNPlan& plan, cudaStream_t stream) { return bwd_typed<float, 4>(p, plan, stream); }
}  // namespace pcb
