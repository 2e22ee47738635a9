// Register kernels of layer norm and the join for __nv_bfloat16, in a translation unit of their own
// so that they compile in parallel.
#include "layer_norm_launch.cuh"

namespace serron {

template cudaError_t norm_launch<__nv_bfloat16>(const NormPlan&, bool, int, const NormArgs<__nv_bfloat16>&, cudaStream_t);

}  // namespace serron
