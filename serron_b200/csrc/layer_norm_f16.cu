// Register kernels of layer norm and the join for __half, in a translation unit of their own
// so that they compile in parallel.
#include "layer_norm_launch.cuh"

namespace serron {

template cudaError_t norm_launch<__half>(const NormPlan&, bool, int, const NormArgs<__half>&, cudaStream_t);

}  // namespace serron
