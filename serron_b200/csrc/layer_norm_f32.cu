// Register kernels of layer norm and the join for float, in a translation unit of their own
// so that they compile in parallel.
#include "layer_norm_launch.cuh"

namespace serron {

template cudaError_t norm_launch<float>(const NormPlan&, bool, int, const NormArgs<float>&, cudaStream_t);

}  // namespace serron
