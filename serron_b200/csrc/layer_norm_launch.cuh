// Launches of the register kernels of layer_norm_fast.cuh for one storage type.
#pragma once

#include "layer_norm_fast.cuh"
#include "layer_plan.h"

namespace serron {

template <typename T>
cudaError_t launch_norm(void (*kernel)(NormArgs<T>), const NormPlan& p, size_t shared, const NormArgs<T>& args,
                        cudaStream_t stream) {
    if (shared > 48 * 1024) {
        const cudaError_t err =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
        if (err != cudaSuccess) return err;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(p.blocks), p.clusters);
    config.blockDim = dim3(p.tx, p.ty);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 1;
    attribute.val.clusterDim.y = p.clusters;
    attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = p.clusters > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args);
}

template <typename T, int V, int NV>
cudaError_t launch_rows(const NormPlan& p, bool backward, bool join, const NormArgs<T>& args, cudaStream_t stream) {
    if (!backward)
        return launch_norm<T>(join ? norm_rows_kernel<T, V, NV, true> : norm_rows_kernel<T, V, NV, false>, p, 0, args,
                              stream);
    const size_t floats = p.ty > 1 ? size_t(NV) * V * p.tx * p.ty : 0;
    return launch_norm<T>(join ? norm_rows_bwd_kernel<T, V, NV, true> : norm_rows_bwd_kernel<T, V, NV, false>, p,
                          sizeof(float) * floats, args, stream);
}

template <typename T, int V, int NV>
cudaError_t launch_columns(const NormPlan& p, bool backward, bool join, const NormArgs<T>& args, cudaStream_t stream) {
    // a tile's partial results: two per row and group, and two per row for the cluster
    const size_t floats = (p.ty > 1 || p.clusters > 1) ? (2 * size_t(p.ty) + 2) * p.tx * V : 0;
    if (!backward)
        return launch_norm<T>(join ? norm_columns_kernel<T, V, NV, true> : norm_columns_kernel<T, V, NV, false>, p,
                              sizeof(float) * floats, args, stream);
    // two tiles' of them; at the end two sums per channel and warp
    const size_t most = std::max(2 * floats, size_t(NV) * p.ty * (p.tx / 32) * 2);
    return launch_norm<T>(join ? norm_columns_bwd_kernel<T, V, NV, true> : norm_columns_bwd_kernel<T, V, NV, false>, p,
                          sizeof(float) * most, args, stream);
}

// The kernel of plan `p`; the cases are those of round_vectors.
template <typename T>
cudaError_t norm_launch(const NormPlan& p, bool backward, bool join, const NormArgs<T>& args, cudaStream_t stream) {
    constexpr int W = 16 / sizeof(T);
#define SERRON_NORM_CASE(layout, v, nv) \
    if (p.V == v && p.NV == nv) return launch_##layout<T, v, nv>(p, backward, join, args, stream);
    if (p.rows) {
        SERRON_NORM_CASE(rows, W, 1)
        SERRON_NORM_CASE(rows, W, 2)
        SERRON_NORM_CASE(rows, W, 4)
        if constexpr (W == 8) {
            SERRON_NORM_CASE(rows, 2, 2)
            SERRON_NORM_CASE(rows, 2, 8)
        }
        SERRON_NORM_CASE(rows, 1, 4)
        SERRON_NORM_CASE(rows, 1, 16)
    } else {
        SERRON_NORM_CASE(columns, 4, 4)
        SERRON_NORM_CASE(columns, 4, 8)
        SERRON_NORM_CASE(columns, 1, 8)
        SERRON_NORM_CASE(columns, 1, 16)
    }
#undef SERRON_NORM_CASE
    return cudaErrorInvalidConfiguration;
}

}  // namespace serron
