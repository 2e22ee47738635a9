// Launches of the register kernels of layer_norm_fast.cuh for one storage type.
#pragma once

#include "layer_norm_fast.cuh"
#include "layer_plan.h"

namespace serron {

template <typename T>
cudaError_t launch_norm(void (*kernel)(NormArgs<T>), const NormPlan& p, bool backward, const NormArgs<T>& args,
                        cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(p.blocks), p.clusters);
    config.blockDim = dim3(p.tx, p.ty);
    config.dynamicSmemBytes = sizeof(float) * plan_shared_floats(p, backward);
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

// The kernel for `join` of the three.
template <typename T>
auto of_join(int join, void (*none)(NormArgs<T>), void (*host)(NormArgs<T>), void (*any)(NormArgs<T>)) {
    return join == kNoJoin ? none : join == kHostSeed ? host : any;
}

template <typename T, int V, int NV, int R, bool SHIFTED>
cudaError_t launch_rows(const NormPlan& p, bool backward, int join, const NormArgs<T>& args, cudaStream_t stream) {
    if (!backward) {
        auto kernel = of_join<T>(join, norm_rows_kernel<T, V, NV, R, kNoJoin, SHIFTED>,
                                 norm_rows_kernel<T, V, NV, R, kHostSeed, SHIFTED>,
                                 norm_rows_kernel<T, V, NV, R, kAnySeed, SHIFTED>);
        return launch_norm<T>(kernel, p, false, args, stream);
    }
    if constexpr (NV * V <= 16) {
        auto kernel = of_join<T>(join, norm_rows_bwd_kernel<T, V, NV, R, kNoJoin, SHIFTED>,
                                 norm_rows_bwd_kernel<T, V, NV, R, kHostSeed, SHIFTED>,
                                 norm_rows_bwd_kernel<T, V, NV, R, kAnySeed, SHIFTED>);
        return launch_norm<T>(kernel, p, true, args, stream);
    }
    return cudaErrorInvalidConfiguration;
}

template <typename T, int V, int NV, bool FULL>
cudaError_t launch_columns(const NormPlan& p, bool backward, int join, const NormArgs<T>& args, cudaStream_t stream) {
    if (!backward) {
        auto kernel = of_join<T>(join, norm_columns_kernel<T, V, NV, kNoJoin, FULL>,
                                 norm_columns_kernel<T, V, NV, kHostSeed, FULL>,
                                 norm_columns_kernel<T, V, NV, kAnySeed, FULL>);
        return launch_norm<T>(kernel, p, false, args, stream);
    }
    if constexpr (NV * V * sizeof(T) <= 64) {
        auto kernel = join == kNoJoin ? norm_columns_bwd_kernel<T, V, NV, kNoJoin, FULL>
                                      : norm_columns_bwd_kernel<T, V, NV, kAnySeed, FULL>;
        return launch_norm<T>(kernel, p, true, args, stream);
    }
    return cudaErrorInvalidConfiguration;
}

// The kernel of plan `p`; the cases are those of plan_rows and plan_columns.
template <typename T>
cudaError_t norm_launch(const NormPlan& p, bool backward, int join, const NormArgs<T>& args, cudaStream_t stream) {
    constexpr int W = 16 / sizeof(T);
#define SERRON_ROWS_CASE(v, nv, r, off) \
    if (p.V == v && p.NV == nv && p.R == r && p.shifted == off) \
        return launch_rows<T, v, nv, r, off>(p, backward, join, args, stream);
#define SERRON_COLUMNS_CASE(v, nv, whole) \
    if (p.V == v && p.NV == nv && p.full == whole) \
        return launch_columns<T, v, nv, whole>(p, backward, join, args, stream);
    if (p.rows) {
        SERRON_ROWS_CASE(W, 1, 4, false)
        SERRON_ROWS_CASE(W, 1, 1, false)
        SERRON_ROWS_CASE(W, 2, 2, false)
        SERRON_ROWS_CASE(W, 2, 1, false)
        SERRON_ROWS_CASE(W, 4, 1, false)
        SERRON_ROWS_CASE(W, 1, 4, true)
        SERRON_ROWS_CASE(W, 1, 1, true)
        SERRON_ROWS_CASE(W, 2, 2, true)
        SERRON_ROWS_CASE(W, 2, 1, true)
        SERRON_ROWS_CASE(W, 4, 1, true)
        SERRON_ROWS_CASE(1, 4, 4, false)
        SERRON_ROWS_CASE(1, 4, 1, false)
        SERRON_ROWS_CASE(1, 16, 1, false)
    } else {
        SERRON_COLUMNS_CASE(4, 4, true)
        SERRON_COLUMNS_CASE(4, 4, false)
        SERRON_COLUMNS_CASE(4, 8, true)
        SERRON_COLUMNS_CASE(4, 8, false)
        if constexpr (sizeof(T) == 2) {
            SERRON_COLUMNS_CASE(4, 16, true)
            SERRON_COLUMNS_CASE(4, 16, false)
        }
        SERRON_COLUMNS_CASE(1, 8, false)
        SERRON_COLUMNS_CASE(1, 16, false)
    }
#undef SERRON_ROWS_CASE
#undef SERRON_COLUMNS_CASE
    return cudaErrorInvalidConfiguration;
}

}  // namespace serron
