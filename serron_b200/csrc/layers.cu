// C ABI of the layer operators: layer norm, dropout and their join with a residual sum (layer_norm.cuh, dropout.cuh).
// Contracts: include/serron_b200.h.
#include "serron_b200.h"

#include <algorithm>
#include <cmath>
#include <limits>

#include "dropout.cuh"
#include "host_guard.h"
#include "layer_norm.cuh"
#include "layer_norm_fast.cuh"
#include "layer_plan.h"

namespace serron {

// the register kernels, instantiated per storage type in layer_norm_<type>.cu
template <typename T>
cudaError_t norm_launch(const NormPlan& p, bool backward, int join, const NormArgs<T>& args, cudaStream_t stream);

namespace {

int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Calls f(T{}) with the storage type of `dtype`.
template <typename F>
void with_type(int dtype, F&& f) {
    switch (dtype) {
    case kF32: f(float{}); break;
    case kF64: f(double{}); break;
    case kF16: f(__half{}); break;
    default: f(__nv_bfloat16{}); break;
    }
}

unsigned grid_of(const char* name, int64_t blocks) {
    SB_CHECK(blocks < (int64_t(1) << 31), name, ": too large (", blocks, " blocks of work)");
    return static_cast<unsigned>(blocks);
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// No kernel can read an element that lies across its own boundary.
template <typename... P>
void check_elements(const char* name, size_t size, P... pointers) {
    SB_CHECK((aligned(pointers, size) && ...), name, ": tensors must start on a boundary of their elements");
}

// ------------------------------------------------------------------------------------------------
// dropout
// ------------------------------------------------------------------------------------------------
DropRule drop_rule(const char* name, double p, uint64_t seed, const void* seed_device, uint64_t sequence) {
    SB_CHECK(p >= 0.0 && p <= 1.0, name, ": p must be between 0 and 1, got ", p);
    SB_CHECK(aligned(seed_device, sizeof(uint64_t)), name, ": a seed in device memory must be aligned to 8 bytes");
    DropRule rule;
    rule.keys.set(seed);
    rule.seed_device = static_cast<const uint64_t*>(seed_device);
    rule.sequence = sequence;
    const double threshold = std::nearbyint(p * 4294967296.0);
    rule.all = threshold >= 4294967296.0;
    rule.threshold = rule.all ? 0xffffffffu : static_cast<uint32_t>(threshold);
    rule.scale = rule.all ? 0.0 : 1.0 / (1.0 - p);
    rule.scale32 = static_cast<float>(rule.scale);
    return rule;
}

constexpr int kDropVectors = 4;  // per thread

template <typename T>
void launch_dropout(const char* name, const void* x_, const void* residual_, void* y_, int64_t n, int64_t span,
                    const DropRule& rule, cudaStream_t stream) {
    const T *x = static_cast<const T*>(x_), *residual = static_cast<const T*>(residual_);
    T* y = static_cast<T*>(y_);
    if constexpr (!std::is_same_v<T, double>) {
        constexpr int V = 16 / sizeof(T), U = kDropVectors;
        const bool wide = aligned(x, 16) && aligned(residual, 16) && aligned(y, 16);
        if (rule.all) span = n;  // one decision for everything, which the kernels of a span look up in the rule
        if (span == 1 && wide && !rule.all) {
            const unsigned blocks = grid_of(name, ceil_div64(n, 256 * U * V));
            auto kernel = rule.seed_device
                              ? (residual ? dropout_kernel<T, V, U, true, true> : dropout_kernel<T, V, U, false, true>)
                              : (residual ? dropout_kernel<T, V, U, true, false> : dropout_kernel<T, V, U, false, false>);
            kernel<<<blocks, 256, 0, stream>>>(x, residual, y, n, rule);
            SB_CUDA(cudaGetLastError());
            return;
        }
        if (wide && span >= V && (span < kLongSpan || (span % V != 0 && span < (int64_t(1) << 30)))) {
            const unsigned blocks = grid_of(name, ceil_div64(n, 256 * U * V));
            auto kernel = rule.seed_device ? (residual ? dropout_spans_kernel<T, V, U, true, true>
                                                       : dropout_spans_kernel<T, V, U, false, true>)
                                           : (residual ? dropout_spans_kernel<T, V, U, true, false>
                                                       : dropout_spans_kernel<T, V, U, false, false>);
            kernel<<<blocks, 256, 0, stream>>>(x, residual, y, n, static_cast<int>(span), rule);
            SB_CUDA(cudaGetLastError());
            return;
        }
        if (span >= 256 && n % span == 0) {
            const int64_t width = wide && span % V == 0 ? V : 1;
            const int64_t pieces = ceil_div64(span, 256 * U * width);
            const unsigned blocks = grid_of(name, n / span * pieces);
            if (width > 1)
                dropout_units_kernel<T, V, U><<<blocks, 256, 0, stream>>>(x, residual, y, span, pieces, rule);
            else
                dropout_units_kernel<T, 1, U><<<blocks, 256, 0, stream>>>(x, residual, y, span, pieces, rule);
            SB_CUDA(cudaGetLastError());
            return;
        }
    }
    dropout_any_kernel<T><<<grid_of(name, ceil_div64(n, 256)), 256, 0, stream>>>(x, residual, y, n, span, rule);
    SB_CUDA(cudaGetLastError());
}

// ------------------------------------------------------------------------------------------------
// layer norm
// ------------------------------------------------------------------------------------------------
struct Norm {
    NormShape shape;
    int chunk = 0, splits = 0;  // a row's cut into chunks
    int rows_per = 0;           // rows a partial sum of the parameters' gradients covers
    int64_t blocks = 0;         // such sums
    int64_t numel() const { return shape.rows * shape.len; }
    int64_t inner = 1;

    // The plan of the widest vectors that the sizes and `fits` (the pointers) allow; not ok where no register kernel
    // takes the call.
    template <typename F>
    NormPlan plan(int dtype, bool backward, F&& fits) const {
        for (const int* v = plan_widths(inner == 1, static_cast<int>(elem_size(dtype))); dtype != kF64 && *v; ++v) {
            if (!fits(*v)) continue;
            const NormPlan p =
                norm_plan(shape.rows, shape.len, inner, *v, static_cast<int>(elem_size(dtype)), backward);
            if (p.ok) return p;
        }
        return NormPlan();
    }
};

// Rows per first-level sum of the parameters' gradients: at most 128 additions in a row (32 per thread where a
// block's threads share a sum), so that the float32 sums stay as exact as a tree's.
constexpr int kRowsPerSum = 128, kColumnsPerSum = 32 * kNormThreads;
// Up to so many rows the gradients of weight and bias are added up straight from the tensors.
constexpr int kDirectRows = 64;

Norm norm_of(const char* name, int64_t outer, int64_t len, int64_t inner) {
    SB_CHECK(outer >= 0 && inner >= 0, name, ": sizes must be non-negative");
    SB_CHECK(len >= 1, name, ": the normalised dimension must not be empty");
    SB_CHECK(len < (int64_t(1) << 31) && inner < (int64_t(1) << 31), name,
             ": the normalised dimension and the elements behind it must be below 2^31");
    // no workspace takes more than 32 bytes an element, and 64 leave room for its alignment
    SB_CHECK(outer == 0 || inner == 0 || outer <= std::numeric_limits<int64_t>::max() / 64 / len / inner, name,
             ": too many elements");
    Norm n;
    n.shape.rows = outer * inner;
    n.shape.len = static_cast<int>(len);
    n.shape.inner = static_cast<int>(std::max<int64_t>(inner, 1));
    n.inner = n.shape.inner;
    n.chunk = static_cast<int>(std::max<int64_t>(inner == 1 ? 8192 : 1024, ceil_div64(len, 65535)));
    n.splits = static_cast<int>(ceil_div64(len, n.chunk));
    n.rows_per = inner == 1 ? kRowsPerSum : kColumnsPerSum;
    n.blocks = ceil_div64(n.shape.rows, n.rows_per);
    return n;
}

// Workspace of the kernels for any length: [partial sums of the rows' chunks][mean, rstd][partial sums of the
// parameters' gradients]; of the register kernels: the last part alone.
struct NormWorkspace {
    int64_t part = 0, stats = 0, params = 0, total = 0;
    NormWorkspace(const Norm& n, size_t acc, bool backward) {
        part = 0;
        stats = part + align256(n.shape.rows * n.splits * 2 * acc);
        params = stats + (backward ? 0 : align256(n.shape.rows * 2 * acc));
        total = params + (backward ? align256(n.blocks * 2 * n.shape.len * acc) : 0);
    }
};

// What a call may need, whatever its pointers' alignment.
int64_t workspace_bytes_of(const Norm& n, int dtype, bool backward) {
    const size_t acc = dtype == kF64 ? 8 : 4;
    bool any = false;  // whether some alignment leaves the call to the kernels for any length
    int64_t bytes = 0;
    for (int width = 1; width <= 8; width *= 2) {
        const NormPlan p = n.plan(dtype, backward, [&](int v) { return v <= width; });
        any = any || !p.ok;
        if (p.ok && backward) bytes = std::max(bytes, align256(p.blocks * 2 * n.shape.len * int64_t(sizeof(float))));
    }
    return n.numel() == 0 ? 0 : any ? std::max(bytes, NormWorkspace(n, acc, backward).total) : bytes;
}

void check_norm(const char* name, int32_t dtype, int32_t param_dtype, const void* weight, const void* bias) {
    SB_CHECK(dtype >= kF32 && dtype <= kBF16, name, ": unsupported dtype code ", dtype);
    if (weight || bias)
        SB_CHECK(param_dtype == dtype || (param_dtype == kF32 && dtype != kF64), name,
                 ": weight and bias must be float32 or have the input's dtype");
}

template <typename T>
constexpr int dtype_of = std::is_same_v<T, float>    ? kF32
                         : std::is_same_v<T, __half> ? kF16
                         : std::is_same_v<T, double> ? kF64
                                                     : kBF16;

int join_kind(bool join, const DropRule& rule) {
    return !join ? kNoJoin : rule.seed_device ? kAnySeed : kHostSeed;
}

// Every pointer on a boundary of `bytes` (null ones are).
template <typename... P>
bool fits(size_t bytes, P... pointers) {
    return (aligned(pointers, bytes) && ...);
}
// Parameters are read V at a time in their own type, float32 ones at most four at a time.
template <typename T, typename... P>
bool params_fit(int V, bool f32, P... pointers) {
    return fits(f32 ? (V >= 4 ? 16 : 4) : V * sizeof(T), pointers...);
}

template <typename T>
void param_final(const typename Storage<T>::acc* sums, int64_t blocks, int len, void* dw, void* db, bool f32,
                 cudaStream_t stream) {
    // eight partial sums or more to a share, at most 32 shares; at least a warp's width of columns
    int shares = 1;
    while (shares < 32 && blocks >= 16 * shares) shares *= 2;
    const int columns = std::max(32, 128 / shares);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(ceil_div64(2ll * len, columns)));
    config.blockDim = dim3(columns, shares);
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    SB_CUDA(cudaLaunchKernelEx(&config, norm_param_final_kernel<T>, sums, static_cast<int>(blocks), len, dw, db, f32));
}

template <typename T>
void norm_forward(const char* name, const Norm& n, const void* x_, const void* weight, const void* bias, bool f32,
                  double eps, void* y, void* mean_, void* rstd_, char* ws, cudaStream_t stream,
                  const void* residual, void* sum, const DropRule& rule) {
    using A = typename Storage<T>::acc;
    const bool join = residual != nullptr;
    if constexpr (!std::is_same_v<T, double>) {
        const NormPlan p = n.plan(dtype_of<T>, false, [&](int v) {
            return fits(v * sizeof(T), x_, residual, sum, y) && params_fit<T>(v, f32, weight, bias);
        });
        if (p.ok) {
            NormArgs<T> a;
            a.x = static_cast<const T*>(x_);
            a.residual = static_cast<const T*>(residual);
            a.weight = weight;
            a.bias = bias;
            a.f32 = f32;
            a.sum = static_cast<T*>(sum);
            a.y = static_cast<T*>(y);
            a.mean = static_cast<float*>(mean_);
            a.rstd = static_cast<float*>(rstd_);
            a.eps = static_cast<float>(eps);
            a.shape = n.shape;
            a.rule = rule;
            a.stats_wide = fits(sizeof(float) * p.V, a.mean, a.rstd);
            a.tiles = p.tiles;
            SB_CUDA(norm_launch<T>(p, false, join_kind(join, rule), a, stream));
            return;
        }
    }
    if (join) {
        launch_dropout<T>(name, x_, residual, sum, n.numel(), 1, rule, stream);
        x_ = sum;
    }
    const NormWorkspace w(n, sizeof(A), false);
    const T* x = static_cast<const T*>(x_);
    A* part = reinterpret_cast<A*>(ws + w.part);
    A* mean = mean_ ? static_cast<A*>(mean_) : reinterpret_cast<A*>(ws + w.stats);
    A* rstd = rstd_ ? static_cast<A*>(rstd_) : reinterpret_cast<A*>(ws + w.stats) + n.shape.rows;
    const bool rows = n.shape.inner == 1;
    const dim3 grid(grid_of(name, rows ? n.shape.rows : ceil_div64(n.shape.rows, 32)), n.splits);
    const unsigned joins = grid_of(name, ceil_div64(n.shape.rows, kNormThreads));
    auto stats = rows ? norm_stats_kernel<T, true> : norm_stats_kernel<T, false>;
    auto apply = rows ? norm_apply_kernel<T, true> : norm_apply_kernel<T, false>;
    stats<<<grid, kNormThreads, 0, stream>>>(x, part, n.shape, n.chunk);
    SB_CUDA(cudaGetLastError());
    norm_join_kernel<A><<<joins, kNormThreads, 0, stream>>>(part, mean, rstd, n.shape, n.chunk, n.splits, eps);
    SB_CUDA(cudaGetLastError());
    apply<<<grid, kNormThreads, 0, stream>>>(x, mean, rstd, weight, bias, f32, static_cast<T*>(y), n.shape, n.chunk);
    SB_CUDA(cudaGetLastError());
}

template <typename T>
void norm_backward(const char* name, const Norm& n, const void* gy_, const void* x_, const void* mean_,
                   const void* rstd_, const void* weight, bool f32, const void* add, const DropRule& rule, void* dx,
                   void* dropped, void* dw, void* db, char* ws, cudaStream_t stream, bool join) {
    using A = typename Storage<T>::acc;
    const T *gy = static_cast<const T*>(gy_), *x = static_cast<const T*>(x_);
    const A *mean = static_cast<const A*>(mean_), *rstd = static_cast<const A*>(rstd_);
    if constexpr (!std::is_same_v<T, double>) {
        const NormPlan p = n.plan(dtype_of<T>, true, [&](int v) {
            return fits(v * sizeof(T), gy_, x_, add, dx, dropped) && params_fit<T>(v, f32, weight);
        });
        if (p.ok) {
            NormArgs<T> a;
            a.x = static_cast<const T*>(x_);
            a.weight = weight;
            a.f32 = f32;
            a.mean = static_cast<float*>(const_cast<void*>(mean_));
            a.rstd = static_cast<float*>(const_cast<void*>(rstd_));
            a.gy = static_cast<const T*>(gy_);
            a.add = static_cast<const T*>(add);
            a.dx = static_cast<T*>(dx);
            a.dropped = static_cast<T*>(dropped);
            // few rows: their partial sums would be as large as the tensors, which are read again instead
            const bool direct = p.rows && n.shape.rows <= kDirectRows;
            a.part = (dw || db) && !direct ? reinterpret_cast<float*>(ws) : nullptr;
            a.shape = n.shape;
            a.rule = rule;
            a.stats_wide = fits(sizeof(float) * p.V, a.mean, a.rstd);
            a.tiles = p.tiles;
            if (!direct || dx || dropped) SB_CUDA(norm_launch<T>(p, true, join_kind(join, rule), a, stream));
            if (a.part) {
                param_final<T>(a.part, p.blocks, n.shape.len, dw, db, f32, stream);
            } else if (dw || db) {
                norm_param_direct_kernel<T><<<ceil_div(n.shape.len, 128), 128, 0, stream>>>(gy, x, mean, rstd, dw, db,
                                                                                            f32, n.shape);
                SB_CUDA(cudaGetLastError());
            }
            return;
        }
    }
    const NormWorkspace w(n, sizeof(A), true);
    A* part = reinterpret_cast<A*>(ws + w.part);
    A* sums = reinterpret_cast<A*>(ws + w.params);
    const bool rows = n.shape.inner == 1;
    if (dx || dropped) {
        const dim3 grid(grid_of(name, rows ? n.shape.rows : ceil_div64(n.shape.rows, 32)), n.splits);
        auto reduce = rows ? norm_bwd_sums_kernel<T, true> : norm_bwd_sums_kernel<T, false>;
        auto apply = rows ? norm_bwd_apply_kernel<T, true> : norm_bwd_apply_kernel<T, false>;
        reduce<<<grid, kNormThreads, 0, stream>>>(gy, x, mean, rstd, weight, f32, part, n.shape, n.chunk);
        SB_CUDA(cudaGetLastError());
        apply<<<grid, kNormThreads, 0, stream>>>(gy, x, mean, rstd, weight, f32, part, static_cast<const T*>(add),
                                                 static_cast<T*>(dx), static_cast<T*>(dropped), rule, n.shape,
                                                 n.chunk);
        SB_CUDA(cudaGetLastError());
    }
    if (dw || db) {
        if (rows) {
            const int tiles = static_cast<int>(ceil_div64(n.shape.len, kNormThreads));
            norm_param_rows_kernel<T><<<grid_of(name, n.blocks * tiles), kNormThreads, 0, stream>>>(
                gy, x, mean, rstd, sums, n.shape, n.rows_per, tiles);
        } else {
            norm_param_columns_kernel<T><<<grid_of(name, n.blocks * n.shape.len), kNormThreads, 0, stream>>>(
                gy, x, mean, rstd, sums, n.shape, n.rows_per);
        }
        SB_CUDA(cudaGetLastError());
        param_final<T>(sums, n.blocks, n.shape.len, dw, db, f32, stream);
    }
}

void check_workspace(const char* name, const void* workspace, int64_t have, int64_t need) {
    if (have < need || (need > 0 && workspace == nullptr))
        throw Failure{SERRON_ERR_WORKSPACE, concat(name, ": workspace of ", have, " bytes, ", need, " needed")};
    SB_CHECK(need == 0 || aligned(workspace, 256), name, ": the workspace must be aligned to 256 bytes");
}

// The kernels write both statistics where they write the mean.
void check_stats(const char* name, int dtype, const void* mean, const void* rstd) {
    check_elements(name, dtype == kF64 ? 8 : 4, mean, rstd);
    SB_CHECK((mean == nullptr) == (rstd == nullptr), name, ": mean and rstd are given both or not at all");
}

// No rows: nothing to normalise, and gradients of the parameters that are sums of nothing.
void zero_params(int len, int param_dtype, void* dw, void* db, cudaStream_t stream) {
    if (dw) SB_CUDA(cudaMemsetAsync(dw, 0, len * elem_size(param_dtype), stream));
    if (db) SB_CUDA(cudaMemsetAsync(db, 0, len * elem_size(param_dtype), stream));
}

int layer_norm_backward(const char* name, bool join, const void* grad_output, const void* grad_sum, const void* input,
                        const void* mean, const void* rstd, int64_t outer, int64_t len, int64_t inner, int32_t dtype,
                        const void* weight, int32_t param_dtype, double p, uint64_t seed, const void* seed_device,
                        uint64_t sequence, void* grad_input, void* grad_dropped, void* grad_weight, void* grad_bias,
                        void* workspace, int64_t workspace_bytes, int32_t device, void* stream_) {
    return guarded([&] {
        check_norm(name, dtype, param_dtype, grad_weight ? grad_weight : weight, grad_bias);
        const Norm n = norm_of(name, outer, len, inner);
        const DropRule rule = drop_rule(name, p, seed, seed_device, sequence);
        const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
        if (n.numel() == 0) {
            if (!grad_weight && !grad_bias) return;
            DeviceScope scope(device);
            return zero_params(n.shape.len, param_dtype, grad_weight, grad_bias, stream);
        }
        SB_CHECK(grad_output && input && mean && rstd, name, ": tensors must not be null");
        check_elements(name, elem_size(dtype), grad_output, grad_sum, input, grad_input, grad_dropped);
        check_elements(name, elem_size(param_dtype), weight, grad_weight, grad_bias);
        check_stats(name, dtype, mean, rstd);
        check_workspace(name, workspace, workspace_bytes, workspace_bytes_of(n, dtype, true));
        DeviceScope scope(device);
        with_type(dtype, [&](auto t) {
            norm_backward<decltype(t)>(name, n, grad_output, input, mean, rstd, weight,
                                       param_dtype == kF32 && dtype != kF32, grad_sum, rule, grad_input, grad_dropped,
                                       grad_weight, grad_bias, static_cast<char*>(workspace), stream, join);
        });
    });
}

}  // namespace
}  // namespace serron

using namespace serron;

extern "C" {

int64_t serron_layer_norm_workspace_bytes(int64_t outer, int64_t len, int64_t inner, int32_t dtype, int32_t backward) {
    int64_t bytes = -1;
    const int rc = guarded([&] {
        check_norm("serron::layer_norm", dtype, dtype, nullptr, nullptr);
        bytes = workspace_bytes_of(norm_of("serron::layer_norm", outer, len, inner), dtype, backward != 0);
    });
    return rc == SERRON_OK ? bytes : -1;
}

int serron_layer_norm(const void* input, int64_t outer, int64_t len, int64_t inner, int32_t dtype, const void* weight,
                      const void* bias, int32_t param_dtype, double eps, void* output, void* mean, void* rstd,
                      void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    const char* name = "serron::layer_norm";
    return guarded([&] {
        check_norm(name, dtype, param_dtype, weight, bias);
        SB_CHECK(eps >= 0.0 && std::isfinite(eps), name, ": eps must be finite and not negative, got ", eps);
        const Norm n = norm_of(name, outer, len, inner);
        check_stats(name, dtype, mean, rstd);
        if (n.numel() == 0) return;
        SB_CHECK(input && output, name, ": tensors must not be null");
        check_elements(name, elem_size(dtype), input, output);
        check_elements(name, elem_size(param_dtype), weight, bias);
        check_workspace(name, workspace, workspace_bytes, workspace_bytes_of(n, dtype, false));
        DeviceScope scope(device);
        with_type(dtype, [&](auto t) {
            norm_forward<decltype(t)>(name, n, input, weight, bias, param_dtype == kF32 && dtype != kF32, eps, output,
                                      mean, rstd, static_cast<char*>(workspace), static_cast<cudaStream_t>(stream),
                                      nullptr, nullptr, DropRule());
        });
    });
}

int serron_layer_norm_backward(const void* grad_output, const void* input, const void* mean, const void* rstd,
                               int64_t outer, int64_t len, int64_t inner, int32_t dtype, const void* weight,
                               int32_t param_dtype, void* grad_input, void* grad_weight, void* grad_bias,
                               void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    return layer_norm_backward("serron::layer_norm_backward", false, grad_output, nullptr, input, mean, rstd, outer, len,
                               inner, dtype, weight, param_dtype, 0.0, 0, nullptr, 0, grad_input, nullptr, grad_weight,
                               grad_bias, workspace, workspace_bytes, device, stream);
}

int serron_dropout(const void* input, const void* residual, int64_t numel, int64_t span, int32_t dtype, double p,
                   uint64_t seed, const void* seed_device, uint64_t sequence, void* output, int32_t device,
                   void* stream) {
    const char* name = "serron::dropout";
    return guarded([&] {
        SB_CHECK(dtype >= kF32 && dtype <= kBF16, name, ": unsupported dtype code ", dtype);
        SB_CHECK(numel >= 0, name, ": sizes must be non-negative");
        SB_CHECK(span >= 1, name, ": a decision must cover at least one element, got ", span);
        const DropRule rule = drop_rule(name, p, seed, seed_device, sequence);
        if (numel == 0) return;
        SB_CHECK(input && output, name, ": tensors must not be null");
        check_elements(name, elem_size(dtype), input, residual, output);
        DeviceScope scope(device);
        with_type(dtype, [&](auto t) {
            launch_dropout<decltype(t)>(name, input, residual, output, numel, span, rule,
                                        static_cast<cudaStream_t>(stream));
        });
    });
}

int serron_dropout_add_layer_norm(const void* input, const void* residual, int64_t outer, int64_t len, int64_t inner,
                                  int32_t dtype, const void* weight, const void* bias, int32_t param_dtype, double p,
                                  uint64_t seed, const void* seed_device, uint64_t sequence, double eps, void* sum,
                                  void* output, void* mean, void* rstd, void* workspace, int64_t workspace_bytes,
                                  int32_t device, void* stream_) {
    const char* name = "serron::dropout_add_layer_norm";
    return guarded([&] {
        check_norm(name, dtype, param_dtype, weight, bias);
        SB_CHECK(eps >= 0.0 && std::isfinite(eps), name, ": eps must be finite and not negative, got ", eps);
        const Norm n = norm_of(name, outer, len, inner);
        const DropRule rule = drop_rule(name, p, seed, seed_device, sequence);
        check_stats(name, dtype, mean, rstd);
        if (n.numel() == 0) return;
        SB_CHECK(input && residual && sum && output, name, ": tensors must not be null");
        check_elements(name, elem_size(dtype), input, residual, sum, output);
        check_elements(name, elem_size(param_dtype), weight, bias);
        check_workspace(name, workspace, workspace_bytes, workspace_bytes_of(n, dtype, false));
        const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
        DeviceScope scope(device);
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            norm_forward<T>(name, n, input, weight, bias, param_dtype == kF32 && dtype != kF32, eps, output, mean, rstd,
                            static_cast<char*>(workspace), stream, residual, sum, rule);
        });
    });
}

int serron_dropout_add_layer_norm_backward(const void* grad_output, const void* grad_sum, const void* sum,
                                           const void* mean, const void* rstd, int64_t outer, int64_t len,
                                           int64_t inner, int32_t dtype, const void* weight, int32_t param_dtype,
                                           double p, uint64_t seed, const void* seed_device, uint64_t sequence,
                                           void* grad_input, void* grad_residual, void* grad_weight, void* grad_bias,
                                           void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    return layer_norm_backward("serron::dropout_add_layer_norm_backward", true, grad_output, grad_sum, sum, mean, rstd,
                               outer, len, inner, dtype, weight, param_dtype, p, seed, seed_device, sequence,
                               grad_residual, grad_input, grad_weight, grad_bias, workspace, workspace_bytes, device,
                               stream);
}

}  // extern "C"
