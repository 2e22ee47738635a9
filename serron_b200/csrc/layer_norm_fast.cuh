// Layer norm, alone or joined with residual + dropout, for rows that fit in registers: each element is read once and
// written once a pass.  Formulas: layer_norm.cuh.
//
// Both layouts work the same way.  A thread keeps NV vectors of V elements; a row's partial results are joined over
// a warp or a block through shared memory and, where a row is too long for one block or rows are few, over a cluster
// of blocks through distributed shared memory.  The forward pass joins (count, mean, sum of squared deviations) of
// parts, each found in two passes over registers, so a level far above the spread costs nothing; the backward pass
// joins two plain sums.
//
//   rows     (inner == 1): a row lies along threadIdx.x, threadIdx.y counts rows of a block
//   columns  (inner  > 1): threadIdx.x counts V neighbouring rows (neighbours in memory), threadIdx.y the strides of
//            the normalised dimension
#pragma once

#include <cooperative_groups.h>

#include "layer_norm.cuh"
#include "layer_vec.cuh"

namespace serron {

namespace cg = cooperative_groups;

template <typename T>
struct NormArgs {
    const T* x = nullptr;         // the input; the join's sum in the backward pass
    const T* residual = nullptr;  // the join
    const void* weight = nullptr;
    const void* bias = nullptr;
    bool f32 = false;  // weight and bias in float32 beside 16-bit activations
    T* sum = nullptr;  // the join
    T* y = nullptr;
    float* mean = nullptr;
    float* rstd = nullptr;
    // backward
    const T* gy = nullptr;
    const T* add = nullptr;  // the gradient that reaches x by another way
    T* dx = nullptr;
    T* dropped = nullptr;    // its masked copy
    float* part = nullptr;   // sums for the gradients of weight and bias
    float eps = 0.0f;
    NormShape shape;
    DropRule rule;
    long long tiles = 0;  // backward: pieces of work that the blocks (clusters) share
};

// h = residual + dropout(x), rounded to T.  Decisions go by the element's index e in memory.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> joined(const Pack<T, V>& x, const Pack<T, V>& residual, long long e,
                                             const DropRule& rule, uint64_t key, float scale) {
    float v[V];
    if (rule.threshold == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = x.get(i) + residual.get(i);
    } else {
        uint32_t words[V];
        drop_words<V>(e, rule.sequence, key, words);
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = (rule.keeps(words[i]) ? scaled(x.get(i), scale) : 0.0f) + residual.get(i);
    }
    Pack<T, V> out;
    out.set(v);
    return out;
}

// ------------------------------------------------------------------------------------------------
// columns
// ------------------------------------------------------------------------------------------------

// Where a thread of a column kernel stands.
struct ColumnPlace {
    long long offset;  // of its first row's first element
    bool live;
};
template <int V>
__device__ __forceinline__ ColumnPlace column_place(const NormShape& s, long long q) {
    const long long vectors = s.rows / V;  // V divides inner
    ColumnPlace p;
    p.live = q < vectors;
    p.offset = 0;
    if (p.live) {
        const unsigned per = s.inner / V;
        // 64-bit division only where the count needs it
        const long long o = vectors < (1ll << 32) ? static_cast<unsigned>(q) / per : q / per;
        p.offset = o * s.len * s.inner + (q - o * per) * V;
    }
    return p;
}

// How many of the positions first, first + step, ... lie below len.
__device__ __forceinline__ int count_below(int first, int step, int len) {
    return first < len ? (len - first + step - 1) / step : 0;
}

template <typename T, int V, int NV, bool JOIN>
__global__ void __launch_bounds__(512, 1) norm_columns_kernel(NormArgs<T> a) {
    using P = Pack<T, V>;
    extern __shared__ float shared[];  // [2][blockDim.y][V][blockDim.x], then [2][V][blockDim.x] for the cluster
    const int lanes = blockDim.x, groups = blockDim.y, lane = threadIdx.x;
    const int clusters = gridDim.y, all = groups * clusters;
    const int group = blockIdx.y * groups + threadIdx.y;
    const int len = a.shape.len;
    const long long q = blockIdx.x * static_cast<long long>(lanes) + lane;
    const ColumnPlace place = column_place<V>(a.shape, q);
    const long long step = static_cast<long long>(all) * a.shape.inner;
    const long long first = place.offset + static_cast<long long>(group) * a.shape.inner;

    P h[NV];
    if (JOIN) {
        P r[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (place.live && group + k * all < len) {
                h[k] = P::load(a.x + first + k * step);
                r[k] = P::load(a.residual + first + k * step);
            }
        }
        const uint64_t key = a.rule.key();
        const float scale = static_cast<float>(a.rule.scale);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (place.live && group + k * all < len) {
                h[k] = joined<T, V>(h[k], r[k], first + k * step, a.rule, key, scale);
                h[k].store(a.sum + first + k * step);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (place.live && group + k * all < len) h[k] = P::load(a.x + first + k * step);
    }

    float mean[V], m2[V];
    const int count = count_below(group, all, len);
#pragma unroll
    for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (group + k * all < len) {
#pragma unroll
            for (int v = 0; v < V; ++v) mean[v] += h[k].get(v);
        }
    }
    if (count > 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) mean[v] /= static_cast<float>(count);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (group + k * all < len) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = h[k].get(v) - mean[v];
                m2[v] += d * d;
            }
        }
    }
    if (groups > 1) {
        float* part = shared;
        const int plane = groups * lanes * V;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            part[(threadIdx.y * V + v) * lanes + lane] = mean[v];
            part[plane + (threadIdx.y * V + v) * lanes + lane] = m2[v];
        }
        __syncthreads();
        // what the whole block holds: its groups are blockIdx.y * groups .. + groups - 1
        int held = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.0f;
        for (int g = 0; g < groups; ++g) {
            const int n = count_below(blockIdx.y * groups + g, all, len);
            held += n;
#pragma unroll
            for (int v = 0; v < V; ++v) mean[v] += static_cast<float>(n) * part[(g * V + v) * lanes + lane];
        }
        if (held > 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) mean[v] /= static_cast<float>(held);
        }
        for (int g = 0; g < groups; ++g) {
            const float n = static_cast<float>(count_below(blockIdx.y * groups + g, all, len));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = part[(g * V + v) * lanes + lane] - mean[v];
                m2[v] += part[plane + (g * V + v) * lanes + lane] + n * d * d;
            }
        }
    }
    if (clusters > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        float* mine = shared + 2 * groups * lanes * V;
        if (threadIdx.y == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                mine[v * lanes + lane] = mean[v];
                mine[(V + v) * lanes + lane] = m2[v];
            }
        }
        cluster.sync();
#pragma unroll
        for (int v = 0; v < V; ++v) mean[v] = m2[v] = 0.0f;
        for (int c = 0; c < clusters; ++c) {
            const float* theirs = cluster.map_shared_rank(mine, c);
            int n = 0;
            for (int g = 0; g < groups; ++g) n += count_below(c * groups + g, all, len);
#pragma unroll
            for (int v = 0; v < V; ++v) mean[v] += static_cast<float>(n) * theirs[v * lanes + lane];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) mean[v] /= static_cast<float>(len);
        for (int c = 0; c < clusters; ++c) {
            const float* theirs = cluster.map_shared_rank(mine, c);
            int n = 0;
            for (int g = 0; g < groups; ++g) n += count_below(c * groups + g, all, len);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = theirs[v * lanes + lane] - mean[v];
                m2[v] += theirs[(V + v) * lanes + lane] + static_cast<float>(n) * d * d;
            }
        }
        cluster.sync();  // no block leaves while another reads it
    }
    if (!place.live) return;
    float rstd[V];
#pragma unroll
    for (int v = 0; v < V; ++v) rstd[v] = inverse_root(m2[v] / static_cast<float>(len) + a.eps);
    if (a.mean != nullptr && group == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a.mean[q * V + v] = mean[v];
            a.rstd[q * V + v] = rstd[v];
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = group + k * all;
        if (c < len) {
            const float w = a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
            const float b = a.bias ? load_param<T>(a.bias, c, a.f32) : 0.0f;
            float v[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (h[k].get(i) - mean[i]) * rstd[i] * w + b;
            P out;
            out.set(v);
            out.store(a.y + first + k * step);
        }
    }
}

// The block (cluster) walks over tiles; a thread adds up its channels' gradients on the way.  `part` gets
// [gridDim.x][2][len] sums.
template <typename T, int V, int NV, bool JOIN>
__global__ void __launch_bounds__(512, 1) norm_columns_bwd_kernel(NormArgs<T> a) {
    using P = Pack<T, V>;
    extern __shared__ float shared[];  // per tile of two: [2][blockDim.y][V][blockDim.x], and for the cluster
                                    // [2][V][blockDim.x] of both behind them
    const int lanes = blockDim.x, groups = blockDim.y, lane = threadIdx.x;
    const int clusters = gridDim.y, all = groups * clusters;
    const int group = blockIdx.y * groups + threadIdx.y;
    const int len = a.shape.len;
    const long long step = static_cast<long long>(all) * a.shape.inner;
    const float inverse = 1.0f / static_cast<float>(len);
    const uint64_t key = JOIN ? a.rule.key() : 0;
    const float scale = static_cast<float>(a.rule.scale);

    float dw[NV], db[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) dw[k] = db[k] = 0.0f;

    int parity = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x, parity ^= 1) {
        const long long q = t * lanes + lane;
        const ColumnPlace place = column_place<V>(a.shape, q);
        const long long first = place.offset + static_cast<long long>(group) * a.shape.inner;
        P gy[NV], x[NV];
        float mean[V], rstd[V];
        if (place.live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (group + k * all < len) {
                    gy[k] = P::load(a.gy + first + k * step);
                    x[k] = P::load(a.x + first + k * step);
                }
            }
#pragma unroll
            for (int v = 0; v < V; ++v) {
                mean[v] = a.mean[q * V + v];
                rstd[v] = a.rstd[q * V + v];
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) mean[v] = rstd[v] = 0.0f;
        }
        float s1[V], s2[V];
#pragma unroll
        for (int v = 0; v < V; ++v) s1[v] = s2[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = group + k * all;
            if (c < len) {
                const float w = a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
                float sw = 0.0f, sb = 0.0f;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float g = gy[k].get(v), gx = g * ((x[k].get(v) - mean[v]) * rstd[v]);
                    sw += gx;
                    sb += g;
                    s1[v] += g * w;
                    s2[v] += gx * w;
                }
                dw[k] += sw;
                db[k] += sb;
            }
        }
        if (groups > 1) {
            const int plane = groups * lanes * V;
            float* part = shared + parity * 2 * plane;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                part[(threadIdx.y * V + v) * lanes + lane] = s1[v];
                part[plane + (threadIdx.y * V + v) * lanes + lane] = s2[v];
            }
            __syncthreads();
#pragma unroll
            for (int v = 0; v < V; ++v) s1[v] = s2[v] = 0.0f;
            for (int g = 0; g < groups; ++g) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    s1[v] += part[(g * V + v) * lanes + lane];
                    s2[v] += part[plane + (g * V + v) * lanes + lane];
                }
            }
        }
        if (clusters > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            float* mine = shared + 4 * groups * lanes * V + parity * 2 * lanes * V;
            if (threadIdx.y == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    mine[v * lanes + lane] = s1[v];
                    mine[(V + v) * lanes + lane] = s2[v];
                }
            }
            cluster.sync();
#pragma unroll
            for (int v = 0; v < V; ++v) s1[v] = s2[v] = 0.0f;
            for (int c = 0; c < clusters; ++c) {
                const float* theirs = cluster.map_shared_rank(mine, c);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    s1[v] += theirs[v * lanes + lane];
                    s2[v] += theirs[(V + v) * lanes + lane];
                }
            }
        }
        if (place.live && (a.dx != nullptr || (JOIN && a.dropped != nullptr))) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                s1[v] *= inverse;
                s2[v] *= inverse;
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = group + k * all;
                if (c < len) {
                    const long long e = first + k * step;
                    const float w = a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
                    float d[V];
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        d[v] = rstd[v] * (gy[k].get(v) * w - s1[v] - ((x[k].get(v) - mean[v]) * rstd[v]) * s2[v]);
                    if (JOIN && a.add != nullptr) {
                        const P add = P::load(a.add + e);
#pragma unroll
                        for (int v = 0; v < V; ++v) d[v] += add.get(v);
                    }
                    P out;
                    if (a.dx != nullptr) {
                        out.set(d);
                        out.store(a.dx + e);
                    }
                    if (JOIN && a.dropped != nullptr) {
                        if (a.rule.threshold != 0) {
                            uint32_t words[V];
                            drop_words<V>(e, a.rule.sequence, key, words);
#pragma unroll
                            for (int v = 0; v < V; ++v) d[v] = a.rule.keeps(words[v]) ? scaled(d[v], scale) : 0.0f;
                        }
                        out.set(d);
                        out.store(a.dropped + e);
                    }
                }
            }
        }
    }
    if (clusters > 1) cg::this_cluster().sync();  // no block leaves while another reads it
    if (a.part == nullptr) return;
    // the lanes of a warp hold the same channels: a warp of the block each, joined through shared memory where a
    // group has several
    const int warps = lanes / 32;
    if (warps > 1) __syncthreads();  // the last tile's use of `shared`
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = group + k * all;
        float w = warp_sum(dw[k]), b = warp_sum(db[k]);
        if (warps > 1) {
            float* part = shared + ((k * groups + threadIdx.y) * warps) * 2;
            if ((lane & 31) == 0) {
                part[(lane >> 5) * 2] = w;
                part[(lane >> 5) * 2 + 1] = b;
            }
            __syncthreads();
            if (lane == 0) {
                w = b = 0.0f;
                for (int i = 0; i < warps; ++i) {
                    w += part[i * 2];
                    b += part[i * 2 + 1];
                }
            }
        }
        if (lane == 0 && c < len) {
            a.part[(blockIdx.x * 2ll) * len + c] = w;
            a.part[(blockIdx.x * 2ll + 1) * len + c] = b;
        }
    }
}

// ------------------------------------------------------------------------------------------------
// rows
// ------------------------------------------------------------------------------------------------

// Joins (count, mean, sum of squared deviations) of 32 lanes' parts; lanes without one give a count of zero.
__device__ __forceinline__ void warp_join(float& n, float& mean, float& m2) {
    const float total = warp_sum(n);
    const float all = total > 0.0f ? warp_sum(n * mean) / total : 0.0f;
    const float d = mean - all;
    m2 = warp_sum(m2 + n * d * d);
    mean = all;
    n = total;
}

template <typename T, int V, int NV, bool JOIN>
__global__ void __launch_bounds__(1024) norm_rows_kernel(NormArgs<T> a) {
    using P = Pack<T, V>;
    __shared__ float shared[32][3], block[3];
    const int width = blockDim.x, lane = threadIdx.x & 31, warps = width / 32;
    const int clusters = gridDim.y, all = width * clusters;
    const int vectors = a.shape.len / V;  // V divides len
    const long long row = blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y;
    const bool live = row < a.shape.rows;
    const int first = blockIdx.y * width + threadIdx.x;
    const long long base = live ? row * a.shape.len : 0;

    P h[NV];
    if (JOIN) {
        P r[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (live && first + k * all < vectors) {
                h[k] = P::load(a.x + base + (first + k * all) * V);
                r[k] = P::load(a.residual + base + (first + k * all) * V);
            }
        }
        const uint64_t key = a.rule.key();
        const float scale = static_cast<float>(a.rule.scale);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (live && first + k * all < vectors) {
                const long long e = base + (first + k * all) * V;
                h[k] = joined<T, V>(h[k], r[k], e, a.rule, key, scale);
                h[k].store(a.sum + e);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (live && first + k * all < vectors) h[k] = P::load(a.x + base + (first + k * all) * V);
    }

    // the warp's elements, in two passes over registers
    float n = static_cast<float>(live ? count_below(first, all, vectors) * V : 0);
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (first + k * all < vectors) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum += h[k].get(v);
        }
    }
    n = warp_sum(n);
    float mean = n > 0.0f ? warp_sum(sum) / n : 0.0f, m2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (first + k * all < vectors) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float d = h[k].get(v) - mean;
                m2 += d * d;
            }
        }
    }
    m2 = warp_sum(m2);
    if (warps > 1) {  // a row a block
        if (lane == 0) {
            shared[threadIdx.x >> 5][0] = n;
            shared[threadIdx.x >> 5][1] = mean;
            shared[threadIdx.x >> 5][2] = m2;
        }
        __syncthreads();
        n = lane < warps ? shared[lane][0] : 0.0f;
        mean = lane < warps ? shared[lane][1] : 0.0f;
        m2 = lane < warps ? shared[lane][2] : 0.0f;
        warp_join(n, mean, m2);
    }
    if (clusters > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) {
            block[0] = n;
            block[1] = mean;
            block[2] = m2;
        }
        cluster.sync();
        const float* theirs = cluster.map_shared_rank(block, lane < clusters ? lane : 0);
        n = lane < clusters ? theirs[0] : 0.0f;
        mean = lane < clusters ? theirs[1] : 0.0f;
        m2 = lane < clusters ? theirs[2] : 0.0f;
        warp_join(n, mean, m2);
        cluster.sync();  // no block leaves while another reads it
    }
    if (!live) return;
    const float rstd = inverse_root(m2 / static_cast<float>(a.shape.len) + a.eps);
    if (a.mean != nullptr && first == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int j = first + k * all;
        if (j < vectors) {
            float v[V], w[V];
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = (h[k].get(i) - mean) * rstd;
            if (a.weight) {
                load_params<T, V>(a.weight, j * V, a.f32, w);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] *= w[i];
            }
            if (a.bias) {
                load_params<T, V>(a.bias, j * V, a.f32, w);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] += w[i];
            }
            P out;
            out.set(v);
            out.store(a.y + base + j * V);
        }
    }
}

// A group of threadIdx.x threads walks over rows; each thread adds up its elements' parameter gradients on the way.
// `part` gets [gridDim.x][2][len] sums, one per block (cluster).
template <typename T, int V, int NV, bool JOIN>
__global__ void __launch_bounds__(512, 1) norm_rows_bwd_kernel(NormArgs<T> a) {
    using P = Pack<T, V>;
    __shared__ float shared[2][16][2], block[2][2];
    extern __shared__ float sums[];  // [NV * V][threads] where a block has several rows
    const int width = blockDim.x, lane = threadIdx.x & 31, warps = width / 32;
    const int clusters = gridDim.y, all = width * clusters;
    const int vectors = a.shape.len / V;
    const int first = blockIdx.y * width + threadIdx.x;
    const float inverse = 1.0f / static_cast<float>(a.shape.len);
    const uint64_t key = JOIN ? a.rule.key() : 0;
    const float scale = static_cast<float>(a.rule.scale);

    float dw[NV][V], db[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) dw[k][v] = db[k][v] = 0.0f;

    int parity = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x, parity ^= 1) {
        const long long row = t * blockDim.y + threadIdx.y;
        const bool live = row < a.shape.rows;
        const long long base = live ? row * a.shape.len : 0;
        P gy[NV], x[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (live && first + k * all < vectors) {
                gy[k] = P::load(a.gy + base + (first + k * all) * V);
                x[k] = P::load(a.x + base + (first + k * all) * V);
            }
        }
        const float mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
        float s1 = 0.0f, s2 = 0.0f;
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = first + k * all;
                if (j < vectors) {
                    float w[V];
                    if (a.weight) load_params<T, V>(a.weight, j * V, a.f32, w);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const float g = gy[k].get(v), gx = g * ((x[k].get(v) - mean) * rstd);
                        dw[k][v] += gx;
                        db[k][v] += g;
                        s1 += a.weight ? g * w[v] : g;
                        s2 += a.weight ? gx * w[v] : gx;
                    }
                }
            }
        }
        s1 = warp_sum(s1);
        s2 = warp_sum(s2);
        if (warps > 1) {
            if (lane == 0) {
                shared[parity][threadIdx.x >> 5][0] = s1;
                shared[parity][threadIdx.x >> 5][1] = s2;
            }
            __syncthreads();
            s1 = warp_sum(lane < warps ? shared[parity][lane][0] : 0.0f);
            s2 = warp_sum(lane < warps ? shared[parity][lane][1] : 0.0f);
        }
        if (clusters > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (threadIdx.x == 0) {
                block[parity][0] = s1;
                block[parity][1] = s2;
            }
            cluster.sync();
            const float* theirs = cluster.map_shared_rank(block[parity], lane < clusters ? lane : 0);
            s1 = warp_sum(lane < clusters ? theirs[0] : 0.0f);
            s2 = warp_sum(lane < clusters ? theirs[1] : 0.0f);
        }
        if (live && (a.dx != nullptr || (JOIN && a.dropped != nullptr))) {
            s1 *= inverse;
            s2 *= inverse;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = first + k * all;
                if (j < vectors) {
                    const long long e = base + j * V;
                    float w[V], d[V];
                    if (a.weight) load_params<T, V>(a.weight, j * V, a.f32, w);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const float g = a.weight ? gy[k].get(v) * w[v] : gy[k].get(v);
                        d[v] = rstd * (g - s1 - ((x[k].get(v) - mean) * rstd) * s2);
                    }
                    if (JOIN && a.add != nullptr) {
                        const P add = P::load(a.add + e);
#pragma unroll
                        for (int v = 0; v < V; ++v) d[v] += add.get(v);
                    }
                    P out;
                    if (a.dx != nullptr) {
                        out.set(d);
                        out.store(a.dx + e);
                    }
                    if (JOIN && a.dropped != nullptr) {
                        if (a.rule.threshold != 0) {
                            uint32_t words[V];
                            drop_words<V>(e, a.rule.sequence, key, words);
#pragma unroll
                            for (int v = 0; v < V; ++v) d[v] = a.rule.keeps(words[v]) ? scaled(d[v], scale) : 0.0f;
                        }
                        out.set(d);
                        out.store(a.dropped + e);
                    }
                }
            }
        }
    }
    if (clusters > 1) cg::this_cluster().sync();  // no block leaves while another reads it
    if (a.part == nullptr) return;
    const long long len = a.shape.len;
    const int rows = blockDim.y, threads = width * rows, tid = threadIdx.y * width + threadIdx.x;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = a.part + (blockIdx.x * 2ll + which) * len;
        if (rows == 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = first + k * all;
                if (j < vectors) {
#pragma unroll
                    for (int v = 0; v < V; ++v) out[static_cast<long long>(j) * V + v] = which ? db[k][v] : dw[k][v];
                }
            }
        } else {
            if (which) __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) sums[(k * V + v) * threads + tid] = which ? db[k][v] : dw[k][v];
            __syncthreads();
            for (int l = tid; l < len; l += threads) {
                const int j = l / V, k = j / width, x = j % width;  // one block a row: no cluster here
                float s = 0.0f;
                for (int r = 0; r < rows; ++r) s += sums[(k * V + l % V) * threads + r * width + x];
                out[l] = s;
            }
        }
    }
}

}  // namespace serron
