// Layer norm, alone or joined with residual + dropout, for rows that fit in registers: each element is read once and
// written once a pass.  Formulas: layer_norm.cuh.
//
// Both layouts work the same way.  A thread keeps vectors of V elements of a row; a row's partial results are joined over
// a warp or a block through shared memory and, where a row is too long for one block or rows are few, over a cluster
// of blocks through distributed shared memory.
//
//   rows     (inner == 1): a row lies along threadIdx.x; threadIdx.y counts groups of threads, each with R rows at a time
//   columns  (inner  > 1): threadIdx.x counts vectors of V neighbouring rows (neighbours in memory), threadIdx.y the
//            strides of the normalised dimension
//
// Forward: a part of a row (a thread's, a warp's or a block's) gives its sum S and the sum Q of squared distances from a
// pivot near its mean; parts of n elements join as  mean = sum S / len  and  sum of squares about it =
// sum (Q + n (pivot - mean)^2),  so a level far above the spread costs nothing.  Backward: two plain sums.
//
// These kernels would be bound by instructions, not by memory, if written one float at a time (31 instructions an element
// of a row, 48 of a column, where 16-bit elements leave about 20 at the memory's rate): elements are unpacked
// once and computed on in pairs (layer_vec.cuh), and divisions are one multiplication and one correction.
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
    bool stats_wide = false;  // mean and rstd may be read and written in vectors (columns)
    long long tiles = 0;      // pieces of work that the blocks (clusters) share
};

// s / n where `inverse` is 1 / n: exact where the quotient is a float.
__device__ __forceinline__ float quotient(float s, float n, float inverse) {
    const float q = s * inverse;
    return fmaf(fmaf(-n, q, s), inverse, q);
}

// 1 / sqrt(v): the approximation and one Newton step (infinite v: zero, as 1 / sqrt gives).
__device__ __forceinline__ float root_inverse(float v) {
    const float r = rsqrtf(v);
    const float better = fmaf(r * 0.5f, fmaf(-(v * r), r, 1.0f), r);
    return v < __int_as_float(0x7f800000) ? better : r;
}

// How many of the positions first, first + step, ... lie below len, for any first < step: one division for all.
struct CountBelow {
    int whole, rest;
    __device__ __forceinline__ CountBelow(int step, int len) : whole(len / step), rest(len - len / step * step) {}
    __device__ __forceinline__ int operator()(int first) const { return whole + (first < rest); }
};

// The generator's keys, in shared memory: a launch takes its seed from the host or from device memory.
__device__ __forceinline__ void share_keys(const DropRule& rule, PhiloxKeys& shared) {
    const int r = threadIdx.y * blockDim.x + threadIdx.x;
    if (r < kPhiloxRounds) {
        const uint64_t seed = rule.seed_device ? __ldg(rule.seed_device) : 0;
        shared.k0[r] = rule.seed_device ? static_cast<uint32_t>(seed) + r * kPhiloxKey0 : rule.keys.k0[r];
        shared.k1[r] = rule.seed_device ? static_cast<uint32_t>(seed >> 32) + r * kPhiloxKey1 : rule.keys.k1[r];
    }
    __syncthreads();
}

// dropout(v) for the elements from e on.
template <int V>
__device__ __forceinline__ Floats<V> drop(const Floats<V>& v, long long e, const DropRule& rule, const PhiloxKeys& keys) {
    if (rule.threshold == 0) return v;
    Floats<V> out;
    if (rule.all) {
        out.fill(0.0f);
        return out;
    }
    uint32_t words[V];
    drop_words<V>(e, rule.sequence, keys, words);
    return dropped<V>(v, words, rule.threshold, static_cast<float>(rule.scale));
}

// h = residual + dropout(x), rounded to T and stored.
template <typename T, int V>
__device__ __forceinline__ Floats<V> join_at(const Pack<T, V>& x, const Pack<T, V>& residual, long long e,
                                             const DropRule& rule, const PhiloxKeys& keys, T* sum) {
    Floats<V> v = drop<V>(x.floats(), e, rule, keys);
    const Floats<V> r = residual.floats();
#pragma unroll
    for (int i = 0; i < Floats<V>::N; ++i) v.e[i] = add(v.e[i], r.e[i]);
    const Pack<T, V> out = Pack<T, V>::of(v);
    out.store(sum + e);
    return out.floats();
}

// What follows dx = v in memory order from e on: the sum with `add`, dx itself, and its masked copy.
template <typename T, int V, bool JOIN>
__device__ __forceinline__ void store_dx(Floats<V> v, long long e, const NormArgs<T>& a, const Pack<T, V>& extra,
                                         const PhiloxKeys& keys) {
    if (JOIN && a.add != nullptr) {
        const Floats<V> f = extra.floats();
#pragma unroll
        for (int i = 0; i < Floats<V>::N; ++i) v.e[i] = add(v.e[i], f.e[i]);
    }
    if (a.dx != nullptr) Pack<T, V>::of(v).store(a.dx + e);
    if (JOIN && a.dropped != nullptr) Pack<T, V>::of(drop<V>(v, e, a.rule, keys)).store(a.dropped + e);
}

// ------------------------------------------------------------------------------------------------
// columns
// ------------------------------------------------------------------------------------------------

// The offset of vector q's first row, and whether there is such a vector.
template <int V>
__device__ __forceinline__ bool column_place(const NormShape& s, long long q, long long& offset) {
    const long long vectors = s.rows / V;  // V divides inner
    offset = 0;
    if (q >= vectors) return false;
    const unsigned per = s.inner / V;
    // a 64-bit division only where the count needs it
    const long long o = vectors < (1ll << 32) ? static_cast<unsigned>(q) / per : q / per;
    offset = o * s.len * s.inner + (q - o * per) * V;
    return true;
}

// V floats of lane `lane` in a plane of `lanes` such, one access each.
template <int V>
__device__ __forceinline__ void put(float* plane, int lane, const Floats<V>& v) {
    Pack<float, V>::of(v).store(plane + lane * V);
}
template <int V>
__device__ __forceinline__ Floats<V> got(const float* plane, int lane) {
    return Pack<float, V>::load(plane + lane * V).floats();
}

// FULL: every thread has all of its NV strides (len is their number times the groups').
template <typename T, int V, int NV, bool JOIN, bool FULL>
__global__ void __launch_bounds__(512, 1) norm_columns_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    // [2 tiles][2][groups][lanes][V], then for the cluster [2 tiles][2][lanes][V]
    extern __shared__ __align__(16) float shared[];
    __shared__ PhiloxKeys keys;
    const int lanes = blockDim.x, groups = blockDim.y, lane = threadIdx.x;
    const int clusters = gridDim.y, all = groups * clusters;
    const int group = blockIdx.y * groups + threadIdx.y;
    const int len = a.shape.len, plane = lanes * V;
    const long long step = static_cast<long long>(all) * a.shape.inner;
    const CountBelow below(all, len);
    const int count = FULL ? NV : below(group);
    const float part_inverse = 1.0f / static_cast<float>(max(count, 1)), len_inverse = 1.0f / static_cast<float>(len);
    if (JOIN) share_keys(a.rule, keys);

    float w[NV], b[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = group + k * all;
        w[k] = (FULL || c < len) && a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
        b[k] = (FULL || c < len) && a.bias ? load_param<T>(a.bias, c, a.f32) : 0.0f;
    }

    int parity = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x, parity ^= 1) {
        const long long q = t * lanes + lane;
        long long offset;
        const bool live = column_place<V>(a.shape, q, offset);
        const long long first = offset + static_cast<long long>(group) * a.shape.inner;
        F h[NV];
        {
            P in[NV], res[JOIN ? NV : 1];
            if (live) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    if (FULL || group + k * all < len) {
                        in[k] = P::load(a.x + first + k * step);
                        if (JOIN) res[k] = P::load(a.residual + first + k * step);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (live && (FULL || group + k * all < len)) {
                    if (JOIN)
                        h[k] = join_at<T, V>(in[k], res[k], first + k * step, a.rule, keys, a.sum);
                    else
                        h[k] = in[k].floats();
                } else {
                    h[k].fill(0.0f);
                }
            }
        }
        // the thread's part of each row: sum, and squares about its mean
        F sum, squares, mean;
        sum.fill(0.0f);
        squares.fill(0.0f);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) sum.e[i] = add(sum.e[i], h[k].e[i]);
        if (all == 1) {
            float s[V];
            sum.to(s);
#pragma unroll
            for (int v = 0; v < V; ++v) s[v] = quotient(s[v], static_cast<float>(len), len_inverse);
            mean.from(s);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) mean.e[i] = mul(sum.e[i], splat<E>(part_inverse));
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (FULL || group + k * all < len) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const E d = sub(h[k].e[i], mean.e[i]);
                    squares.e[i] = fma(d, d, squares.e[i]);
                }
            }
        }
        if (groups > 1) {
            float* sums = shared + parity * 2 * groups * plane;
            float* sqs = sums + groups * plane;
            put<V>(sums + threadIdx.y * plane, lane, sum);
            put<V>(sqs + threadIdx.y * plane, lane, squares);
            __syncthreads();
            // the block's part: its groups are blockIdx.y * groups .. + groups - 1
            sum.fill(0.0f);
            int held = 0;
            for (int g = 0; g < groups; ++g) {
                const F s = got<V>(sums + g * plane, lane);
                held += below(blockIdx.y * groups + g);
#pragma unroll
                for (int i = 0; i < N; ++i) sum.e[i] = add(sum.e[i], s.e[i]);
            }
            const float n = static_cast<float>(max(held, 1)), n_inverse = clusters == 1 ? len_inverse : 1.0f / n;
            float m[V];
            sum.to(m);
#pragma unroll
            for (int v = 0; v < V; ++v) m[v] = quotient(m[v], n, n_inverse);
            mean.from(m);
            squares.fill(0.0f);
            const float more_inverse = 1.0f / static_cast<float>(below.whole + 1);
            const float whole_inverse = 1.0f / static_cast<float>(max(below.whole, 1));
            for (int g = 0; g < groups; ++g) {
                const bool more = blockIdx.y * groups + g < below.rest;
                const float gn = static_cast<float>(below.whole + more), inverse = more ? more_inverse : whole_inverse;
                const F s = got<V>(sums + g * plane, lane), sq = got<V>(sqs + g * plane, lane);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const E d = sub(mul(s.e[i], splat<E>(inverse)), mean.e[i]);
                    squares.e[i] = add(squares.e[i], fma(mul(d, splat<E>(gn)), d, sq.e[i]));
                }
            }
        }
        if (clusters > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            float* mine = shared + (4 * groups + parity * 2) * plane;
            if (threadIdx.y == 0) {
                put<V>(mine, lane, sum);
                put<V>(mine + plane, lane, squares);
            }
            cluster.sync();
            sum.fill(0.0f);
            for (int c = 0; c < clusters; ++c) {
                const F s = got<V>(cluster.map_shared_rank(mine, c), lane);
#pragma unroll
                for (int i = 0; i < N; ++i) sum.e[i] = add(sum.e[i], s.e[i]);
            }
            float m[V];
            sum.to(m);
#pragma unroll
            for (int v = 0; v < V; ++v) m[v] = quotient(m[v], static_cast<float>(len), len_inverse);
            mean.from(m);
            squares.fill(0.0f);
            for (int c = 0; c < clusters; ++c) {
                const float* theirs = cluster.map_shared_rank(mine, c);
                const F s = got<V>(theirs, lane), sq = got<V>(theirs + plane, lane);
                const float n = static_cast<float>(
                    max(groups * below.whole + min(max(below.rest - c * groups, 0), groups), 1));
                float ms[V];
                s.to(ms);
#pragma unroll
                for (int v = 0; v < V; ++v) ms[v] = quotient(ms[v], n, 1.0f / n);
                F d;
                d.from(ms);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const E e = sub(d.e[i], mean.e[i]);
                    squares.e[i] = add(squares.e[i], fma(mul(e, splat<E>(n)), e, sq.e[i]));
                }
            }
        }
        if (!live) continue;
        F rstd;
        {
            float m[V], r[V];
            mean.to(m);
            squares.to(r);
#pragma unroll
            for (int v = 0; v < V; ++v) r[v] = root_inverse(fmaf(r[v], len_inverse, a.eps));
            rstd.from(r);
            if (a.mean != nullptr && group == 0) {
                if (a.stats_wide) {
                    put<V>(a.mean + q * V, 0, mean);
                    put<V>(a.rstd + q * V, 0, rstd);
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        a.mean[q * V + v] = m[v];
                        a.rstd[q * V + v] = r[v];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (FULL || group + k * all < len) {
                F out;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    out.e[i] = fma(mul(sub(h[k].e[i], mean.e[i]), rstd.e[i]), splat<E>(w[k]), splat<E>(b[k]));
                P::of(out).store(a.y + first + k * step);
            }
        }
    }
    if (clusters > 1) cg::this_cluster().sync();  // no block leaves while another reads it
}

// A thread adds up its channels' gradients over the tiles that its block (cluster) walks over.  `part` gets
// [gridDim.x][2][len] sums.
template <typename T, int V, int NV, bool JOIN, bool FULL>
__global__ void __launch_bounds__(512, 1) norm_columns_bwd_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    // [2 tiles][2][groups][lanes][V], then for the cluster [2 tiles][2][lanes][V]; at the end two floats a channel and warp
    extern __shared__ __align__(16) float shared[];
    __shared__ PhiloxKeys keys;
    const int lanes = blockDim.x, groups = blockDim.y, lane = threadIdx.x;
    const int clusters = gridDim.y, all = groups * clusters;
    const int group = blockIdx.y * groups + threadIdx.y;
    const int len = a.shape.len, plane = lanes * V;
    const long long step = static_cast<long long>(all) * a.shape.inner;
    const float inverse = 1.0f / static_cast<float>(len);
    const bool stores = a.dx != nullptr || (JOIN && a.dropped != nullptr);
    if (JOIN) share_keys(a.rule, keys);

    float w[NV];
    E dw[NV], db[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = group + k * all;
        w[k] = (FULL || c < len) && a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
        dw[k] = db[k] = splat<E>(0.0f);
    }

    int parity = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x, parity ^= 1) {
        const long long q = t * lanes + lane;
        long long offset;
        const bool live = column_place<V>(a.shape, q, offset);
        const long long first = offset + static_cast<long long>(group) * a.shape.inner;
        P gy[NV], x[NV], extra[JOIN ? NV : 1];
        F mean, rstd, s1, s2;
        s1.fill(0.0f);
        s2.fill(0.0f);
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || group + k * all < len) {
                    gy[k] = P::load(a.gy + first + k * step);
                    x[k] = P::load(a.x + first + k * step);
                }
            }
            if (a.stats_wide) {
                mean = got<V>(a.mean + q * V, 0);
                rstd = got<V>(a.rstd + q * V, 0);
            } else {
                float m[V], r[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    m[v] = a.mean[q * V + v];
                    r[v] = a.rstd[q * V + v];
                }
                mean.from(m);
                rstd.from(r);
            }
            if (JOIN && a.add != nullptr) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    if (FULL || group + k * all < len) extra[k] = P::load(a.add + first + k * step);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || group + k * all < len) {
                    const F g = gy[k].floats(), h = x[k].floats();
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const E gx = mul(g.e[i], mul(sub(h.e[i], mean.e[i]), rstd.e[i]));
                        dw[k] = add(dw[k], gx);
                        db[k] = add(db[k], g.e[i]);
                        s1.e[i] = fma(g.e[i], splat<E>(w[k]), s1.e[i]);
                        s2.e[i] = fma(gx, splat<E>(w[k]), s2.e[i]);
                    }
                }
            }
        }
        if (groups > 1) {
            float* sums = shared + parity * 2 * groups * plane;
            float* sums2 = sums + groups * plane;
            put<V>(sums + threadIdx.y * plane, lane, s1);
            put<V>(sums2 + threadIdx.y * plane, lane, s2);
            __syncthreads();
            s1.fill(0.0f);
            s2.fill(0.0f);
            for (int g = 0; g < groups; ++g) {
                const F p1 = got<V>(sums + g * plane, lane), p2 = got<V>(sums2 + g * plane, lane);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s1.e[i] = add(s1.e[i], p1.e[i]);
                    s2.e[i] = add(s2.e[i], p2.e[i]);
                }
            }
        }
        if (clusters > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            float* mine = shared + (4 * groups + parity * 2) * plane;
            if (threadIdx.y == 0) {
                put<V>(mine, lane, s1);
                put<V>(mine + plane, lane, s2);
            }
            cluster.sync();
            s1.fill(0.0f);
            s2.fill(0.0f);
            for (int c = 0; c < clusters; ++c) {
                const float* theirs = cluster.map_shared_rank(mine, c);
                const F p1 = got<V>(theirs, lane), p2 = got<V>(theirs + plane, lane);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    s1.e[i] = add(s1.e[i], p1.e[i]);
                    s2.e[i] = add(s2.e[i], p2.e[i]);
                }
            }
        }
        if (live && stores) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s1.e[i] = mul(s1.e[i], splat<E>(-inverse));
                s2.e[i] = mul(s2.e[i], splat<E>(-inverse));
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || group + k * all < len) {
                    const F g = gy[k].floats(), h = x[k].floats();
                    F d;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const E xhat = mul(sub(h.e[i], mean.e[i]), rstd.e[i]);
                        d.e[i] = mul(rstd.e[i], fma(xhat, s2.e[i], fma(g.e[i], splat<E>(w[k]), s1.e[i])));
                    }
                    store_dx<T, V, JOIN>(d, first + k * step, a, extra[JOIN ? k : 0], keys);
                }
            }
        }
    }
    if (clusters > 1) cg::this_cluster().sync();  // no block leaves while another reads it
    if (a.part == nullptr) return;
    // the lanes of a warp hold the same channels; a group has several warps
    const int warps = lanes / 32;
    if (warps > 1) __syncthreads();  // the last tile's use of `shared`
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const float sw = warp_sum(total(dw[k])), sb = warp_sum(total(db[k]));
        if ((lane & 31) == 0) {
            if (warps > 1) {
                float* part = shared + ((k * groups + threadIdx.y) * warps + (lane >> 5)) * 2;
                part[0] = sw;
                part[1] = sb;
            } else if (group + k * all < len) {
                a.part[(blockIdx.x * 2ll) * len + group + k * all] = sw;
                a.part[(blockIdx.x * 2ll + 1) * len + group + k * all] = sb;
            }
        }
    }
    if (warps > 1) {
        __syncthreads();
        for (int k = lane; k < NV; k += lanes) {
            if (group + k * all < len) {
                const float* part = shared + (k * groups + threadIdx.y) * warps * 2;
                float sw = 0.0f, sb = 0.0f;
                for (int i = 0; i < warps; ++i) {
                    sw += part[i * 2];
                    sb += part[i * 2 + 1];
                }
                a.part[(blockIdx.x * 2ll) * len + group + k * all] = sw;
                a.part[(blockIdx.x * 2ll + 1) * len + group + k * all] = sb;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// rows
// ------------------------------------------------------------------------------------------------

// Sum over the `width` neighbouring lanes (a power of two up to 32) of a row.
__device__ __forceinline__ float lanes_sum(float v, int width) {
    for (int d = width >> 1; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// blockDim.x threads a row: a power of two up to 32, or whole warps (then blockDim.y is 1).  Each group of threads
// takes R rows at a time, whose loads are in flight together and which share the parameters' loads.
template <typename T, int V, int NV, int R, bool JOIN>
__global__ void __launch_bounds__(512, 1) norm_rows_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    __shared__ float parts[16][R][2], counts[16], block[R][2];
    __shared__ PhiloxKeys keys;
    const int width = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int warps = width > 32 ? width >> 5 : 1;
    const int clusters = gridDim.y, all = width * clusters;
    const int len = a.shape.len, vectors = len / V;  // V divides len
    const int first = blockIdx.y * width + threadIdx.x;
    const float n = static_cast<float>(len), inverse = 1.0f / n;
    const long long row = (blockIdx.x * static_cast<long long>(blockDim.y) + threadIdx.y) * R;
    const long long base = row * len + static_cast<long long>(first) * V;
    if (JOIN) share_keys(a.rule, keys);

    F h[R][NV];
    {
        P in[R][NV], res[JOIN ? R : 1][NV];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (row + r < a.shape.rows && first + k * all < vectors) {
                    const long long e = base + static_cast<long long>(r) * len + k * all * V;
                    in[r][k] = P::load(a.x + e);
                    if (JOIN) res[r][k] = P::load(a.residual + e);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (row + r < a.shape.rows && first + k * all < vectors) {
                    const long long e = base + static_cast<long long>(r) * len + k * all * V;
                    if (JOIN)
                        h[r][k] = join_at<T, V>(in[r][k], res[r][k], e, a.rule, keys, a.sum);
                    else
                        h[r][k] = in[r][k].floats();
                } else {
                    h[r][k].fill(0.0f);
                }
            }
        }
    }

    float mean[R], squares[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        E s = splat<E>(0.0f);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) s = add(s, h[r][k].e[i]);
        mean[r] = total(s);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) mean[r] = lanes_sum(mean[r], min(width, 32));
    const bool whole = warps == 1 && clusters == 1;  // the warp has whole rows: their sums are what the mean is of
    // the warp's elements of a row
    float count = 0.0f, count_inverse = 0.0f;
    if (!whole) {
        int c = 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) c += max(0, min(32, vectors - (first - lane) - k * all));
        count = static_cast<float>(c * V);
        count_inverse = 1.0f / fmaxf(count, 1.0f);
    }
    float sum[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        sum[r] = mean[r];
        mean[r] = whole ? quotient(sum[r], n, inverse) : sum[r] * count_inverse;
        const E m = splat<E>(mean[r]);
        E q = splat<E>(0.0f);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (first + k * all < vectors) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const E d = sub(h[r][k].e[i], m);
                    q = fma(d, d, q);
                }
            }
        }
        squares[r] = total(q);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) squares[r] = lanes_sum(squares[r], min(width, 32));
    if (!whole) {
        if (lane == 0) {
            counts[warp] = count;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                parts[warp][r][0] = sum[r];
                parts[warp][r][1] = squares[r];
            }
        }
        __syncthreads();
        float held = 0.0f;
        for (int i = 0; i < warps; ++i) held += counts[i];
        if (clusters == 1) held = n;
        const float held_inverse = 1.0f / fmaxf(held, 1.0f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sum[r] = squares[r] = 0.0f;
            for (int i = 0; i < warps; ++i) sum[r] += parts[i][r][0];
            mean[r] = quotient(sum[r], held, held_inverse);
        }
        for (int i = 0; i < warps; ++i) {
            const float c = counts[i], c_inverse = 1.0f / fmaxf(c, 1.0f);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float d = parts[i][r][0] * c_inverse - mean[r];
                squares[r] += fmaf(c * d, d, parts[i][r][1]);
            }
        }
    }
    if (clusters > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                block[r][0] = sum[r];
                block[r][1] = squares[r];
            }
        }
        cluster.sync();
#pragma unroll
        for (int r = 0; r < R; ++r) sum[r] = squares[r] = 0.0f;
        for (int c = 0; c < clusters; ++c) {
            const float* theirs = cluster.map_shared_rank(&block[0][0], c);
#pragma unroll
            for (int r = 0; r < R; ++r) sum[r] += theirs[2 * r];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) mean[r] = quotient(sum[r], n, inverse);
        for (int c = 0; c < clusters; ++c) {
            const float* theirs = cluster.map_shared_rank(&block[0][0], c);
            int held = 0;  // what block c has of a row
#pragma unroll
            for (int k = 0; k < NV; ++k) held += max(0, min(width, vectors - c * width - k * all));
            const float cn = fmaxf(static_cast<float>(held) * V, 1.0f), c_inverse = 1.0f / cn;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float d = quotient(theirs[2 * r], cn, c_inverse) - mean[r];
                squares[r] += fmaf(cn * d, d, theirs[2 * r + 1]);
            }
        }
        cluster.sync();  // no block leaves while another reads it
    }
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        rstd[r] = root_inverse(fmaf(squares[r], inverse, a.eps));
        if (a.mean != nullptr && first == 0 && row + r < a.shape.rows) {
            a.mean[row + r] = mean[r];
            a.rstd[row + r] = rstd[r];
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int j = first + k * all;
        if (j < vectors) {
            F w, b;
            w.fill(1.0f);
            b.fill(0.0f);
            if (a.weight) w = load_params<T, V>(a.weight, j * V, a.f32);
            if (a.bias) b = load_params<T, V>(a.bias, j * V, a.f32);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (row + r < a.shape.rows) {
                    F out;
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        out.e[i] = fma(mul(sub(h[r][k].e[i], splat<E>(mean[r])), splat<E>(rstd[r])), w.e[i], b.e[i]);
                    P::of(out).store(a.y + base + static_cast<long long>(r) * len + k * all * V);
                }
            }
        }
    }
}

// The groups of a block walk over tiles of blockDim.y * R rows; a thread adds up its elements' parameter gradients on
// the way.  `part` gets [gridDim.x][2][len] sums, one pair per block (cluster).
template <typename T, int V, int NV, int R, bool JOIN>
__global__ void __launch_bounds__(512, 1) norm_rows_bwd_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    __shared__ float parts[2][16][R][2], block[2][R][2];
    extern __shared__ __align__(16) float sums[];  // [NV][threads][V] where a block has several groups
    __shared__ PhiloxKeys keys;
    const int width = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int warps = width > 32 ? width >> 5 : 1;
    const int clusters = gridDim.y, all = width * clusters;
    const int len = a.shape.len, vectors = len / V;
    const int first = blockIdx.y * width + threadIdx.x;
    const float inverse = 1.0f / static_cast<float>(len);
    const bool stores = a.dx != nullptr || (JOIN && a.dropped != nullptr);
    if (JOIN) share_keys(a.rule, keys);

    F dw[NV], db[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        dw[k].fill(0.0f);
        db[k].fill(0.0f);
    }

    int parity = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x, parity ^= 1) {
        const long long row = (t * blockDim.y + threadIdx.y) * R;
        const long long base = row * len + static_cast<long long>(first) * V;
        P gy[R][NV], x[R][NV], extra[JOIN ? R : 1][NV];
        float mean[R], rstd[R], s1[R], s2[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool live = row + r < a.shape.rows;
            mean[r] = live ? a.mean[row + r] : 0.0f;
            rstd[r] = live ? a.rstd[row + r] : 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (live && first + k * all < vectors) {
                    const long long e = base + static_cast<long long>(r) * len + k * all * V;
                    gy[r][k] = P::load(a.gy + e);
                    x[r][k] = P::load(a.x + e);
                    if (JOIN && a.add != nullptr) extra[r][k] = P::load(a.add + e);
                }
            }
        }
        E p1[R], p2[R];
#pragma unroll
        for (int r = 0; r < R; ++r) p1[r] = p2[r] = splat<E>(0.0f);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = first + k * all;
            if (j < vectors) {
                F w;
                w.fill(1.0f);
                if (a.weight) w = load_params<T, V>(a.weight, j * V, a.f32);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (row + r < a.shape.rows) {
                        const F g = gy[r][k].floats(), h = x[r][k].floats();
#pragma unroll
                        for (int i = 0; i < N; ++i) {
                            const E gx =
                                mul(g.e[i], mul(sub(h.e[i], splat<E>(mean[r])), splat<E>(rstd[r])));
                            dw[k].e[i] = add(dw[k].e[i], gx);
                            db[k].e[i] = add(db[k].e[i], g.e[i]);
                            p1[r] = fma(g.e[i], w.e[i], p1[r]);
                            p2[r] = fma(gx, w.e[i], p2[r]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s1[r] = lanes_sum(total(p1[r]), min(width, 32));
            s2[r] = lanes_sum(total(p2[r]), min(width, 32));
        }
        if (warps > 1) {
            if (lane == 0) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    parts[parity][warp][r][0] = s1[r];
                    parts[parity][warp][r][1] = s2[r];
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < R; ++r) s1[r] = s2[r] = 0.0f;
            for (int i = 0; i < warps; ++i) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    s1[r] += parts[parity][i][r][0];
                    s2[r] += parts[parity][i][r][1];
                }
            }
        }
        if (clusters > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (threadIdx.x == 0) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    block[parity][r][0] = s1[r];
                    block[parity][r][1] = s2[r];
                }
            }
            cluster.sync();
#pragma unroll
            for (int r = 0; r < R; ++r) s1[r] = s2[r] = 0.0f;
            for (int c = 0; c < clusters; ++c) {
                const float* theirs = cluster.map_shared_rank(&block[parity][0][0], c);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    s1[r] += theirs[2 * r];
                    s2[r] += theirs[2 * r + 1];
                }
            }
        }
        if (stores) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = first + k * all;
                if (j < vectors) {
                    F w;
                    w.fill(1.0f);
                    if (a.weight) w = load_params<T, V>(a.weight, j * V, a.f32);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        if (row + r < a.shape.rows) {
                            const E m1 = splat<E>(-s1[r] * inverse), m2 = splat<E>(-s2[r] * inverse);
                            const F g = gy[r][k].floats(), h = x[r][k].floats();
                            F d;
#pragma unroll
                            for (int i = 0; i < N; ++i) {
                                const E xhat = mul(sub(h.e[i], splat<E>(mean[r])), splat<E>(rstd[r]));
                                d.e[i] = mul(splat<E>(rstd[r]), fma(xhat, m2, fma(g.e[i], w.e[i], m1)));
                            }
                            store_dx<T, V, JOIN>(d, base + static_cast<long long>(r) * len + k * all * V, a,
                                                 extra[JOIN ? r : 0][k], keys);
                        }
                    }
                }
            }
        }
    }
    if (clusters > 1) cg::this_cluster().sync();  // no block leaves while another reads it
    if (a.part == nullptr) return;
    const int groups = blockDim.y, threads = width * groups, tid = threadIdx.y * width + threadIdx.x;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = a.part + (blockIdx.x * 2ll + which) * len;
        if (groups == 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = first + k * all;
                if (j < vectors) {
                    float v[V];
                    (which ? db : dw)[k].to(v);
#pragma unroll
                    for (int i = 0; i < V; ++i) out[static_cast<long long>(j) * V + i] = v[i];
                }
            }
        } else {  // several groups, no cluster
            if (which) __syncthreads();
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float v[V];
                (which ? db : dw)[k].to(v);
#pragma unroll
                for (int i = 0; i < V; ++i) sums[(k * V + i) * threads + tid] = v[i];
            }
            __syncthreads();
            for (int l = tid; l < len; l += threads) {
                const int j = l / V, k = j / width;
                const float* from = sums + (k * V + l % V) * threads + (j - k * width);
                float s = 0.0f;
                for (int g = 0; g < groups; ++g) s += from[g * width];
                out[l] = s;
            }
        }
    }
}

}  // namespace serron
