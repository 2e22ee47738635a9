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
// The forward pass adds up a row twice over its registers, for the mean and for the squares about that mean, so that a
// level far above the spread costs nothing; the backward pass adds up two numbers once.  Statistics, sums and
// products are float32; what is stored in 16 bits is rounded once.
//
// What bounds them: the latency of loads and of dependent instructions, with too few warps to hide it.  Registers leave
// room for 14 to 28 warps an SM, which issue in 52 to 68 % of the cycles and wait first for memory (rows, the columns'
// backward pass) or for the previous instruction (columns forward, the join).  Fewer instructions are therefore time won: the memory's rate leaves 16-bit
// elements about 20 each at full issue.  One float at a time the forward pass took 31 an element of a row and 48 of a
// column; computed on in pairs (layer_vec.cuh), with divisions as one multiplication and one correction, it takes 23
// and 15, the backward pass 25 and 24, and the generator adds 22 to 26 in the join.
//   (64,32,256,256) bfloat16, columns: norm 98 us forward (5.5 TB/s, 84 % of the copy rate of 6.55), 165 backward (75 %);
//   join 254 (65 %) and 361 (57 %).  (8192,1024) bfloat16, rows: 10.9 and 21.3 us; join 19.9 and 31.5.
// The join moves four passes where dropout with a residual and the norm after it move five, but its 41 instructions an
// element are more than their 18 and 15: of the columns above it takes 254 us, they take 116 + 98; of (32,64,128,128)
// bfloat16 70 us against 32 + 28.  Of rows it takes what they take: 19.9 us against 10.8 + 10.9, (2048,4096) float16 22.1
// against 10.4 + 13.5.
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

// s / n where `inverse` is 1 / n: a product, corrected by its remainder (Markstein, "Computation of elementary functions on
// the IBM RISC System/6000 processor", IBM J. Res. Dev. 34, 1990), so that it is exact where the quotient is a float.
template <typename E>
__device__ __forceinline__ E quotient(E s, float n, float inverse) {
    const E q = mul(s, splat<E>(inverse));
    return fma(fma(splat<E>(-n), q, s), splat<E>(inverse), q);
}

// 1 / sqrt(v), v >= 0: the approximation and one step of Newton's iteration.  The step has 0 * infinity in it at zero and
// at infinity, where the approximation is exact (infinity and zero): it is taken where v's bits are those of a float between.
// (A comparison of the result with itself took 1 % longer over the columns: 99.5 us against 97.7 at (64,32,256,256) bfloat16.)
__device__ __forceinline__ float root_inverse(float v) {
    const float r = rsqrtf(v);
    const float better = fmaf(r * 0.5f, fmaf(-(v * r), r, 1.0f), r);
    return __float_as_uint(v) - 1u < 0x7f7fffffu ? better : r;
}

// What the kernels are compiled for: the norm alone, or the join with the generator's keys as operands in constant memory
// (a seed from the host) or in shared memory (any seed).  The backward pass of columns always has them in shared
// memory: beside its other registers, operands made it slower (378 us against 361 at (64,32,256,256) bfloat16).
enum Join : int { kNoJoin = 0, kHostSeed = 1, kAnySeed = 2 };

template <int JOIN>
__device__ __forceinline__ const PhiloxKeys& join_keys(const DropRule& rule, PhiloxKeys& shared) {
    if (JOIN != kAnySeed) return rule.keys;
    const int r = threadIdx.y * blockDim.x + threadIdx.x;
    if (r < kPhiloxRounds) {
        // the first round's keys are the seed
        const uint64_t seed = rule.seed_device ? __ldg(rule.seed_device)
                                               : rule.keys.k[0] | static_cast<uint64_t>(rule.keys.k[1]) << 32;
        shared.k[2 * r] = static_cast<uint32_t>(seed) + r * kPhiloxKey0;
        shared.k[2 * r + 1] = static_cast<uint32_t>(seed >> 32) + r * kPhiloxKey1;
    }
    __syncthreads();
    return shared;
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
    return dropped<V>(v, words, rule.threshold, rule.scale32);
}

// residual + dropout(x), rounded to T: it is an output, and the norm (and its backward pass, which reads it back) is of
// that output.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> joined(const Pack<T, V>& x, const Pack<T, V>& residual, long long e,
                                             const DropRule& rule, const PhiloxKeys& keys) {
    Floats<V> v = drop<V>(x.floats(), e, rule, keys);
    const Floats<V> r = residual.floats();
#pragma unroll
    for (int i = 0; i < Floats<V>::N; ++i) v.e[i] = add(v.e[i], r.e[i]);
    return Pack<T, V>::of(v);
}

// V elements at p; of an incomplete vector only those from lo to hi.
template <typename T, int V>
__device__ __forceinline__ void store_part(T* p, const Pack<T, V>& v, bool whole, int lo, int hi) {
    if (whole) {
        v.store(p);
    } else {
        float f[V];
        v.floats().to(f);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i >= lo && i < hi) p[i] = Storage<T>::store(f[i]);
    }
}

// What follows dx = v from element e on: the sum with `extra`, dx itself, and its masked copy.
template <typename T, int V, int JOIN>
__device__ __forceinline__ void store_dx(Floats<V> v, long long e, const NormArgs<T>& a, const Pack<T, V>& extra,
                                         const PhiloxKeys& keys, bool whole = true, int lo = 0, int hi = V) {
    if (JOIN && a.add != nullptr) {
        const Floats<V> f = extra.floats();
#pragma unroll
        for (int i = 0; i < Floats<V>::N; ++i) v.e[i] = add(v.e[i], f.e[i]);
    }
    if (a.dx != nullptr) store_part<T, V>(a.dx + e, Pack<T, V>::of(v), whole, lo, hi);
    if (JOIN && a.dropped != nullptr)
        store_part<T, V>(a.dropped + e, Pack<T, V>::of(drop<V>(v, e, a.rule, keys)), whole, lo, hi);
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

// Brings a thread's strides of the next tile from DRAM to the L2 while the present one is computed on.  The lanes of a warp
// share the lines: kPer lanes' vectors lie in one, and each of those asks for another stride or tensor, at its own
// place in the row.  (16,64,128,128) float32: 25 us forward against 30, 51 backward against 58.  Copies of whole tiles into
// shared memory instead, ahead of their use, cost more instructions than they saved waiting (16-bit: 113 us against 105
// forward, 176 against 165 backward).
template <typename T, int V, int NV>
__device__ __forceinline__ void fetch_ahead(const T* const (&from)[3], int tensors, unsigned step, int count) {
    constexpr int kBytes = V * static_cast<int>(sizeof(T)), kPer = kBytes >= 4 ? 128 / kBytes : 32;
    for (int i = static_cast<int>(threadIdx.x & 31) % kPer; i < tensors * NV; i += kPer) {
        const int m = i / NV, k = i % NV;
        const T* p = (m == 0 ? from[0] : m == 1 ? from[1] : from[2]) + k * step;
        if (k < count) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    }
}

// Sums M numbers for each of a lane's V rows over the groups of a block, then over the blocks of a cluster.  `shared`:
// [2 phases][M][groups][lanes][V], then for the cluster [2 phases][M][lanes][V]; `phase` alternates from call to call, so
// that a call's reads and the next but one's writes have a barrier between them.
template <int V, int M>
__device__ __forceinline__ void column_totals(Floats<V> (&v)[M], float* shared, int& phase) {
    const int lanes = blockDim.x, groups = blockDim.y, lane = threadIdx.x, clusters = gridDim.y, plane = lanes * V;
    if (groups > 1) {
        float* mine = shared + phase * M * groups * plane;
#pragma unroll
        for (int m = 0; m < M; ++m) put<V>(mine + (m * groups + threadIdx.y) * plane, lane, v[m]);
        __syncthreads();
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = got<V>(mine + m * groups * plane, lane);
        for (int g = 1; g < groups; ++g) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const Floats<V> p = got<V>(mine + (m * groups + g) * plane, lane);
#pragma unroll
                for (int i = 0; i < Floats<V>::N; ++i) v[m].e[i] = add(v[m].e[i], p.e[i]);
            }
        }
    }
    if (clusters > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        float* mine = shared + (2 * groups + phase) * M * plane;
        if (threadIdx.y == 0) {
#pragma unroll
            for (int m = 0; m < M; ++m) put<V>(mine + m * plane, lane, v[m]);
        }
        cluster.sync();
#pragma unroll
        for (int m = 0; m < M; ++m) v[m].fill(0.0f);
        for (int c = 0; c < clusters; ++c) {
            const float* theirs = cluster.map_shared_rank(mine, c);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const Floats<V> p = got<V>(theirs + m * plane, lane);
#pragma unroll
                for (int i = 0; i < Floats<V>::N; ++i) v[m].e[i] = add(v[m].e[i], p.e[i]);
            }
        }
    }
    phase ^= 1;
}

// FULL: every thread has all of its NV strides (len is their number times the groups').
// Registers: at 96 (five blocks of 128 threads to an SM) the norm at (64,32,256,256) bfloat16 took 102 us, at 128 110, at 80 106, at
// 64 (spilling) 128; the join 278 at 128 and 318, 331, 402 at 96, 80, 64.
template <typename T, int V, int NV, int JOIN, bool FULL>
__global__ void __maxnreg__(JOIN ? 128 : 96) norm_columns_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    extern __shared__ __align__(16) float shared[];
    __shared__ PhiloxKeys own_keys;
    const int lanes = blockDim.x, lane = threadIdx.x;
    const int clusters = gridDim.y, all = blockDim.y * clusters;
    const int group = blockIdx.y * blockDim.y + threadIdx.y;
    const int len = a.shape.len;
    const unsigned step = static_cast<unsigned>(all) * a.shape.inner;  // a sample's elements are counted in 31 bits here
    const int count = (len - group + all - 1) / all;                    // of this thread's strides
    const float n = static_cast<float>(len), inverse = 1.0f / n;
    const PhiloxKeys& keys = join_keys<JOIN>(a.rule, own_keys);

    float w[NV], b[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = group + k * all;
        w[k] = (FULL || k < count) && a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
        b[k] = (FULL || k < count) && a.bias ? load_param<T>(a.bias, c, a.f32) : 0.0f;
    }

    int phase = 0;
    long long next = 0;  // where the thread's part of the next tile begins
    bool next_live = false;
    const auto look = [&](long long t) {
        next_live = column_place<V>(a.shape, t * lanes + lane, next);
        next += static_cast<long long>(group) * a.shape.inner;
    };
    look(blockIdx.x);
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        const long long q = t * lanes + lane, first = next;
        const bool live = next_live;
        P h[NV];
        F sum[1], squares[1];
        sum[0].fill(0.0f);
        squares[0].fill(0.0f);
        if (live) {
            P res[JOIN ? NV : 1];
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || k < count) {
                    h[k] = P::load(a.x + first + k * step);
                    if (JOIN) res[k] = P::load(a.residual + first + k * step);
                }
            }
            if (t + gridDim.x < a.tiles) {
                look(t + gridDim.x);
                if (next_live)
                    fetch_ahead<T, V, NV>({a.x + next, JOIN ? a.residual + next : nullptr, nullptr}, JOIN ? 2 : 1, step,
                                          count);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || k < count) {
                    if (JOIN) {
                        h[k] = joined<T, V>(h[k], res[k], first + k * step, a.rule, keys);
                        h[k].store(a.sum + first + k * step);
                    }
                    const F f = h[k].floats();
#pragma unroll
                    for (int i = 0; i < N; ++i) sum[0].e[i] = add(sum[0].e[i], f.e[i]);
                }
            }
        }
        column_totals<V, 1>(sum, shared, phase);
        F mean;
#pragma unroll
        for (int i = 0; i < N; ++i) mean.e[i] = quotient(sum[0].e[i], n, inverse);
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || k < count) {
                    const F f = h[k].floats();
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const E d = sub(f.e[i], mean.e[i]);
                        squares[0].e[i] = fma(d, d, squares[0].e[i]);
                    }
                }
            }
        }
        column_totals<V, 1>(squares, shared, phase);
        if (!live) continue;
        F rstd;
        float r[V];
        squares[0].to(r);
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = root_inverse(fmaf(r[v], inverse, a.eps));
        rstd.from(r);
        if (a.mean != nullptr && group == 0) {
            if (a.stats_wide) {
                put<V>(a.mean + q * V, 0, mean);
                put<V>(a.rstd + q * V, 0, rstd);
            } else {
                float m[V];
                mean.to(m);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    a.mean[q * V + v] = m[v];
                    a.rstd[q * V + v] = r[v];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (FULL || k < count) {
                const F f = h[k].floats();
                F out;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    out.e[i] = fma(mul(sub(f.e[i], mean.e[i]), rstd.e[i]), splat<E>(w[k]), splat<E>(b[k]));
                P::of(out).store(a.y + first + k * step);
            }
        }
    }
    if (clusters > 1) cg::this_cluster().sync();  // no block leaves while another reads it
}

// A thread adds up its channels' gradients over the tiles that its block (cluster) walks over.  `part` gets
// [gridDim.x][2][len] sums.  Four blocks of 128 threads to an SM hide more than what fewer registers spill: 167 us at 128
// registers, 174, 227, 292 at 112, 96, 80, and 246 with 144 (three blocks).
template <typename T, int V, int NV, int JOIN, bool FULL>
__global__ void __maxnreg__(128) norm_columns_bwd_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    extern __shared__ __align__(16) float shared[];  // column_totals'; at the end two floats a channel and warp
    __shared__ PhiloxKeys own_keys;
    const int lanes = blockDim.x, groups = blockDim.y, lane = threadIdx.x;
    const int clusters = gridDim.y, all = groups * clusters;
    const int group = blockIdx.y * groups + threadIdx.y;
    const int len = a.shape.len;
    const unsigned step = static_cast<unsigned>(all) * a.shape.inner;  // a sample's elements are counted in 31 bits here
    const int count = (len - group + all - 1) / all;                    // of this thread's strides
    const float inverse = 1.0f / static_cast<float>(len);
    const bool stores = a.dx != nullptr || (JOIN && a.dropped != nullptr);
    const PhiloxKeys& keys = join_keys<JOIN>(a.rule, own_keys);

    float w[NV];
    E dw[NV], db[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = group + k * all;
        w[k] = (FULL || k < count) && a.weight ? load_param<T>(a.weight, c, a.f32) : 1.0f;
        dw[k] = db[k] = splat<E>(0.0f);
    }

    // the join of 16-bit vectors has no registers left for the next tile's place: 361 us at (64,32,256,256) bfloat16, 372
    // with it
    constexpr bool kFetch = !(JOIN && sizeof(T) == 2 && V > 1);
    int phase = 0;
    long long next = 0;  // where the thread's part of the next tile begins
    bool next_live = false;
    const auto look = [&](long long t) {
        next_live = column_place<V>(a.shape, t * lanes + lane, next);
        next += static_cast<long long>(group) * a.shape.inner;
    };
    if (kFetch) look(blockIdx.x);
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        if (!kFetch) look(t);
        const long long q = t * lanes + lane, first = next;
        const bool live = next_live;
        P gy[NV], x[NV], extra[JOIN ? NV : 1];
        F mean, rstd, s[2];
        s[0].fill(0.0f);
        s[1].fill(0.0f);
        if (live) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || k < count) {
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
                    if (FULL || k < count) extra[k] = P::load(a.add + first + k * step);
            }
            if (kFetch && t + gridDim.x < a.tiles) {
                look(t + gridDim.x);
                if (next_live)
                    fetch_ahead<T, V, NV>({a.gy + next, a.x + next, JOIN ? a.add + next : nullptr},
                                          JOIN && a.add != nullptr ? 3 : 2, step, count);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || k < count) {
                    const F g = gy[k].floats(), h = x[k].floats();
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const E gx = mul(g.e[i], mul(sub(h.e[i], mean.e[i]), rstd.e[i]));
                        dw[k] = add(dw[k], gx);
                        db[k] = add(db[k], g.e[i]);
                        s[0].e[i] = fma(g.e[i], splat<E>(w[k]), s[0].e[i]);
                        s[1].e[i] = fma(gx, splat<E>(w[k]), s[1].e[i]);
                    }
                }
            }
        }
        column_totals<V, 2>(s, shared, phase);
        if (live && stores) {
            // dx = rstd (g w - mean(g w) - xhat mean(g w xhat)), with xhat's rstd multiplied into the mean, which is the same
            // for a row; rstd^2 would leave float32's range for rows of tiny spread, whose dx does not
            F scale, shift;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                shift.e[i] = mul(s[0].e[i], splat<E>(-inverse));
                scale.e[i] = mul(mul(s[1].e[i], splat<E>(-inverse)), rstd.e[i]);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (FULL || k < count) {
                    const F g = gy[k].floats(), h = x[k].floats();
                    F d;
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        d.e[i] = mul(fma(sub(h.e[i], mean.e[i]), scale.e[i], fma(g.e[i], splat<E>(w[k]), shift.e[i])),
                                     rstd.e[i]);
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
            } else if (k < count) {
                a.part[(blockIdx.x * 2ll) * len + group + k * all] = sw;
                a.part[(blockIdx.x * 2ll + 1) * len + group + k * all] = sb;
            }
        }
    }
    if (warps > 1) {
        __syncthreads();
        for (int k = lane; k < NV; k += lanes) {
            if (k < count) {
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
//
// blockDim.x threads a row: a power of two up to 32, or whole warps (then blockDim.y is 1).  Each group of threads takes
// R rows at a time, whose loads are in flight together.
//
// Where V does not divide len (SHIFTED), vectors are laid over the memory and not over the row: the row's first
// element is number `shift` of its first vector, and the first and the last vector hold elements of other rows, which
// are put aside.  `shift` is the row's number times len, mod V, so a block takes rows that are V apart: they all have
// the same, and a thread keeps the same elements of every row.
// ------------------------------------------------------------------------------------------------

// Sums M numbers over the threads of a row: of a warp or a part of it, of a block, of a cluster.  Two phases, as above.
template <int M>
struct RowScratch {
    float warps[2][16][M], block[2][M];
};
template <int M>
__device__ __forceinline__ void row_totals(float (&v)[M], RowScratch<M>& scratch, int& phase) {
    const int width = blockDim.x, clusters = gridDim.y;
    if (width >= 32) {
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = warp_sum(v[m]);
    } else {
        for (int d = width >> 1; d > 0; d >>= 1) {
#pragma unroll
            for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(0xffffffffu, v[m], d);
        }
    }
    if (width > 32) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int m = 0; m < M; ++m) scratch.warps[phase][threadIdx.x >> 5][m] = v[m];
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = scratch.warps[phase][0][m];
        for (int i = 1; i < width >> 5; ++i) {
#pragma unroll
            for (int m = 0; m < M; ++m) v[m] += scratch.warps[phase][i][m];
        }
    }
    if (clusters > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int m = 0; m < M; ++m) scratch.block[phase][m] = v[m];
        }
        cluster.sync();
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = 0.0f;
        for (int c = 0; c < clusters; ++c) {
            const float* theirs = cluster.map_shared_rank(scratch.block[phase], c);
#pragma unroll
            for (int m = 0; m < M; ++m) v[m] += theirs[m];
        }
    }
    phase ^= 1;
}

// Where a thread of a row kernel stands: its vectors are first, first + all, ...
template <int V, bool SHIFTED>
struct RowPlace {
    int shift, vectors, first, all, len;

    __device__ __forceinline__ explicit RowPlace(const NormShape& s) {
        len = s.len;
        shift = SHIFTED ? static_cast<int>(static_cast<long long>(blockIdx.x % V) * len % V) : 0;
        vectors = SHIFTED ? (len + shift + V - 1) / V : len / V;
        all = blockDim.x * gridDim.y;
        first = blockIdx.y * blockDim.x + threadIdx.x;
    }
    // the first row of tile t that this thread's group takes; the others are kStep apart
    static constexpr int kStep = SHIFTED ? V : 1;
    __device__ __forceinline__ long long row(long long t, int R) const {
        if (!SHIFTED) return (t * blockDim.y + threadIdx.y) * R;
        return t % V + (t / V * blockDim.y + threadIdx.y) * static_cast<long long>(R * V);
    }
    // the first element of the thread's first vector of a row in memory
    __device__ __forceinline__ long long at(long long row) const {
        return row * len + (static_cast<long long>(first) * V - shift);
    }
    __device__ __forceinline__ int lo(int j) const { return SHIFTED && j == 0 ? shift : 0; }
    __device__ __forceinline__ int hi(int j) const {
        return SHIFTED && j == vectors - 1 ? len + shift - j * V : V;
    }
    __device__ __forceinline__ bool whole(int j) const {
        return !SHIFTED || ((j > 0 || shift == 0) && len + shift - j * V >= V);
    }
    // the parameters of vector j's elements; `fill` beside the row
    template <typename T>
    __device__ __forceinline__ Floats<V> params(const void* p, int j, bool f32, float fill) const {
        Floats<V> out;
        if (p == nullptr) {
            out.fill(fill);
        } else if (!SHIFTED) {
            out = load_params<T, V>(p, j * V, f32);
        } else {
            // aligned groups of a vector's width, from which the vector is cut at `off`, the same place for all threads
            const int from = j * V - shift, off = (V - shift) % V;
            float f[2 * V];
            if (from >= 0 && from - off + 2 * V <= len) {
                const Floats<V> a = load_params<T, V>(p, from - off, f32), b = load_params<T, V>(p, from - off + V, f32);
                float parts[V];
                a.to(parts);
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = parts[i];
                b.to(parts);
#pragma unroll
                for (int i = 0; i < V; ++i) f[V + i] = parts[i];
                // by one, two and four places where off has that bit
#pragma unroll
                for (int bit = 1; bit < V; bit *= 2) {
                    if (off & bit) {
#pragma unroll
                        for (int i = 0; i < 2 * V - bit; ++i) f[i] = f[i + bit];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    f[i] = from + i >= 0 && from + i < len ? load_param<T>(p, from + i, f32) : fill;
            }
            float cut[V];
#pragma unroll
            for (int i = 0; i < V; ++i) cut[i] = f[i];
            out.from(cut);
        }
        return out;
    }
};

// An incomplete vector with zeros in the place of other rows' elements, before lo and from hi on.  `inside`: it lies in the tensor
// and was read as a whole (all but the tensor's last are); else its own elements are read now, one by one.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> trimmed(const Pack<T, V>& v, const T* p, bool inside, int lo, int hi) {
    float f[V];
    v.floats().to(f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (!inside) f[i] = i < hi ? Storage<T>::load(p[i]) : 0.0f;
        f[i] = i >= lo && i < hi ? f[i] : 0.0f;
    }
    Floats<V> out;
    out.from(f);
    return Pack<T, V>::of(out);
}

// Registers: 64 for whole vectors (11.1 us at (8192,1024) bfloat16; at 80, 96, 128 12.2, 12.1, 12.4), 80 in the join, which at 64
// is slower for short rows (200,000 of 64: 33 us against 30); 32 more where vectors are shifted, of which the kernels of
// four 16-bit vectors a thread still spill (76 to 92 bytes).  Swept in bfloat16; float32 and single elements take the same.
template <typename T, int V, int NV, int R, int JOIN, bool SHIFTED>
__global__ void __maxnreg__((JOIN ? 80 : 64) + (SHIFTED ? 32 : 0))
    norm_rows_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    constexpr bool kKeepParams = SHIFTED && NV <= 2;  // unaligned parameters are read once
    __shared__ RowScratch<R> scratch;
    __shared__ PhiloxKeys own_keys;
    const RowPlace<V, SHIFTED> place(a.shape);
    const float n = static_cast<float>(place.len), inverse = 1.0f / n;
    const long long row_step = static_cast<long long>(place.len) * place.kStep, numel = a.shape.rows * place.len;
    const PhiloxKeys& keys = join_keys<JOIN>(a.rule, own_keys);
    F w[NV], b[NV];
    if (kKeepParams) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            w[k] = place.template params<T>(a.weight, place.first + k * place.all, a.f32, 1.0f);
            b[k] = place.template params<T>(a.bias, place.first + k * place.all, a.f32, 0.0f);
        }
    }

    int phase = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        P h[R][NV];
        float sum[R], squares[R], mean[R], rstd[R];
        const long long row0 = place.row(t, R), base = place.at(row0);
        const int rows =
            static_cast<int>(min((a.shape.rows - row0 + place.kStep - 1) / place.kStep, static_cast<long long>(R)));
        {
            P res[JOIN ? R : 1][NV];
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int j = place.first + k * place.all;
                    if (r < rows && j < place.vectors) {
                        const long long e = base + r * row_step + k * place.all * V;
                        if (!SHIFTED || e + V <= numel) {
                            h[r][k] = P::load(a.x + e);
                            if (JOIN) res[r][k] = P::load(a.residual + e);
                        }
                    }
                }
            }
            if (SHIFTED) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
                        const int j = place.first + k * place.all;
                        if (r < rows && j < place.vectors && !place.whole(j)) {
                            const long long e = base + r * row_step + k * place.all * V;
                            const bool inside = e + V <= numel;
                            h[r][k] = trimmed<T, V>(h[r][k], a.x + e, inside, place.lo(j), place.hi(j));
                            if (JOIN)
                                res[r][k] = trimmed<T, V>(res[r][k], a.residual + e, inside, place.lo(j), place.hi(j));
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                E s = splat<E>(0.0f);
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int j = place.first + k * place.all;
                    if (r < rows && j < place.vectors) {
                        if (JOIN) {  // beside the row: dropout and sum of zeros
                            const long long e = base + r * row_step + k * place.all * V;
                            h[r][k] = joined<T, V>(h[r][k], res[r][k], e, a.rule, keys);
                            store_part<T, V>(a.sum + e, h[r][k], place.whole(j), place.lo(j), place.hi(j));
                        }
                        const F f = h[r][k].floats();
#pragma unroll
                        for (int i = 0; i < N; ++i) s = add(s, f.e[i]);
                    }
                }
                sum[r] = total(s);
            }
        }
        row_totals<R>(sum, scratch, phase);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mean[r] = quotient(sum[r], n, inverse);
            E s = splat<E>(0.0f);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = place.first + k * place.all;
                if (r < rows && j < place.vectors) {
                    F f = h[r][k].floats();
#pragma unroll
                    for (int i = 0; i < N; ++i) f.e[i] = sub(f.e[i], splat<E>(mean[r]));
                    if (SHIFTED && !place.whole(j)) {
                        float d[V];
                        f.to(d);
                        const int lo = place.lo(j), hi = place.hi(j);
#pragma unroll
                        for (int i = 0; i < V; ++i) d[i] = i >= lo && i < hi ? d[i] : 0.0f;
                        f.from(d);
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) s = fma(f.e[i], f.e[i], s);
                }
            }
            squares[r] = total(s);
        }
        row_totals<R>(squares, scratch, phase);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            rstd[r] = root_inverse(fmaf(squares[r], inverse, a.eps));
            if (a.mean != nullptr && place.first == 0 && r < rows) {
                a.mean[row0 + r * place.kStep] = mean[r];
                a.rstd[row0 + r * place.kStep] = rstd[r];
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = place.first + k * place.all;
            if (j < place.vectors) {
                const F wk = kKeepParams ? w[k] : place.template params<T>(a.weight, j, a.f32, 1.0f);
                const F bk = kKeepParams ? b[k] : place.template params<T>(a.bias, j, a.f32, 0.0f);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < rows) {
                        const F f = h[r][k].floats();
                        F out;
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            out.e[i] = fma(mul(sub(f.e[i], splat<E>(mean[r])), splat<E>(rstd[r])), wk.e[i], bk.e[i]);
                        store_part<T, V>(a.y + base + r * row_step + k * place.all * V, P::of(out), place.whole(j),
                                         place.lo(j), place.hi(j));
                    }
                }
            }
        }
    }
    if (gridDim.y > 1) cg::this_cluster().sync();  // no block leaves while another reads it
}

// `part` gets [gridDim.x][2][len] sums of the parameters' gradients, one pair per block (cluster).  Registers: 22 us at
// (8192,1024) bfloat16 with 128; 25, 27, 34 with 96, 80, 64.
template <typename T, int V, int NV, int R, int JOIN, bool SHIFTED>
__global__ void __maxnreg__(128) norm_rows_bwd_kernel(const __grid_constant__ NormArgs<T> a) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    using E = typename F::E;
    constexpr int N = F::N;
    constexpr bool kKeepParams = SHIFTED && NV <= 2;
    __shared__ RowScratch<2 * R> scratch;
    extern __shared__ __align__(16) float sums[];  // [NV][V][threads] where a block has several groups
    __shared__ PhiloxKeys own_keys;
    const RowPlace<V, SHIFTED> place(a.shape);
    const float inverse = 1.0f / static_cast<float>(place.len);
    const long long row_step = static_cast<long long>(place.len) * place.kStep, numel = a.shape.rows * place.len;
    const bool stores = a.dx != nullptr || (JOIN && a.dropped != nullptr);
    const PhiloxKeys& keys = join_keys<JOIN>(a.rule, own_keys);

    F dw[NV], db[NV], w[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        dw[k].fill(0.0f);
        db[k].fill(0.0f);
        if (kKeepParams) w[k] = place.template params<T>(a.weight, place.first + k * place.all, a.f32, 1.0f);
    }

    int phase = 0;
    for (long long t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        P gy[R][NV], x[R][NV], extra[JOIN ? R : 1][NV];
        float mean[R], rstd[R], s[2 * R];
        const long long row0 = place.row(t, R), base = place.at(row0);
        const int rows =
            static_cast<int>(min((a.shape.rows - row0 + place.kStep - 1) / place.kStep, static_cast<long long>(R)));
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool live = r < rows;
            mean[r] = live ? a.mean[row0 + r * place.kStep] : 0.0f;
            rstd[r] = live ? a.rstd[row0 + r * place.kStep] : 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = place.first + k * place.all;
                const long long e = base + r * row_step + k * place.all * V;
                if (live && j < place.vectors && (!SHIFTED || e + V <= numel)) {
                    gy[r][k] = P::load(a.gy + e);
                    x[r][k] = P::load(a.x + e);
                    if (JOIN && a.add != nullptr) extra[r][k] = P::load(a.add + e);
                }
            }
        }
        if (SHIFTED) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int j = place.first + k * place.all;
                    if (r < rows && j < place.vectors && !place.whole(j)) {
                        const long long e = base + r * row_step + k * place.all * V;
                        const bool inside = e + V <= numel;
                        const int lo = place.lo(j), hi = place.hi(j);
                        gy[r][k] = trimmed<T, V>(gy[r][k], a.gy + e, inside, lo, hi);
                        x[r][k] = trimmed<T, V>(x[r][k], a.x + e, inside, lo, hi);
                        if (JOIN && a.add != nullptr)
                            extra[r][k] = trimmed<T, V>(extra[r][k], a.add + e, inside, lo, hi);
                    }
                }
            }
        }
        if (t + gridDim.x < a.tiles) {
            // the next tile from DRAM to the L2: eight lanes' vectors lie in a line, each asks for another one's
            constexpr int kPer = V * sizeof(T) == 16 ? 8 : 32;
            const long long ahead = place.row(t + gridDim.x, R);
            for (int i = threadIdx.x % kPer; i < 2 * R * NV; i += kPer) {
                const int r = i / NV % R, j = place.first + i % NV * place.all;
                const long long row = ahead + r * place.kStep;
                const T* p = (i < R * NV ? a.gy : a.x) + place.at(ahead) + r * row_step + i % NV * place.all * V;
                if (row < a.shape.rows && j < place.vectors) asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
            }
        }
        E p1[R], p2[R];
#pragma unroll
        for (int r = 0; r < R; ++r) p1[r] = p2[r] = splat<E>(0.0f);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = place.first + k * place.all;
            if (j < place.vectors) {
                const F wk = kKeepParams ? w[k] : place.template params<T>(a.weight, j, a.f32, 1.0f);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < rows) {
                        const F g = gy[r][k].floats(), h = x[r][k].floats();
#pragma unroll
                        for (int i = 0; i < N; ++i) {  // beside the row g is zero
                            const E gx = mul(g.e[i], mul(sub(h.e[i], splat<E>(mean[r])), splat<E>(rstd[r])));
                            dw[k].e[i] = add(dw[k].e[i], gx);
                            db[k].e[i] = add(db[k].e[i], g.e[i]);
                            p1[r] = fma(g.e[i], wk.e[i], p1[r]);
                            p2[r] = fma(gx, wk.e[i], p2[r]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[2 * r] = total(p1[r]);
            s[2 * r + 1] = total(p2[r]);
        }
        row_totals<2 * R>(s, scratch, phase);
        if (stores) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = place.first + k * place.all;
                if (j < place.vectors) {
                    const F wk = kKeepParams ? w[k] : place.template params<T>(a.weight, j, a.f32, 1.0f);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        if (r < rows) {
                            const E shift = splat<E>(-s[2 * r] * inverse);
                            const E scale = splat<E>(-s[2 * r + 1] * inverse * rstd[r]);
                            const F g = gy[r][k].floats(), h = x[r][k].floats();
                            F d;
#pragma unroll
                            for (int i = 0; i < N; ++i)
                                d.e[i] = mul(fma(sub(h.e[i], splat<E>(mean[r])), scale, fma(g.e[i], wk.e[i], shift)),
                                             splat<E>(rstd[r]));
                            store_dx<T, V, JOIN>(d, base + r * row_step + k * place.all * V, a, extra[JOIN ? r : 0][k],
                                                 keys, place.whole(j), place.lo(j), place.hi(j));
                        }
                    }
                }
            }
        }
    }
    if (gridDim.y > 1) cg::this_cluster().sync();  // no block leaves while another reads it
    if (a.part == nullptr) return;
    const int len = place.len, width = blockDim.x, groups = blockDim.y;
    const int threads = width * groups, tid = threadIdx.y * width + threadIdx.x;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = a.part + (blockIdx.x * 2ll + which) * len;
        if (groups == 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int j = place.first + k * place.all;
                if (j < place.vectors) {
                    const int lo = place.lo(j), hi = place.hi(j);
                    float v[V];
                    (which ? db : dw)[k].to(v);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (!SHIFTED || (i >= lo && i < hi)) out[static_cast<long long>(j) * V + i - place.shift] = v[i];
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
                const int p = l + place.shift, j = p / V, k = j / width;
                const float* from = sums + (k * V + p % V) * threads + (j - k * width);
                float sum = 0.0f;
                for (int g = 0; g < groups; ++g) sum += from[g * width];
                out[l] = sum;
            }
        }
    }
}

}  // namespace serron
