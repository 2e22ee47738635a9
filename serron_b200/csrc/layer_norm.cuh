// Layer norm over one dimension of a dense tensor seen as (outer, len, inner): row r = (o, i) holds the len elements
// x[o, :, i], `inner` apart.
//
//   mean = sum x / len,  rstd = 1 / sqrt(sum (x - mean)^2 / len + eps),  xhat = (x - mean) * rstd
//   forward    y = xhat * w + b
//   backward   g = gy * w,  dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),
//              dw = sum over rows of gy * xhat,  db = sum over rows of gy
//
// Statistics and sums are float32 (double for double) whatever the storage type.
#pragma once

#include "layer_common.cuh"

namespace serron {

struct NormShape {
    long long rows = 0;  // outer * inner
    int len = 0, inner = 1;

    // first element of row r; its elements are `inner` apart
    __device__ __forceinline__ long long base(long long r) const {
        return inner == 1 ? r * len : (r / inner) * static_cast<long long>(len) * inner + r % inner;
    }
};

// ------------------------------------------------------------------------------------------------
// kernels for any length and layout: rows are cut into chunks of `chunk` elements, each block reduces one chunk of
// one row (inner == 1: 256 threads along the row) or of 32 neighbouring rows (inner > 1: 32 x 8 threads, neighbouring
// rows being neighbours in memory), and the chunks' results are joined where they are used.
//
// Bound by loads of single elements, and by reading x three times (twice from DRAM where a chunk stays in the caches) and in
// a backward pass gy and x three times.  Forward and backward, of the copy rate: (16,32,256,256) float64 205 and 448 us (40
// and 27 %), (8192,1024) float64 47 and 124 us (44 and 25 %), (400,70000) bfloat16 70 and 168 us (24 and 15 %),
// (16,2100,32,32) bfloat16 106 and 251 us (20 and 13 %).
// ------------------------------------------------------------------------------------------------
constexpr int kNormThreads = 256;

// Block-wide sum over the threads of one row: all 256 of a block (ROWS), or the 8 of a column of 32 x 8.
template <bool ROWS, typename A>
__device__ __forceinline__ A row_sum(A v, A* shared) {
    const int t = threadIdx.x;
    __syncthreads();  // the last use of `shared`
    if (ROWS) {
        v = warp_sum(v);
        if ((t & 31) == 0) shared[t >> 5] = v;
        __syncthreads();
        A s = A(0);
        for (int w = 0; w < kNormThreads / 32; ++w) s += shared[w];
        return s;
    }
    shared[t] = v;
    __syncthreads();
    A s = A(0);
    for (int w = 0; w < kNormThreads / 32; ++w) s += shared[w * 32 + (t & 31)];
    return s;
}

// What a thread of the chunk kernels works on: elements first, first + step, ... below `end` of a row.  A row may have
// 2^31 - 1 elements, and the index that leaves the loop lies up to `step` beyond them.
struct ChunkPlace {
    long long row, offset;
    unsigned first, step, end;
    bool live;
};
template <bool ROWS>
__device__ __forceinline__ ChunkPlace chunk_place(const NormShape& s, int chunk, int split) {
    ChunkPlace p;
    p.row = ROWS ? static_cast<long long>(blockIdx.x) : blockIdx.x * 32ll + (threadIdx.x & 31);
    p.live = p.row < s.rows;
    p.offset = p.live ? s.base(p.row) : 0;
    const long long begin = static_cast<long long>(split) * chunk;
    p.end = p.live ? static_cast<unsigned>(min(begin + chunk, static_cast<long long>(s.len))) : 0u;
    p.first = static_cast<unsigned>(begin) + (ROWS ? threadIdx.x : threadIdx.x >> 5);
    p.step = ROWS ? kNormThreads : kNormThreads / 32;
    return p;
}

// Mean and sum of squared deviations of each chunk (two passes over it, the second from the caches).
template <typename T, bool ROWS>
__global__ void __launch_bounds__(kNormThreads)
    norm_stats_kernel(const T* __restrict__ x, typename Storage<T>::acc* __restrict__ part, NormShape s, int chunk) {
    using S = Storage<T>;
    using A = typename S::acc;
    __shared__ A shared[kNormThreads];
    const int split = blockIdx.y;
    const ChunkPlace p = chunk_place<ROWS>(s, chunk, split);
    const int count = min(chunk, s.len - split * chunk);
    A sum = A(0);
    for (unsigned l = p.first; l < p.end; l += p.step) sum += S::load(x[p.offset + static_cast<long long>(l) * s.inner]);
    const A mean = row_sum<ROWS>(sum, shared) / A(count);
    A m2 = A(0);
    for (unsigned l = p.first; l < p.end; l += p.step) {
        const A d = S::load(x[p.offset + static_cast<long long>(l) * s.inner]) - mean;
        m2 += d * d;
    }
    m2 = row_sum<ROWS>(m2, shared);
    if (p.live && (ROWS ? threadIdx.x == 0 : threadIdx.x < 32)) {
        part[(p.row * gridDim.y + split) * 2] = mean;
        part[(p.row * gridDim.y + split) * 2 + 1] = m2;
    }
}

// Joins the chunks of each row: with count n, mean m and sum of squares q of two parts,
// m = m1 + (m2 - m1) n2 / n and q = q1 + q2 + (m2 - m1)^2 n1 n2 / n.
template <typename A>
__global__ void norm_join_kernel(const A* __restrict__ part, A* __restrict__ mean_out, A* __restrict__ rstd_out,
                                 NormShape s, int chunk, int splits, double eps) {
    const long long row = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (row >= s.rows) return;
    A mean = part[row * splits * 2], m2 = part[row * splits * 2 + 1], n = A(min(chunk, s.len));
    for (int k = 1; k < splits; ++k) {
        const A count = A(min(chunk, s.len - k * chunk));
        const A d = part[(row * splits + k) * 2] - mean;
        const A total = n + count;
        mean += d * (count / total);
        m2 += part[(row * splits + k) * 2 + 1] + d * d * (n * (count / total));
        n = total;
    }
    mean_out[row] = mean;
    rstd_out[row] = inverse_root<A>(m2 / A(s.len) + A(eps));
}

template <typename T, bool ROWS>
__global__ void __launch_bounds__(kNormThreads)
    norm_apply_kernel(const T* __restrict__ x, const typename Storage<T>::acc* __restrict__ mean,
                      const typename Storage<T>::acc* __restrict__ rstd, const void* __restrict__ weight,
                      const void* __restrict__ bias, bool f32, T* __restrict__ y, NormShape s, int chunk) {
    using S = Storage<T>;
    using A = typename S::acc;
    const ChunkPlace p = chunk_place<ROWS>(s, chunk, blockIdx.y);
    if (!p.live) return;
    const A m = mean[p.row], r = rstd[p.row];
    for (unsigned l = p.first; l < p.end; l += p.step) {
        const long long e = p.offset + static_cast<long long>(l) * s.inner;
        A v = (S::load(x[e]) - m) * r;
        if (weight) v *= load_param<T>(weight, l, f32);
        if (bias) v += load_param<T>(bias, l, f32);
        y[e] = S::store(v);
    }
}

// Sums of g and g * xhat of each chunk.
template <typename T, bool ROWS>
__global__ void __launch_bounds__(kNormThreads)
    norm_bwd_sums_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                         const typename Storage<T>::acc* __restrict__ mean,
                         const typename Storage<T>::acc* __restrict__ rstd, const void* __restrict__ weight, bool f32,
                         typename Storage<T>::acc* __restrict__ part, NormShape s, int chunk) {
    using S = Storage<T>;
    using A = typename S::acc;
    __shared__ A shared[kNormThreads];
    const ChunkPlace p = chunk_place<ROWS>(s, chunk, blockIdx.y);
    const A m = p.live ? mean[p.row] : A(0), r = p.live ? rstd[p.row] : A(0);
    A s1 = A(0), s2 = A(0);
    for (unsigned l = p.first; l < p.end; l += p.step) {
        const long long e = p.offset + static_cast<long long>(l) * s.inner;
        A g = S::load(gy[e]);
        if (weight) g *= load_param<T>(weight, l, f32);
        s1 += g;
        s2 += g * ((S::load(x[e]) - m) * r);
    }
    s1 = row_sum<ROWS>(s1, shared);
    s2 = row_sum<ROWS>(s2, shared);
    if (p.live && (ROWS ? threadIdx.x == 0 : threadIdx.x < 32)) {
        part[(p.row * gridDim.y + blockIdx.y) * 2] = s1;
        part[(p.row * gridDim.y + blockIdx.y) * 2 + 1] = s2;
    }
}

// dx (plus `add`, the gradient that reaches x by another way), and for the join its masked copy `dropped`.
template <typename T, bool ROWS>
__global__ void __launch_bounds__(kNormThreads)
    norm_bwd_apply_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                          const typename Storage<T>::acc* __restrict__ mean,
                          const typename Storage<T>::acc* __restrict__ rstd, const void* __restrict__ weight, bool f32,
                          const typename Storage<T>::acc* __restrict__ part, const T* __restrict__ add,
                          T* __restrict__ dx, T* __restrict__ dropped, DropRule rule, NormShape s, int chunk) {
    using S = Storage<T>;
    using A = typename S::acc;
    const ChunkPlace p = chunk_place<ROWS>(s, chunk, blockIdx.y);
    if (!p.live) return;
    A s1 = A(0), s2 = A(0);
    for (int k = 0; k < static_cast<int>(gridDim.y); ++k) {
        s1 += part[(p.row * gridDim.y + k) * 2];
        s2 += part[(p.row * gridDim.y + k) * 2 + 1];
    }
    s1 /= A(s.len);
    s2 /= A(s.len);
    const A m = mean[p.row], r = rstd[p.row];
    for (unsigned l = p.first; l < p.end; l += p.step) {
        const long long e = p.offset + static_cast<long long>(l) * s.inner;
        A g = S::load(gy[e]);
        if (weight) g *= load_param<T>(weight, l, f32);
        A v = r * (g - s1 - ((S::load(x[e]) - m) * r) * s2);
        if (add) v += S::load(add[e]);
        if (dx) dx[e] = S::store(v);
        if (dropped) {
            const bool kept =
                word_of(philox(e >> 2, rule.sequence, rule.own_keys()), e & 3) >= rule.threshold && !rule.all;
            dropped[e] = S::store(kept ? scaled<A>(v, A(rule.scale)) : A(0));
        }
    }
}

// ------------------------------------------------------------------------------------------------
// gradients of weight and bias: sums over rows, first of `rows_per` rows each in A, then of those in double, each in
// an order that the sizes set
// ------------------------------------------------------------------------------------------------

// inner == 1: a thread owns an element of the row and walks down rows_per rows.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
    norm_param_rows_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                           const typename Storage<T>::acc* __restrict__ mean,
                           const typename Storage<T>::acc* __restrict__ rstd,
                           typename Storage<T>::acc* __restrict__ part, NormShape s, int rows_per, int tiles) {
    using S = Storage<T>;
    using A = typename S::acc;
    const long long block = blockIdx.x / tiles;
    const int l = static_cast<int>(blockIdx.x % tiles) * kNormThreads + threadIdx.x;
    if (l >= s.len) return;
    const long long first = block * rows_per, end = min(first + rows_per, s.rows);
    A dw = A(0), db = A(0);
    for (long long r = first; r < end; ++r) {
        const A g = S::load(gy[r * s.len + l]);
        dw += g * ((S::load(x[r * s.len + l]) - mean[r]) * rstd[r]);
        db += g;
    }
    part[(block * 2) * s.len + l] = dw;
    part[(block * 2 + 1) * s.len + l] = db;
}

// inner == 1 and few rows: a thread owns an element of the row, and what it adds up is the gradient.  Partial sums of so
// few rows would be as large as the tensors: 16 rows of 65536 bfloat16 take 14 us with this, 31 with them.
template <typename T>
__global__ void __launch_bounds__(128)
    norm_param_direct_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                             const typename Storage<T>::acc* __restrict__ mean,
                             const typename Storage<T>::acc* __restrict__ rstd, void* __restrict__ dw,
                             void* __restrict__ db, bool f32, NormShape s) {
    using S = Storage<T>;
    using A = typename S::acc;
    const int l = blockIdx.x * 128 + threadIdx.x;
    if (l >= s.len) return;
    A w = A(0), b = A(0);
#pragma unroll 8
    for (int r = 0; r < static_cast<int>(s.rows); ++r) {
        const long long e = static_cast<long long>(r) * s.len + l;
        const A g = S::load(gy[e]);
        w += g * ((S::load(x[e]) - mean[r]) * rstd[r]);
        b += g;
    }
    if (dw) store_param<T>(dw, l, f32, w);
    if (db) store_param<T>(db, l, f32, b);
}

// inner > 1: a block sums rows_per neighbouring rows at one element of them.
template <typename T>
__global__ void __launch_bounds__(kNormThreads)
    norm_param_columns_kernel(const T* __restrict__ gy, const T* __restrict__ x,
                              const typename Storage<T>::acc* __restrict__ mean,
                              const typename Storage<T>::acc* __restrict__ rstd,
                              typename Storage<T>::acc* __restrict__ part, NormShape s, int rows_per) {
    using S = Storage<T>;
    using A = typename S::acc;
    __shared__ A shared[kNormThreads];
    const long long block = blockIdx.x / s.len;
    const int l = static_cast<int>(blockIdx.x % s.len);
    const long long end = min((block + 1) * rows_per, s.rows);
    A dw = A(0), db = A(0);
    for (long long r = block * rows_per + threadIdx.x; r < end; r += kNormThreads) {
        const long long e = s.base(r) + static_cast<long long>(l) * s.inner;
        const A g = S::load(gy[e]);
        dw += g * ((S::load(x[e]) - mean[r]) * rstd[r]);
        db += g;
    }
    dw = row_sum<true>(dw, shared);
    db = row_sum<true>(db, shared);
    if (threadIdx.x == 0) {
        part[(block * 2) * s.len + l] = dw;
        part[(block * 2 + 1) * s.len + l] = db;
    }
}

// A block sums blockDim.x of the 2 * len columns (dw, then db), each in blockDim.y shares of the partial sums.  It is
// launched while the kernel that writes them still runs, and waits for its end: a backward pass takes 0.7 to 1.2 us less.
constexpr int kParamThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kParamThreads)
    norm_param_final_kernel(const typename Storage<T>::acc* __restrict__ part, int blocks, int len,
                            void* __restrict__ dw, void* __restrict__ db, bool f32) {
    __shared__ double shared[kParamThreads];
    const int shares = blockDim.y, at = threadIdx.y * blockDim.x + threadIdx.x;
    const long long width = 2ll * len, column = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    double sum = 0.0;
    cudaGridDependencySynchronize();
    if (column < width) {
        const typename Storage<T>::acc* p = part + column;
#pragma unroll 8
        for (int k = threadIdx.y; k < blocks; k += shares) sum += p[k * width];
    }
    if (shares > 1) {
        shared[at] = sum;
        for (int half = shares >> 1; half > 0; half >>= 1) {  // a power of two of shares
            __syncthreads();
            if (threadIdx.y < half) shared[at] = sum += shared[at + half * blockDim.x];
        }
    }
    void* out = column < len ? dw : db;
    if (threadIdx.y == 0 && column < width && out != nullptr)
        store_param<T>(out, column < len ? column : column - len, f32, sum);
}

}  // namespace serron
