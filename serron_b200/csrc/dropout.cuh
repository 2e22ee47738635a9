// Dropout: y = kept ? x / (1 - p) : 0, plus a residual where there is one.  The mask is a function of the element's
// index, the seed and the sequence number alone, so the backward pass is the same kernel over grad_output and
// nothing is stored between the two.
#pragma once

#include "layer_vec.cuh"

namespace serron {

// Decisions by element, p < 1.  A thread takes U vectors of V consecutive elements, 256 vectors apart, all loads issued
// before the first is used; a block of the generator serves four elements.  A block's elements start at a multiple of
// their number, a power of two, so the upper word of the generator's counter is the same for all of them.
template <typename T, int V, int U, bool RESIDUAL, bool DEVICE_SEED>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
                   const __grid_constant__ DropRule rule) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    const long long start = blockIdx.x * (256ll * U * V);
    const uint32_t high = static_cast<uint32_t>(start >> 34), low = static_cast<uint32_t>(start >> 2);
    const float scale = rule.scale32;
    PhiloxKeys own;
    if (DEVICE_SEED) own.set(__ldg(rule.seed_device));
    const PhiloxKeys& keys = DEVICE_SEED ? own : rule.keys;
    const int left = static_cast<int>(min(n - start, 256ll * U * V));  // of the block
    const T *xs = x + start, *rs = residual + (RESIDUAL ? start : 0);
    T* ys = y + start;
    P in[U], res[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = (u * 256 + threadIdx.x) * V;
        if (e + V <= left) {
            in[u] = P::load(xs + e);
            if (RESIDUAL) res[u] = P::load(rs + e);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = (u * 256 + threadIdx.x) * V;
        if (e >= left) return;
        uint32_t words[V];
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const uint4 w = philox(low + (e + k) / 4, high, rule.sequence, keys);
            words[k] = w.x;
            words[k + 1] = w.y;
            words[k + 2] = w.z;
            words[k + 3] = w.w;
        }
        if (e + V <= left) {
            F v = dropped<V>(in[u].floats(), words, rule.threshold, scale);
            if (RESIDUAL) {
                const F r = res[u].floats();
#pragma unroll
                for (int i = 0; i < F::N; ++i) v.e[i] = add(v.e[i], r.e[i]);
            }
            P::of(v).store(ys + e);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) {  // the last, incomplete vector
                if (e + k < left) {
                    float v = words[k] >= rule.threshold ? scaled(Storage<T>::load(xs[e + k]), scale) : 0.0f;
                    if (RESIDUAL) v += Storage<T>::load(rs[e + k]);
                    ys[e + k] = Storage<T>::store(v);
                }
            }
        }
    }
}

// Any alignment, any type and any `span` (the elements that share a decision), an element at a time.
template <typename T>
__global__ void __launch_bounds__(256)
    dropout_any_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
                       long long span, const __grid_constant__ DropRule rule) {
    using S = Storage<T>;
    using A = typename S::acc;
    const long long e = blockIdx.x * 256ll + threadIdx.x;
    if (e >= n) return;
    const long long unit = span == 1 ? e : e / span;
    const uint4 words = philox(unit >> 2, rule.sequence, rule.own_keys());
    const bool kept = word_of(words, unit & 3) >= rule.threshold && !rule.all;
    A v = kept ? scaled<A>(S::load(x[e]), A(rule.scale)) : A(0);
    if (residual) v = v + S::load(residual[e]);
    y[e] = S::store(v);
}

// Decisions by channel or sample: a block takes a piece of one unit, decides once and reads the input only where it is
// kept.  Grid: pieces of a unit, units.
template <typename T, int V, int U>
__global__ void __launch_bounds__(256)
    dropout_units_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long span,
                         unsigned pieces, const __grid_constant__ DropRule rule) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    const unsigned unit = blockIdx.x / pieces;
    const long long at = (blockIdx.x - unit * pieces) * (256ll * U * V);
    const long long base = unit * span + at;
    const int left = static_cast<int>(min(span - at, 256ll * U * V));
    const bool kept =
        word_of(philox(unit >> 2, rule.sequence, rule.own_keys()), unit & 3) >= rule.threshold && !rule.all;
    const float scale = rule.scale32;
    P in[U], res[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = (u * 256 + threadIdx.x) * V;
        if (e < left) {
            if (kept) in[u] = P::load(x + base + e);
            if (residual) res[u] = P::load(residual + base + e);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = (u * 256 + threadIdx.x) * V;
        if (e >= left) return;
        F v;
        v.fill(0.0f);
        if (kept) {
            v = in[u].floats();
#pragma unroll
            for (int i = 0; i < F::N; ++i) v.e[i] = mul(v.e[i], splat<typename F::E>(scale));
        }
        if (residual) {
            const F r = res[u].floats();
#pragma unroll
            for (int i = 0; i < F::N; ++i) v.e[i] = add(v.e[i], r.e[i]);
        }
        P::of(v).store(y + base + e);
    }
}

}  // namespace serron
