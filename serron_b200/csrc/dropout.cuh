// Dropout: y = kept ? x / (1 - p) : 0, plus a residual where there is one.  The mask is a function of the element's
// index, the seed and the sequence number alone, so the backward pass is the same kernel over grad_output and
// nothing is stored between the two.
#pragma once

#include "layer_vec.cuh"

namespace serron {

// Decisions by element.  A thread takes U vectors of V consecutive elements, 256 vectors apart, all loads issued before
// the first is used; a block of the generator serves four elements.
template <typename T, int V, int U, bool RESIDUAL>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
                   DropRule rule) {
    using P = Pack<T, V>;
    const long long first = (blockIdx.x * (256ll * U) + threadIdx.x) * V;
    const uint64_t key = rule.key();
    const float scale = static_cast<float>(rule.scale);
    P in[U], res[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long e = first + u * (256 * V);
        if (e + V <= n) {
            in[u] = P::load(x + e);
            if (RESIDUAL) res[u] = P::load(residual + e);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long e = first + u * (256 * V);
        if (e >= n) return;
        uint32_t words[V];
        drop_words<V>(e, rule.sequence, key, words);
        if (e + V <= n) {
            float v[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[k] = rule.keeps(words[k]) ? scaled(in[u].get(k), scale) : 0.0f;
                if (RESIDUAL) v[k] += res[u].get(k);
            }
            P out;
            out.set(v);
            out.store(y + e);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) {  // the last, incomplete vector
                if (e + k < n) {
                    float v = rule.keeps(words[k]) ? scaled(Storage<T>::load(x[e + k]), scale) : 0.0f;
                    if (RESIDUAL) v += Storage<T>::load(residual[e + k]);
                    y[e + k] = Storage<T>::store(v);
                }
            }
        }
    }
}

// Any alignment, any type and any `span` (the elements that share a decision), an element at a time.
template <typename T>
__global__ void __launch_bounds__(256)
    dropout_any_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
                       long long span, DropRule rule) {
    using S = Storage<T>;
    using A = typename S::acc;
    const long long e = blockIdx.x * 256ll + threadIdx.x;
    if (e >= n) return;
    const long long unit = span == 1 ? e : e / span;
    const uint4 words = philox(unit >> 2, rule.sequence, rule.key());
    A v = rule.keeps(word_of(words, unit & 3)) ? scaled<A>(S::load(x[e]), A(rule.scale)) : A(0);
    if (residual) v = v + S::load(residual[e]);
    y[e] = S::store(v);
}

// Decisions by channel or sample: a block takes `vectors` vectors of one unit (grid: pieces of a unit, units), decides
// once and reads the input only where it is kept.
template <typename T, int V, int U>
__global__ void __launch_bounds__(256)
    dropout_units_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long span,
                         unsigned pieces, DropRule rule) {
    using P = Pack<T, V>;
    const long long unit = blockIdx.x / pieces;
    const long long at = ((blockIdx.x % pieces) * (256ll * U) + threadIdx.x) * V;
    const long long base = unit * span;
    const bool kept = rule.keeps(word_of(philox(unit >> 2, rule.sequence, rule.key()), unit & 3));
    const float scale = static_cast<float>(rule.scale);
    P in[U], res[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long e = at + u * (256 * V);
        if (e < span) {
            if (kept) in[u] = P::load(x + base + e);
            if (residual) res[u] = P::load(residual + base + e);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long e = at + u * (256 * V);
        if (e >= span) return;
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            v[k] = kept ? scaled(in[u].get(k), scale) : 0.0f;
            if (residual) v[k] += res[u].get(k);
        }
        P out;
        out.set(v);
        out.store(y + base + e);
    }
}

}  // namespace serron
