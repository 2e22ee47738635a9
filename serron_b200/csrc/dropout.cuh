// Dropout: y = kept ? x / (1 - p) : 0, plus a residual where there is one.  The mask is a function of the element's
// index, the seed and the sequence number alone, so the backward pass is the same kernel over grad_output and
// nothing is stored between the two.
#pragma once

#include "layer_common.cuh"

namespace serron {

// `span` elements share a decision: 1, a channel's H * W, or a sample's C * H * W.
template <typename T>
__global__ void __launch_bounds__(256)
    dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
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

}  // namespace serron
