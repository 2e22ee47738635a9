// Dropout: y = kept ? x / (1 - p) : 0, plus a residual where there is one.  The mask is a function of the element's
// index, the seed and the sequence number alone, so the backward pass is the same kernel over grad_output and
// nothing is stored between the two.
#pragma once

#include "layer_vec.cuh"

namespace serron {

// Decisions by element, p < 1.  A thread takes U vectors of V consecutive elements, 256 vectors apart, all loads issued
// before the first is used; a block of the generator serves four elements.  A block's elements start at a multiple of
// their number, a power of two, so the upper word of the generator's counter is the same for all of them, and with it
// half of the first two rounds.  The round keys are operands in constant memory where the seed is the host's.
//
// 16-bit elements are bound by the generator: five 32 x 32 -> 64 bit products an element, 17 instructions in all (26 with keys
// made in the kernel and elements unpacked one at a time).  (64,32,256,256) bfloat16: 103 to 113 us from run to run (72 to
// 80 % of the copy rate), with a residual 117 (at the copy rate, part of it from the L2); float32 runs at 88 to 100 % of it.
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

// Any alignment, any type and any `span` (the elements that share a decision), an element and a block of the generator at a
// time: 706 us at (64,32,256,256) bfloat16 an element off the boundary of a vector, seven times the vectors' time.
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

// Decisions by channel or sample, `span` elements each, V <= span < 2^30: small maps, of which a block holds many, and any
// that begin off a vector's boundary.  Vectors as above; a vector's first unit is found from where the block begins, and
// a vector may hold the end of one unit and the beginning of the next.  The input is read only where something is kept.
// (64,512,14,14) float16: 10.3 us; a decision for every element by itself took 40.
constexpr int kLongSpan = 8192;
template <typename T, int V, int U, bool RESIDUAL, bool DEVICE_SEED>
__global__ void __launch_bounds__(256)
    dropout_spans_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
                         int span, const __grid_constant__ DropRule rule) {
    using P = Pack<T, V>;
    using F = Floats<V>;
    static_assert(256 * U * V <= kLongSpan);
    const long long start = blockIdx.x * (256ll * U * V);
    const long long first = n < (1ll << 32) ? static_cast<unsigned>(start) / static_cast<unsigned>(span) : start / span;
    const int rest = static_cast<int>(start - first * span);  // of unit `first` before the block
    const float inverse = 1.0f / static_cast<float>(span);
    PhiloxKeys own;
    if (DEVICE_SEED) own.set(__ldg(rule.seed_device));
    const PhiloxKeys& keys = DEVICE_SEED ? own : rule.keys;
    const auto keeps = [&](long long unit) {
        return word_of(philox(unit >> 2, rule.sequence, keys), unit & 3) >= rule.threshold && !rule.all;
    };
    const int left = static_cast<int>(min(n - start, 256ll * U * V));  // of the block
    const T *xs = x + start, *rs = residual + (RESIDUAL ? start : 0);
    T* ys = y + start;
    P in[U], res[U];
    bool kept[U], after[U];
    int ends[U];  // the vector's elements in its first unit
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = (u * 256 + threadIdx.x) * V;
        // a block reaches into the unit after a long one at most; below 2 * kLongSpan the product is off by less than the
        // half that is added
        const int at = rest + e;
        const int unit = span >= kLongSpan ? at >= span : static_cast<int>((static_cast<float>(at) + 0.5f) * inverse);
        ends[u] = (unit + 1) * span - at;
        kept[u] = keeps(first + unit);
        after[u] = ends[u] < V && keeps(first + unit + 1);
        if (e + V <= left) {
            if (kept[u] || after[u]) in[u] = P::load(xs + e);
            if (RESIDUAL) res[u] = P::load(rs + e);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = (u * 256 + threadIdx.x) * V;
        if (e >= left) return;
        if (e + V <= left) {
            F v;
            v.fill(0.0f);
            if (kept[u] || after[u]) {
                v = in[u].floats();
                float f[V];
#pragma unroll
                for (int i = 0; i < F::N; ++i) v.e[i] = mul(v.e[i], splat<typename F::E>(rule.scale32));
                v.to(f);
#pragma unroll
                for (int k = 0; k < V; ++k) f[k] = (k < ends[u] ? kept[u] : after[u]) ? f[k] : 0.0f;
                v.from(f);
            }
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
                    const bool keep = k < ends[u] ? kept[u] : after[u];
                    float v = keep ? scaled(Storage<T>::load(xs[e + k]), rule.scale32) : 0.0f;
                    if (RESIDUAL) v += Storage<T>::load(rs[e + k]);
                    ys[e + k] = Storage<T>::store(v);
                }
            }
        }
    }
}

// Decisions by channel or sample of kLongSpan elements or more, in whole vectors: a block takes a piece of one unit, decides
// once and reads the input only where it is kept (70 us at (64,32,256,256) bfloat16 with p = 1/4: 7/8 of two passes at the
// copy rate).  Grid: pieces of a unit, units.
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
