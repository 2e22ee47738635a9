// What the layer operators (layer norm, dropout and their join) share: the counter-based generator, the dropout
// rule, and parameters held in float32 or in the activations' type.
#pragma once

#include <cstdint>

#include "common.cuh"

namespace serron {

// ------------------------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds
// of two 32 x 32 -> 64 bit products over a counter, under a key that grows by a constant a round.  Block j of
// sequence q under seed s is the cipher of counter (j, q) with key s, all 64 bits wide, low word first.
// ------------------------------------------------------------------------------------------------
constexpr int kPhiloxRounds = 10;
constexpr uint32_t kPhiloxMul0 = 0xD2511F53u, kPhiloxMul1 = 0xCD9E8D57u;
constexpr uint32_t kPhiloxKey0 = 0x9E3779B9u, kPhiloxKey1 = 0xBB67AE85u;

// The keys of all rounds, both words of a round side by side.
struct alignas(16) PhiloxKeys {
    uint32_t k[2 * kPhiloxRounds];

    __host__ __device__ __forceinline__ void set(uint64_t seed) {
        for (int r = 0; r < kPhiloxRounds; ++r) {
            k[2 * r] = static_cast<uint32_t>(seed) + r * kPhiloxKey0;
            k[2 * r + 1] = static_cast<uint32_t>(seed >> 32) + r * kPhiloxKey1;
        }
    }
};

// The words of block (low, high).  Where `high` and `sequence` are the same for all threads, so is half of the first two
// rounds, and the compiler computes it once.
__device__ __forceinline__ uint4 philox(uint32_t low, uint32_t high, uint64_t sequence, const PhiloxKeys& keys) {
    uint32_t c0 = low, c1 = high;
    uint32_t c2 = static_cast<uint32_t>(sequence), c3 = static_cast<uint32_t>(sequence >> 32);
#pragma unroll
    for (int r = 0; r < kPhiloxRounds; ++r) {
        const uint64_t a = static_cast<uint64_t>(c0) * kPhiloxMul0;
        const uint64_t b = static_cast<uint64_t>(c2) * kPhiloxMul1;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ keys.k[2 * r];
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ keys.k[2 * r + 1];
        c3 = static_cast<uint32_t>(a);
    }
    return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ uint4 philox(long long block, uint64_t sequence, const PhiloxKeys& keys) {
    return philox(static_cast<uint32_t>(block), static_cast<uint32_t>(block >> 32), sequence, keys);
}

__device__ __forceinline__ uint32_t word_of(const uint4& block, int i) {
    return i == 0 ? block.x : i == 1 ? block.y : i == 2 ? block.z : block.w;
}

// The dropout rule: decision j keeps its elements when word j % 4 of block j / 4 is at least `threshold`.
struct DropRule {
    PhiloxKeys keys;                        // of the seed, unless it is in device memory
    const uint64_t* seed_device = nullptr;  // read by the kernel in place of `keys` where set
    uint64_t sequence = 0;
    uint32_t threshold = 0;  // round(p * 2^32)
    bool all = false;        // p rounds to one: every element is dropped
    double scale = 1.0;      // 1 / (1 - p)
    float scale32 = 1.0f;

    // the keys wherever the seed is (in registers)
    __device__ __forceinline__ PhiloxKeys own_keys() const {
        PhiloxKeys k = keys;
        if (seed_device) k.set(__ldg(seed_device));
        return k;
    }
};

// A kept element, scaled; a dropped one is zero whatever it held (NaN and infinities too).  The product is rounded
// before anything is added to it, so that the sum with a residual has the bits of the two-step formula.
template <typename A>
__device__ __forceinline__ A scaled(A v, A scale);
template <>
__device__ __forceinline__ float scaled<float>(float v, float scale) { return __fmul_rn(v, scale); }
template <>
__device__ __forceinline__ double scaled<double>(double v, double scale) { return __dmul_rn(v, scale); }

// ------------------------------------------------------------------------------------------------
// weight and bias: float32, or the activations' own type
// ------------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ typename Storage<T>::acc load_param(const void* p, long long i, bool f32) {
    using A = typename Storage<T>::acc;
    return f32 ? A(static_cast<const float*>(p)[i]) : A(Storage<T>::load(static_cast<const T*>(p)[i]));
}
template <typename T, typename V>
__device__ __forceinline__ void store_param(void* p, long long i, bool f32, V v) {
    if (f32)
        static_cast<float*>(p)[i] = static_cast<float>(v);
    else
        static_cast<T*>(p)[i] = Storage<T>::store(static_cast<typename Storage<T>::acc>(v));
}

template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

template <typename A>
__device__ __forceinline__ A inverse_root(A v);
template <>
__device__ __forceinline__ float inverse_root<float>(float v) { return 1.0f / sqrtf(v); }
template <>
__device__ __forceinline__ double inverse_root<double>(double v) { return 1.0 / sqrt(v); }

}  // namespace serron
