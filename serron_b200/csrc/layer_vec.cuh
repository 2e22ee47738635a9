// Short vectors of stored elements, read and written in one access, and computed on as floats.
#pragma once

#include "layer_common.cuh"

namespace serron {

template <int BYTES>
struct RawOf;
template <>
struct RawOf<2> { using type = uint16_t; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<16> { using type = uint4; };

// V elements of T as they lie in memory, aligned to their size.
template <typename T, int V>
struct Pack {
    using Raw = typename RawOf<V * static_cast<int>(sizeof(T))>::type;
    union {
        Raw raw;
        T e[V];
    };
    __device__ __forceinline__ Pack() : raw() {}
    static __device__ __forceinline__ Pack load(const T* p) {
        Pack out;
        out.raw = *reinterpret_cast<const Raw*>(p);
        return out;
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
    __device__ __forceinline__ float get(int i) const { return Storage<T>::load(e[i]); }
    // all V at once: two conversions to 16 bits are one instruction
    __device__ __forceinline__ void set(const float (&v)[V]) {
        if constexpr (V % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                if constexpr (std::is_same_v<T, __half>)
                    *reinterpret_cast<__half2*>(&e[i]) = __floats2half2_rn(v[i], v[i + 1]);
                else
                    *reinterpret_cast<__nv_bfloat162*>(&e[i]) = __floats2bfloat162_rn(v[i], v[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = Storage<T>::store(v[i]);
        }
    }
};

// V parameters from index i on (a multiple of V), float32 or of type T.
template <typename T, int V>
__device__ __forceinline__ void load_params(const void* p, int i, bool f32, float (&out)[V]) {
    if (f32) {
        if constexpr (V >= 4) {
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const float4 q = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + k);
                out[k] = q.x;
                out[k + 1] = q.y;
                out[k + 2] = q.z;
                out[k + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) out[k] = static_cast<const float*>(p)[i + k];
        }
    } else {
        const Pack<T, V> q = Pack<T, V>::load(static_cast<const T*>(p) + i);
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = q.get(k);
    }
}

// The words of decisions e .. e + V - 1, where e is a multiple of min(V, 4).
template <int V>
__device__ __forceinline__ void drop_words(long long e, uint64_t sequence, uint64_t key, uint32_t (&out)[V]) {
    if constexpr (V >= 4) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const uint4 w = philox((e >> 2) + k / 4, sequence, key);
            out[k] = w.x;
            out[k + 1] = w.y;
            out[k + 2] = w.z;
            out[k + 3] = w.w;
        }
    } else {
        const uint4 w = philox(e >> 2, sequence, key);
        if constexpr (V == 2) {
            out[0] = e & 2 ? w.z : w.x;
            out[1] = e & 2 ? w.w : w.y;
        } else {
            out[0] = word_of(w, e & 3);
        }
    }
}

}  // namespace serron
