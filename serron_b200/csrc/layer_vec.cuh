// Short vectors of stored elements, read and written in one access, and computed on as floats, two to an instruction.
#pragma once

#include <type_traits>

#include "layer_common.cuh"

namespace serron {

// ------------------------------------------------------------------------------------------------
// two floats in one register pair: sm_100 adds, multiplies and fuses both in one instruction (each lane rounded as
// the scalar instruction rounds).  The same names work on single floats, so that code is written once.
// ------------------------------------------------------------------------------------------------
struct Two {
    unsigned long long bits;
};

__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.bits) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 parts(Two v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v.bits));
    return r;
}
__device__ __forceinline__ Two add(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two sub(Two a, Two b) {
    Two r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}
__device__ __forceinline__ float total(Two v) {
    const float2 p = parts(v);
    return p.x + p.y;
}
__device__ __forceinline__ float add(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ float sub(float a, float b) { return __fsub_rn(a, b); }
__device__ __forceinline__ float mul(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float fma(float a, float b, float c) { return __fmaf_rn(a, b, c); }
__device__ __forceinline__ float total(float v) { return v; }

template <typename E>
__device__ __forceinline__ E splat(float v);
template <>
__device__ __forceinline__ Two splat<Two>(float v) { return two(v, v); }
template <>
__device__ __forceinline__ float splat<float>(float v) { return v; }


// V floats: pairs where V is even.
template <int V>
struct Floats {
    using E = std::conditional_t<V % 2 == 0, Two, float>;
    static constexpr int N = V % 2 == 0 ? V / 2 : V;
    E e[N];

    __device__ __forceinline__ void fill(float v) {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = splat<E>(v);
    }
    __device__ __forceinline__ void to(float (&out)[V]) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (V % 2 == 0) {
                const float2 p = parts(e[i]);
                out[2 * i] = p.x;
                out[2 * i + 1] = p.y;
            } else {
                out[i] = e[i];
            }
        }
    }
    __device__ __forceinline__ void from(const float (&in)[V]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (V % 2 == 0)
                e[i] = two(in[2 * i], in[2 * i + 1]);
            else
                e[i] = in[i];
        }
    }
};

// ------------------------------------------------------------------------------------------------
// V elements of T as they lie in memory, aligned to their size
// ------------------------------------------------------------------------------------------------
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

template <typename T, int V>
struct Pack {
    using Raw = typename RawOf<V * static_cast<int>(sizeof(T))>::type;
    static constexpr int kWords = V * static_cast<int>(sizeof(T)) / 4;
    union {
        Raw raw;
        uint32_t word[kWords > 0 ? kWords : 1];
    };

    static __device__ __forceinline__ Pack load(const T* p) {
        Pack out;
        out.raw = *reinterpret_cast<const Raw*>(p);
        return out;
    }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }

    __device__ __forceinline__ Floats<V> floats() const {
        Floats<V> out;
        if constexpr (sizeof(T) == 4) {
            if constexpr (V == 1) {
                out.e[0] = __uint_as_float(raw);
            } else {
#pragma unroll
                for (int i = 0; i < V / 2; ++i)
                    out.e[i] = two(__uint_as_float(word[2 * i]), __uint_as_float(word[2 * i + 1]));
            }
        } else if constexpr (V == 1) {
            if constexpr (std::is_same_v<T, __half>)
                out.e[0] = __half2float(__ushort_as_half(raw));
            else
                out.e[0] = __uint_as_float(static_cast<uint32_t>(raw) << 16);
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                if constexpr (std::is_same_v<T, __half>) {
                    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&word[i]));
                    out.e[i] = two(p.x, p.y);
                } else {  // a bfloat16 is the upper half of its float
                    out.e[i] = two(__uint_as_float(word[i] << 16), __uint_as_float(word[i] & 0xffff0000u));
                }
            }
        }
        return out;
    }

    static __device__ __forceinline__ Pack of(const Floats<V>& f) {
        Pack out;
        if constexpr (sizeof(T) == 4) {
            if constexpr (V == 1) {
                out.raw = __float_as_uint(f.e[0]);
            } else {
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float2 p = parts(f.e[i]);
                    out.word[2 * i] = __float_as_uint(p.x);
                    out.word[2 * i + 1] = __float_as_uint(p.y);
                }
            }
        } else if constexpr (V == 1) {
            if constexpr (std::is_same_v<T, __half>)
                out.raw = __half_as_ushort(__float2half_rn(f.e[0]));
            else
                out.raw = __bfloat16_as_ushort(__float2bfloat16_rn(f.e[0]));
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float2 p = parts(f.e[i]);
                if constexpr (std::is_same_v<T, __half>) {
                    const __half2 h = __floats2half2_rn(p.x, p.y);
                    out.word[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);
                    out.word[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
        }
        return out;
    }
};

// V parameters from index i on (a multiple of V), float32 or of type T.
template <typename T, int V>
__device__ __forceinline__ Floats<V> load_params(const void* p, int i, bool f32) {
    if (sizeof(T) == 2 && !f32) return Pack<T, V>::load(static_cast<const T*>(p) + i).floats();
    const float* q = static_cast<const float*>(p) + i;
    if constexpr (V <= 4) {
        return Pack<float, V>::load(q).floats();
    } else {
        Floats<V> out;
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const Floats<4> four = Pack<float, 4>::load(q + k).floats();
            out.e[k / 2] = four.e[0];
            out.e[k / 2 + 1] = four.e[1];
        }
        return out;
    }
}

// The words of decisions e .. e + V - 1 (below 2^34), where e is a multiple of V.
template <int V>
__device__ __forceinline__ void drop_words(long long e, uint64_t sequence, const PhiloxKeys& keys, uint32_t (&out)[V]) {
    if constexpr (V >= 4) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const uint4 w = philox(static_cast<uint32_t>(e >> 2) + k / 4, 0u, sequence, keys);
            out[k] = w.x;
            out[k + 1] = w.y;
            out[k + 2] = w.z;
            out[k + 3] = w.w;
        }
    } else {
        static_assert(V == 1);
        out[0] = word_of(philox(static_cast<uint32_t>(e >> 2), 0u, sequence, keys), e & 3);
    }
}

// The dropped v, scaled.
template <int V>
__device__ __forceinline__ Floats<V> dropped(const Floats<V>& v, const uint32_t (&words)[V], uint32_t threshold,
                                             float scale) {
    Floats<V> s;
#pragma unroll
    for (int i = 0; i < Floats<V>::N; ++i) s.e[i] = mul(v.e[i], splat<typename Floats<V>::E>(scale));
    float f[V];
    s.to(f);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = words[i] >= threshold ? f[i] : 0.0f;
    s.from(f);
    return s;
}

}  // namespace serron
