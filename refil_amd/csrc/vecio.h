// Element types of the block operators (linrec.hip, norm_gate.hip, gated_ff.hip): fp32, bf16 and fp16 in memory, fp32 in registers.
// A vector access needs the ELEMENT's alignment only (gfx950 takes global accesses at any byte address), so odd widths and strides run
// through the same kernels; the ragged end of a row is moved element by element.
#pragma once
#include "common.h"

namespace refil {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <class T> constexpr int VEC_OF = 16 / (int)sizeof(T);

template <int BYTES, int ALIGN> struct IoWord;
template <> struct IoWord<16, 4> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct IoWord<16, 2> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct IoWord<8, 2> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(2))); };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
// (round to nearest even: half a step of the type)
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// the raw words of V elements, kept packed until the values are needed
template <class T, int V = VEC_OF<T>> struct Raw { unsigned w[V * sizeof(T) / 4]; };

// a word full of -inf (an element that is not there, where the value's exponential is to vanish)
template <class T> inline constexpr unsigned NEG_INF_WORD = 0xFF800000u;
template <> inline constexpr unsigned NEG_INF_WORD<bf16_t> = 0xFF80FF80u;
template <> inline constexpr unsigned NEG_INF_WORD<f16_t> = 0xFC00FC00u;

// V elements moved down by m (0 <= m < V), zeros coming in on top
template <class T, int V>
__device__ __forceinline__ Raw<T, V> raw_down(Raw<T, V> r, int m) {
    constexpr int W = V * sizeof(T) / 4;
    const int words = sizeof(T) == 4 ? m : m >> 1;
#pragma unroll
    for (int b = 1; b < W; b *= 2) {
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = (words & b) ? (i + b < W ? r.w[i + b] : 0u) : r.w[i];
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = (m & 1) ? (r.w[i] >> 16) | (i + 1 < W ? r.w[i + 1] << 16 : 0u) : r.w[i];
    }
    return r;
}
// elements [p, p + n) of V; the others are `absent` (a bit pattern per word; n is 0, or V but for the ragged end of a row)
template <class T, int V = VEC_OF<T>>
__device__ __forceinline__ Raw<T, V> ld_raw(const T* p, int n, unsigned absent = 0u) {
    constexpr int W = V * sizeof(T) / 4;
    typedef typename IoWord<V * sizeof(T), sizeof(T)>::type Word;
    Raw<T, V> r;
    if (n >= V) {
        const Word v = *reinterpret_cast<const Word*>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = v[i];
        return r;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = absent;
    if (n > 0) {
        // (V loads at once from places that exist, one wait, then the choice)
        T e[V];
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = p[i < n ? i : n - 1];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) r.w[i] = i < n ? __builtin_bit_cast(unsigned, e[i]) : absent;
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const unsigned lo = i < n ? __builtin_bit_cast(unsigned short, e[i]) : (absent & 0xFFFFu);
                const unsigned hi = i + 1 < n ? (unsigned)__builtin_bit_cast(unsigned short, e[i + 1]) << 16 : (absent & 0xFFFF0000u);
                r.w[i >> 1] = lo | hi;
            }
        }
    }
    return r;
}
template <class T, int V>
__device__ __forceinline__ float raw_get(const Raw<T, V>& r, int i) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
    else if constexpr (__is_same(T, bf16_t)) return __uint_as_float((i & 1) ? (r.w[i >> 1] & 0xFFFF0000u) : (r.w[i >> 1] << 16));
    else return (float)__builtin_bit_cast(f16_t, (unsigned short)(r.w[i >> 1] >> (16 * (i & 1))));
}
template <class T, int V = VEC_OF<T>>
__device__ __forceinline__ Raw<T, V> raw_pack(const float* v) {
    Raw<T, V> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) r.w[i] = __float_as_uint(v[i]);
    } else {
        typedef float F2 __attribute__((ext_vector_type(2)));
        typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < V / 2; ++i) r.w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((F2{v[2 * i], v[2 * i + 1]}), T2));
    }
    return r;
}
template <class T, int V>
__device__ __forceinline__ void st_raw(T* p, const Raw<T, V>& r, int n) {
    constexpr int W = V * sizeof(T) / 4;
    typedef typename IoWord<V * sizeof(T), sizeof(T)>::type Word;
    if (n >= V) {
        Word v;
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = r.w[i];
        *reinterpret_cast<Word*>(p) = v;
        return;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = __builtin_bit_cast(T, r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = __builtin_bit_cast(T, (unsigned short)(r.w[i >> 1] >> (16 * (i & 1))));
    }
}

// e^x at the hardware's rate: the exponent's product costs |x| half steps of the result, v_exp_f32 one
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(1.44269504088896341f * x); }

}  // namespace refil
