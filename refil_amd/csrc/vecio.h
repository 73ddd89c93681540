// Element types of the block operators (linrec.hip, norm_gate.hip, gated_ff.hip): fp32, bf16 and fp16 in memory, fp32 in registers.
// A vector access is 16 bytes wide and needs the ELEMENT's alignment only (gfx950 takes global accesses at any byte address), so odd
// widths and strides run through the same kernels; the ragged end of a row is moved element by element.
#pragma once
#include "common.h"

namespace refil {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

typedef unsigned u32x4_e4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_e2 __attribute__((ext_vector_type(4), aligned(2)));
template <class T> struct IoVec { typedef u32x4_e2 type; };
template <> struct IoVec<float> { typedef u32x4_e4 type; };

template <class T> constexpr int VEC_OF = 16 / (int)sizeof(T);

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
// (round to nearest even: half a step of the type)
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// the raw 16 bytes of a vector, kept packed until the values are needed
struct Raw { unsigned w[4]; };

// elements [p, p + n), n <= VEC, missing ones zero
template <class T>
__device__ __forceinline__ Raw ld_raw(const T* p, int n) {
    Raw r;
    if (n >= VEC_OF<T>) {
        const typename IoVec<T>::type v = *reinterpret_cast<const typename IoVec<T>::type*>(p);
        r.w[0] = v[0]; r.w[1] = v[1]; r.w[2] = v[2]; r.w[3] = v[3];
        return r;
    }
    r.w[0] = r.w[1] = r.w[2] = r.w[3] = 0u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) r.w[i] = __builtin_bit_cast(unsigned, p[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) r.w[i >> 1] |= (unsigned)__builtin_bit_cast(unsigned short, p[i]) << (16 * (i & 1));
    }
    return r;
}
template <class T> __device__ __forceinline__ float raw_get(const Raw& r, int i);
template <> __device__ __forceinline__ float raw_get<float>(const Raw& r, int i) { return __uint_as_float(r.w[i]); }
template <> __device__ __forceinline__ float raw_get<bf16_t>(const Raw& r, int i) {
    const unsigned w = r.w[i >> 1];
    return __uint_as_float((i & 1) ? (w & 0xFFFF0000u) : (w << 16));
}
template <> __device__ __forceinline__ float raw_get<f16_t>(const Raw& r, int i) {
    return (float)__builtin_bit_cast(f16_t, (unsigned short)(r.w[i >> 1] >> (16 * (i & 1))));
}
template <class T>
__device__ __forceinline__ Raw raw_pack(const float* v) {
    Raw r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.w[i] = (unsigned)__builtin_bit_cast(unsigned short, from_f32<T>(v[2 * i])) | ((unsigned)__builtin_bit_cast(unsigned short, from_f32<T>(v[2 * i + 1])) << 16);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void st_raw(T* p, const Raw& r, int n) {
    if (n >= VEC_OF<T>) {
        typename IoVec<T>::type v;
        v[0] = r.w[0]; v[1] = r.w[1]; v[2] = r.w[2]; v[3] = r.w[3];
        *reinterpret_cast<typename IoVec<T>::type*>(p) = v;
        return;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = __builtin_bit_cast(T, r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = __builtin_bit_cast(T, (unsigned short)(r.w[i >> 1] >> (16 * (i & 1))));
    }
}

// exp(x) = 2^(x log2 e) with the rounding of the product put back as a first-order factor: 1-2 ulp over the whole range (the bare
// product loses |x| half steps). v_exp_f32 flushes nothing that matters here: results below 2^-126 are zero to every consumer.
__device__ __forceinline__ float exp_acc(float x) {
    const float t = x * 1.44269504088896341f;
    const float lo = fmaf(x, 1.44269504088896341f, -t) + x * 1.92596299e-8f;      // log2 e = 1.442695041 (fp32) + 1.926e-8
    const float e = __builtin_amdgcn_exp2f(t);
    // (t infinite: lo is NaN and the exponential already is 0 or inf)
    return fabsf(t) < 256.f ? fmaf(e, lo * 0.693147181f, e) : e;
}
// 1 / (1 + e^-x); saturates to 0 and 1
__device__ __forceinline__ float sigmoid_acc(float x) { return 1.0f / (1.0f + exp_acc(-x)); }

// the per-type choice: 16-bit results are rounded at 2^-9 (bf16) / 2^-12 (fp16) of their value, the 1e-6 of the hardware-rate forms below
// vanishes there; fp32 results get the accurate forms
template <class T> __device__ __forceinline__ float sigmoid_t(float x) { return fast_sigmoid(x); }
template <> __device__ __forceinline__ float sigmoid_t<float>(float x) {
    const float d = 1.0f + exp_acc(-x);
    float r = __builtin_amdgcn_rcpf(d);
    return d < 1e38f ? fmaf(fmaf(-d, r, 1.0f), r, r) : 0.0f;     // one Newton step on the hardware reciprocal
}
template <class T> __device__ __forceinline__ float exp_t(float x) { return __builtin_amdgcn_exp2f(1.44269504088896341f * x); }
template <> __device__ __forceinline__ float exp_t<float>(float x) { return exp_acc(x); }

}  // namespace refil
