// Element types of the training-block operators (fp32, bf16, fp16): four consecutive values between memory and fp32 registers.  Stores round
// once, to nearest even.  load / store want 4 * sizeof(T) alignment, one / put the element's own.
#pragma once
#include "common.h"

template <typename T> struct Quad;                                  // four consecutive values of a parameter or gradient
template <> struct Quad<float> {
    static __device__ __forceinline__ void load(const float *p, float *v) { const float4 t = ldg4(p); v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; }
    static __device__ __forceinline__ void store(float *p, const float *v) { stg4(p, make_float4(v[0], v[1], v[2], v[3])); }
    static __device__ __forceinline__ float one(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
};
template <> struct Quad<__bf16> {
    static __device__ __forceinline__ void load(const __bf16 *p, float *v) {
        const uint2 t = *reinterpret_cast<const uint2 *>(p);
        v[0] = __uint_as_float(t.x << 16); v[1] = __uint_as_float(t.x & 0xffff0000u);
        v[2] = __uint_as_float(t.y << 16); v[3] = __uint_as_float(t.y & 0xffff0000u);
    }
    static __device__ __forceinline__ unsigned short rn(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }
    static __device__ __forceinline__ void store(__bf16 *p, const float *v) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(rn(v[0]) | (unsigned)rn(v[1]) << 16, rn(v[2]) | (unsigned)rn(v[3]) << 16);
    }
    static __device__ __forceinline__ float one(const __bf16 *p) { return __uint_as_float((unsigned)*reinterpret_cast<const unsigned short *>(p) << 16); }
    static __device__ __forceinline__ void put(__bf16 *p, float v) { *reinterpret_cast<unsigned short *>(p) = rn(v); }
};
template <> struct Quad<_Float16> {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ void load(const _Float16 *p, float *v) {
        const h4 t = *reinterpret_cast<const h4 *>(p);
        v[0] = (float)t[0]; v[1] = (float)t[1]; v[2] = (float)t[2]; v[3] = (float)t[3];
    }
    static __device__ __forceinline__ void store(_Float16 *p, const float *v) { *reinterpret_cast<h4 *>(p) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]}; }
    static __device__ __forceinline__ float one(const _Float16 *p) { return (float)*p; }
    static __device__ __forceinline__ void put(_Float16 *p, float v) { *p = (_Float16)v; }
};

// N consecutive values (16 bytes, or one value for rows that 16-byte loads do not fit)
template <typename T, int N> struct Vec {
    static_assert(N == 1 || N * sizeof(T) == 16, "one value or 16 bytes");
    static __device__ __forceinline__ void load(const T *p, float *v) {
        if constexpr (N == 1) v[0] = Quad<T>::one(p);
        else if constexpr (sizeof(T) == 4) Quad<T>::load(p, v);
        else {
            const uint4 t = *reinterpret_cast<const uint4 *>(p);
            const unsigned w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (__is_same(T, __bf16)) {
                    v[2 * j] = __uint_as_float(w[j] << 16);
                    v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                } else {
                    v[2 * j] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[j] & 0xffffu));
                    v[2 * j + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[j] >> 16));
                }
            }
        }
    }
    static __device__ __forceinline__ void store(T *p, const float *v) {
        if constexpr (N == 1) Quad<T>::put(p, v[0]);
        else if constexpr (sizeof(T) == 4) Quad<T>::store(p, v);
        else {
            unsigned w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = __builtin_bit_cast(unsigned short, (T)v[2 * j]) | (unsigned)__builtin_bit_cast(unsigned short, (T)v[2 * j + 1]) << 16;
            *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};
