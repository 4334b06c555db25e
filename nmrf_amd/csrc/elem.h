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

// 16 bytes of values as they lie in memory, at any alignment of the element (gfx950 takes unaligned 16-byte accesses), and their fp32 values.
// Loads are split from unpacking so that a row can be asked for long before it is used.
template <typename T> struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ uint4 raw(const T *p) {
        uint4 t;
        __builtin_memcpy(&t, p, 16);
        return t;
    }
    static __device__ __forceinline__ void unpack(const uint4 &t, float *v) {
        const unsigned w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) v[j] = __uint_as_float(w[j]);
            else if constexpr (__is_same(T, __bf16)) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            } else {
                v[2 * j] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[j] & 0xffffu));
                v[2 * j + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[j] >> 16));
            }
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *v) {
        unsigned w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[j]);
            else w[j] = __builtin_bit_cast(unsigned short, (T)v[2 * j]) | (unsigned)__builtin_bit_cast(unsigned short, (T)v[2 * j + 1]) << 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void store(T *p, const float *v) {
        const uint4 t = pack(v);
        __builtin_memcpy(p, &t, 16);
    }
    // the first n < N values, zeros behind them
    static __device__ __forceinline__ uint4 raw_part(const T *p, int n) {
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < n) {
                if constexpr (sizeof(T) == 4) w[k] = __builtin_bit_cast(unsigned, p[k]);
                else w[k / 2] |= (unsigned)__builtin_bit_cast(unsigned short, p[k]) << (16 * (k & 1));
            }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // the first n <= N values, zeros behind them, where `room` values from p on may be read
    static __device__ __forceinline__ uint4 raw_masked(const T *p, int n, int64_t room) {
        if (room < N) return raw_part(p, n < room ? n : (int)room);
        const uint4 t = raw(p);
        unsigned w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) w[j] = j < n ? w[j] : 0u;
            else w[j] &= (2 * j < n ? 0xffffu : 0u) | (2 * j + 1 < n ? 0xffff0000u : 0u);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void store_part(T *p, const float *v, int n) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < n) p[k] = (T)v[k];
    }
};
