// AdamW over many tensors at once, with the moments in 32 or in 8 bits, and the global gradient norm behind it (the reference builds
// torch.optim.AdamW, main.py:186-245, and clips with clip_grad_norm_, main.py:413-430).  Per element, every operation rounded by itself in fp32:
//     g' = c g                  c = min(1, max_norm / (|g| + 1e-6)) over ALL tensors, read from device memory (no read-back)
//     m  = b1 m + (1 - b1) g'   v = b2 v + (1 - b2) g'^2      r = sqrt(v)
//     p  = p (1 - lr wd) - (m lr / (1 - b1^t)) / (r / sqrt(1 - b2^t) + eps)
// Nothing is contracted into an fma here: the 8-bit codes are decided next to borders, and with plain roundings the same inputs give the
// same bits in any elementwise implementation of the formula.
//
// A launch takes its tensor list by value (kernel arguments, < 4 KB: 84 tensors with 32-bit moments, 56 with 8-bit ones), so a step needs no
// table in device memory, no copy and no lifetime rule; a block owns 4 096 elements of one tensor and finds it by one ballot over the list.
//
// Bound by memory: p, m and v in and out, g in (and once more for the norm).  Measured, 202 M elements: bf16 with 32-bit moments 806 us (4.45 GB,
// 5.5 TB/s), the norm before it 126 us (0.40 GB, 3.2 TB/s); fp32 with 8-bit moments 822 us (3.25 GB, 4.0 TB/s), bf16 with 8-bit moments 753 us
// (2.03 GB, 2.7 TB/s: the rounding's VALU work is that of fp32), reading a moment out 204 us (1.01 GB, 4.9 TB/s).  A model of 180 tensors and
// 3 M elements: 3 x 5.7 us with 32-bit moments, 4 x 9.8 us with 8-bit ones, 9 us for the norm.
#include "common.h"
#include "elem.h"
#include <algorithm>
#include <vector>

#pragma clang fp contract(off)

#define ADAMW_CHUNK 4096            // elements of a block: 16 per thread
#define ADAMW_BLOCK 256             // elements that share a scale (8-bit moments): 4 per lane of one wave
#define SQSUM_CHUNK 8192

namespace {

struct AdamwHyper { float decay, step, inv_bc2, eps; };            // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps

template <int NT, bool Q>
struct AdamwArgs {
    uint64_t p[NT], g[NT], m[NT], v[NT];
    uint64_t ms[Q ? NT : 1], vs[Q ? NT : 1];
    int64_t n[NT];
    unsigned first[NT];             // first block of a tensor
    unsigned key[Q ? NT : 1];
    AdamwHyper hyper[8];
    unsigned char which[NT];        // its entry of hyper
    float b1, ob1, b2, ob2;
    const float *grad_scale;
    int nt;
};
constexpr int NT32 = 84, NT8 = 56;
static_assert(sizeof(AdamwArgs<NT32, false>) <= 4096 && sizeof(AdamwArgs<NT8, true>) <= 4096, "kernel argument segment");

template <int NT>
struct SqsumArgs {
    uint64_t g[NT];
    int64_t n[NT];
    unsigned first[NT];
    double *out;
    int nt;
};
constexpr int NTS = 200;
static_assert(sizeof(SqsumArgs<NTS>) <= 4096, "kernel argument segment");

// index of the tensor a block works on: the number of list entries that begin at or before it, minus one (all lanes compare one entry each)
template <int NT>
__device__ __forceinline__ int find_tensor(const unsigned (&first)[NT], int nt, unsigned block) {
    const int lane = threadIdx.x & 63;
    int k = -1;
#pragma unroll
    for (int b = 0; b < NT; b += 64) k += __popcll(__ballot(b + lane < nt && first[b + lane < NT ? b + lane : NT - 1] <= block));
    return __builtin_amdgcn_readfirstlane(k);
}

struct Elem { float b1, ob1, b2, ob2, c; AdamwHyper h; };

// one element; m and v hold the old moments and become the new ones.  Returns the new parameter, r = sqrt(v)
__device__ __forceinline__ float adamw_elem(const Elem &e, float p, float g, float &m, float &v, float &r) {
    g = g * e.c;
    const float m0 = m * e.b1, m1 = g * e.ob1;
    m = m0 + m1;
    const float gg = g * g, v0 = v * e.b2, v1 = gg * e.ob2;
    v = v0 + v1;
    r = sqrtf(v);
    p = p * e.h.decay;
    const float den = r * e.h.inv_bc2 + e.h.eps;
    return p - (m * e.h.step) / den;
}

template <typename T>
__global__ __launch_bounds__(256) void adamw32_kernel(AdamwArgs<NT32, false> a) {
    const int t = find_tensor(a.first, a.nt, blockIdx.x);
    T *p = reinterpret_cast<T *>(a.p[t]);
    const T *g = reinterpret_cast<const T *>(a.g[t]);
    float *m = reinterpret_cast<float *>(a.m[t]), *v = reinterpret_cast<float *>(a.v[t]);
    const int64_t n = a.n[t], base = (int64_t)(blockIdx.x - a.first[t]) * ADAMW_CHUNK;
    Elem e{a.b1, a.ob1, a.b2, a.ob2, a.grad_scale ? *a.grad_scale : 1.0f, a.hyper[a.which[t]]};
    const bool vec = ((a.m[t] | a.v[t]) & 15) == 0 && ((a.p[t] | a.g[t]) & (4 * sizeof(T) - 1)) == 0;
    float pv[4][4], gv[4][4], mv[4][4], vv[4][4];
    // all loads of a block first; a tensor's last elements, or storage that is not aligned, go one by one
    auto at = [&](int u) { return base + u * 1024 + threadIdx.x * 4; };
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t i = at(u);
        if (vec && i + 4 <= n) {
            Quad<T>::load(p + i, pv[u]);
            Quad<T>::load(g + i, gv[u]);
            Quad<float>::load(m + i, mv[u]);
            Quad<float>::load(v + i, vv[u]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const bool in = i + k < n;
                pv[u][k] = in ? Quad<T>::one(p + i + k) : 0.f;
                gv[u][k] = in ? Quad<T>::one(g + i + k) : 0.f;
                mv[u][k] = in ? m[i + k] : 0.f;
                vv[u][k] = in ? v[i + k] : 0.f;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t i = at(u);
        float r;
#pragma unroll
        for (int k = 0; k < 4; ++k) pv[u][k] = adamw_elem(e, pv[u][k], gv[u][k], mv[u][k], vv[u][k], r);
        if (vec && i + 4 <= n) {
            Quad<T>::store(p + i, pv[u]);
            Quad<float>::store(m + i, mv[u]);
            Quad<float>::store(v + i, vv[u]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) {
                    Quad<T>::put(p + i + k, pv[u][k]);
                    m[i + k] = mv[u][k];
                    v[i + k] = vv[u][k];
                }
        }
    }
}

// ---- 8-bit moments ---------------------------------------------------------------------------------------------------------------
// 256 consecutive values share a scale 2^floor(log2 max|x|); x / scale in [0, 2) is held in 3 exponent and M mantissa bits (subnormals
// below 2^-6): m with a sign and M = 4, and -- because v spans twice the octaves -- sqrt(v) with M = 5, no sign.  The scale is a power of
// two so that scaling is exact and a value that does not change keeps its code.  Rounding is probabilistic, up with the probability of the
// dropped fraction: the second moment changes by 0.1 % a step (b2 = 0.999) against half a step of 1.6 ... 3 % of the value, so that rounding
// to the nearest code would never move it (simulated over 2 000 steps after half a block's gradients shrank to 0.3: sqrt(v) off by 52 % of a
// standard deviation with nearest rounding and a scale of max|x|, by 9 % here, without bias).  A value above the top code, (2 - 2^-M) scale, is
// cut to it where it got there in one step; where the block already stood there it would be cut again at every step, and a value that grows
// by less than a code a step would never reach 2 scale: then the scale doubles (simulated, normal gradients that grow from 1.6 to 2.2: sqrt(v)
// 12 % low and falling without, 0.4 % high with it, as if nothing were ever cut; m that grows 0.03 % a step: 11 % low, exact).  A value whose
// v is not zero never gets code zero (the step would divide by eps alone).  A gradient that is not finite makes its block's scale NaN, as it
// makes its element's moments.
__device__ __forceinline__ unsigned adamw_random(unsigned index, unsigned key) {
    unsigned x = index * 0x9E3779B9u + key;
    x = (x ^ (x >> 16)) * 0x6C62272Du;
    x = (x ^ (x >> 15)) * 0x2C9277B5u;
    return x ^ (x >> 16);
}
template <int M>
__device__ __forceinline__ unsigned q8_encode(float x, unsigned rnd) {              // x in [0, 2), rnd: 23 - M random bits
    const unsigned normal = ((__float_as_uint(x) + rnd) >> (23 - M)) - (120u << M);
    const unsigned small = ((unsigned)(int)(x * 536870912.0f) + rnd) >> (23 - M);
    const unsigned code = x >= 0.015625f ? normal : small;
    return code > (8u << M) - 1 ? (8u << M) - 1 : code;
}
template <int M>
__device__ __forceinline__ float q8_decode(unsigned code, float scale) {
    const unsigned field = code >> M, man = code & ((1u << M) - 1);
    const float normal = __uint_as_float((field + 120u) << 23 | man << (23 - M));
    const float small = (float)man * (1.0f / (64 << M));
    return (field ? normal : small) * scale;
}
__device__ __forceinline__ float q8_decode_m(unsigned c, float scale) {
    const float x = q8_decode<4>(c & 127u, scale);
    return c & 128u ? -x : x;
}
// the top code's mantissa bits, and whether a block's largest magnitude (as bits) lies above it and may still be doubled
template <int M> __device__ __forceinline__ constexpr unsigned q8_top() { return ((1u << M) - 1) << (23 - M); }
template <int M> __device__ __forceinline__ bool q8_over(unsigned top) { return (top & 0x7fffffu) > q8_top<M>() && top < 0x7f000000u; }
// scale and its inverse from the block's largest magnitude (as bits: NaN is largest)
__device__ __forceinline__ float q8_scale(unsigned top, float &inv) {
    const float s = __uint_as_float(top & 0x7f800000u);
    const bool some = top >= 0x0d800000u;                          // 2^-100: everything below is zero
    inv = some ? 1.0f / s : 0.f;
    return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : (some ? s : 0.f);
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o));
    return v;
}

template <typename T>
__global__ __launch_bounds__(256) void adamw8_kernel(AdamwArgs<NT8, true> a) {
    const int t = find_tensor(a.first, a.nt, blockIdx.x);
    T *p = reinterpret_cast<T *>(a.p[t]);
    const T *g = reinterpret_cast<const T *>(a.g[t]);
    uint8_t *m = reinterpret_cast<uint8_t *>(a.m[t]), *v = reinterpret_cast<uint8_t *>(a.v[t]);
    float *ms = reinterpret_cast<float *>(a.ms[t]), *vs = reinterpret_cast<float *>(a.vs[t]);
    const int64_t n = a.n[t], base = (int64_t)(blockIdx.x - a.first[t]) * ADAMW_CHUNK;
    const unsigned key = a.key[t];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Elem e{a.b1, a.ob1, a.b2, a.ob2, a.grad_scale ? *a.grad_scale : 1.0f, a.hyper[a.which[t]]};
    const bool vec = ((a.m[t] | a.v[t]) & 3) == 0 && ((a.p[t] | a.g[t]) & (4 * sizeof(T) - 1)) == 0;
    float pv[4][4], gv[4][4];
    unsigned mc[4], vc[4];
    float msc[4], vsc[4];
    // a wave's four blocks of 256: all loads first
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t b0 = base + (u * 4 + wave) * ADAMW_BLOCK, i = b0 + lane * 4;
        mc[u] = vc[u] = 0;
        msc[u] = vsc[u] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) pv[u][k] = gv[u][k] = 0.f;
        if (b0 >= n) continue;
        msc[u] = ms[b0 / ADAMW_BLOCK];
        vsc[u] = vs[b0 / ADAMW_BLOCK];
        if (vec && b0 + ADAMW_BLOCK <= n) {
            Quad<T>::load(p + i, pv[u]);
            Quad<T>::load(g + i, gv[u]);
            mc[u] = *reinterpret_cast<const unsigned *>(m + i);
            vc[u] = *reinterpret_cast<const unsigned *>(v + i);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) {
                    pv[u][k] = Quad<T>::one(p + i + k);
                    gv[u][k] = Quad<T>::one(g + i + k);
                    mc[u] |= (unsigned)m[i + k] << (8 * k);
                    vc[u] |= (unsigned)v[i + k] << (8 * k);
                }
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t b0 = base + (u * 4 + wave) * ADAMW_BLOCK, i = b0 + lane * 4;
        if (b0 >= n) continue;                                     // (uniform over the wave)
        float mn[4], rn[4];
        unsigned mt = 0, rt = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            mn[k] = q8_decode_m((mc[u] >> (8 * k)) & 255u, msc[u]);
            const float r0 = q8_decode<5>((vc[u] >> (8 * k)) & 255u, vsc[u]);
            float vv = r0 * r0;
            pv[u][k] = adamw_elem(e, pv[u][k], gv[u][k], mn[k], vv, rn[k]);
            const bool in = i + k < n;                             // (elements behind the end take no part in the scale)
            mt = max(mt, in ? __float_as_uint(mn[k]) & 0x7fffffffu : 0u);
            rt = max(rt, in ? __float_as_uint(rn[k]) & 0x7fffffffu : 0u);
        }
        unsigned mtop = __builtin_amdgcn_readfirstlane(wave_umax(mt)), rtop = __builtin_amdgcn_readfirstlane(wave_umax(rt));
        if (q8_over<4>(mtop)) {                                    // (4.6 % of the blocks, 2.3 % of the roots')
            const float edge = __uint_as_float((mtop & 0x7f800000u) | q8_top<4>());
            bool held = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) held |= q8_decode<4>((mc[u] >> (8 * k)) & 127u, msc[u]) >= edge;
            if (__any(held)) mtop += 0x800000u;
        }
        if (q8_over<5>(rtop)) {
            const float edge = __uint_as_float((rtop & 0x7f800000u) | q8_top<5>());
            bool held = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) held |= q8_decode<5>((vc[u] >> (8 * k)) & 255u, vsc[u]) >= edge;
            if (__any(held)) rtop += 0x800000u;
        }
        float minv, rinv;
        const float mscale = q8_scale(mtop, minv), rscale = q8_scale(rtop, rinv);
        unsigned mo = 0, ro = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned rnd = adamw_random((unsigned)(i + k), key);
            unsigned cm = q8_encode<4>(__builtin_fabsf(mn[k]) * minv, (rnd >> 18) << 5);
            cm |= mn[k] < 0.f ? 128u : 0u;
            unsigned cr = q8_encode<5>(rn[k] * rinv, rnd & 0x3ffffu);
            if (rn[k] > 0.f && rinv > 0.f && cr == 0) cr = 1;
            mo |= cm << (8 * k);
            ro |= cr << (8 * k);
        }
        if (vec && b0 + ADAMW_BLOCK <= n) {
            Quad<T>::store(p + i, pv[u]);
            *reinterpret_cast<unsigned *>(m + i) = mo;
            *reinterpret_cast<unsigned *>(v + i) = ro;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < n) {
                    Quad<T>::put(p + i + k, pv[u][k]);
                    m[i + k] = (uint8_t)(mo >> (8 * k));
                    v[i + k] = (uint8_t)(ro >> (8 * k));
                }
        }
        if (lane == 0) {
            ms[b0 / ADAMW_BLOCK] = mscale;
            vs[b0 / ADAMW_BLOCK] = rscale;
        }
    }
}

__global__ __launch_bounds__(256) void adamw_moment_kernel(const uint8_t *__restrict__ code, const float *__restrict__ scale, int64_t n, int squared,
                                                           float *__restrict__ out) {
    const bool vec = (reinterpret_cast<uintptr_t>(code) & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q * 4 < n; q += (int64_t)gridDim.x * 256) {
        const int64_t i = q * 4;
        const float s = scale[i / ADAMW_BLOCK];
        auto value = [&](unsigned c) {
            if (!squared) return q8_decode_m(c, s);
            const float r = q8_decode<5>(c, s);
            return r * r;
        };
        if (vec && i + 4 <= n) {
            const unsigned c = *reinterpret_cast<const unsigned *>(code + i);
            stg4(out + i, make_float4(value(c & 255u), value((c >> 8) & 255u), value((c >> 16) & 255u), value(c >> 24)));
        } else {
            for (int k = 0; k < 4 && i + k < n; ++k) out[i + k] = value(code[i + k]);
        }
    }
}

// ---- the gradient norm: squares and sums in 64 bits (202 million addends), one partial per block, summed in a fixed order ------------------
__device__ __forceinline__ double block_sum(double s) {
    __shared__ double sh[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
template <typename T>
__global__ __launch_bounds__(256) void grad_sqsum_kernel(SqsumArgs<NTS> a) {
    const int t = find_tensor(a.first, a.nt, blockIdx.x);
    const T *g = reinterpret_cast<const T *>(a.g[t]);
    const int64_t n = a.n[t], base = (int64_t)(blockIdx.x - a.first[t]) * SQSUM_CHUNK;
    const bool vec = (a.g[t] & (4 * sizeof(T) - 1)) == 0;
    constexpr int U = SQSUM_CHUNK / 1024;
    float gv[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = base + u * 1024 + threadIdx.x * 4;
        if (vec && i + 4 <= n) {
            Quad<T>::load(g + i, gv[u]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) gv[u][k] = i + k < n ? Quad<T>::one(g + i + k) : 0.f;
        }
    }
    double s[4] = {0., 0., 0., 0.};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = fma((double)gv[u][k], (double)gv[u][k], s[k]);
    const double b = block_sum((s[0] + s[1]) + (s[2] + s[3]));
    if (threadIdx.x == 0) a.out[blockIdx.x] = b;
}
__global__ __launch_bounds__(256) void grad_norm_kernel(const double *__restrict__ parts, int64_t n, float max_norm, float *__restrict__ out) {
    double s[4] = {0., 0., 0., 0.};
    int64_t i = threadIdx.x;
    for (; i + 768 < n; i += 1024)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] += parts[i + 256 * k];
    for (; i < n; i += 256) s[0] += parts[i];
    const double b = block_sum((s[0] + s[1]) + (s[2] + s[3]));
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(b), c = max_norm / (norm + 1e-6f);
        out[0] = norm;
        out[1] = c > 1.0f ? 1.0f : c;                              // (a norm that is NaN makes every gradient NaN, as clip_grad_norm_ does)
    }
}

template <typename T>
int adamw_launch(int state_bits, const AdamwArgs<NT32, false> &a, const AdamwArgs<NT8, true> &q, unsigned blocks, hipStream_t st) {
    if (state_bits == 32) hipLaunchKernelGGL((adamw32_kernel<T>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((adamw8_kernel<T>), dim3(blocks), dim3(256), 0, st, q);
    return nmrf_launch_status();
}

// fills launches of up to NT tensors; `go` launches one
template <int NT, bool Q, typename F>
int adamw_fill(AdamwArgs<NT, Q> &a, int n, const uint64_t *p, const uint64_t *g, const uint64_t *m, const uint64_t *v, const uint64_t *ms,
               const uint64_t *vs, const int64_t *numel, const float *hyper, const uint32_t *key, F go) {
    unsigned blocks = 0;
    int nh = 0;
    a.nt = 0;
    for (int i = 0; i <= n; ++i) {
        int h = 0;
        int64_t nb = 0;
        AdamwHyper want{};
        if (i < n) {
            if (numel[i] == 0) continue;
            want = AdamwHyper{hyper[4 * i], hyper[4 * i + 1], hyper[4 * i + 2], hyper[4 * i + 3]};
            while (h < nh && __builtin_memcmp(&a.hyper[h], &want, sizeof want) != 0) ++h;
            nb = ceil_div64(numel[i], ADAMW_CHUNK);
        }
        if (a.nt && (i == n || a.nt == NT || h == 8 || (int64_t)blocks + nb > 0x7fffffff)) {
            const int rc = go(blocks);
            if (rc != NMRF_OK) return rc;
            blocks = 0;
            nh = a.nt = 0;
            h = 0;
        }
        if (i == n) break;
        if (h == nh) a.hyper[nh++] = want;
        const int k = a.nt++;
        a.p[k] = p[i]; a.g[k] = g[i]; a.m[k] = m[i]; a.v[k] = v[i];
        a.n[k] = numel[i];
        a.first[k] = blocks;
        a.which[k] = (unsigned char)h;
        if constexpr (Q) { a.ms[k] = ms[i]; a.vs[k] = vs[i]; a.key[k] = key[i]; }
        blocks += (unsigned)nb;
    }
    return NMRF_OK;
}

}  // namespace

extern "C" int nmrf_adamw_step(int n, const uint64_t *p, const uint64_t *g, const uint64_t *m, const uint64_t *v, const uint64_t *m_scale,
                               const uint64_t *v_scale, const int64_t *numel, const float *hyper, const uint32_t *key, const float *betas,
                               int dtype, int state_bits, const float *grad_scale, void *stream) {
    if (!p || !g || !m || !v || !numel || !hyper || !betas) return NMRF_ENULL;
    if (state_bits != 32 && state_bits != 8) return NMRF_EINVAL;
    if (state_bits == 8 && (!m_scale || !v_scale || !key)) return NMRF_ENULL;
    if (n < 1 || dtype < NMRF_F32 || dtype > NMRF_F16) return NMRF_EINVAL;
    const uint64_t el = dtype == NMRF_F32 ? 3 : 1;
    for (int i = 0; i < n; ++i) {
        if (numel[i] < 0 || numel[i] > (int64_t)0x7fffffff * ADAMW_CHUNK) return NMRF_EINVAL;
        if (numel[i] == 0) continue;
        if (!p[i] || !g[i] || !m[i] || !v[i] || (state_bits == 8 && (!m_scale[i] || !v_scale[i]))) return NMRF_ENULL;
        if (((p[i] | g[i]) & el) || (state_bits == 32 ? ((m[i] | v[i]) & 3) : ((m_scale[i] | v_scale[i]) & 3))) return NMRF_EINVAL;
    }
    try {                                                          // one parameter twice would be updated by two blocks at once
        std::vector<uint64_t> seen;
        seen.reserve(n);
        for (int i = 0; i < n; ++i) if (numel[i]) seen.push_back(p[i]);
        std::sort(seen.begin(), seen.end());
        if (std::adjacent_find(seen.begin(), seen.end()) != seen.end()) return NMRF_EINVAL;
    } catch (...) {
        return NMRF_EINVAL;
    }
    AdamwArgs<NT32, false> a;
    AdamwArgs<NT8, true> q;
    a.b1 = q.b1 = betas[0]; a.ob1 = q.ob1 = betas[1]; a.b2 = q.b2 = betas[2]; a.ob2 = q.ob2 = betas[3];
    a.grad_scale = q.grad_scale = grad_scale;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](unsigned blocks) {
        if (dtype == NMRF_F32) return adamw_launch<float>(state_bits, a, q, blocks, st);
        if (dtype == NMRF_BF16) return adamw_launch<__bf16>(state_bits, a, q, blocks, st);
        return adamw_launch<_Float16>(state_bits, a, q, blocks, st);
    };
    if (state_bits == 32) return adamw_fill(a, n, p, g, m, v, m_scale, v_scale, numel, hyper, key, go);
    return adamw_fill(q, n, p, g, m, v, m_scale, v_scale, numel, hyper, key, go);
}

extern "C" int nmrf_adamw_moment_f32(const uint8_t *code, const float *scale, int64_t n, int squared, float *out, void *stream) {
    if (!code || !scale || !out) return NMRF_ENULL;
    if (n < 1 || (reinterpret_cast<uintptr_t>(scale) & 3) || (reinterpret_cast<uintptr_t>(out) & 3)) return NMRF_EINVAL;
    int64_t blocks = ceil_div64(n, 1024);
    if (blocks > 16384) blocks = 16384;
    hipLaunchKernelGGL(adamw_moment_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, code, scale, n, squared, out);
    return nmrf_launch_status();
}

static int64_t grad_sqsum_parts(int n, const int64_t *numel) {
    int64_t total = 0;
    for (int i = 0; numel && i < n; ++i) total += numel[i] > 0 ? ceil_div64(numel[i], SQSUM_CHUNK) : 0;
    return total;
}

extern "C" int nmrf_grad_sqsum(int n, const uint64_t *g, const int64_t *numel, int dtype, double *parts, int64_t capacity, void *stream) {
    if (!g || !numel || !parts) return NMRF_ENULL;
    if (n < 1 || dtype < NMRF_F32 || dtype > NMRF_F16) return NMRF_EINVAL;
    const uint64_t el = dtype == NMRF_F32 ? 3 : 1;
    for (int i = 0; i < n; ++i) {
        if (numel[i] < 0 || numel[i] > (int64_t)0x7fffffff * SQSUM_CHUNK) return NMRF_EINVAL;
        if (numel[i] && !g[i]) return NMRF_ENULL;
        if (numel[i] && (g[i] & el)) return NMRF_EINVAL;
    }
    if (grad_sqsum_parts(n, numel) > capacity) return NMRF_EINVAL;
    SqsumArgs<NTS> a;
    a.out = parts;
    a.nt = 0;
    int64_t blocks = 0;
    hipStream_t st = (hipStream_t)stream;
    for (int i = 0; i <= n; ++i) {
        if (i < n && numel[i] == 0) continue;
        const int64_t nb = i < n ? ceil_div64(numel[i], SQSUM_CHUNK) : 0;
        if (a.nt && (i == n || a.nt == NTS || blocks + nb > 0x7fffffff)) {
            if (dtype == NMRF_F32) hipLaunchKernelGGL(grad_sqsum_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, a);
            else if (dtype == NMRF_BF16) hipLaunchKernelGGL(grad_sqsum_kernel<__bf16>, dim3((unsigned)blocks), dim3(256), 0, st, a);
            else hipLaunchKernelGGL(grad_sqsum_kernel<_Float16>, dim3((unsigned)blocks), dim3(256), 0, st, a);
            const int rc = nmrf_launch_status();
            if (rc != NMRF_OK) return rc;
            a.out += blocks;
            blocks = 0;
            a.nt = 0;
        }
        if (i == n) break;
        a.g[a.nt] = g[i];
        a.n[a.nt] = numel[i];
        a.first[a.nt++] = (unsigned)blocks;
        blocks += nb;
    }
    return NMRF_OK;
}

extern "C" int nmrf_grad_norm(const double *parts, int64_t count, float max_norm, float *out, void *stream) {
    if (!parts || !out) return NMRF_ENULL;
    if (count < 1 || !(max_norm > 0.f)) return NMRF_EINVAL;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, parts, count, max_norm, out);
    return nmrf_launch_status();
}
