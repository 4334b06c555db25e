// The gated feed-forward block, forward and backward:
//     g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u,  y = h Wd^T + bd                 x [T, D], Wg, Wu [F, D], Wd [Do, F]
//     dh = dy Wd,  du = dh act(g),  dg = dh u act'(g)                                    act: silu, gelu (erf), relu
//     dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h,  biases: column sums
// (the framework's own feed-forward is the two-matrix form fc2(gelu(fc1 x)), nmrf/models/NMP.py:337, 537, 675).
//
// Bound by the matrix pipe: 6 T D F operations forward, 12 T D F backward, all in ONE tile kernel with operands that lie either way -- along the
// contraction (x Wg^T) or across it (dh = dy Wd, every weight gradient) -- and the elementwise work in its epilogue: both projections share a
// block (half its columns are Wg's, half Wu's, so that a lane holds g and u of the same element), dg and du come out of the product dh
// without dh being written.  16-bit types feed v_mfma_f32_16x16x32 directly.  fp32 is multiplied as fp16 pairs (hi, lo) in three products, as
// everywhere in this library, with each operand first scaled by a power of two that puts its largest magnitude at 2^13 (split_mfma.h):
// errors relative to the tensor's largest entry, no range limit.  Sums in fp32.
//
// Few tokens (up to 64): the weights are read once and nothing else matters; ffn_few_kernel streams them from memory into the matrix pipe's
// operand layout without LDS, a block's 8 waves sharing the contraction.
#include "common.h"
#include "elem.h"
#include <initializer_list>
#include <type_traits>

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

template <typename T> using Half = std::conditional_t<__is_same(T, float), _Float16, T>;      // what the matrix pipe reads

__device__ __forceinline__ f32x4 mma(const uint4 &a, const uint4 &b, f32x4 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const uint4 &a, const uint4 &b, f32x4 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };
__device__ __forceinline__ float act_value(float g, int act) {
    if (act == ACT_SILU) return g / (1.0f + expf(-g));
    if (act == ACT_GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678118654752440f));
    return g > 0.f ? g : (g != g ? g : 0.f);
}
__device__ __forceinline__ float act_slope(float g, int act) {
    if (act == ACT_SILU) {
        const float s = 1.0f / (1.0f + expf(-g));
        return s * (1.0f + g * (1.0f - s));
    }
    if (act == ACT_GELU) return 0.5f * (1.0f + erff(g * 0.70710678118654752440f)) + g * 0.39894228040143267794f * expf(-0.5f * g * g);
    return g > 0.f ? 1.f : 0.f;
}

// ---- largest magnitudes (fp32 operands): per tensor 64 slots, of which a product takes the maximum --------------------------------------
enum { SLOT_X = 0, SLOT_W = 1, SLOT_WD = 2, SLOT_H = 3, SLOT_DY = 4, SLOT_DG = 5, NSLOT = 6 };
struct AbsmaxArgs { const float *p[5]; int64_t n[5]; int slot[5]; int count; unsigned *out; int zero; };      // zero: bit i clears slot i
__global__ __launch_bounds__(256) void ffn_absmax_kernel(AbsmaxArgs a) {
    __shared__ float sh[4];
    const int which = blockIdx.y;
    const float *p = a.p[which];
    const int64_t n = a.n[which], per = (n + gridDim.x - 1) / gridDim.x, i0 = blockIdx.x * per, i1 = min(n, i0 + per);
    float m[4] = {0.f, 0.f, 0.f, 0.f};
    int64_t i = i0 + threadIdx.x * 4;
    for (; i + 4 <= i1; i += 1024) {
        float v[4];
        Vec16<float>::unpack(Vec16<float>::raw(p + i), v);
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = fmaxf(m[k], fabsf(v[k]));
    }
    for (; i < i1; ++i) m[0] = fmaxf(m[0], fabsf(p[i]));          // (a lane's last quad, cut short)
    float x = wave_max(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        x = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
        unsigned *o = a.out + a.slot[which] * 64 + (blockIdx.x & 63);     // (cleared by the launch before; the maximum does not depend on the order)
        atomicMax(o, __float_as_uint(x));
    }
}
__global__ void ffn_zero_kernel(unsigned *out, int zero) {
    if (zero >> blockIdx.x & 1) out[blockIdx.x * 64 + threadIdx.x] = 0u;
}
// power of two that puts the largest magnitude at [2^13, 2^14); 1 for zero, infinity and NaN
__device__ __forceinline__ int slot_shift(const unsigned *amax, int slot) {
    if (!amax) return 0;
    float m = wave_max(__uint_as_float(amax[slot * 64 + (threadIdx.x & 63)]));
    if (!(m > 0.f) || !(m < INFINITY)) return 0;
    const int e = (int)((__float_as_uint(m) >> 23) & 0xffu) - 127, sh = 13 - (e < -100 ? -100 : e);
    return __builtin_amdgcn_readfirstlane(sh);
}

// ---- the tile kernel ----------------------------------------------------------------------------------------------------------------------
//     C[m, n] = sum over segments s and k of P_s[m, k] Q_s[n, k]
// An operand lies ALONG k (row m: k contiguous, stride ld) or ACROSS it (row k: m contiguous, stride ld).
enum { EPI_DUAL = 0, EPI_PLAIN = 1, EPI_DH = 2 };
struct GemmArgs {
    const void *P[2], *Q[2];
    int64_t ldp, ldq, ldc;
    int M, N, K, segs;                           // K of one segment
    void *C, *C2, *C3;                           // EPI_DUAL: h, g, u (C2, C3 may be null); EPI_PLAIN: the product; EPI_DH: dg, du in C, C2
    const void *g, *u;                           // EPI_DH
    const void *bias, *bias2;
    float *parts;                                // EPI_PLAIN with splits > 1: fp32 partial products [splits][M][N]
    unsigned *amax;                              // fp32: the slots above
    int slot_p, slot_q, slot_out;                // slot_out: where the largest magnitude of the output goes (-1: nowhere)
    int act, splits, tiles_m, tiles_n, z;        // z problems side by side (P[z], C / C2): the two weight gradients of dg and du
};

template <typename T, int ROWS, int BK, bool ALONG, int THREADS> struct Stage {
    using H = Half<T>;
    static constexpr int CH = ROWS * BK / 8, N = CH / THREADS, V = sizeof(T) == 4 ? 2 : 1, PL = sizeof(T) == 4 ? 2 : 1;
    static constexpr int CPR = ALONG ? BK / 8 : ROWS / 8;          // 8-element chunks of an LDS row
    static constexpr int PLANE = ROWS * BK;                        // elements of one plane (fp32: hi plane, lo plane)
    static_assert(CH % THREADS == 0, "chunks per thread");
    uint4 r[N][V];
    // Position of chunk c of LDS row i.  Rows of 64 or 128 bytes (ALONG) take the same chunk from 16 consecutive rows: the rows that share a
    // 256-byte line of banks differ in their offset, the others in the exclusive-or.  Rows of 256 or 512 bytes (ACROSS) are read 8 at a time
    // (k, k+1, k+2, k+3 and 8 further), 32 bytes each: chunk pairs change places by those three bits of k.
    static __device__ __forceinline__ int slot(int i, int c) {
        if constexpr (ALONG) return c ^ ((i / (16 / CPR)) & (CPR - 1));
        else return c ^ ((2 * ((i & 3) | ((i >> 3) & 1) << 2)) & (CPR - 1));
    }
    // base: the operand's element (m0, k0) (block and k tile), rows: valid rows m, kleft: valid k.  row(m): offset of row m from base.
    template <typename RowOf>
    __device__ __forceinline__ void load(const T *base, int64_t ld, int rows, int kleft, bool whole, RowOf row_of) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = threadIdx.x + n * THREADS, i = id / CPR, c = id % CPR;
            if constexpr (ALONG) {
                const T *p = row_of(i) + c * 8;
                if (whole) {
#pragma unroll
                    for (int v = 0; v < V; ++v) r[n][v] = Vec16<T>::raw(p + v * (8 / V));
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) r[n][v] = Vec16<T>::raw_part(p + v * (8 / V), max(0, min(8 / V, kleft - c * 8 - v * (8 / V))));
                }
            } else {
                if (whole) {
                    const T *p = base + (int64_t)(unsigned)(i * (int)ld) + (c * 8 < rows ? c * 8 : 0);
#pragma unroll
                    for (int v = 0; v < V; ++v) r[n][v] = Vec16<T>::raw(p + v * (8 / V));
                } else {
                    const int left = i < kleft ? rows - c * 8 : 0;
                    const T *p = base + (int64_t)(i < kleft ? i : 0) * ld + (left > 0 ? c * 8 : 0);
#pragma unroll
                    for (int v = 0; v < V; ++v) r[n][v] = Vec16<T>::raw_part(p + v * (8 / V), max(0, min(8 / V, left - v * (8 / V))));
                }
            }
        }
    }
    __device__ __forceinline__ void put(H *lds, float mul) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = threadIdx.x + n * THREADS, i = id / CPR, c = id % CPR;
            H *q = lds + (ALONG ? i * BK : i * ROWS) + slot(i, c) * 8;
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<uint4 *>(q) = r[n][0];
            } else {
                float v[8];
                Vec16<float>::unpack(r[n][0], v);
                Vec16<float>::unpack(r[n][1], v + 4);
                h8 hi, lo;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float s = v[k] * mul;
                    hi[k] = (_Float16)s;
                    lo[k] = (_Float16)(s - (float)hi[k]);
                }
                *reinterpret_cast<h8 *>(q) = hi;
                *reinterpret_cast<h8 *>(q + PLANE) = lo;
            }
        }
    }
    // operand fragment of 16 rows from row m0 on, k = 32 kk + 8 (lane / 16) ... + 7
    static __device__ __forceinline__ uint4 frag(const H *lds, int m0, int kk) {
        const int l = threadIdx.x & 63;
        if constexpr (ALONG) {
            const int i = m0 + (l & 15);
            return *reinterpret_cast<const uint4 *>(lds + i * BK + slot(i, kk * 4 + (l >> 4)) * 8);
        } else {
            // a transposing read: 16 lanes fetch 4 rows k of 16 values and each gets the 4 values of its column
            const int k = 32 * kk + 8 * (l >> 4) + ((l & 15) >> 2), m = m0 + 4 * (l & 3);
            typedef __attribute__((address_space(3))) s4 lds_s4;
            union { s4 v[2]; uint4 u; } o;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int kr = k + 4 * h;
                H *q = const_cast<H *>(lds) + kr * ROWS + slot(kr, m >> 3) * 8 + (m & 7);
                o.v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(q));
            }
            return o.u;
        }
    }
};

template <typename T, int BM, int BN, int WM, int WN, int BK, bool PA, bool QA, int EPI>
__global__ __launch_bounds__(64 * WM * WN) void ffn_gemm_kernel(GemmArgs a) {
    using H = Half<T>;
    constexpr int THREADS = 64 * WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, PL = sizeof(T) == 4 ? 2 : 1;
    using SP = Stage<T, BM, BK, PA, THREADS>;
    using SQ = Stage<T, BN, BK, QA, THREADS>;
    __shared__ __align__(16) H lds[2][PL * (BM + BN) * BK];
    // blocks go to the 8 XCDs in turn: give each one a run of neighbouring tiles (its L2 then holds their operands), 8 row tiles deep
    const int per_z = a.tiles_m * a.tiles_n, all = per_z * a.splits * a.z;
    int t;
    {
        const int xcd = blockIdx.x & 7, q = all >> 3, rem = all & 7;
        t = xcd * q + min(xcd, rem) + (blockIdx.x >> 3);
    }
    const int zz = t / (per_z * a.splits), sp = t / per_z % a.splits;
    t %= per_z;
    const int band = t / (8 * a.tiles_n), deep = min(8, a.tiles_m - band * 8), in_band = t - band * 8 * a.tiles_n;
    const int tm = band * 8 + in_band % deep, tn = in_band / deep;
    constexpr int BNC = EPI == EPI_DUAL ? BN / 2 : BN;             // columns of the result
    const int m0 = tm * BM, n0 = tn * BNC;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN, lane = threadIdx.x & 63;

    float pmul = 1.f, qmul = 1.f;
    int unshift = 0;
    if constexpr (PL == 2) {
        const int sp_ = slot_shift(a.amax, a.slot_p), sq_ = slot_shift(a.amax, a.slot_q);
        pmul = ldexpf(1.f, sp_);
        qmul = ldexpf(1.f, sq_);
        unshift = -(sp_ + sq_);
    }
    const int ktiles_seg = (a.K + BK - 1) / BK, ktiles = ktiles_seg * a.segs;
    const int per = (ktiles + a.splits - 1) / a.splits, kt0 = sp * per, kt1 = min(ktiles, kt0 + per);
    const int prow = a.M - m0, qrow = a.N - n0;
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    SP sP;
    SQ sQ;
    auto fetch = [&](int kt) {
        const int seg = kt / ktiles_seg, k0 = (kt - seg * ktiles_seg) * BK, kleft = a.K - k0;
        const T *P = static_cast<const T *>(a.z > 1 ? (zz ? a.P[1] : a.P[0]) : (seg ? a.P[1] : a.P[0]));
        const T *Q = static_cast<const T *>(EPI != EPI_DUAL && seg ? a.Q[1] : a.Q[0]);
        const bool kw = kleft >= BK;
        // (a row behind the last is read as the last: its products are not stored)
        if constexpr (PA) {
            const T *b = P + (int64_t)m0 * a.ldp + k0;
            sP.load(nullptr, 0, 0, kleft, kw, [&](int i) { return b + (unsigned)(min(i, prow - 1) * (int)a.ldp); });
        } else {
            sP.load(P + (int64_t)k0 * a.ldp + m0, a.ldp, prow, kleft, kw && (prow >= BM || (a.M & 7) == 0), [](int) { return (const T *)nullptr; });
        }
        if constexpr (QA) {
            if constexpr (EPI == EPI_DUAL) {
                // of a wave's 16-column tiles the first half are Wg's rows, the second half Wu's
                const T *b0 = Q + (int64_t)n0 * a.ldq + k0, *b1 = static_cast<const T *>(a.Q[1]) + (int64_t)n0 * a.ldq + k0;
                sQ.load(nullptr, 0, 0, kleft, kw, [&](int i) {
                    const int w = i / (TN * 16), j = i / 16 % TN, n = w * (TN * 8) + j % (TN / 2) * 16 + i % 16;
                    return (j < TN / 2 ? b0 : b1) + (unsigned)(min(n, qrow - 1) * (int)a.ldq);
                });
            } else {
                const T *b = Q + (int64_t)n0 * a.ldq + k0;
                sQ.load(nullptr, 0, 0, kleft, kw, [&](int i) { return b + (unsigned)(min(i, qrow - 1) * (int)a.ldq); });
            }
        } else {
            sQ.load(Q + (int64_t)k0 * a.ldq + n0, a.ldq, qrow, kleft, kw && (qrow >= BN || (a.N & 7) == 0), [](int) { return (const T *)nullptr; });
        }
    };
    if (kt0 < kt1) {
        fetch(kt0);
        sP.put(lds[0], pmul);
        sQ.put(lds[0] + PL * BM * BK, qmul);
    }
    __syncthreads();
    int cur = 0;
    for (int kt = kt0; kt < kt1; ++kt) {
        if (kt + 1 < kt1) fetch(kt + 1);                           // on its way while this tile is multiplied
        const H *lp = lds[cur], *lq = lds[cur] + PL * BM * BK;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            uint4 fp[TM], fq[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) fp[i] = SP::frag(lp, (wm * TM + i) * 16, kk);
#pragma unroll
            for (int j = 0; j < TN; ++j) fq[j] = SQ::frag(lq, (wn * TN + j) * 16, kk);
            if constexpr (PL == 2) {
                uint4 fl[TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) fl[j] = SQ::frag(lq + SQ::PLANE, (wn * TN + j) * 16, kk);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = mma(fl[j], fp[i], acc[i][j], H{});
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const uint4 pl = SP::frag(lp + SP::PLANE, (wm * TM + i) * 16, kk);
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = mma(fq[j], pl, acc[i][j], H{});
                }
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mma(fq[j], fp[i], acc[i][j], H{});
        }
        if (kt + 1 < kt1) {
            sP.put(lds[cur ^ 1], pmul);
            sQ.put(lds[cur ^ 1] + PL * BM * BK, qmul);
        }
        __syncthreads();
        cur ^= 1;
    }
    // lane: row m = lane % 16 of a tile, columns n = 4 (lane / 16) ... + 3
    float top = 0.f;
    auto put4 = [&](void *base, int64_t at, int left, const float *v) {
        T *p = static_cast<T *>(base) + at;
        if (left >= 4) {
            if constexpr (sizeof(T) == 4) {
                Vec16<float>::store(p, v);
            } else {
                T o[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
                __builtin_memcpy(p, o, 8);
            }
        } else {
            for (int k = 0; k < left; ++k) p[k] = (T)v[k];
        }
    };
    auto get4 = [&](const void *base, int64_t at, int left, float *v) {
        const T *p = static_cast<const T *>(base) + at;
        if (left >= 4) {
            T o[4];
            __builtin_memcpy(o, p, 4 * sizeof(T));
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = (float)o[k];
        } else {
            for (int k = 0; k < 4; ++k) v[k] = k < left ? (float)p[k] : 0.f;
        }
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = m0 + (wm * TM + i) * 16 + (lane & 15);
        constexpr int JN = EPI == EPI_DUAL ? TN / 2 : TN;
#pragma unroll
        for (int j = 0; j < JN; ++j) {
            const int n = n0 + (wn * JN + j) * 16 + 4 * (lane >> 4), left = a.N - n;
            if (m >= a.M || left <= 0) continue;
            const int64_t at = (int64_t)m * a.ldc + n;
            float v[4], w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = PL == 2 ? ldexpf(acc[i][j][k], unshift) : acc[i][j][k];
            if constexpr (EPI == EPI_DUAL) {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = PL == 2 ? ldexpf(acc[i][j + JN][k], unshift) : acc[i][j + JN][k];
                if (a.bias) {
                    float b[4];
                    get4(a.bias, n, left, b);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] += b[k];
                }
                if (a.bias2) {
                    float b[4];
                    get4(a.bias2, n, left, b);
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] += b[k];
                }
                if (a.C2) {
                    put4(a.C2, at, left, v);
                    put4(a.C3, at, left, w);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[k] = act_value(v[k], a.act) * w[k];
                    if (k < left) top = fmaxf(top, fabsf(v[k]));
                }
                put4(a.C, at, left, v);
            } else if constexpr (EPI == EPI_DH) {
                float g[4], u[4];
                get4(a.g, at, left, g);
                get4(a.u, at, left, u);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    w[k] = v[k] * act_value(g[k], a.act);
                    v[k] = v[k] * u[k] * act_slope(g[k], a.act);
                    if (k < left) top = fmaxf(top, fmaxf(fabsf(v[k]), fabsf(w[k])));
                }
                put4(a.C, at, left, v);
                put4(a.C2, at, left, w);
            } else {
                if (a.parts) {
                    float *p = a.parts + ((int64_t)(zz * a.splits + sp) * a.M + m) * a.N + n;
                    if (left >= 4) Vec16<float>::store(p, v);
                    else for (int k = 0; k < left; ++k) p[k] = v[k];
                } else {
                    if (a.bias) {
                        float b[4];
                        get4(a.bias, n, left, b);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] += b[k];
                    }
                    put4(zz ? a.C2 : a.C, at, left, v);
                }
            }
        }
    }
    if constexpr (PL == 2 && EPI != EPI_PLAIN) {
        if (a.slot_out >= 0) {
            top = wave_max(top);
            if (lane == 0) atomicMax(a.amax + a.slot_out * 64 + (blockIdx.x & 63), __float_as_uint(top));
        }
    }
}

// partial products -> the product, in ascending order of the splits; z outputs
template <typename T>
__global__ __launch_bounds__(256) void ffn_join_kernel(const float *__restrict__ parts, int splits, int64_t n, T *c0, T *c1) {
    const float *p = parts + (int64_t)blockIdx.y * splits * n;
    T *c = blockIdx.y ? c1 : c0;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        const bool whole = i + 4 <= n;
        for (int k = 0; k < splits; ++k) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            const float *q = p + (int64_t)k * n + i;
            if (whole) Vec16<float>::unpack(Vec16<float>::raw(q), v);
            else for (int e = 0; e < 4 && i + e < n; ++e) v[e] = q[e];
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) c[i + e] = (T)s[e];
    }
}

// column sums (bias gradients): a block adds its rows of 64 columns (4 row lanes), the second launch adds the blocks' partials
template <typename T>
__global__ __launch_bounds__(256) void ffn_colsum_kernel(const T *__restrict__ x, int64_t T_, int N, int64_t rows, float *__restrict__ parts) {
    __shared__ float sh[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), l = threadIdx.x >> 6;
    const int64_t r0 = (int64_t)blockIdx.y * rows, r1 = min(T_, r0 + rows);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < N) {
        int64_t r = r0 + l;
        for (; r + 12 < r1; r += 16)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += (float)x[(r + 4 * k) * N + c];
        for (; r < r1; r += 4) s[0] += (float)x[r * N + c];
    }
    sh[l][threadIdx.x & 63] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (l == 0 && c < N) parts[(int64_t)blockIdx.y * N + c] = (sh[0][threadIdx.x] + sh[1][threadIdx.x]) + (sh[2][threadIdx.x] + sh[3][threadIdx.x]);
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------------------------
// A block owns 16 rows of the weights (of Wg and of Wu: NW = 2; of Wd: NW = 1); its 8 waves share the contraction; lane l reads 16 bytes of row
// l % 16, which is the matrix pipe's operand layout; tokens are the other operand, 16 at a time.  fp32 runs on v_mfma_f32_16x16x4_f32: 4 steps
// take the 4 values of a lane (both operands permute k alike).
struct FewArgs {
    const void *x, *w0, *w1, *b0, *b1;
    void *out;
    int M, N, K, act;
    int64_t ldx, ldw, ldo;
};
template <typename T, int NW, int MT>
__global__ __launch_bounds__(512) void ffn_few_kernel(FewArgs a) {
    constexpr int V = 16 / sizeof(T), STEP = 4 * V, U = 4;         // values of a lane, k of a step, steps in flight
    __shared__ f32x4 red[8][NW * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 16;
    const int row = min(n0 + (lane & 15), a.N - 1);
    const T *w[2] = {static_cast<const T *>(a.w0) + (int64_t)row * a.ldw, static_cast<const T *>(NW == 2 ? a.w1 : a.w0) + (int64_t)row * a.ldw};
    const T *x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = static_cast<const T *>(a.x) + (int64_t)min(t * 16 + (lane & 15), a.M - 1) * a.ldx;
    f32x4 acc[NW][MT];
#pragma unroll
    for (int s = 0; s < NW; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[s][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = (a.K + STEP - 1) / STEP, per = (steps + 7) / 8, s0 = wave * per, s1 = min(steps, s0 + per);
    auto fma1 = [&](const uint4 &p, const uint4 &q, f32x4 c) {
        if constexpr (sizeof(T) == 4) {
            float pv[4], qv[4];
            Vec16<float>::unpack(p, pv);
            Vec16<float>::unpack(q, qv);
#pragma unroll
            for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(pv[k], qv[k], c, 0, 0, 0);
            return c;
        } else {
            return mma(p, q, c, T{});
        }
    };
    int st = s0;
    for (; st + U <= s1 && (st + U) * STEP <= a.K; st += U) {
        uint4 wv[U][NW], xv[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (st + u) * STEP + V * (lane >> 4);
#pragma unroll
            for (int s = 0; s < NW; ++s) wv[u][s] = Vec16<T>::raw(w[s] + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) xv[u][t] = Vec16<T>::raw(x[t] + k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < NW; ++s)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[s][t] = fma1(wv[u][s], xv[u][t], acc[s][t]);
    }
    for (; st < s1; ++st) {
        const int k = st * STEP + V * (lane >> 4), left = max(0, min(V, a.K - k)), kk = left ? k : 0;
        uint4 xv[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[t] = Vec16<T>::raw_part(x[t] + kk, left);
#pragma unroll
        for (int s = 0; s < NW; ++s) {
            const uint4 wv = Vec16<T>::raw_part(w[s] + kk, left);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[s][t] = fma1(wv, xv[t], acc[s][t]);
        }
    }
#pragma unroll
    for (int s = 0; s < NW; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) red[wave][s * MT + t][lane] = acc[s][t];
    __syncthreads();
    // wave t adds token tile t over the 8 waves in ascending order
    for (int t = wave; t < MT; t += 8) {
        f32x4 v[NW];
#pragma unroll
        for (int s = 0; s < NW; ++s) {
            v[s] = red[0][s * MT + t][lane];
            for (int k = 1; k < 8; ++k) v[s] += red[k][s * MT + t][lane];
        }
        const int m = t * 16 + (lane & 15), n = n0 + 4 * (lane >> 4);
        if (m < a.M)
            for (int k = 0; k < 4; ++k)
                if (n + k < a.N) {
                    float o = v[0][k] + (a.b0 ? (float)static_cast<const T *>(a.b0)[n + k] : 0.f);
                    if constexpr (NW == 2) o = act_value(o, a.act) * (v[1][k] + (a.b1 ? (float)static_cast<const T *>(a.b1)[n + k] : 0.f));
                    static_cast<T *>(a.out)[(int64_t)m * a.ldo + n + k] = (T)o;
                }
    }
}
template <typename T, int NW>
void few_launch(const FewArgs &a, hipStream_t st) {
    const dim3 g((unsigned)((a.N + 15) / 16)), b(512);
    if (a.M <= 16) hipLaunchKernelGGL((ffn_few_kernel<T, NW, 1>), g, b, 0, st, a);
    else if (a.M <= 32) hipLaunchKernelGGL((ffn_few_kernel<T, NW, 2>), g, b, 0, st, a);
    else hipLaunchKernelGGL((ffn_few_kernel<T, NW, 4>), g, b, 0, st, a);
}

template <typename T, bool PA, bool QA, int EPI>
int gemm_launch(GemmArgs a, hipStream_t st) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64, BM = 128, BN = 128, BNC = EPI == EPI_DUAL ? BN / 2 : BN;
    a.tiles_m = (a.M + BM - 1) / BM;
    a.tiles_n = (a.N + BNC - 1) / BNC;
    const int64_t blocks = (int64_t)a.tiles_m * a.tiles_n * a.splits * a.z;
    if (blocks > 0x7fffffff) return NMRF_EINVAL;
    hipLaunchKernelGGL((ffn_gemm_kernel<T, BM, BN, 2, 2, BK, PA, QA, EPI>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    return nmrf_launch_status();
}

struct FfnShape { int64_t T; int D, F, Do; };
bool ffn_bad(const FfnShape &s, int dtype, int act) {
    // (offsets inside a tile are 32-bit: 128 rows of 2^22 elements)
    return s.T < 0 || s.T > 0x7fffffff - 256 || s.D < 1 || s.F < 1 || s.Do < 1 || s.D > 1 << 22 || s.F > 1 << 22 || s.Do > 1 << 22 ||
           dtype < NMRF_F32 || dtype > NMRF_F16 || act < 0 || act > 2;
}
bool ffn_misaligned(std::initializer_list<const void *> ps, int dtype) {
    uintptr_t o = 0;
    for (const void *p : ps) o |= reinterpret_cast<uintptr_t>(p);
    return o & (dtype == NMRF_F32 ? 3 : 1);
}
int absmax(const float *const *p, const int64_t *n, const int *slot, int count, unsigned *amax, int zero, hipStream_t st) {
    AbsmaxArgs a{};
    for (int i = 0; i < count; ++i) { a.p[i] = p[i]; a.n[i] = n[i]; a.slot[i] = slot[i]; }
    a.out = amax;
    hipLaunchKernelGGL(ffn_zero_kernel, dim3(NSLOT), dim3(64), 0, st, amax, zero);
    if (count) hipLaunchKernelGGL(ffn_absmax_kernel, dim3(256, (unsigned)count), dim3(256), 0, st, a);
    return nmrf_launch_status();
}

template <typename T>
int ffn_forward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, const void *bg, const void *bu, const void *bd,
                int act, void *h, void *g, void *u, void *y, unsigned *amax, hipStream_t st) {
    if (s.T <= 64 && !g) {
        FewArgs f{x, wg, wu, bg, bu, h, (int)s.T, s.F, s.D, act, s.D, s.D, s.F};
        few_launch<T, 2>(f, st);
        FewArgs d{h, wd, wd, bd, nullptr, y, (int)s.T, s.Do, s.F, act, s.F, s.F, s.Do};
        few_launch<T, 1>(d, st);
        return nmrf_launch_status();
    }
    if constexpr (sizeof(T) == 4) {
        const float *p[4] = {(const float *)x, (const float *)wg, (const float *)wu, (const float *)wd};
        const int64_t n[4] = {s.T * s.D, (int64_t)s.F * s.D, (int64_t)s.F * s.D, (int64_t)s.Do * s.F};
        const int slot[4] = {SLOT_X, SLOT_W, SLOT_W, SLOT_WD};
        const int rc = absmax(p, n, slot, 4, amax, 1 << SLOT_X | 1 << SLOT_W | 1 << SLOT_WD | 1 << SLOT_H, st);
        if (rc != NMRF_OK) return rc;
    }
    GemmArgs a{};
    a.P[0] = x; a.Q[0] = wg; a.Q[1] = wu; a.ldp = a.ldq = s.D; a.ldc = s.F;
    a.M = (int)s.T; a.N = s.F; a.K = s.D; a.segs = 1; a.splits = 1; a.z = 1;
    a.C = h; a.C2 = g; a.C3 = u; a.bias = bg; a.bias2 = bu; a.act = act; a.amax = amax; a.slot_p = SLOT_X; a.slot_q = SLOT_W; a.slot_out = SLOT_H;
    int rc = gemm_launch<T, true, true, EPI_DUAL>(a, st);
    if (rc != NMRF_OK) return rc;
    GemmArgs b{};
    b.P[0] = h; b.Q[0] = wd; b.ldp = b.ldq = s.F; b.ldc = s.Do;
    b.M = (int)s.T; b.N = s.Do; b.K = s.F; b.segs = 1; b.splits = 1; b.z = 1;
    b.C = y; b.bias = bd; b.amax = amax; b.slot_p = SLOT_H; b.slot_q = SLOT_WD; b.slot_out = -1;
    return gemm_launch<T, true, true, EPI_PLAIN>(b, st);
}

// weight gradient: z products P_z^T Q over all T tokens, the contraction split until the chip is full
int wgrad_splits(int64_t T, int M, int N, int z, int bk) {
    const int64_t tiles = (int64_t)((M + 127) / 128) * ((N + 127) / 128) * z, ktiles = (T + bk - 1) / bk;
    int64_t s = tiles >= 384 ? 1 : 768 / tiles;
    if (s > ktiles / 4) s = ktiles / 4;
    return (int)(s < 1 ? 1 : s);
}
int64_t colsum_blocks(int64_t T) { return T < 2048 ? 1 : (T / 256 < 128 ? T / 256 : 128); }

template <typename T>
int wgrad(const void *p0, const void *p1, const void *q, int64_t tokens, int M, int N, void *c0, void *c1, float *ws, unsigned *amax, int slot_p, int slot_q,
          hipStream_t st) {
    GemmArgs a{};
    a.P[0] = p0; a.P[1] = p1; a.Q[0] = q; a.ldp = M; a.ldq = N; a.ldc = N;
    a.M = M; a.N = N; a.K = (int)tokens; a.segs = 1; a.z = p1 ? 2 : 1;
    a.C = c0; a.C2 = c1; a.amax = amax; a.slot_p = slot_p; a.slot_q = slot_q; a.slot_out = -1;
    a.splits = wgrad_splits(tokens, M, N, a.z, sizeof(T) == 4 ? 32 : 64);
    a.parts = a.splits > 1 ? ws : nullptr;
    const int rc = gemm_launch<T, false, false, EPI_PLAIN>(a, st);
    if (rc != NMRF_OK || a.splits == 1) return rc;
    const int64_t n = (int64_t)M * N;
    int64_t blocks = ceil_div64(n, 1024);
    if (blocks > 4096) blocks = 4096;
    hipLaunchKernelGGL(ffn_join_kernel<T>, dim3((unsigned)blocks, (unsigned)a.z), dim3(256), 0, st, ws, a.splits, n, (T *)c0, (T *)c1);
    return nmrf_launch_status();
}
template <typename T>
int colsum(const void *x, int64_t tokens, int N, void *out, float *ws, hipStream_t st) {
    const int64_t nb = colsum_blocks(tokens), rows = ceil_div64(tokens, nb);
    hipLaunchKernelGGL(ffn_colsum_kernel<T>, dim3((unsigned)((N + 63) / 64), (unsigned)nb), dim3(256), 0, st, (const T *)x, tokens, N, rows, ws);
    int64_t blocks = ceil_div64(N, 1024);
    hipLaunchKernelGGL(ffn_join_kernel<T>, dim3((unsigned)blocks, 1), dim3(256), 0, st, ws, (int)nb, (int64_t)N, (T *)out, (T *)nullptr);
    return nmrf_launch_status();
}

template <typename T>
int ffn_backward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, const void *h, const void *g, const void *u, const void *dy,
                 int act, void *dg, void *du, void *dx, void *dwg, void *dwu, void *dwd, void *dbg, void *dbu, void *dbd, unsigned *amax, float *ws,
                 hipStream_t st) {
    int rc;
    if constexpr (sizeof(T) == 4) {
        const float *p[1] = {(const float *)dy};
        const int64_t n[1] = {s.T * s.Do};
        const int slot[1] = {SLOT_DY};
        if ((rc = absmax(p, n, slot, 1, amax, 1 << SLOT_DY | 1 << SLOT_DG, st)) != NMRF_OK) return rc;
    }
    GemmArgs a{};
    a.P[0] = dy; a.Q[0] = wd; a.ldp = s.Do; a.ldq = s.F; a.ldc = s.F;
    a.M = (int)s.T; a.N = s.F; a.K = s.Do; a.segs = 1; a.splits = 1; a.z = 1;
    a.C = dg; a.C2 = du; a.g = g; a.u = u; a.act = act; a.amax = amax; a.slot_p = SLOT_DY; a.slot_q = SLOT_WD; a.slot_out = SLOT_DG;
    if ((rc = gemm_launch<T, true, false, EPI_DH>(a, st)) != NMRF_OK) return rc;
    if (dx) {
        GemmArgs b{};
        b.P[0] = dg; b.P[1] = du; b.Q[0] = wg; b.Q[1] = wu; b.ldp = s.F; b.ldq = s.D; b.ldc = s.D;
        b.M = (int)s.T; b.N = s.D; b.K = s.F; b.segs = 2; b.splits = 1; b.z = 1;
        b.C = dx; b.amax = amax; b.slot_p = SLOT_DG; b.slot_q = SLOT_W; b.slot_out = -1;
        if ((rc = gemm_launch<T, true, false, EPI_PLAIN>(b, st)) != NMRF_OK) return rc;
    }
    if (dwg && dwu) {
        if ((rc = wgrad<T>(dg, du, x, s.T, s.F, s.D, dwg, dwu, ws, amax, SLOT_DG, SLOT_X, st)) != NMRF_OK) return rc;
    } else if (dwg || dwu) {
        if ((rc = wgrad<T>(dwg ? dg : du, nullptr, x, s.T, s.F, s.D, dwg ? dwg : dwu, nullptr, ws, amax, SLOT_DG, SLOT_X, st)) != NMRF_OK) return rc;
    }
    if (dwd && (rc = wgrad<T>(dy, nullptr, h, s.T, s.Do, s.F, dwd, nullptr, ws, amax, SLOT_DY, SLOT_H, st)) != NMRF_OK) return rc;
    if (dbg && (rc = colsum<T>(dg, s.T, s.F, dbg, ws, st)) != NMRF_OK) return rc;
    if (dbu && (rc = colsum<T>(du, s.T, s.F, dbu, ws, st)) != NMRF_OK) return rc;
    if (dbd && (rc = colsum<T>(dy, s.T, s.Do, dbd, ws, st)) != NMRF_OK) return rc;
    return NMRF_OK;
}

}  // namespace

extern "C" int nmrf_gated_ffn(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *b_gate, const void *b_up,
                              const void *b_down, int64_t T, int D, int F, int Do, int dtype, int act, void *h, void *g, void *u, void *y,
                              uint32_t *amax, void *stream) {
    const FfnShape s{T, D, F, Do};
    if (ffn_bad(s, dtype, act)) return NMRF_EINVAL;
    if (T == 0) return NMRF_OK;
    if (!x || !w_gate || !w_up || !w_down || !h || !y || (dtype == NMRF_F32 && !amax)) return NMRF_ENULL;
    if ((g == nullptr) != (u == nullptr) || ffn_misaligned({x, w_gate, w_up, w_down, b_gate, b_up, b_down, h, g, u, y}, dtype)) return NMRF_EINVAL;
    if (reinterpret_cast<uintptr_t>(amax) & 3) return NMRF_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NMRF_F32) return ffn_forward<float>(s, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, h, g, u, y, amax, st);
    if (dtype == NMRF_BF16) return ffn_forward<__bf16>(s, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, h, g, u, y, amax, st);
    return ffn_forward<_Float16>(s, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, h, g, u, y, amax, st);
}

extern "C" int nmrf_gated_ffn_bwd_size(int64_t T, int D, int F, int Do, int dtype, int64_t *floats) {
    if (!floats) return NMRF_ENULL;
    if (ffn_bad(FfnShape{T, D, F, Do}, dtype, 0) || T < 1) return NMRF_EINVAL;
    const int bk = dtype == NMRF_F32 ? 32 : 64;
    int64_t n = 0;
    const int s2 = wgrad_splits(T, F, D, 2, bk), s1 = wgrad_splits(T, F, D, 1, bk), sd = wgrad_splits(T, Do, F, 1, bk);
    const int64_t a = s2 > 1 ? 2 * (int64_t)s2 * F * D : 0, b = s1 > 1 ? (int64_t)s1 * F * D : 0, c = sd > 1 ? (int64_t)sd * Do * F : 0;
    n = a > b ? a : b;
    n = n > c ? n : c;
    const int64_t cs = colsum_blocks(T) * (int64_t)(F > Do ? F : Do);
    *floats = n > cs ? n : cs;
    return NMRF_OK;
}

extern "C" int nmrf_gated_ffn_bwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *h, const void *g, const void *u,
                                  const void *dy, int64_t T, int D, int F, int Do, int dtype, int act, void *dg, void *du, void *dx, void *dw_gate,
                                  void *dw_up, void *dw_down, void *db_gate, void *db_up, void *db_down, uint32_t *amax, float *ws,
                                  int64_t ws_floats, void *stream) {
    const FfnShape s{T, D, F, Do};
    if (ffn_bad(s, dtype, act) || T < 1) return NMRF_EINVAL;
    if (!x || !w_gate || !w_up || !w_down || !h || !g || !u || !dy || !dg || !du || !ws || (dtype == NMRF_F32 && !amax)) return NMRF_ENULL;
    if (ffn_misaligned({x, w_gate, w_up, w_down, h, g, u, dy, dg, du, dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down}, dtype)) return NMRF_EINVAL;
    if ((reinterpret_cast<uintptr_t>(amax) | reinterpret_cast<uintptr_t>(ws)) & 3) return NMRF_EINVAL;
    int64_t need = 0;
    const int rc = nmrf_gated_ffn_bwd_size(T, D, F, Do, dtype, &need);
    if (rc != NMRF_OK || need > ws_floats) return NMRF_EINVAL;
    hipStream_t st = (hipStream_t)stream;
#define NMRF_FFN_BWD(TYPE) ffn_backward<TYPE>(s, x, w_gate, w_up, w_down, h, g, u, dy, act, dg, du, dx, dw_gate, dw_up, dw_down, db_gate, db_up, \
                                              db_down, amax, ws, st)
    if (dtype == NMRF_F32) return NMRF_FFN_BWD(float);
    if (dtype == NMRF_BF16) return NMRF_FFN_BWD(__bf16);
    return NMRF_FFN_BWD(_Float16);
#undef NMRF_FFN_BWD
}
