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
//
// Measured (kernel time): bf16, T = 8 192, D = 2 048, F = 5 504: both projections 549 us (369 GFLOP, 673 TFLOP/s), the second matrix 218 us (848),
// dg and du 439 us (420: 541 MB of g, u, dg and du go through its epilogue), dx 369 us (1 001), weight gradients 722 us (767).  fp32, T = 29 952,
// D = 128, F = 512: 102, 36, 91, 57 and 60 us (43 to 198 TFLOP/s of fp32 work, three products each).  One token, bf16, D = 4 096,
// F = 11 008: 33 + 20 us (270 MB, 5.1 TB/s); 16 tokens 39 + 29, 64 tokens 81 + 62; in fp32 one token 70 + 41 (541 MB, 4.9 TB/s), 64 tokens
// 203 + 132 (four k steps of v_mfma_f32_16x16x4_f32 for every 16-byte load).
#include "common.h"
#include "elem.h"
#include <algorithm>
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

// act(g) and its derivative.  gelu: Phi(g) from erfc(|g| / sqrt 2) = 2^(-t P(t)), t = min(|g|, 7), the polynomial of gelu_fast (common.h: off by
// 5.3e-8 in Phi's scale), one more exponential for the density in the derivative.  Below -7 the value is zero (g Phi(g) > -9e-12; Phi held at
// its value at -7 would come back times any g), the slope held (-6e-11).
enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
__device__ __forceinline__ void act_both(float g, int act, float &value, float &slope) {
    if (act == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + exp_of(-g));  // (1 ulp; a division is ten instructions a hidden value)
        value = g == -INFINITY ? 0.f : g * s;
        slope = fmaf(value, 1.0f - s, s);
    } else if (act == ACT_GELU) {
        const float t = fminf(fabsf(g), 7.0f);
        float p = fmaf(-3.0177725420799106e-05f, t, 0.0007414184510707855f);
        p = fmaf(p, t, -0.007980725727975368f);
        p = fmaf(p, t, 0.053240980952978134f);
        p = fmaf(p, t, 0.45891475677490234f);
        p = fmaf(p, t, 1.151147484779358f);
        const float half = 0.5f * __builtin_amdgcn_exp2f(-t * p), phi = g < 0.f ? half : 1.0f - half;
        value = g < -7.0f ? 0.f : g * phi;
        slope = fmaf(t * (g < 0.f ? -0.39894228040143267794f : 0.39894228040143267794f), exp_of(-0.5f * t * t), phi);
        if (g != g) value = slope = g;
    } else {
        value = g > 0.f ? g : (g != g ? g : 0.f);
        slope = g > 0.f ? 1.f : 0.f;
    }
}
__device__ __forceinline__ float act_value(float g, int act) {
    float v, s;
    act_both(g, act, v, s);
    return v;
}

// ---- largest magnitudes (fp32 operands): per tensor 256 slots, of which a product takes the maximum --------------------------------------
enum { SLOT_X = 0, SLOT_WG = 1, SLOT_WU = 2, SLOT_WD = 3, SLOT_H = 4, SLOT_DY = 5, SLOT_DG = 6 };
// (values that are not finite do not count: they spoil their own row whatever the scale, and must not take the others' bits)
__device__ __forceinline__ float magnitude(float v) {
    v = fabsf(v);
    return v < INFINITY ? v : 0.f;
}
struct AbsmaxArgs { const float *p[5]; int64_t n[5]; int slot[5]; unsigned *out; };      // p null: clear the slot (a later kernel fills it)
__global__ __launch_bounds__(256) void ffn_absmax_kernel(AbsmaxArgs a) {
    __shared__ float sh[4];
    const int which = blockIdx.y;
    const float *p = a.p[which];
    const int64_t n = p ? a.n[which] : 0, per = (n + 1023) / 1024 * 4, i0 = blockIdx.x * per, i1 = min(n, i0 + per);
    float m[4] = {0.f, 0.f, 0.f, 0.f};
    int64_t i = i0 + threadIdx.x * 4;
    for (; i + 3076 <= i1; i += 4096) {                            // four loads in flight
        float v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u) Vec16<float>::unpack(Vec16<float>::raw(p + i + 1024 * u), v[u]);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) m[k] = fmaxf(m[k], magnitude(v[u][k]));
    }
    for (; i < i1; i += 1024)
        for (int k = 0; k < 4 && i + k < i1; ++k) m[k] = fmaxf(m[k], magnitude(p[i + k]));
    float x = wave_max(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) a.out[a.slot[which] * 256 + blockIdx.x] = __float_as_uint(fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3])));
}
// the power of two that puts the largest magnitude at [2^13, 2^14), 0 where all are zero
__device__ __forceinline__ int slot_shift(const unsigned *amax, int slot, int count) {
    float m = 0.f;
    for (int i = threadIdx.x & 63; i < 256 * count; i += 64) m = fmaxf(m, __uint_as_float(amax[slot * 256 + i]));
    m = wave_max(m);
    if (!(m > 0.f)) return 0;
    const int e = (int)((__float_as_uint(m) >> 23) & 0xffu) - 127, sh = 13 - (e < -100 ? -100 : e);
    return __builtin_amdgcn_readfirstlane(sh);
}

// ---- the tile kernel ----------------------------------------------------------------------------------------------------------------------
//     C[m, n] = sum over segments s and k of P_s[m, k] Q_s[n, k]
// An operand lies ALONG k (row m: k contiguous, stride ld) or ACROSS it (row k: m contiguous, stride ld).
enum { EPI_DUAL = 0, EPI_PLAIN = 1, EPI_DH = 2 };
struct Problem {
    const void *P[2], *Q[2];                     // the segments of a contraction (EPI_DUAL: Q = Wg, Wu)
    int64_t ldp, ldq, ldc;
    int M, N, K, segs;                           // K of one segment
    void *C, *C2, *C3;                           // EPI_DUAL: h, g, u (C2, C3 fp32, may be null); EPI_PLAIN: the product; EPI_DH: dg, du in C, C2
    const float *g, *u;                          // EPI_DH
    const void *bias, *bias2;
    float *parts;                                // EPI_PLAIN with splits > 1: fp32 partial products [splits][M][N]
    float *sum1, *sum2;                          // EPI_DH: column sums of dg, du over each wave's rows, [2 tiles_m][N] (may be null)
    int slot_p, slot_q, slot_out;                // fp32: slots of the operands' and the output's largest magnitudes (slot_out -1: none)
    int splits, tiles_m, tiles_n, blocks;
};
struct GemmArgs {
    Problem p[3];                                // side by side in one launch
    int count, act;
    unsigned *amax;
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
    unsigned off[N];                                               // byte offsets of the chunks from the tile's first value: they do not change with k
    // ALONG: of_row(i): the matrix row of tile row i (a row behind the last is read as another one: its products are not stored)
    template <typename OfRow> __device__ __forceinline__ void init(int ld, int rows, OfRow of_row) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int id = threadIdx.x + n * THREADS, i = id / CPR, c = id % CPR * 8;
            off[n] = (unsigned)(ALONG ? of_row(i) * ld + c : i * ld + (c < rows ? c : 0)) * (unsigned)sizeof(T);
        }
    }
    // base_of(i): the tile's first value and the end of its tensor (by tile row: two matrices may share a tile); left: values of k from there on
    template <typename BaseOf>
    __device__ __forceinline__ void load(int ld, int rows, int left, BaseOf base_of) {
        // ACROSS reads over a row's end into the rows behind it (8 of them hold 8 values whatever their width) unless the rows end with a chunk
        if (left >= (ALONG || (rows & 7) == 0 ? BK : BK + 8)) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const T *end, *p = base_of((threadIdx.x + n * THREADS) / CPR, end);
                const char *q = reinterpret_cast<const char *>(p) + off[n];
#pragma unroll
                for (int v = 0; v < V; ++v) __builtin_memcpy(&r[n][v], q + 16 * v, 16);
            }
            return;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {                              // the last tile: a value of k behind the last is zero
            const int id = threadIdx.x + n * THREADS, i = id / CPR, c = id % CPR * 8;
            const T *end, *p = base_of(i, end);
            p += ALONG ? off[n] / sizeof(T) : (unsigned)((i < left ? i : 0) * ld + (c < rows ? c : 0));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const T *q = p + v * (8 / V);
                r[n][v] = Vec16<T>::raw_masked(q, ALONG ? max(0, left - c - v * (8 / V)) : (i < left ? 8 : 0), end - q);
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
__global__ __launch_bounds__(64 * WM * WN, 2) void ffn_gemm_kernel(GemmArgs args) {
    using H = Half<T>;
    constexpr int THREADS = 64 * WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, PL = sizeof(T) == 4 ? 2 : 1;
    using SP = Stage<T, BM, BK, PA, THREADS>;
    using SQ = Stage<T, BN, BK, QA, THREADS>;
    __shared__ __align__(16) H lds[2][PL * (BM + BN) * BK];
    int bid = blockIdx.x, which = 0;
    while (which + 1 < args.count && bid >= args.p[which].blocks) bid -= args.p[which++].blocks;
    const Problem &a = args.p[which];
    // blocks go to the 8 XCDs in turn: give each one a run of neighbouring tiles (its L2 then holds their operands), 8 row tiles deep
    const int per_split = a.tiles_m * a.tiles_n, q8 = a.blocks >> 3, rem = a.blocks & 7, xcd = bid & 7;
    int t = xcd * q8 + min(xcd, rem) + (bid >> 3);
    const int sp = t / per_split;
    t -= sp * per_split;
    const int band = t / (8 * a.tiles_n), deep = min(8, a.tiles_m - band * 8), in_band = t - band * 8 * a.tiles_n;
    const int tm = band * 8 + in_band % deep, tn = in_band / deep;
    constexpr int BNC = EPI == EPI_DUAL ? BN / 2 : BN;             // columns of the result
    const int m0 = tm * BM, n0 = tn * BNC;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN, lane = threadIdx.x & 63;

    float pmul = 1.f, qmul = 1.f;
    int unshift = 0;
    if constexpr (PL == 2) {
        const int sp_ = slot_shift(args.amax, a.slot_p, 1), sq_ = slot_shift(args.amax, a.slot_q, a.slot_q == SLOT_WG ? 2 : 1);
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
        const int seg = kt / ktiles_seg, k0 = (kt - seg * ktiles_seg) * BK, left = a.K - k0;
        const T *P = static_cast<const T *>(seg ? a.P[1] : a.P[0]);
        const T *Q = static_cast<const T *>(EPI != EPI_DUAL && seg ? a.Q[1] : a.Q[0]);
        const T *pb = P + (PA ? (int64_t)m0 * a.ldp + k0 : (int64_t)k0 * a.ldp + m0), *pe = P + (int64_t)(PA ? a.M : a.K) * a.ldp;
        sP.load((int)a.ldp, prow, left, [&](int, const T *&end) { end = pe; return pb; });
        const int64_t qo = QA ? (int64_t)n0 * a.ldq + k0 : (int64_t)k0 * a.ldq + n0, qn = (int64_t)(QA ? a.N : a.K) * a.ldq;
        const T *Q1 = static_cast<const T *>(a.Q[1]);
        sQ.load((int)a.ldq, qrow, left, [&](int i, const T *&end) {
            const T *q = EPI == EPI_DUAL && i / 16 % TN >= TN / 2 ? Q1 : Q;
            end = q + qn;
            return q + qo;
        });
    };
    sP.init((int)a.ldp, prow, [&](int i) { return min(i, prow - 1); });
    // (EPI_DUAL: of a wave's 16-column tiles the first half are Wg's rows, the second half Wu's)
    sQ.init((int)a.ldq, qrow, [&](int i) { return min(EPI == EPI_DUAL ? i / (TN * 16) * (TN * 8) + i / 16 % (TN / 2) * 16 + i % 16 : i, qrow - 1); });
    constexpr int JN = EPI == EPI_DUAL ? TN / 2 : TN, GM = EPI == EPI_DH ? TM : 1, GJ = EPI == EPI_DH ? TN : 1, EARLY = EPI == EPI_DH && TN == 2 ? 2 : 0;
    // EPI_DH: g and u of a tile that lies inside, all before the first store (a load between stores is waited for by itself): before the contraction
    // where the registers hold them beside it (64 x 64), else behind it
    const bool inside = EPI == EPI_DH && m0 + BM <= a.M && n0 + BN <= a.N;
    uint4 gw[GJ][GM], uw[GJ][GM];
    typedef unsigned w4 __attribute__((ext_vector_type(4), aligned(4)));
    auto once = [&](const float *p) { return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const w4 *>(p))); };
    auto ask = [&](int j) {
#pragma unroll
        for (int i = 0; i < GM; ++i) {
            const int64_t at = (int64_t)(m0 + (wm * TM + i) * 16 + (lane & 15)) * a.ldc + n0 + (wn * JN + j) * 16 + 4 * (lane >> 4);
            gw[j][i] = once(a.g + at);
            uw[j][i] = once(a.u + at);
        }
    };
    if (EARLY && inside)
#pragma unroll
        for (int j = 0; j < EARLY; ++j) ask(j);
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
        if constexpr (PL == 1) {
            // two fragments of P ahead of the products, Q's next ones half way: the LDS is read under the matrix pipe
            constexpr int S = BK / 32 * TM;
            uint4 fq[2][TN], fp[4];
#pragma unroll
            for (int j = 0; j < TN; ++j) fq[0][j] = SQ::frag(lq, (wn * TN + j) * 16, 0);
            fp[0] = SP::frag(lp, wm * TM * 16, 0);
            fp[1] = SP::frag(lp, (wm * TM + 1) * 16, 0);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const int kk = s / TM, i = s % TM;
                if (s + 2 < S) fp[(s + 2) & 3] = SP::frag(lp, (wm * TM + (s + 2) % TM) * 16, (s + 2) / TM);
                if (i == TM / 2 && kk + 1 < BK / 32)
#pragma unroll
                    for (int j = 0; j < TN; ++j) fq[(kk + 1) & 1][j] = SQ::frag(lq, (wn * TN + j) * 16, kk + 1);
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mma(fq[kk & 1][j], fp[s & 3], acc[i][j], H{});
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < BK / 32; ++kk) {
                uint4 fp[TM], fq[TN], fl[TN];
#pragma unroll
                for (int i = 0; i < TM; ++i) fp[i] = SP::frag(lp, (wm * TM + i) * 16, kk);
#pragma unroll
                for (int j = 0; j < TN; ++j) fl[j] = SQ::frag(lq + SQ::PLANE, (wn * TN + j) * 16, kk);
#pragma unroll
                for (int j = 0; j < TN; ++j) fq[j] = SQ::frag(lq, (wn * TN + j) * 16, kk);
                // the small products first: lo hi, hi lo, hi hi
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
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = mma(fq[j], fp[i], acc[i][j], H{});
            }
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
    auto putf = [&](float *p, int left, const float *v) {
        if (left >= 4) Vec16<float>::store(p, v);
        else for (int k = 0; k < left; ++k) p[k] = v[k];
    };
    typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
    auto putn = [&](float *p, int left, const float *v) {
        if (left >= 4) __builtin_nontemporal_store(f4u{v[0], v[1], v[2], v[3]}, reinterpret_cast<f4u *>(p));
        else for (int k = 0; k < left; ++k) p[k] = v[k];
    };
    auto getf = [&](const float *p, int left, float *v) {
        if (left >= 4) Vec16<float>::unpack(Vec16<float>::raw(p), v);
        else for (int k = 0; k < 4; ++k) v[k] = k < left ? p[k] : 0.f;
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
    if (EPI == EPI_DH && inside)
#pragma unroll
        for (int j = EARLY; j < JN; ++j) ask(j);
#pragma unroll
    for (int j = 0; j < JN; ++j) {
        const int n = n0 + (wn * JN + j) * 16 + 4 * (lane >> 4), left = a.N - n;
        float s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + (wm * TM + i) * 16 + (lane & 15);
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
                // (kept in fp32: rounded to 16 bits they would add a third to the gradients' error; past the caches, which then still hold h and,
                // behind the product that reads g and u, dg and du for the next one: T = 29 952 in fp32 380 -> 348 us (350 ... 361 since, by the caches), T = 8 192, D = 2 048 in
                // bf16 2 202 -> 2 151 us forward and backward; loads alone: 358, 2 172)
                if (a.C2) {
                    putn(static_cast<float *>(a.C2) + at, left, v);
                    putn(static_cast<float *>(a.C3) + at, left, w);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[k] = act_value(v[k], args.act) * w[k];
                    if (PL == 2 && k < left) top = fmaxf(top, magnitude(v[k]));
                }
                put4(a.C, at, left, v);
            } else if constexpr (EPI == EPI_DH) {
                float g[4], u[4];
                if (inside) {
                    Vec16<float>::unpack(gw[j][i], g);
                    Vec16<float>::unpack(uw[j][i], u);
                } else {
                    getf(a.g + at, left, g);
                    getf(a.u + at, left, u);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float value, slope;
                    act_both(g[k], args.act, value, slope);
                    w[k] = v[k] * value;
                    v[k] = v[k] * u[k] * slope;
                    if (PL == 2 && k < left) top = fmaxf(top, fmaxf(magnitude(v[k]), magnitude(w[k])));
                }
                put4(a.C, at, left, v);
                put4(a.C2, at, left, w);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s1[k] += v[k];
                    s2[k] += w[k];
                }
            } else {
                if (a.parts) {
                    putf(a.parts + ((int64_t)sp * a.M + m) * a.N + n, left, v);
                } else {
                    if (a.bias) {
                        float b[4];
                        get4(a.bias, n, left, b);
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] += b[k];
                    }
                    put4(a.C, at, left, v);
                }
            }
        }
        if constexpr (EPI == EPI_DH) {
            if (a.sum1 || a.sum2) {                                // bias gradients: over the wave's rows, 16 lanes of a row group
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s1[k] += NMRF_ROW_ROR(s1[k], 8);
                    s2[k] += NMRF_ROW_ROR(s2[k], 8);
                    s1[k] += NMRF_ROW_ROR(s1[k], 4);
                    s2[k] += NMRF_ROW_ROR(s2[k], 4);
                    s1[k] += NMRF_ROW_ROR(s1[k], 2);
                    s2[k] += NMRF_ROW_ROR(s2[k], 2);
                    s1[k] += NMRF_ROW_ROR(s1[k], 1);
                    s2[k] += NMRF_ROW_ROR(s2[k], 1);
                }
                if ((lane & 15) == 0 && left > 0) {
                    const int64_t at = (int64_t)(tm * WM + wm) * a.N + n;
                    if (a.sum1) putf(a.sum1 + at, left, s1);
                    if (a.sum2) putf(a.sum2 + at, left, s2);
                }
            }
        }
    }
    if constexpr (PL == 2 && EPI != EPI_PLAIN) {
        if (a.slot_out >= 0) {
            top = wave_max(top);
            if (lane == 0) atomicMax(args.amax + a.slot_out * 256 + (blockIdx.x & 255), __float_as_uint(top));
        }
    }
}

// partial results [splits][n] -> the results (the first one plus a bias of `cols` values), several in one launch: a block owns 32 values; its 32
// row lanes add the splits l, l + 32, ... and 32 threads the lane sums, in a fixed order (bias sums have a partial for every 32 or 64 rows of
// tokens and few columns: long chains want many lanes)
struct JoinArgs { const float *parts[7]; void *c[7]; int64_t n[7]; int splits[7], blocks[7]; const void *bias; int cols, count; };
template <typename T>
__global__ __launch_bounds__(256) void ffn_join_kernel(JoinArgs a) {
    __shared__ float sh[32][33];
    int bid = blockIdx.x, which = 0;
    while (which + 1 < a.count && bid >= a.blocks[which]) bid -= a.blocks[which++];
    const int64_t n = a.n[which];
    const int splits = a.splits[which], blocks = a.blocks[which];
    const float *p = a.parts[which];
    T *c = static_cast<T *>(a.c[which]);
    const void *bias = which ? nullptr : a.bias;
    const int l = threadIdx.x >> 3, q4 = (threadIdx.x & 7) * 4;
    for (int64_t i0 = (int64_t)bid * 32; i0 < n; i0 += (int64_t)blocks * 32) {
        const int64_t i = i0 + q4;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        if (i + 4 <= n) {
            int k = l;
            for (; k + 96 < splits; k += 128) {                    // four loads in flight
                float v[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) Vec16<float>::unpack(Vec16<float>::raw(p + (int64_t)(k + 32 * q) * n + i), v[q]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += (v[0][e] + v[1][e]) + (v[2][e] + v[3][e]);
            }
            for (; k < splits; k += 32) {
                float v[4];
                Vec16<float>::unpack(Vec16<float>::raw(p + (int64_t)k * n + i), v);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += v[e];
            }
        } else {
            for (int k = l; k < splits; k += 32)
                for (int e = 0; e < 4; ++e)
                    if (i + e < n) s[e] += p[(int64_t)k * n + i + e];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) sh[l][q4 + e] = s[e];
        __syncthreads();
        const int64_t j = i0 + threadIdx.x;
        if (threadIdx.x < 32 && j < n) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k & 3] += sh[k][threadIdx.x];
            float o = (v[0] + v[1]) + (v[2] + v[3]);
            if (bias) o += (float)static_cast<const T *>(bias)[j % a.cols];
            c[j] = (T)o;
        }
    }
}

// column sums of dy (dg's and du's come out of the kernel that makes them): a block adds its rows of 64 columns (16 row lanes of 16 column
// lanes), a join adds the blocks' partials
struct ColsumArgs { const void *x; float *parts; int cols; int64_t rows, per; };
template <typename T>
__global__ __launch_bounds__(256) void ffn_colsum_kernel(ColsumArgs a) {
    __shared__ float sh[16][65];
    const int N = a.cols, c = blockIdx.x * 64 + (threadIdx.x & 15) * 4, l = threadIdx.x >> 4;
    const T *x = static_cast<const T *>(a.x);
    const int64_t r0 = blockIdx.y * a.per, r1 = min(a.rows, r0 + a.per);
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c + 4 <= N) {
        int64_t r = r0 + l;
        for (; r + 48 < r1; r += 64) {                             // four loads in flight
            T v[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) __builtin_memcpy(v[k], x + (r + 16 * k) * N + c, 4 * sizeof(T));
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += ((float)v[0][e] + (float)v[1][e]) + ((float)v[2][e] + (float)v[3][e]);
        }
        for (; r < r1; r += 16) {
            T v[4];
            __builtin_memcpy(v, x + r * N + c, 4 * sizeof(T));
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += (float)v[e];
        }
    } else {
        for (int64_t r = r0 + l; r < r1; r += 16)
            for (int e = 0; e < 4 && c + e < N; ++e) s[e] += (float)x[r * N + c + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sh[l][(threadIdx.x & 15) * 4 + e] = s[e];
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.x * 64 + (int)threadIdx.x < N) {
        float v = sh[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 16; ++k) v += sh[k][threadIdx.x];
        a.parts[(int64_t)blockIdx.y * N + blockIdx.x * 64 + threadIdx.x] = v;
    }
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
    constexpr int V = 16 / sizeof(T), STEP = 4 * V, U = NW * MT == 1 ? 8 : 4;      // values of a lane, k of a step, steps in flight
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
    // whole steps, U at a time; those behind the last one read it again and count as zeros (a step by itself waits for memory by itself), and 8 in
    // flight for one matrix and one token tile, which have the registers: second matrix of one token, D = 4 096, F = 11 008, 27 -> 20 us
    const int whole = min(s1, a.K / STEP);
    int st = s0;
    for (; st < whole; st += U) {
        uint4 wv[U][NW], xv[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(st + u, whole - 1) * STEP + V * (lane >> 4);
#pragma unroll
            for (int s = 0; s < NW; ++s) wv[u][s] = Vec16<T>::raw(w[s] + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) xv[u][t] = Vec16<T>::raw(x[t] + k);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool on = st + u < whole;
#pragma unroll
            for (int t = 0; t < MT; ++t) xv[u][t] = on ? xv[u][t] : uint4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NW; ++s) {
                wv[u][s] = on ? wv[u][s] : uint4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[s][t] = fma1(wv[u][s], xv[u][t], acc[s][t]);
            }
        }
    }
    for (st = max(s0, whole); st < s1; ++st) {
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

// The tile of a launch.  fp32 with a short contraction (k <= 256): 64 x 64 -- loads, the split into halves and the epilogue outweigh the products,
// and five waves a SIMD cover each other where two do not (T = 29 952, D = 128: both projections 106 -> 102 us, dg and du 109 -> 90 us).
// 16-bit types with k >= 512: 256 x 256 (8 waves) where its rounds of 256 blocks cost less than those of 512 blocks of 128 x 128, a product of
// the large tile taking 0.77 (operand across: dx 505 -> 386 us at T = 8 192, D = 2 048, F = 5 504) to 0.86 of the time (weight gradients:
// 761 us in five rounds of the small one, 868 in three of the large) -- but not for dg and du, whose epilogue the one block a CU cannot hide
// (474 us with the small tile, 576 with the large).  Else 128 x 128 where it fills the chip, 64 x 64 where it does not (192 of the 256 CUs).  A plain
// product with too few tiles splits its contraction over about two blocks a CU, 4 k tiles each at least, and is joined by a second launch.
struct GemmPlan { int tile, tiles_m, tiles_n, splits; };
enum { PLAN_PLAIN, PLAN_DUAL, PLAN_DH };
// z: problems in the launch; tile: that of the launch, 0: to be chosen
GemmPlan gemm_plan(int64_t M, int64_t N, int64_t k, int z, int bk, int what, int tile) {
    GemmPlan p;
    auto tiles = [&](int t) {
        p.tile = t;
        p.tiles_m = (int)((M + t - 1) / t);
        p.tiles_n = (int)(what == PLAN_DUAL ? (N + t / 2 - 1) / (t / 2) : (N + t - 1) / t);
        return (int64_t)p.tiles_m * p.tiles_n * z;
    };
    const int64_t kt = (k + bk - 1) / bk;
    if (!tile && bk == 32 && k <= 256) tile = 64;
    if (!tile && bk == 64 && k >= 512 && what != PLAN_DH) {
        const int64_t big = ceil_div64(tiles(256), 256) * 256 * 4, small = ceil_div64(tiles(128), 512) * 512;
        if (tiles(256) >= 192 && big * 86 < small * 100) tile = 256;
    }
    int64_t n = tiles(tile ? tile : 128);
    const bool split = what == PLAN_PLAIN;
    if (!tile && n < 192 && !(split && n * (kt / 4) >= 192)) n = tiles(64);
    p.splits = split && n < 192 ? (int)std::max<int64_t>(1, std::min<int64_t>(512 / n, kt / 4)) : 1;
    return p;
}

// the outputs that wait for the join at the end of a pass, and the workspace behind them
struct Pending {
    JoinArgs j{};
    float *ws;
    explicit Pending(float *w) : ws(w) {}
    float *add(int64_t n, int splits, void *c) {
        float *at = ws;
        const int k = j.count++;
        j.parts[k] = at;
        j.c[k] = c;
        j.n[k] = n;
        j.splits[k] = splits;
        j.blocks[k] = (int)std::min<int64_t>(ceil_div64(n, 32), 8192);
        ws += (int64_t)splits * n;
        return at;
    }
    template <typename T> int go(hipStream_t st) {
        if (!j.count) return NMRF_OK;
        unsigned blocks = 0;
        for (int k = 0; k < j.count; ++k) blocks += (unsigned)j.blocks[k];
        hipLaunchKernelGGL(ffn_join_kernel<T>, dim3(blocks), dim3(256), 0, st, j);
        return nmrf_launch_status();
    }
};

template <typename T, bool PA, bool QA, int EPI>
int gemm_launch(GemmArgs &a, Pending &wait, hipStream_t st) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64;
    int tile = 0;
    int64_t blocks = 0;
    for (int i = 0; i < a.count; ++i) {
        Problem &q = a.p[i];
        const GemmPlan p = gemm_plan(q.M, q.N, (int64_t)q.K * q.segs, a.count, BK, EPI == EPI_DUAL ? PLAN_DUAL : EPI == EPI_DH ? PLAN_DH : PLAN_PLAIN, tile);
        tile = p.tile;                                             // (problems of one launch share the first one's tile)
        q.tiles_m = p.tiles_m;
        q.tiles_n = p.tiles_n;
        q.splits = p.splits;
        q.parts = p.splits > 1 ? wait.add((int64_t)q.M * q.N, p.splits, q.C) : nullptr;
        const int64_t n = (int64_t)p.tiles_m * p.tiles_n * p.splits;
        blocks += n;
        if (blocks > 0x7fffffff) return NMRF_EINVAL;
        q.blocks = (int)n;
    }
    if (tile == 256) {
        if constexpr (sizeof(T) == 2 && EPI != EPI_DH) hipLaunchKernelGGL((ffn_gemm_kernel<T, 256, 256, 2, 4, BK, PA, QA, EPI>), dim3((unsigned)blocks), dim3(512), 0, st, a);
    } else if (tile == 128) hipLaunchKernelGGL((ffn_gemm_kernel<T, 128, 128, 2, 2, BK, PA, QA, EPI>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((ffn_gemm_kernel<T, 64, 64, 2, 2, BK, PA, QA, EPI>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    return nmrf_launch_status();
}
// floats a plain product keeps in the workspace: alone in its launch, or at most, whatever shares it
int64_t gemm_floats(int64_t M, int64_t N, int64_t k, int bk, bool alone) {
    int64_t n = 0;
    for (int z = 1; z <= (alone ? 1 : 3); ++z)
        for (int tile : {0, 64, 128, 256}) {
            const int s = gemm_plan(M, N, k, z, bk, PLAN_PLAIN, tile).splits;
            n = std::max(n, s > 1 ? (int64_t)s * M * N : 0);
            if (alone) return n;
        }
    return n;
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
int64_t colsum_blocks(int64_t T) { return T < 512 ? 1 : std::min<int64_t>(T / 256, 128); }
constexpr int64_t FEW = 64;                                        // rows that stream the weights once

template <typename T>
int ffn_forward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, const void *bg, const void *bu, const void *bd,
                int act, void *h, float *g, float *u, void *y, unsigned *amax, float *ws, hipStream_t st) {
    if (s.T <= FEW && !g) {
        FewArgs f{x, wg, wu, bg, bu, h, (int)s.T, s.F, s.D, act, s.D, s.D, s.F};
        few_launch<T, 2>(f, st);
        FewArgs d{h, wd, wd, bd, nullptr, y, (int)s.T, s.Do, s.F, act, s.F, s.F, s.Do};
        few_launch<T, 1>(d, st);
        return nmrf_launch_status();
    }
    if constexpr (sizeof(T) == 4) {
        AbsmaxArgs m{{(const float *)x, (const float *)wg, (const float *)wu, (const float *)wd, nullptr},
                     {s.T * s.D, (int64_t)s.F * s.D, (int64_t)s.F * s.D, (int64_t)s.Do * s.F, 0},
                     {SLOT_X, SLOT_WG, SLOT_WU, SLOT_WD, SLOT_H}, amax};
        hipLaunchKernelGGL(ffn_absmax_kernel, dim3(256, 5), dim3(256), 0, st, m);
    }
    Pending wait(ws);
    GemmArgs a{};
    a.count = 1; a.act = act; a.amax = amax;
    Problem &p = a.p[0];
    p.P[0] = x; p.Q[0] = wg; p.Q[1] = wu; p.ldp = p.ldq = s.D; p.ldc = s.F;
    p.M = (int)s.T; p.N = s.F; p.K = s.D; p.segs = 1;
    p.C = h; p.C2 = g; p.C3 = u; p.bias = bg; p.bias2 = bu; p.slot_p = SLOT_X; p.slot_q = SLOT_WG; p.slot_out = SLOT_H;
    int rc = gemm_launch<T, true, true, EPI_DUAL>(a, wait, st);
    if (rc != NMRF_OK) return rc;
    p = Problem{};
    p.P[0] = h; p.Q[0] = wd; p.ldp = p.ldq = s.F; p.ldc = s.Do;
    p.M = (int)s.T; p.N = s.Do; p.K = s.F; p.segs = 1;
    p.C = y; p.bias = bd; p.slot_p = SLOT_H; p.slot_q = SLOT_WD; p.slot_out = -1;
    if ((rc = gemm_launch<T, true, true, EPI_PLAIN>(a, wait, st)) != NMRF_OK) return rc;
    wait.j.bias = bd;
    wait.j.cols = s.Do;
    return wait.go<T>(st);
}

template <typename T>
int ffn_backward(const FfnShape &s, const void *x, const void *wg, const void *wu, const void *wd, const void *h, const float *g, const float *u,
                 const void *dy, int act, void *dg, void *du, void *dx, void *dwg, void *dwu, void *dwd, void *dbg, void *dbu, void *dbd, unsigned *amax,
                 float *ws, hipStream_t st) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64;
    int rc;
    if constexpr (sizeof(T) == 4) {
        AbsmaxArgs m{{(const float *)dy, nullptr}, {s.T * s.Do, 0}, {SLOT_DY, SLOT_DG}, amax};
        hipLaunchKernelGGL(ffn_absmax_kernel, dim3(256, 2), dim3(256), 0, st, m);
    }
    Pending wait(ws);
    GemmArgs a{};
    a.count = 1; a.act = act; a.amax = amax;
    Problem &p = a.p[0];
    p.P[0] = dy; p.Q[0] = wd; p.ldp = s.Do; p.ldq = s.F; p.ldc = s.F;
    p.M = (int)s.T; p.N = s.F; p.K = s.Do; p.segs = 1;
    p.C = dg; p.C2 = du; p.g = g; p.u = u; p.slot_p = SLOT_DY; p.slot_q = SLOT_WD; p.slot_out = SLOT_DG;
    const int sums = 2 * gemm_plan(s.T, s.F, s.Do, 1, BK, PLAN_DH, 0).tiles_m;
    if (dbg) p.sum1 = wait.add(s.F, sums, dbg);
    if (dbu) p.sum2 = wait.add(s.F, sums, dbu);
    if ((rc = gemm_launch<T, true, false, EPI_DH>(a, wait, st)) != NMRF_OK) return rc;
    if (dx) {
        p = Problem{};
        p.P[0] = dg; p.P[1] = du; p.Q[0] = wg; p.Q[1] = wu; p.ldp = s.F; p.ldq = s.D; p.ldc = s.D;
        p.M = (int)s.T; p.N = s.D; p.K = s.F; p.segs = 2;
        p.C = dx; p.slot_p = SLOT_DG; p.slot_q = SLOT_WG; p.slot_out = -1;
        if ((rc = gemm_launch<T, true, false, EPI_PLAIN>(a, wait, st)) != NMRF_OK) return rc;
    }
    // weight gradients: products P^T Q over all T tokens, in one launch
    a.count = 0;
    auto wgrad = [&](const void *pp, const void *qq, int M, int N, void *c, int slot_p, int slot_q) {
        if (!c) return;
        Problem &w = a.p[a.count++];
        w = Problem{};
        w.P[0] = pp; w.Q[0] = qq; w.ldp = M; w.ldq = N; w.ldc = N;
        w.M = M; w.N = N; w.K = (int)s.T; w.segs = 1;
        w.C = c; w.slot_p = slot_p; w.slot_q = slot_q; w.slot_out = -1;
    };
    wgrad(dg, x, s.F, s.D, dwg, SLOT_DG, SLOT_X);
    wgrad(du, x, s.F, s.D, dwu, SLOT_DG, SLOT_X);
    wgrad(dy, h, s.Do, s.F, dwd, SLOT_DY, SLOT_H);
    if (a.count && (rc = gemm_launch<T, false, false, EPI_PLAIN>(a, wait, st)) != NMRF_OK) return rc;
    if (dbd) {
        const int64_t nb = colsum_blocks(s.T);
        ColsumArgs c{dy, wait.add(s.Do, (int)nb, dbd), s.Do, s.T, ceil_div64(s.T, nb)};
        hipLaunchKernelGGL(ffn_colsum_kernel<T>, dim3((unsigned)((s.Do + 63) / 64), (unsigned)nb), dim3(256), 0, st, c);
    }
    return wait.go<T>(st);
}

}  // namespace

extern "C" int nmrf_gated_ffn_size(int64_t T, int D, int F, int Do, int dtype, int backward, int64_t *floats) {
    if (!floats) return NMRF_ENULL;
    if (ffn_bad(FfnShape{T, D, F, Do}, dtype, 0)) return NMRF_EINVAL;
    const int bk = dtype == NMRF_F32 ? 32 : 64;
    int64_t n = 0;
    if (T > 0 && !backward) n = gemm_floats(T, Do, F, bk, true);
    if (T > 0 && backward)
        n = gemm_floats(T, D, 2 * (int64_t)F, bk, true) + 2 * gemm_floats(F, D, T, bk, false) + gemm_floats(Do, F, T, bk, false) + colsum_blocks(T) * Do +
            4 * (int64_t)F * gemm_plan(T, F, Do, 1, bk, PLAN_DH, 0).tiles_m;
    *floats = n;
    return NMRF_OK;
}

extern "C" int nmrf_gated_ffn(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *b_gate, const void *b_up,
                              const void *b_down, int64_t T, int D, int F, int Do, int dtype, int act, void *h, float *g, float *u, void *y,
                              uint32_t *amax, float *ws, int64_t ws_floats, void *stream) {
    const FfnShape s{T, D, F, Do};
    if (ffn_bad(s, dtype, act)) return NMRF_EINVAL;
    if (T == 0) return NMRF_OK;
    if (!x || !w_gate || !w_up || !w_down || !h || !y || (dtype == NMRF_F32 && !amax)) return NMRF_ENULL;
    if ((g == nullptr) != (u == nullptr) || ffn_misaligned({x, w_gate, w_up, w_down, b_gate, b_up, b_down, h, y}, dtype)) return NMRF_EINVAL;
    if (ffn_misaligned({amax, ws, g, u}, NMRF_F32)) return NMRF_EINVAL;
    int64_t need = 0;
    if (T > FEW || g) {
        const int rc = nmrf_gated_ffn_size(T, D, F, Do, dtype, 0, &need);
        if (rc != NMRF_OK || need > ws_floats) return NMRF_EINVAL;
        if (need && !ws) return NMRF_ENULL;
    }
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NMRF_F32) return ffn_forward<float>(s, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, h, g, u, y, amax, ws, st);
    if (dtype == NMRF_BF16) return ffn_forward<__bf16>(s, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, h, g, u, y, amax, ws, st);
    return ffn_forward<_Float16>(s, x, w_gate, w_up, w_down, b_gate, b_up, b_down, act, h, g, u, y, amax, ws, st);
}

extern "C" int nmrf_gated_ffn_bwd(const void *x, const void *w_gate, const void *w_up, const void *w_down, const void *h, const float *g, const float *u,
                                  const void *dy, int64_t T, int D, int F, int Do, int dtype, int act, void *dg, void *du, void *dx, void *dw_gate,
                                  void *dw_up, void *dw_down, void *db_gate, void *db_up, void *db_down, uint32_t *amax, float *ws,
                                  int64_t ws_floats, void *stream) {
    const FfnShape s{T, D, F, Do};
    if (ffn_bad(s, dtype, act) || T < 1) return NMRF_EINVAL;
    if (!x || !w_gate || !w_up || !w_down || !h || !g || !u || !dy || !dg || !du || !ws || (dtype == NMRF_F32 && !amax)) return NMRF_ENULL;
    if (ffn_misaligned({x, w_gate, w_up, w_down, h, dy, dg, du, dx, dw_gate, dw_up, dw_down, db_gate, db_up, db_down}, dtype)) return NMRF_EINVAL;
    if (ffn_misaligned({amax, ws, g, u}, NMRF_F32)) return NMRF_EINVAL;
    int64_t need = 0;
    const int rc = nmrf_gated_ffn_size(T, D, F, Do, dtype, 1, &need);
    if (rc != NMRF_OK || need > ws_floats) return NMRF_EINVAL;
    hipStream_t st = (hipStream_t)stream;
#define NMRF_FFN_BWD(TYPE) ffn_backward<TYPE>(s, x, w_gate, w_up, w_down, h, g, u, dy, act, dg, du, dx, dw_gate, dw_up, dw_down, db_gate, db_up, \
                                              db_down, amax, ws, st)
    if (dtype == NMRF_F32) return NMRF_FFN_BWD(float);
    if (dtype == NMRF_BF16) return NMRF_FFN_BWD(__bf16);
    return NMRF_FFN_BWD(_Float16);
#undef NMRF_FFN_BWD
}
