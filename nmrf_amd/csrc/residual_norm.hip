// The norms around a block, fused with its gate and residual scale, and their backward pass.  Per row of C channels:
//     z   = post ? norm(y) * post_w + post_b : y            y: what the block returned
//     out = x + s a z                                        s: a number times a vector over C; a = act(gate), act: none, sigmoid, tanh
//     h   = norm(out) * next_w + next_b                      what the next block reads (optional)
// norm: (v - mean) / sqrt(var + eps) or v / sqrt(mean(v^2) + eps).  The gate is one value per element, per row, per group of R consecutive
// rows, or per group and channel.  (The framework's add + LayerNorm kernel, nmrf_add_ln_concat_f32, is the form x + y, LayerNorm at C = 128.)
//
// Bound by memory: x and y in, out and h out -- 4 T C elements forward, 6 T C backward (x, y and both gradients in, dx and dy out) and
// nothing else per row.  One pass: a row sits in the registers of its lanes (16 lanes up to 128 channels, a wave up to 512, a block of 4 waves up to
// 2 048, of 8 up to 8 192; 8 elements a lane, 16 above 4 096 channels), the mean is subtracted before squares are summed (fp32), and h is formed from the fp32
// values of out, not from its rounded copy.  The backward pass recomputes that row from x and y -- the same bytes as reading a saved out --
// and keeps the sums over rows (parameters, group gates) in registers: a block writes one partial row at its end, and one more launch adds the
// partials in a fixed order.  No atomics: the same bits every run.
//
// Measured (kernel time): fp32 [29 952, 128], LayerNorm, scale: forward 12 us (61 MB, 5.1 TB/s), backward 19 + 5 us (92 MB, 4.8 TB/s); bf16
// [16 384, 4 096], post norm and a tanh gate per sample: forward 98 us (537 MB, 5.5 TB/s), backward 215 + 8 us (805 MB, 3.7 TB/s: one row a CU
// in flight, four sums over 8 waves a row).  Loads a row ahead, no load under a branch (each is waited for before the next: 264 -> 233 us),
// consecutive rows to a block so that a group's gate is read once (forward 161 -> 105 us).
#include "common.h"
#include "elem.h"
#include <initializer_list>

namespace {

enum { GATE_NONE = 0, GATE_ELEM = 1, GATE_ROW = 2, GATE_GROUP = 3, GATE_GROUP_ONE = 4 };
enum { P_NEXT_W = 0, P_NEXT_B = 1, P_SCALE = 2, P_POST_W = 3, P_POST_B = 4, NPARAM = 5 };

struct RnArgs {
    const void *x, *y, *gate, *post_w, *post_b, *next_w, *next_b, *scale;
    void *out, *h;                               // forward
    const void *d_out, *d_h;                     // backward
    void *dx, *dy, *dgate;
    float *parts, *gparts;                       // [gridDim][NPARAM][C], [items][C or 1]
    int64_t T, R;                                // R: rows that share a gate row
    int64_t span, items, chunks, rows_per_item;  // backward: items are (span of rows, chunk of it) pairs
    int C, gate_mode, gate_act, pf32, rms, post, next, want;      // want: bit P_* = that gradient is asked for, bit 8: dgate
    float eps, scale_value;
};

template <int LPR> __device__ __forceinline__ float lanes_sum(float v) {            // over the LPR (<= 64) lanes of a row
    if constexpr (LPR == 64) return wave_sum_nolds(v);
    v += NMRF_ROW_ROR(v, 8);
    v += NMRF_ROW_ROR(v, 4);
    v += NMRF_ROW_ROR(v, 2);
    v += NMRF_ROW_ROR(v, 1);
    return v;
}
// sums of a (and b) over the lanes of a row; rows of several waves meet in LDS (two buffers in turn: one barrier a sum)
template <int LPR> struct RowSum {
    float (*sh)[2][8];
    int turn = 0;
    __device__ __forceinline__ void two(float &a, float &b) {
        if constexpr (LPR <= 64) {
            a = lanes_sum<LPR>(a);
            b = lanes_sum<LPR>(b);
        } else {
            a = wave_sum_nolds(a);
            b = wave_sum_nolds(b);
            if ((threadIdx.x & 63) == 0) {
                sh[turn][0][threadIdx.x >> 6] = a;
                sh[turn][1][threadIdx.x >> 6] = b;
            }
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < LPR / 64; ++w) {
                a += sh[turn][0][w];
                b += sh[turn][1][w];
            }
            turn ^= 1;
        }
    }
    __device__ __forceinline__ float one(float a) {
        if constexpr (LPR <= 64) return lanes_sum<LPR>(a);
        a = wave_sum_nolds(a);
        if ((threadIdx.x & 63) == 0) sh[turn][0][threadIdx.x >> 6] = a;
        __syncthreads();
        a = 0.f;
#pragma unroll
        for (int w = 0; w < LPR / 64; ++w) a += sh[turn][0][w];
        turn ^= 1;
        return a;
    }
};

__device__ __forceinline__ float gate_value(float g, int act) {
    return act == 1 ? 1.0f / (1.0f + expf(-g)) : (act == 2 ? tanhf(g) : g);
}
__device__ __forceinline__ float gate_slope(float a, int act) { return act == 1 ? a * (1.0f - a) : (act == 2 ? 1.0f - a * a : 1.0f); }

// The lanes' elements against the row: EXACT -- each one a channel (powers of two from 64 on); ANY; TINY -- fewer channels than a 16-byte
// vector holds.  (Clamped addresses and masks cost half as many instructions again as the arithmetic of a row of 128 channels.)
enum { EXACT = 0, ANY = 1, TINY = 2 };
template <typename T, int LPR, int E, int FIT> struct Row {
    static constexpr int N = Vec16<T>::N, K = N * E;
    int C, lane;
    bool tail;                                   // (uniform) the last vector of a row is not whole
    __device__ __forceinline__ Row(int c, int l) : C(FIT == EXACT ? LPR * K : c), lane(l), tail(FIT != EXACT && c % N != 0) {}
    __device__ __forceinline__ int at(int j) const { return (j * LPR + lane) * N; }
    __device__ __forceinline__ bool in(int e) const { return FIT == EXACT || at(e / N) + e % N < C; }
    // Every lane loads, whatever it holds of the row (a load under a branch is waited for before the next one): a vector that the row's end cuts
    // short comes from the last N channels and is moved into place by place(), one behind the end from the row's start and is dropped there.
    __device__ __forceinline__ int from(int j) const { return FIT == EXACT || at(j) + N <= C ? at(j) : (at(j) < C ? C - N : 0); }
    __device__ __forceinline__ void place(float *v) const {
        if constexpr (FIT == EXACT) return;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            float *x = v + j * N;
            if (FIT == ANY && tail) {
                const int m = at(j) < C && at(j) + N > C ? at(j) + N - C : 0;
#pragma unroll
                for (int s = N / 2; s > 0; s /= 2)
#pragma unroll
                    for (int k = 0; k < N; ++k) x[k] = m & s ? (k + s < N ? x[k + s < N ? k + s : 0] : 0.f) : x[k];
            }
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = at(j) < C ? x[k] : 0.f;
        }
    }
    __device__ __forceinline__ void ask(const void *p, int64_t base, uint4 *w) const {
        const T *q = static_cast<const T *>(p) + base;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if constexpr (FIT == TINY) w[j] = Vec16<T>::raw_part(q, j == 0 && lane == 0 ? C : 0);
            else w[j] = Vec16<T>::raw(q + from(j));
        }
    }
    __device__ __forceinline__ void take(const uint4 *w, float *v) const {
#pragma unroll
        for (int j = 0; j < E; ++j) Vec16<T>::unpack(w[j], v + j * N);
        place(v);
    }
    __device__ __forceinline__ void store(void *p, int64_t base, const float *v) const {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            T *q = static_cast<T *>(p) + base + at(j);
            if (FIT == EXACT || at(j) + N <= C) Vec16<T>::store(q, v + j * N);
            else if (tail && at(j) < C) Vec16<T>::store_part(q, v + j * N, C - at(j));
        }
    }
    // a vector over the channels, in the rows' type or in fp32; `none` where there is none, 0 behind the last channel
    __device__ __forceinline__ void param(const RnArgs &a, const void *p, float none, float *v) const {
        if (!p) {
#pragma unroll
            for (int e = 0; e < K; ++e) v[e] = in(e) ? none : 0.f;
        } else if (!a.pf32) {
            uint4 w[E];
            ask(p, 0, w);
            take(w, v);
        } else {
            const float *q = static_cast<const float *>(p);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if constexpr (FIT == TINY) {
#pragma unroll
                    for (int k = 0; k < N; ++k) v[j * N + k] = q[at(j) + k < C ? at(j) + k : 0];
                } else {
#pragma unroll
                    for (int k = 0; k < N; k += 4) Vec16<float>::unpack(Vec16<float>::raw(q + from(j) + k), v + j * N + k);
                }
            }
            if (FIT == TINY)
#pragma unroll
                for (int e = 0; e < K; ++e) v[e] = in(e) ? v[e] : 0.f;
            else place(v);
        }
    }
    // v -> (v - mean) * rstd (layer) or v * rstd (rms); returns rstd
    __device__ __forceinline__ float norm(float *v, int rms, float eps, RowSum<LPR> &rs) const {
        const float inv = 1.0f / C;
        if (!rms) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < K; ++e) s += v[e];
            const float mean = rs.one(s) * inv;
#pragma unroll
            for (int e = 0; e < K; ++e) v[e] -= mean;
            if (FIT != EXACT)
#pragma unroll
                for (int e = 0; e < K; ++e) v[e] = in(e) ? v[e] : 0.f;
        }
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < K; ++e) q = fmaf(v[e], v[e], q);
        const float rstd = 1.0f / sqrtf(rs.one(q) * inv + eps);
#pragma unroll
        for (int e = 0; e < K; ++e) v[e] *= rstd;
        return rstd;
    }
    // u = gradient of the normalised values -> gradient of the values: rstd (u - mean(u) - vhat mean(u vhat)), without mean(u) for rms
    __device__ __forceinline__ void norm_back(float *u, const float *vhat, float rstd, int rms, RowSum<LPR> &rs) const {
        float su = 0.f, sx = 0.f;
#pragma unroll
        for (int e = 0; e < K; ++e) {
            su += u[e];
            sx = fmaf(u[e], vhat[e], sx);
        }
        if (rms) {
            sx = rs.one(sx);
            su = 0.f;
        } else {
            rs.two(su, sx);
        }
        su *= 1.0f / C;
        sx *= 1.0f / C;
#pragma unroll
        for (int e = 0; e < K; ++e) u[e] = rstd * (u[e] - su - vhat[e] * sx);
    }
    // act(gate) of row r, read again only when the row's gate row is another one: one value (GV false), or one for each element
    template <bool GV> __device__ __forceinline__ void gate(const RnArgs &a, int64_t r, int64_t &held, float *g) const {
        if (a.gate_mode == GATE_NONE) return;
        const int64_t gr = a.R == 1 ? r : r / a.R;
        if (gr == held) return;
        held = gr;
        if constexpr (GV) {
            uint4 w[E];
            ask(a.gate, gr * a.C, w);
            take(w, g);
#pragma unroll
            for (int e = 0; e < K; ++e) g[e] = gate_value(g[e], a.gate_act);
        } else {
            g[0] = gate_value(Quad<T>::one(static_cast<const T *>(a.gate) + gr), a.gate_act);
        }
    }
};

template <int LPR> constexpr int rn_threads() { return LPR <= 256 ? 256 : LPR; }

template <typename T, int LPR, int E, int FIT>
__global__ __launch_bounds__(rn_threads<LPR>()) void residual_norm_fwd_kernel(RnArgs a) {
    constexpr int K = Row<T, LPR, E, FIT>::K, ROWS = rn_threads<LPR>() / LPR;
    __shared__ float sh[2][2][8];
    RowSum<LPR> rs{sh};
    const Row<T, LPR, E, FIT> row(a.C, (int)(threadIdx.x % LPR));
    const bool gv = a.gate_mode == GATE_ELEM || a.gate_mode == GATE_GROUP;
    float pw[K], pb[K], nw[K], nb[K], sc[K], g[K];
    // (a block owns consecutive rows: they share their gate row as long as they can)
    const int64_t r1 = min(a.T, (int64_t)(blockIdx.x + 1) * a.rows_per_item);
    int64_t r = (int64_t)blockIdx.x * a.rows_per_item + threadIdx.x / LPR, held = -1;
    uint4 wx[E], wy[E];
    if (r < r1) {
        row.ask(a.y, r * a.C, wy);
        row.ask(a.x, r * a.C, wx);
    }
    row.param(a, a.post_w, 1.f, pw);
    row.param(a, a.post_b, 0.f, pb);
    row.param(a, a.next_w, 1.f, nw);
    row.param(a, a.next_b, 0.f, nb);
    row.param(a, a.scale, 1.f, sc);
#pragma unroll
    for (int e = 0; e < K; ++e) {
        sc[e] *= a.scale_value;
        g[e] = 1.f;
    }
    // (rows of one wave or less: lanes behind the last row leave; a row of several waves has the whole block's barriers in step)
    for (; r < r1; r += ROWS) {
        float x[K], z[K];
        row.take(wy, z);
        row.take(wx, x);
        if (r + ROWS < r1) {                                       // the next row is on its way while this one waits for its sums
            row.ask(a.y, (r + ROWS) * a.C, wy);
            row.ask(a.x, (r + ROWS) * a.C, wx);
        }
        if (gv) {
            row.template gate<true>(a, r, held, g);
        } else if (a.gate_mode != GATE_NONE) {
            row.template gate<false>(a, r, held, g);
#pragma unroll
            for (int e = 1; e < K; ++e) g[e] = g[0];
        }
        if (a.post) {
            row.norm(z, a.rms, a.eps, rs);
#pragma unroll
            for (int e = 0; e < K; ++e) z[e] = fmaf(z[e], pw[e], pb[e]);
        }
#pragma unroll
        for (int e = 0; e < K; ++e) x[e] = fmaf(sc[e] * g[e], z[e], x[e]);
        row.store(a.out, r * a.C, x);
        if (a.next) {
            row.norm(x, a.rms, a.eps, rs);
#pragma unroll
            for (int e = 0; e < K; ++e) x[e] = fmaf(x[e], nw[e], nb[e]);
            row.store(a.h, r * a.C, x);
        }
    }
}

// sum of a lane's K values over the rows a block holds side by side -> dst [C], written by the lanes of its first row
template <typename T, int LPR, int E, int FIT>
__device__ __forceinline__ void block_columns(const Row<T, LPR, E, FIT> &row, float *v, float mul, float *dst) {
    constexpr int K = Row<T, LPR, E, FIT>::K, N = Row<T, LPR, E, FIT>::N;
    if constexpr (LPR < 64) {
#pragma unroll
        for (int e = 0; e < K; ++e) {
            v[e] += __shfl_xor(v[e], 16);
            v[e] += __shfl_xor(v[e], 32);
        }
    }
    if constexpr (LPR <= 64) {
        __shared__ float cols[4][LPR * K];
        __syncthreads();
        if ((threadIdx.x & 63) < LPR)
#pragma unroll
            for (int e = 0; e < K; ++e) cols[threadIdx.x >> 6][(threadIdx.x & 63) * K + e] = v[e];
        __syncthreads();
        if (threadIdx.x < LPR)
#pragma unroll
            for (int e = 0; e < K; ++e) {
                const int i = threadIdx.x * K + e;
                v[e] = (cols[0][i] + cols[1][i]) + (cols[2][i] + cols[3][i]);
            }
    }
    if (threadIdx.x < LPR)
#pragma unroll
        for (int e = 0; e < K; ++e)
            if (row.in(e)) dst[row.at(e / N) + e % N] = v[e] * mul;
}

// GV: the gate is a vector over the channels (one value a row, or none, keeps 2 K registers free)
template <typename T, int LPR, int E, int FIT, bool GV>
__global__ __launch_bounds__(rn_threads<LPR>()) void residual_norm_bwd_kernel(RnArgs a) {
    constexpr int K = Row<T, LPR, E, FIT>::K, THREADS = rn_threads<LPR>(), ROWS = THREADS / LPR, GK = GV ? K : 1;
    __shared__ float sh[2][2][8];
    __shared__ float ones[THREADS / 64];
    RowSum<LPR> rs{sh};
    const Row<T, LPR, E, FIT> row(a.C, (int)(threadIdx.x % LPR));
    float pw[K], nw[K], sc[K], g[GK], acc[NPARAM][K];
    row.param(a, a.post_w, 1.f, pw);
    row.param(a, a.next_w, 1.f, nw);
    row.param(a, a.scale, 1.f, sc);
#pragma unroll
    for (int e = 0; e < K; ++e) sc[e] *= a.scale_value;
#pragma unroll
    for (int e = 0; e < GK; ++e) g[e] = 1.f;
#pragma unroll
    for (int q = 0; q < NPARAM; ++q)
#pragma unroll
        for (int e = 0; e < K; ++e) acc[q][e] = 0.f;
    int64_t held = -1;
    for (int64_t item = blockIdx.x; item < a.items; item += gridDim.x) {
        const int64_t group = item / a.chunks, first = (item - group * a.chunks) * a.rows_per_item;
        const int64_t r1 = group * a.span + (first + a.rows_per_item < a.span ? first + a.rows_per_item : a.span);
        float ga[GK];
#pragma unroll
        for (int e = 0; e < GK; ++e) ga[e] = 0.f;
        uint4 wx[E], wy[E], wh[E], wd[E];
#pragma unroll
        for (int j = 0; j < E; ++j) wh[j] = wd[j] = make_uint4(0, 0, 0, 0);
        auto ask = [&](int64_t r) {
            row.ask(a.y, r * a.C, wy);
            row.ask(a.x, r * a.C, wx);
            if (a.d_h) row.ask(a.d_h, r * a.C, wh);
            if (a.d_out) row.ask(a.d_out, r * a.C, wd);
        };
        int64_t r = group * a.span + first + threadIdx.x / LPR;
        if (r < r1) ask(r);
        for (; r < r1; r += ROWS) {
            float z[K], t[K], d[K], u[K], zz[K];
            row.take(wy, z);
            row.take(wx, t);
            row.take(wh, u);
            row.take(wd, d);
            if (r + ROWS < r1) ask(r + ROWS);
            row.template gate<GV>(a, r, held, g);
            float zr = 0.f;
            if (a.post) {
                zr = row.norm(z, a.rms, a.eps, rs);                // z holds zhat from here on
                row.param(a, a.post_b, 0.f, zz);
#pragma unroll
                for (int e = 0; e < K; ++e) zz[e] = fmaf(z[e], pw[e], zz[e]);
            } else {
#pragma unroll
                for (int e = 0; e < K; ++e) zz[e] = z[e];
            }
            if (a.d_h) {
#pragma unroll
                for (int e = 0; e < K; ++e) t[e] = fmaf(sc[e] * g[GV ? e : 0], zz[e], t[e]);
                const float hr = row.norm(t, a.rms, a.eps, rs);
#pragma unroll
                for (int e = 0; e < K; ++e) {
                    acc[P_NEXT_W][e] = fmaf(u[e], t[e], acc[P_NEXT_W][e]);
                    acc[P_NEXT_B][e] += u[e];
                    u[e] *= nw[e];
                }
                row.norm_back(u, t, hr, a.rms, rs);
#pragma unroll
                for (int e = 0; e < K; ++e) d[e] += u[e];
            }
            row.store(a.dx, r * a.C, d);
            float gs = 0.f;
#pragma unroll
            for (int e = 0; e < K; ++e) {
                const float dz = d[e] * zz[e];                     // gradient of the factor scale_value * scale * a
                acc[P_SCALE][e] = fmaf(dz, g[GV ? e : 0], acc[P_SCALE][e]);
                u[e] = dz * sc[e];                                 // gradient of a
                if constexpr (GV) ga[e] += u[e];
                else gs += u[e];
                d[e] *= sc[e] * g[GV ? e : 0];                     // gradient of z
            }
            if (a.want & 256) {
                if constexpr (GV) {
                    if (a.gate_mode == GATE_ELEM) {
#pragma unroll
                        for (int e = 0; e < K; ++e) u[e] *= gate_slope(g[e], a.gate_act);
                        row.store(a.dgate, r * a.C, u);
                    }
                } else if (a.gate_mode == GATE_ROW) {
                    gs = rs.one(gs) * gate_slope(g[0], a.gate_act);
                    if (row.lane == 0) Quad<T>::put(static_cast<T *>(a.dgate) + r, gs);
                } else {
                    ga[0] += gs;
                }
            }
            if (a.post) {
#pragma unroll
                for (int e = 0; e < K; ++e) {
                    acc[P_POST_W][e] = fmaf(d[e], z[e], acc[P_POST_W][e]);
                    acc[P_POST_B][e] += d[e];
                    d[e] *= pw[e];
                }
                row.norm_back(d, z, zr, a.rms, rs);
            }
            row.store(a.dy, r * a.C, d);
        }
        if (a.want & 256) {
            if constexpr (GV) {
                if (a.gate_mode == GATE_GROUP) block_columns(row, ga, 1.f, a.gparts + item * a.C);
            } else if (a.gate_mode == GATE_GROUP_ONE) {
                const float s1 = wave_sum_nolds(ga[0]);
                __syncthreads();
                if ((threadIdx.x & 63) == 0) ones[threadIdx.x >> 6] = s1;
                __syncthreads();
                if (threadIdx.x == 0) {
                    float s = 0.f;
                    for (int w = 0; w < THREADS / 64; ++w) s += ones[w];
                    a.gparts[item] = s;
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q < NPARAM; ++q)
        if (a.want >> q & 1) block_columns(row, acc[q], q == P_SCALE ? a.scale_value : 1.f, a.parts + ((int64_t)blockIdx.x * NPARAM + q) * a.C);
}

// the second launch: parameter columns over all blocks, gate groups over their chunks.  A block owns 16 columns; its 16 row lanes add the
// partials i, i + 16, ... in ascending order and lane 0 adds the 16 lane sums: a fixed order.
struct RnReduce {
    const float *parts, *gparts;
    void *to[NPARAM];
    void *dgate;
    const void *gate;
    int64_t chunks, gcols;      // gcols: gate columns altogether (groups x C, or groups), 0: none
    int blocks, C, pf32, gate_act, pblocks, gC;
};
template <typename T>
__global__ __launch_bounds__(256) void residual_norm_reduce_kernel(RnReduce a) {
    __shared__ float sh[16][17];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4;
    const bool params = (int)blockIdx.x < a.pblocks;
    const int64_t col = params ? (int64_t)blockIdx.x * 16 + c : (int64_t)(blockIdx.x - a.pblocks) * 16 + c;
    const int q = params ? (int)(col / a.C) : 0;
    const bool on = params ? (q < NPARAM && a.to[q < NPARAM ? q : 0]) : col < a.gcols;
    const float *p = nullptr;
    int64_t stride = 0, count = 0;
    if (on) {
        if (params) {
            p = a.parts + col;
            stride = (int64_t)NPARAM * a.C;
            count = a.blocks;
        } else {
            const int64_t group = col / a.gC;
            p = a.gparts + group * a.chunks * a.gC + (col - group * a.gC);
            stride = a.gC;
            count = a.chunks;
        }
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    int64_t i = l;
    for (; i + 48 < count; i += 64)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] += p[(i + 16 * k) * stride];
    for (; i < count; i += 16) s[0] += p[i * stride];
    sh[l][c] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (l == 0 && on) {
        float v = sh[0][c];
#pragma unroll
        for (int k = 1; k < 16; ++k) v += sh[k][c];
        if (params) {
            const int64_t cc = col - (int64_t)q * a.C;
            if (a.pf32) static_cast<float *>(a.to[q])[cc] = v;
            else Quad<T>::put(static_cast<T *>(a.to[q]) + cc, v);
        } else {
            v *= gate_slope(gate_value(Quad<T>::one(static_cast<const T *>(a.gate) + col), a.gate_act), a.gate_act);
            Quad<T>::put(static_cast<T *>(a.dgate) + col, v);
        }
    }
}

// lanes of a row and 16-byte vectors of a lane: 16 lanes while 8 elements each hold the row, then a wave, then 4, then 8 waves.  (16 elements
// a lane take all 256 VGPRs of the backward kernel and spill: above 4 096 channels only, where it is slow for it.  bf16, [8 192, 8 192]: forward
// 93 us (5.8 TB/s), backward 560 us (1.4 TB/s); [8 192, 5 120], whose lanes are not all at work: 176 and 648 us.)
struct RnShape { int lpr, e; };
RnShape rn_shape(int C, int n) {
    RnShape s{C <= 128 ? 16 : (C <= 512 ? 64 : (C <= 2048 ? 256 : 512)), 8 / n};
    if (s.lpr == 512 && C > 4096) s.e *= 2;
    if (n == 4 && s.lpr < 512 && C <= s.lpr * 4) s.e = 1;
    return s;
}
template <typename T, int LPR, int E, int FIT>
void rn_fit(bool bwd, const RnArgs &a, unsigned grid, hipStream_t st) {
    const dim3 b(rn_threads<LPR>());
    if (!bwd) hipLaunchKernelGGL((residual_norm_fwd_kernel<T, LPR, E, FIT>), dim3(grid), b, 0, st, a);
    else if (a.gate_mode == GATE_ELEM || a.gate_mode == GATE_GROUP) hipLaunchKernelGGL((residual_norm_bwd_kernel<T, LPR, E, FIT, true>), dim3(grid), b, 0, st, a);
    else hipLaunchKernelGGL((residual_norm_bwd_kernel<T, LPR, E, FIT, false>), dim3(grid), b, 0, st, a);
}
template <typename T, int LPR, int E>
void rn_go(bool bwd, const RnArgs &a, unsigned grid, hipStream_t st) {
    if (a.C == LPR * E * Vec16<T>::N) rn_fit<T, LPR, E, EXACT>(bwd, a, grid, st);
    else rn_fit<T, LPR, E, ANY>(bwd, a, grid, st);
}
template <typename T, int LPR>
void rn_e(int e, bool bwd, const RnArgs &a, unsigned grid, hipStream_t st) {
    constexpr int E = 8 / Vec16<T>::N;
    if constexpr (E == 2 && LPR < 512) if (e == 1) return rn_go<T, LPR, 1>(bwd, a, grid, st);
    if constexpr (LPR == 512) if (e == 2 * E) return rn_go<T, LPR, 2 * E>(bwd, a, grid, st);
    rn_go<T, LPR, E>(bwd, a, grid, st);
}
template <typename T>
int rn_launch(const RnShape &s, bool bwd, const RnArgs &a, unsigned grid, hipStream_t st) {
    if (a.C < Vec16<T>::N) rn_fit<T, 16, 1, TINY>(bwd, a, grid, st);
    else if (s.lpr == 16) rn_e<T, 16>(s.e, bwd, a, grid, st);
    else if (s.lpr == 64) rn_e<T, 64>(s.e, bwd, a, grid, st);
    else if (s.lpr == 256) rn_e<T, 256>(s.e, bwd, a, grid, st);
    else rn_e<T, 512>(s.e, bwd, a, grid, st);
    return nmrf_launch_status();
}
int rn_dispatch(int dtype, const RnShape &s, bool bwd, const RnArgs &a, unsigned grid, hipStream_t st) {
    if (dtype == NMRF_F32) return rn_launch<float>(s, bwd, a, grid, st);
    if (dtype == NMRF_BF16) return rn_launch<__bf16>(s, bwd, a, grid, st);
    return rn_launch<_Float16>(s, bwd, a, grid, st);
}

int rn_gate_mode(const void *gate, int64_t T, int C, int64_t R, int cols) {
    if (!gate) return GATE_NONE;
    if (R < 1 || T % R != 0 || (cols != 1 && cols != C)) return -1;
    if (cols == C && C > 1) return R == 1 ? GATE_ELEM : GATE_GROUP;
    return R == 1 ? GATE_ROW : GATE_GROUP_ONE;
}
// the backward grid: items of rows of one gate group each, about 512 blocks (2 per CU; rows of 8 waves: one per CU,
// which is what their registers leave room for: more partial rows cost more than they hide)
struct RnPlan { int64_t items, chunks, rows; int blocks; };
RnPlan rn_plan(int64_t T, int64_t span, int lpr) {
    const int side = lpr <= 256 ? 256 / lpr : 1;                   // rows a block works on at once
    const int64_t target = lpr == 512 ? 256 : 512, groups = T / span;
    RnPlan p;
    int64_t chunks = groups >= target ? 1 : target / groups;
    const int64_t most = ceil_div64(span, side);
    if (chunks > most) chunks = most;
    p.rows = ceil_div64(ceil_div64(span, chunks), side) * side;
    p.chunks = ceil_div64(span, p.rows);
    p.items = groups * p.chunks;
    p.blocks = (int)(p.items < target ? p.items : target);
    return p;
}
bool rn_aligned(std::initializer_list<const void *> ps, uintptr_t mask) {
    uintptr_t o = 0;
    for (const void *p : ps) o |= reinterpret_cast<uintptr_t>(p);
    return (o & mask) == 0;
}
int rn_check(const RnArgs &a, int gate_act, int kind, int dtype, int params_f32) {
    if (a.T < 0 || a.C < 1 || a.C > 8192 || dtype < NMRF_F32 || dtype > NMRF_F16 || gate_act < 0 || gate_act > 2 || kind < 0 || kind > 1) return NMRF_EINVAL;
    if (!(a.eps >= 0.f) || a.gate_mode < 0 || a.T > ((int64_t)1 << 50) / a.C) return NMRF_EINVAL;
    const uintptr_t el = dtype == NMRF_F32 ? 3 : 1, pe = params_f32 ? 3 : el;
    if (!rn_aligned({a.x, a.y, a.gate, a.out, a.h, a.d_out, a.d_h, a.dx, a.dy, a.dgate}, el) ||
        !rn_aligned({a.post_w, a.post_b, a.next_w, a.next_b, a.scale}, pe)) return NMRF_EINVAL;
    return NMRF_OK;
}

}  // namespace

extern "C" int nmrf_residual_norm(const void *x, const void *y, int64_t T, int C, int dtype, int kind, float eps, const void *gate,
                                  int64_t gate_rows, int gate_cols, int gate_act, float scale_value, const void *scale, int post,
                                  const void *post_w, const void *post_b, const void *next_w, const void *next_b, int params_f32, void *out,
                                  void *h, void *stream) {
    RnArgs a{};
    a.x = x; a.y = y; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.next_w = next_w; a.next_b = next_b; a.scale = scale;
    a.out = out; a.h = h; a.T = T; a.C = C; a.R = gate ? gate_rows : 1; a.gate_act = gate_act; a.pf32 = params_f32; a.rms = kind; a.post = post;
    a.next = h != nullptr; a.eps = eps; a.scale_value = scale_value;
    a.gate_mode = rn_gate_mode(gate, T, C, gate_rows, gate_cols);
    const int rc = rn_check(a, gate_act, kind, dtype, params_f32);
    if (rc != NMRF_OK) return rc;
    if (T == 0) return NMRF_OK;
    if (!x || !y || !out) return NMRF_ENULL;
    const RnShape s = rn_shape(C, dtype == NMRF_F32 ? 4 : 8);
    const int rows = s.lpr <= 256 ? 256 / s.lpr : 1;
    const int64_t most = s.lpr < 256 ? 2048 : (s.lpr == 256 ? 1024 : 512);
    a.rows_per_item = ceil_div64(ceil_div64(T, most), rows) * rows;
    const int64_t grid = ceil_div64(T, a.rows_per_item);
    return rn_dispatch(dtype, s, false, a, (unsigned)grid, (hipStream_t)stream);
}

extern "C" int nmrf_residual_norm_bwd_size(int64_t T, int C, int64_t gate_rows, int64_t *floats) {
    if (!floats) return NMRF_ENULL;
    if (T < 1 || C < 1 || C > 8192 || gate_rows < 1 || T % gate_rows != 0) return NMRF_EINVAL;
    // (an upper bound over the row layouts: blocks <= 512, items <= max(groups, 512))
    const int64_t groups = T / gate_rows;
    *floats = ((int64_t)512 * NPARAM + (groups > 512 ? groups : 512)) * C;
    return NMRF_OK;
}

extern "C" int nmrf_residual_norm_bwd(const void *x, const void *y, const void *d_out, const void *d_h, int64_t T, int C, int dtype, int kind,
                                      float eps, const void *gate, int64_t gate_rows, int gate_cols, int gate_act, float scale_value,
                                      const void *scale, int post, const void *post_w, const void *post_b, const void *next_w, int params_f32,
                                      void *dx, void *dy, void *dgate, void *d_scale, void *d_post_w, void *d_post_b, void *d_next_w,
                                      void *d_next_b, float *ws, int64_t ws_floats, void *stream) {
    RnArgs a{};
    a.x = x; a.y = y; a.gate = gate; a.post_w = post_w; a.post_b = post_b; a.next_w = next_w; a.scale = scale;
    a.d_out = d_out; a.d_h = d_h; a.dx = dx; a.dy = dy; a.dgate = dgate;
    a.T = T; a.C = C; a.gate_act = gate_act; a.pf32 = params_f32; a.rms = kind; a.post = post; a.eps = eps; a.scale_value = scale_value;
    a.gate_mode = rn_gate_mode(gate, T, C, gate_rows, gate_cols);
    const int rc = rn_check(a, gate_act, kind, dtype, params_f32);
    if (rc != NMRF_OK) return rc;
    if (T < 1) return NMRF_EINVAL;
    if (!x || !y || !dx || !dy || !ws || (!d_out && !d_h)) return NMRF_ENULL;
    if ((dgate && !gate) || ((d_next_w || d_next_b) && !d_h) || ((d_post_w || d_post_b) && !post)) return NMRF_EINVAL;
    const uintptr_t pe = params_f32 || dtype == NMRF_F32 ? 3 : 1;
    if (!rn_aligned({d_scale, d_post_w, d_post_b, d_next_w, d_next_b}, pe) || !rn_aligned({ws}, 3)) return NMRF_EINVAL;
    void *to[NPARAM] = {d_next_w, d_next_b, d_scale, d_post_w, d_post_b};
    for (int q = 0; q < NPARAM; ++q) a.want |= to[q] ? 1 << q : 0;
    if (dgate) a.want |= 256;
    const RnShape s = rn_shape(C, dtype == NMRF_F32 ? 4 : 8);
    // rows are dealt out group by group only where a gate gradient is summed over them
    const bool grouped = dgate && (a.gate_mode == GATE_GROUP || a.gate_mode == GATE_GROUP_ONE);
    a.R = gate ? gate_rows : 1;
    a.span = grouped ? gate_rows : T;
    const RnPlan p = rn_plan(T, a.span, s.lpr);
    const int gC = a.gate_mode == GATE_GROUP ? C : 1;
    if ((int64_t)p.blocks * NPARAM * C + (grouped ? p.items * gC : 0) > ws_floats) return NMRF_EINVAL;
    a.parts = ws;
    a.gparts = ws + (int64_t)p.blocks * NPARAM * C;
    a.items = p.items; a.chunks = p.chunks; a.rows_per_item = p.rows;
    const int64_t groups = T / a.span;
    hipStream_t st = (hipStream_t)stream;
    const int rc2 = rn_dispatch(dtype, s, true, a, (unsigned)p.blocks, st);
    if (rc2 != NMRF_OK || !(a.want & 31 || grouped)) return rc2;
    RnReduce r{};
    r.parts = a.parts; r.gparts = a.gparts; r.dgate = dgate; r.gate = gate; r.chunks = p.chunks; r.blocks = p.blocks; r.C = C; r.pf32 = params_f32;
    r.gate_act = gate_act; r.gC = gC; r.gcols = grouped ? groups * gC : 0;
    for (int q = 0; q < NPARAM; ++q) r.to[q] = to[q];
    r.pblocks = a.want & 31 ? (int)ceil_div64((int64_t)NPARAM * C, 16) : 0;
    const int64_t grid = r.pblocks + ceil_div64(r.gcols, 16);
    if (grid > 0x7fffffff) return NMRF_EINVAL;
    if (dtype == NMRF_F32) hipLaunchKernelGGL(residual_norm_reduce_kernel<float>, dim3((unsigned)grid), dim3(256), 0, st, r);
    else if (dtype == NMRF_BF16) hipLaunchKernelGGL(residual_norm_reduce_kernel<__bf16>, dim3((unsigned)grid), dim3(256), 0, st, r);
    else hipLaunchKernelGGL(residual_norm_reduce_kernel<_Float16>, dim3((unsigned)grid), dim3(256), 0, st, r);
    return nmrf_launch_status();
}
