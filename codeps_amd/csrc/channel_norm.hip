// Norms over the channels of a row (a pixel of an NHWC map, a token) before and behind a residual block, forward and backward.
//   norm only:  h = n(x) w + b
//   block end:  a = n(x) w + b  (or x),   y = r + alpha act(g) a,   h = n'(y) w' + b'     -- one pass: y and h leave together
//   n(v) = (v - mu) rho with rho = (var + eps)^-1/2 ("layer"), or v rho with rho = (mean v^2 + eps)^-1/2 ("rms")
// Backward, with u = n(x), u' = n'(y) and n^T(t) = rho (t - [mean t] - u mean(t u))   ([..]: layer only):
//   D = dy + n'^T(dh w');  dr = D;  dA = alpha act(g) D;  dg = alpha a D act'(g);  dx = n^T(dA w)
//   dw = sum_rows dA u;  db = sum_rows dA;  dw' = sum_rows dh u';  db' = sum_rows dh
// y is formed again from x, r and g in the backward pass instead of being read: the same bytes, and the sums see y before it was rounded to
// its type.  Everything between a load and a store is fp32; each output is rounded once.
//
// A row stays in registers between its reductions, so every tensor crosses HBM once: the pass is bound by bandwidth.  One lane holds E = 4 or 8
// channels as 16-byte pieces; 2^k lanes of a wave share a row up to 512 channels (several rows per wave), beyond that a block of 128 .. 512
// threads holds one row with 8 or 16 channels per thread (two-stage sums through LDS, one barrier each).  Column sums (dw, db, dg, dw', db') live in registers across the rows of
// a block, go to one slab per block and are added in a fixed order by a second launch: no atomics, bitwise reproducible.
#include <algorithm>

#include "common.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));              // rows start at any multiple of the element size
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));

struct bf16 { unsigned short v; };
struct f16 { unsigned short v; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(bf16 x) { return __uint_as_float((unsigned)x.v << 16); }
__device__ __forceinline__ float widen(f16 x) { return (float)__builtin_bit_cast(_Float16, x.v); }
// round to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
__device__ __forceinline__ void narrow(float x, float& o) { o = x; }
__device__ __forceinline__ void narrow(float x, bf16& o) { o.v = __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ __forceinline__ void narrow(float x, f16& o) { o.v = __builtin_bit_cast(unsigned short, (_Float16)x); }

template <int V> __device__ __forceinline__ void load_full(const float* p, float* o) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
        const f32x4u q = *reinterpret_cast<const f32x4u*>(p + 4 * k);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * k + e] = q[e];
    }
}
template <int V, typename T> __device__ __forceinline__ void load_full16(const T* p, float* o) {
    if constexpr (V == 8) {
        const u16x8u q = *reinterpret_cast<const u16x8u*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = widen(T{q[e]});
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = widen(p[e]);
    }
}
template <int V> __device__ __forceinline__ void load_full(const bf16* p, float* o) { load_full16<V, bf16>(p, o); }
template <int V> __device__ __forceinline__ void load_full(const f16* p, float* o) { load_full16<V, f16>(p, o); }

template <int V> __device__ __forceinline__ void store_full(float* p, const float* v) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
        f32x4u q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = v[4 * k + e];
        *reinterpret_cast<f32x4u*>(p + 4 * k) = q;
    }
}
template <int V, typename T> __device__ __forceinline__ void store_full16(T* p, const float* v) {
    if constexpr (V == 8) {
        u16x8u q;
#pragma unroll
        for (int e = 0; e < 8; ++e) { T t; narrow(v[e], t); q[e] = t.v; }
        *reinterpret_cast<u16x8u*>(p) = q;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) narrow(v[e], p[e]);
    }
}
template <int V> __device__ __forceinline__ void store_full(bf16* p, const float* v) { store_full16<V, bf16>(p, v); }
template <int V> __device__ __forceinline__ void store_full(f16* p, const float* v) { store_full16<V, f16>(p, v); }

// element c of a row as a 32-bit byte offset from the row's address: where the row is the same for all lanes, that stays in scalar registers
template <typename T> __device__ __forceinline__ const T* at(const T* row, int c) { return (const T*)((const char*)row + (unsigned)c * (unsigned)sizeof(T)); }
template <typename T> __device__ __forceinline__ T* at(T* row, int c) { return (T*)((char*)row + (unsigned)c * (unsigned)sizeof(T)); }

// V channels from c0 on; the ones past the row's end read as `fill` and are not touched
template <int V, typename T> __device__ __forceinline__ void load_piece(const T* row, int c0, int C, float fill, float* o) {
    if (c0 + V <= C) {
        load_full<V>(at(row, c0), o);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = c0 + e < C ? widen(at(row, c0)[e]) : fill;
    }
}
template <int V, typename T> __device__ __forceinline__ void store_piece(T* row, int c0, int C, const float* v) {
    if (c0 + V <= C) {
        store_full<V>(at(row, c0), v);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c0 + e < C) narrow(v[e], at(row, c0)[e]);
    }
}
// the same behind a type known at run time (weights, gates); the branch is the same for every lane
template <int V> __device__ __forceinline__ void load_any(const void* row, int type, size_t first, int c0, int C, float fill, float* o) {
    if (type == CODEPS_F32) load_piece<V>((const float*)row + first, c0, C, fill, o);
    else if (type == CODEPS_BF16) load_piece<V>((const bf16*)row + first, c0, C, fill, o);
    else load_piece<V>((const f16*)row + first, c0, C, fill, o);
}
template <int V> __device__ __forceinline__ void store_any(void* row, int type, size_t first, int c0, int C, const float* v) {
    if (type == CODEPS_F32) store_piece<V>((float*)row + first, c0, C, v);
    else if (type == CODEPS_BF16) store_piece<V>((bf16*)row + first, c0, C, v);
    else store_piece<V>((f16*)row + first, c0, C, v);
}

template <int V> __device__ __forceinline__ void add_piece(float* row, int c0, int C, const float* v) {
    float o[V];
    load_piece<V>(row, c0, C, 0.f, o);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] += v[e];
    store_piece<V>(row, c0, C, o);
}

struct Args {
    const void *x, *r, *gate, *w, *b, *nw, *nb, *dy, *dh;
    void *y, *h, *dx, *dr, *dgate;
    float *stats, *slab, *gate_slab;
    const float* stats_in;
    long long rows, xp, rp, gp, dyp, dhp;
    int C, kind, next, gate_mode, act, rpi, wt, gt, nt, lpr_log2, items, slices, cols;      // cols: which column sums are wanted (COL_*)
    float scale, eps, neps, inv_c;
};
enum { COL_W = 1, COL_B = 2, COL_NW = 4, COL_NB = 8, COL_G = 16 };

constexpr int WAVE_THREADS = 256;

// Sum over the lanes that share a row, the result in each of them.  `red`: two sets of 16 floats used in turn, so that one barrier per sum is enough
// (a wave reaches the second sum after this one, and with it the same set again, only when all waves have read this one).
template <bool BLOCK> __device__ __forceinline__ float row_sum(float v, int lpr_log2, float (*red)[32], int& turn) {
    if constexpr (!BLOCK) {
        for (int o = (1 << lpr_log2) >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
        return v;
    } else {
        v = wave_sum(v);
        if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = v;
        __syncthreads();
        const int nw = blockDim.x >> 6;
        float t = 0.f;
        for (int i = 0; i < nw; ++i) t += red[turn][i];
        turn ^= 1;
        return t;
    }
}
template <bool BLOCK> __device__ __forceinline__ void row_sum2(float& v, float& q, int lpr_log2, float (*red)[32], int& turn) {
    if constexpr (!BLOCK) {
        for (int o = (1 << lpr_log2) >> 1; o > 0; o >>= 1) { v += __shfl_xor(v, o, 64); q += __shfl_xor(q, o, 64); }
    } else {
        v = wave_sum(v);
        q = wave_sum(q);
        if ((threadIdx.x & 63) == 0) { red[turn][threadIdx.x >> 6] = v; red[turn][16 + (threadIdx.x >> 6)] = q; }
        __syncthreads();
        const int nw = blockDim.x >> 6;
        v = q = 0.f;
        for (int i = 0; i < nw; ++i) { v += red[turn][i]; q += red[turn][16 + i]; }
        turn ^= 1;
    }
}

// mean and 1 / deviation of the row that v holds.  The deviations are summed around the mean, in a second sweep over registers: the difference
// of two large sums would lose them where the mean is large.
template <int V, int NCH, bool BLOCK>
__device__ __forceinline__ void row_stats(const float* v, int kind, float eps, float inv_c, int C, int lane, int lpr, int lpr_log2, float (*red)[32],
                                          int& turn, float& mu, float& rho) {
    mu = 0.f;
    if (kind == CODEPS_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NCH * V; ++k) s += v[k];                          // (channels past the end are zeros)
        mu = row_sum<BLOCK>(s, lpr_log2, red, turn) * inv_c;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        const int c0 = (j * lpr + lane) * V;
        if (c0 + V <= C) {
#pragma unroll
            for (int e = 0; e < V; ++e) { const float d = v[j * V + e] - mu; q += d * d; }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) { const float d = c0 + e < C ? v[j * V + e] - mu : 0.f; q += d * d; }
        }
    }
    q = row_sum<BLOCK>(q, lpr_log2, red, turn);
    rho = 1.f / sqrtf(q * inv_c + eps);
}

__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == CODEPS_GATE_LINEAR) return g;
    const float s = 1.f / (1.f + expf(-g));
    return act == CODEPS_GATE_SIGMOID ? s : g * s;
}
__device__ __forceinline__ void gate_both(float g, int act, float& val, float& slope) {
    if (act == CODEPS_GATE_LINEAR) { val = g; slope = 1.f; return; }
    const float s = 1.f / (1.f + expf(-g));
    if (act == CODEPS_GATE_SIGMOID) { val = s; slope = s * (1.f - s); }
    else { val = g * s; slope = s * (1.f + g * (1.f - s)); }
}
// row of the gate tensor that belongs to a row of x
__device__ __forceinline__ size_t gate_at(const Args& a, long long row) {
    if (a.gate_mode == CODEPS_GATE_CHANNEL) return 0;
    if (a.gate_mode == CODEPS_GATE_ITEM) return (size_t)((unsigned)row / (unsigned)a.rpi) * a.gp;
    return (size_t)row * a.gp;
}

// --------------------------------------------------------------------------------------------------------------------------- forward
template <typename TX, typename TR, int NCH, bool FULL, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? 512 : WAVE_THREADS) void channel_norm_fwd_kernel(Args a) {
    constexpr int V = sizeof(TX) == 4 ? 4 : 8, E = V * NCH;
    __shared__ float red[2][32];
    int turn = 0;
    const int lpr_log2 = a.lpr_log2, lpr = BLOCK ? (int)blockDim.x : 1 << lpr_log2, C = a.C;
    const int lane = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (lpr - 1);
    const int group = BLOCK ? 0 : (int)threadIdx.x >> lpr_log2, rpb = BLOCK ? 1 : WAVE_THREADS >> lpr_log2;

    float w[E], b[E], nw[FULL ? E : 1], nb[FULL ? E : 1];                        // the vectors stay in registers over the rows of a block
    const auto vec = [&](const void* p, int type, int j, float fill, float* o) {
        if (p) load_any<V>(p, type, 0, (j * lpr + lane) * V, C, fill, o);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fill;
        }
    };
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        vec(a.w, a.wt, j, 1.f, w + j * V);
        vec(a.b, a.wt, j, 0.f, b + j * V);
        if constexpr (FULL) {
            vec(a.nw, a.nt, j, 1.f, nw + j * V);
            vec(a.nb, a.nt, j, 0.f, nb + j * V);
        }
    }
    for (long long row = (long long)blockIdx.x * rpb + group; row < a.rows; row += (long long)gridDim.x * rpb) {
        const TX* px = (const TX*)a.x + (size_t)row * a.xp;
        float v[E], rv[FULL ? E : 1], g[FULL ? E : 1];
#pragma unroll
        for (int j = 0; j < NCH; ++j) load_piece<V>(px, (j * lpr + lane) * V, C, 0.f, v + j * V);
        if constexpr (FULL) {
            const TR* pr = (const TR*)a.r + (size_t)row * a.rp;
            const size_t ga = a.gate_mode ? gate_at(a, row) : 0;
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const int c0 = (j * lpr + lane) * V;
                if (a.r) load_piece<V>(pr, c0, C, 0.f, rv + j * V);
                else {
#pragma unroll
                    for (int e = 0; e < V; ++e) rv[j * V + e] = 0.f;
                }
                if (a.gate_mode) load_any<V>(a.gate, a.gt, ga, c0, C, 0.f, g + j * V);
            }
        }
        float mu = 0.f, rho = 1.f, nmu = 0.f, nrho = 1.f;
        if (a.kind) row_stats<V, NCH, BLOCK>(v, a.kind, a.eps, a.inv_c, C, lane, lpr, lpr_log2, red, turn, mu, rho);
#pragma unroll
        for (int k = 0; k < E; ++k) v[k] = (v[k] - mu) * rho * w[k] + b[k];
        if constexpr (!FULL) {
            TX* ph = (TX*)a.h + (size_t)row * C;
#pragma unroll
            for (int j = 0; j < NCH; ++j) store_piece<V>(ph, (j * lpr + lane) * V, C, v + j * V);
            if (a.stats && lane == 0) *reinterpret_cast<float2*>(a.stats + (size_t)row * 2) = make_float2(mu, rho);
        } else {
            TR* py = (TR*)a.y + (size_t)row * C;
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const int c0 = (j * lpr + lane) * V;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int k = j * V + e;
                    const float s = a.gate_mode ? a.scale * gate_value(g[k], a.act) : a.scale;
                    v[k] = c0 + e < C ? rv[k] + s * v[k] : 0.f;
                }
                store_piece<V>(py, c0, C, v + j * V);
            }
            if (a.next) {
                row_stats<V, NCH, BLOCK>(v, a.next, a.neps, a.inv_c, C, lane, lpr, lpr_log2, red, turn, nmu, nrho);
                TX* ph = (TX*)a.h + (size_t)row * C;
#pragma unroll
                for (int k = 0; k < E; ++k) v[k] = (v[k] - nmu) * nrho * nw[k] + nb[k];
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    store_piece<V>(ph, (j * lpr + lane) * V, C, v + j * V);
                }
            }
            if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + (size_t)row * 4) = make_float4(mu, rho, nmu, nrho);
        }
    }
}

// -------------------------------------------------------------------------------------------------------------------------- backward
// Column sums of one kind over the rows this block has seen -> dst[C].  Several rows per block: the row groups meet in LDS, in a fixed order.
template <int V, int NCH, bool BLOCK>
__device__ __forceinline__ void put_columns(const float* acc, float* lds, float* dst, int C, int lane, int group, int lpr, int rpb) {
    if constexpr (BLOCK) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) store_piece<V>(dst, (j * lpr + lane) * V, C, acc + j * V);
    } else {
        const int width = lpr * V * NCH;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) lds[group * width + (j * lpr + lane) * V + e] = acc[j * V + e];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += WAVE_THREADS) {
            float t = 0.f;
            for (int g = 0; g < rpb; ++g) t += lds[g * width + c];
            dst[c] = t;
        }
    }
}

// MEM (16 channels per thread): the column sums are kept in the block's slab (each thread adds to its own columns) and the vectors are read again where they
// are used: five sums and three vectors would take 128 registers next to four tensors of the row
template <typename TX, typename TR, int NCH, bool FULL, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? 512 : WAVE_THREADS) void channel_norm_bwd_kernel(Args a) {
    constexpr int V = sizeof(TX) == 4 ? 4 : 8, E = V * NCH;
    constexpr bool MEM = E > 8;
    __shared__ float red[2][32];
    __shared__ float lds[BLOCK ? 1 : WAVE_THREADS * E];
    int turn = 0;
    const int lpr_log2 = a.lpr_log2, lpr = BLOCK ? (int)blockDim.x : 1 << lpr_log2, C = a.C;
    const int lane = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (lpr - 1);
    const int group = BLOCK ? 0 : (int)threadIdx.x >> lpr_log2, rpb = BLOCK ? 1 : WAVE_THREADS >> lpr_log2;
    const auto vec = [&](const void* p, int type, int j, float fill, float* o) {
        if (p) load_any<V>(p, type, 0, (j * lpr + lane) * V, C, fill, o);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fill;
        }
    };
    float w[E], b[FULL ? E : 1], nw[FULL ? E : 1];
    if constexpr (!MEM) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            vec(a.w, a.wt, j, 1.f, w + j * V);
            if constexpr (FULL) {
                vec(a.b, a.wt, j, 0.f, b + j * V);
                vec(a.nw, a.nt, j, 1.f, nw + j * V);
            }
        }
    }
    float aw[MEM ? 1 : E], ab[MEM ? 1 : E], anw[!MEM && FULL ? E : 1], anb[!MEM && FULL ? E : 1], ag[!MEM && FULL ? E : 1];
    float* const my = a.slab + (size_t)blockIdx.x * 4 * C;                       // [dw | db | dw' | db'] of this block
    const int S = a.slices, slice = (int)(blockIdx.x % (unsigned)S);
    float* myg = nullptr;
    if constexpr (!MEM) {
#pragma unroll
        for (int k = 0; k < E; ++k) aw[k] = ab[k] = 0.f;
        if constexpr (FULL) {
#pragma unroll
            for (int k = 0; k < E; ++k) anw[k] = anb[k] = 0.f;
        }
    } else {
        const float zero[V] = {};
#pragma unroll
        for (int j = 0; j < NCH; ++j)
            for (int q = 0; q < 4; ++q) store_piece<V>(my + q * C, (j * lpr + lane) * V, C, zero);
    }
    const int per = (a.rpi + S - 1) / S;
    for (int item = (int)(blockIdx.x / (unsigned)S); item < a.items; item += (int)(gridDim.x / (unsigned)S)) {
        if constexpr (FULL) {
            myg = a.gate_slab + ((size_t)item * S + slice) * C;
            if constexpr (!MEM) {
#pragma unroll
                for (int k = 0; k < E; ++k) ag[k] = 0.f;
            } else if (a.cols & COL_G) {
                const float zero[V] = {};
#pragma unroll
                for (int j = 0; j < NCH; ++j) store_piece<V>(myg, (j * lpr + lane) * V, C, zero);
            }
        }
        const int first = slice * per, last = min(a.rpi, first + per);
        for (int i = first + group; i < last; i += rpb) {
            const long long row = (long long)item * a.rpi + i;
            float u[E], d[E];                                                  // u = n(x), d: the gradient that runs backward
            const TX* px = (const TX*)a.x + (size_t)row * a.xp;
#pragma unroll
            for (int j = 0; j < NCH; ++j) load_piece<V>(px, (j * lpr + lane) * V, C, 0.f, u + j * V);
            float mu = 0.f, rho = 1.f, nmu = 0.f, nrho = 1.f;
            if constexpr (!FULL) {
                const TX* pd = (const TX*)a.dh + (size_t)row * a.dhp;
#pragma unroll
                for (int j = 0; j < NCH; ++j) load_piece<V>(pd, (j * lpr + lane) * V, C, 0.f, d + j * V);
                const float2 st = *reinterpret_cast<const float2*>(a.stats_in + (size_t)row * 2);
                mu = st.x; rho = st.y;
#pragma unroll
                for (int k = 0; k < E; ++k) u[k] = (u[k] - mu) * rho;
            } else {
                float al[E], dal[E], t[E], y[E];                               // alpha act(g), d(alpha act(g)) / dg * a; dh; r
                const float4 st = *reinterpret_cast<const float4*>(a.stats_in + (size_t)row * 4);
                mu = st.x; rho = st.y; nmu = st.z; nrho = st.w;
                const size_t ga = a.gate_mode ? gate_at(a, row) : 0;
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const int c0 = (j * lpr + lane) * V;
                    if (a.dy) load_piece<V>((const TR*)a.dy + (size_t)row * a.dyp, c0, C, 0.f, d + j * V);
                    else {
#pragma unroll
                        for (int e = 0; e < V; ++e) d[j * V + e] = 0.f;
                    }
                    if (a.next) {
                        load_piece<V>((const TX*)a.dh + (size_t)row * a.dhp, c0, C, 0.f, t + j * V);
                        if (a.r) load_piece<V>((const TR*)a.r + (size_t)row * a.rp, c0, C, 0.f, y + j * V);
                        else {
#pragma unroll
                            for (int e = 0; e < V; ++e) y[j * V + e] = 0.f;
                        }
                    }
                    if (a.gate_mode) load_any<V>(a.gate, a.gt, ga, c0, C, 0.f, al + j * V);
                }
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    if constexpr (MEM) { vec(a.w, a.wt, j, 1.f, w + j * V); vec(a.b, a.wt, j, 0.f, b + j * V); }
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int k = j * V + e;
                        u[k] = (u[k] - mu) * rho;
                        const float an = u[k] * w[k] + b[k];
                        float val = 1.f, slope = 0.f;
                        if (a.gate_mode) gate_both(al[k], a.act, val, slope);
                        al[k] = a.scale * val;
                        dal[k] = a.scale * slope * an;
                        if (a.next) y[k] += al[k] * an;
                    }
                }
                if (a.next) {                                                  // d += n'^T(dh w')
                    float s1 = 0.f, s2 = 0.f;
#pragma unroll
                    for (int j = 0; j < NCH; ++j) {
                        if constexpr (MEM) vec(a.nw, a.nt, j, 1.f, nw + j * V);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const int k = j * V + e;
                            y[k] = (y[k] - nmu) * nrho;
                            if constexpr (!MEM) { anw[k] += t[k] * y[k]; anb[k] += t[k]; }
                        }
                        if constexpr (MEM) {
                            float q[V];
#pragma unroll
                            for (int e = 0; e < V; ++e) q[e] = t[j * V + e] * y[j * V + e];
                            if (a.cols & COL_NW) add_piece<V>(my + 2 * C, (j * lpr + lane) * V, C, q);
                            if (a.cols & COL_NB) add_piece<V>(my + 3 * C, (j * lpr + lane) * V, C, t + j * V);
                        }
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const int k = j * V + e;
                            t[k] *= nw[k];
                            s1 += t[k];                                        // (dh is 0 past the end)
                            s2 += t[k] * y[k];
                        }
                    }
                    row_sum2<BLOCK>(s1, s2, lpr_log2, red, turn);
                    s1 = a.next == CODEPS_NORM_LAYER ? s1 * a.inv_c : 0.f;
                    s2 *= a.inv_c;
#pragma unroll
                    for (int k = 0; k < E; ++k) d[k] += nrho * (t[k] - s1 - y[k] * s2);
                }
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    const int c0 = (j * lpr + lane) * V;
                    if (c0 + V > C) {
#pragma unroll
                        for (int e = 0; e < V; ++e)
                            if (c0 + e >= C) d[j * V + e] = 0.f;
                    }
                    if (a.dr) store_piece<V>((TR*)a.dr + (size_t)row * C, c0, C, d + j * V);
                    if (a.gate_mode) {
#pragma unroll
                        for (int e = 0; e < V; ++e) dal[j * V + e] *= d[j * V + e];
                        if (a.gate_mode == CODEPS_GATE_ELEMENT) {
                            if (a.dgate) store_any<V>(a.dgate, a.gt, (size_t)row * C, c0, C, dal + j * V);
                        } else {
                            if constexpr (!MEM) {
#pragma unroll
                                for (int e = 0; e < V; ++e) ag[j * V + e] += dal[j * V + e];
                            } else if (a.cols & COL_G) {
                                add_piece<V>(myg, c0, C, dal + j * V);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) d[j * V + e] *= al[j * V + e];
                }
            }
            // d = the gradient of a: its column sums, then through n
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                if constexpr (MEM) vec(a.w, a.wt, j, 1.f, w + j * V);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int k = j * V + e;
                    if constexpr (!MEM) { aw[k] += d[k] * u[k]; ab[k] += d[k]; }
                }
                if constexpr (MEM) {
                    float q[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) q[e] = d[j * V + e] * u[j * V + e];
                    if (a.cols & COL_W) add_piece<V>(my, (j * lpr + lane) * V, C, q);
                    if (a.cols & COL_B) add_piece<V>(my + C, (j * lpr + lane) * V, C, d + j * V);
                }
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int k = j * V + e;
                    d[k] *= w[k];
                    s1 += d[k];
                    s2 += d[k] * u[k];
                }
            }
            if (a.kind) {
                row_sum2<BLOCK>(s1, s2, lpr_log2, red, turn);
                s1 = a.kind == CODEPS_NORM_LAYER ? s1 * a.inv_c : 0.f;
                s2 *= a.inv_c;
#pragma unroll
                for (int k = 0; k < E; ++k) d[k] = rho * (d[k] - s1 - u[k] * s2);
            }
            if (a.dx) {
                TX* pdx = (TX*)a.dx + (size_t)row * C;
#pragma unroll
                for (int j = 0; j < NCH; ++j) store_piece<V>(pdx, (j * lpr + lane) * V, C, d + j * V);
            }
        }
        if constexpr (FULL && !MEM) {
            if (a.cols & COL_G) put_columns<V, NCH, BLOCK>(ag, lds, myg, C, lane, group, lpr, rpb);
        }
    }
    if constexpr (!MEM) {
        if (a.cols & COL_W) put_columns<V, NCH, BLOCK>(aw, lds, my, C, lane, group, lpr, rpb);
        if (a.cols & COL_B) put_columns<V, NCH, BLOCK>(ab, lds, my + C, C, lane, group, lpr, rpb);
        if constexpr (FULL) {
            if (a.cols & COL_NW) put_columns<V, NCH, BLOCK>(anw, lds, my + 2 * C, C, lane, group, lpr, rpb);
            if (a.cols & COL_NB) put_columns<V, NCH, BLOCK>(anb, lds, my + 3 * C, C, lane, group, lpr, rpb);
        }
    }
}

// out[g][c] (+)= sum over n of part[(g * n + i) * pitch + c], in a fixed order: 16 columns x 16 strided streams per block
struct Finish {
    const float* part[5];
    void* out[5];
    int type[5], groups[5], n[5], pitch[5], accumulate[5];
    int C;
};
__global__ __launch_bounds__(256) void channel_norm_finish_kernel(Finish f) {
    __shared__ float red[16][17];
    const int k = blockIdx.z, g = blockIdx.y, c = blockIdx.x * 16 + (threadIdx.x & 15), s = threadIdx.x >> 4;
    if (g >= f.groups[k]) return;
    const int n = f.n[k];
    const size_t pitch = f.pitch[k];
    float t0 = 0.f, t1 = 0.f, t2 = 0.f, t3 = 0.f;
    if (c < f.C) {
        const float* p = f.part[k] + (size_t)g * n * pitch + c;
        int i = s;
        for (; i + 48 < n; i += 64) {
            t0 += p[(size_t)i * pitch];
            t1 += p[(size_t)(i + 16) * pitch];
            t2 += p[(size_t)(i + 32) * pitch];
            t3 += p[(size_t)(i + 48) * pitch];
        }
        for (; i < n; i += 16) t0 += p[(size_t)i * pitch];
    }
    red[s][threadIdx.x & 15] = (t0 + t1) + (t2 + t3);
    __syncthreads();
    if (s == 0 && c < f.C) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += red[i][threadIdx.x & 15];
        const size_t at = (size_t)g * f.C + c;
        if (f.type[k] == CODEPS_F32) { float* o = (float*)f.out[k] + at; *o = f.accumulate[k] ? *o + t : t; }
        else if (f.type[k] == CODEPS_BF16) narrow(t, ((bf16*)f.out[k])[at]);
        else narrow(t, ((f16*)f.out[k])[at]);
    }
}

// --------------------------------------------------------------------------------------------------------------------------- launch
constexpr int MAX_C = 8192, MAX_BLOCKS = 1024;

// lanes per row and channels per lane: in one wave while 8 channels per lane do (16-byte loads, no barrier), then a block of up to 512 threads with 8
// channels per thread, then with 16
struct Shape { bool block; int nch, lpr_log2, threads, rpb; };
Shape shape_of(const codeps_channel_norm_desc* d) {
    const int V = d->x_type == CODEPS_F32 ? 4 : 8, C = d->channels;
    Shape s{false, 1, 0, WAVE_THREADS, 0};
    if (C <= 64 * 8) {
        s.nch = V == 4 && C > 64 * 4 ? 2 : 1;
        while ((V * s.nch << s.lpr_log2) < C) ++s.lpr_log2;
        s.rpb = WAVE_THREADS >> s.lpr_log2;
        return s;
    }
    s.block = true;
    s.rpb = 1;
    const int E = C <= 512 * 8 ? 8 : 16;
    s.nch = E / V;
    s.threads = cdiv(cdiv(C, E), 64) * 64;
    return s;
}
struct Plan { Shape s; int items, rpi, slices, blocks; size_t slab, gate_slab; };
Plan plan_of(const codeps_channel_norm_desc* d) {
    Plan p;
    p.s = shape_of(d);
    const bool per_item = d->gate_mode == CODEPS_GATE_ITEM;
    p.rpi = per_item ? d->rows_per_item : (int)d->rows;
    p.items = per_item ? std::max(1, (int)(d->rows / d->rows_per_item)) : 1;
    // enough blocks to fill 256 CUs, and at least 8 rows for each row group of a block where there are that many: the column sums' slabs are a cost per block
    const long long want = std::max<long long>(256, std::min<long long>(MAX_BLOCKS, d->rows / (8LL * p.s.rpb)));
    const long long most = std::max<long long>(1, cdiv(p.rpi, p.s.rpb));
    p.slices = (int)std::max<long long>(1, std::min<long long>(most, want / p.items));
    p.blocks = (int)std::min<long long>(p.items, std::max<long long>(1, MAX_BLOCKS / p.slices)) * p.slices;
    p.slab = (size_t)p.blocks * 4 * d->channels;
    p.gate_slab = d->gate_mode == CODEPS_GATE_CHANNEL || per_item ? (size_t)(per_item ? p.items : 1) * p.slices * d->channels : 0;
    return p;
}

int check_desc(const codeps_channel_norm_desc* d, const char* who) {
    CODEPS_REQUIRE(d, CODEPS_ERR_ARG, "%s: null descriptor", who);
    const auto type_ok = [](int t) { return t == CODEPS_F32 || t == CODEPS_BF16 || t == CODEPS_F16; };
    CODEPS_REQUIRE(d->rows >= 0 && d->rows < (1LL << 31) && d->channels >= 1 && d->channels <= MAX_C, CODEPS_ERR_ARG,
                   "%s: %lld rows of %d channels (at most 2^31 - 1 rows, 1 .. %d channels)", who, (long long)d->rows, d->channels, MAX_C);
    CODEPS_REQUIRE(type_ok(d->x_type) && type_ok(d->res_type) && type_ok(d->weight_type) && type_ok(d->gate_type) && type_ok(d->next_weight_type),
                   CODEPS_ERR_ARG, "%s: unknown element type", who);
    CODEPS_REQUIRE(d->res_type == d->x_type || d->res_type == CODEPS_F32, CODEPS_ERR_ARG, "%s: the residual has x's type or fp32", who);
    CODEPS_REQUIRE(d->kind >= CODEPS_NORM_NONE && d->kind <= CODEPS_NORM_RMS && d->next_kind >= CODEPS_NORM_NONE && d->next_kind <= CODEPS_NORM_RMS,
                   CODEPS_ERR_ARG, "%s: unknown norm", who);
    CODEPS_REQUIRE(d->gate_mode >= CODEPS_GATE_NONE && d->gate_mode <= CODEPS_GATE_ELEMENT && d->gate_act >= CODEPS_GATE_LINEAR &&
                   d->gate_act <= CODEPS_GATE_SILU, CODEPS_ERR_ARG, "%s: unknown gate", who);
    CODEPS_REQUIRE(d->gate_mode != CODEPS_GATE_ITEM || (d->rows_per_item >= 1 && d->rows % d->rows_per_item == 0), CODEPS_ERR_ARG,
                   "%s: %lld rows are not whole items of %d", who, (long long)d->rows, d->rows_per_item);
    const long long C = d->channels;
    CODEPS_REQUIRE(d->x_pitch >= C && (d->full == 0 || d->res_pitch >= C) && (d->gate_mode < CODEPS_GATE_ITEM || d->gate_pitch >= C), CODEPS_ERR_ARG,
                   "%s: a row pitch is smaller than the row", who);
    CODEPS_REQUIRE(d->full || (d->kind != CODEPS_NORM_NONE && d->next_kind == CODEPS_NORM_NONE && d->gate_mode == CODEPS_GATE_NONE), CODEPS_ERR_ARG,
                   "%s: a norm on its own has a kind and neither gate nor next norm", who);
    return CODEPS_OK;
}

Args args_of(const codeps_channel_norm_desc* d, const Shape& s) {
    Args a{};
    a.rows = d->rows; a.C = d->channels; a.xp = d->x_pitch; a.rp = d->res_pitch; a.gp = d->gate_pitch; a.dyp = d->dy_pitch; a.dhp = d->dh_pitch;
    a.kind = d->kind; a.next = d->next_kind; a.gate_mode = d->gate_mode; a.act = d->gate_act; a.rpi = d->rows_per_item;
    a.wt = d->weight_type; a.gt = d->gate_type; a.nt = d->next_weight_type;
    a.scale = d->scale; a.eps = d->eps; a.neps = d->next_eps; a.inv_c = (float)(1.0 / d->channels);
    a.lpr_log2 = s.lpr_log2; a.items = 1; a.slices = 1;
    return a;
}

template <typename TX> constexpr int pieces_of = sizeof(TX) == 4 ? 2 : 1;          // 16-byte pieces that are 8 channels
template <typename TX, typename TR, int NCH, bool FULL>
void launch_fwd(const Args& a, const Shape& s, hipStream_t st) {
    const int blocks = (int)std::min<long long>((a.rows + s.rpb - 1) / s.rpb, 4096);
    if constexpr (NCH >= pieces_of<TX>)
        if (s.block) hipLaunchKernelGGL((channel_norm_fwd_kernel<TX, TR, NCH, FULL, true>), dim3(blocks), dim3(s.threads), 0, st, a);
    if constexpr (NCH <= pieces_of<TX>)
        if (!s.block) hipLaunchKernelGGL((channel_norm_fwd_kernel<TX, TR, NCH, FULL, false>), dim3(blocks), dim3(s.threads), 0, st, a);
}
template <typename TX, typename TR, int NCH, bool FULL>
void launch_bwd(const Args& a, const Shape& s, int blocks, hipStream_t st) {
    if constexpr (NCH >= pieces_of<TX>)
        if (s.block) hipLaunchKernelGGL((channel_norm_bwd_kernel<TX, TR, NCH, FULL, true>), dim3(blocks), dim3(s.threads), 0, st, a);
    if constexpr (NCH <= pieces_of<TX>)
        if (!s.block) hipLaunchKernelGGL((channel_norm_bwd_kernel<TX, TR, NCH, FULL, false>), dim3(blocks), dim3(s.threads), 0, st, a);
}
// every (type, pieces per lane) that shape_of can ask for
template <typename F> void dispatch(const codeps_channel_norm_desc* d, const Shape& s, F&& f) {
    const auto pieces = [&](auto tx, auto tr) {
        if constexpr (sizeof(tx) == 4) {
            if (s.nch == 1) f(tx, tr, std::integral_constant<int, 1>{});
            else if (s.nch == 2) f(tx, tr, std::integral_constant<int, 2>{});
            else f(tx, tr, std::integral_constant<int, 4>{});
        } else {
            if (s.nch == 1) f(tx, tr, std::integral_constant<int, 1>{});
            else f(tx, tr, std::integral_constant<int, 2>{});
        }
    };
    if (d->x_type == CODEPS_F32) pieces(float{}, float{});
    else if (d->x_type == CODEPS_BF16) { if (d->res_type == CODEPS_F32 && d->full) pieces(bf16{}, float{}); else pieces(bf16{}, bf16{}); }
    else { if (d->res_type == CODEPS_F32 && d->full) pieces(f16{}, float{}); else pieces(f16{}, f16{}); }
}

}  // namespace

// =============================================================================================== C ABI
extern "C" int codeps_channel_norm_fwd(const codeps_channel_norm_desc* d, const void* x, const void* residual, const void* gate, const void* weight,
                                       const void* bias, const void* next_weight, const void* next_bias, void* y, void* h, float* stats,
                                       codeps_stream_t stream) {
    const int rc = check_desc(d, "channel_norm_fwd");
    if (rc != CODEPS_OK) return rc;
    if (d->rows == 0) return CODEPS_OK;
    CODEPS_REQUIRE(x && (d->full ? y != nullptr : h != nullptr) && (!d->next_kind || h) && (!d->gate_mode || gate), CODEPS_ERR_ARG,
                   "channel_norm_fwd: null pointer");
    const Shape s = shape_of(d);
    Args a = args_of(d, s);
    a.x = x; a.r = residual; a.gate = gate; a.w = weight; a.b = bias; a.nw = next_weight; a.nb = next_bias; a.y = y; a.h = h; a.stats = stats;
    hipStream_t st = (hipStream_t)stream;
    dispatch(d, s, [&](auto tx, auto tr, auto nch) {
        using TX = decltype(tx);
        using TR = decltype(tr);
        constexpr int NCH = decltype(nch)::value;
        if (d->full) launch_fwd<TX, TR, NCH, true>(a, s, st);
        else if constexpr (std::is_same<TX, TR>::value) launch_fwd<TX, TR, NCH, false>(a, s, st);
    });
    CODEPS_CHECK_LAUNCH("channel_norm_fwd_kernel");
    return CODEPS_OK;
}

extern "C" size_t codeps_channel_norm_bwd_workspace_bytes(const codeps_channel_norm_desc* d) {
    if (check_desc(d, "channel_norm_bwd_workspace_bytes") != CODEPS_OK) return 0;
    const Plan p = plan_of(d);
    return std::max<size_t>(256, (p.slab + p.gate_slab) * sizeof(float));
}

extern "C" int codeps_channel_norm_bwd(const codeps_channel_norm_desc* d, const void* x, const void* residual, const void* gate, const void* weight,
                                       const void* bias, const void* next_weight, const float* stats, const void* dy, const void* dh, void* dx,
                                       void* dresidual, void* dgate, void* dweight, void* dbias, void* dnext_weight, void* dnext_bias, int accumulate,
                                       void* workspace, size_t workspace_bytes, codeps_stream_t stream) {
    const int rc = check_desc(d, "channel_norm_bwd");
    if (rc != CODEPS_OK) return rc;
    const Plan p = plan_of(d);
    CODEPS_REQUIRE(workspace && workspace_bytes >= codeps_channel_norm_bwd_workspace_bytes(d), CODEPS_ERR_WORKSPACE,
                   "channel_norm_bwd: %zu bytes of workspace, %zu are needed", workspace_bytes, codeps_channel_norm_bwd_workspace_bytes(d));
    CODEPS_REQUIRE((accumulate & ~(CODEPS_ACC_WEIGHT | CODEPS_ACC_BIAS | CODEPS_ACC_NEXT_WEIGHT | CODEPS_ACC_NEXT_BIAS)) == 0, CODEPS_ERR_ARG,
                   "channel_norm_bwd: unknown accumulate bits %d", accumulate);
    CODEPS_REQUIRE((!(accumulate & (CODEPS_ACC_WEIGHT | CODEPS_ACC_BIAS)) || d->weight_type == CODEPS_F32) &&
                   (!(accumulate & (CODEPS_ACC_NEXT_WEIGHT | CODEPS_ACC_NEXT_BIAS)) || d->next_weight_type == CODEPS_F32), CODEPS_ERR_ARG,
                   "channel_norm_bwd: gradients are accumulated in fp32 only");
    if (d->rows > 0) {
        CODEPS_REQUIRE(x && stats && (!d->gate_mode || gate) && (d->full ? (dy || d->next_kind) : dh != nullptr) && (!d->next_kind || dh), CODEPS_ERR_ARG,
                       "channel_norm_bwd: null pointer");
        CODEPS_REQUIRE((!dy || d->dy_pitch >= d->channels) && (!dh || d->dh_pitch >= d->channels), CODEPS_ERR_ARG,
                       "channel_norm_bwd: a row pitch is smaller than the row");
    }
    hipStream_t st = (hipStream_t)stream;
    float* slab = (float*)workspace;
    const bool columns = d->gate_mode == CODEPS_GATE_CHANNEL || d->gate_mode == CODEPS_GATE_ITEM;
    if (d->rows > 0) {
        Args a = args_of(d, p.s);
        a.x = x; a.r = residual; a.gate = gate; a.w = weight; a.b = bias; a.nw = next_weight; a.stats_in = stats; a.dy = dy; a.dh = dh;
        a.dx = dx; a.dr = dresidual; a.dgate = dgate; a.slab = slab; a.gate_slab = slab + p.slab;
        a.items = p.items; a.rpi = p.rpi; a.slices = p.slices;
        a.cols = (dweight ? COL_W : 0) | (dbias ? COL_B : 0) | (dnext_weight && d->next_kind ? COL_NW : 0) | (dnext_bias && d->next_kind ? COL_NB : 0) |
                 (dgate && columns ? COL_G : 0);
        dispatch(d, p.s, [&](auto tx, auto tr, auto nch) {
            using TX = decltype(tx);
            using TR = decltype(tr);
            constexpr int NCH = decltype(nch)::value;
            if (d->full) launch_bwd<TX, TR, NCH, true>(a, p.s, p.blocks, st);
            else if constexpr (std::is_same<TX, TR>::value) launch_bwd<TX, TR, NCH, false>(a, p.s, p.blocks, st);
        });
        CODEPS_CHECK_LAUNCH("channel_norm_bwd_kernel");
    }
    Finish f{};
    int k = 0, groups = 1;
    f.C = d->channels;
    const auto add = [&](const float* part, void* out, int type, int g, int n, int pitch, int acc) {
        if (!out) return;
        f.part[k] = part; f.out[k] = out; f.type[k] = type; f.groups[k] = g; f.n[k] = d->rows > 0 ? n : 0; f.pitch[k] = pitch; f.accumulate[k] = acc;
        groups = std::max(groups, g);
        ++k;
    };
    const int C = d->channels;
    add(slab, dweight, d->weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_WEIGHT);
    add(slab + C, dbias, d->weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_BIAS);
    if (d->next_kind) {
        add(slab + 2 * C, dnext_weight, d->next_weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_NEXT_WEIGHT);
        add(slab + 3 * C, dnext_bias, d->next_weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_NEXT_BIAS);
    }
    if (columns && (d->rows > 0 || d->gate_mode == CODEPS_GATE_CHANNEL)) add(slab + p.slab, dgate, d->gate_type, p.items, p.slices, C, 0);
    // (items behind the 65535th have their own launch: a grid's second dimension ends there)
    for (int g0 = 0; k > 0 && g0 < groups; g0 += 65535) {
        Finish part = f;
        for (int i = 0; i < k; ++i) {
            const int skip = std::min(g0, f.groups[i]);
            part.groups[i] = std::min(f.groups[i] - skip, 65535);
            part.part[i] = f.part[i] + (size_t)skip * f.n[i] * f.pitch[i];
            part.out[i] = (char*)f.out[i] + (size_t)skip * C * (f.type[i] == CODEPS_F32 ? 4 : 2);
        }
        hipLaunchKernelGGL(channel_norm_finish_kernel, dim3(cdiv(C, 16), std::min(groups - g0, 65535), k), dim3(256), 0, st, part);
        CODEPS_CHECK_LAUNCH("channel_norm_finish_kernel");
    }
    return CODEPS_OK;
}
