// What the forward and the backward kernel of the channel norms share (channel_norm_fwd.hip, channel_norm_bwd.hip).
//
//   norm only:  h = n(x) w + b
//   block end:  a = n(x) w + b  (or x w + b),   y = r + alpha act(g) a,   h = n'(y) w' + b'     -- one pass: y and h leave together
//   n(v) = (v - mu) rho with rho = (var + eps)^-1/2 ("layer"), or v rho with rho = (mean v^2 + eps)^-1/2 ("rms")
//
// A row (the channels of a pixel or token) stays in registers between its sums, so every tensor crosses HBM once: the pass is bound by bandwidth, and by
// instructions where rows are short.  A lane holds E = 4 or 8 channels as 16-byte pieces; 2^k lanes of a wave share a row up to 512 channels (several rows
// per wave), beyond that a block of 128 .. 1024 threads holds one row with 8 channels per thread (two-stage sums through LDS, one barrier each).
// Everything between a load and a store is fp32; each output is rounded once.
//
// Kernels come in two forms: rows of whole pieces (channels a multiple of 4 or 8), whose loads have no branch -- a branch per load makes the compiler
// wait for each one before the next -- and rows that end inside a piece, whose last piece is loaded from the row's end and shifted.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));              // rows start at any multiple of the element size
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned int u32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

struct bf16 { unsigned short v; };
struct f16 { unsigned short v; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(bf16 x) { return __uint_as_float((unsigned)x.v << 16); }
__device__ __forceinline__ float widen(f16 x) { return (float)__builtin_bit_cast(_Float16, x.v); }
// round to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
__device__ __forceinline__ void narrow(float x, float& o) { o = x; }
__device__ __forceinline__ void narrow(float x, bf16& o) { o.v = __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ __forceinline__ void narrow(float x, f16& o) { o.v = __builtin_bit_cast(unsigned short, (_Float16)x); }

template <int V, typename T> __device__ __forceinline__ void load_full(const T* p, float* o) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int k = 0; k < V / 4; ++k) {
            const f32x4u q = *reinterpret_cast<const f32x4u*>(p + 4 * k);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[4 * k + e] = q[e];
        }
    } else if constexpr (V == 8) {
        const u16x8u q = *reinterpret_cast<const u16x8u*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = widen(T{q[e]});
    } else {                                                        // (a 16-bit vector next to fp32 rows: outside the row loop only)
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = widen(p[e]);
    }
}
template <int V, typename T> __device__ __forceinline__ void store_full(T* p, const float* v) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int k = 0; k < V / 4; ++k) {
            f32x4u q;
#pragma unroll
            for (int e = 0; e < 4; ++e) q[e] = v[4 * k + e];
            *reinterpret_cast<f32x4u*>(p + 4 * k) = q;
        }
    } else {
        static_assert(V == 8, "16-bit rows have pieces of 8");
        u16x8u q;
#pragma unroll
        for (int e = 0; e < 8; ++e) { T t; narrow(v[e], t); q[e] = t.v; }
        *reinterpret_cast<u16x8u*>(p) = q;
    }
}

// element c from a row's address on, as a 32-bit byte offset.  Row addresses are the same for all lanes of a wave (the wave's first row; lanes of its other rows
// carry their distance in c): they stay in scalar registers, and the lanes' offsets do not change from row to row.
template <typename T> __device__ __forceinline__ const T* at(const T* row, int c) { return (const T*)((const char*)row + (unsigned)c * (unsigned)sizeof(T)); }
template <typename T> __device__ __forceinline__ T* at(T* row, int c) { return (T*)((char*)row + (unsigned)c * (unsigned)sizeof(T)); }

// V channels from c0 on of the row that lies `off` elements behind `row`, as they lie in memory.  Whole pieces (TAIL false): a lane behind the row's end reads
// the row's first piece, which its caller leaves out of every sum and every store.  TAIL: the piece that crosses the end is read from the row's last V
// elements and shifted by widen_piece; elements past the end are 0.
template <int V, typename T> struct Raw { unsigned w[V * sizeof(T) / 4]; };
template <int V, bool TAIL, typename T> __device__ __forceinline__ Raw<V, T> raw_piece(const T* row, int off, int c0, int C) {
    constexpr int PER = 4 / sizeof(T), W = V / PER;                           // elements per word, words
    Raw<V, T> r;
    if (TAIL && C < V) {
#pragma unroll
        for (int e = 0; e < W; ++e) r.w[e] = 0;
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c0 + e < C) r.w[e / PER] |= (PER == 1 ? ((const unsigned*)(const void*)at(row, off + c0))[e]
                                                      : (unsigned)((const unsigned short*)(const void*)at(row, off + c0))[e] << (16 * (e % PER)));
    } else {
        const char* p = reinterpret_cast<const char*>(at(row, off + (TAIL ? min(c0, C - V) : c0 < C ? c0 : 0)));
#pragma unroll
        for (int k = 0; k < W / 4; ++k) {
            const u32x4u q = *reinterpret_cast<const u32x4u*>(p + 16 * k);
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[4 * k + e] = q[e];
        }
    }
    return r;
}
template <int V, bool TAIL, typename T> __device__ __forceinline__ void widen_piece(Raw<V, T> r, int c0, int C, float* o) {
    constexpr int PER = 4 / sizeof(T), W = V / PER;
    if (TAIL && C >= V) {                                                     // the shift works on whole words, two 16-bit elements at a time
        const int sh = c0 - min(c0, C - V);
#pragma unroll
        for (int s = W / 2; s > 0; s /= 2)
#pragma unroll
            for (int e = 0; e < W; ++e) r.w[e] = (sh & (s * PER)) ? (e + s < W ? r.w[e + s] : 0u) : r.w[e];
        if constexpr (PER == 2) {
            const unsigned bits = (sh & 1) * 16;
#pragma unroll
            for (int e = 0; e < W; ++e) r.w[e] = __builtin_amdgcn_alignbit(e + 1 < W ? r.w[e + 1] : 0u, r.w[e], bits);
        }
#pragma unroll
        for (int e = 0; e < W; ++e) r.w[e] = sh >= V ? 0u : r.w[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if constexpr (PER == 1) o[e] = __uint_as_float(r.w[e]);
        else o[e] = widen(T{(unsigned short)(e % 2 ? r.w[e / 2] >> 16 : r.w[e / 2] & 0xffffu)});
    }
}
template <int V, bool TAIL, typename T> __device__ __forceinline__ void load_piece(const T* row, int off, int c0, int C, float* o) {
    widen_piece<V, TAIL>(raw_piece<V, TAIL>(row, off, c0, C), c0, C, o);
}
template <int V, bool TAIL, typename T> __device__ __forceinline__ void store_piece(T* row, int off, int c0, int C, const float* v) {
    if (c0 + V <= C) {
        store_full<V>(at(row, off + c0), v);
    } else if constexpr (TAIL) {                                     // V / 2, V / 4, .. elements at a time, by the bits of what is left
        const int left = max(C - c0, 0);
        T* p = at(row, off + c0);
        T t[V];
#pragma unroll
        for (int e = 0; e < V; ++e) narrow(v[e], t[e]);
#pragma unroll
        for (int n = V / 2; n > 0; n /= 2) {
            if (left & n) {
                __builtin_memcpy(p, t, n * sizeof(T));
                p += n;
#pragma unroll
                for (int e = 0; e < n; ++e) t[e] = t[e + n];
            }
        }
    }
}
// a vector [C] of a type known at run time (outside the row loop); absent: fill
template <int V> __device__ __forceinline__ void load_vector(const void* p, int type, size_t first, int c0, int C, float fill, float* o) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = fill;
    if (!p) return;
    if (c0 + V <= C) {
        if (type == CODEPS_F32) load_full<V>((const float*)p + first + c0, o);
        else if (type == CODEPS_BF16) load_full<V>((const bf16*)p + first + c0, o);
        else load_full<V>((const f16*)p + first + c0, o);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c0 + e < C) {
                if (type == CODEPS_F32) o[e] = ((const float*)p)[first + c0 + e];
                else if (type == CODEPS_BF16) o[e] = widen(((const bf16*)p)[first + c0 + e]);
                else o[e] = widen(((const f16*)p)[first + c0 + e]);
            }
    }
}

struct Args {
    const void *x, *r, *gate, *w, *b, *nw, *nb, *dy, *dh;
    void *y, *h, *dx, *dr, *dgate;
    float *stats, *slab, *gate_slab, *row_sums;
    const float* stats_in;
    long long rows, xp, rp, gp, dyp, dhp;
    int C, kind, next, act, rpi, shared_lines, wt, gt, nt, lpr_log2, items, slices, cols;      // cols: which column sums are wanted (COL_*)
    float scale, eps, neps, inv_c;
};
enum { COL_W = 1, COL_B = 2, COL_NW = 4, COL_NB = 8, COL_G = 16 };
enum { GATE_NONE, GATE_HELD, GATE_ROWS };           // no gate | one row of it for all rows of an item, kept in registers | as many rows as x

constexpr int WAVE_THREADS = 256;

// Which rows and channels a thread works on.  first: the wave's first row of the block's turn (the same for all lanes), sub: this lane's row behind it.
struct Place { int lpr, lane, first, sub, rpb; };
template <bool BLOCK> __device__ __forceinline__ Place place_of(int lpr_log2) {
    if constexpr (BLOCK) return {(int)blockDim.x, (int)threadIdx.x, 0, 0, 1};
    const int per_wave = 64 >> lpr_log2, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), in_wave = (int)threadIdx.x & 63;
    return {1 << lpr_log2, in_wave & ((1 << lpr_log2) - 1), wave * per_wave, in_wave >> lpr_log2, WAVE_THREADS >> lpr_log2};
}

// The slice of a block.  Blocks go to the 8 XCDs in turn.  Where a row is not a whole number of 128-byte lines, neighbouring slices, whose rows share lines, are
// given to blocks of one XCD, and its L2 merges their parts of a line: norm alone, bf16, forward and backward, 32768 x 1000 86 -> 82 us, 32768 x 1001 109 -> 106;
// whole lines are better off in turn (262144 x 256 132 against 137 us).
__device__ __forceinline__ int slice_of(unsigned block, int S, bool shared_lines) {
    const int s = (int)(block % (unsigned)S);
    return shared_lines && S % 8 == 0 ? (s & 7) * (S >> 3) + (s >> 3) : s;
}

// ---- sums over the lanes that share a row: lanes 1, 2, 4, 8 away over DPP, 16 and 32 away by exchanging half rows (no LDS, no waits)
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float add16(float v) {
    const u32x2 q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
__device__ __forceinline__ float add32(float v) {
    const u32x2 q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
template <int N> __device__ __forceinline__ void lanes_sum(float (&v)[N], int log2) {
    const auto step = [&](auto f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = f(v[i]);
    };
    if (log2 > 0) step([](float x) { return x + dpp<0xB1>(x); });       // quad: 1 0 3 2
    if (log2 > 1) step([](float x) { return x + dpp<0x4E>(x); });       // quad: 2 3 0 1
    if (log2 > 2) step([](float x) { return x + dpp<0x141>(x); });      // half row mirrored (quads are uniform by now)
    if (log2 > 3) step([](float x) { return x + dpp<0x140>(x); });      // row mirrored
    if (log2 > 4) step([](float x) { return add16(x); });
    if (log2 > 5) step([](float x) { return add32(x); });
}
// N sums at once, each lane gets them.  BLOCK: `red` has two sets used in turn, so that one barrier per call is enough (a wave reaches the second call after
// this one, and with it the same set again, only when all waves have read this one).
template <bool BLOCK, int N> __device__ __forceinline__ void row_sums(float (&v)[N], int lpr_log2, float (*red)[32], int& turn) {
    if constexpr (!BLOCK) {
        lanes_sum(v, lpr_log2);
    } else {
        lanes_sum(v, 6);
        const int waves = blockDim.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) red[turn][16 * i + (threadIdx.x >> 6)] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
            for (int k = 0; k < waves; ++k) v[i] += red[turn][16 * i + k];
        }
        turn ^= 1;
    }
}
// sum over one piece of what lies inside the row.  TAIL: keep[e] = all ones inside the row, 0 behind it; not needed where the values behind it are zeros.
template <int V, bool TAIL, bool ZEROS> __device__ __forceinline__ float piece_sum(const float* v, int left, const unsigned* keep) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) s += TAIL && !ZEROS ? __uint_as_float(__float_as_uint(v[e]) & keep[e]) : v[e];
    return TAIL || left > 0 ? s : 0.f;
}

// 1 / (1 + exp(-g)) on the hardware's 2^x and reciprocal (1 step each); the rounding of g log2(e) is carried along, or it would cost |g| steps.  That
// rounding, lo, is far below 1 while e counts; for g = +inf and finite gates whose product overflows it is infinite or NaN beside e = 0, hence the minimum.
__device__ __forceinline__ float sigmoid(float g) {
    const float hi = g * -1.44269504f, lo = __builtin_fmaf(g, -1.44269504f, -hi) + g * -1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(hi), t = __builtin_fmaf(e, fminf(lo, 1.f) * 0.69314718f, e);
    return __builtin_amdgcn_rcpf(1.f + (hi > 126.f ? __builtin_inff() : t));
}
__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == CODEPS_GATE_LINEAR) return g;
    const float s = sigmoid(g);
    return act == CODEPS_GATE_SIGMOID ? s : g * s;
}
__device__ __forceinline__ void gate_both(float g, int act, float& val, float& slope) {
    if (act == CODEPS_GATE_LINEAR) { val = g; slope = 1.f; return; }
    const float s = sigmoid(g);
    if (act == CODEPS_GATE_SIGMOID) { val = s; slope = s * (1.f - s); }
    else { val = g * s; slope = s * (1.f + g * (1.f - s)); }
}

// ---- host side
constexpr int MAX_C = 8192, CUS = 256;
constexpr long long MAX_PITCH = (1 << 24) - 1;                 // 64 rows are within 32-bit byte offsets

// lanes per row and channels per lane: in one wave while 8 channels per lane do (16-byte loads, no barrier), then a block with 8 channels per thread
// (16 of them spill in the backward pass)
struct Shape { bool block, tail; int nch, lpr_log2, threads, rpb; };
inline Shape shape_of(const codeps_channel_norm_desc* d) {
    const int V = d->x_type == CODEPS_F32 ? 4 : 8, C = d->channels;
    Shape s{false, C % V != 0, 1, 0, WAVE_THREADS, 0};
    if (C <= 64 * 8) {
        s.nch = V == 4 && C > 64 * 4 ? 2 : 1;
        while ((V * s.nch << s.lpr_log2) < C) ++s.lpr_log2;
        s.rpb = WAVE_THREADS >> s.lpr_log2;
        return s;
    }
    s.block = true;
    s.rpb = 1;
    s.nch = 8 / V;
    s.threads = cdiv(cdiv(C, 8), 64) * 64;
    return s;
}
// Blocks work on rows of one item (the rows that share an ITEM gate; all rows otherwise): block (item, slice) takes every slices-th group of rows, so that the
// chip walks through memory in step (contiguous ranges per block: norm alone, 262144 x 256 bf16, backward kernel 98 instead of 77 us).  Blocks loop over items.
inline bool shared_lines(const codeps_channel_norm_desc* d) { return d->channels * (d->x_type == CODEPS_F32 ? 4 : 2) % 128 != 0; }
struct Plan { Shape s; int items, rpi, slices, blocks; };
inline Plan plan_of(const codeps_channel_norm_desc* d, int want, int resident) {
    Plan p;
    p.s = shape_of(d);
    const bool per_item = d->gate_mode == CODEPS_GATE_ITEM;
    p.rpi = per_item ? d->rows_per_item : (int)d->rows;
    p.items = per_item ? std::max(1, (int)(d->rows / d->rows_per_item)) : 1;
    const int most = (int)std::max<long long>(1, ((long long)p.rpi + p.s.rpb - 1) / p.s.rpb);
    p.slices = std::max(1, std::min(most, want / p.items));
    if (p.slices > 8 && shared_lines(d)) p.slices &= ~7;                       // (whole rounds over the XCDs: slice_of)
    p.blocks = std::min(p.items, std::max(1, resident / p.slices)) * p.slices;
    return p;
}

inline int check_desc(const codeps_channel_norm_desc* d, const char* who) {
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
    CODEPS_REQUIRE(d->gate_mode != CODEPS_GATE_ELEMENT || d->gate_type == d->x_type, CODEPS_ERR_ARG, "%s: an element-wise gate has x's type", who);
    const long long C = d->channels;
    CODEPS_REQUIRE(d->x_pitch >= C && (d->full == 0 || d->res_pitch >= C) && (d->gate_mode < CODEPS_GATE_ITEM || d->gate_pitch >= C), CODEPS_ERR_ARG,
                   "%s: a row pitch is smaller than the row", who);
    CODEPS_REQUIRE(d->x_pitch <= MAX_PITCH && d->res_pitch <= MAX_PITCH && d->gate_pitch <= MAX_PITCH && d->dy_pitch <= MAX_PITCH && d->dh_pitch <= MAX_PITCH,
                   CODEPS_ERR_ARG, "%s: a row pitch of 2^24 elements or more", who);
    CODEPS_REQUIRE(d->full || (d->kind != CODEPS_NORM_NONE && d->next_kind == CODEPS_NORM_NONE && d->gate_mode == CODEPS_GATE_NONE), CODEPS_ERR_ARG,
                   "%s: a norm on its own has a kind and neither gate nor next norm", who);
    return CODEPS_OK;
}

inline Args args_of(const codeps_channel_norm_desc* d, const Plan& p) {
    Args a{};
    a.rows = d->rows; a.C = d->channels; a.xp = d->x_pitch; a.rp = d->res_pitch; a.gp = d->gate_pitch; a.dyp = d->dy_pitch; a.dhp = d->dh_pitch;
    a.kind = d->kind; a.next = d->next_kind; a.act = d->gate_act;
    a.wt = d->weight_type; a.gt = d->gate_type; a.nt = d->next_weight_type;
    a.scale = d->scale; a.eps = d->eps; a.neps = d->next_eps; a.inv_c = (float)(1.0 / d->channels);
    a.shared_lines = shared_lines(d);
    a.lpr_log2 = p.s.lpr_log2; a.items = p.items; a.rpi = p.rpi; a.slices = p.slices;
    if (d->gate_mode == CODEPS_GATE_CHANNEL) a.gp = 0;                          // (the one item's row)
    return a;
}

template <typename TX> constexpr int pieces_of = sizeof(TX) == 4 ? 2 : 1;       // 16-byte pieces that are 8 channels
template <int N> using num = std::integral_constant<int, N>;
// f(x type, residual type, pieces per lane, block, tail, full, gate) for every combination that shape_of can ask for
template <typename F> void dispatch(const codeps_channel_norm_desc* d, const Shape& s, F&& f) {
    const auto gates = [&](auto tx, auto tr, auto nch, auto block, auto tail) {
        if (!d->full) {
            if constexpr (std::is_same<decltype(tx), decltype(tr)>::value) f(tx, tr, nch, block, tail, std::false_type{}, num<GATE_NONE>{});
        } else if (d->gate_mode == CODEPS_GATE_NONE) f(tx, tr, nch, block, tail, std::true_type{}, num<GATE_NONE>{});
        else if (d->gate_mode == CODEPS_GATE_ELEMENT) f(tx, tr, nch, block, tail, std::true_type{}, num<GATE_ROWS>{});
        else f(tx, tr, nch, block, tail, std::true_type{}, num<GATE_HELD>{});
    };
    const auto tails = [&](auto tx, auto tr, auto nch, auto block) {
        if (s.tail) gates(tx, tr, nch, block, std::true_type{});
        else gates(tx, tr, nch, block, std::false_type{});
    };
    const auto pieces = [&](auto tx, auto tr) {
        constexpr int P = pieces_of<decltype(tx)>;
        if (s.block) tails(tx, tr, num<P>{}, std::true_type{});
        else if (s.nch == P) tails(tx, tr, num<P>{}, std::false_type{});
        else if constexpr (P > 1) tails(tx, tr, num<1>{}, std::false_type{});
    };
    const bool wide = d->res_type == CODEPS_F32 && d->full;
    if (d->x_type == CODEPS_F32) pieces(float{}, float{});
    else if (d->x_type == CODEPS_BF16) { if (wide) pieces(bf16{}, float{}); else pieces(bf16{}, bf16{}); }
    else { if (wide) pieces(f16{}, float{}); else pieces(f16{}, f16{}); }
}

}  // namespace
