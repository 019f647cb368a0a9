// Backward pass of the channel norms (formulas and row layout: channel_norm.h).  With u = n(x), u' = n'(y) and
// n^T(t) = rho (t - [mean t] - u mean(t u))   ([..]: layer only):
//   D = dy + n'^T(dh w');  dr = D;  dA = alpha act(g) D;  dg = alpha a D act'(g);  dx = n^T(dA w)
//   dw = sum_rows dA u;  db = sum_rows dA;  dw' = sum_rows dh u';  db' = sum_rows dh
// y is formed again from x, r and g instead of being read: the same bytes, and the sums see y before it was rounded to its type.
//
// Column sums (dw, db, dg, dw', db') live in registers across the rows of a block, go to one slab per block and are added in a fixed order by a second
// launch: no atomics, bitwise reproducible.
#include "channel_norm.h"

namespace {

// Column sums of one kind over the rows this block has seen -> dst[C].  Several rows per block: the row groups meet in LDS, in a fixed order.
template <int V, int NCH, bool BLOCK>
__device__ __forceinline__ void put_columns(const float* acc, float* lds, float* dst, const int* c0, int C, const Place& at_) {
    if constexpr (BLOCK) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) store_piece<V, true>(dst, 0, c0[j], C, acc + j * V);
    } else {
        const int width = at_.lpr * V * NCH, group = (int)threadIdx.x / at_.lpr;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) lds[group * width + c0[j] + e] = acc[j * V + e];
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += WAVE_THREADS) {
            float t = 0.f;
            for (int g = 0; g < at_.rpb; ++g) t += lds[g * width + c];
            dst[c] = t;
        }
    }
}

enum { SUMS_APART, SUMS_HERE, SUMS_WIDE };
// A row's tensors as they lie in memory.
template <int V, int NCH, typename TX, typename TR, bool ROWS> struct Row {
    Raw<V, TX> x[NCH], dh[NCH], g[ROWS ? NCH : 1];
    Raw<V, TR> r[NCH], dy[NCH];
    float4 st;                                       // mean and 1 / deviation of both norms
};

// Times below are forward and backward together, bf16 in and out, layer norms with weight and bias, "next": with the next block's norm.
//
// Rows of more than 4096 channels take blocks of more than 512 threads, which have 128 registers each.  SUMS_WIDE: the column sums fit there (norm alone; 16-bit
// block ends without a gate: 4096 x 5000, next, 175 us, apart 204).  SUMS_APART: channel_norm_columns_kernel forms them from the row's two sums of n'^T.  In place
// they spill 8 - 276 bytes (4096 x 5000, next: around an fp32 residual 228 -> 250 us, a gate per element 250 -> 273, per channel 272 -> 392); fp32 rows
// without a gate would bear it (4096 x 8192, next, 442 -> 416), but no kernel here uses scratch.
//
// Loads of a row are issued together, before anything is widened.  AHEAD: those of the next row as well, before the current one's arithmetic: for gates held over
// 16-bit rows, where the sums' registers allow two waves per SIMD either way, and for a norm alone in wide rows, where one block fills a CU (4096 x 8192
// 117 -> 102 us).  Held gates: 8192 x 4096, channel gate, next, 233 -> 214 us; 32768 x 2048, channel gate, next, 352 -> 333, without next 218 -> 190;
// 20485 x 768 around an fp32 residual, item gate, next, 117 -> 114; but 32768 x 2048 around fp32, channel gate, next, 392 -> 413.  (Three waves per SIMD without
// it spill; 32768 x 2048, channel gate, next, took 316 us that way.)  Elsewhere it costs a wave or scratch (gate per element, next, 32768 x 1024 203 -> 239;
// 4096 x 5000, next, 175 -> 235) or gains nothing (65536 x 1024, next, 300 -> 303; fp32 rows 273 -> 274).
template <typename TX, bool BLOCK, bool FULL, int GATE, int SUMS> struct Form {
    static constexpr bool held = BLOCK && SUMS == SUMS_HERE && GATE == GATE_HELD;
    static constexpr bool ahead = (held && sizeof(TX) == 2) || (SUMS == SUMS_WIDE && !FULL);
    static constexpr int threads = SUMS != SUMS_HERE ? 1024 : BLOCK ? 512 : WAVE_THREADS;
};
constexpr bool sums_fit(bool full, int gate, bool all_16_bit) { return !full || (gate == GATE_NONE && all_16_bit); }
template <typename TX, typename TR, int NCH, bool BLOCK, bool TAIL, bool FULL, int GATE, int SUMS>
__global__ __launch_bounds__((Form<TX, BLOCK, FULL, GATE, SUMS>::threads)) void channel_norm_bwd_kernel(Args a) {
    constexpr int V = sizeof(TX) == 4 ? 4 : 8, E = V * NCH;
    constexpr bool HELD = FULL && GATE == GATE_HELD, ROWS = FULL && GATE == GATE_ROWS, AHEAD = Form<TX, BLOCK, FULL, GATE, SUMS>::ahead;
    __shared__ float red[2][32];
    __shared__ float lds[BLOCK ? 1 : WAVE_THREADS * E];
    int turn = 0;
    const int lpr_log2 = a.lpr_log2, C = a.C;
    const Place at_ = place_of<BLOCK>(lpr_log2);
    const int lane = at_.lane, sub = at_.sub;
    // this lane's row behind the wave's first, in elements
    const int ox = sub * (int)a.xp, orr = sub * (int)a.rp, og = sub * (int)a.gp, ody = sub * (int)a.dyp, odh = sub * (int)a.dhp, oc = sub * C;
    int c0[NCH], left[NCH];
    unsigned keep[TAIL && FULL ? E : 1];
    float w[E], b[FULL ? E : 1], nw[FULL ? E : 1];
    float gv[HELD ? E : 1], gs[HELD ? E : 1];                                     // alpha act(g), alpha act'(g) of the item
    float aw[SUMS ? E : 1], ab[SUMS ? E : 1], anw[SUMS && FULL ? E : 1], anb[SUMS && FULL ? E : 1], ag[SUMS && HELD ? E : 1];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        c0[j] = (j * at_.lpr + lane) * V;
        left[j] = C - c0[j];
        if constexpr (TAIL && FULL) {
#pragma unroll
            for (int e = 0; e < V; ++e) keep[j * V + e] = e < left[j] ? ~0u : 0u;
        }
        load_vector<V>(a.w, a.wt, 0, c0[j], C, 1.f, w + j * V);
        if constexpr (FULL) {
            load_vector<V>(a.b, a.wt, 0, c0[j], C, 0.f, b + j * V);
            load_vector<V>(a.nw, a.nt, 0, c0[j], C, 1.f, nw + j * V);
        }
    }
    if constexpr (SUMS) {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            aw[k] = ab[k] = 0.f;
            if constexpr (FULL) anw[k] = anb[k] = 0.f;
        }
    }
    const int S = a.slices, slice = slice_of(blockIdx.x, S, a.shared_lines);
    const bool has_r = a.r != nullptr;
    for (unsigned item = blockIdx.x / (unsigned)S; item < (unsigned)a.items; item += gridDim.x / (unsigned)S) {
        if constexpr (HELD) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                load_vector<V>(a.gate, a.gt, (size_t)item * a.gp, c0[j], C, 0.f, gv + j * V);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int k = j * V + e;
                    float val, slope;
                    gate_both(gv[k], a.act, val, slope);
                    gv[k] = a.scale * val;
                    gs[k] = a.scale * slope;
                    if constexpr (SUMS) ag[k] = 0.f;
                }
            }
        }
        const auto fetch = [&](size_t row) {                                   // the wave's first row
            Row<V, NCH, TX, TR, ROWS> q;
            const TX* px = (const TX*)a.x + row * a.xp;
#pragma unroll
            for (int j = 0; j < NCH; ++j) q.x[j] = raw_piece<V, TAIL>(px, ox, c0[j], C);
            if constexpr (!FULL) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) q.dh[j] = raw_piece<V, TAIL>((const TX*)a.dh + row * a.dhp, odh, c0[j], C);
                const float2 st = *reinterpret_cast<const float2*>(a.stats_in + (row + sub) * 2);
                q.st = make_float4(st.x, st.y, 0.f, 1.f);
            } else {
                q.st = *reinterpret_cast<const float4*>(a.stats_in + (row + sub) * 4);
                if constexpr (ROWS) {
#pragma unroll
                    for (int j = 0; j < NCH; ++j) q.g[j] = raw_piece<V, TAIL>((const TX*)a.gate + row * a.gp, og, c0[j], C);
                }
                if (a.next) {
                    // without a residual x's row stands in for it (then both have one type) and counts as zeros: no branch around the load
                    const TR* pr = has_r ? (const TR*)a.r + row * a.rp : (const TR*)(const void*)px;
#pragma unroll
                    for (int j = 0; j < NCH; ++j) {
                        q.dh[j] = raw_piece<V, TAIL>((const TX*)a.dh + row * a.dhp, odh, c0[j], C);
                        q.r[j] = raw_piece<V, TAIL>(pr, has_r ? orr : ox, c0[j], C);
                    }
                }
                if (a.dy) {
#pragma unroll
                    for (int j = 0; j < NCH; ++j) q.dy[j] = raw_piece<V, TAIL>((const TR*)a.dy + row * a.dyp, ody, c0[j], C);
                }
            }
            return q;
        };
        const long long i0 = (long long)slice * at_.rpb + at_.first, step = (long long)S * at_.rpb;
        Row<V, NCH, TX, TR, ROWS> now, ahead;
        if constexpr (AHEAD) {
            if (i0 + sub < a.rpi) ahead = fetch((size_t)item * a.rpi + i0);
        }
        for (long long i = i0; i + sub < a.rpi; i += step) {
            const size_t row = (size_t)item * a.rpi + i;
            if constexpr (AHEAD) {
                now = ahead;
                if (i + step + sub < a.rpi) ahead = fetch(row + step);
            } else {
                now = fetch(row);
            }
            float u[E], d[E];                                                  // u = n(x), d: the gradient that runs backward
#pragma unroll
            for (int j = 0; j < NCH; ++j) widen_piece<V, TAIL>(now.x[j], c0[j], C, u + j * V);
            const float mu = now.st.x, rho = now.st.y, nmu = now.st.z, nrho = now.st.w;
            if constexpr (!FULL) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) widen_piece<V, TAIL>(now.dh[j], c0[j], C, d + j * V);
#pragma unroll
                for (int k = 0; k < E; ++k) u[k] = (u[k] - mu) * rho;
            } else {
                float t[E], y[E], al[ROWS ? E : 1], as[ROWS ? E : 1];          // dh; r, then u'; alpha act(g), alpha act'(g) of the row
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    if constexpr (ROWS) widen_piece<V, TAIL>(now.g[j], c0[j], C, al + j * V);
                    if (a.next) {
                        widen_piece<V, TAIL>(now.dh[j], c0[j], C, t + j * V);
                        widen_piece<V, TAIL>(now.r[j], c0[j], C, y + j * V);
                    }
                    if (a.dy) {
                        widen_piece<V, TAIL>(now.dy[j], c0[j], C, d + j * V);
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) d[j * V + e] = 0.f;
                    }
                }
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    u[k] = (u[k] - mu) * rho;
                    if constexpr (ROWS) {
                        float val, slope;
                        gate_both(al[k], a.act, val, slope);
                        al[k] = a.scale * val;
                        as[k] = a.scale * slope;
                    }
                }
                const auto val = [&](int k) { if constexpr (ROWS) return al[k]; else if constexpr (HELD) return gv[k]; else return a.scale; };
                const auto slope = [&](int k) { if constexpr (ROWS) return as[k]; else return gs[k]; };
                if (a.next) {                                                  // d += n'^T(dh w')
                    float s[2] = {0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < NCH; ++j) {
                        float q[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const int k = j * V + e;
                            y[k] = ((has_r ? y[k] : 0.f) + val(k) * (u[k] * w[k] + b[k]) - nmu) * nrho;
                            q[e] = t[k] * y[k];
                            if constexpr (SUMS) { anw[k] += q[e]; anb[k] += t[k]; }
                            q[e] *= nw[k];
                            t[k] *= nw[k];
                        }
                        s[0] += piece_sum<V, TAIL, true>(t + j * V, left[j], keep);        // (dh is 0 behind the row's end)
                        s[1] += piece_sum<V, TAIL, true>(q, left[j], keep);
                    }
                    row_sums<BLOCK>(s, lpr_log2, red, turn);
                    s[0] = a.next == CODEPS_NORM_LAYER ? s[0] * a.inv_c : 0.f;
                    s[1] *= a.inv_c;
                    if constexpr (!SUMS) {
                        if (lane == 0) *reinterpret_cast<float2*>(a.row_sums + (row + sub) * 2) = make_float2(s[0], s[1]);
                    }
#pragma unroll
                    for (int k = 0; k < E; ++k) d[k] += nrho * (t[k] - s[0] - y[k] * s[1]);
                }
#pragma unroll
                for (int j = 0; j < NCH; ++j) {
                    if (a.dr) store_piece<V, TAIL>((TR*)a.dr + row * C, oc, c0[j], C, d + j * V);
                    if constexpr (GATE != GATE_NONE && (SUMS || ROWS)) {
                        float q[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const int k = j * V + e;
                            q[e] = slope(k) * (u[k] * w[k] + b[k]) * d[k];
                            if constexpr (HELD) ag[k] += q[e];
                        }
                        if constexpr (ROWS) {
                            if (a.dgate) store_piece<V, TAIL>((TX*)a.dgate + row * C, oc, c0[j], C, q);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) d[j * V + e] *= val(j * V + e);
                }
            }
            // d = the gradient of a: its column sums, then through n
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                float q[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int k = j * V + e;
                    q[e] = d[k] * u[k];
                    if constexpr (SUMS) { aw[k] += q[e]; ab[k] += d[k]; }
                    q[e] *= w[k];
                    d[k] *= w[k];
                }
                s[0] += piece_sum<V, TAIL, !FULL>(d + j * V, left[j], keep + (TAIL && FULL ? j * V : 0));
                s[1] += piece_sum<V, TAIL, !FULL>(q, left[j], keep + (TAIL && FULL ? j * V : 0));
            }
            if (a.kind) {
                row_sums<BLOCK>(s, lpr_log2, red, turn);
                s[0] = a.kind == CODEPS_NORM_LAYER ? s[0] * a.inv_c : 0.f;
                s[1] *= a.inv_c;
#pragma unroll
                for (int k = 0; k < E; ++k) d[k] = rho * (d[k] - s[0] - u[k] * s[1]);
            }
            if (a.dx) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) store_piece<V, TAIL>((TX*)a.dx + row * C, oc, c0[j], C, d + j * V);
            }
        }
        if constexpr (HELD && SUMS) {
            if (a.cols & COL_G) put_columns<V, NCH, BLOCK>(ag, lds, a.gate_slab + ((size_t)item * S + slice) * C, c0, C, at_);
        }
    }
    if constexpr (SUMS) {
        float* const my = a.slab + (size_t)blockIdx.x * 4 * C;                   // [dw | db | dw' | db'] of this block
        if (a.cols & COL_W) put_columns<V, NCH, BLOCK>(aw, lds, my, c0, C, at_);
        if (a.cols & COL_B) put_columns<V, NCH, BLOCK>(ab, lds, my + C, c0, C, at_);
        if constexpr (FULL) {
            if (a.cols & COL_NW) put_columns<V, NCH, BLOCK>(anw, lds, my + 2 * C, c0, C, at_);
            if (a.cols & COL_NB) put_columns<V, NCH, BLOCK>(anb, lds, my + 3 * C, c0, C, at_);
        }
    }
}

// The column sums alone, for SUMS_APART: a thread owns V channels of every row of its slice and forms D from the row's statistics and
// sums.  Reads the row's tensors a second time (from the L2s and the memory-side cache where few rows lie between).
template <typename TX, typename TR, bool TAIL, int GATE>
__global__ __launch_bounds__(256) void channel_norm_columns_kernel(Args a) {
    constexpr int V = sizeof(TX) == 4 ? 4 : 8;
    constexpr bool HELD = GATE == GATE_HELD, ROWS = GATE == GATE_ROWS;
    const int C = a.C, S = a.slices, slice = slice_of(blockIdx.x, S, a.shared_lines), c0 = (int)(blockIdx.y * 256 + threadIdx.x) * V;
    float w[V], b[V], nw[V], gv[V], gs[V], aw[V] = {}, ab[V] = {}, anw[V] = {}, anb[V] = {}, ag[V];
    load_vector<V>(a.w, a.wt, 0, c0, C, 1.f, w);
    load_vector<V>(a.b, a.wt, 0, c0, C, 0.f, b);
    load_vector<V>(a.nw, a.nt, 0, c0, C, 1.f, nw);
    const bool has_r = a.r != nullptr;
    for (unsigned item = blockIdx.x / (unsigned)S; item < (unsigned)a.items; item += gridDim.x / (unsigned)S) {
        if constexpr (HELD) {
            load_vector<V>(a.gate, a.gt, (size_t)item * a.gp, c0, C, 0.f, gv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                gate_both(gv[e], a.act, gv[e], gs[e]);
                gv[e] *= a.scale;
                gs[e] *= a.scale;
                ag[e] = 0.f;
            }
        }
        for (long long i = slice; i < a.rpi; i += S) {
            const size_t row = (size_t)item * a.rpi + i;
            const TX* px = (const TX*)a.x + row * a.xp;
            float u[V], d[V];
            load_piece<V, TAIL>(px, 0, c0, C, u);
            const float4 st = *reinterpret_cast<const float4*>(a.stats_in + row * 4);
            float t[V], y[V];
            if constexpr (ROWS) load_piece<V, TAIL>((const TX*)a.gate + row * a.gp, 0, c0, C, gv);
            if (a.next) {
                load_piece<V, TAIL>((const TX*)a.dh + row * a.dhp, 0, c0, C, t);
                load_piece<V, TAIL>(has_r ? (const TR*)a.r + row * a.rp : (const TR*)(const void*)px, 0, c0, C, y);
            }
            if (a.dy) load_piece<V, TAIL>((const TR*)a.dy + row * a.dyp, 0, c0, C, d);
            else {
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = 0.f;
            }
            const float2 s = a.next ? *reinterpret_cast<const float2*>(a.row_sums + row * 2) : make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                u[e] = (u[e] - st.x) * st.y;
                const float an = u[e] * w[e] + b[e];
                float val = a.scale, slope = 0.f;
                if constexpr (ROWS) { gate_both(gv[e], a.act, val, slope); val *= a.scale; }
                if constexpr (HELD) { val = gv[e]; slope = gs[e]; }
                if (a.next) {
                    y[e] = ((has_r ? y[e] : 0.f) + val * an - st.z) * st.w;
                    anw[e] += t[e] * y[e];
                    anb[e] += t[e];
                    d[e] += st.w * (t[e] * nw[e] - s.x - y[e] * s.y);
                }
                if constexpr (HELD) ag[e] += slope * an * d[e];
                d[e] *= val;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) { aw[e] += d[e] * u[e]; ab[e] += d[e]; }
        }
        if constexpr (HELD) {
            if (a.cols & COL_G) store_piece<V, true>(a.gate_slab + ((size_t)item * S + slice) * C, 0, c0, C, ag);
        }
    }
    float* const my = a.slab + (size_t)blockIdx.x * 4 * C;
    if (a.cols & COL_W) store_piece<V, true>(my, 0, c0, C, aw);
    if (a.cols & COL_B) store_piece<V, true>(my + C, 0, c0, C, ab);
    if (a.cols & COL_NW) store_piece<V, true>(my + 2 * C, 0, c0, C, anw);
    if (a.cols & COL_NB) store_piece<V, true>(my + 3 * C, 0, c0, C, anb);
}

// out[g][c] (+)= sum over n of part[(g * n + i) * pitch + c], in a fixed order: 16 columns x 64 strided streams per block
struct Finish {
    const float* part[5];
    void* out[5];
    int type[5], groups[5], n[5], pitch[5], accumulate[5];
    int C;
};
constexpr int FINISH_STREAMS = 64;
__global__ __launch_bounds__(16 * FINISH_STREAMS) void channel_norm_finish_kernel(Finish f) {
    __shared__ float red[FINISH_STREAMS][17];
    const int k = blockIdx.z, g = blockIdx.y, col = threadIdx.x & 15, c = blockIdx.x * 16 + col, s = threadIdx.x >> 4;
    if (g >= f.groups[k]) return;
    const int n = f.n[k];
    const size_t pitch = f.pitch[k];
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < f.C) {
        const float* p = f.part[k] + (size_t)g * n * pitch + c;
        int i = s;
        for (; i + 3 * FINISH_STREAMS < n; i += 4 * FINISH_STREAMS)
#pragma unroll
            for (int q = 0; q < 4; ++q) t[q] += p[(size_t)(i + q * FINISH_STREAMS) * pitch];
        for (; i < n; i += FINISH_STREAMS) t[0] += p[(size_t)i * pitch];
    }
    red[s][col] = (t[0] + t[1]) + (t[2] + t[3]);
    __syncthreads();
    if (s < 4) {                                                       // one wave: 16 columns x 4 quarters of the streams
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < FINISH_STREAMS / 4; ++i) v += red[s * (FINISH_STREAMS / 4) + i][col];
        v += __shfl_xor(v, 16, 64);
        v += __shfl_xor(v, 32, 64);
        if (s == 0 && c < f.C) {
            const size_t o = (size_t)g * f.C + c;
            if (f.type[k] == CODEPS_F32) { float* p = (float*)f.out[k] + o; *p = f.accumulate[k] ? *p + v : v; }
            else if (f.type[k] == CODEPS_BF16) narrow(v, ((bf16*)f.out[k])[o]);
            else narrow(v, ((f16*)f.out[k])[o]);
        }
    }
}

// Blocks: as many as are resident at once, by the registers of the kernel that runs -- more leave a tail of late blocks, fewer leave lanes idle.  Forward and
// backward together at 8 / 12 / 16 waves per CU, us: norm alone, 65536 x 768 bf16 147 / 127 / 119, 16384 x 2048 fp32 130 / 132 / 138; block end in one 16-bit
// type, next norm, no gate, 65536 x 1024 327 / 300 / 308, gate per element, 32768 x 1024 217 / 202 / 224, channel gate, 65536 x 1024 330 / 380 / 396; 16-bit blocks
// around an fp32 residual, next norm, 32768 x 2048, channel gate 416 / 422 / 422, 20485 x 768, item gate 114 / 127 / 133; all fp32, next norm, 20485 x 768, item gate
// 152 / 174 / 185, 32768 x 1024, channel gate 272 / 294 / 319.
// A block takes at least 8 rows per row group where there are that many: its column sums' slab is a cost of its own.
Plan bwd_plan(const codeps_channel_norm_desc* d) {
    const Shape s = shape_of(d);
    const bool half = d->x_type != CODEPS_F32, held = d->gate_mode == CODEPS_GATE_CHANNEL || d->gate_mode == CODEPS_GATE_ITEM;
    const int waves = !half || d->res_type != d->x_type ? 8 : !d->full ? 16 : held ? 8 : 12;
    const int resident = CUS * std::max(1, waves / (s.threads / 64));
    return plan_of(d, (int)std::max<long long>(CUS, std::min<long long>(resident, d->rows / (8LL * s.rpb))), resident);
}
size_t slab_floats(const codeps_channel_norm_desc* d, const Plan& p) { return (size_t)p.blocks * 4 * d->channels; }
bool columns_apart(const codeps_channel_norm_desc* d, const Shape& s) {
    const int gate = d->gate_mode == CODEPS_GATE_NONE ? GATE_NONE : d->gate_mode == CODEPS_GATE_ELEMENT ? GATE_ROWS : GATE_HELD;
    return s.threads > 512 && !sums_fit(d->full, gate, d->x_type != CODEPS_F32 && d->res_type == d->x_type);
}
size_t row_floats(const codeps_channel_norm_desc* d, const Plan& p) { return columns_apart(d, p.s) && d->next_kind ? (size_t)d->rows * 2 : 0; }
size_t gate_floats(const codeps_channel_norm_desc* d, const Plan& p) {
    return d->gate_mode == CODEPS_GATE_CHANNEL || d->gate_mode == CODEPS_GATE_ITEM ? (size_t)p.items * p.slices * d->channels : 0;
}

}  // namespace

extern "C" size_t codeps_channel_norm_bwd_workspace_bytes(const codeps_channel_norm_desc* d) {
    if (check_desc(d, "channel_norm_bwd_workspace_bytes") != CODEPS_OK) return 0;
    const Plan p = bwd_plan(d);
    return std::max<size_t>(256, (row_floats(d, p) + slab_floats(d, p) + gate_floats(d, p)) * sizeof(float));
}

extern "C" int codeps_channel_norm_bwd(const codeps_channel_norm_desc* d, const void* x, const void* residual, const void* gate, const void* weight,
                                       const void* bias, const void* next_weight, const float* stats, const void* dy, const void* dh, void* dx,
                                       void* dresidual, void* dgate, void* dweight, void* dbias, void* dnext_weight, void* dnext_bias, int accumulate,
                                       void* workspace, size_t workspace_bytes, codeps_stream_t stream) {
    const int rc = check_desc(d, "channel_norm_bwd");
    if (rc != CODEPS_OK) return rc;
    const Plan p = bwd_plan(d);
    CODEPS_REQUIRE(workspace && workspace_bytes >= codeps_channel_norm_bwd_workspace_bytes(d), CODEPS_ERR_WORKSPACE,
                   "channel_norm_bwd: %zu bytes of workspace, %zu are needed", workspace_bytes, codeps_channel_norm_bwd_workspace_bytes(d));
    CODEPS_REQUIRE((accumulate & ~(CODEPS_ACC_WEIGHT | CODEPS_ACC_BIAS | CODEPS_ACC_NEXT_WEIGHT | CODEPS_ACC_NEXT_BIAS)) == 0, CODEPS_ERR_ARG,
                   "channel_norm_bwd: unknown accumulate bits %d", accumulate);
    CODEPS_REQUIRE((!(accumulate & (CODEPS_ACC_WEIGHT | CODEPS_ACC_BIAS)) || d->weight_type == CODEPS_F32) &&
                   (!(accumulate & (CODEPS_ACC_NEXT_WEIGHT | CODEPS_ACC_NEXT_BIAS)) || d->next_weight_type == CODEPS_F32), CODEPS_ERR_ARG,
                   "channel_norm_bwd: gradients are accumulated in fp32 only");
    const void* const outs[] = {dx, dresidual, dgate, dweight, dbias, dnext_weight, dnext_bias};
    for (int i = 0; i < 7; ++i)
        for (int j = 0; j < i; ++j)
            CODEPS_REQUIRE(!outs[i] || outs[i] != outs[j], CODEPS_ERR_ARG, "channel_norm_bwd: two gradients have one address");
    if (d->rows > 0) {
        CODEPS_REQUIRE(x && stats && (!d->gate_mode || gate) && (d->full ? (dy || d->next_kind) : dh != nullptr) && (!d->next_kind || dh), CODEPS_ERR_ARG,
                       "channel_norm_bwd: null pointer");
        CODEPS_REQUIRE((!dy || d->dy_pitch >= d->channels) && (!dh || d->dh_pitch >= d->channels), CODEPS_ERR_ARG,
                       "channel_norm_bwd: a row pitch is smaller than the row");
        CODEPS_REQUIRE(!d->next_kind || residual || d->res_type == d->x_type, CODEPS_ERR_ARG, "channel_norm_bwd: without a residual y has x's type");
    }
    hipStream_t st = (hipStream_t)stream;
    float *slab = (float*)workspace + row_floats(d, p), *gate_slab = slab + slab_floats(d, p);          // [rows][2] first: 8-byte aligned
    const int C = d->channels;
    const bool columns = d->gate_mode == CODEPS_GATE_CHANNEL || d->gate_mode == CODEPS_GATE_ITEM;
    if (d->rows > 0) {
        Args a = args_of(d, p);
        a.x = x; a.r = residual; a.gate = gate; a.w = weight; a.b = bias; a.nw = next_weight; a.stats_in = stats; a.dy = dy; a.dh = dh;
        a.dx = dx; a.dr = dresidual; a.dgate = dgate; a.slab = slab; a.gate_slab = gate_slab; a.row_sums = (float*)workspace;
        a.cols = (dweight ? COL_W : 0) | (dbias ? COL_B : 0) | (dnext_weight && d->next_kind ? COL_NW : 0) | (dnext_bias && d->next_kind ? COL_NB : 0) |
                 (dgate && columns ? COL_G : 0);
        dispatch(d, p.s, [&](auto tx, auto tr, auto nch, auto block, auto tail, auto full, auto gmode) {
            using TX = decltype(tx);
            using TR = decltype(tr);
            constexpr bool BLOCK = decltype(block)::value, TAIL = decltype(tail)::value, FULL = decltype(full)::value;
            constexpr int NCH = decltype(nch)::value, GATE = decltype(gmode)::value;
            if (BLOCK && p.s.threads > 512) {
                if constexpr (BLOCK) {
                    constexpr int SUMS = sums_fit(FULL, GATE, sizeof(TX) == 2 && std::is_same<TX, TR>::value) ? SUMS_WIDE : SUMS_APART;
                    hipLaunchKernelGGL((channel_norm_bwd_kernel<TX, TR, NCH, true, TAIL, FULL, GATE, SUMS>), dim3(p.blocks), dim3(p.s.threads), 0, st, a);
                    if constexpr (SUMS == SUMS_APART) {
                        if (a.cols)
                            hipLaunchKernelGGL((channel_norm_columns_kernel<TX, TR, TAIL, GATE>),
                                               dim3(p.blocks, cdiv(d->channels, 256 * (sizeof(TX) == 4 ? 4 : 8))), dim3(256), 0, st, a);
                    }
                }
            } else {
                hipLaunchKernelGGL((channel_norm_bwd_kernel<TX, TR, NCH, BLOCK, TAIL, FULL, GATE, SUMS_HERE>), dim3(p.blocks), dim3(p.s.threads), 0, st, a);
            }
        });
        CODEPS_CHECK_LAUNCH("channel_norm_bwd_kernel");
    }
    Finish f{};
    int k = 0, groups = 1;
    f.C = C;
    const auto add = [&](const float* part, void* out, int type, int g, int n, int pitch, int acc) {
        if (!out) return;
        f.part[k] = part; f.out[k] = out; f.type[k] = type; f.groups[k] = g; f.n[k] = d->rows > 0 ? n : 0; f.pitch[k] = pitch; f.accumulate[k] = acc;
        groups = std::max(groups, g);
        ++k;
    };
    add(slab, dweight, d->weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_WEIGHT);
    add(slab + C, dbias, d->weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_BIAS);
    if (d->next_kind) {
        add(slab + 2 * C, dnext_weight, d->next_weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_NEXT_WEIGHT);
        add(slab + 3 * C, dnext_bias, d->next_weight_type, 1, p.blocks, 4 * C, accumulate & CODEPS_ACC_NEXT_BIAS);
    }
    if (columns && (d->rows > 0 || d->gate_mode == CODEPS_GATE_CHANNEL)) add(gate_slab, dgate, d->gate_type, p.items, p.slices, C, 0);
    // (items behind the 65535th have their own launch: a grid's second dimension ends there)
    for (long long g0 = 0; k > 0 && g0 < groups; g0 += 65535) {
        Finish part = f;
        for (int i = 0; i < k; ++i) {
            const int skip = (int)std::min<long long>(g0, f.groups[i]);
            part.groups[i] = std::min(f.groups[i] - skip, 65535);
            part.part[i] = f.part[i] + (size_t)skip * f.n[i] * f.pitch[i];
            part.out[i] = (char*)f.out[i] + (size_t)skip * C * (f.type[i] == CODEPS_F32 ? 4 : 2);
        }
        hipLaunchKernelGGL(channel_norm_finish_kernel, dim3(cdiv(C, 16), (unsigned)std::min<long long>(groups - g0, 65535), k), dim3(16 * FINISH_STREAMS), 0, st, part);
        CODEPS_CHECK_LAUNCH("channel_norm_finish_kernel");
    }
    return CODEPS_OK;
}
