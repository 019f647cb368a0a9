// Forward pass of the channel norms (formulas and row layout: channel_norm.h).
#include "channel_norm.h"

namespace {

// mean and 1 / deviation of the row that v holds.  The deviations are summed around the mean, in a second sweep over registers: the difference of two
// large sums would lose them where the mean is large.
template <int V, int NCH, bool BLOCK, bool TAIL, bool ZEROS>
__device__ __forceinline__ void row_stats(const float* v, const int* left, const unsigned* keep, int kind, float eps, float inv_c, int lpr_log2, float (*red)[32], int& turn,
                                          float& mu, float& rho) {
    float s[1];
    mu = 0.f;
    if (kind == CODEPS_NORM_LAYER) {
        s[0] = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) s[0] += piece_sum<V, TAIL, ZEROS>(v + j * V, left[j], keep + (TAIL ? j * V : 0));
        row_sums<BLOCK>(s, lpr_log2, red, turn);
        mu = s[0] * inv_c;
    }
    s[0] = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        float q[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { const float t = v[j * V + e] - mu; q[e] = t * t; }
        s[0] += piece_sum<V, TAIL, false>(q, left[j], keep + (TAIL ? j * V : 0));
    }
    row_sums<BLOCK>(s, lpr_log2, red, turn);
    rho = 1.f / sqrtf(s[0] * inv_c + eps);
}

template <typename TX, typename TR, int NCH, bool BLOCK, bool TAIL, bool FULL, int GATE>
__global__ __launch_bounds__(BLOCK ? 1024 : WAVE_THREADS) void channel_norm_fwd_kernel(Args a) {
    constexpr int V = sizeof(TX) == 4 ? 4 : 8, E = V * NCH;
    __shared__ float red[2][32];
    int turn = 0;
    const int lpr_log2 = a.lpr_log2, C = a.C;
    const Place at_ = place_of<BLOCK>(lpr_log2);
    const int lpr = at_.lpr, lane = at_.lane, sub = at_.sub;
    const int ox = sub * (int)a.xp, orr = sub * (int)a.rp, og = sub * (int)a.gp, oc = sub * C;        // this lane's row behind the wave's first, in elements
    int c0[NCH], left[NCH];
    unsigned keep[TAIL ? E : 1];
    float w[E], b[E], nw[FULL ? E : 1], nb[FULL ? E : 1], g[FULL && GATE != GATE_NONE ? E : 1];     // the vectors stay in registers over the rows of a block
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        c0[j] = (j * lpr + lane) * V;
        left[j] = C - c0[j];
        if constexpr (TAIL) {
#pragma unroll
            for (int e = 0; e < V; ++e) keep[j * V + e] = e < left[j] ? ~0u : 0u;
        }
        load_vector<V>(a.w, a.wt, 0, c0[j], C, 1.f, w + j * V);
        load_vector<V>(a.b, a.wt, 0, c0[j], C, 0.f, b + j * V);
        if constexpr (FULL) {
            load_vector<V>(a.nw, a.nt, 0, c0[j], C, 1.f, nw + j * V);
            load_vector<V>(a.nb, a.nt, 0, c0[j], C, 0.f, nb + j * V);
        }
    }
    const int S = a.slices, slice = slice_of(blockIdx.x, S, a.shared_lines);
    const bool has_r = a.r != nullptr;
    for (unsigned item = blockIdx.x / (unsigned)S; item < (unsigned)a.items; item += gridDim.x / (unsigned)S) {
        if constexpr (FULL && GATE == GATE_HELD) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                load_vector<V>(a.gate, a.gt, (size_t)item * a.gp, c0[j], C, 0.f, g + j * V);
#pragma unroll
                for (int e = 0; e < V; ++e) g[j * V + e] = a.scale * gate_value(g[j * V + e], a.act);
            }
        }
        for (long long i = (long long)slice * at_.rpb + at_.first; i + sub < a.rpi; i += (long long)S * at_.rpb) {
            const size_t row = (size_t)item * a.rpi + i;                       // the wave's first row
            const TX* px = (const TX*)a.x + row * a.xp;
            float v[E], rv[FULL ? E : 1];
#pragma unroll
            for (int j = 0; j < NCH; ++j) load_piece<V, TAIL>(px, ox, c0[j], C, v + j * V);
            if constexpr (FULL) {
                // without a residual x's row stands in for it (then both have one type) and counts as zeros: no branch around the load
                const TR* pr = has_r ? (const TR*)a.r + row * a.rp : (const TR*)(const void*)px;
#pragma unroll
                for (int j = 0; j < NCH; ++j) load_piece<V, TAIL>(pr, has_r ? orr : ox, c0[j], C, rv + j * V);
                if constexpr (GATE == GATE_ROWS) {
#pragma unroll
                    for (int j = 0; j < NCH; ++j) load_piece<V, TAIL>((const TX*)a.gate + row * a.gp, og, c0[j], C, g + j * V);
                }
            }
            float mu = 0.f, rho = 1.f, nmu = 0.f, nrho = 1.f;
            if (a.kind) row_stats<V, NCH, BLOCK, TAIL, true>(v, left, keep, a.kind, a.eps, a.inv_c, lpr_log2, red, turn, mu, rho);
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = (v[k] - mu) * rho * w[k] + b[k];
            if constexpr (!FULL) {
#pragma unroll
                for (int j = 0; j < NCH; ++j) store_piece<V, TAIL>((TX*)a.h + row * C, oc, c0[j], C, v + j * V);
                if (a.stats && lane == 0) *reinterpret_cast<float2*>(a.stats + (row + sub) * 2) = make_float2(mu, rho);
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float s = GATE == GATE_NONE ? a.scale : GATE == GATE_HELD ? g[GATE ? k : 0] : a.scale * gate_value(g[GATE ? k : 0], a.act);
                    v[k] = (has_r ? rv[k] : 0.f) + s * v[k];
                }
#pragma unroll
                for (int j = 0; j < NCH; ++j) store_piece<V, TAIL>((TR*)a.y + row * C, oc, c0[j], C, v + j * V);
                if (a.next) {
                    row_stats<V, NCH, BLOCK, TAIL, false>(v, left, keep, a.next, a.neps, a.inv_c, lpr_log2, red, turn, nmu, nrho);
#pragma unroll
                    for (int k = 0; k < E; ++k) v[k] = (v[k] - nmu) * nrho * nw[k] + nb[k];
#pragma unroll
                    for (int j = 0; j < NCH; ++j) store_piece<V, TAIL>((TX*)a.h + row * C, oc, c0[j], C, v + j * V);
                }
                if (a.stats && lane == 0) *reinterpret_cast<float4*>(a.stats + (row + sub) * 4) = make_float4(mu, rho, nmu, nrho);
            }
        }
    }
}

}  // namespace

extern "C" int codeps_channel_norm_fwd(const codeps_channel_norm_desc* d, const void* x, const void* residual, const void* gate, const void* weight,
                                       const void* bias, const void* next_weight, const void* next_bias, void* y, void* h, float* stats,
                                       codeps_stream_t stream) {
    const int rc = check_desc(d, "channel_norm_fwd");
    if (rc != CODEPS_OK) return rc;
    if (d->rows == 0) return CODEPS_OK;
    CODEPS_REQUIRE(x && (d->full ? y != nullptr : h != nullptr) && (!d->next_kind || h) && (!d->gate_mode || gate), CODEPS_ERR_ARG,
                   "channel_norm_fwd: null pointer");
    CODEPS_REQUIRE(!d->full || residual || d->res_type == d->x_type, CODEPS_ERR_ARG, "channel_norm_fwd: without a residual y has x's type");
    const Plan p = plan_of(d, 4096, 4096);
    Args a = args_of(d, p);
    a.x = x; a.r = residual; a.gate = gate; a.w = weight; a.b = bias; a.nw = next_weight; a.nb = next_bias; a.y = y; a.h = h; a.stats = stats;
    dispatch(d, p.s, [&](auto tx, auto tr, auto nch, auto block, auto tail, auto full, auto gmode) {
        hipLaunchKernelGGL((channel_norm_fwd_kernel<decltype(tx), decltype(tr), decltype(nch)::value, decltype(block)::value, decltype(tail)::value,
                                                    decltype(full)::value, decltype(gmode)::value>),
                           dim3(p.blocks), dim3(p.s.threads), 0, (hipStream_t)stream, a);
    });
    CODEPS_CHECK_LAUNCH("channel_norm_fwd_kernel");
    return CODEPS_OK;
}
