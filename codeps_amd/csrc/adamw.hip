// AdamW over many tensors at once and the global norm of their gradients.
//   g' = g s c,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,  p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
// A step is two launches (with clipping one more, for the norm): a small one that advances every tensor's count t and turns it into the tensor's factors
// (64 bits: 1 - b2^t of a young tensor loses its digits in 32), and the update itself.  Nothing of a step depends on host values but its scalars, so a
// captured step replays as the next one.  The update reads and writes every byte once: 28 bytes per element with 32-bit states, 16 with 8-bit ones (fp32
// gradients); it is bound by bandwidth: 99.6 M elements in 8 bits take 301 - 309 us (5.2 - 5.3 TB/s), 23.5 M in 32 bits with an average (36 bytes) 140 - 153 us
// (5.6 - 6.0 TB/s).
//
// Tensors are cut into chunks of 2048 elements, one block each; a table gives the tensor of a chunk.  The static part of a tensor (addresses, state
// offsets) lies in a device table, gradient addresses travel in the launch's arguments: they change from step to step.
//
// 8-bit states: a wave owns a block of 256 elements (4 per lane), finds its largest magnitude (integer maximum of the bit patterns: NaN and infinity
// win), takes the smallest power of two under which it fits, and rounds stochastically:
//   q = floor(t / quantum + rho / 65536),  rho = 16 random bits
// in integers: t 2^16 / quantum is below 2^21, its whole part plus rho is shifted by 16.  The fp32 value behind it is off by a unit at most, so the
// result can differ from the exact one only where the sum lies within two units of a multiple of 65536: there (about 8 elements in 100 000) the
// moments are formed again in 64 bits.  So are those of a whole block whose largest magnitude lies next to a border between two units (about two blocks
// in 100 000).  The root is held over the whole range of fp32, but its square is not: a block goes through 64 bits as a whole, its unit
// and the parameters' update included, where a square would overflow (roots of 2^62 or more) or lose bits that a code could see.  Those are squares below
// 2^-120 that are not exactly zero, in blocks whose largest root is below 2^-36, or beside an eps below 2^-50: elsewhere, what a subnormal square loses (2^-74
// of the root) is less than the 2^-16 quanta of the lowest codes (2^-70) and a rounding of the update's denominator.
#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int CHUNK = 2048, QB = 256, THREADS = 256, PER_LAUNCH = 320;
constexpr int MANT_M = 3, MANT_R = 4;
constexpr long long MAX_GRID = 1 << 23;         // work groups per launch: a grid has fewer than 2^32 lanes
constexpr int MAX_GROUPS = 16, PER_NORM = 160, NCHUNK = 4096, NORM_BLOCKS = 1024, ONE_BLOCK_CHUNKS = 32;

struct Item {                                   // one tensor, in device memory
    float* p;
    float* ema;
    void* copy;
    long long n, off, packed;                   // elements; offset into the flat states (bits = 8: multiple of 256); offset among the 8-bit tensors, packed
    long long chunk0;
    int bits, copy_type, group, pad;
};
struct Factors {                                // of one tensor and step, in the workspace
    double b1, ob1, b2, ob2, gs;                // 64 bits for the borders of the 8-bit codes
    float fb1, fob1, fb2, fob2, fgs;
    float keep, rate, root, eps;                // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t), eps
    unsigned k0, k1;                            // random keys
    int live;                                   // 0: no gradient, or the step is skipped
    int skipped;                                // the whole step is (nothing changes, EMA included)
    int with64;                                 // WITH64_*
};

enum { WITH64_SCALE = 1, WITH64_ROOT = 2 };      // fp32 does not hold gs as a normal number | eps is too small to hide what a root below 2^-60 has lost

struct Grads {                                  // launch argument: the gradients of up to PER_LAUNCH tensors
    const void* g[PER_LAUNCH];
    unsigned char type[PER_LAUNCH];
};
struct NormTensors {                            // launch argument: the tensors one norm launch sums over
    const void* g[PER_NORM];
    long long n[PER_NORM];
    unsigned chunk0[PER_NORM + 1];              // chunks of NCHUNK elements in front of a tensor
    unsigned char type[PER_NORM];
    int count;
};
struct Group { double lr, b1, b2, eps, wd; const float* lr_dev; };
struct Groups { Group g[MAX_GROUPS]; unsigned live[(PER_LAUNCH + 31) / 32]; };

__device__ __forceinline__ float grad_at(const void* g, int type, long long i) {
    if (type == CODEPS_F32) return ((const float*)g)[i];
    const unsigned short h = ((const unsigned short*)g)[i];
    return type == CODEPS_BF16 ? __uint_as_float((unsigned)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
// Four elements from i on.  TAIL: the ones from n on read as zero and are not stored; otherwise all four are inside (no branch: a branch per load makes the
// compiler wait for each one before the next).
template <bool TAIL> __device__ __forceinline__ void load4(const float* p, long long i, long long n, float* o) {
    if (!TAIL || i + 4 <= n) {
        const f32x4u q = *reinterpret_cast<const f32x4u*>(p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = q[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = i + e < n ? p[i + e] : 0.f;
    }
}
template <bool TAIL> __device__ __forceinline__ void store4(float* p, long long i, long long n, const float* v) {
    if (!TAIL || i + 4 <= n) {
        f32x4u q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = v[e];
        *reinterpret_cast<f32x4u*>(p + i) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) p[i + e] = v[e];
    }
}
template <bool TAIL> __device__ __forceinline__ void grad4(const void* g, int type, long long i, long long n, float* o) {
    if (type == CODEPS_F32) {
        load4<TAIL>((const float*)g, i, n, o);
    } else if (!TAIL || i + 4 <= n) {
        const u16x4u q = *reinterpret_cast<const u16x4u*>((const unsigned short*)g + i);
        if (type == CODEPS_BF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __uint_as_float((unsigned)q[e] << 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (float)__builtin_bit_cast(_Float16, (unsigned short)q[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = i + e < n ? grad_at(g, type, i + e) : 0.f;
    }
}
__device__ __forceinline__ unsigned short narrow16(float v, int type) {
    return type == CODEPS_BF16 ? __builtin_bit_cast(unsigned short, (__bf16)v) : __builtin_bit_cast(unsigned short, (_Float16)v);
}
template <bool TAIL> __device__ __forceinline__ void store4_16(void* p, int type, long long i, long long n, const float* v) {
    unsigned short* d = (unsigned short*)p + i;
    if (!TAIL || i + 4 <= n) {
        u16x4u q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = narrow16(v[e], type);
        *reinterpret_cast<u16x4u*>(d) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < n) d[e] = narrow16(v[e], type);
    }
}

// ------------------------------------------------------------------------------------------------------------------ gradient norm
// Sum of squares in 64 bits: an fp32 square overflows at 2e19, and sums over 10^8 elements lose digits.  A block walks a contiguous range of chunks, one
// partial per block, added in a fixed order by the launch that needs the norm.
template <int NT> __device__ __forceinline__ double block_sum64(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) s += red[i];
    return s;
}

// Each group of GT threads walks its own contiguous range of chunks.  norm != NULL (one block): the norm itself, no partials and no second launch.  One block
// (8 groups of 128) up to 32 chunks against two launches, per call: 12 tensors of 3000 elements 6.3 / 9.3 us, 32 of 4096 8.8 / 9.5 us, one of 131072
// 7.9 / 9.4 us; 4 groups of 256 take 10.0, 16 of 64 8.6 us for the 32.
template <int NT, int GT> __global__ __launch_bounds__(NT) void grad_norm_kernel(NormTensors t, double* __restrict__ part, double scale, float* __restrict__ norm) {
    __shared__ double red[NT / 64];
    constexpr int GROUPS = NT / GT, K = NCHUNK / (GT * 4);
    const int tid = threadIdx.x & (GT - 1);
    const unsigned total = t.chunk0[t.count], group = blockIdx.x * GROUPS + (unsigned)__builtin_amdgcn_readfirstlane((int)threadIdx.x / GT), groups = gridDim.x * GROUPS;
    const unsigned c0 = (unsigned)((unsigned long long)total * group / groups), c1 = (unsigned)((unsigned long long)total * (group + 1) / groups);
    int lo = 0, hi = t.count - 1;                                  // the last tensor that starts at or before chunk c0
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.chunk0[mid] <= c0) lo = mid; else hi = mid - 1;
    }
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    for (unsigned c = c0; c < c1; ++c) {
        while (t.chunk0[lo + 1] <= c) ++lo;
        const void* g = t.g[lo];
        const long long n = t.n[lo], i0 = (long long)(c - t.chunk0[lo]) * NCHUNK + tid * 4;
        const int type = t.type[lo];
        const auto chunk = [&](auto tail) {
            float v[K][4];
#pragma unroll
            for (int k = 0; k < K; ++k) grad4<decltype(tail)::value>(g, type, i0 + k * GT * 4, n, v[k]);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += (double)v[k][e] * (double)v[k][e];
        };
        if ((long long)(c - t.chunk0[lo] + 1) * NCHUNK <= n) chunk(std::false_type{});
        else chunk(std::true_type{});
    }
    const double sum = block_sum64<NT>((s[0] + s[1]) + (s[2] + s[3]), red);
    if (threadIdx.x == 0) {
        if (norm) norm[0] = (float)(fabs(scale) * sqrt(sum));
        else part[blockIdx.x] = sum;
    }
}

__device__ __forceinline__ double norm_of(const double* part, int n_part, double scale, double* red) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n_part; i += THREADS) s += part[i];
    return fabs(scale) * sqrt(block_sum64<THREADS>(s, red));
}
__global__ __launch_bounds__(THREADS) void grad_norm_finish_kernel(const double* __restrict__ part, int n_part, double scale, float* __restrict__ norm) {
    __shared__ double red[4];
    const double v = norm_of(part, n_part, scale, red);
    if (threadIdx.x == 0) norm[0] = (float)v;
}

// ---------------------------------------------------------------------------------------------------------- a step's factors per tensor
__global__ __launch_bounds__(THREADS) void adamw_factors_kernel(Groups groups, const Item* __restrict__ items, int base, int count, long long* __restrict__ steps,
                                                                const double* __restrict__ part, int n_part, double grad_scale, double max_norm,
                                                                int skip_nonfinite, float* __restrict__ norm_out, unsigned long long seed,
                                                                Factors* __restrict__ out) {
    __shared__ double red[4];
    double gs = grad_scale;
    bool skip = false;
    if (n_part > 0) {
        const double norm = norm_of(part, n_part, grad_scale, red);
        if (max_norm > 0.0 && norm > max_norm) gs *= max_norm / norm;
        skip = skip_nonfinite && !isfinite(norm);
        if (norm_out && threadIdx.x == 0) norm_out[0] = (float)norm;
    }
    for (int i = threadIdx.x; i < count; i += THREADS) {
        const Group g = groups.g[items[base + i].group & (MAX_GROUPS - 1)];
        const bool live = !skip && (groups.live[i >> 5] >> (i & 31) & 1);
        long long t = steps[base + i];
        if (live) steps[base + i] = ++t;
        Factors f;
        f.live = live; f.skipped = skip;
        f.b1 = g.b1; f.ob1 = 1.0 - g.b1; f.b2 = g.b2; f.ob2 = 1.0 - g.b2; f.gs = gs;
        f.fb1 = (float)f.b1; f.fob1 = (float)f.ob1; f.fb2 = (float)f.b2; f.fob2 = (float)f.ob2; f.fgs = (float)gs;
        const double lr = g.lr_dev ? (double)*g.lr_dev : g.lr;
        f.keep = (float)(1.0 - lr * g.wd);
        f.rate = (float)(lr / (1.0 - pow(g.b1, (double)t)));
        f.root = (float)(1.0 / sqrt(1.0 - pow(g.b2, (double)t)));
        f.eps = (float)g.eps;
        f.with64 = (gs != 0.0 && !(fabs(gs) >= 0x1p-126 && fabs(gs) < 0x1p127) ? WITH64_SCALE : 0) | (f.eps >= f.root * 0x1p-50f ? 0 : WITH64_ROOT);
        // keys: the 64-bit finaliser of Steele, Lea and Flood, "Fast splittable pseudorandom number generators" (2014), over seed, step and tensor
        unsigned long long z = seed + (unsigned long long)t * 0x9E3779B97F4A7C15ull + (unsigned long long)(base + i) * 0xD1B54A32D192ED03ull;
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
        z ^= z >> 31;
        f.k0 = (unsigned)z; f.k1 = (unsigned)(z >> 32);
        out[base + i] = f;
    }
}

// --------------------------------------------------------------------------------------------------------------------- 8-bit codes
// Biased exponent of the block's unit for its largest magnitude (bit pattern): the next power of two when the mantissa would not fit below 2 - 2^-MANT.
template <int MANT> __device__ __forceinline__ int unit_of(unsigned top) {
    const unsigned e = (top + ((1u << (23 - MANT)) - 1)) >> 23;
    return top < 0x00800000u ? 0 : (int)min(e, 255u);
}
// a code's bits, shifted to where fp32 has exponent and mantissa, are the value times 2^-112 -- field 0 included, as fp32's own subnormals
template <int MANT> __device__ __forceinline__ float decode(unsigned code, int unit) {
    return __builtin_ldexpf(__uint_as_float(code << (23 - MANT)), unit - 15);            // (a block that is not finite holds zeros: its caller makes them NaN)
}
// log2 of the quantum at |x| = a, in units of the block (fp32: a's biased exponent is good enough, units from 14 on have nothing smaller than a subnormal code
// that they could not hold)
template <int MANT> __device__ __forceinline__ int place_of(float a, int unit) { return max((int)(__float_as_uint(a) >> 23) - unit, -14); }
// |x| = a -> code at place `low`.  slack: how far (in 2^-16 quanta) a may be from the exact value; unsure: whether that could change the code.
template <int MANT> __device__ __forceinline__ unsigned encode(float a, int unit, int low, unsigned rho, unsigned slack, bool& unsure) {
    const unsigned k = (unsigned)__builtin_ldexpf(a, 143 + MANT - unit - low) + rho;
    unsure = ((k + slack) & 0xffffu) <= 2 * slack;
    return ((unsigned)(low + 14) << MANT) + (k >> 16);
}
template <int MANT> __device__ __forceinline__ unsigned encode64(double a, int unit, unsigned rho) {
    a = unit == 0 ? 0.0 : a;
    const int low = a == 0.0 ? -14 : max(__builtin_amdgcn_frexp_exp(a) - 1 + 127 - unit, -14);
    const unsigned k = (unsigned)ldexp(a, 143 + MANT - unit - low) + rho;
    return min(((unsigned)(low + 14) << MANT) + (k >> 16), (16u << MANT) - 1u);
}
// whether a magnitude that is off by `steps` of its last place at most could have another unit
template <int MANT> __device__ __forceinline__ bool next_to_border(unsigned top, unsigned steps) {
    return ((top + ((1u << (23 - MANT)) - 1) + steps) & 0x7fffffu) <= 2 * steps;
}
// unit_of in 64 bits
template <int MANT> __device__ __forceinline__ unsigned unit64(double a) {
    const unsigned e = (unsigned)(((unsigned long long)__double_as_longlong(a) + ((1ull << (52 - MANT)) - 1)) >> 52) - (1023 - 127);
    return a < 0x1p-126 ? 0u : min(e, 255u);
}
// 32 random bits of an element: a multiply-xorshift mix of two rounds (shifts and multipliers of Wellons's search for low-bias 32-bit hashes), keyed per tensor
// and step
__device__ __forceinline__ unsigned random_bits(long long i, unsigned k0, unsigned k1) {
    unsigned x = (unsigned)i + (unsigned)(i >> 32) * 0x9E3779B1u + k0;
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x = x ^ (x >> 15) ^ k1;
    x *= 0x846CA68Bu;
    return x ^ (x >> 16);
}
// largest of a wave's values, in every lane: lanes 1, 2, 4, 8 away over DPP, 16 and 32 away by exchanging half rows
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
    v = dpp_max<0xB1>(v);
    v = dpp_max<0x4E>(v);
    v = dpp_max<0x141>(v);
    v = dpp_max<0x140>(v);
    u32x2 q = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(q[0], q[1]);
    q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (unsigned)__builtin_amdgcn_readfirstlane((int)max(q[0], q[1]));
}

// ------------------------------------------------------------------------------------------------------------------------ the update
struct States { float *m, *v; unsigned char *mc, *me, *rc, *re; };

// The new moments in 64 bits, every operation rounded by itself: 16-bit gradients and codes lie on coarse grids, sums fall exactly on borders between codes,
// and there the last bit decides.
__device__ __forceinline__ void moments64(const Factors& f, double m0, double r0, double g, double& m, double& v) {
#pragma clang fp contract(off)
    const double gg = g * f.gs, a = f.b1 * m0, b = f.ob1 * gg, c = f.b2 * (r0 * r0), d = f.ob2 * gg * gg;
    m = a + b;
    v = c + d;
}

// One chunk of a tensor; WIDE: 32-bit states.  The update divides by a reciprocal that is off by a step (2^-23 of the update, one of the handful of roundings
// that it takes in fp32), an 8-bit root is a square root off by a step, which the two units of `encode` allow for.  The gradients are loaded last: their type is
// known at run time, and where the branches meet the compiler waits.
template <bool WIDE, bool TAIL>
__device__ __forceinline__ void update_chunk(const Item& it, const Factors& f, const void* gp, int gt, float* const ema, long long start, const States& st, float al, float oal) {
    constexpr int K = CHUNK / (THREADS * 4);
    const long long n = it.n, first = start + (long long)threadIdx.x * 4;
    float p[K][4], g[K][4], a[K][4], b[K][4], em[K][4];
    unsigned mc[K], rc[K];
    int mu[K], ru[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = first + k * THREADS * 4;
        load4<TAIL>(it.p, i, n, p[k]);
        if (ema) load4<TAIL>(ema, i, n, em[k]);
        if constexpr (WIDE) {
            load4<TAIL>(st.m + it.off, i, n, a[k]);
            load4<TAIL>(st.v + it.off, i, n, b[k]);
        } else if (!TAIL || (i & ~(long long)(QB - 1)) < n) {                  // the same for a whole wave: it owns the 256 elements from here on
            const long long q = it.off + i;
            mc[k] = *reinterpret_cast<const unsigned*>(st.mc + q);
            rc[k] = *reinterpret_cast<const unsigned*>(st.rc + q);
            const long long blk = (it.off + start + k * THREADS * 4) / QB + (threadIdx.x >> 6);
            mu[k] = st.me[blk];
            ru[k] = st.re[blk];
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) grad4<TAIL>(gp, gt, first + k * THREADS * 4, n, g[k]);
    float fgs = f.fgs;
    if constexpr (WIDE) {
        if (__builtin_expect(f.with64 & WITH64_SCALE, false)) {                // (clipping gradients of 1e38: the factor has few bits in fp32, or none)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) g[k][e] = (float)((double)g[k][e] * f.gs);
            fgs = 1.f;
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long long i = first + k * THREADS * 4;
        if constexpr (WIDE) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float gg = g[k][e] * fgs;
                a[k][e] = f.fb1 * a[k][e] + f.fob1 * gg;
                b[k][e] = f.fb2 * b[k][e] + f.fob2 * gg * gg;
                p[k][e] = p[k][e] * f.keep - f.rate * a[k][e] * __builtin_amdgcn_rcpf(sqrtf(b[k][e]) * f.root + f.eps);
            }
            store4<TAIL>(st.m + it.off, i, n, a[k]);
            store4<TAIL>(st.v + it.off, i, n, b[k]);
        } else {
            if (TAIL && (i & ~(long long)(QB - 1)) >= n) continue;
            const int um = __builtin_amdgcn_readfirstlane(mu[k]), ur = __builtin_amdgcn_readfirstlane(ru[k]);
            const float bad_m = um == 255 ? __uint_as_float(0x7fc00000u) : 0.f, bad_r = ur == 255 ? __uint_as_float(0x7fc00000u) : 0.f;
            float m0[4], r0[4], c[4];
            unsigned mtop = 0, rtop = 0;
            bool deep = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned code = mc[k] >> (8 * e);
                const float q = decode<MANT_M>(code & 127u, um) + bad_m;
                m0[e] = __uint_as_float(__float_as_uint(q) | (code & 128u) << 24);
                r0[e] = decode<MANT_R>(rc[k] >> (8 * e) & 255u, ur) + bad_r;
                const float gg = g[k][e] * fgs;
                c[e] = f.fob1 * gg;
                a[k][e] = __builtin_fmaf(f.fb1, m0[e], c[e]);
                b[k][e] = __builtin_amdgcn_sqrtf(__builtin_fmaf(f.fb2, r0[e] * r0[e], f.fob2 * gg * gg));
                mtop = max(mtop, __float_as_uint(a[k][e]) & 0x7fffffffu);
                rtop = max(rtop, __float_as_uint(b[k][e]) & 0x7fffffffu);
            }
            mtop = wave_umax(mtop);
            rtop = wave_umax(rtop);
            int nm = unit_of<MANT_M>(mtop), nr = unit_of<MANT_R>(rtop);
            // The largest magnitudes are off by 2^-21 of the root and 2^-21 of m's terms.  Those are below |m| + 2 |b1 m0|, and m0 below 2 of its block's units: at most
            // 32 steps of m's last place, and twice as many for every binary place by which m has come out below m0's unit.
            const bool unsure = next_to_border<MANT_M>(mtop, 32u << min(max(um + 1 - (int)(mtop >> 23), 0), 17)) || next_to_border<MANT_R>(rtop, 16u);
            if (__builtin_expect(nr < 91 || (f.with64 & WITH64_ROOT), false)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) deep = deep || (b[k][e] < 0x1p-60f && (r0[e] != 0.f || g[k][e] != 0.f));
                deep = __builtin_amdgcn_ballot_w64(deep) != 0;
            }
            unsigned ncm = 0, ncr = 0;
            const bool ends = nm < 14 || nr < 14 || nm == 255 || nr > 189;
            if (__builtin_expect(unsure || deep || ends || (f.with64 & WITH64_SCALE), false)) {      // the same for the whole wave
                // (a block of zeros, states and gradients: what a row without gradients keeps is 10 % of the whole step in 64 bits)
                bool some = ((mc[k] & 0x7f7f7f7fu) | rc[k]) != 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) some = some || g[k][e] != 0.f;
                if (nm == 0 && nr == 0 && f.eps > 0.f && __builtin_amdgcn_ballot_w64(some) == 0) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[k][e] *= f.keep;
                } else {
                    double m[4], r[4];
                    unsigned tm = 0, tr = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        double v;
                        moments64(f, (double)m0[e], (double)r0[e], (double)g[k][e], m[e], v);
                        r[e] = sqrt(v);
                        p[k][e] = (float)((double)p[k][e] * f.keep - (double)f.rate * m[e] / (r[e] * f.root + f.eps));
                        tm = max(tm, unit64<MANT_M>(fabs(m[e])));
                        tr = max(tr, unit64<MANT_R>(r[e]));
                    }
                    nm = (int)wave_umax(tm);
                    nr = (int)wave_umax(tr);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const unsigned rnd = random_bits(i + e, f.k0, f.k1);
                        ncm |= (encode64<MANT_M>(fabs(m[e]), nm, rnd & 0xffffu) | (m[e] < 0.0 ? 128u : 0u)) << (8 * e);
                        ncr |= encode64<MANT_R>(r[e], nr, rnd >> 16) << (8 * e);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[k][e] = p[k][e] * f.keep - f.rate * a[k][e] * __builtin_amdgcn_rcpf(b[k][e] * f.root + f.eps);
                    const unsigned rnd = random_bits(i + e, f.k0, f.k1);
                    bool dm, dr;
                    // m may come out of a cancellation: its error is that of its two terms, (|b1 m| + |(1 - b1) g'|) 2^-22, in units of 2^-16 quanta
                    const float am = fabsf(a[k][e]), size = fabsf(f.fb1 * m0[e]) + fabsf(c[e]);
                    const int low = place_of<MANT_M>(am, nm);
                    const unsigned slack = 2u + (unsigned)fminf(__builtin_ldexpf(size, 143 + MANT_M - 22 - nm - low), 33000.f);    // (2 * 33002 covers every remainder)
                    bool minus = a[k][e] < 0.f;
                    unsigned cm = encode<MANT_M>(am, nm, low, rnd & 0xffffu, slack, dm);
                    unsigned cr = encode<MANT_R>(b[k][e], nr, place_of<MANT_R>(b[k][e], nr), rnd >> 16, 2u, dr);
                    if (__builtin_expect(dm || dr, false)) {
                        double m, v;
                        moments64(f, (double)m0[e], (double)r0[e], (double)g[k][e], m, v);
                        minus = m < 0.0;
                        cm = encode64<MANT_M>(fabs(m), nm, rnd & 0xffffu);
                        cr = encode64<MANT_R>(sqrt(v), nr, rnd >> 16);
                    }
                    ncm |= (cm | (minus ? 128u : 0u)) << (8 * e);
                    ncr |= cr << (8 * e);
                }
            }
            if (nm == 255) ncm = 0;
            if (nr == 255) ncr = 0;
            const long long q = it.off + i;
            *reinterpret_cast<unsigned*>(st.mc + q) = ncm;
            *reinterpret_cast<unsigned*>(st.rc + q) = ncr;
            if ((threadIdx.x & 63) == 0) {
                st.me[q / QB] = (unsigned char)nm;
                st.re[q / QB] = (unsigned char)nr;
            }
        }
        store4<TAIL>(it.p, i, n, p[k]);
        if (it.copy) store4_16<TAIL>(it.copy, it.copy_type, i, n, p[k]);
        if (ema) {
#pragma unroll
            for (int e = 0; e < 4; ++e) em[k][e] = al * em[k][e] + oal * p[k][e];
            store4<TAIL>(ema, i, n, em[k]);
        }
    }
}

__global__ __launch_bounds__(THREADS) void adamw_step_kernel(Grads grads, const Item* __restrict__ items, const int* __restrict__ chunk_items,
                                                             const Factors* __restrict__ factors, int base, long long first_chunk, States st, float al, float oal) {
    const long long chunk = first_chunk + blockIdx.x;
    const int t = chunk_items[chunk];
    const Item it = items[t];
    const Factors& f = factors[t];
    float* const ema = al >= 0.f ? it.ema : nullptr;
    if (f.skipped || (!f.live && !ema)) return;
    const long long start = (chunk - it.chunk0) * CHUNK;
    if (!f.live) {                                                             // no gradient: the average follows the parameter as it is
        for (int k = 0; k < CHUNK / (THREADS * 4); ++k) {
            const long long i = start + (k * THREADS + threadIdx.x) * 4;
            float p[4], em[4];
            load4<true>(it.p, i, it.n, p);
            load4<true>(ema, i, it.n, em);
#pragma unroll
            for (int e = 0; e < 4; ++e) em[e] = al * em[e] + oal * p[e];
            store4<true>(ema, i, it.n, em);
        }
        return;
    }
    const void* gp = grads.g[t - base];
    const int gt = grads.type[t - base];
    const bool whole = start + CHUNK <= it.n;
    if (it.bits == 32) {
        if (whole) update_chunk<true, false>(it, f, gp, gt, ema, start, st, al, oal);
        else update_chunk<true, true>(it, f, gp, gt, ema, start, st, al, oal);
    } else {
        if (whole) update_chunk<false, false>(it, f, gp, gt, ema, start, st, al, oal);
        else update_chunk<false, true>(it, f, gp, gt, ema, start, st, al, oal);
    }
}

__global__ __launch_bounds__(THREADS) void adamw_moments_kernel(const Item* __restrict__ items, const int* __restrict__ chunk_items, const unsigned char* __restrict__ mc,
                                                                const unsigned char* __restrict__ me, const unsigned char* __restrict__ rc,
                                                                const unsigned char* __restrict__ re, long long first_chunk, void* __restrict__ om,
                                                                void* __restrict__ orr) {
    const long long chunk = first_chunk + blockIdx.x;
    const Item it = items[chunk_items[chunk]];
    if (it.bits != 8) return;
    const long long n = it.n, start = (chunk - it.chunk0) * CHUNK;
#pragma unroll
    for (int k = 0; k < CHUNK / (THREADS * 4); ++k) {
        const long long i = start + k * THREADS * 4 + threadIdx.x * 4, q = it.off + i;
        if (i >= n) continue;
        const unsigned cm = *reinterpret_cast<const unsigned*>(mc + q), cr = *reinterpret_cast<const unsigned*>(rc + q);
        const int mu = me[q / QB], ru = re[q / QB];
        const float bad_m = mu == 255 ? __uint_as_float(0x7fc00000u) : 0.f, bad_r = ru == 255 ? __uint_as_float(0x7fc00000u) : 0.f;
        float m[4], r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned c = cm >> (8 * e) & 255u;
            const float v = decode<MANT_M>(c & 127u, mu) + bad_m;
            m[e] = c & 128u ? -v : v;
            r[e] = decode<MANT_R>(cr >> (8 * e) & 255u, ru) + bad_r;
        }
        store4_16<true>((unsigned short*)om + it.packed, CODEPS_BF16, i, n, m);
        store4_16<true>((unsigned short*)orr + it.packed, CODEPS_BF16, i, n, r);
    }
}

bool grad_type_ok(int t) { return t == CODEPS_F32 || t == CODEPS_BF16 || t == CODEPS_F16; }

// partial sums of squares of all tensors into `part`; the number of partials, or a negative code.  norm != NULL: where one block does it all, the norm is
// stored there and -- since nothing is left to add -- 0 returned as *finished = true.
int norm_partials(const void* const* grads, const unsigned char* types, const long long* numels, int n, double* part, hipStream_t st, double scale = 1.0,
                  float* norm = nullptr, bool* finished = nullptr) {
    int parts = 0;
    for (int base = 0; base < n;) {
        NormTensors t;
        t.count = 0;
        long long chunks = 0;
        while (base < n && t.count < PER_NORM) {
            const long long c = grads[base] ? (numels[base] + NCHUNK - 1) / NCHUNK : 0;            // (32 bits: check_grads bounds the sum)
            t.g[t.count] = grads[base]; t.n[t.count] = numels[base]; t.type[t.count] = types[base];
            t.chunk0[t.count++] = (unsigned)chunks;
            chunks += c;
            ++base;
        }
        t.chunk0[t.count] = (unsigned)chunks;
        if (chunks == 0) continue;
        if (norm && chunks <= ONE_BLOCK_CHUNKS && t.count == n) {
            hipLaunchKernelGGL((grad_norm_kernel<1024, 128>), dim3(1), dim3(1024), 0, st, t, part, scale, norm);
            CODEPS_CHECK_LAUNCH("grad_norm_kernel");
            *finished = true;
            return 0;
        }
        const int blocks = (int)std::min<long long>(chunks, NORM_BLOCKS);
        hipLaunchKernelGGL((grad_norm_kernel<THREADS, THREADS>), dim3(blocks), dim3(THREADS), 0, st, t, part + parts, 1.0, (float*)nullptr);
        CODEPS_CHECK_LAUNCH("grad_norm_kernel");
        parts += blocks;
    }
    return parts;
}
size_t norm_bytes(int n) { return (size_t)cdiv(n, PER_NORM) * NORM_BLOCKS * sizeof(double); }

int check_grads(const void* const* grads, const unsigned char* types, const long long* numels, int n, const char* who) {
    CODEPS_REQUIRE(grads && types && numels && n >= 1 && n <= (1 << 24), CODEPS_ERR_ARG, "%s: null array, or not 1 .. 2^24 tensors", who);
    long long total = 0;
    for (int i = 0; i < n; ++i) {
        CODEPS_REQUIRE(numels[i] >= 0 && numels[i] <= (1LL << 40) && (total += numels[i]) <= (1LL << 43), CODEPS_ERR_ARG, "%s: tensor %d has %lld elements (at most 2^40, 2^43 together)", who, i, numels[i]);
        CODEPS_REQUIRE(!grads[i] || grad_type_ok(types[i]), CODEPS_ERR_ARG, "%s: gradient %d has the unknown type %d", who, i, (int)types[i]);
        CODEPS_REQUIRE(((uintptr_t)grads[i] & (types[i] == CODEPS_F32 ? 3 : 1)) == 0, CODEPS_ERR_ARG, "%s: gradient %d is not aligned to its elements", who, i);
    }
    return CODEPS_OK;
}

}  // namespace

// =============================================================================================== C ABI
extern "C" size_t codeps_adamw_item_bytes(void) { return sizeof(Item); }

extern "C" long long codeps_adamw_item_fill(void* item, float* param, float* ema, void* copy, int copy_type, long long numel, int bits,
                                            long long state_offset, long long packed_offset, int group, long long chunk0) {
    CODEPS_REQUIRE(item && (param || numel == 0) && numel >= 0 && numel <= (1LL << 40), CODEPS_ERR_ARG, "adamw_item_fill: null pointer or bad element count");
    CODEPS_REQUIRE(bits == 32 || bits == 8, CODEPS_ERR_ARG, "adamw_item_fill: states have 32 or 8 bits, not %d", bits);
    CODEPS_REQUIRE(state_offset >= 0 && packed_offset >= 0 && chunk0 >= 0 && (bits == 32 || state_offset % QB == 0), CODEPS_ERR_ARG,
                   "adamw_item_fill: state offset %lld (8-bit states start at multiples of %d)", state_offset, QB);
    CODEPS_REQUIRE(group >= 0 && group < MAX_GROUPS, CODEPS_ERR_ARG, "adamw_item_fill: group %d of at most %d", group, MAX_GROUPS);
    CODEPS_REQUIRE(!copy || copy_type == CODEPS_BF16 || copy_type == CODEPS_F16, CODEPS_ERR_ARG, "adamw_item_fill: a copy is bf16 or fp16");
    CODEPS_REQUIRE((((uintptr_t)param | (uintptr_t)ema) & 3) == 0 && ((uintptr_t)copy & 1) == 0, CODEPS_ERR_ARG, "adamw_item_fill: unaligned pointer");
    const Item it = {param, ema, copy, numel, state_offset, packed_offset, chunk0, bits, copy_type, group, 0};
    memcpy(item, &it, sizeof(it));
    return (numel + CHUNK - 1) / CHUNK;
}

extern "C" size_t codeps_adamw_workspace_bytes(int n_items) {
    if (n_items < 1) { codeps_set_error("adamw_workspace_bytes: %d tensors", n_items); return 0; }
    return align_up((size_t)n_items * sizeof(Factors), 256) + norm_bytes(n_items);
}

extern "C" int codeps_adamw_step(const void* items, int n_items, const int* chunk_items, const long long* chunk0, const void* const* grads,
                                 const unsigned char* grad_types, const long long* numels, const codeps_adamw_group* groups, int n_groups,
                                 long long* steps, float* exp_avg, float* exp_avg_sq, unsigned char* exp_avg_codes, unsigned char* exp_avg_exponents,
                                 unsigned char* root_codes, unsigned char* root_exponents, double grad_scale, double max_norm, int skip_nonfinite,
                                 float* norm, unsigned long long seed, double ema_alpha, void* workspace, size_t workspace_bytes,
                                 codeps_stream_t stream) {
    const int rc = check_grads(grads, grad_types, numels, n_items, "adamw_step");
    if (rc != CODEPS_OK) return rc;
    CODEPS_REQUIRE(items && chunk_items && chunk0 && steps && groups && workspace, CODEPS_ERR_ARG, "adamw_step: null pointer");
    CODEPS_REQUIRE(n_groups >= 1 && n_groups <= MAX_GROUPS, CODEPS_ERR_ARG, "adamw_step: %d groups (1 .. %d)", n_groups, MAX_GROUPS);
    CODEPS_REQUIRE(workspace_bytes >= codeps_adamw_workspace_bytes(n_items), CODEPS_ERR_WORKSPACE, "adamw_step: %zu bytes of workspace, %zu are needed",
                   workspace_bytes, codeps_adamw_workspace_bytes(n_items));
    CODEPS_REQUIRE((exp_avg == nullptr) == (exp_avg_sq == nullptr) && (exp_avg_codes == nullptr) == (root_codes == nullptr) &&
                   (exp_avg_codes == nullptr) == (exp_avg_exponents == nullptr) && (exp_avg_codes == nullptr) == (root_exponents == nullptr) &&
                   (exp_avg || exp_avg_codes), CODEPS_ERR_ARG, "adamw_step: incomplete states");
    for (int i = 0; i < n_groups; ++i) {
        const codeps_adamw_group& g = groups[i];
        CODEPS_REQUIRE(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0 && g.eps >= 0.0, CODEPS_ERR_ARG,
                       "adamw_step: group %d has betas (%g, %g), eps %g", i, g.beta1, g.beta2, g.eps);
    }
    for (int i = 0; i < n_items; ++i)
        CODEPS_REQUIRE(chunk0[i + 1] - chunk0[i] == (numels[i] + CHUNK - 1) / CHUNK, CODEPS_ERR_ARG, "adamw_step: tensor %d: chunk table and element count differ", i);
    hipStream_t st = (hipStream_t)stream;
    Factors* factors = (Factors*)workspace;
    double* part = (double*)((char*)workspace + align_up((size_t)n_items * sizeof(Factors), 256));
    int parts = 0;
    if (max_norm > 0.0 || skip_nonfinite || norm) {
        parts = norm_partials(grads, grad_types, numels, n_items, part, st);
        if (parts < 0) return parts;
    }
    Groups gs;
    for (int i = 0; i < MAX_GROUPS; ++i) {
        const codeps_adamw_group& g = groups[std::min(i, n_groups - 1)];
        gs.g[i] = {g.lr, g.beta1, g.beta2, g.eps, g.weight_decay, g.lr_device};
    }
    const States states = {exp_avg, exp_avg_sq, exp_avg_codes, exp_avg_exponents, root_codes, root_exponents};
    for (int base = 0; base < n_items; base += PER_LAUNCH) {
        const int count = std::min(PER_LAUNCH, n_items - base);
        memset(gs.live, 0, sizeof(gs.live));
        Grads gr;
        for (int i = 0; i < count; ++i) {
            gr.g[i] = grads[base + i];
            gr.type[i] = grad_types[base + i];
            if (grads[base + i]) gs.live[i >> 5] |= 1u << (i & 31);
        }
        // (without gradients at all there are no partials: the norm is 0)
        if (parts == 0 && norm && base == 0) {
            hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(THREADS), 0, st, (const double*)part, 0, grad_scale, norm);
            CODEPS_CHECK_LAUNCH("grad_norm_finish_kernel");
        }
        hipLaunchKernelGGL(adamw_factors_kernel, dim3(1), dim3(THREADS), 0, st, gs, (const Item*)items, base, count, steps, (const double*)part, parts,
                           grad_scale, max_norm, skip_nonfinite, norm, seed, factors);
        CODEPS_CHECK_LAUNCH("adamw_factors_kernel");
        long long first = chunk0[base];
        const long long end = chunk0[base + count];
        for (; first < end; first += MAX_GRID) {
            hipLaunchKernelGGL(adamw_step_kernel, dim3((unsigned)std::min<long long>(end - first, MAX_GRID)), dim3(THREADS), 0, st, gr, (const Item*)items,
                               chunk_items, (const Factors*)factors, base, first, states, (float)ema_alpha, (float)(1.0 - ema_alpha));
            CODEPS_CHECK_LAUNCH("adamw_step_kernel");
        }
    }
    return CODEPS_OK;
}

extern "C" int codeps_adamw_moments_8bit(const void* items, int n_items, const int* chunk_items, long long n_chunks, const unsigned char* exp_avg_codes,
                                         const unsigned char* exp_avg_exponents, const unsigned char* root_codes, const unsigned char* root_exponents,
                                         void* exp_avg_bf16, void* root_bf16, codeps_stream_t stream) {
    CODEPS_REQUIRE(items && n_items >= 1 && chunk_items && n_chunks >= 1 && n_chunks < (1LL << 31) && exp_avg_codes && exp_avg_exponents && root_codes &&
                   root_exponents && exp_avg_bf16 && root_bf16, CODEPS_ERR_ARG, "adamw_moments_8bit: bad arguments");
    for (long long first = 0; first < n_chunks; first += MAX_GRID) {
        hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)std::min<long long>(n_chunks - first, MAX_GRID)), dim3(THREADS), 0, (hipStream_t)stream,
                           (const Item*)items, chunk_items, exp_avg_codes, exp_avg_exponents, root_codes, root_exponents, first, exp_avg_bf16, root_bf16);
        CODEPS_CHECK_LAUNCH("adamw_moments_kernel");
    }
    return CODEPS_OK;
}

extern "C" size_t codeps_grad_norm_workspace_bytes(int n_tensors) {
    if (n_tensors < 1) { codeps_set_error("grad_norm_workspace_bytes: %d tensors", n_tensors); return 0; }
    return norm_bytes(n_tensors);
}

extern "C" int codeps_grad_norm(const void* const* grads, const unsigned char* grad_types, const long long* numels, int n_tensors, double scale,
                                float* norm, void* workspace, size_t workspace_bytes, codeps_stream_t stream) {
    const int rc = check_grads(grads, grad_types, numels, n_tensors, "grad_norm");
    if (rc != CODEPS_OK) return rc;
    CODEPS_REQUIRE(norm && workspace && workspace_bytes >= norm_bytes(n_tensors), CODEPS_ERR_WORKSPACE, "grad_norm: null pointer or workspace too small");
    hipStream_t st = (hipStream_t)stream;
    bool finished = false;
    const int parts = norm_partials(grads, grad_types, numels, n_tensors, (double*)workspace, st, scale, norm, &finished);
    if (parts < 0 || finished) return parts;
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(THREADS), 0, st, (const double*)workspace, parts, scale, norm);
    CODEPS_CHECK_LAUNCH("grad_norm_finish_kernel");
    return CODEPS_OK;
}
