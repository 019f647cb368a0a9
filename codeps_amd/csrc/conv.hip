// NHWC fp32 implicit-GEMM convolution engine on the gfx950 matrix cores:
// forward (+fused nearest-x2 upsample of source 0, concat-by-pointer of two sources, zero / reflect
// padding, per-channel affine (folded eval BatchNorm or bias), residual add, ReLU / ELU), data gradient
// and weight gradient.  fp32 in, fp32 out, fp32 accumulation.  The main forward / data-gradient kernel feeds the bf16 MFMA
// (v_mfma_f32_32x32x16_bf16) with every fp32 operand split EXACTLY into three bf16 pieces and sums the six piece products of
// order <= 2 (error <= 2^-24 per product, below fp32 rounding; 2.7x fewer MFMA cycles than v_mfma_f32_32x32x2_f32, which
// weight gradients, 16-column kernels and CODEPS_SPLIT=0 use).  No reduced precision.
//
// Replaces the ATen/cuDNN convolutions behind: torchvision ResNet (models/resnet_encoder.py:115-126),
// DepthHead / SemanticHead decoders (models/depth_head.py:60-71, models/semantic_head.py:50-72),
// InstanceHead 1x1 convs (models/instance_head.py:24-57,99-111), PoseHead (models/pose_head.py:36-44).
//
// GEMM view:  forward  Y[m][n] = sum_{tap,c} X(m,tap,c) * Wf[n][tap][c]      m = output pixel, n = out channel
//             dgrad    dX[m][n] = sum_{tap,c} dZ(m,tap,c) * Wd[n][tap][c]    m = input pixel,  n = in channel
//             wgrad    dW[m][n](tap) = sum_p dZ[p][m] * X(p,tap,n)           m = out channel,  n = in channel
// Block tile (32*WM*TM) x (32*WN*TN), 256 threads = 4 waves (WM x WN), wave tile TM x TN MFMA tiles of
// 32x32; K-step BK channels of one tap.  Per block a gather table (byte offset of every row x tap, out-of-range marker
// for zero padding) is built once; the K loop is buffer_load (hardware zero fill) -> registers -> one LDS stage ->
// ds_read_b128 fragments -> MFMA, the next stage's loads in flight during the MFMAs.  LDS rows padded to BK+4 floats =>
// conflict-free ds_read_b128 fragment reads (row stride 36 or 20 dwords walks all 16 four-bank slots).  blockIdx is
// remapped so that the N-tiles of one M-tile run on the same XCD (they share the A tile through that XCD's L2).
// Variants: 16-column kernels (N <= 16, v_mfma_f32_16x16x4_f32, operands straight to registers), split-K for small-M
// launches, per-tap / halo-tile / stem weight-gradient kernels.  DESIGN.md section 3 has the measurements behind each choice.
#include <stdlib.h>
#include <type_traits>

#include "common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

enum { MODE_FWD = 0, MODE_DGRAD = 1 };

// Tuning aid (never set in the shipped build): -DCODEPS_ABLATE=1 drops the global loads of the K loop, =2 also the
// LDS stores and barriers, =3 also the LDS fragment reads -- results are garbage, timings bound each pipeline stage.
#ifndef CODEPS_ABLATE
#define CODEPS_ABLATE 0
#endif
#ifndef CODEPS_IGEMM_SWZ
#define CODEPS_IGEMM_SWZ 1       // A/B builds only: 0 = the padded 208-byte LDS rows of rounds 2-3 in conv_igemm_kernel<split3>
#endif
#ifndef CODEPS_HALO_SWZ
#define CODEPS_HALO_SWZ 1        // A/B builds only: 0 = the 208-byte activation pitch and unswizzled weight tiles of rounds 2-3
#endif

struct ConvP {
    // geometry (see codeps_conv_desc)
    int B, H, W;          // logical input size (after the optional x2 upsample of source 0)
    int C0, C1, Ct;       // channels of source 0 / 1, Ct = C0 + C1
    int up0;
    int Co, Ho, Wo;
    int KH, KW, stride, pad, pad_mode;   // stride / pad: vertical;  stride_w / pad_w: horizontal
    int stride_w, pad_w;
    int pitch0, wrow0;    // forward, source 0 as overlapping pixels: floats between pixel starts / pixels per stored row (0 = dense)
    int act;
    int M, N;             // GEMM rows / cols of this launch
    int n_mt, n_nt;       // tile counts
    int src;              // dgrad: which source's gradient (0/1)
    int Cs;               // dgrad: channels of that source;  c_off = its channel offset in the packed weights
    int c_off;
    // stride-2 dgrad by input-parity class: rows enumerate the pixels (2y'+py, 2x'+px) only and the K loop walks just the
    // taps whose parity can reach them (3x3: 1, 2, 2 or 4 taps instead of 9 mostly-zero ones)
    int par, py, px, ky0, kx0, nky, nkx, Hc, Wc;
    // par == 2 (round 5): ALL parity classes in one launch -- blockIdx.z = class, its (py, px, ky0, kx0, nky, nkx) in pcls; Hc / Wc / M
    // are the same for every class (even H and W).  Four launches of 96-192 blocks each left 25-60 % of the CUs idle.
    int pcls[4][6];
    int grid_mult;        // launches that repeat the tile grid (4 parity classes): what the tile cost model multiplies the blocks by
    // split-K (small-M launches): gridDim.y slices of `ksteps` K-steps each write raw partial sums to part[slice][M][N]
    int ksplit, ksteps;
    float* part;
    size_t part_bytes;
    // weights of this launch pre-split into three bf16 pieces ([row][K group of 32][piece][32], written by the weight pack
    // behind its fp32 part); the 3-piece kernel stages its B operand from here with plain copies
    const void* w3;
    // ... and as two fp16 pieces of w * 2^kb ([row][K group of 32][piece][32]); w2s[0] = 2^-kb (the pack's per-tensor scale, inverted)
    const void* w2;
    const float* w2s;
    // epilogue extras (codeps_conv_epilogue; all optional, applied to the value the epilogue is about to store, after the residual /
    // second-gradient add):  a GATE  v *= g'  and per-M-tile COLUMN STATISTICS of the gated v
    const float* ex_gate;       // gate 1 / 2: the activation's output [M][N];  gate 3: the block output when a residual fed the ReLU (else null)
    int ex_gate_act;            // 0 none, 1 ReLU' (gate > 0), 2 ELU' (gate > 0 ? 1 : gate + 1), 3 train-mode BatchNorm (+ ReLU) backward
    int ex_stat;                // 0 none, 1 (shift, sum (v - shift), sum (v - shift)^2), 2 sum v, 3 (sum v, sum v * xhat)
    float* ex_part;             // [tile][rows of the mode][N]
    int ex_tile0;               // tile index of this launch's first M tile (the stride-2 parity classes are four launches)
    int ex_img_rows;            // gate 3 / stat 1 with the generic kernels: GEMM rows per image (a multiple of the tile's rows)
    int ex_fin;                 // K slices: the extras run in splitk_finish_ex_kernel (64-row tiles) instead of the GEMM kernel's epilogue
    const float* ex_bn_x;       // gate 3: BatchNorm's input z [M][N], mean / invstd [groups][N], gamma / beta [N]
    const float* ex_bn_mean; const float* ex_bn_invstd; const float* ex_bn_gamma; const float* ex_bn_beta;
    int ex_bn_relu, ex_bn_ng;
    int ex_bn_b0[8];            // first image of every statistic group
    // forward, source 0 arrives as the INPUT of a train-mode BatchNorm + ReLU (codeps_conv2d_fwd_in): [image][mean | invstd | gamma | beta][Ct];
    // the kernel normalises on its operand load -- the normalised tensor is never written
    const float* in_aff;
};


typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

// Split-precision operands (CODEPS_SPLIT, default 3 pieces): x = p0 + p1 (+ p2) with bf16 pieces (round to nearest each time);
// bf16 x bf16 products are exact in fp32, so NP = 3 with the six products of order <= 2 reproduces the fp32 product to
// ~6e-9 relative, NP = 2 with three products to ~4e-6 (tools/split_precision_study.py).
// eight bf16 values (k .. k + 7) as one 16-byte LDS store
__device__ __forceinline__ i32x4 pack8(const u16x4 a, const u16x4 b) {
    return i32x4{(int)((unsigned)a[0] | ((unsigned)a[1] << 16)), (int)((unsigned)a[2] | ((unsigned)a[3] << 16)),
                 (int)((unsigned)b[0] | ((unsigned)b[1] << 16)), (int)((unsigned)b[2] | ((unsigned)b[3] << 16))};
}

template <int NP>
__device__ __forceinline__ void split_bf16(const f32x4 v, u16x4 (&pc)[NP]) {
    f32x4 r = v;
#pragma unroll
    for (int q = 0; q < NP; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned short h = __builtin_bit_cast(unsigned short, (__bf16)r[e]);
            pc[q][e] = h;
            r[e] -= __builtin_bit_cast(float, (unsigned)h << 16);
        }
}

// ---- Two-piece fp16 arithmetic (round 6; ARITH = 16 in the kernels that have it, CODEPS_SPLIT=16 / codeps_conv2d_set_arith(16)).
// x s = hi + lo with hi = rn16(x s), lo = rn16(x s - hi): |x s - hi - lo| <= 2^-22 |x s| (two 11-bit significands and the sign of lo),
// and the THREE products hi hi + hi lo + lo hi on v_mfma_f32_16x16x32_f16 (fp16 x fp16 is exact in fp32, fp32 accumulation) drop a term
// <= 2^-24: half the matrix instructions of the 3 x bf16 split and 4 instead of 6 bytes per element in LDS, at an operand error of the size
// of fp32's own rounding.  fp16 has 5 exponent bits, so every operand carries a power-of-two scale s that puts its largest magnitude
// just below 2^15: weights per tensor, found by the pack (pack_amax_kernel); activations / gradients per BLOCK and K chunk inside the
// kernel (the running maximum exponent of the tiles staged so far; when it grows the accumulators are multiplied by the exact ratio),
// so no tensor needs a side channel for its range.  Elements more than 2^17 below the block's maximum lose their lo piece gradually
// (fp16 subnormals, honoured by the instruction: tools/f16_mfma_probe.py): absolute error <= 2^-40 of that maximum.
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr int F16_TARGET = 14;      // |x s| < 2^(F16_TARGET + 1)
constexpr int F16_EMIN = 27;        // operands below 2^-100 count as 2^-100 when the scale is chosen

__device__ __forceinline__ void split_f16(const f32x4 v, const float s, u16x4& hi, u16x4& lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const _Float16 h = (_Float16)(v[e] * s);
        const _Float16 l = (_Float16)__builtin_fmaf(v[e], s, -(float)h);
        hi[e] = __builtin_bit_cast(unsigned short, h);
        lo[e] = __builtin_bit_cast(unsigned short, l);
    }
}
// biased exponent of the largest magnitude among the wave's values m (>= 0): every lane returns it
__device__ __forceinline__ int wave_max_exponent(float m) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    return (int)(__builtin_bit_cast(unsigned, m) >> 23);
}
// scale 2^(F16_TARGET - (e - 127)) of a tile whose maximum exponent is e, its inverse, and the factor 2^(e_old - e_new) that re-bases sums
__device__ __forceinline__ float f16_scale_of(int e) { return __builtin_bit_cast(float, (unsigned)(254 + F16_TARGET - e) << 23); }
__device__ __forceinline__ float f16_inv_scale_of(int e) { return __builtin_bit_cast(float, (unsigned)(e - F16_TARGET) << 23); }
__device__ __forceinline__ float f16_rebase(int e_old, int e_new) {
    const int d = e_old - e_new;
    return d < -126 ? 0.f : __builtin_bit_cast(float, (unsigned)(127 + d) << 23);
}

CODEPS_STAMP_DECL(conv)

// 16 zero floats in global memory: what a gathered load reads when its tap falls into the zero padding
__device__ __attribute__((aligned(64))) float zero_page[16];

// Gather-table entry of a zero-padding tap: a byte offset past the end of every buffer resource, so the hardware
// range check of buffer_load returns 0 for it (no compare / select / branch in the K loop).
constexpr unsigned GATHER_OOB = 0xFFFF0000u;

// Raw buffer resource (stride 0 -> num_records in bytes) over [base, base + bytes); bytes saturates below GATHER_OOB.
// base and bytes must be wave-uniform (they are functions of blockIdx only); readfirstlane pins them to SGPRs so the
// compiler never has to wrap the loads in a waterfall loop.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const float* base, size_t bytes) {
    const unsigned long long a = reinterpret_cast<unsigned long long>(base);
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    const unsigned n = __builtin_amdgcn_readfirstlane((unsigned)(bytes < (size_t)GATHER_OOB ? bytes : (size_t)GATHER_OOB));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((unsigned long long)hi << 32) | lo), 0, (int)n, 0x00020000);
}

__device__ __forceinline__ int reflect_idx(int i, int n) {
    i = i < 0 ? -i : i;
    return i >= n ? 2 * (n - 1) - i : i;
}

__device__ __forceinline__ float apply_act(float v, int act) {
    if (act == 1) return v > 0.f ? v : 0.f;
    if (act == 2) return v > 0.f ? v : expm1f(v);
    return v;
}

// ---- epilogue extras (ConvP.ex_*).  Per thread: the column quad n .. n + 3 of some rows of ONE M tile whose rows lie in one image.
struct EpiCtx { f32x4 sh, s1, s2, mu, is, ga, be; };

// img: image of the tile (block-uniform); n: first column of this thread's quad (n < p.N)
__device__ __forceinline__ void epi_begin(const ConvP& p, EpiCtx& ec, int img, int n) {
    ec.sh = ec.s1 = ec.s2 = f32x4{0.f, 0.f, 0.f, 0.f};
    ec.mu = ec.be = f32x4{0.f, 0.f, 0.f, 0.f};
    ec.is = ec.ga = f32x4{1.f, 1.f, 1.f, 1.f};
    if (p.ex_gate_act == 3 && n < p.N) {
        int g = 0;
#pragma unroll
        for (int i = 1; i < 8; ++i) g += (i < p.ex_bn_ng && img >= p.ex_bn_b0[i]) ? 1 : 0;
        ec.mu = *reinterpret_cast<const f32x4*>(p.ex_bn_mean + (size_t)g * p.N + n);
        ec.is = *reinterpret_cast<const f32x4*>(p.ex_bn_invstd + (size_t)g * p.N + n);
        if (p.ex_bn_relu && !p.ex_gate) {
            ec.ga = *reinterpret_cast<const f32x4*>(p.ex_bn_gamma + n);
            ec.be = *reinterpret_cast<const f32x4*>(p.ex_bn_beta + n);
        }
    }
}

// What a gate reads from memory at out[idx] (the BatchNorm's input, the gate tensor).  The kernels fetch these for ALL rows of an
// epilogue pass before the pass's first store: the stores go to `out`, which the compiler cannot prove distinct from the gate tensors, so
// loads written inside the store loop are issued one row at a time, each behind the previous row's store -- a memory latency per row
// (8 rows x 2 passes per block: most of the 35-40 us a BatchNorm-gate data gradient cost over the plain one).
struct EpiPre { f32x4 x, g; };
__device__ __forceinline__ EpiPre epi_prefetch(const ConvP& p, size_t idx, bool ok) {
    EpiPre e{f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    if (!ok) return e;
    if (p.ex_gate_act == 3) {
        e.x = *reinterpret_cast<const f32x4*>(p.ex_bn_x + idx);
        if (p.ex_bn_relu && p.ex_gate) e.g = *reinterpret_cast<const f32x4*>(p.ex_gate + idx);
    } else if (p.ex_gate_act) {
        e.g = *reinterpret_cast<const f32x4*>(p.ex_gate + idx);
    }
    return e;
}

// v = the value about to be stored at out[idx]: gate it, account for it in the tile's statistics
__device__ __forceinline__ f32x4 epi_apply(const ConvP& p, EpiCtx& ec, f32x4 v, const EpiPre& pre) {
    if (p.ex_gate_act == 1 || p.ex_gate_act == 2) {
        const f32x4 g = pre.g;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= g[e] > 0.f ? 1.f : (p.ex_gate_act == 2 ? g[e] + 1.f : 0.f);      // = act_bwd_kernel's product
    }
    if (p.ex_gate_act == 3) {
        const f32x4 xh = (pre.x - ec.mu) * ec.is;
        if (p.ex_bn_relu) {
            const f32x4 yy = p.ex_gate ? pre.g : xh * ec.ga + ec.be;    // bn_bwd_reduce_mg_kernel's mask
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = yy[e] > 0.f ? v[e] : 0.f;
        }
        if (p.ex_stat == 3) { ec.s1 += v; ec.s2 += v * xh; }
    }
    if (p.ex_stat == 1) { const f32x4 d = v - ec.sh; ec.s1 += d; ec.s2 += d * d; }
    if (p.ex_stat == 2) ec.s1 += v;
    return v;
}

// After the last store: the tile's statistics -> p.ex_part[tile][rows][N].  Threads tid = k * V4 + c4 (k < RPASS) hold column quad c4;
// `red` = 2 * (threads of the block) f32x4 of LDS nobody reads any more (a barrier is taken first).  Fixed summation order.
__device__ __forceinline__ void epi_flush(const ConvP& p, const EpiCtx& ec, float* red, int tid, int V4, int RPASS, int tile, int n) {
    if (!p.ex_stat) return;
    const int NT = V4 * RPASS;                                     // threads of the block (256, or 512 in the wave-specialised kernel)
    __syncthreads();
    f32x4* r = reinterpret_cast<f32x4*>(red);
    r[tid] = ec.s1; r[NT + tid] = ec.s2;
    __syncthreads();
    if (tid < V4 && n < p.N) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < RPASS; ++k) { a += r[k * V4 + tid]; b += r[NT + k * V4 + tid]; }
        const int rows = p.ex_stat == 1 ? 3 : (p.ex_stat == 2 ? 1 : 2);
        float* dst = p.ex_part + ((size_t)(p.ex_tile0 + tile) * rows) * p.N + n;
        if (p.ex_stat == 1) {
            *reinterpret_cast<f32x4*>(dst) = ec.sh; *reinterpret_cast<f32x4*>(dst + p.N) = a; *reinterpret_cast<f32x4*>(dst + 2 * (size_t)p.N) = b;
        } else {
            *reinterpret_cast<f32x4*>(dst) = a;
            if (p.ex_stat == 3) *reinterpret_cast<f32x4*>(dst + p.N) = b;
        }
    }
}

// The extras are compiled into the EX = true instantiation of a kernel only: with them in every instantiation the epilogue, not the
// K loop, set the register count (conv_igemm_kernel 128 x 128: 166 -> 176 registers, 3 -> 2 waves per SIMD).
__device__ __forceinline__ f32x4 epi_apply(const ConvP& p, EpiCtx& ec, f32x4 v, size_t idx) { return epi_apply(p, ec, v, epi_prefetch(p, idx, true)); }
template <bool EX>
__device__ __forceinline__ f32x4 epi_apply_t(const ConvP& p, EpiCtx& ec, f32x4 v, size_t idx) {
    if constexpr (EX) return epi_apply(p, ec, v, idx);
    else return v;
}
template <bool EX>
__device__ __forceinline__ f32x4 epi_apply_t(const ConvP& p, EpiCtx& ec, f32x4 v, const EpiPre& pre) {
    if constexpr (EX) return epi_apply(p, ec, v, pre);
    else return v;
}

// XCD-aware bijective block remap (guide T1): blocks with equal blockIdx % 8 share an XCD.
__device__ __forceinline__ int xcd_remap(int bid, int nblk) {
    const int q = nblk / 8, r = nblk % 8, x = bid % 8, i = bid / 8;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
}

// The parity class of this block: the launch's (par == 1: one launch per class) or blockIdx.z's (par == 2).  Read-only on purpose:
// WRITING the selected class back into the kernel's by-value ConvP made the compiler keep the whole struct in scratch (400 bytes per
// lane in every data-gradient instantiation, every data-gradient launch 30-50 % slower -- measured on the pre-training configurations).
struct ParSel { int py, px, ky0, kx0, nky, nkx, tile_off; };
__device__ __forceinline__ ParSel parity_class(const ConvP& p) {
    ParSel s{p.py, p.px, p.ky0, p.kx0, p.nky, p.nkx, 0};
    if (p.par == 2) {
        const int c = blockIdx.z;
#define PCLS(k) (c == 0 ? p.pcls[0][k] : c == 1 ? p.pcls[1][k] : c == 2 ? p.pcls[2][k] : p.pcls[3][k])
        s.py = PCLS(0); s.px = PCLS(1); s.ky0 = PCLS(2); s.kx0 = PCLS(3); s.nky = PCLS(4); s.nkx = PCLS(5);
#undef PCLS
        s.tile_off = c * p.n_mt;
    }
    return s;
}

// Gather table of one block of BM rows (see conv_igemm_kernel): tab[source][tap][row] = byte offset of the pixel that row
// reads through that tap, relative to the first image the block touches (GATHER_OOB = zero padding / row past M), plus
// the buffer resources of the source(s) rebased to that image.  Ends with a barrier.
template <int MODE, int BM>
__device__ __forceinline__ void build_gather(const ConvP& p, int m0, int ntap, unsigned* tab, const float* a0, const float* a1,
                                             __amdgpu_buffer_rsrc_t& rs0, __amdgpu_buffer_rsrc_t& rs1, const ParSel pc) {
    const int tid = threadIdx.x;
    const bool two_src = MODE == MODE_FWD && p.C1 > 0;
    const bool parc = MODE == MODE_DGRAD && p.par;
    const bool upd = MODE == MODE_DGRAD && p.up0 && p.src == 0;
    const int HWm = (MODE == MODE_FWD) ? p.Ho * p.Wo : (parc ? p.Hc * p.Wc : (upd ? (p.H / 2) * (p.W / 2) : p.H * p.W));
    const int Wm = (MODE == MODE_FWD) ? p.Wo : (parc ? p.Wc : (upd ? p.W / 2 : p.W));
    const int b_first = m0 / HWm;                                // block-uniform: offsets stay < 4 GB whatever the tensor size
    // source geometry: fwd source 0 (maybe at half resolution), fwd source 1, or dZ for dgrad
    const int H0 = (MODE == MODE_FWD) ? (p.up0 ? p.H / 2 : p.H) : p.Ho, W0 = (MODE == MODE_FWD) ? (p.up0 ? p.W / 2 : p.W) : p.Wo;
    const int cs0 = (MODE == MODE_FWD) ? p.C0 : p.Co;
    for (int e = tid; e < ntap * BM; e += 256) {
        const int row = e % BM, tap = e / BM;
        const int m = m0 + row;
        unsigned v0 = GATHER_OOB, v1 = GATHER_OOB;
        if (m < p.M) {
            const int bb = m / HWm - b_first, rem = m % HWm;
            const int y = rem / Wm, x = rem % Wm;
            if (MODE == MODE_FWD) {
                const int ky = tap / p.KW, kx = tap % p.KW;
                int iy = y * p.stride - p.pad + ky, ix = x * p.stride_w - p.pad_w + kx;
                if (p.pad_mode == 1) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
                if (iy >= 0 && iy < p.H && ix >= 0 && ix < p.W) {
                    v1 = (unsigned)((bb * p.H + iy) * p.W + ix) * (unsigned)(p.C1 * 4);
                    v0 = p.up0 ? (unsigned)((bb * H0 + (iy >> 1)) * W0 + (ix >> 1)) * (unsigned)(cs0 * 4)      // fused nearest x2 of source 0
                       : p.pitch0 ? (unsigned)((bb * p.H + iy) * p.wrow0 + ix) * (unsigned)(p.pitch0 * 4)      // overlapping pixels
                               : (unsigned)((bb * p.H + iy) * p.W + ix) * (unsigned)(cs0 * 4);
                }
            } else {
                // dgrad: the output pixel (ty, tx) that read this input pixel through tap (ky, kx)
                int ky, kx, qy = 0, qx = 0;
                if (parc) { ky = pc.ky0 + 2 * (tap / pc.nkx); kx = pc.kx0 + 2 * (tap % pc.nkx); }
                else if (upd) {
                    const int q = tap / (p.KH * p.KW), t2 = tap % (p.KH * p.KW);
                    qy = q >> 1; qx = q & 1; ky = t2 / p.KW; kx = t2 % p.KW;
                } else { ky = tap / p.KW; kx = tap % p.KW; }
                int iy = y, ix = x;
                if (parc) { iy = 2 * iy + pc.py; ix = 2 * ix + pc.px; }
                if (upd) { iy = 2 * iy + qy; ix = 2 * ix + qx; }
                int ty = iy + p.pad - ky, tx = ix + p.pad - kx;
                bool ok = ty >= 0 && tx >= 0;
                if (p.stride == 2) { ok = ok && !(ty & 1) && !(tx & 1); ty >>= 1; tx >>= 1; }
                if (ok && ty < p.Ho && tx < p.Wo) v0 = (unsigned)((bb * p.Ho + ty) * p.Wo + tx) * (unsigned)(cs0 * 4);
            }
        }
        tab[e] = v0;
        if (two_src) tab[ntap * BM + e] = v1;
    }
    __syncthreads();
    const int Btot = p.M > 0 ? (p.M + HWm - 1) / HWm : 1;        // images addressed by the rows of this launch (= batch)
    const size_t img0 = (MODE == MODE_FWD && p.pitch0) ? (size_t)p.H * p.wrow0 * p.pitch0 : (size_t)H0 * W0 * cs0, img1 = (size_t)p.H * p.W * p.C1;
    rs0 = make_rsrc(a0 + (size_t)b_first * img0, (size_t)(Btot - b_first) * img0 * 4);
    rs1 = two_src ? make_rsrc(a1 + (size_t)b_first * img1, (size_t)(Btot - b_first) * img1 * 4) : rs0;
}

// One implicit-GEMM kernel for forward and dgrad.
//   A rows: pixels.  B rows: GEMM columns n (weights packed [n][tap][c], c contiguous).
template <int MODE, int WM, int WN, int TM, int TN, int BK, int NBUF, int NP = 0, bool EX = false>
__global__ __launch_bounds__(256) void conv_igemm_kernel(ConvP p, const float* __restrict__ a0,
                                                         const float* __restrict__ a1, const float* __restrict__ wq,
                                                         const float* __restrict__ scale,
                                                         const float* __restrict__ shift,
                                                         const float* __restrict__ residual, float* __restrict__ out) {
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
    static_assert(NP == 0 || ((BK == 32 || (BK == 16 && NP == 3)) && NBUF == 1), "split-precision variant: BK = 32 (or 16 with pre-split weights), single LDS stage");
    // LDS row (floats).  f32 operands: BK + 4 (padded).  Split operands at BK = 32 (round 4): UNPADDED rows of 192 bytes = [piece][4 k
    // groups of 16 bytes] with the k group stored at position kg ^ ((row >> 2) & 3).  With the 208-byte padded rows of rounds 2-3 the
    // staging `ds_write_b128` (8 contiguous lanes = 2 rows x 4 chunks) hit one 16-byte slot twice per lane group: bank-conflict cycles
    // = 10-13 % of these kernels' CU cycles (PMC, round 4).  At a 192-byte pitch two consecutive rows fill all eight slots, and the
    // swizzle spreads the fragment reads (lane = row, 16 rows per ds_read_b128 lane group, 12 r mod 16 takes four values only) over
    // all sixteen -- both conflict-free under the documented lane groups (MI355X_MICROARCH.md, LDS); 8 % less LDS per block.
    // NP = 2 (round 6): TWO fp16 pieces of x 2^k (split_f16; block-local running scale for the gathered operand, the pack's per-tensor scale for
    // the weights), rows of 128 bytes = [piece][4 k groups]: besides the k-group swizzle the two pieces swap places in rows 2, 3 (mod 4), so that
    // the 16 lanes of a staging store (4 rows x 4 chunks) and the 16 rows of a fragment-read lane group each cover all sixteen 16-byte slots.
    constexpr bool H16 = NP == 2;
    constexpr int EB = NP * 2;                        // bytes per element of the pre-split weights
    constexpr bool SWZ = (CODEPS_IGEMM_SWZ || H16) && NP > 0 && BK == 32;
    constexpr int LDK = NP == 0 ? BK + 4 : (SWZ ? NP * BK / 2 : (NP * BK + 8) / 2);
    constexpr int KPT = NP > 0 ? 8 : 4;               // consecutive k values staged per thread and row (split kernel: 8, so that each bf16
                                                      // piece goes to LDS as one 16-B write)
    constexpr int SUB = KPT / 4;                      // 16-B global loads per staged chunk
    constexpr int CPR = BK / KPT;                     // chunks per row
    constexpr int RPP = 256 / CPR;                    // rows covered per pass of the 256 threads
    constexpr int APASS = (BM + RPP - 1) / RPP, BPASS = (BN + RPP - 1) / RPP;
    extern __shared__ __attribute__((aligned(16))) float smem[];
    // NBUF = 2: LDS double buffer, one barrier per K-step.  NBUF = 1: the next stage lives only in registers, two
    // barriers per K-step, half the LDS -> twice the co-resident blocks per CU (4 waves per SIMD hide each other's
    // load / store / barrier phases behind MFMAs).
    float* As = smem;                                 // [NBUF][BM][LDK]
    float* Bs = smem + NBUF * BM * LDK;               // [NBUF][BN][LDK]
    CODEPS_STAMP_BEGIN();
    const ParSel pc = parity_class(p);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    const int logical = xcd_remap(blockIdx.x, p.n_mt * p.n_nt);
    const int nt = logical % p.n_nt, mt = logical / p.n_nt;
    const int m0 = mt * BM, n0 = nt * BN;

    // ---- K-step enumeration: (tap, source segment, channel chunk)
    const int ntap = (MODE == MODE_DGRAD && p.par) ? pc.nky * pc.nkx
                   : ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW);
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;          // channels per tap in the packed weights
    const int steps_per_tap = Kc / BK;
    const int nsteps = ntap * steps_per_tap;

    // ---- gather table (built once per block): tab[source][tap][row] = BYTE offset of the pixel that row reads through
    //      that tap, relative to the first image this block touches; GATHER_OOB = zero padding.  The K loop then costs
    //      one broadcast LDS read + one add per 16-B buffer_load (whose range check supplies the zeros) instead of the
    //      div / mod / bounds / reflect / upsample arithmetic and its branches (measured: with the address arithmetic in
    //      the loop the MFMA pipe idled 20-45 % of the time behind VALU work).
    unsigned* tab = reinterpret_cast<unsigned*>(smem + NBUF * (BM + BN) * LDK);
    __amdgpu_buffer_rsrc_t rs0, rs1;
    // in_aff (forward only; tiles lie inside one image): the image's [mean | invstd | gamma | beta][Ct] behind the table and the maxima slot
    float* aff = reinterpret_cast<float*>(tab + ((MODE == MODE_FWD && p.C1 > 0) ? 2 : 1) * ntap * BM + 4);
    if (MODE == MODE_FWD && p.in_aff) {
        const float* src = p.in_aff + (size_t)(m0 / (p.Ho * p.Wo)) * 4 * p.Ct;
        for (int e = tid; e < p.Ct; e += 256) *reinterpret_cast<f32x4*>(aff + e * 4) = *reinterpret_cast<const f32x4*>(src + e * 4);
    }
    build_gather<MODE, BM>(p, m0, ntap, tab, a0, a1, rs0, rs1, pc);

    // ---- per-thread staging roles: 16-B chunk `chunk` of rows rbase + RPP * i
    const int chunk = tid % CPR, rbase = tid / CPR;
    const int wchunk = SWZ ? (chunk ^ ((rbase >> 2) & 3)) : chunk;       // where this thread's k group goes inside an LDS row (RPP % 16 == 0)
    constexpr bool AGUARD = (BM % RPP) != 0, BGUARD = (BN % RPP) != 0;
    // B rows (weights): row n = n0 + rbase + RPP*i, K-contiguous; rows past N are clamped (their columns are never stored)
    const size_t wrow = (MODE == MODE_FWD) ? (size_t)p.KH * p.KW * p.Ct : (size_t)p.KH * p.KW * p.Co;     // floats per packed weight row
    // 3-piece arithmetic: the weights arrive pre-split (6 bytes per element, laid out like an LDS row), so the B operand is
    // staged with copies only -- every weight element would otherwise be converted again by each of the M / BM row tiles
    constexpr bool BPRE = NP >= 2;
    constexpr int BREGS = BPRE ? NP : SUB;            // 16-byte registers per staged B row chunk
    const __amdgpu_buffer_rsrc_t rsB = BPRE ? make_rsrc(static_cast<const float*>(H16 ? p.w2 : p.w3), (size_t)p.N * wrow * EB) : make_rsrc(wq, (size_t)p.N * wrow * 4);
    unsigned boff[BPASS];
#pragma unroll
    for (int i = 0; i < BPASS; ++i) {
        const size_t row = (size_t)min(n0 + rbase + RPP * i, p.N - 1) * wrow;
        boff[i] = BPRE ? (unsigned)(row * EB + chunk * 16) : (unsigned)((row + chunk * KPT) * 4);
    }

    f32x4 areg[APASS * SUB], breg[BPASS * BREGS];
    int areg_c = 0;                                           // channel offset of the tile `areg` holds (in_aff)

    auto load_step = [&](int step) {
        const int tap = step / steps_per_tap;
        const int cstep = (step - tap * steps_per_tap) * BK;   // channel offset within the tap
        areg_c = cstep;
        // ---- A operand
        const bool s1 = MODE == MODE_FWD && cstep >= p.C0;        // which source this chunk belongs to
        const __amdgpu_buffer_rsrc_t rs = s1 ? rs1 : rs0;
        const unsigned coff = (unsigned)((s1 ? cstep - p.C0 : cstep) + chunk * KPT) * 4u;
        const unsigned* t = tab + ((s1 ? ntap : 0) + tap) * BM + rbase;
#pragma unroll
        for (int i = 0; i < APASS; ++i) {
            const unsigned off = t[(AGUARD && rbase + RPP * i >= BM) ? 0 : RPP * i];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
                areg[i * SUB + u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + coff + 16 * u, 0, 0));
        }
        // ---- B operand (packed weights, K contiguous)
        int koff;
        if (MODE == MODE_DGRAD && p.par) koff = ((pc.ky0 + 2 * (tap / pc.nkx)) * p.KW + pc.kx0 + 2 * (tap % pc.nkx)) * Kc + cstep;
        else if (MODE == MODE_DGRAD && p.up0 && p.src == 0) koff = ((tap % (p.KH * p.KW)) * Kc) + cstep;
        else koff = tap * Kc + cstep;
#pragma unroll
        for (int i = 0; i < BPASS; ++i)
#pragma unroll
            for (int u = 0; u < BREGS; ++u)
                breg[i * BREGS + u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    rsB, BPRE ? boff[i] + (unsigned)(koff >> 5) * (unsigned)(32 * EB) + (unsigned)(koff & 31) * 2u + 64 * u : boff[i] + (unsigned)koff * 4u + 16 * u, 0, 0));
    };
    // in_aff: the tile in `areg` is BatchNorm's INPUT -- normalise + ReLU in registers (bn_norm_relu: the expression of bn_apply_mg_kernel, so
    // the product equals the one over the materialised tensor bit for bit).  1x1 / no padding only: every gathered element is a real pixel.
    auto transform_a = [&]() {
        if (MODE == MODE_FWD && p.in_aff) {
            const float* a = aff + areg_c + chunk * KPT;
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const f32x4 mu = *reinterpret_cast<const f32x4*>(a + 4 * u), is = *reinterpret_cast<const f32x4*>(a + p.Ct + 4 * u);
                const f32x4 ga = *reinterpret_cast<const f32x4*>(a + 2 * p.Ct + 4 * u), be = *reinterpret_cast<const f32x4*>(a + 3 * p.Ct + 4 * u);
#pragma unroll
                for (int i = 0; i < APASS; ++i) areg[i * SUB + u] = bn_norm_relu(areg[i * SUB + u], mu, is, ga, be);
            }
        }
    };
    // NP = 2: the exponent of the largest magnitude of the gathered tile in `areg` -> amax_slot[wave] (read behind the next barrier)
    int* amax_slot = reinterpret_cast<int*>(tab + ((MODE == MODE_FWD && p.C1 > 0) ? 2 : 1) * ntap * BM);
    auto publish_amax = [&]() {
        if constexpr (H16) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < APASS * SUB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(areg[i][e]));
            const int ex = wave_max_exponent(m);
            if (lane == 0) amax_slot[wave] = ex;
        }
    };
    float a_scale = 1.f;
    const int psw = H16 ? (rbase >> 1) & 1 : 0;        // NP = 2: rows 2, 3 (mod 4) keep their pieces in swapped places (RPP % 4 == 0)
    auto store_step = [&](int buf) {
        float* Ab = As + buf * BM * LDK;
        float* Bb = Bs + buf * BN * LDK;
#pragma unroll
        for (int i = 0; i < APASS; ++i)
            if (!AGUARD || rbase + RPP * i < BM) {
                if constexpr (NP == 0) {
                    *reinterpret_cast<f32x4*>(Ab + (rbase + RPP * i) * LDK + chunk * 4) = areg[i];
                } else {                                     // row = [piece][32 bf16]; this thread's 8 k values of every piece: one b128 each
                    u16x4 lo[NP > 0 ? NP : 1], hi[NP > 0 ? NP : 1];
                    if constexpr (H16) {
                        split_f16(areg[i * SUB], a_scale, lo[0], lo[1]);
                        split_f16(areg[i * SUB + SUB - 1], a_scale, hi[0], hi[1]);
                    } else {
                        split_bf16<(NP > 0 ? NP : 1)>(areg[i * SUB], lo);
                        split_bf16<(NP > 0 ? NP : 1)>(areg[i * SUB + SUB - 1], hi);
                    }
                    unsigned short* row = reinterpret_cast<unsigned short*>(Ab + (rbase + RPP * i) * LDK);
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        *reinterpret_cast<i32x4*>(row + (q ^ psw) * BK + wchunk * 8) = pack8(lo[q], hi[q]);
                }
            }
#pragma unroll
        for (int i = 0; i < BPASS; ++i)
            if (!BGUARD || rbase + RPP * i < BN) {
                if constexpr (NP == 0) {
                    *reinterpret_cast<f32x4*>(Bb + (rbase + RPP * i) * LDK + chunk * 4) = breg[i];
                } else if constexpr (BPRE) {
                    unsigned short* row = reinterpret_cast<unsigned short*>(Bb + (rbase + RPP * i) * LDK);
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        *reinterpret_cast<i32x4*>(row + (q ^ psw) * BK + wchunk * 8) = __builtin_bit_cast(i32x4, breg[i * BREGS + q]);
                } else {
                    u16x4 lo[NP > 0 ? NP : 1], hi[NP > 0 ? NP : 1];
                    split_bf16<(NP > 0 ? NP : 1)>(breg[i * SUB], lo);
                    split_bf16<(NP > 0 ? NP : 1)>(breg[i * SUB + SUB - 1], hi);
                    unsigned short* row = reinterpret_cast<unsigned short*>(Bb + (rbase + RPP * i) * LDK);
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        *reinterpret_cast<i32x4*>(row + q * BK + wchunk * 8) = pack8(lo[q], hi[q]);
                }
            }
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int s_begin = p.ksplit > 1 ? (int)blockIdx.y * p.ksteps : 0;
    const int s_end = p.ksplit > 1 ? min(nsteps, s_begin + p.ksteps) : nsteps;
    // NP = 2: the running maximum exponent of the gathered tiles -> the scale of the next tile's split; when it grows the sums so far are
    // multiplied by the exact ratio.  Called between the barrier that publishes the waves' maxima and the tile's LDS stores.
    int run_e = F16_EMIN;
    auto rescale = [&]() {
        if constexpr (H16) {
            const i32x4 pe = *reinterpret_cast<const i32x4*>(amax_slot);
            const int e_new = __builtin_amdgcn_readfirstlane(max(max(max(pe[0], pe[1]), max(pe[2], pe[3])), run_e));
            if (e_new != run_e) {
                const float rb = f16_rebase(run_e, e_new);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] *= rb;
                run_e = e_new;
            }
            a_scale = f16_scale_of(run_e);
        }
    };
    load_step(s_begin);
    transform_a();
    if constexpr (H16) { publish_amax(); __syncthreads(); rescale(); }
    store_step(0);
    __syncthreads();

    const int lrow = lane & 31, lhalf = lane >> 5;
    for (int step = s_begin; step < s_end; ++step) {
        const int buf = NBUF == 2 ? ((step - s_begin) & 1) : 0;
        CODEPS_STAMP_PHASE_START();
        if (step + 1 < s_end && CODEPS_ABLATE < 1) load_step(step + 1);           // global loads in flight during the MFMAs
        const float* Ab = As + buf * BM * LDK + (wm * TM * 32 + lrow) * LDK;
        const float* Bb = Bs + buf * BN * LDK + (wn * TN * 32 + lrow) * LDK;
        if constexpr (NP == 0) {
#pragma unroll
            for (int g = 0; g < BK / 8; ++g) {
                f32x4 af[TM], bf[TN];
                const int fo = (2 * g + lhalf) * 4;               // lanes < 32 / >= 32 take k and k + 4 of each 8-deep group
#pragma unroll
                for (int i = 0; i < TM; ++i) af[i] = *reinterpret_cast<const f32x4*>(Ab + i * 32 * LDK + fo);
#pragma unroll
                for (int j = 0; j < TN; ++j) bf[j] = *reinterpret_cast<const f32x4*>(Bb + j * 32 * LDK + fo);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(af[i][e], bf[j][e], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_s_setprio(0);
            }
        } else {
            // v_mfma_f32_32x32x16_bf16: lane (row = lane % 32, half = lane / 32) holds the 8 consecutive k values 8 * half .. of a
            // 16-deep chunk; per chunk the products p_a * p_b with a + b < NP, smallest terms first
#pragma unroll
            for (int kc = 0; kc < BK / 16; ++kc) {
                typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
                frag_t af[TM][NP > 0 ? NP : 1], bf[TN][NP > 0 ? NP : 1];
                const int pr = H16 ? (lrow >> 1) & 1 : 0;
                // halfword offset of this lane's k group inside a piece (swizzled layout: group (2 kc + half) ^ ((row >> 2) & 3))
                const int ho = SWZ ? (((kc * 2 + lhalf) ^ ((lrow >> 2) & 3)) * 8) : kc * 16 + lhalf * 8;
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        af[i][q] = *reinterpret_cast<const frag_t*>(reinterpret_cast<const unsigned short*>(Ab + i * 32 * LDK) + (q ^ pr) * BK + ho);
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        bf[j][q] = *reinterpret_cast<const frag_t*>(reinterpret_cast<const unsigned short*>(Bb + j * 32 * LDK) + (q ^ pr) * BK + ho);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                    for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                        for (int i = 0; i < TM; ++i)
#pragma unroll
                            for (int j = 0; j < TN; ++j)
                                if constexpr (H16) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[i][qa], bf[j][ord - qa], acc[i][j], 0, 0, 0);
                                else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[i][qa], bf[j][ord - qa], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_s_setprio(0);
            }
        }
#if CODEPS_ABLATE >= 2
        continue;
#endif
        CODEPS_STAMP_PHASE_A();                               // A: loads issued + fragment reads + MFMAs of this wave
        CODEPS_STAMP_PHASE_START();
        if (step + 1 < s_end) transform_a();
        if (H16 && step + 1 < s_end) publish_amax();          // (the next tile's loads have had the MFMAs to land)
        if (NBUF == 1) __syncthreads();                       // every wave is done reading the single buffer
        if (step + 1 < s_end) { rescale(); store_step(NBUF == 2 ? (buf ^ 1) : 0); }
        __syncthreads();
        CODEPS_STAMP_PHASE_B();                               // B: barrier + (wait for the loads) split + LDS stores + barrier
    }

    // ---- epilogue: accumulators -> LDS tile [BM][BN+4] -> coalesced float4 rows (512 B per 32 lanes at BN = 128),
    //      affine / residual / activation applied on the vectorised side.  (MFMA C layout: lane holds column
    //      n = lane&31 of each 32x32 tile, rows (r&3) + 8*(r>>2) + 4*(lane>>5); stored directly that would be one
    //      128-B segment per half-wave per row.)
    constexpr int LDC = BN + 4;
    float* Cs = smem;                                  // reuses the staging buffers (all waves passed the last barrier)
    constexpr int V4 = BN / 4;                         // float4 per tile row
    constexpr int RPASS = 256 / V4;                    // rows per pass
    const int c4 = tid % V4, r0 = tid / V4;
    const int n = n0 + c4 * 4;
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (MODE == MODE_FWD && n < p.N) {
        if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    }
    EpiCtx ec;
    if constexpr (EX) epi_begin(p, ec, p.ex_img_rows ? m0 / p.ex_img_rows : 0, n);
    if constexpr (H16) {                                      // sums of (x 2^ka)(w 2^kb): back to the operands' units (exact)
        const float inv = f16_inv_scale_of(run_e) * p.w2s[0];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] *= inv;
    }
    // one pass per row-tile index i: staging holds WM*32 rows (keeps the LDS footprint at <= 34 KB so that the
    // K-loop buffers, not the epilogue, decide how many blocks fit on a CU)
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (i > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                Cs[(wm * 32 + (r & 3) + 8 * (r >> 2) + 4 * lhalf) * LDC + (wn * TN + j) * 32 + lrow] = acc[i][j][r];
        // the residual rows of this pass are requested before the barrier: their latency overlaps the LDS round trip (short-K
        // 1x1 layers spend a fifth of a block's life in this epilogue)
        constexpr int NRES = (WM * 32 + RPASS - 1) / RPASS;
        f32x4 resv[NRES];
        EpiPre pre[NRES];                                     // (the gates' tensors: all rows at once, see EpiPre)
        const bool use_res = residual != nullptr && p.ksplit <= 1 && n < p.N;
        auto row_of = [&](int u, int& rr) -> int {            // output row (pixel index) of this thread's u-th row of the pass, -1 = none
            rr = r0 + u * RPASS;
            int m = m0 + ((rr >> 5) * TM + i) * 32 + (rr & 31);
            if (rr >= WM * 32 || m >= p.M) return -1;
            if (MODE == MODE_DGRAD && p.par) {                // class row -> pixel of the full-resolution gradient
                const int bb = m / (p.Hc * p.Wc), rem = m % (p.Hc * p.Wc);
                m = (bb * p.H + 2 * (rem / p.Wc) + pc.py) * p.W + 2 * (rem % p.Wc) + pc.px;
            }
            return m;
        };
        if (use_res || EX) {
#pragma unroll
            for (int u = 0; u < NRES; ++u) {
                int rr;
                const int m = row_of(u, rr);
                const bool live = m >= 0 && p.ksplit <= 1 && n < p.N;
                resv[u] = (use_res && live) ? *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n) : f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (EX) pre[u] = epi_prefetch(p, (size_t)(m < 0 ? 0 : m) * p.N + n, live);
            }
        }
        __syncthreads();
        if constexpr (EX) if (i == 0 && p.ex_stat == 1) ec.sh = *reinterpret_cast<const f32x4*>(Cs + c4 * 4) * sc + sh;     // the tile's first row = the statistics' shift
        if (n < p.N) {
#pragma unroll
            for (int u = 0; u < NRES; ++u) {
                int rr;
                const int m = row_of(u, rr);
                if (m < 0) continue;
                f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * LDC + c4 * 4);
                if (p.ksplit > 1) {                           // raw partial sum of this K slice; splitk_finish_kernel does the rest
                    // (K slices never meet the parity classes: the rows of `part` are the output's rows)
                    *reinterpret_cast<f32x4*>(p.part + ((size_t)blockIdx.y * p.M + m) * p.N + n) = v;
                    continue;
                }
                if (MODE == MODE_FWD) {
                    v = v * sc + sh;
                    if (use_res) v += resv[u];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
                } else if (use_res) {                         // data gradient + the gradient that reached the same tensor by another path
                    v += resv[u];
                }
                *reinterpret_cast<f32x4*>(out + (size_t)m * p.N + n) = epi_apply_t<EX>(p, ec, v, pre[u]);
            }
        }
    }
    if constexpr (EX) epi_flush(p, ec, smem, tid, V4, RPASS, mt + pc.tile_off, n);
    CODEPS_STAMP_END(conv);
}

// ---------------------------------------------------------------------------------- wave-specialised variant (deep K)
// Same GEMM, same 3-piece arithmetic and pre-split weights as conv_igemm_kernel<.., 32, 1, 3>, for launches whose K loop is
// long enough to amortise a block that owns a whole CU: 512 threads = 4 CONSUMER waves (the 2x2 wave grid, fragment reads +
// MFMAs only) + 4 PRODUCER waves (global loads, bf16 split of the activations, LDS writes), one of each per SIMD, LDS double
// buffered, ONE barrier per K-step.  In the 256-thread kernel every wave runs load -> convert -> write -> barrier -> read ->
// MFMA -> barrier in sequence and the matrix pipe idles ~63 % of the time (PMC); here a SIMD's producer wave
// converts and writes K-step s + 1 while its consumer wave multiplies K-step s.
// ARITH 16 (round 6): two fp16 pieces.  A producer wave stages one whole 32-row MFMA tile of the gathered operand (rows 32 w ..), so the
// scale is per ROW TILE: the wave that stages a tile finds its largest exponent alone (no exchange), leaves the running exponent beside the
// tile, and the consumer that multiplies the tile re-bases that row tile's sums when it grew.
template <int MODE, int TN, bool EX = false, int ARITH = 3>
__global__ __launch_bounds__(512) void conv_igemm_ws_kernel(ConvP p, const float* __restrict__ a0, const float* __restrict__ a1,
                                                            const float* __restrict__ scale, const float* __restrict__ shift,
                                                            const float* __restrict__ residual, float* __restrict__ out) {
    constexpr int WM = 2, WN = 2, TM = 2, BK = 32, NP = ARITH == 16 ? 2 : 3;
    constexpr bool H16 = ARITH == 16;
    constexpr int EB = NP * 2;
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
    constexpr int LDK = (NP * BK + 8) / 2;            // floats per LDS row: [piece][32 bf16] + pad
    constexpr int CPR = BK / 8, RPP = 256 / CPR;      // producer threads: 8 consecutive k per thread and row, 64 rows per pass
    constexpr int APASS = BM / RPP, BPASS = BN / RPP;
    extern __shared__ __attribute__((aligned(16))) float smem[];
    float* As = smem;                                 // [2][BM][LDK]
    float* Bs = smem + 2 * BM * LDK;                  // [2][BN][LDK]
    unsigned* tab = reinterpret_cast<unsigned*>(smem + 2 * (BM + BN) * LDK);
    const ParSel pc = parity_class(p);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool producer = wave >= 4;
    const int cw = wave & 3, wm = cw / WN, wn = cw % WN;
    const int logical = xcd_remap(blockIdx.x, p.n_mt * p.n_nt);
    const int nt = logical % p.n_nt, mt = logical / p.n_nt;
    const int m0 = mt * BM, n0 = nt * BN;
    const int ntap = (MODE == MODE_DGRAD && p.par) ? pc.nky * pc.nkx
                   : ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW);
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;
    const int steps_per_tap = Kc / BK;
    const int nsteps = ntap * steps_per_tap;
    __amdgpu_buffer_rsrc_t rs0, rs1;
    build_gather<MODE, BM>(p, m0, ntap, tab, a0, a1, rs0, rs1, pc);
    int* slots = reinterpret_cast<int*>(tab + ((MODE == MODE_FWD && p.C1 > 0) ? 2 : 1) * ntap * BM);      // ARITH 16: [buffer][row tile] running exponents
    int run_e[TM] = {F16_EMIN, F16_EMIN};             // consumer: of its two row tiles; producer: [0] = of the row tile it stages

    const int s_begin = p.ksplit > 1 ? (int)blockIdx.y * p.ksteps : 0;
    const int s_end = p.ksplit > 1 ? min(nsteps, s_begin + p.ksteps) : nsteps;
    const int lrow = lane & 31, lhalf = lane >> 5;

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    if (producer) {
        const int ptid = tid - 256, chunk = ptid % CPR, rbase = ptid / CPR;
        const int pw = wave - 4;
        // rows of the gathered operand this thread stages: passes of 64 rows over the block (three pieces), or the producer wave's own row tile
        const int abase = H16 ? pw * 32 + (lane >> 2) : rbase;
        constexpr int ASTEP = H16 ? 16 : RPP;
        const size_t wrow = (MODE == MODE_FWD) ? (size_t)p.KH * p.KW * p.Ct : (size_t)p.KH * p.KW * p.Co;
        const __amdgpu_buffer_rsrc_t rsB = make_rsrc(static_cast<const float*>(H16 ? p.w2 : p.w3), (size_t)p.N * wrow * EB);
        unsigned boff[BPASS];
#pragma unroll
        for (int i = 0; i < BPASS; ++i) boff[i] = (unsigned)((size_t)min(n0 + rbase + RPP * i, p.N - 1) * wrow * EB + chunk * 16);
        f32x4 areg[APASS * 2], breg[BPASS * NP];
        auto load_step = [&](int step) {
            const int tap = step / steps_per_tap;
            const int cstep = (step - tap * steps_per_tap) * BK;
            const bool s1 = MODE == MODE_FWD && cstep >= p.C0;
            const __amdgpu_buffer_rsrc_t rs = s1 ? rs1 : rs0;
            const unsigned coff = (unsigned)((s1 ? cstep - p.C0 : cstep) + chunk * 8) * 4u;
            const unsigned* t = tab + ((s1 ? ntap : 0) + tap) * BM + abase;
#pragma unroll
            for (int i = 0; i < APASS; ++i) {
                const unsigned off = t[ASTEP * i];
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    areg[i * 2 + u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + coff + 16 * u, 0, 0));
            }
            int koff;
            if (MODE == MODE_DGRAD && p.par) koff = ((pc.ky0 + 2 * (tap / pc.nkx)) * p.KW + pc.kx0 + 2 * (tap % pc.nkx)) * Kc + cstep;
            else if (MODE == MODE_DGRAD && p.up0 && p.src == 0) koff = ((tap % (p.KH * p.KW)) * Kc) + cstep;
            else koff = tap * Kc + cstep;
#pragma unroll
            for (int i = 0; i < BPASS; ++i)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    breg[i * NP + q] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsB, boff[i] + (unsigned)koff * (unsigned)EB + 64 * q, 0, 0));
        };
        auto store_step = [&](int buf) {
            float* Ab = As + buf * BM * LDK;
            float* Bb = Bs + buf * BN * LDK;
            float a_scale = 1.f;
            if constexpr (H16) {                                  // this wave's row tile: largest exponent so far -> scale, left beside the tile
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < APASS * 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(areg[i][e]));
                run_e[0] = max(run_e[0], wave_max_exponent(m));
                a_scale = f16_scale_of(run_e[0]);
                if (lane == 0) slots[buf * 4 + pw] = run_e[0];
            }
#pragma unroll
            for (int i = 0; i < APASS; ++i) {
                u16x4 lo[NP], hi[NP];
                if constexpr (H16) {
                    split_f16(areg[i * 2], a_scale, lo[0], lo[1]);
                    split_f16(areg[i * 2 + 1], a_scale, hi[0], hi[1]);
                } else {
                    split_bf16<NP>(areg[i * 2], lo);
                    split_bf16<NP>(areg[i * 2 + 1], hi);
                }
                unsigned short* row = reinterpret_cast<unsigned short*>(Ab + (abase + ASTEP * i) * LDK);
#pragma unroll
                for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(row + q * BK + chunk * 8) = pack8(lo[q], hi[q]);
            }
#pragma unroll
            for (int i = 0; i < BPASS; ++i) {
                unsigned short* row = reinterpret_cast<unsigned short*>(Bb + (rbase + RPP * i) * LDK);
#pragma unroll
                for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(row + q * BK + chunk * 8) = __builtin_bit_cast(i32x4, breg[i * NP + q]);
            }
        };
        load_step(s_begin);
        store_step(0);
        if (s_begin + 1 < s_end) load_step(s_begin + 1);
        __syncthreads();                                          // stage 0 is visible
        for (int step = s_begin; step < s_end; ++step) {
            const int buf = (step - s_begin) & 1;
            if (step + 1 < s_end) store_step(buf ^ 1);            // the consumers read `buf` meanwhile
            if (step + 2 < s_end) load_step(step + 2);            // stays in flight across the barrier
            __syncthreads();
        }
    } else {
        __syncthreads();
        for (int step = s_begin; step < s_end; ++step) {
            const int buf = (step - s_begin) & 1;
            const float* Ab = As + buf * BM * LDK + (wm * TM * 32 + lrow) * LDK;
            const float* Bb = Bs + buf * BN * LDK + (wn * TN * 32 + lrow) * LDK;
            if constexpr (H16) {                                  // the row tiles' scales of this K-step: re-base a tile's sums when its scale grew (exact)
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const int e_new = __builtin_amdgcn_readfirstlane(slots[buf * 4 + wm * TM + i]);
                    if (e_new != run_e[i]) {
                        const float rb = f16_rebase(run_e[i], e_new);
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] *= rb;
                        run_e[i] = e_new;
                    }
                }
            }
#pragma unroll
            for (int kc = 0; kc < BK / 16; ++kc) {
                typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
                frag_t af[TM][NP], bf[TN][NP];
                const int ho = kc * 16 + lhalf * 8;
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        af[i][q] = *reinterpret_cast<const frag_t*>(reinterpret_cast<const unsigned short*>(Ab + i * 32 * LDK) + q * BK + ho);
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        bf[j][q] = *reinterpret_cast<const frag_t*>(reinterpret_cast<const unsigned short*>(Bb + j * 32 * LDK) + q * BK + ho);
#pragma unroll
                for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                    for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                        for (int i = 0; i < TM; ++i)
#pragma unroll
                            for (int j = 0; j < TN; ++j)
                                if constexpr (H16) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[i][qa], bf[j][ord - qa], acc[i][j], 0, 0, 0);
                                else acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[i][qa], bf[j][ord - qa], acc[i][j], 0, 0, 0);
            }
            __syncthreads();
        }
    }

    // ---- epilogue (as in conv_igemm_kernel; the consumer waves hold the accumulators, all 512 threads move rows)
    constexpr int LDC = BN + 4;
    float* Cs = smem;
    constexpr int V4 = BN / 4, RPASS = 512 / V4;
    const int c4 = tid % V4, r0 = tid / V4;
    const int n = n0 + c4 * 4;
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (MODE == MODE_FWD && n < p.N) {
        if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    }
    EpiCtx ec;
    if constexpr (EX) epi_begin(p, ec, p.ex_img_rows ? m0 / p.ex_img_rows : 0, n);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (i > 0) __syncthreads();
        if (!producer) {
            const float inv = H16 ? f16_inv_scale_of(run_e[i]) * p.w2s[0] : 1.f;      // back to the operands' units (exact)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    Cs[(wm * 32 + (r & 3) + 8 * (r >> 2) + 4 * lhalf) * LDC + (wn * TN + j) * 32 + lrow] = H16 ? acc[i][j][r] * inv : acc[i][j][r];
        }
        __syncthreads();
        if constexpr (EX) if (i == 0 && p.ex_stat == 1) ec.sh = *reinterpret_cast<const f32x4*>(Cs + c4 * 4) * sc + sh;
        if (n < p.N) {
#pragma unroll 2
            for (int rr = r0; rr < WM * 32; rr += RPASS) {
                int m = m0 + ((rr >> 5) * TM + i) * 32 + (rr & 31);
                if (m >= p.M) continue;
                if (MODE == MODE_DGRAD && p.par) {
                    const int bb = m / (p.Hc * p.Wc), rem = m % (p.Hc * p.Wc);
                    m = (bb * p.H + 2 * (rem / p.Wc) + pc.py) * p.W + 2 * (rem % p.Wc) + pc.px;
                }
                f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * LDC + c4 * 4);
                if (p.ksplit > 1) {
                    *reinterpret_cast<f32x4*>(p.part + ((size_t)blockIdx.y * p.M + m) * p.N + n) = v;
                    continue;
                }
                if (MODE == MODE_FWD) {
                    v = v * sc + sh;
                    if (residual) v += *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
                } else if (residual) {
                    v += *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n);
                }
                *reinterpret_cast<f32x4*>(out + (size_t)m * p.N + n) = epi_apply_t<EX>(p, ec, v, (size_t)m * p.N + n);
            }
        }
    }
    if constexpr (EX) epi_flush(p, ec, smem, tid, V4, RPASS, mt + pc.tile_off, n);
}

// ---------------------------------------------------------------------------------- halo-tile variant (3x3, stride 1)
// conv_igemm_kernel stages a 128-pixel x 32-channel activation tile once per TAP: for a 3x3 layer every activation element is
// loaded, split and written to LDS nine times per column tile.  Here the block's 128 output pixels are a 4 x 32 rectangle and
// the 6 x 34 halo rectangle of one 32-channel chunk (of either concat source; nearest x2 of source 0 fused) is staged ONCE; the nine taps read their A fragments from shifted rows
// of it (a tap is a row offset in the [pixel][piece][32] layout: aligned, no gather table).  Only the pre-split weights of
// (tap, chunk) move per K-step, through a double buffer: one barrier per tap.  Same arithmetic, same epilogue.
// MODE_DGRAD (stride 1): input pixel p sums dZ(p + (1 - ky, 1 - kx)) x W[ci][tap][co]: the same kernel with mirrored taps.
// WM x WN waves: 2 x 2 = 4 x 32 output pixels x (64 TN) columns (two blocks per CU at TN = 1); 4 x 1 (round 4) = 8 x 32 pixels x 32
// columns for the layers with <= 32 output channels (the decoders' half-resolution stage), which the generic kernel ran at 84-119 TFLOP/s.
template <int MODE, int TN, int WM = 2, int WN = 2, bool EX = false, int ARITH = 3>
__global__ __launch_bounds__(256) void conv_halo3_kernel(ConvP p, const float* __restrict__ a0, const float* __restrict__ a1,
                                                         const float* __restrict__ scale, const float* __restrict__ shift,
                                                         const float* __restrict__ residual, float* __restrict__ out) {
    constexpr int TM = 2, BK = 32, NP = ARITH == 16 ? 2 : 3;       // ARITH 16: two fp16 pieces, block-local scales (see split_f16)
    constexpr bool H16 = ARITH == 16;
    constexpr int EB = NP * 2, SEGD = NP * 4;                      // bytes per pre-split weight element; 16-byte segments per (row, K group)
    constexpr int TH = 2 * WM, TW = 32, HH = TH + 2, HW = TW + 2, HPIX = HH * HW;  // WM = 2: 128 outputs, 204 halo pixels; WM = 4: 256 / 340
    constexpr int BN = 32 * WN * TN;
    constexpr int LDK = (NP * BK + 8) / 2;                                        // floats per LDS row
    constexpr int LDKA = CODEPS_HALO_SWZ ? LDK + 4 : LDK;                         // activation rows: 224 bytes (conv_halo3r_kernel explains)
    constexpr int APASS = (HPIX * 4 + 255) / 256;                                 // (pixel, 8-channel chunk) tasks per thread
    extern __shared__ __attribute__((aligned(16))) float smem[];
    float* As = smem;                                  // [HPIX][LDKA]
    float* Bs = smem + HPIX * LDKA;                    // [2][BN][LDK]
    int* amax_slot = reinterpret_cast<int*>(Bs + 2 * BN * LDK);        // ARITH 16: the waves' maximum exponents of the activation tile in flight
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    const int logical = xcd_remap(blockIdx.x, p.n_mt * p.n_nt);
    const int nt = logical % p.n_nt, mt = logical / p.n_nt;
    const int n0 = nt * BN;
    const int Hm = (MODE == MODE_FWD) ? p.Ho : p.H, Wm = (MODE == MODE_FWD) ? p.Wo : p.W;       // = input size (stride 1, pad 1)
    const int tiles_x = Wm / TW, tiles_y = Hm / TH;
    const int b = mt / (tiles_x * tiles_y), tr = mt % (tiles_x * tiles_y);
    const int y0 = (tr / tiles_x) * TH, x0 = (tr % tiles_x) * TW;
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;                                           // channels of the staged tensor
    const int nchunks = Kc / BK;
    // forward: source 0 (C0 channels, optionally at half resolution: nearest x2 fused into the load) ++ source 1 (C1 channels)
    const bool up = MODE == MODE_FWD && p.up0;
    const int H0 = up ? Hm / 2 : Hm, W0 = up ? Wm / 2 : Wm;
    const int cs0 = (MODE == MODE_FWD) ? p.C0 : p.Co;
    const float* img0 = a0 + (size_t)b * H0 * W0 * cs0;
    const float* img1 = (MODE == MODE_FWD && p.C1 > 0) ? a1 + (size_t)b * Hm * Wm * p.C1 : nullptr;

    // A staging roles
    const int achunk = tid & 3;
    // B staging roles: a (tap, chunk) row of the pre-split pack is 192 contiguous bytes = 12 16-byte segments, and so is its LDS
    // row ([piece][32]): task t = tid + 256 i copies segment t % 12 of row t / 12 -- twelve neighbouring lanes move one row, so
    // both the global read and the LDS write are contiguous (the 4-lanes-per-row mapping left the writes on a 2-way bank conflict)
    constexpr int BTASK = (BN * SEGD + 255) / 256;                                   // (BN = 32: 384 segments, the second pass half empty)
    const size_t wrow = (size_t)9 * Kc;
    const __amdgpu_buffer_rsrc_t rsB = make_rsrc(static_cast<const float*>(H16 ? p.w2 : p.w3), (size_t)p.N * wrow * EB);
    unsigned boff[BTASK], bdst[BTASK];
#pragma unroll
    for (int i = 0; i < BTASK; ++i) {
        const int t = min(tid + 256 * i, BN * SEGD - 1), row = t / SEGD, seg = t % SEGD;        // (surplus lanes repeat the last segment: same data, same slot)
        boff[i] = (unsigned)((size_t)min(n0 + row, p.N - 1) * wrow * EB + seg * 16);
        bdst[i] = (unsigned)(row * LDK * 4 + (seg ^ (CODEPS_HALO_SWZ ? (((row >> 2) ^ (row >> 3)) & 1) : 0)) * 16);    // k groups of rows 4 .. 11 swapped pairwise
    }

    f32x4 areg[APASS * 2], breg[BTASK];
    auto load_a = [&](int chunk) {
        const int cstep = chunk * BK;
        const bool s1 = MODE == MODE_FWD && cstep >= p.C0;
        const float* base = s1 ? img1 + (cstep - p.C0) + achunk * 8 : img0 + cstep + achunk * 8;
        const int cs = s1 ? p.C1 : cs0, ws = s1 ? Wm : W0, sh = (!s1 && up) ? 1 : 0;
#pragma unroll
        for (int i = 0; i < APASS; ++i) {
            const int pos = (tid >> 2) + 64 * i;
            const int iy = y0 + pos / HW - 1, ix = x0 + pos % HW - 1;
            const bool ok = pos < HPIX && iy >= 0 && iy < Hm && ix >= 0 && ix < Wm;
            const float* src = base + ((size_t)(iy >> sh) * ws + (ix >> sh)) * cs;
            areg[i * 2] = ok ? *reinterpret_cast<const f32x4*>(src) : f32x4{0.f, 0.f, 0.f, 0.f};
            areg[i * 2 + 1] = ok ? *reinterpret_cast<const f32x4*>(src + 4) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    auto publish_amax = [&]() {                                   // ARITH 16 (as in conv_halo3r_kernel)
        if constexpr (H16) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < APASS * 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(areg[i][e]));
            const int ex = wave_max_exponent(m);
            if (lane == 0) amax_slot[wave] = ex;
        }
    };
    float a_scale = 1.f;
    auto store_a = [&]() {
#pragma unroll
        for (int i = 0; i < APASS; ++i) {
            const int pos = (tid >> 2) + 64 * i;
            if (pos >= HPIX) continue;
            u16x4 lo[NP], hi[NP];
            if constexpr (H16) {
                split_f16(areg[i * 2], a_scale, lo[0], lo[1]);
                split_f16(areg[i * 2 + 1], a_scale, hi[0], hi[1]);
            } else {
                split_bf16<NP>(areg[i * 2], lo);
                split_bf16<NP>(areg[i * 2 + 1], hi);
            }
            unsigned short* row = reinterpret_cast<unsigned short*>(As + pos * LDKA);
#pragma unroll
            for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(row + q * BK + achunk * 8) = pack8(lo[q], hi[q]);
        }
    };
    auto load_b = [&](int tap, int chunk) {
        const unsigned koff = (unsigned)(tap * Kc + chunk * BK) * (unsigned)EB;
#pragma unroll
        for (int i = 0; i < BTASK; ++i)
            breg[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsB, boff[i] + koff, 0, 0));
    };
    auto store_b = [&](int buf) {
        char* Bb = reinterpret_cast<char*>(Bs + buf * BN * LDK);
#pragma unroll
        for (int i = 0; i < BTASK; ++i) *reinterpret_cast<i32x4*>(Bb + bdst[i]) = __builtin_bit_cast(i32x4, breg[i]);
    };

    // v_mfma_f32_16x16x32_bf16: one MFMA per 16 x 16 tile and 32-channel K-step (lane = (row l16, k group kg of 8)); the wave's
    // 64 x (32 TN) tile is 4 x (2 TN) of them
    constexpr int NA = 4, NB = 2 * TN;
    const int l16 = lane & 15, kg = lane >> 4;
    const int kgb = kg ^ (CODEPS_HALO_SWZ ? (((l16 >> 2) ^ (l16 >> 3)) & 1) : 0);      // weight tiles: swizzled k group of this lane's row
    f32x4 acc[NA][NB];
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // halo position of this lane's output pixel for row tile i (tap (0, 0)): pixel = wm * 64 + i * 16 + l16
    int apos[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int pix = wm * 64 + i * 16 + l16;
        apos[i] = (pix / TW) * HW + pix % TW;
    }

    load_a(0);
    load_b(0, 0);
    publish_amax();
    int run_e = F16_EMIN;
    int bbuf = 0;
    for (int chunk = 0; chunk < nchunks; ++chunk) {
        __syncthreads();                                          // the previous chunk's fragment reads are done
        if constexpr (H16) {
            const i32x4 pe = *reinterpret_cast<const i32x4*>(amax_slot);
            const int e_new = __builtin_amdgcn_readfirstlane(max(max(max(pe[0], pe[1]), max(pe[2], pe[3])), run_e));
            if (e_new != run_e) {                                 // re-base the sums so far to the larger tile's scale (exact)
                const float rb = f16_rebase(run_e, e_new);
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j] *= rb;
                run_e = e_new;
            }
            a_scale = f16_scale_of(run_e);
        }
        store_a();
        if (chunk == 0) store_b(0);
        __syncthreads();
        if (chunk + 1 < nchunks) load_a(chunk + 1);               // in flight during the nine taps
#pragma unroll 1
        for (int tap = 0; tap < 9; ++tap) {
            const bool last = chunk + 1 == nchunks && tap == 8;
            if (!last) load_b(tap == 8 ? 0 : tap + 1, tap == 8 ? chunk + 1 : chunk);
            const int ky = tap / 3, kx = tap % 3;
            const int toff = (MODE == MODE_FWD) ? ky * HW + kx : (2 - ky) * HW + (2 - kx);
            const float* Bb = Bs + bbuf * BN * LDK + (wn * TN * 32 + l16) * LDK;
            if (H16 && tap == 4 && chunk + 1 < nchunks) publish_amax();      // the next tile has landed by now; read behind the chunk's last barrier
            {
                typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
                frag_t af[NA][NP], bf[NB][NP];
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        af[i][q] = *reinterpret_cast<const frag_t*>(reinterpret_cast<const unsigned short*>(As + (apos[i] + toff) * LDKA) + q * BK + kg * 8);
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        bf[j][q] = *reinterpret_cast<const frag_t*>(reinterpret_cast<const unsigned short*>(Bb + j * 16 * LDK) + q * BK + kgb * 8);
#pragma unroll
                for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                    for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                        for (int i = 0; i < NA; ++i)
#pragma unroll
                            for (int j = 0; j < NB; ++j)
                                if constexpr (H16) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[i][qa], bf[j][ord - qa], acc[i][j], 0, 0, 0);
                                else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[i][qa], bf[j][ord - qa], acc[i][j], 0, 0, 0);
            }
            if (!last) store_b(bbuf ^ 1);                         // the other buffer: nobody reads it during this tap
            bbuf ^= 1;
            __syncthreads();
        }
    }

    // ---- epilogue (as in conv_igemm_kernel, rows mapped through the 4 x 32 tile)
    constexpr int LDC = BN + 4;
    float* Cs = smem;
    constexpr int V4 = BN / 4, RPASS = 256 / V4;
    const int c4 = tid % V4, r0 = tid / V4;
    const int n = n0 + c4 * 4;
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (MODE == MODE_FWD && n < p.N) {
        if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    }
    EpiCtx ec;
    if constexpr (EX) epi_begin(p, ec, b, n);
    if constexpr (H16) {                                          // sums of (x 2^ka)(w 2^kb): back to the operands' units (exact)
        const float inv = f16_inv_scale_of(run_e) * p.w2s[0];
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] *= inv;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (i > 0) __syncthreads();
        // pass i holds row tiles 2 i, 2 i + 1 of every wave; C layout of the 16 x 16 tile: column = l16, row = 4 kg + reg
#pragma unroll
        for (int ih = 0; ih < 2; ++ih)
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    Cs[(wm * 32 + ih * 16 + 4 * kg + r) * LDC + (wn * NB + j) * 16 + l16] = acc[2 * i + ih][j][r];
        // what the rows of this pass read from memory (residual / second gradient, the gates' tensors): requested before the barrier,
        // all rows at once (see EpiPre)
        constexpr int NRW = WM * 32 / RPASS;
        f32x4 resv[NRW];
        EpiPre pre[NRW];
#pragma unroll
        for (int u = 0; u < NRW; ++u) {
            const int rr = r0 + u * RPASS, pix = ((rr >> 5) * TM + i) * 32 + (rr & 31);
            const size_t idx = (((size_t)b * Hm + y0 + pix / TW) * Wm + x0 + pix % TW) * p.N + n;
            resv[u] = (residual && n < p.N) ? *reinterpret_cast<const f32x4*>(residual + idx) : f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (EX) pre[u] = epi_prefetch(p, idx, n < p.N);
        }
        __syncthreads();
        if constexpr (EX) if (i == 0 && p.ex_stat == 1) ec.sh = *reinterpret_cast<const f32x4*>(Cs + c4 * 4) * sc + sh;     // the tile's first row = the statistics' shift
        if (n < p.N) {
#pragma unroll
            for (int u = 0; u < NRW; ++u) {
                const int rr = r0 + u * RPASS, pix = ((rr >> 5) * TM + i) * 32 + (rr & 31);
                const size_t m = ((size_t)b * Hm + y0 + pix / TW) * Wm + x0 + pix % TW;
                f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * LDC + c4 * 4);
                if (MODE == MODE_FWD) {
                    v = v * sc + sh;
                    if (residual) v += resv[u];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
                } else if (residual) {
                    v += resv[u];
                }
                *reinterpret_cast<f32x4*>(out + m * p.N + n) = epi_apply_t<EX>(p, ec, v, pre[u]);
            }
        }
    }
    if constexpr (EX) epi_flush(p, ec, smem, tid, V4, RPASS, mt, n);
}

// ---------------------------------------------------------------------------------- halo-tile variant, weights by LDS DMA
// conv_halo3_kernel re-timed around two facts.  (1) The pre-split weights are plain copies, so they go global -> LDS without
// passing registers: `buffer_load_dwordx4 ... lds` into a ring of four (tap, chunk) tiles, issued as soon as a slot's
// fragments have been read, two taps before the tile is needed.  (2) The activation tile is constant for the nine taps of
// a chunk, so tap t + 1's A and B fragments are read while tap t's MFMAs run (taps fully unrolled, one fragment read per
// four MFMAs pinned with sched_group_barrier -- left alone the scheduler sinks the reads behind the MFMAs).  One barrier per
// tap.  The DMA is issued through inline assembly and its completion is counted by hand (vector-memory operations return
// in order): through the builtin the compiler orders every later LDS read behind the transfer with vmcnt(0), which
// also drains the activation loads in flight.  Measured on the ResNet-101 layer3 3x3 (B 8, 32 x 64, 256 -> 256): 120 -> 105 us
// back to back, -0.37 ms per step with the streams serialised, -0.13 ms with them overlapped (149 KB of LDS: nothing of
// the pose stream shares the CU).  128 output columns only: with 64 (two chunks of nine taps per block, 96 KB) it loses
// the second block per CU and measures 10 % slower than conv_halo3_kernel.  CODEPS_HALO_RING=0 selects conv_halo3_kernel.
// Tuning aid (never set in the shipped build): -DCODEPS_ABLATE_RING=bits -- 1: no weight DMA after the first ring fill, 2: the
// activation tile is written without the bf16 split, 4: the fragments of tap 0 serve every tap (no LDS fragment reads in the
// tap loop).  Results are garbage; the timings bound what each stage costs.
#ifndef CODEPS_ABLATE_RING
#define CODEPS_ABLATE_RING 0
#endif
#ifndef CODEPS_RING_ADB
#define CODEPS_RING_ADB 0        // A/B builds only: 1 = the fp16-pair ring kernel with TWO activation tiles, the next one staged under taps 3 .. (measured: 56.8 vs 56.1 us with eight waves, 67.8 vs 59.0 with four -- not kept)
#endif
#ifndef CODEPS_RING_BREG
#define CODEPS_RING_BREG 0       // A/B builds only: 1 = the fp16-pair ring kernel fills its weight ring through registers (measured 61.2 vs 58.6 us on ResNet-101 layer3: not kept)
#endif

// ARITH 3: three bf16 pieces, six products (rounds 2-5).  ARITH 16: two fp16 pieces, three products, block-local scales (round 6).
// NW = 8 (round 6, fp16 form): EIGHT waves, two per SIMD, on the same 4 x 32 pixel x 128 column tile (wave = 64 pixels x 32 columns).  With half
// the matrix instructions per tap a wave's own DMA issue, waits and barrier idle its SIMD's matrix pipe for as long as its MFMAs take; a
// second wave per SIMD multiplies meanwhile.  Same LDS image, ring and arithmetic (bit-identical results).
template <int MODE, int TN, bool EX = false, int ARITH = 3, int NW = 4>
__global__ __launch_bounds__(64 * NW) void conv_halo3r_kernel(ConvP p, const float* __restrict__ a0, const float* __restrict__ a1,
                                                          const float* __restrict__ scale, const float* __restrict__ shift,
                                                          const float* __restrict__ residual, float* __restrict__ out) {
    constexpr int WM = 2, WN = NW / 2, TM = 2, BK = 32, NP = ARITH == 16 ? 2 : 3;
    constexpr int NT = 64 * NW;                               // threads of the block
    constexpr bool H16 = ARITH == 16;
    constexpr int EB = NP * 2;                                // bytes per element of the pre-split weights
    constexpr int NPROD = NP * (NP + 1) / 2;
    constexpr int TH = 4, TW = 32, HH = TH + 2, HW = TW + 2, HPIX = HH * HW;
    constexpr int BN = 32 * WN * TN;
    constexpr int LDK = (NP * BK + 8) / 2;
    // Fragment reads (ds_read_b128, lane = (row l16, k group kg)) are serviced in the lane groups {0-3, 12-15, 20-27}, {4-11, 16-19, 28-31},
    // ... (MI355X_MICROARCH.md, LDS): with a 208-byte row pitch the rows of kg = 0 and the rows of kg = 1 of one group share 16-byte
    // slots -- every fragment read cost 8 LDS cycles instead of 4 (PMC, round 4: bank-conflict cycles = 13 % of the kernel's CU
    // cycles).  Activation tile: 224-byte pitch (14 slots per row: conflict-free for every alignment of the 16 consecutive halo
    // positions a fragment reads).  Weight tiles: the pitch stays 208 (LDS DMA image = pack rows + one pad segment) and the k groups
    // of rows 4 .. 11 (mod 16) are stored pairwise swapped -- the DMA picks the source segment per lane, the reader flips bit 0 of kg.
    // Two pieces: weight rows 144 bytes (9 slots: odd, so the pairwise swap works as above), activation rows 160 bytes (10 slots == -6 mod 16:
    // the 16 consecutive positions of a fragment at k group 0 cover the even slots, k group 1 the odd ones, for every alignment).
    constexpr int LDKA = CODEPS_HALO_SWZ ? LDK + 4 : LDK;
    constexpr int SEG = LDK / 4;                              // 16-byte slots per weight row in LDS (the last one is padding)
    constexpr int APASS = (HPIX * 4 + NT - 1) / NT, NALOAD = APASS * 2;
    constexpr int RING = 4;
    extern __shared__ __attribute__((aligned(16))) float smem[];
    // CODEPS_RING_ADB=1 (A/B builds; NOT the default): TWO activation tiles in the fp16 form (2 x 33 KB + 74 KB of weight ring).  The next
    // chunk's tile is split and stored between the MFMAs of taps 3 .. of the current chunk and the taps run on across the chunk boundary
    // instead of barrier -> split + store -> barrier -> first fragment reads (in-kernel stamps put a quarter of a chunk's time there).
    // Bit-identical; measured no faster with eight waves and 15 % slower with four (256 registers): the staging's instructions among the
    // MFMAs cost what the boundary cost.
    constexpr bool ADB = H16 && CODEPS_RING_ADB;
    constexpr int ATILE = (HPIX + 1) * LDKA;           // floats per activation tile
    float* As = smem;                                  // [ADB ? 2 : 1][HPIX + 1][LDKA]  (row HPIX: staging tasks past the tile)
    float* Bs = smem + (ADB ? 2 : 1) * ATILE;          // [RING][BN][LDK]
    int* amax_slot = reinterpret_cast<int*>(Bs + RING * BN * LDK);     // ARITH 16: the waves' maximum exponents of the activation tile in flight
    CODEPS_STAMP_BEGIN();
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    const int logical = xcd_remap(blockIdx.x, p.n_mt * p.n_nt);
    const int nt = logical % p.n_nt, mt = logical / p.n_nt;
    const int n0 = nt * BN;
    const int Hm = (MODE == MODE_FWD) ? p.Ho : p.H, Wm = (MODE == MODE_FWD) ? p.Wo : p.W;
    const int tiles_x = Wm / TW, tiles_y = Hm / TH;
    const int b = mt / (tiles_x * tiles_y), tr = mt % (tiles_x * tiles_y);
    const int y0 = (tr / tiles_x) * TH, x0 = (tr % tiles_x) * TW;
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;
    // split-K (grids that cannot fill the chip: gridDim.y slices of p.ksteps channel chunks each; raw partial sums go to
    // p.part[slice][M][N] and splitk_finish_kernel applies the epilogue): this block walks chunks [cbase, cbase + nchunks)
    const int cbase = p.ksplit > 1 ? (int)blockIdx.y * p.ksteps : 0;
    const int nchunks = p.ksplit > 1 ? min(p.ksteps, Kc / BK - cbase) : Kc / BK;
    const bool up = MODE == MODE_FWD && p.up0;
    const int H0 = up ? Hm / 2 : Hm, W0 = up ? Wm / 2 : Wm;
    const int cs0 = (MODE == MODE_FWD) ? p.C0 : p.Co;
    const float* img0 = a0 + (size_t)b * H0 * W0 * cs0;
    const float* img1 = (MODE == MODE_FWD && p.C1 > 0) ? a1 + (size_t)b * Hm * Wm * p.C1 : nullptr;
    const int achunk = tid & 3;

    // weights: lane L of the tile's linear 16-byte segment index copies segment L % 13 of row L / 13 (13th = pad); every wave
    // issues BPW instructions per tile (the waves past the last partial group repeat their previous instruction)
    const size_t wrow = (size_t)9 * Kc;
    constexpr int BINS = BN * SEG / 64, BPW = (BINS + NW - 1) / NW;
    static_assert((BN * SEG) % 64 == 0 && LDK * 4 == SEG * 16 && (SEG & 1) && BPW + NALOAD < 16, "linear DMA layout; vmcnt immediates");
    const int wave_u = __builtin_amdgcn_readfirstlane(wave);
    unsigned boff[BPW], bins[BPW];
#pragma unroll
    for (int i = 0; i < BPW; ++i) {
        const int ins = wave_u + NW * i < BINS ? wave_u + NW * i : wave_u + NW * (i - 1);
        const int L = ins * 64 + lane, row = L / SEG, seg = L % SEG;
        const int swz = CODEPS_HALO_SWZ ? (((row >> 2) ^ (row >> 3)) & 1) : 0;       // rows 4 .. 11 (mod 16): k groups swapped pairwise
        bins[i] = (unsigned)ins * 1024u;
        boff[i] = (unsigned)((size_t)min(n0 + row, p.N - 1) * wrow * EB + (seg < SEG - 1 ? (seg ^ swz) : 0) * 16);
    }
    i32x4 rsBv;
    {
        const unsigned long long a = reinterpret_cast<unsigned long long>(H16 ? p.w2 : p.w3);
        const size_t bytes = (size_t)p.N * wrow * EB;
        rsBv[0] = (int)__builtin_amdgcn_readfirstlane((unsigned)a);
        rsBv[1] = (int)(__builtin_amdgcn_readfirstlane((unsigned)(a >> 32)) & 0xFFFFu);
        rsBv[2] = (int)__builtin_amdgcn_readfirstlane((unsigned)(bytes < (size_t)GATHER_OOB ? bytes : (size_t)GATHER_OOB));
        rsBv[3] = 0x00020000;
    }
    const unsigned bs_lds = (unsigned)(size_t)(__attribute__((address_space(3))) char*)(Bs);
    auto dma_b = [&](int tap, int chunk, int slot) {
        const unsigned koff = (unsigned)__builtin_amdgcn_readfirstlane((tap * Kc + (cbase + chunk) * BK) * EB);
#pragma unroll
        for (int i = 0; i < BPW; ++i) {
            const unsigned dst = (unsigned)__builtin_amdgcn_readfirstlane(bs_lds + slot * BN * LDK * 4 + bins[i]);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(dst), "v"(boff[i]), "s"(rsBv), "s"(koff) : "memory");
        }
    };

    // CODEPS_RING_BREG=1 (A/B builds; NOT the default): the weight tiles of the fp16 form travel global -> registers -> LDS instead of by LDS
    // DMA.  With half the matrix instructions per tap the five DMA instructions every wave issues per tap are the largest item next to the
    // MFMAs (the kernel without them: 58.9 -> 52.2 us on ResNet-101 layer3, -DCODEPS_ABLATE_RING=1), but four 16-byte loads + four
    // ds_write_b128 per thread and tap (and 25 more registers) cost as much: 61.2 us.  The loads of tile g + 4 are issued behind the barrier
    // that ends tap g and written in front of the next one; plain builtins, the compiler counts vmcnt itself.
    constexpr bool BREG = H16 && CODEPS_RING_BREG;
    constexpr int BTASK = BN * (SEG - 1) / NT;                // 16-byte segments per thread and tile (the pad segment is not copied)
    static_assert(!BREG || (BN * (SEG - 1)) % NT == 0, "weight tile: whole segments per thread");
    const __amdgpu_buffer_rsrc_t rsBr = make_rsrc(static_cast<const float*>(H16 ? p.w2 : p.w3), (size_t)p.N * wrow * EB);
    unsigned rboff[BTASK], rbdst[BTASK];
#pragma unroll
    for (int i = 0; i < BTASK; ++i) {
        const int t = tid + NT * i, row = t / (SEG - 1), seg = t % (SEG - 1);
        const int swz = CODEPS_HALO_SWZ ? (((row >> 2) ^ (row >> 3)) & 1) : 0;
        rboff[i] = (unsigned)((size_t)min(n0 + row, p.N - 1) * wrow * EB + seg * 16);
        rbdst[i] = (unsigned)(row * LDK * 4 + (seg ^ swz) * 16);
    }
    f32x4 breg[BTASK];
    auto load_b = [&](int tap, int chunk, f32x4 (&r)[BTASK]) {
        const unsigned koff = (unsigned)__builtin_amdgcn_readfirstlane((tap * Kc + (cbase + chunk) * BK) * EB);
#pragma unroll
        for (int i = 0; i < BTASK; ++i) r[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsBr, rboff[i], koff, 0));
    };
    auto store_b = [&](int slot, const f32x4 (&r)[BTASK]) {
        char* Bb = reinterpret_cast<char*>(Bs + slot * BN * LDK);
#pragma unroll
        for (int i = 0; i < BTASK; ++i) *reinterpret_cast<f32x4*>(Bb + rbdst[i]) = r[i];
    };

    const __amdgpu_buffer_rsrc_t rsA0 = make_rsrc(img0, (size_t)H0 * W0 * cs0 * 4);
    const __amdgpu_buffer_rsrc_t rsA1 = make_rsrc(img1 ? img1 : img0, img1 ? (size_t)Hm * Wm * p.C1 * 4 : 0);
    f32x4 areg[NALOAD];
    auto load_a = [&](int chunk) {
        const int cstep = (cbase + chunk) * BK;
        const bool s1 = MODE == MODE_FWD && cstep >= p.C0;
        const int cs = s1 ? p.C1 : cs0, ws = s1 ? Wm : W0, sh = (!s1 && up) ? 1 : 0;
        const unsigned cbyte = (unsigned)((s1 ? cstep - p.C0 : cstep) + achunk * 8) * 4u;
#pragma unroll
        for (int i = 0; i < APASS; ++i) {
            const int pos = (tid >> 2) + (NT / 4) * i;
            const int iy = y0 + pos / HW - 1, ix = x0 + pos % HW - 1;
            const bool ok = pos < HPIX && iy >= 0 && iy < Hm && ix >= 0 && ix < Wm;
            const unsigned off = ok ? (unsigned)(((iy >> sh) * ws + (ix >> sh)) * cs) * 4u + cbyte : GATHER_OOB;
            if (s1) {
                areg[i * 2] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsA1, off, 0, 0));
                areg[i * 2 + 1] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsA1, off, 16, 0));
            } else {
                areg[i * 2] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsA0, off, 0, 0));
                areg[i * 2 + 1] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsA0, off, 16, 0));
            }
        }
    };
    // ARITH 16: the exponent of the largest magnitude in the tile `areg` holds -> amax_slot[wave] (read behind the next barrier)
    auto publish_amax = [&]() {
        if constexpr (H16) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < NALOAD; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(areg[i][e]));
            const int ex = wave_max_exponent(m);
            if (lane == 0) amax_slot[wave] = ex;
        }
    };
    float a_scale = 1.f;
    auto store_a_pos = [&](int i, float* Adst, float sc) {           // ADB: staging task i of this thread -> tile Adst
        const int pos = min((tid >> 2) + (NT / 4) * i, HPIX);
        u16x4 lo[NP], hi[NP];
        if constexpr (H16) {
            split_f16(areg[i * 2], sc, lo[0], lo[1]);
            split_f16(areg[i * 2 + 1], sc, hi[0], hi[1]);
        } else {
            split_bf16<NP>(areg[i * 2], lo);
            split_bf16<NP>(areg[i * 2 + 1], hi);
        }
        unsigned short* row = reinterpret_cast<unsigned short*>(Adst + pos * LDKA);
#pragma unroll
        for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(row + q * BK + achunk * 8) = pack8(lo[q], hi[q]);
    };
    auto store_a = [&]() {
#pragma unroll
        for (int i = 0; i < APASS; ++i) {
            const int pos = min((tid >> 2) + (NT / 4) * i, HPIX);
            u16x4 lo[NP], hi[NP];
#if CODEPS_ABLATE_RING & 2
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                lo[q] = u16x4{(unsigned short)__builtin_bit_cast(unsigned, areg[i * 2][q]), 1, 2, 3};
                hi[q] = u16x4{(unsigned short)__builtin_bit_cast(unsigned, areg[i * 2 + 1][q]), 1, 2, 3};
            }
#else
            if constexpr (H16) {
                split_f16(areg[i * 2], a_scale, lo[0], lo[1]);
                split_f16(areg[i * 2 + 1], a_scale, hi[0], hi[1]);
            } else {
                split_bf16<NP>(areg[i * 2], lo);
                split_bf16<NP>(areg[i * 2 + 1], hi);
            }
#endif
            unsigned short* row = reinterpret_cast<unsigned short*>(As + pos * LDKA);
#pragma unroll
            for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(row + q * BK + achunk * 8) = pack8(lo[q], hi[q]);
        }
    };

    constexpr int NA = 4, NB = 2 * TN;
    const int l16 = lane & 15, kg = lane >> 4;
    f32x4 acc[NA][NB];
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const unsigned short* arow[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int pix = wm * 64 + i * 16 + l16;
        arow[i] = reinterpret_cast<const unsigned short*>(As + ((pix / TW) * HW + pix % TW) * LDKA) + kg * 8;
    }
    const int bswz = CODEPS_HALO_SWZ ? (((l16 >> 2) ^ (l16 >> 3)) & 1) : 0;
    const unsigned short* brow = reinterpret_cast<const unsigned short*>(Bs + (wn * TN * 32 + l16) * LDK) + (kg ^ bswz) * 8;

    typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
    struct Frag { frag_t a[NA][NP], b[NB][NP]; };
    auto read_frags = [&](int tap, int slot, Frag& f, int abuf = 0) {   // tap: compile-time after unrolling; slot, abuf (activation tile): wave-uniform
        const int ky = tap / 3, kx = tap % 3;
        const int toff = ((MODE == MODE_FWD) ? ky * HW + kx : (2 - ky) * HW + (2 - kx)) * LDKA * 2;     // halfwords
        const unsigned short* bp = brow + slot * (BN * LDK * 2);
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int q = 0; q < NP; ++q) f.a[i][q] = *reinterpret_cast<const frag_t*>(arow[i] + abuf * (ATILE * 2) + toff + q * BK);
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int q = 0; q < NP; ++q) f.b[j][q] = *reinterpret_cast<const frag_t*>(bp + j * 16 * LDK * 2 + q * BK);
    };
    auto mfmas = [&](const Frag& f) {
#pragma unroll
        for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
            for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        if constexpr (H16) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.a[i][qa], f.b[j][ord - qa], acc[i][j], 0, 0, 0);
                        else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.a[i][qa], f.b[j][ord - qa], acc[i][j], 0, 0, 0);
    };
    const int T = 9 * nchunks;
    load_a(0);
    if constexpr (BREG) {                                         // tiles 0 .. 2 into the ring, tile 3 into the registers (written at the end of tap 0)
        f32x4 b1[BTASK], b2[BTASK];
        load_b(0, 0, breg); load_b(1, 0, b1); load_b(2, 0, b2);
        store_b(0, breg); store_b(1, b1); store_b(2, b2);
        load_b(3, 0, breg);
    } else {
#pragma unroll
        for (int g = 0; g < RING; ++g) dma_b(g, 0, g);            // nchunks >= 1: taps 0 .. 3 exist
        __builtin_amdgcn_s_waitcnt(0x0F70);                       // the first activation tile and four weight tiles have landed
#pragma unroll
        for (int i = 0; i < NALOAD; ++i) asm volatile("" : "+v"(areg[i]));
    }
    publish_amax();
    int run_e = F16_EMIN;                                         // ARITH 16: the largest exponent among the activation tiles staged so far
    auto block_exponent = [&](int floor_e) {                      // the waves' published exponents and `floor_e`: every thread the same value
        i32x4 pe = *reinterpret_cast<const i32x4*>(amax_slot);
        if constexpr (NW == 8) {
            const i32x4 pe2 = *reinterpret_cast<const i32x4*>(amax_slot + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) pe[e] = max(pe[e], pe2[e]);
        }
        return __builtin_amdgcn_readfirstlane(max(max(max(pe[0], pe[1]), max(pe[2], pe[3])), floor_e));
    };
    if constexpr (ADB) {
        __syncthreads();                                          // the exponents of tile 0
        run_e = block_exponent(run_e);
        a_scale = f16_scale_of(run_e);
#pragma unroll
        for (int i = 0; i < APASS; ++i) store_a_pos(i, As, a_scale);
        __syncthreads();
        Frag fr[2];
        read_frags(0, 0, fr[0], 0);
        int e_next = run_e;
        float s_next = a_scale;
        for (int chunk = 0; chunk < nchunks; ++chunk) {
            const int g0 = chunk * 9, par = chunk & 1;
            const bool more = chunk + 1 < nchunks;
            float* Anext = As + (par ^ 1) * ATILE;
            __builtin_amdgcn_sched_barrier(0);
            if (more) load_a(chunk + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int tap = 0; tap < 9; ++tap) {
                const int g = g0 + tap;
                CODEPS_STAMP_PHASE_START();
                const bool pre = tap < 8 || more;                   // the next tap exists (tap 8: tap 0 of the next chunk, from the other tile)
                if (tap < 8) read_frags(tap + 1, (g + 1) & 3, fr[(tap + 1) & 1], par);
                else if (more) read_frags(0, (g + 1) & 3, fr[1], par ^ 1);
                const bool stage = more && tap >= 3 && tap < 3 + APASS;      // this tap carries a staging task of the next tile
                if (stage) {
                    if (tap == 3) { e_next = block_exponent(run_e); s_next = f16_scale_of(e_next); }      // published in front of tap 2's barrier
                    store_a_pos(tap - 3, Anext, s_next);
                }
                mfmas(fr[tap & 1]);
                if (pre) {                                          // one fragment read, its share of the MFMAs, then room for the staging's instructions
#pragma unroll
                    for (int k = 0; k < NA * NP + NB * NP; ++k) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, (NA * NB * NPROD) / (NA * NP + NB * NP), 0);
                        if (stage) __builtin_amdgcn_sched_group_barrier(0x202, 6, 0);
                    }
                }
                const bool t3 = g + 3 < T;
                CODEPS_STAMP_PHASE_A();
                CODEPS_STAMP_PHASE_START();
                if (tap < 2 && more) {
                    if (t3) __builtin_amdgcn_s_waitcnt(0x0F70 | (BPW + NALOAD));
                    else __builtin_amdgcn_s_waitcnt(0x0F70 | NALOAD);
                } else {
                    if (t3) __builtin_amdgcn_s_waitcnt(0x0F70 | BPW);
                    else __builtin_amdgcn_s_waitcnt(0x0F70);
                }
                if (tap == 2) {
#pragma unroll
                    for (int i = 0; i < NALOAD; ++i) asm volatile("" : "+v"(areg[i]));
                    if (more) publish_amax();
                }
                __syncthreads();
                if (g + 4 < T) dma_b((tap + 4) % 9, chunk + (tap + 4) / 9, g & 3);
                CODEPS_STAMP_PHASE_B();
            }
            if (more) {
                if (e_next != run_e) {                            // the next tile was staged at a larger scale: re-base the sums (exact)
                    const float rb = f16_rebase(run_e, e_next);
#pragma unroll
                    for (int i = 0; i < NA; ++i)
#pragma unroll
                        for (int j = 0; j < NB; ++j) acc[i][j] *= rb;
                    run_e = e_next;
                }
                fr[0] = fr[1];                                    // (tap 8 runs from fr[0] and fetched the next chunk's tap 0 into fr[1])
            }
        }
    } else
    for (int chunk = 0; chunk < nchunks; ++chunk) {
        const int g0 = chunk * 9;
        const bool more = chunk + 1 < nchunks;
        __syncthreads();                                          // the previous chunk's fragment reads are done
        if constexpr (H16) {
            i32x4 pe = *reinterpret_cast<const i32x4*>(amax_slot);
            if constexpr (NW == 8) {
                const i32x4 pe2 = *reinterpret_cast<const i32x4*>(amax_slot + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) pe[e] = max(pe[e], pe2[e]);
            }
            const int e_new = __builtin_amdgcn_readfirstlane(max(max(max(pe[0], pe[1]), max(pe[2], pe[3])), run_e));
            if (e_new != run_e) {                                 // the tile outgrew the scale of the sums so far: re-base them (exact)
                const float rb = f16_rebase(run_e, e_new);
#pragma unroll
                for (int i = 0; i < NA; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j] *= rb;
                run_e = e_new;
            }
            a_scale = f16_scale_of(run_e);
        }
        store_a();
        __syncthreads();
        Frag fr[2];
        read_frags(0, g0 & 3, fr[0]);
        __builtin_amdgcn_sched_barrier(0);
        if (more) load_a(chunk + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int tap = 0; tap < 9; ++tap) {
            const int g = g0 + tap;
            CODEPS_STAMP_PHASE_START();
#if CODEPS_ABLATE_RING & 4
            mfmas(fr[0]);
            if (false) {
#else
            if (tap < 8) read_frags(tap + 1, (g + 1) & 3, fr[(tap + 1) & 1]);   // tile g + 1 landed before the barrier that ended tap g - 1
            mfmas(fr[tap & 1]);
            if (tap < 8) {
#endif                                         // one fragment read per four MFMAs (the scheduler would sink the reads)
#pragma unroll
                for (int k = 0; k < NA * NP + NB * NP; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, (NA * NB * NPROD) / (NA * NP + NB * NP), 0);
                }
            }
            // End of tap g: tile g + 2 (issued after the barrier that ended tap g - 2) must have landed.  Younger operations
            // that may stay in flight: tile g + 3 (BPW instructions, if it exists) and, at taps 0 and 1, the next chunk's
            // activation loads (issued at the chunk's start, after tiles g0 + 2 and g0 + 3).  Tile g0 + 4 is younger than
            // those loads, so tap 2's wait completes them -- told to the compiler there (an empty asm that "uses" the
            // registers), or it would count them against the DMA instructions in flight when store_a reads them.
            const bool t3 = g + 3 < T;
            CODEPS_STAMP_PHASE_A();                                // A: fragment reads of tap + 1 issued, 96 MFMAs of tap issued
            CODEPS_STAMP_PHASE_START();
            if constexpr (BREG) {
                // tile g + 3 (loaded during this tap) -> its slot, which held tile g - 1 (last read during tap g - 2); behind the barrier the
                // loads of tile g + 4.  sched_barriers: the stores stay behind the tap's MFMAs, the loads behind the barrier
                __builtin_amdgcn_sched_barrier(0);
                if (t3) store_b((g + 3) & 3, breg);
                if (tap == 2 && more) publish_amax();
                __syncthreads();
                if (g + 4 < T) load_b((tap + 4) % 9, chunk + (tap + 4) / 9, breg);
                __builtin_amdgcn_sched_barrier(0);
            } else {
            if (tap < 2 && more) {
                if (t3) __builtin_amdgcn_s_waitcnt(0x0F70 | (BPW + NALOAD));
                else __builtin_amdgcn_s_waitcnt(0x0F70 | NALOAD);
            } else {
                if (t3) __builtin_amdgcn_s_waitcnt(0x0F70 | BPW);
                else __builtin_amdgcn_s_waitcnt(0x0F70);
            }
            if (tap == 2) {                                        // unconditional: the waitcnt pass is not path-sensitive
#pragma unroll
                for (int i = 0; i < NALOAD; ++i) asm volatile("" : "+v"(areg[i]));
                if (more) publish_amax();                          // (the slot's previous values were read at this chunk's start, barriers ago)
            }
            __syncthreads();
            // every wave has read tile g's fragments (during tap g - 1, or at the chunk's start): its slot takes tile g + 4
            if (g + 4 < T && !(CODEPS_ABLATE_RING & 1)) dma_b((tap + 4) % 9, chunk + (tap + 4) / 9, g & 3);
            }
            CODEPS_STAMP_PHASE_B();                                // B: wait for tile g + 2, barrier, DMA of tile g + 4 issued
        }
    }
    if constexpr (!BREG) __builtin_amdgcn_s_waitcnt(0x0F70);

    // ---- epilogue (as in conv_halo3_kernel)
    constexpr int LDC = BN + 4;
    float* Cs = smem;
    constexpr int V4 = BN / 4, RPASS = NT / V4;
    const int c4 = tid % V4, r0 = tid / V4;
    const int n = n0 + c4 * 4;
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (MODE == MODE_FWD && n < p.N) {
        if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    }
    EpiCtx ec;
    if constexpr (EX) epi_begin(p, ec, b, n);
    if constexpr (H16) {                                          // sums of (x 2^ka)(w 2^kb): back to the operands' units (exact)
        const float inv = f16_inv_scale_of(run_e) * p.w2s[0];
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] *= inv;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        __syncthreads();
#pragma unroll
        for (int ih = 0; ih < 2; ++ih)
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    Cs[(wm * 32 + ih * 16 + 4 * kg + r) * LDC + (wn * NB + j) * 16 + l16] = acc[2 * i + ih][j][r];
        // what the rows of this pass read from memory (residual / second gradient, the gates' tensors): requested before the barrier,
        // all rows at once (see EpiPre); K slices: nothing (the finish pass applies the epilogue)
        constexpr int NRW = WM * 32 / RPASS;
        f32x4 resv[NRW];
        EpiPre pre[NRW];
#pragma unroll
        for (int u = 0; u < NRW; ++u) {
            const int rr = r0 + u * RPASS, pix = ((rr >> 5) * TM + i) * 32 + (rr & 31);
            const size_t idx = (((size_t)b * Hm + y0 + pix / TW) * Wm + x0 + pix % TW) * p.N + n;
            const bool live = p.ksplit <= 1 && n < p.N;
            resv[u] = (residual && live) ? *reinterpret_cast<const f32x4*>(residual + idx) : f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (EX) pre[u] = epi_prefetch(p, idx, live);
        }
        __syncthreads();
        if constexpr (EX) if (i == 0 && p.ex_stat == 1) ec.sh = *reinterpret_cast<const f32x4*>(Cs + c4 * 4) * sc + sh;     // the tile's first row = the statistics' shift
        if (n < p.N) {
#pragma unroll
            for (int u = 0; u < NRW; ++u) {
                const int rr = r0 + u * RPASS, pix = ((rr >> 5) * TM + i) * 32 + (rr & 31);
                const size_t m = ((size_t)b * Hm + y0 + pix / TW) * Wm + x0 + pix % TW;
                f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * LDC + c4 * 4);
                if (p.ksplit > 1) {                           // raw partial sum of this K slice; splitk_finish_kernel does the rest
                    *reinterpret_cast<f32x4*>(p.part + ((size_t)blockIdx.y * p.M + m) * p.N + n) = v;
                    continue;
                }
                if (MODE == MODE_FWD) {
                    v = v * sc + sh;
                    if (residual) v += resv[u];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
                } else if (residual) {
                    v += resv[u];
                }
                *reinterpret_cast<f32x4*>(out + m * p.N + n) = epi_apply_t<EX>(p, ec, v, pre[u]);
            }
        }
    }
    if constexpr (EX) if (p.ksplit <= 1) epi_flush(p, ec, smem, tid, V4, RPASS, mt, n);
    CODEPS_STAMP_END(conv);
}

// ---------------------------------------------------------------------------------- halo-tile ring kernel, producer / consumer waves
// conv_halo3r_kernel with the staging taken out of the matrix waves' instruction streams.  In-kernel stamps of that kernel
// (tools/clock_cycles.py, profiles/r04_clock_cycles.json; ResNet-101 layer3 3x3, 2.2-2.3 GHz in the kernel) put 57 % of a block's
// lifetime into issuing MFMAs, 18 % into the wait + barrier + the seven LDS-DMA instructions every wave issues per tap, 8 % into the
// bf16 split of the activation tile -- and a second wave on a SIMD that only issues vector / memory instructions does not cost the MFMA
// wave a cycle (32.04 cycles per v_mfma_f32_32x32x16_bf16 with 0 .. 16 v_fma_f32 per MFMA in the partner wave).  So: 384 threads =
// waves 0-3 CONSUMERS (the 2 x 2 wave grid: LDS fragment reads + MFMAs, nothing else in the tap loop) + waves 4-5 PRODUCERS (all
// 26 LDS-DMA instructions of a weight tile, and load -> split -> store of the next chunk's activation tile while the consumers run
// the chunk's last tap).  Same LDS image, same ring of four weight tiles, same arithmetic and summation order as conv_halo3r_kernel
// (bit-identical results); one barrier per tap.  Six waves on four SIMDs leave 256 registers per wave, so the consumers keep ONE set
// of A fragments and reload row tile i for the next tap right after its 24 MFMAs (the MFMAs run row tile by row tile), a second
// set only for row tile 3, and two sets of B fragments.
template <int MODE, int TN>
__global__ __launch_bounds__(384) void conv_halo3p_kernel(ConvP p, const float* __restrict__ a0, const float* __restrict__ a1,
                                                          const float* __restrict__ scale, const float* __restrict__ shift,
                                                          const float* __restrict__ residual, float* __restrict__ out) {
    constexpr int WM = 2, WN = 2, TM = 2, BK = 32, NP = 3;
    constexpr int TH = 4, TW = 32, HH = TH + 2, HW = TW + 2, HPIX = HH * HW;
    constexpr int BN = 32 * WN * TN;
    constexpr int LDK = (NP * BK + 8) / 2;
    constexpr int PT = 128;                                         // producer threads
    constexpr int ATASK = (HPIX * 4 + PT - 1) / PT, NALOAD = ATASK * 2;      // (pixel, 8-channel group) tasks / 16-byte loads per producer thread
    constexpr int BINS = BN * 13 / 64, BPW = BINS / 2;              // LDS-DMA instructions per weight tile / per producer wave
    static_assert((BN * 13) % 128 == 0 && LDK * 4 == 13 * 16 && BPW + NALOAD < 64, "linear DMA layout; vmcnt immediates");
    extern __shared__ __attribute__((aligned(16))) float smem[];
    float* As = smem;                                  // [HPIX + 1][LDK]  (row HPIX: staging tasks past the tile)
    float* Bs = smem + (HPIX + 1) * LDK;               // [4][BN][LDK]
    CODEPS_STAMP_BEGIN();
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool producer = wave >= 4;
    const int wm = (wave & 3) / WN, wn = (wave & 3) % WN;
    const int logical = xcd_remap(blockIdx.x, p.n_mt * p.n_nt);
    const int nt = logical % p.n_nt, mt = logical / p.n_nt;
    const int n0 = nt * BN;
    const int Hm = (MODE == MODE_FWD) ? p.Ho : p.H, Wm = (MODE == MODE_FWD) ? p.Wo : p.W;
    const int tiles_x = Wm / TW, tiles_y = Hm / TH;
    const int b = mt / (tiles_x * tiles_y), tr = mt % (tiles_x * tiles_y);
    const int y0 = (tr / tiles_x) * TH, x0 = (tr % tiles_x) * TW;
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;
    const int cbase = p.ksplit > 1 ? (int)blockIdx.y * p.ksteps : 0;
    const int nchunks = p.ksplit > 1 ? min(p.ksteps, Kc / BK - cbase) : Kc / BK;
    const int T = 9 * nchunks;
    constexpr int NA = 4, NB = 2 * TN;
    const int l16 = lane & 15, kg = lane >> 4;
    f32x4 acc[NA][NB];

    if (producer) {
        // ============================================================ producers: weight tiles by LDS DMA, activation tiles
        const int pw = wave - 4, ptid = tid - 256;
        const bool up = MODE == MODE_FWD && p.up0;
        const int H0 = up ? Hm / 2 : Hm, W0 = up ? Wm / 2 : Wm;
        const int cs0 = (MODE == MODE_FWD) ? p.C0 : p.Co;
        const float* img0 = a0 + (size_t)b * H0 * W0 * cs0;
        const float* img1 = (MODE == MODE_FWD && p.C1 > 0) ? a1 + (size_t)b * Hm * Wm * p.C1 : nullptr;
        const int achunk = ptid & 3;
        const size_t wrow = (size_t)9 * Kc;
        unsigned boff[BPW], bins[BPW];
#pragma unroll
        for (int i = 0; i < BPW; ++i) {
            const int ins = pw + 2 * i;
            const int L = ins * 64 + lane, row = L / 13, seg = L % 13;
            bins[i] = (unsigned)ins * 1024u;
            boff[i] = (unsigned)((size_t)min(n0 + row, p.N - 1) * wrow * 6 + (seg < 12 ? seg : 0) * 16);
        }
        auto rsrc_of = [](const void* base, size_t bytes) {
            const unsigned long long a = reinterpret_cast<unsigned long long>(base);
            i32x4 r;
            r[0] = (int)__builtin_amdgcn_readfirstlane((unsigned)a);
            r[1] = (int)(__builtin_amdgcn_readfirstlane((unsigned)(a >> 32)) & 0xFFFFu);
            r[2] = (int)__builtin_amdgcn_readfirstlane((unsigned)(bytes < (size_t)GATHER_OOB ? bytes : (size_t)GATHER_OOB));
            r[3] = 0x00020000;
            return r;
        };
        const i32x4 rsBv = rsrc_of(p.w3, (size_t)p.N * wrow * 6);
        const i32x4 rsA0 = rsrc_of(img0, (size_t)H0 * W0 * cs0 * 4);
        const i32x4 rsA1 = rsrc_of(img1 ? img1 : img0, img1 ? (size_t)Hm * Wm * p.C1 * 4 : 0);
        const unsigned bs_lds = (unsigned)(size_t)(__attribute__((address_space(3))) char*)(Bs);
        auto dma_b = [&](int g) {                                   // weight tile g (global tap index of this block) -> slot g & 3
            const int tap = g % 9, chunk = g / 9;
            const unsigned koff = (unsigned)__builtin_amdgcn_readfirstlane((tap * Kc + (cbase + chunk) * BK) * 6);
#pragma unroll
            for (int i = 0; i < BPW; ++i) {
                const unsigned dst = (unsigned)__builtin_amdgcn_readfirstlane(bs_lds + (g & 3) * BN * LDK * 4 + bins[i]);
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                             :: "s"(dst), "v"(boff[i]), "s"(rsBv), "s"(koff) : "memory");
            }
        };
        // The activation loads are inline assembly too: every vector-memory operation of these waves is then counted by hand (they
        // retire in order), and the compiler -- which takes an asm destination for written at once -- gets the registers back only
        // through the "claim" statement that carries the wait.
        f32x4 areg[NALOAD];
        auto load_a = [&](int chunk) {
            const int cstep = (cbase + chunk) * BK;
            const bool s1 = MODE == MODE_FWD && cstep >= p.C0;
            const int cs = s1 ? p.C1 : cs0, ws = s1 ? Wm : W0, sh = (!s1 && up) ? 1 : 0;
            const unsigned cbyte = (unsigned)((s1 ? cstep - p.C0 : cstep) + achunk * 8) * 4u;
            const i32x4 rs = s1 ? rsA1 : rsA0;
#pragma unroll
            for (int i = 0; i < ATASK; ++i) {
                const int pos = (ptid >> 2) + 32 * i;
                const int iy = y0 + pos / HW - 1, ix = x0 + pos % HW - 1;
                const bool ok = pos < HPIX && iy >= 0 && iy < Hm && ix >= 0 && ix < Wm;
                const unsigned off = ok ? (unsigned)(((iy >> sh) * ws + (ix >> sh)) * cs) * 4u + cbyte : GATHER_OOB;
                asm volatile("buffer_load_dwordx4 %0, %1, %2, 0 offen" : "=v"(areg[i * 2]) : "v"(off), "s"(rs) : "memory");
                asm volatile("buffer_load_dwordx4 %0, %1, %2, 0 offen offset:16" : "=v"(areg[i * 2 + 1]) : "v"(off), "s"(rs) : "memory");
            }
        };
        auto store_a = [&]() {
#pragma unroll
            for (int i = 0; i < ATASK; ++i) {
                const int pos = min((ptid >> 2) + 32 * i, HPIX);
                u16x4 lo[NP], hi[NP];
                split_bf16<NP>(areg[i * 2], lo);
                split_bf16<NP>(areg[i * 2 + 1], hi);
                unsigned short* row = reinterpret_cast<unsigned short*>(As + pos * LDK);
#pragma unroll
                for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(row + q * BK + achunk * 8) = pack8(lo[q], hi[q]);
            }
        };
#define HALO3P_CLAIM(WAIT)                                                                                                       \
    asm volatile(WAIT : "+v"(areg[0]), "+v"(areg[1]), "+v"(areg[2]), "+v"(areg[3]), "+v"(areg[4]), "+v"(areg[5]), "+v"(areg[6]),   \
                 "+v"(areg[7]), "+v"(areg[8]), "+v"(areg[9]), "+v"(areg[10]), "+v"(areg[11]), "+v"(areg[12]), "+v"(areg[13]) :: "memory")
        static_assert(NALOAD == 14, "HALO3P_CLAIM lists 14 registers");
        // ---- prologue: first activation tile + four weight tiles; everything landed, tile written, next tile's loads in flight
        load_a(0);
#pragma unroll
        for (int g = 0; g < 4; ++g) dma_b(g);                       // nchunks >= 1: taps 0 .. 3 exist
        HALO3P_CLAIM("s_waitcnt vmcnt(0)");
        __builtin_amdgcn_sched_barrier(0);
        store_a();
        if (nchunks > 1) load_a(1);
        __syncthreads();                                            // S: tile 0 .. 3 and the first activation tile are visible
        for (int chunk = 0; chunk < nchunks; ++chunk) {
            const int g0 = chunk * 9;
#pragma unroll
            for (int tap = 0; tap < 9; ++tap) {
                const int g = g0 + tap;
                // (1) the slot of tile g - 1 is free (its fragments were read before barrier g - 1): tile g + 3 goes there
                if (g >= 1 && g + 3 < T) dma_b(g + 3);
                // (2) last tap of the chunk: the consumers read nothing of the activation tile any more (tap 8's A fragments were
                //     read during tap 7): write the next chunk's tile, then start the loads of the one after it
                if (tap == 8 && chunk + 1 < nchunks) {
                    store_a();
                    if (chunk + 2 < nchunks) load_a(chunk + 2);
                }
                // (3) tile g + 2 must have landed before barrier g (the consumers read its fragments during tap g + 1).  Younger
                //     operations that may stay in flight: tile g + 3 (BPW instructions) and the activation loads issued in (2) of
                //     this tap or of the tap before (tap 0: issued at the previous chunk's tap 8, or in the prologue).
                const bool t3 = g >= 1 && g + 3 < T;
                const bool al = (tap == 8 && chunk + 2 < nchunks) || (tap == 0 && chunk + 1 < nchunks);
                if (t3 && al) asm volatile("s_waitcnt vmcnt(27)" ::: "memory");
                else if (t3) asm volatile("s_waitcnt vmcnt(13)" ::: "memory");
                else if (al) asm volatile("s_waitcnt vmcnt(14)" ::: "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                // tap 1's wait leaves at most tile g + 3 in flight: the activation loads (older) have landed -- claimed here,
                // unconditionally (harmless when no loads were issued: the registers are then not read before the next load_a)
                if (tap == 1) { HALO3P_CLAIM(""); }
                static_assert(BPW == 13 && NALOAD == 14, "vmcnt immediates above");
                __syncthreads();                                    // barrier g
            }
        }
#undef HALO3P_CLAIM
    } else {
        // ============================================================ consumers: fragment reads + MFMAs
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const unsigned short* arow[NA];
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int pix = wm * 64 + i * 16 + l16;
            arow[i] = reinterpret_cast<const unsigned short*>(As + ((pix / TW) * HW + pix % TW) * LDK) + kg * 8;
        }
        const unsigned short* brow = reinterpret_cast<const unsigned short*>(Bs + (wn * TN * 32 + l16) * LDK) + kg * 8;
        auto toff_of = [](int tap) {                                // halfwords
            const int ky = tap / 3, kx = tap % 3;
            return ((MODE == MODE_FWD) ? ky * HW + kx : (2 - ky) * HW + (2 - kx)) * LDK * 2;
        };
        auto read_a = [&](int tap, int i, bf16x8 (&f)[NP]) {
#pragma unroll
            for (int q = 0; q < NP; ++q) f[q] = *reinterpret_cast<const bf16x8*>(arow[i] + toff_of(tap) + q * BK);
        };
        auto read_b = [&](int slot, bf16x8 (&f)[NB][NP]) {           // slot: wave-uniform
            const unsigned short* bp = brow + slot * (BN * LDK * 2);
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int q = 0; q < NP; ++q) f[j][q] = *reinterpret_cast<const bf16x8*>(bp + j * 16 * LDK * 2 + q * BK);
        };
        auto row_mfmas = [&](int i, const bf16x8 (&a)[NP], const bf16x8 (&bq)[NB][NP]) {
#pragma unroll
            for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                    for (int j = 0; j < NB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[qa], bq[j][ord - qa], acc[i][j], 0, 0, 0);
        };
        bf16x8 af[3][NP], a3[2][NP], bq[2][NB][NP];
        __syncthreads();                                            // S
        for (int chunk = 0; chunk < nchunks; ++chunk) {
            const int g0 = chunk * 9;
            // chunk start (behind barrier S or barrier g0 - 1): this chunk's activation tile and weight tile g0 are in LDS
#pragma unroll
            for (int i = 0; i < 3; ++i) read_a(0, i, af[i]);
            read_a(0, 3, a3[0]);
            read_b(g0 & 3, bq[0]);
#pragma unroll
            for (int tap = 0; tap < 9; ++tap) {
                const int g = g0 + tap;
                CODEPS_STAMP_PHASE_START();
                if (tap < 8) {                                      // the next tap's weight fragments and row tile 3: free registers
                    read_b((g + 1) & 3, bq[(tap + 1) & 1]);
                    read_a(tap + 1, 3, a3[(tap + 1) & 1]);
                }
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    row_mfmas(i, af[i], bq[tap & 1]);
                    if (tap < 8) read_a(tap + 1, i, af[i]);         // reloaded in place once its 24 MFMAs have been issued
                }
                row_mfmas(3, a3[tap & 1], bq[tap & 1]);
                if (tap < 8) {                                      // one fragment read per four MFMAs
#pragma unroll
                    for (int k = 0; k < NA * NP + NB * NP; ++k) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, (NA * NB * 6) / (NA * NP + NB * NP), 0);
                    }
                }
                CODEPS_STAMP_PHASE_A();                             // A: fragment reads + 96 MFMAs issued
                CODEPS_STAMP_PHASE_START();
                __syncthreads();                                    // barrier g
                CODEPS_STAMP_PHASE_B();                             // B: waiting at the barrier (the producers, the other consumers)
            }
        }
    }

    // ---- epilogue (as in conv_halo3r_kernel; the consumer waves hold the accumulators, all 384 threads move rows)
    constexpr int LDC = BN + 4;
    float* Cs = smem;
    constexpr int V4 = BN / 4, RPASS = 384 / V4;
    const int c4 = tid % V4, r0 = tid / V4;
    const int n = n0 + c4 * 4;
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (MODE == MODE_FWD && n < p.N) {
        if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        if (i > 0) __syncthreads();                               // (pass 0: the loop's last barrier already separates the fragment reads)
        if (!producer) {
#pragma unroll
            for (int ih = 0; ih < 2; ++ih)
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        Cs[(wm * 32 + ih * 16 + 4 * kg + r) * LDC + (wn * NB + j) * 16 + l16] = acc[2 * i + ih][j][r];
        }
        __syncthreads();
        if (n < p.N) {
            for (int rr = r0; rr < WM * 32; rr += RPASS) {
                const int pix = ((rr >> 5) * TM + i) * 32 + (rr & 31);
                const size_t m = ((size_t)b * Hm + y0 + pix / TW) * Wm + x0 + pix % TW;
                f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * LDC + c4 * 4);
                if (p.ksplit > 1) {                           // raw partial sum of this K slice; splitk_finish_kernel does the rest
                    *reinterpret_cast<f32x4*>(p.part + ((size_t)blockIdx.y * p.M + m) * p.N + n) = v;
                    continue;
                }
                if (MODE == MODE_FWD) {
                    v = v * sc + sh;
                    if (residual) v += *reinterpret_cast<const f32x4*>(residual + m * p.N + n);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
                } else if (residual) {
                    v += *reinterpret_cast<const f32x4*>(residual + m * p.N + n);
                }
                *reinterpret_cast<f32x4*>(out + m * p.N + n) = v;
            }
        }
    }
    CODEPS_STAMP_END(conv);
}

// ---------------------------------------------------------------------------------- 16-column variant
// N <= 16 (disparity / class / centre-offset outputs, the 16-channel full-resolution decoder tail and their data
// gradients): v_mfma_f32_16x16x4_f32 tiles, so no MFMA work is spent on zero-padded output columns.
// With a single 16-wide column tile every A element feeds exactly one MFMA, i.e. there is NO reuse to stage for:
// both operands go global -> VGPR directly (lane (l&15, q=l>>4) loads 16 B = k 4q..4q+3 of its own pixel row / weight
// row for each 16-deep k group; 4 lanes cover one 64-B run), software-pipelined one K-step ahead in registers.
// No LDS and no barrier in the main loop; waves run independently (64 rows = 4 row tiles per wave).
// Forward of the double-pixel stem (ResNet conv1 as 7 x 4 taps of 16 channels, stride (2, 1), padding (3, 0), 64 output channels:
// codeps_amd.functional.stem_conv2d) as a halo-tile kernel.  The generic kernel runs it in 28 K-steps of one tap each and stages
// a 128-row operand tile for every one of them -- 100 TFLOP/s; here an 8 x 32 output tile's input (21 rows x 35 double pixels) is
// split and stored in LDS ONCE, as [row][double pixel][piece][16 ch] at a 112-byte pitch (28 dwords: conflict-free 16-byte fragment
// reads), and every tap reads its fragments from that image at a shifted address.  The pre-split weights of one tap row (4 taps x 64
// channels, 25 KB) ride in a two-slot ring filled through registers one tap row ahead.  Eight waves, two per SIMD (one hides the
// other's fragment-read and barrier latencies: with four waves of two rows each the kernel measured 490 us, 50 % of its MFMA time);
// wave w owns output row w of the tile (one 32-pixel MFMA row tile x two 32-channel column tiles): 48 MFMAs per tap row against
// 12 + 24 fragment reads.  Blocks walk `tiles_per_block` tiles; the next tile's loads are issued under the last tap rows of the
// current one.
// ARITH 16 (round 6): two fp16 pieces; the input tile's scale per tile (block-wide maximum in front of the tile's first barrier), the weights'
// from the pack.
template <int ARITH = 3>
__global__ __launch_bounds__(512) void conv_stem74f_kernel(ConvP p, int tiles_x, int tiles_y, int tiles_per_block, const float* __restrict__ x,
                                                           const float* __restrict__ scale, const float* __restrict__ shift, float* __restrict__ y) {
    constexpr int NP = ARITH == 16 ? 2 : 3, EB = NP * 2;
    constexpr bool H16 = ARITH == 16;
    typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
    __shared__ float stem_red[8];                      // ARITH 16: the waves' largest magnitudes of the input tile in flight
    constexpr int TH = 8, TW = 32, KH = 7, KW = 4, XH = 2 * TH + KH - 2, XW = TW + KW - 1, PIT = NP * 16 + 8;      // PIT: halfwords per double pixel
    constexpr int WROW = 2 * NP * 32 + 8;              // halfwords per output channel and tap row: [2 groups][NP pieces][32] + pad (100 / 68 dwords)
    constexpr int WSEG = 2 * NP * 4;                   // 16-byte segments of such a row
    constexpr int NT = 512, NTASK = XH * XW * 4, NRAW = (NTASK + NT - 1) / NT, NWSEG = 64 * WSEG / NT;
    extern __shared__ __attribute__((aligned(16))) unsigned short lds16[];
    unsigned short* Xs = lds16;                        // [XH][XW][PIT]
    unsigned short* Ws = lds16 + XH * XW * PIT;        // [2][64][WROW]
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blockIdx.x * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    const size_t ximg = (size_t)p.H * p.W * 16;
    const char* w3 = static_cast<const char*>(H16 ? p.w2 : p.w3);

    // input tasks: (row r, double pixel c, channel quad c4); thread tid owns tasks tid + 512 k
    int t_off[NRAW], t_row[NRAW], t_dst[NRAW];
#pragma unroll
    for (int k = 0; k < NRAW; ++k) {
        const int t = tid + NT * k, c4 = t & 3, pc = t >> 2, c = pc % XW, r = pc / XW;
        t_row[k] = t < NTASK ? r : 1 << 20;            // (a row no image has)
        t_off[k] = ((r * p.W + c) * 16 + c4 * 4) * 4;
        t_dst[k] = (r * XW + c) * PIT + c4 * 4;
    }
    f32x4 raw[NRAW];
    auto load_x = [&](int tile, bool valid) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);             // (scalar)
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(x + (size_t)b * ximg, ximg * 4);
        const int iy0 = 2 * ty0 - p.pad, org = (iy0 * p.W + tx0) * 64;
#pragma unroll
        for (int k = 0; k < NRAW; ++k) {
            const unsigned vo = (valid && (unsigned)(iy0 + t_row[k]) < (unsigned)p.H) ? (unsigned)(org + t_off[k]) : GATHER_OOB;
            raw[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, 0, 0));
        }
    };
    float a_scale = 1.f;
    auto store_x = [&]() {
#pragma unroll
        for (int k = 0; k < NRAW; ++k) {
            if (tid + NT * k >= NTASK) continue;
            u16x4 pc[NP];
            if constexpr (H16) split_f16(raw[k], a_scale, pc[0], pc[1]);
            else split_bf16<NP>(raw[k], pc);
#pragma unroll
            for (int q = 0; q < NP; ++q) *reinterpret_cast<u16x4*>(Xs + t_dst[k] + q * 16) = pc[q];
        }
    };
    // weights of tap row ky: per output channel 384 contiguous bytes of the pre-split pack ([co][14 groups][3 pieces][32 bf16], groups 2 ky, 2 ky + 1)
    i32x4 wreg[NWSEG];
    auto load_w = [&](int ky) {
#pragma unroll
        for (int i = 0; i < NWSEG; ++i) {
            const int seg = tid + NT * i, co = seg / WSEG, s16 = seg % WSEG;
            wreg[i] = *reinterpret_cast<const i32x4*>(w3 + ((size_t)co * 14 + 2 * ky) * (32 * EB) + s16 * 16);
        }
    };
    auto store_w = [&](int slot) {
#pragma unroll
        for (int i = 0; i < NWSEG; ++i) {
            const int seg = tid + NT * i, co = seg / WSEG, s16 = seg % WSEG;
            *reinterpret_cast<i32x4*>(Ws + (slot * 64 + co) * WROW + s16 * 8) = wreg[i];
        }
    };

    if (t_beg < t_end) load_x(t_beg, true);
    for (int tile = t_beg; tile < t_end; ++tile) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
        load_w(0);
        int e_tile = F16_EMIN;
        if constexpr (H16) {
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < NRAW; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(raw[k][e]));
            m = wave_max(m);
            if (lane == 0) stem_red[wave] = m;
        }
        __syncthreads();                                            // the previous tile's fragment reads are done
        if constexpr (H16) {
            float m = 0.f;
#pragma unroll
            for (int w8 = 0; w8 < 8; ++w8) m = fmaxf(m, stem_red[w8]);
            e_tile = max((int)(__builtin_bit_cast(unsigned, m) >> 23), F16_EMIN);
            a_scale = f16_scale_of(e_tile);
        }
        store_x();
        store_w(0);
        __syncthreads();
        f32x16 acc[2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[nt][e] = 0.f;
#pragma unroll
        for (int ky = 0; ky < KH; ++ky) {
            if (ky + 1 < KH) load_w(ky + 1);
            if (ky == KH - 3) load_x(min(tile + 1, t_end - 1), tile + 1 < t_end);       // (lands under the last tap rows)
            const unsigned short* W = Ws + (ky & 1) * 64 * WROW;
#pragma unroll
            for (int kx = 0; kx < KW; ++kx) {
                frag_t bw[2][NP];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        bw[nt][q] = *reinterpret_cast<const frag_t*>(W + (nt * 32 + l32) * WROW + ((kx >> 1) * NP + q) * 32 + (kx & 1) * 16 + h * 8);
                const int row = 2 * wave + ky;
                frag_t a[NP];
#pragma unroll
                for (int q = 0; q < NP; ++q) a[q] = *reinterpret_cast<const frag_t*>(Xs + (row * XW + l32 + kx) * PIT + q * 16 + h * 8);
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa) {
                            if constexpr (H16) acc[nt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[qa], bw[nt][ord - qa], acc[nt], 0, 0, 0);
                            else acc[nt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[qa], bw[nt][ord - qa], acc[nt], 0, 0, 0);
                        }
            }
            if (ky + 1 < KH) {
                store_w((ky + 1) & 1);                              // the slot tap row ky - 1 was read from: every wave is past the barrier behind it
                __syncthreads();
            }
        }
        if constexpr (H16) {                                        // back to the operands' units (exact)
            const float inv = f16_inv_scale_of(e_tile) * p.w2s[0];
            acc[0] *= inv; acc[1] *= inv;
        }
        // epilogue: C layout of the 32 x 32 tile: column (channel) = lane & 31, row (pixel) = (reg & 3) + 8 * (reg >> 2) + 4 * (lane >> 5)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            const int co = nt * 32 + l32;
            const float sc = scale ? scale[co] : 1.f, sh = shift ? shift[co] : 0.f;
            float* orow = y + (((size_t)b * p.Ho + ty0 + wave) * p.Wo + tx0) * 64 + co;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = (e & 3) + 8 * (e >> 2) + 4 * h;
                orow[(size_t)m * 64] = apply_act(acc[nt][e] * sc + sh, p.act);
            }
        }
        if (p.ex_stat == 1) {
            // the tile's statistics for the train-mode BatchNorm behind the stem (ConvP.ex_stat 1: shift = the tile's first pixel, sum (z - shift),
            // sum (z - shift)^2 per channel; no scale / shift in that configuration): 16 values per lane, the other half-wave by a shuffle,
            // the eight waves (= output rows of the tile) in LDS in a fixed order -- instead of a 400 MB pass over the stem's output
            float* st_sh = reinterpret_cast<float*>(lds16 + XH * XW * PIT + 2 * 64 * WROW);      // [64] shift, then [8 waves][2][64] partial sums
            float* st_part = st_sh + 64;
            if (wave == 0 && h == 0) { st_sh[l32] = acc[0][0]; st_sh[32 + l32] = acc[1][0]; }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const float s0 = st_sh[nt * 32 + l32];
                float a = 0.f, q = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) { const float d = acc[nt][e] - s0; a += d; q += d * d; }
                a += __shfl_xor(a, 32, 64); q += __shfl_xor(q, 32, 64);
                if (h == 0) { st_part[(wave * 2 + 0) * 64 + nt * 32 + l32] = a; st_part[(wave * 2 + 1) * 64 + nt * 32 + l32] = q; }
            }
            __syncthreads();
            if (tid < 64) {
                float a = 0.f, q = 0.f;
#pragma unroll
                for (int w8 = 0; w8 < 8; ++w8) { a += st_part[(w8 * 2 + 0) * 64 + tid]; q += st_part[(w8 * 2 + 1) * 64 + tid]; }
                float* dst = p.ex_part + (size_t)tile * 3 * 64 + tid;
                dst[0] = st_sh[tid]; dst[64] = a; dst[128] = q;
            }
        }
    }
}

// ---------------------------------------------------------------------------------- 3x3 layers of 16 / 32 channels, split arithmetic
// The full-resolution tail of the depth decoder (models/depth_head.py:60-71: 32 -> 16 and 16 -> 16 at 256 x 512 and 512 x 1024) ran on
// the f32 MFMA in conv_igemm16_kernel / conv_igemm_kernel<f32>: 45-68 TFLOP/s of 157 and 0.8-2.1 TB/s -- neither roof.  With 16
// channels a K-step of v_mfma_f32_16x16x32_bf16 is TWO TAPS x 16 channels (k group kg of a lane: tap 2 s + (kg >> 1), channels
// 8 (kg & 1) ..): five steps for the nine taps, the tenth half-step against zero weights.  The A fragment of a lane is then 8
// consecutive channels of ITS pixel shifted by ITS tap -- an aligned 16-byte read at a per-lane address of the halo tile, which is split
// into the three bf16 pieces once for all nine taps ([pixel][piece][16 channels], 112-byte pitch).  The weights (<= 32 x 9 x 32
// floats) never touch LDS: every lane builds its B fragments from the fp32 pack once per block (persistent over its tiles) and keeps
// them in registers (60 per 16 x 16 channel block).  Block = 8 x 32 output pixels, wave = two rows = four 16-pixel row tiles; the next
// tile's loads are in flight under the MFMAs; the epilogue goes through LDS so that stores are 16 bytes per lane and the epilogue extras
// (gates 1 / 2, column sums) are the common code.  MODE_DGRAD: the same kernel on the [ci][tap][co] pack with mirrored tap geometry.
// ARITH 16 (round 6): two fp16 pieces.  The weights' scale is found by the block itself (<= 9216 floats, once per persistent block: these
// packs are too small to carry the pack's slot), the activation tile's per tile (the sums start at zero with every tile).
template <int MODE, int NT, int KH, bool EX = false, int ARITH = 3>
__global__ __launch_bounds__(256, KH == 2 ? 1 : 2) void conv_halo3n16_kernel(ConvP p, int tiles_x, int tiles_y, int tiles_per_block, const float* __restrict__ x,
                                                                const float* __restrict__ wq, const float* __restrict__ scale,
                                                                const float* __restrict__ shift, const float* __restrict__ residual,
                                                                float* __restrict__ out) {
    constexpr int NP = ARITH == 16 ? 2 : 3;
    constexpr bool H16 = ARITH == 16;
    constexpr int TH = 8, TW = 32, XH = TH + 2, XW = TW + 2, PIT = NP * 16 + 8, CI = 16 * KH, CO = 16 * NT;
    __shared__ float n16_red[4];                                  // ARITH 16: the waves' largest magnitudes (weights once, then every tile)
    typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
    constexpr int NTASK = XH * XW * (CI / 4), NRAW = (NTASK + 255) / 256;
    constexpr int LDC = CO + 4;
    extern __shared__ __attribute__((aligned(16))) unsigned short lds16[];
    unsigned short* Xs = lds16;                                   // [KH][XH * XW][PIT]
    float* Cs = reinterpret_cast<float*>(lds16);                  // [256][LDC] (epilogue: aliases the activation tile)
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int Hm = (MODE == MODE_FWD) ? p.Ho : p.H, Wm = (MODE == MODE_FWD) ? p.Wo : p.W;      // (= the input's size: stride 1, pad 1)
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blockIdx.x * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    const size_t ximg = (size_t)Hm * Wm * CI;

    // ---- B fragments from the fp32 pack (row n: [tap][CI]); lane = (column l16, k group kg): tap 2 s + (kg >> 1), channels 8 (kg & 1) ..
    float w_scale = 1.f, w_inv = 1.f;
    if constexpr (H16) {
        float m = 0.f;
        for (int i = tid; i < CO * 9 * CI / 4; i += 256) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(wq + (size_t)i * 4);
            m = fmaxf(fmaxf(m, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
        }
        m = wave_max(m);
        if (lane == 0) n16_red[wave] = m;
        __syncthreads();
        m = fmaxf(fmaxf(n16_red[0], n16_red[1]), fmaxf(n16_red[2], n16_red[3]));
        __syncthreads();
        const int e = max((int)(__builtin_bit_cast(unsigned, m) >> 23), F16_EMIN);
        w_scale = f16_scale_of(e); w_inv = f16_inv_scale_of(e);
    }
    frag_t bfr[NT][KH][5][NP];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int hf = 0; hf < KH; ++hf)
#pragma unroll
            for (int st = 0; st < 5; ++st) {
                const int tap = 2 * st + (kg >> 1);
                f32x4 w0 = {0.f, 0.f, 0.f, 0.f}, w1 = {0.f, 0.f, 0.f, 0.f};
                if (tap < 9) {
                    const float* wp = wq + ((size_t)(j * 16 + l16) * 9 + tap) * CI + hf * 16 + (kg & 1) * 8;
                    w0 = *reinterpret_cast<const f32x4*>(wp);
                    w1 = *reinterpret_cast<const f32x4*>(wp + 4);
                }
                u16x4 p0[NP], p1[NP];
                if constexpr (H16) { split_f16(w0, w_scale, p0[0], p0[1]); split_f16(w1, w_scale, p1[0], p1[1]); }
                else { split_bf16<NP>(w0, p0); split_bf16<NP>(w1, p1); }
#pragma unroll
                for (int q = 0; q < NP; ++q) bfr[j][hf][st][q] = __builtin_bit_cast(frag_t, pack8(p0[q], p1[q]));
            }
    // ---- A fragment offsets (halfwords) of this lane's tap per K-step: forward pixel + (ky, kx), data gradient pixel + (2 - ky, 2 - kx)
    int aoff[5];
#pragma unroll
    for (int st = 0; st < 5; ++st) {
        const int tap = min(2 * st + (kg >> 1), 8);                // (the tenth half-step multiplies zero weights: any valid address)
        const int ky = tap / 3, kx = tap % 3;
        const int gy = (MODE == MODE_FWD) ? ky : 2 - ky, gx = (MODE == MODE_FWD) ? kx : 2 - kx;
        aoff[st] = (gy * XW + gx) * PIT + (kg & 1) * 8;
    }

    // ---- staging tasks: (halo pixel pc, channel quad c4); thread tid owns tasks tid + 256 k
    int t_off[NRAW], t_rc[NRAW], t_dst[NRAW];                       // t_rc: halo row << 8 | halo column (one register: this kernel is at its register limit)
#pragma unroll
    for (int k = 0; k < NRAW; ++k) {
        const int t = tid + 256 * k, c4 = t % (CI / 4), pc = t / (CI / 4), c = pc % XW, r = pc / XW;
        t_rc[k] = ((t < NTASK ? r : 1 << 20) << 8) | c;            // (a row no image has)
        t_off[k] = ((r * Wm + c) * CI + c4 * 4) * 4;
        t_dst[k] = (c4 / 4) * (XH * XW * PIT) + pc * PIT + (c4 % 4) * 4;
    }
    f32x4 raw[NRAW];
    auto load_x = [&](int tile, bool valid) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);             // (scalar)
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(x + (size_t)b * ximg, ximg * 4);
        const int iy0 = ty0 - 1, ix0 = tx0 - 1, org = (iy0 * Wm + ix0) * CI * 4;
#pragma unroll
        for (int k = 0; k < NRAW; ++k) {
            const bool ok = valid && (unsigned)(iy0 + (t_rc[k] >> 8)) < (unsigned)Hm && (unsigned)(ix0 + (t_rc[k] & 255)) < (unsigned)Wm;
            const unsigned vo = ok ? (unsigned)(org + t_off[k]) : GATHER_OOB;
            raw[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, 0, 0));
        }
    };
    float a_scale = 1.f;
    auto store_x = [&]() {
#pragma unroll
        for (int k = 0; k < NRAW; ++k) {
            if (tid + 256 * k >= NTASK) continue;
            u16x4 pc[NP];
            if constexpr (H16) split_f16(raw[k], a_scale, pc[0], pc[1]);
            else split_bf16<NP>(raw[k], pc);
#pragma unroll
            for (int q = 0; q < NP; ++q) *reinterpret_cast<u16x4*>(Xs + t_dst[k] + q * 16) = pc[q];
        }
    };

    // epilogue roles: thread = (column quad c4e, row r0e + RPASS k)
    constexpr int V4 = CO / 4, RPASS = 256 / V4, NROW = 256 / RPASS;
    const int c4e = tid % V4, r0e = tid / V4, n = c4e * 4;
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (MODE == MODE_FWD && n < p.N) {
        if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    }

    if (t_beg < t_end) load_x(t_beg, true);
    for (int tile = t_beg; tile < t_end; ++tile) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
        int e_tile = F16_EMIN;
        if constexpr (H16) {                                        // this tile's largest magnitude (its loads have had the previous tile to land)
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < NRAW; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(raw[k][e]));
            m = wave_max(m);
            if (lane == 0) n16_red[wave] = m;
        }
        __syncthreads();                                            // the previous tile's epilogue has read Cs
        if constexpr (H16) {
            const float m = fmaxf(fmaxf(n16_red[0], n16_red[1]), fmaxf(n16_red[2], n16_red[3]));
            e_tile = max((int)(__builtin_bit_cast(unsigned, m) >> 23), F16_EMIN);
            a_scale = f16_scale_of(e_tile);
        }
        store_x();
        __syncthreads();
        load_x(min(tile + 1, t_end - 1), tile + 1 < t_end);         // in flight under the MFMAs and the epilogue
        f32x4 acc[4][NT];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[m][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hf = 0; hf < KH; ++hf)
#pragma unroll
            for (int st = 0; st < 5; ++st)
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int base = ((2 * wave + (m >> 1)) * XW + (m & 1) * 16 + l16) * PIT + hf * (XH * XW * PIT) + aoff[st];
                    frag_t a[NP];
#pragma unroll
                    for (int q = 0; q < NP; ++q) a[q] = *reinterpret_cast<const frag_t*>(Xs + base + q * 16);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                            for (int qa = 0; qa <= ord; ++qa) {
                                if constexpr (H16) acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[qa], bfr[j][hf][st][ord - qa], acc[m][j], 0, 0, 0);
                                else acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[qa], bfr[j][hf][st][ord - qa], acc[m][j], 0, 0, 0);
                            }
                }
        __syncthreads();                                            // every wave is done with the activation tile: Cs may overwrite it
        // C layout of a 16 x 16 tile: column = l16, row = 4 kg + reg; tile row index = pixel (yy * 32 + xx) of the 8 x 32 tile
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    Cs[((2 * wave + (m >> 1)) * TW + (m & 1) * 16 + 4 * kg + r) * LDC + j * 16 + l16] =
                        H16 ? acc[m][j][r] * (f16_inv_scale_of(e_tile) * w_inv) : acc[m][j][r];
        __syncthreads();
        f32x4 colsum = {0.f, 0.f, 0.f, 0.f};                        // (extras of this kernel: gates 1 / 2 and statistics 2 only -- written out here:
        if (n < p.N) {                                              //  the common EpiCtx keeps 28 registers live that this kernel does not have)
            // residual / gate rows: requested before the stores (see EpiPre), four rows at a time (two in the 32-column form, which is at its register limit)
            constexpr int CH = NT == 2 ? 2 : 4;
#pragma unroll
            for (int k0 = 0; k0 < NROW; k0 += CH) {
            f32x4 resv[CH], gv[CH];
#pragma unroll
            for (int kk = 0; kk < CH; ++kk) {
                const int k = k0 + kk;
                const int rr = r0e + k * RPASS;
                const size_t idx = (((size_t)b * Hm + ty0 + rr / TW) * Wm + tx0 + rr % TW) * p.N + n;
                resv[kk] = residual ? *reinterpret_cast<const f32x4*>(residual + idx) : f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (EX) gv[kk] = p.ex_gate_act ? *reinterpret_cast<const f32x4*>(p.ex_gate + idx) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int kk = 0; kk < CH; ++kk) {
                const int k = k0 + kk;
                const int rr = r0e + k * RPASS;                     // pixel of the tile
                const size_t idx = (((size_t)b * Hm + ty0 + rr / TW) * Wm + tx0 + rr % TW) * p.N + n;
                f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * LDC + c4e * 4);
                if (MODE == MODE_FWD) {
                    v = v * sc + sh;
                    if (residual) v += resv[kk];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
                } else if (residual) {                              // data gradient + the gradient that reached the same tensor by another path
                    v += resv[kk];
                }
                if constexpr (EX) {
                    if (p.ex_gate_act) {                            // = epi_apply's gates 1 / 2
                        const f32x4 g = gv[kk];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] *= g[e] > 0.f ? 1.f : (p.ex_gate_act == 2 ? g[e] + 1.f : 0.f);
                    }
                    colsum += v;
                }
                *reinterpret_cast<f32x4*>(out + idx) = v;
            }
            }
        }
        if constexpr (EX) {
            if (p.ex_stat == 2) {                                   // = epi_flush for statistics 2: the tile's column sums, fixed order
                f32x4* red = reinterpret_cast<f32x4*>(Cs + 256 * LDC);      // (behind the C tile: the activation tile's space, free until the next store_x)
                __syncthreads();
                red[tid] = colsum;
                __syncthreads();
                if (tid < V4 && n < p.N) {
                    f32x4 a = {0.f, 0.f, 0.f, 0.f};
                    for (int k = 0; k < RPASS; ++k) a += red[k * V4 + tid];
                    *reinterpret_cast<f32x4*>(p.ex_part + (size_t)(p.ex_tile0 + tile) * p.N + n) = a;
                }
            }
        }
    }
}

template <int MODE, int BK, bool EX = false>
__global__ __launch_bounds__(256) void conv_igemm16_kernel(ConvP p, const float* __restrict__ a0, const float* __restrict__ a1,
                                                           const float* __restrict__ wq, const float* __restrict__ scale,
                                                           const float* __restrict__ shift, const float* __restrict__ residual,
                                                           float* __restrict__ out) {
    constexpr int BM = 256, TM = 4, G = BK / 16;
    __shared__ __attribute__((aligned(16))) float Cs[BM * 20];
    extern __shared__ __attribute__((aligned(16))) float smem[];         // gather table [sources][taps][BM]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.x * BM;
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;
    const int ntap = (MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW;
    const int steps_per_tap = Kc / BK, nsteps = ntap * steps_per_tap;
    unsigned* tab = reinterpret_cast<unsigned*>(smem);
    __amdgpu_buffer_rsrc_t rs0, rs1;
    build_gather<MODE, BM>(p, m0, ntap, tab, a0, a1, rs0, rs1, parity_class(p));
    // weight row of this lane's column; columns past N read row N - 1 (their results are never stored)
    const float* brow = wq + (size_t)min(l16, p.N - 1) * p.KH * p.KW * Kc + q * 4;
    const int rrow = wave * 64 + l16;                            // this lane's row in tile i: rrow + 16 * i

    auto load_step = [&](int step, f32x4 (&af)[TM][G], f32x4 (&bf)[G]) {
        const int tap = step / steps_per_tap, cstep = (step - tap * steps_per_tap) * BK;
        const bool s1 = MODE == MODE_FWD && cstep >= p.C0;
        const __amdgpu_buffer_rsrc_t rs = s1 ? rs1 : rs0;
        const unsigned coff = (unsigned)((s1 ? cstep - p.C0 : cstep) + q * 4) * 4u;
        const unsigned* t = tab + ((s1 ? ntap : 0) + tap) * BM + rrow;
        const int koff = ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? (tap % (p.KH * p.KW)) : tap) * Kc + cstep;
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const unsigned off = t[16 * i] + coff;
#pragma unroll
            for (int g = 0; g < G; ++g)
                af[i][g] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + g * 64, 0, 0));
        }
#pragma unroll
        for (int g = 0; g < G; ++g) bf[g] = *reinterpret_cast<const f32x4*>(brow + koff + g * 16);
    };

    f32x4 acc[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 a_cur[TM][G], b_cur[G], a_nxt[TM][G], b_nxt[G];
    load_step(0, a_cur, b_cur);
    for (int step = 0; step < nsteps; ++step) {
        if (step + 1 < nsteps) load_step(step + 1, a_nxt, b_nxt);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a_cur[i][g][e], b_cur[g][e], acc[i], 0, 0, 0);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            b_cur[g] = b_nxt[g];
#pragma unroll
            for (int i = 0; i < TM; ++i) a_cur[i][g] = a_nxt[i][g];
        }
    }
    // epilogue through LDS: C layout col = lane&15, row = (lane>>4)*4 + reg  ->  one float4 per (row, 4 columns)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) Cs[(wave * 64 + i * 16 + q * 4 + r) * 20 + l16] = acc[i][r];
    __syncthreads();
    const int c4 = tid & 3, r0 = tid >> 2;                   // 4 float4 per row, 64 rows per pass
    const int n = c4 * 4;
    EpiCtx ec;
    if constexpr (EX) epi_begin(p, ec, p.ex_img_rows ? m0 / p.ex_img_rows : 0, n);
    if (n < p.N) {
        f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
        if (MODE == MODE_FWD) {
            if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
            if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
        }
        if constexpr (EX) if (p.ex_stat == 1) ec.sh = *reinterpret_cast<const f32x4*>(Cs + n) * sc + sh;
#pragma unroll
        for (int rr = r0; rr < BM; rr += 64) {
            const int m = m0 + rr;
            if (m >= p.M) break;
            f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * 20 + n);
            if (MODE == MODE_FWD) {
                v = v * sc + sh;
                if (residual) v += *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
            } else if (residual) {
                v += *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n);
            }
            *reinterpret_cast<f32x4*>(out + (size_t)m * p.N + n) = epi_apply_t<EX>(p, ec, v, (size_t)m * p.N + n);
        }
    }
    if constexpr (EX) epi_flush(p, ec, Cs, tid, 4, 64, blockIdx.x, n);
}

// LDS-staged flavour of the 16-column kernel for deep K (e.g. the 240-channel GUDA conv): full 128-B row segments are
// fetched once per K-step by 8 adjacent lanes and re-read from LDS as fragments, which keeps the texture path off the
// critical path when K per tap is large; the register-direct flavour above wins for the K = 144 decoder tail.
template <int MODE, int BK, bool EX = false>
__global__ __launch_bounds__(256) void conv_igemm16_lds_kernel(ConvP p, const float* __restrict__ a0, const float* __restrict__ a1,
                                                               const float* __restrict__ wq, const float* __restrict__ scale,
                                                               const float* __restrict__ shift, const float* __restrict__ residual,
                                                               float* __restrict__ out) {
    constexpr int BM = 256, BN = 16, TM = 4;
    constexpr int LDK = BK + 4, CPR = BK / 4, RPP = 256 / CPR, APASS = BM / RPP;
    __shared__ __attribute__((aligned(16))) float As[2][BM * LDK];
    __shared__ __attribute__((aligned(16))) float Bs[2][BN * LDK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m0 = blockIdx.x * BM;
    const int chunk = tid % CPR, rbase = tid / CPR;
    int rb[APASS], ry[APASS], rx[APASS];
#pragma unroll
    for (int i = 0; i < APASS; ++i) {
        const int m = m0 + rbase + RPP * i;
        if (m < p.M) {
            const bool upd = MODE == MODE_DGRAD && p.up0 && p.src == 0;
            const int HWm = (MODE == MODE_FWD) ? p.Ho * p.Wo : (upd ? (p.H / 2) * (p.W / 2) : p.H * p.W);
            const int Wm = (MODE == MODE_FWD) ? p.Wo : (upd ? p.W / 2 : p.W);
            rb[i] = m / HWm;
            const int rem = m % HWm;
            ry[i] = rem / Wm; rx[i] = rem % Wm;
        } else { rb[i] = -1; ry[i] = 0; rx[i] = 0; }
    }
    const int Kc = (MODE == MODE_FWD) ? p.Ct : p.Co;
    const float* brow = nullptr;
    if (tid < BN * CPR && tid / CPR < p.N) brow = wq + (size_t)(tid / CPR) * p.KH * p.KW * Kc + chunk * 4;
    const int ntap = (MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW;
    const int steps_per_tap = Kc / BK, nsteps = ntap * steps_per_tap;
    f32x4 areg[APASS], breg;
    auto load_step = [&](int step) {
        const int tap = step / steps_per_tap, cstep = (step % steps_per_tap) * BK;
        int ky, kx, qy = 0, qx = 0;
        if (MODE == MODE_DGRAD && p.up0 && p.src == 0) {
            const int qq = tap / (p.KH * p.KW), t2 = tap % (p.KH * p.KW);
            qy = qq >> 1; qx = qq & 1; ky = t2 / p.KW; kx = t2 % p.KW;
        } else { ky = tap / p.KW; kx = tap % p.KW; }
        if (MODE == MODE_FWD) {
            const bool s1 = cstep >= p.C0;
            const float* src = s1 ? a1 : a0;
            const int cs = s1 ? p.C1 : p.C0, c = (s1 ? cstep - p.C0 : cstep) + chunk * 4;
            const bool up = p.up0 && !s1;
            const int Hs = up ? p.H / 2 : p.H, Ws = up ? p.W / 2 : p.W;
#pragma unroll
            for (int i = 0; i < APASS; ++i) {
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
                if (rb[i] >= 0) {
                    int iy = ry[i] * p.stride - p.pad + ky, ix = rx[i] * p.stride - p.pad + kx;
                    if (p.pad_mode == 1) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
                    if (iy >= 0 && iy < p.H && ix >= 0 && ix < p.W) {
                        if (up) { iy >>= 1; ix >>= 1; }
                        v = *reinterpret_cast<const f32x4*>(src + (((size_t)rb[i] * Hs + iy) * Ws + ix) * cs + c);
                    }
                }
                areg[i] = v;
            }
        } else {
            const int c = cstep + chunk * 4;
#pragma unroll
            for (int i = 0; i < APASS; ++i) {
                f32x4 v = {0.f, 0.f, 0.f, 0.f};
                if (rb[i] >= 0) {
                    int iy = ry[i], ix = rx[i];
                    if (p.up0 && p.src == 0) { iy = 2 * iy + qy; ix = 2 * ix + qx; }
                    int ty = iy + p.pad - ky, tx = ix + p.pad - kx;
                    bool ok = ty >= 0 && tx >= 0;
                    if (p.stride == 2) { ok = ok && !(ty & 1) && !(tx & 1); ty >>= 1; tx >>= 1; }
                    if (ok && ty < p.Ho && tx < p.Wo)
                        v = *reinterpret_cast<const f32x4*>(a0 + (((size_t)rb[i] * p.Ho + ty) * p.Wo + tx) * p.Co + c);
                }
                areg[i] = v;
            }
        }
        const int koff = ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? (tap % (p.KH * p.KW)) : tap) * Kc + cstep;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (brow) v = *reinterpret_cast<const f32x4*>(brow + koff);
        breg = v;
    };
    auto store_step = [&](int buf) {
#pragma unroll
        for (int i = 0; i < APASS; ++i) *reinterpret_cast<f32x4*>(&As[buf][(rbase + RPP * i) * LDK + chunk * 4]) = areg[i];
        if (tid < BN * CPR) *reinterpret_cast<f32x4*>(&Bs[buf][(tid / CPR) * LDK + chunk * 4]) = breg;
    };
    f32x4 acc[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    load_step(0);
    store_step(0);
    __syncthreads();
    const int l16 = lane & 15, q = lane >> 4;
    for (int step = 0; step < nsteps; ++step) {
        const int buf = step & 1;
        if (step + 1 < nsteps) load_step(step + 1);
        const float* Ab = &As[buf][(wave * 64 + l16) * LDK + q * 4];
        const float* Bb = &Bs[buf][l16 * LDK + q * 4];
#pragma unroll
        for (int g = 0; g < BK / 16; ++g) {
            const f32x4 bf = *reinterpret_cast<const f32x4*>(Bb + g * 16);
            f32x4 af[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) af[i] = *reinterpret_cast<const f32x4*>(Ab + i * 16 * LDK + g * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < TM; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(af[i][e], bf[e], acc[i], 0, 0, 0);
        }
        if (step + 1 < nsteps) store_step(buf ^ 1);
        __syncthreads();
    }
    float* Cs = &As[0][0];                                   // [256][20]
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) Cs[(wave * 64 + i * 16 + q * 4 + r) * 20 + l16] = acc[i][r];
    __syncthreads();
    const int c4 = tid & 3, r0 = tid >> 2;
    const int n = c4 * 4;
    EpiCtx ec;
    if constexpr (EX) epi_begin(p, ec, p.ex_img_rows ? m0 / p.ex_img_rows : 0, n);
    if (n < p.N) {
        f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
        if (MODE == MODE_FWD) {
            if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
            if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
        }
        if constexpr (EX) if (p.ex_stat == 1) ec.sh = *reinterpret_cast<const f32x4*>(Cs + n) * sc + sh;
#pragma unroll
        for (int rr = r0; rr < BM; rr += 64) {
            const int m = m0 + rr;
            if (m >= p.M) break;
            f32x4 v = *reinterpret_cast<const f32x4*>(Cs + rr * 20 + n);
            if (MODE == MODE_FWD) {
                v = v * sc + sh;
                if (residual) v += *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], p.act);
            } else if (residual) {
                v += *reinterpret_cast<const f32x4*>(residual + (size_t)m * p.N + n);
            }
            *reinterpret_cast<f32x4*>(out + (size_t)m * p.N + n) = epi_apply_t<EX>(p, ec, v, (size_t)m * p.N + n);
        }
    }
    if constexpr (EX) epi_flush(p, ec, Cs, tid, 4, 64, blockIdx.x, n);
}

// ---------------------------------------------------------------------------------- wgrad
// dW[co][tap][ci] partial over a pixel range.  A = dZ^T (LDS [k=pixel][m=co]), B = X(tap) (LDS [k][n=ci]).
struct WgradP {
    int B, H, W, C0, C1, Ct, up0, Co, Ho, Wo, KH, KW, stride, pad, pad_mode, stride_w, pad_w;
    int n_mt, n_nt, splits, pix_per_split, P;     // P = B*Ho*Wo output pixels
    int fast;                                     // wgrad_halo64s_kernel: the layer-wide conditions of its FAST address path hold
    const float* in_aff;                          // wgrad_1x1s_kernel: x is the INPUT of a train-mode BatchNorm + ReLU, [image][mean | invstd | gamma | beta][Ct]
};

template <int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(256) void conv_wgrad_kernel(WgradP p, const float* __restrict__ x0,
                                                         const float* __restrict__ x1, const float* __restrict__ dz,
                                                         float* __restrict__ part) {
    constexpr int KS = 4 / (WM * WN);              // narrow tiles: the spare waves split K (pixel rows) inside the block
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, BKP = KS == 4 ? 32 : 16;   // pixels per K-step
    constexpr int LDM = BM + 4, LDN = BN + 4;
    extern __shared__ __attribute__((aligned(16))) float smem[];
    float* As = smem;                        // [2][BKP][LDM]
    float* Bs = smem + 2 * BKP * LDM;        // [2][BKP][LDN]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wt = wave % (WM * WN), kw = wave / (WM * WN);      // tile position, K-split lane of this wave
    const int wm = wt / WN, wn = wt % WN;
    // block -> (tile group g = (split, nt, mt), tap): the KH*KW tap blocks of one group read the same dZ rows and the same
    // (shifted) X rows, so they are given consecutive-by-8 block ids = the same XCD, close in dispatch order: the
    // operands come from HBM once and from that XCD's L2 for the other taps (measured before: 9x the HBM reads)
    const int ntap = p.KH * p.KW, Gt = p.splits * p.n_nt * p.n_mt, G8 = (Gt / 8) * 8;
    int g, tap;
    if ((int)blockIdx.x < G8 * ntap) {
        const int chunk = blockIdx.x / (8 * ntap), r = blockIdx.x % (8 * ntap);
        tap = r / 8; g = chunk * 8 + (r % 8);
    } else {
        const int r = blockIdx.x - G8 * ntap, rest = Gt - G8;
        tap = r / rest; g = G8 + r % rest;
    }
    const int split = g % p.splits;
    const int nt = (g / p.splits) % p.n_nt;
    const int mt = g / (p.splits * p.n_nt);
    const int ky = tap / p.KW, kx = tap % p.KW;
    const int m0 = mt * BM, n0 = nt * BN;
    const int pbeg = split * p.pix_per_split, pend = min(pbeg + p.pix_per_split, p.P);

    // loader mapping: A: BKP x BM floats, 16-B chunks along m;  B: BKP x BN along n
    constexpr int ACH = BM / 4, BCH = BN / 4;                 // chunks per pixel row
    constexpr int AIT = (BKP * ACH + 255) / 256, BIT = (BKP * BCH + 255) / 256;
    f32x4 areg[AIT], breg[BIT];

    // No division, bounds branch or source decision inside the K loop (they used to cost more issue slots than the
    // MFMAs): every thread keeps the pixel coordinates of its chunks and steps them by BKP pixels per K-step.
    //   A (dZ, dense rows): buffer_load through a resource that ends at this split's last pixel -> the tail reads 0.
    //   B (x gathered through this block's tap): global_load from the pixel address, or from zero_page when the tap
    //     falls into the padding / past the split (select on the address, loads are unconditional).
    const __amdgpu_buffer_rsrc_t rsA = make_rsrc(dz + (size_t)pbeg * p.Co, (size_t)max(pend - pbeg, 0) * p.Co * 4);
    unsigned a_off[AIT];
#pragma unroll
    for (int i = 0; i < AIT; ++i) {
        const int idx = tid + 256 * i, kr = idx / ACH, m = m0 + (idx % ACH) * 4;
        a_off[i] = (idx < BKP * ACH && m < p.Co) ? (unsigned)(kr * p.Co + m) * 4u : GATHER_OOB;
    }
    const unsigned a_stride = (unsigned)(BKP * p.Co) * 4u;
    const float* b_src[BIT];
    int b_x[BIT], b_y[BIT], b_b[BIT];
    bool b_s1[BIT], b_okn[BIT];
    int pix0 = pbeg + tid / BCH;                               // pixel of chunk 0; chunk i sits 256 * i / BCH pixels further
#pragma unroll
    for (int i = 0; i < BIT; ++i) {
        const int idx = tid + 256 * i, kr = idx / BCH, n = n0 + (idx % BCH) * 4;
        b_okn[i] = idx < BKP * BCH && n < p.Ct;
        b_s1[i] = n >= p.C0;
        b_src[i] = b_s1[i] ? x1 + (n - p.C0) : x0 + n;
        const int pix = pbeg + kr;
        b_b[i] = pix / (p.Ho * p.Wo);
        const int rem = pix % (p.Ho * p.Wo);
        b_y[i] = rem / p.Wo; b_x[i] = rem % p.Wo;
    }

    auto load_step = [&](int step) {
#pragma unroll
        for (int i = 0; i < AIT; ++i) {
            const unsigned off = a_off[i] == GATHER_OOB ? GATHER_OOB : a_off[i] + (unsigned)step * a_stride;
            areg[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsA, off, 0, 0));
        }
#pragma unroll
        for (int i = 0; i < BIT; ++i) {
            int iy = b_y[i] * p.stride - p.pad + ky, ix = b_x[i] * p.stride_w - p.pad_w + kx;
            if (p.pad_mode == 1) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
            const bool ok = b_okn[i] && pix0 + (256 * i) / BCH < pend && iy >= 0 && iy < p.H && ix >= 0 && ix < p.W;
            const bool up = p.up0 && !b_s1[i];
            const int sh = up ? 1 : 0;
            const int Hs = p.H >> sh, Ws = p.W >> sh, cs = b_s1[i] ? p.C1 : p.C0;
            const float* ptr = b_src[i] + (size_t)(unsigned)((b_b[i] * Hs + (iy >> sh)) * Ws + (ix >> sh)) * cs;
            breg[i] = *reinterpret_cast<const f32x4*>(ok ? ptr : zero_page);
            // advance this chunk's pixel by BKP (branch-free; rows narrower than BKP take the uniform slow path)
            if (p.Wo >= BKP) {
                b_x[i] += BKP;
                const bool wx = b_x[i] >= p.Wo;
                b_x[i] -= wx ? p.Wo : 0; b_y[i] += wx ? 1 : 0;
                const bool wy = b_y[i] >= p.Ho;
                b_y[i] -= wy ? p.Ho : 0; b_b[i] += wy ? 1 : 0;
            } else {
                const int pix = pix0 + (256 * i) / BCH + BKP;
                b_b[i] = pix / (p.Ho * p.Wo);
                const int rem = pix % (p.Ho * p.Wo);
                b_y[i] = rem / p.Wo; b_x[i] = rem % p.Wo;
            }
        }
        pix0 += BKP;
    };
    auto store_step = [&](int buf) {
#pragma unroll
        for (int i = 0; i < AIT; ++i) {
            const int idx = tid + 256 * i;
            if (idx < BKP * ACH) *reinterpret_cast<f32x4*>(As + buf * BKP * LDM + (idx / ACH) * LDM + (idx % ACH) * 4) = areg[i];
        }
#pragma unroll
        for (int i = 0; i < BIT; ++i) {
            const int idx = tid + 256 * i;
            if (idx < BKP * BCH) *reinterpret_cast<f32x4*>(Bs + buf * BKP * LDN + (idx / BCH) * LDN + (idx % BCH) * 4) = breg[i];
        }
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int nsteps = (pend - pbeg + BKP - 1) / BKP;
    const int lrow = lane & 31, lhalf = lane >> 5;
    if (nsteps > 0) {
        load_step(0);
        store_step(0);
        __syncthreads();
        for (int step = 0; step < nsteps; ++step) {
            const int buf = step & 1;
            if (step + 1 < nsteps && CODEPS_ABLATE < 1) load_step(step + 1);
            const float* Ab = As + buf * BKP * LDM + wm * TM * 32 + lrow;
            const float* Bb = Bs + buf * BKP * LDN + wn * TN * 32 + lrow;
#pragma unroll
            for (int g = 0; g < BKP / 8; ++g) {
                if (KS > 1 && (g % KS) != kw) continue;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int kr = g * 8 + lhalf * 4 + e;
                    float af[TM], bf[TN];
#if CODEPS_ABLATE >= 3
#pragma unroll
                    for (int i = 0; i < TM; ++i) af[i] = (float)(kr + i + step);
#pragma unroll
                    for (int j = 0; j < TN; ++j) bf[j] = (float)(kr - j);
#else
#pragma unroll
                    for (int i = 0; i < TM; ++i) af[i] = Ab[kr * LDM + i * 32];
#pragma unroll
                    for (int j = 0; j < TN; ++j) bf[j] = Bb[kr * LDN + j * 32];
#endif
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(af[i], bf[j], acc[i][j], 0, 0, 0);
                }
            }
#if CODEPS_ABLATE >= 2
            continue;
#endif
            if (step + 1 < nsteps) store_step(buf ^ 1);
            __syncthreads();
        }
    }
    if (KS > 1) {                                  // fixed-order sum of the K-split waves through LDS
        static_assert(KS == 1 || BM * BN <= 2 * BKP * (LDM + LDN), "reduction tile must fit in the staging LDS");
        float* red = smem;
        for (int w = 0; w < KS; ++w) {
            __syncthreads();
            if (kw != w) continue;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        float* d = red + (((wm * TM + i) * 32 + (r & 3) + 8 * (r >> 2) + 4 * lhalf) * BN) + (wn * TN + j) * 32 + lrow;
                        const float v = (w == 0 ? 0.f : *d) + acc[i][j][r];
                        if (w == KS - 1) acc[i][j][r] = v; else *d = v;
                    }
        }
        if (kw != KS - 1) return;                  // the last K-split wave holds the block's total
    }
    // partial slab [split][co][tap][ci]
    float* dst = part + (size_t)split * p.Co * p.KH * p.KW * p.Ct;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = n0 + (wn * TN + j) * 32 + lrow;
        if (n >= p.Ct) continue;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + (wm * TM + i) * 32 + (r & 3) + 8 * (r >> 2) + 4 * lhalf;
                if (m < p.Co) dst[((size_t)m * p.KH * p.KW + tap) * p.Ct + n] = acc[i][j][r];
            }
    }
}

// ---------------------------------------------------------------------------------- wgrad of 1x1 convolutions, split arithmetic
// dW[co][ci] = sum over pixels dZ[pix][co] X[pix'][ci] (pix' = pix, or the stride-2 sample of a down-sampling shortcut): a GEMM whose K
// is the pixel axis, the SLOW axis of both NHWC operands.  conv_wgrad_kernel runs it on v_mfma_f32_32x32x2f32 (1/16 of the bf16 rate:
// 50-60 us per bottleneck convolution of the pre-training configurations, 2.6 ms per step).  Here, as in wgrad_halo64s_kernel: a task
// is 8 consecutive pixels x 4 channels (eight 16-byte loads, 64 contiguous bytes per pixel over four lanes), split into the three bf16
// pieces in registers and written TRANSPOSED -- per channel and piece the 8 pixels as one 16-byte LDS store -- so that the fragments
// of v_mfma_f32_32x32x16_bf16 (8 consecutive k per lane) are aligned 16-byte reads.  Block = 256 channels of the wider operand (A) x
// 128 (TB = 2) or 64 (TB = 1) of the other (B) x K-steps of 32 pixels; wave = 128 x (TB x 32).  The tile is that large because every
// block streams its A and B rows over ALL its pixels: a 128 x 64 tile (the first form of this kernel) moved ~200 MB per layer through
// the memory system whatever the layer and ran at the f32 kernel's speed (60-70 us, ~3.3 TB/s).  The next K-step's loads are in flight
// under the MFMAs.  SWAP: A = X, B = dZ (Ci > Co).  One partial slab [co][ci] per block, summed in a fixed order by wgrad_reduce_kernel.
// ARITH 16 (round 6): two fp16 pieces; both operands are activations, each with a running block-local scale: the waves publish the largest
// exponent of the K-step they hold in registers in front of the barrier that precedes its LDS stores.
// (three pieces at TB = 1 need 264 - 272 registers: one wave per SIMD.  Two would spill 72 - 88 bytes and are no faster, per call with the reduction: B4 128 x 256,
// 64 -> 256 channels 64.5 / 66.3 us, 256 -> 64 66.2 / 70.3 us)
template <bool SWAP, int TB, int ARITH = 3>
__global__ __launch_bounds__(256, TB == 1 && ARITH == 16 ? 2 : 1) void wgrad_1x1s_kernel(WgradP p, const float* __restrict__ x, const float* __restrict__ dz,
                                                                          float* __restrict__ part) {
    constexpr int NP = ARITH == 16 ? 2 : 3;
    constexpr bool H16 = ARITH == 16;
    typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
    __shared__ int w1_slots[8];                              // ARITH 16: [operand][wave] largest exponents of the K-step in flight
    constexpr int KP = 32, ZP = NP * KP + 8;                  // pixels per K-step; halfwords per channel row (pad: conflict-free fragment reads)
    constexpr int TA = 4, BA = 2 * TA * 32, BB = 2 * TB * 32;
    constexpr int NBT = BB / 4 * (KP / 8);                   // B tasks per K-step (A: 256)
    extern __shared__ __attribute__((aligned(16))) unsigned short lds16[];
    unsigned short* As = lds16;                             // [BA][ZP]
    unsigned short* Bs = lds16 + BA * ZP;                   // [BB][ZP]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, h = lane >> 5;
    const int wa = wave >> 1, wb = wave & 1;                // wave tile: A channels wa * 128 .., B channels wb * TB * 32 ..
    const int CA = SWAP ? p.Ct : p.Co, CB = SWAP ? p.Co : p.Ct;
    const int n_bt = (CB + BB - 1) / BB;
    const int a0 = (blockIdx.y / n_bt) * BA, b0 = (blockIdx.y % n_bt) * BB;
    const int split = blockIdx.x;
    const int pbeg = split * p.pix_per_split, pend = min(pbeg + p.pix_per_split, p.P);
    const bool strided = p.stride != 1 || p.stride_w != 1;

    // Loads without branches: buffer loads whose byte offset is GATHER_OOB (-> zeros from the hardware range check) for pixels behind
    // the slab's end and channels behind the operand's last -- sixteen `if (ok) load` made sixteen exec-mask regions per K-step, and the
    // first form of this kernel spent its time there (434 v_mul_lo_u32 and 187 s_cbranch_execz in 4300 instructions, 60 TF/s).
    const __amdgpu_buffer_rsrc_t rs_x = make_rsrc(x, (size_t)p.B * p.H * p.W * p.Ct * 4), rs_z = make_rsrc(dz, (size_t)p.P * p.Co * 4);
    const __amdgpu_buffer_rsrc_t rs_a = SWAP ? rs_x : rs_z, rs_b = SWAP ? rs_z : rs_x;
    // tasks: A 64 quads x 4 pixel groups = 256 (thread tid), B (BB / 4) x 4 = 128 / 64 (the first threads).  Task -> (quad, group): the
    // quad's low two bits over four consecutive lanes (64 contiguous bytes per pixel), then the pixel group, then the quad's high bits
    const int t_c4 = (tid & 3) | ((tid >> 4) << 2), t_g = (tid >> 2) & 3;
    const bool b_on = tid < NBT;
    const int ca = a0 + t_c4 * 4, cb = b0 + t_c4 * 4;
    const bool a_ok = ca < CA, b_ok = b_on && cb < CB;
    // element offset of output pixel q in X (dZ: q * Co)
    auto x_pix = [&](int q) -> unsigned {
        if (!strided) return (unsigned)q * (unsigned)p.Ct;
        const int b = q / (p.Ho * p.Wo), rem = q % (p.Ho * p.Wo);
        return (unsigned)(((b * p.H + (rem / p.Wo) * p.stride) * p.W + (rem % p.Wo) * p.stride_w)) * (unsigned)p.Ct;
    };
    f32x4 ra[8], rb[8];
    // in_aff: x = BatchNorm's input; this thread's channel quad of the K-step's image (K-steps lie inside one image: codeps_conv2d_in_affine_ok)
    f32x4 nmu, nis, nga, nbe;
    int q_cur = pbeg;
    const int cx = SWAP ? ca : cb;
    const bool x_ok = SWAP ? a_ok : b_ok;
    auto load_step = [&](int q0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int qa = q0 + t_g * 8 + i;
            const bool ok = qa < pend;
            const unsigned ox = x_pix(qa), oz = (unsigned)qa * (unsigned)p.Co;
            const unsigned va = (ok && a_ok) ? ((SWAP ? ox : oz) + ca) * 4u : GATHER_OOB;
            const unsigned vb = (ok && b_ok) ? ((SWAP ? oz : ox) + cb) * 4u : GATHER_OOB;
            ra[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs_a, va, 0, 0));
            rb[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs_b, vb, 0, 0));     // (threads without a B task: out of range, no traffic)
        }
        if (p.in_aff) {
            const float* t = p.in_aff + (size_t)(q0 / (p.Ho * p.Wo)) * 4 * p.Ct + (x_ok ? cx : 0);
            nmu = *reinterpret_cast<const f32x4*>(t); nis = *reinterpret_cast<const f32x4*>(t + p.Ct);
            nga = *reinterpret_cast<const f32x4*>(t + 2 * p.Ct); nbe = *reinterpret_cast<const f32x4*>(t + 3 * p.Ct);
            q_cur = q0;
        }
    };
    auto normalise = [&](f32x4 (&r)[8]) {                       // relu(BatchNorm(x)) in registers; pixels behind the slab's end stay zero
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const f32x4 v = bn_norm_relu(r[i], nmu, nis, nga, nbe);
            r[i] = (x_ok && q_cur + t_g * 8 + i < pend) ? v : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    auto store_task = [&](const f32x4 (&r)[8], unsigned short* dst, float sc) {      // dst = row of the quad's first channel, at this pixel group
        u16x4 pc[8][NP];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (H16) split_f16(r[i], sc, pc[i][0], pc[i][1]);
            else split_bf16<NP>(r[i], pc[i]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const u16x4 lo = {pc[0][q][e], pc[1][q][e], pc[2][q][e], pc[3][q][e]}, hi = {pc[4][q][e], pc[5][q][e], pc[6][q][e], pc[7][q][e]};
                *reinterpret_cast<i32x4*>(dst + e * ZP + q * KP) = pack8(lo, hi);
            }
    };

    f32x16 acc[TA][TB];
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int nsteps = (pend - pbeg + KP - 1) / KP;
    if (nsteps > 0) load_step(pbeg);
    int ea_run = F16_EMIN, eb_run = F16_EMIN;
    for (int step = 0; step < nsteps; ++step) {
        float sa = 1.f, sb = 1.f;
        if (p.in_aff) { if constexpr (SWAP) normalise(ra); else normalise(rb); }
        if constexpr (H16) {
            float ma = 0.f, mb = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) { ma = fmaxf(ma, fabsf(ra[i][e])); mb = fmaxf(mb, fabsf(rb[i][e])); }
            const int xa = wave_max_exponent(ma), xb = wave_max_exponent(mb);
            if (lane == 0) { w1_slots[wave] = xa; w1_slots[4 + wave] = xb; }
        }
        __syncthreads();                                     // the previous K-step's fragment reads are done
        if constexpr (H16) {
            const i32x4 pa = *reinterpret_cast<const i32x4*>(w1_slots), pb = *reinterpret_cast<const i32x4*>(w1_slots + 4);
            const int ea = __builtin_amdgcn_readfirstlane(max(max(max(pa[0], pa[1]), max(pa[2], pa[3])), ea_run));
            const int eb = __builtin_amdgcn_readfirstlane(max(max(max(pb[0], pb[1]), max(pb[2], pb[3])), eb_run));
            if (ea + eb != ea_run + eb_run) {                // re-base the sums to the larger tiles' scales (exact)
                const float rbs = f16_rebase(ea_run + eb_run, ea + eb);
#pragma unroll
                for (int i = 0; i < TA; ++i)
#pragma unroll
                    for (int j = 0; j < TB; ++j) acc[i][j] *= rbs;
            }
            ea_run = ea; eb_run = eb;
            sa = f16_scale_of(ea); sb = f16_scale_of(eb);
        }
        store_task(ra, As + (t_c4 * 4) * ZP + t_g * 8, sa);
        if (b_on) store_task(rb, Bs + (t_c4 * 4) * ZP + t_g * 8, sb);
        __syncthreads();
        if (step + 1 < nsteps) load_step(pbeg + (step + 1) * KP);
#pragma unroll
        for (int ks = 0; ks < KP / 16; ++ks) {
            frag_t fb[TB][NP];
#pragma unroll
            for (int j = 0; j < TB; ++j)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    fb[j][q] = *reinterpret_cast<const frag_t*>(Bs + ((wb * TB + j) * 32 + l32) * ZP + q * KP + ks * 16 + h * 8);
#pragma unroll
            for (int i = 0; i < TA; ++i) {
                frag_t fa[NP];
#pragma unroll
                for (int q = 0; q < NP; ++q) fa[q] = *reinterpret_cast<const frag_t*>(As + ((wa * TA + i) * 32 + l32) * ZP + q * KP + ks * 16 + h * 8);
#pragma unroll
                for (int j = 0; j < TB; ++j)
#pragma unroll
                    for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa) {
                            // (the lanes of the result run along the SECOND operand: always the input channels, the slab's fast axis)
                            if constexpr (H16)
                                acc[i][j] = SWAP ? __builtin_amdgcn_mfma_f32_32x32x16_f16(fb[j][ord - qa], fa[qa], acc[i][j], 0, 0, 0)
                                                 : __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[qa], fb[j][ord - qa], acc[i][j], 0, 0, 0);
                            else
                                acc[i][j] = SWAP ? __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[j][ord - qa], fa[qa], acc[i][j], 0, 0, 0)
                                                 : __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[qa], fb[j][ord - qa], acc[i][j], 0, 0, 0);
                        }
            }
        }
    }
    // partial slab [split][co][ci]; C layout: column = lane & 31 (ci), row = (reg & 3) + 8 * (reg >> 2) + 4 * (lane >> 5) (co)
    float* dst = part + (size_t)split * p.Co * p.Ct;
    const float inv = H16 ? f16_inv_scale_of(ea_run) * f16_inv_scale_of(eb_run) : 1.f;
#pragma unroll
    for (int j = 0; j < TB; ++j)
#pragma unroll
        for (int i = 0; i < TA; ++i) {
            const int ta = a0 + (wa * TA + i) * 32, tb = b0 + (wb * TB + j) * 32;          // first A / B channel of this 32 x 32 tile
            const int ci = (SWAP ? ta : tb) + l32;
            if (ci >= p.Ct) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int co = (SWAP ? tb : ta) + (r & 3) + 8 * (r >> 2) + 4 * h;
                if (co < p.Co) dst[(size_t)co * p.Ct + ci] = H16 ? acc[i][j][r] * inv : acc[i][j][r];
            }
        }
}

// ---------------------------------------------------------------------------------- wgrad, small channel counts
// Weight gradient of stride-1 1x1 / 3x3 convs with <= 32 output channels (the full-resolution decoder tail, the
// disparity / class convs, the 240-channel GUDA conv): K (= pixels) is huge and the output is tiny, so the generic
// one-tap-per-block kernel above is latency bound.  Here a block walks over 8x32 pixel tiles; per tile the dZ tile
// and ONE halo tile of X (a 32-channel chunk) are staged in LDS and every tap reads its shifted window from that halo
// (X is fetched once instead of once per tap); each wave owns 64 of the 256 pixels and keeps all (m-tile, n-tile, tap)
// accumulators of v_mfma_f32_16x16x4_f32 in registers across tiles; per-wave partial slabs, fixed-order reduce.
template <int MT, int NT, int KH, int KW, int SH, int SW, int TH, int TW>
__global__ __launch_bounds__(256) void wgrad_small_kernel(WgradP p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                          const float* __restrict__ x0, const float* __restrict__ x1,
                                                          const float* __restrict__ dz, float* __restrict__ part) {
    constexpr int XH = (TH - 1) * SH + KH, XW = (TW - 1) * SW + KW, TAPS = KH * KW, PIX = TH * TW;
    static_assert(PIX % 64 == 0 && (PIX * MT * 4) % 256 == 0, "tile must give every wave whole MFMA k-steps");
    const int co_base = blockIdx.y * MT * 16;                    // output-channel group of this block (stem: 4 groups of 16)
    constexpr int LDZ = MT * 16 + 4, LDX = NT * 16 + 4;
    constexpr int SLAB = MT * 16 * TAPS * NT * 16;              // floats of one block slab (cross-wave reduction buffer)
    constexpr int STAGE = TH * TW * LDZ + XH * XW * LDX;
    __shared__ __attribute__((aligned(16))) float lds_all[STAGE > SLAB ? STAGE : SLAB];
    float* dZs = lds_all;
    float* Xs = lds_all + TH * TW * LDZ;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
    const int chunk = blockIdx.x % ci_chunks, blk = blockIdx.x / ci_chunks;
    const int c_base = chunk * NT * 16;                         // first input channel of this block's chunk
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    // source of this channel chunk (chunks never straddle the two concat sources: C0 is a multiple of NT*16 or C1 == 0)
    const bool s1 = c_base >= p.C0;
    const float* src = s1 ? x1 : x0;
    const int cs = s1 ? p.C1 : p.C0, c_src = s1 ? c_base - p.C0 : c_base;
    const bool up = p.up0 && !s1;
    const int Hs = up ? p.H / 2 : p.H, Ws = up ? p.W / 2 : p.W;

    f32x4 acc[MT][NT][TAPS];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int t = 0; t < TAPS; ++t) acc[a][b][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    // in_aff (1x1 only): x is the INPUT of a train-mode BatchNorm + ReLU; a thread's channel quad is the same for all its loads (NT * 4 divides
    // 256), its four BatchNorm vectors are reloaded when the tile's image changes
    f32x4 nmu = {0.f, 0.f, 0.f, 0.f}, nis = nmu, nga = nmu, nbe = nmu;
    int n_img = -1;
    for (int tile = t_beg; tile < t_end; ++tile) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
        if constexpr (TAPS == 1 && 256 % (NT * 4) == 0) {
            if (p.in_aff && b != n_img) {
                const int cq = c_src + (tid % (NT * 4)) * 4;
                const float* t = p.in_aff + (size_t)b * 4 * p.Ct + (cq < cs ? cq : 0);
                nmu = *reinterpret_cast<const f32x4*>(t); nis = *reinterpret_cast<const f32x4*>(t + p.Ct);
                nga = *reinterpret_cast<const f32x4*>(t + 2 * p.Ct); nbe = *reinterpret_cast<const f32x4*>(t + 3 * p.Ct);
                n_img = b;
            }
        }
        // all global loads of the tile are issued into registers first, then written to LDS (one latency, not one per
        // element: a load -> ds_write pair per loop iteration would wait for every load separately)
        constexpr int NZ = PIX * MT * 4 / 256, NX = (XH * XW * NT * 4 + 255) / 256;
        f32x4 zr[NZ], xr_[NX];
#pragma unroll
        for (int u = 0; u < NZ; ++u) {                          // dZ tile: [pixel][MT*16] as float4
            const int i = tid + 256 * u;
            const int pix = i / (MT * 4), c4 = i % (MT * 4);
            const int gy = ty0 + pix / TW, gx = tx0 + pix % TW;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (gy < p.Ho && gx < p.Wo && co_base + c4 * 4 < p.Co)
                v = *reinterpret_cast<const f32x4*>(dz + (((size_t)b * p.Ho + gy) * p.Wo + gx) * p.Co + co_base + c4 * 4);
            zr[u] = v;
        }
#pragma unroll
        for (int u = 0; u < NX; ++u) {                          // X halo tile: [position][NT*16] as float4
            const int i = tid + 256 * u;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (i < XH * XW * NT * 4) {
                const int pos = i / (NT * 4), c4 = i % (NT * 4);
                int iy = ty0 * SH + pos / XW - p.pad, ix = tx0 * SW + pos % XW - p.pad_w;
                if (p.pad_mode == 1) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
                if (iy >= 0 && iy < p.H && ix >= 0 && ix < p.W && c_src + c4 * 4 < cs) {
                    if (up) { iy >>= 1; ix >>= 1; }
                    v = *reinterpret_cast<const f32x4*>(src + (((size_t)b * Hs + iy) * Ws + ix) * cs + c_src + c4 * 4);
                    if constexpr (TAPS == 1 && 256 % (NT * 4) == 0) { if (p.in_aff) v = bn_norm_relu(v, nmu, nis, nga, nbe); }
                }
            }
            xr_[u] = v;
        }
        __syncthreads();                                        // previous tile's MFMAs are done with the LDS
#pragma unroll
        for (int u = 0; u < NZ; ++u) {
            const int i = tid + 256 * u;
            *reinterpret_cast<f32x4*>(dZs + (i / (MT * 4)) * LDZ + (i % (MT * 4)) * 4) = zr[u];
        }
#pragma unroll
        for (int u = 0; u < NX; ++u) {
            const int i = tid + 256 * u;
            if (i < XH * XW * NT * 4) *reinterpret_cast<f32x4*>(Xs + (i / (NT * 4)) * LDX + (i % (NT * 4)) * 4) = xr_[u];
        }
        __syncthreads();
#pragma unroll 4
        for (int j = 0; j < PIX / 16; ++j) {                    // MFMA k-steps of 4 pixels over this wave's PIX/4 pixels
            const int pix = wave * (PIX / 4) + j * 4 + q;
            const int py = pix / TW, px = pix % TW;
            float af[MT];
#pragma unroll
            for (int a = 0; a < MT; ++a) af[a] = dZs[pix * LDZ + a * 16 + l16];
#pragma unroll
            for (int ky = 0; ky < KH; ++ky)
#pragma unroll
                for (int kx = 0; kx < KW; ++kx) {
                    const float* xr = Xs + ((py * SH + ky) * XW + px * SW + kx) * LDX + l16;
#pragma unroll
                    for (int bb = 0; bb < NT; ++bb) {
                        const float bv = xr[bb * 16];
#pragma unroll
                        for (int a = 0; a < MT; ++a)
                            acc[a][bb][ky * KW + kx] = __builtin_amdgcn_mfma_f32_16x16x4f32(af[a], bv, acc[a][bb][ky * KW + kx], 0, 0, 0);
                    }
                }
        }
    }
    // cross-wave sum through LDS, then ONE partial slab [co][tap][ci] per block.
    // C layout: column (ci) = lane&15, row (co) = (lane>>4)*4 + reg
    float* red = lds_all;
    for (int w = 0; w < 4; ++w) {                               // waves add their accumulators in turn (fixed order)
        __syncthreads();
        if (wave != w) continue;
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int bb = 0; bb < NT; ++bb)
#pragma unroll
                for (int t = 0; t < TAPS; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float* d = red + ((a * 16 + q * 4 + r) * TAPS + t) * (NT * 16) + bb * 16 + l16;
                        *d = (w == 0 ? 0.f : *d) + acc[a][bb][t][r];
                    }
    }
    __syncthreads();
    float* dst = part + (size_t)blk * p.Co * TAPS * p.Ct;
    for (int i = tid; i < SLAB; i += 256) {
        const int cl = i % (NT * 16), t = (i / (NT * 16)) % TAPS, co = i / (NT * 16 * TAPS);
        const int ci = c_base + cl;
        if (co_base + co < p.Co && ci < p.Ct) dst[((size_t)(co_base + co) * TAPS + t) * p.Ct + ci] = red[i];
    }
}

// wgrad_halo64_kernel on the bf16 matrix cores (same tiles, same grid, same partial-sum layout; CODEPS_WGRAD_SPLIT).
// The weight gradient contracts over PIXELS, and v_mfma_f32_32x32x16_bf16 wants 8 consecutive k values per lane, so both
// operands are transposed while they are staged: a thread loads 8 pixels x 4 channels (eight 16-byte loads), splits each
// channel's 8 values into the three bf16 pieces and writes one 16-byte LDS row segment per (channel, piece):
//   dZs [64 co][piece][64 px]              X rows: [64 ci][piece][6 rows][ -1 | 16 px | 16 ] at elements 7 | 8..23 | 24
// A tap (ky, kx) reads X row py + ky at column offset kx - 1: the kx = 1 fragment is an aligned 16-byte read, the other two
// are built in registers from the neighbouring aligned groups (v_alignbit, 4 per fragment) -- no unaligned LDS access, no
// second copy of the tile.  Every X row's fragments are read once per tile and used by the up to three (py, ky) pairs that
// touch it: 66 fragment reads for 216 MFMAs (9 taps x 6 piece products x 4 k-chunks) per wave and tile.
// CO32 (layers with <= 32 output channels: the decoders' 1/2-resolution stages): one 32-row co tile, so the waves that would hold
// the second co tile split the PIXELS instead -- wave = (pixel half ph, ci tile): output rows 2 ph, 2 ph + 1 of every tile -- and
// each pixel half writes its own partial slab (the slab reduction sums them like any other split).
// This is the GENERIC body (reflect padding, ragged maps, a chunk split between the sources elsewhere than at 32): per-pixel address
// arithmetic behind exec-mask branches -- stamped in the diagnostic build (-DCODEPS_WG_STAMP_LOADS), issuing a tile's 17 loads that way
// is 22-25 % of a block's lifetime, the split + store phase another 20 %.  Every block of the shipped configurations takes
// wgrad_halo64d_body below instead.
template <bool CO32>
__device__ __forceinline__ void wgrad_halo64s_body(const WgradP& p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                   const float* __restrict__ x0, const float* __restrict__ x1,
                                                   const float* __restrict__ dz, float* __restrict__ part, unsigned short* lds16) {
    constexpr int TH = 4, TW = 16, XH = TH + 2, PIX = TH * TW, XROW = 32;
    constexpr int ZP = 3 * PIX + 8;                    // halfwords per dZ channel (pad: conflict-free 16-byte fragment reads)
    constexpr int XQ = XH * XROW, XP = 3 * XQ + 8;     // halfwords per X piece / per X channel
    unsigned short* dZs = lds16;                       // [64][ZP]
    unsigned short* Xs = lds16 + 64 * ZP;              // [64][XP]
    CODEPS_STAMP_BEGIN();
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, h = lane >> 5;
    const int wco = CO32 ? 0 : (wave & 1), wci = wave >> 1;
    const int ph = __builtin_amdgcn_readfirstlane(wave & 1);       // CO32: this wave's pixel half
    const int co_base = blockIdx.y * 64;
    const int chunk = blockIdx.x % ci_chunks, blk = blockIdx.x / ci_chunks;
    const int c_base = chunk * 64;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    // source of a channel quad of this chunk (a 64-channel chunk may straddle the two concat sources: picked per quad)
    auto src_of = [&](int c4, const float*& src, int& cs, int& c_src, bool& up) {
        const int ch = c_base + c4 * 4;
        const bool s1 = ch >= p.C0;
        src = s1 ? x1 : x0;
        cs = s1 ? p.C1 : p.C0;
        c_src = s1 ? ch - p.C0 : ch;
        up = p.up0 && !s1;
    };

    f32x16 acc[9];
#pragma unroll
    for (int t = 0; t < 9; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

    // staging tasks: "big" = 8 pixels x 4 channels (128 dZ tasks, then 192 X tasks: 6 rows x 2 groups x 16 channel quads),
    // "small" = one halo pixel x 4 channels (6 rows x 2 sides x 16).  Thread tid owns big tasks tid and tid + 256 (< 320) and,
    // from thread 64 on, small task tid - 64.  Task -> (channel quad, pixel group): the quad's low two bits run over four
    // consecutive lanes (64 contiguous bytes per pixel in HBM), then the pixel group, then the quad's high bits -- with the
    // quad fastest, eight neighbouring lanes would write LDS rows 4 channels apart, which all fall on two bank groups.
    f32x4 bigr[2][8], smallr;
    auto task_of = [](int t, int ngrp, int& c4, int& grp) {               // t in [0, 16 * ngrp)
        c4 = (t & 3) | ((t / (4 * ngrp)) << 2);
        grp = (t >> 2) % ngrp;
    };
    // X task index of this thread's two big tasks (u = 0: threads 128.., u = 1: threads 0..63).  Opaque to the compiler on
    // purpose: with both written as bt - 128 it narrows the / 48 and % 12 to 16-bit multiplies of ONE register (tid - 128 and
    // tid + 128 agree in the low byte), hoists that out of the tile loop and feeds the u = 1 lanes 0xff80 + tid -- wrong
    // channel quads for a quarter of the X tile as soon as the per-quad source selection depends on them (ROCm 7.2 clang).
    int xt0 = tid - 128, xt1 = tid + 128;
    asm volatile("" : "+v"(xt0), "+v"(xt1));
    // eight consecutive pixels (iy, ix0 .. ix0 + 7) of the X source, 4 channels from c4 * 4; zero outside the image
    auto x_row8 = [&](int b, int iy, int ix0, int c4, f32x4 (&dst)[8]) {
        const float* src; int cs, c_src; bool up;
        src_of(c4, src, cs, c_src, up);
        const int Hs = up ? p.H / 2 : p.H, Ws = up ? p.W / 2 : p.W;
        if (p.pad_mode == 1) iy = reflect_idx(iy, p.H);
        const bool rowok = iy >= 0 && iy < p.H && c_src < cs;
        const float* rowp = src + ((size_t)b * Hs + (up ? iy >> 1 : iy)) * Ws * cs + c_src;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int ix = ix0 + i;
            if (p.pad_mode == 1) ix = reflect_idx(ix, p.W);
            const bool ok = rowok && ix >= 0 && ix < p.W;
            dst[i] = ok ? *reinterpret_cast<const f32x4*>(rowp + (size_t)(up ? ix >> 1 : ix) * cs) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    auto x_pixel = [&](int b, int iy, int ix, int c4) -> f32x4 {
        const float* src; int cs, c_src; bool up;
        src_of(c4, src, cs, c_src, up);
        const int Hs = up ? p.H / 2 : p.H, Ws = up ? p.W / 2 : p.W;
        if (p.pad_mode == 1) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
        if (iy >= 0 && iy < p.H && ix >= 0 && ix < p.W && c_src < cs) {
            if (up) { iy >>= 1; ix >>= 1; }
            return *reinterpret_cast<const f32x4*>(src + (((size_t)b * Hs + iy) * Ws + ix) * cs + c_src);
        }
        return f32x4{0.f, 0.f, 0.f, 0.f};
    };
    auto load_tile = [&](int tile) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int bt = tid + 256 * u;
            if (bt >= 320) break;
            int c4, grp;
            if (bt < 128) {                                          // dZ: channel quad c4, pixel group grp (8 per tile)
                task_of(bt, 8, c4, grp);
                const int gy = ty0 + (grp >> 1), gx0 = tx0 + (grp & 1) * 8;
                const bool rowok = gy < p.Ho && co_base + c4 * 4 < p.Co;
                const float* rowp = dz + (((size_t)b * p.Ho + gy) * p.Wo + gx0) * p.Co + co_base + c4 * 4;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    bigr[u][i] = (rowok && gx0 + i < p.Wo) ? *reinterpret_cast<const f32x4*>(rowp + (size_t)i * p.Co) : f32x4{0.f, 0.f, 0.f, 0.f};
            } else {                                                 // X interior: grp = row r * 2 + group g (12 per tile)
                task_of(u == 0 ? xt0 : xt1, 12, c4, grp);
                x_row8(b, ty0 + (grp >> 1) - 1, tx0 + (grp & 1) * 8, c4, bigr[u]);
            }
        }
        if (tid >= 64) {
            const int t = tid - 64, c4 = t & 15, rs = t >> 4, r = rs >> 1, side = rs & 1;
            smallr = x_pixel(b, ty0 + r - 1, tx0 + (side ? TW : -1), c4);
        }
    };
    auto store_tile = [&]() {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int bt = tid + 256 * u;
            if (bt >= 320) break;
            unsigned short* dst;                                     // element 0 of this task's 8-pixel segment, piece 0, channel c4 * 4
            int cstride, qstride, c4, grp;
            if (bt < 128) {
                task_of(bt, 8, c4, grp);
                dst = dZs + (c4 * 4) * ZP + grp * 8; cstride = ZP; qstride = PIX;
            } else {
                task_of(u == 0 ? xt0 : xt1, 12, c4, grp);
                dst = Xs + (c4 * 4) * XP + (grp >> 1) * XROW + 8 + (grp & 1) * 8; cstride = XP; qstride = XQ;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {                            // transpose in registers: channel e of the 8 pixels
                const f32x4 lo4 = {bigr[u][0][e], bigr[u][1][e], bigr[u][2][e], bigr[u][3][e]};
                const f32x4 hi4 = {bigr[u][4][e], bigr[u][5][e], bigr[u][6][e], bigr[u][7][e]};
                u16x4 lo[3], hi[3];
                split_bf16<3>(lo4, lo);
                split_bf16<3>(hi4, hi);
#pragma unroll
                for (int q = 0; q < 3; ++q) *reinterpret_cast<i32x4*>(dst + e * cstride + q * qstride) = pack8(lo[q], hi[q]);
            }
        }
        if (tid >= 64) {
            const int t = tid - 64, c4 = t & 15, rs = t >> 4, r = rs >> 1, side = rs & 1;
            u16x4 pc[3];
            split_bf16<3>(smallr, pc);
            unsigned short* dst = Xs + (c4 * 4) * XP + r * XROW + (side ? 24 : 7);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int q = 0; q < 3; ++q) dst[e * XP + q * XQ] = pc[q][e];
        }
    };

    if (t_beg < t_end) load_tile(t_beg);
    const unsigned short* zrow = dZs + (wco * 32 + l32) * ZP + h * 8;
    const unsigned short* xrow = Xs + (wci * 32 + l32) * XP + h * 8;
    for (int tile = t_beg; tile < t_end; ++tile) {
        CODEPS_STAMP_PHASE_START();
        __syncthreads();                                            // the previous tile's fragment reads are done
        store_tile();
        __syncthreads();
        CODEPS_STAMP_PHASE_B();                                     // B: barrier + (wait for the loads) split + transpose + LDS stores + barrier
        CODEPS_STAMP_PHASE_START();
        if (tile + 1 < t_end) load_tile(tile + 1);
#ifdef CODEPS_WG_STAMP_LOADS                                         // diagnostic split of phase A: A = issuing the next tile's loads only
        CODEPS_STAMP_PHASE_A();
#endif
        bf16x8 zf[TH][3];
#pragma unroll
        for (int py = 0; py < TH; ++py) {
            if (CO32 && (py >> 1) != ph) continue;                  // (wave-uniform)
#pragma unroll
            for (int q = 0; q < 3; ++q) zf[py][q] = *reinterpret_cast<const bf16x8*>(zrow + q * PIX + py * TW);
        }
#pragma unroll
        for (int r = 0; r < XH; ++r) {
            if (CO32 && (r < 2 * ph || r > 2 * ph + 3)) continue;   // X rows this wave's two output rows read
            bf16x8 xf[3][3];                                         // [kx][piece]
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const unsigned short* g0 = xrow + q * XQ + r * XROW;
                const i32x4 prev = *reinterpret_cast<const i32x4*>(g0), cur = *reinterpret_cast<const i32x4*>(g0 + 8),
                            next = *reinterpret_cast<const i32x4*>(g0 + 16);
                i32x4 left, right;
                left[0] = (int)__builtin_amdgcn_alignbit((unsigned)cur[0], (unsigned)prev[3], 16);
                right[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)cur[3], 16);
#pragma unroll
                for (int i = 1; i < 4; ++i) left[i] = (int)__builtin_amdgcn_alignbit((unsigned)cur[i], (unsigned)cur[i - 1], 16);
#pragma unroll
                for (int i = 0; i < 3; ++i) right[i] = (int)__builtin_amdgcn_alignbit((unsigned)cur[i + 1], (unsigned)cur[i], 16);
                xf[0][q] = __builtin_bit_cast(bf16x8, left);
                xf[1][q] = __builtin_bit_cast(bf16x8, cur);
                xf[2][q] = __builtin_bit_cast(bf16x8, right);
            }
#pragma unroll
            for (int ky = 0; ky < 3; ++ky) {
                const int py = r - ky;
                if (py < 0 || py >= TH) continue;
                if (CO32 && (py >> 1) != ph) continue;
#pragma unroll
                for (int kx = 0; kx < 3; ++kx)
#pragma unroll
                    for (int ord = 2; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa)
                            acc[ky * 3 + kx] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(zf[py][qa], xf[kx][ord - qa], acc[ky * 3 + kx], 0, 0, 0);
            }
        }
#ifndef CODEPS_WG_STAMP_LOADS
        CODEPS_STAMP_PHASE_A();                                     // A: next tile's loads issued + fragment reads + 216 MFMAs of this wave
#endif
    }
    // partial slab [blk][co][tap][ci]; C layout: column (ci) = lane & 31, row (co) = (reg & 3) + 8 * (reg >> 2) + 4 * (lane >> 5)
    float* dst = part + (size_t)(CO32 ? blk * 2 + ph : blk) * p.Co * 9 * p.Ct;
    const int ci = c_base + wci * 32 + l32;
    if (ci < p.Ct) {
#pragma unroll
        for (int t = 0; t < 9; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int co = co_base + wco * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
                if (co < p.Co) dst[((size_t)co * 9 + t) * p.Ct + ci] = acc[t][r];
            }
    }
    CODEPS_STAMP_END(conv);
}

#ifndef WG_FILL
#define WG_FILL 4                                       // staging instructions offered to the scheduler per MFMA (A/B builds: 3 and 5 measured slower)
#endif

// The blocks with constant-offset addressing (p.fast, see the kernel wrapper), double-buffered (wgrad_halo64s_body spends a quarter
// of a block's lifetime staging -- split, transpose, LDS stores between two barriers -- and as much issuing its loads, with the
// matrix pipe idle: one wave per SIMD, nothing else to issue).  Every address here is (scalar tile origin) + (per-thread constant),
// padding is the range check of the buffer resource (an offset past its end reads 0).  A 4 x 16
// tile is two 2 x 16 sub-tiles and LDS holds two of them (2 x 66 KB): while the waves run the 108 MFMAs of sub-tile j from one
// buffer, the same waves split and store sub-tile j + 1 into the other between those MFMAs (vector slots the MFMAs leave free) and
// issue the loads of sub-tile j + 2 into the second register set -- one barrier per sub-tile (in front of its last 18 MFMAs, which
// need registers only: the first fragment reads of the next sub-tile ride under them), no staging phase.  The price is the halo
// rows staged twice (4 X rows per 2 output rows instead of 6 per 4); the work is hidden, the extra reads hit L2.
// Tasks per sub-tile: 64 dZ (8 pixels x 4 channels; wave 0), 128 X interior (waves 1, 2), 128 halo pixels (two per lane; wave 3).
// The sub-tile loop exists three times, once per role: a wave runs its own staging instructions between its MFMAs, in one basic block
// (one shared instruction stream with the other roles' stores sent to a scrap area measured SLOWER than the single-buffered body: the
// LDS pipe was then busy longer than the matrix pipe).
// Sources: a chunk's 64 channels are two halves of 32 (quads 0-7, 8-15); each half lies in ONE source (host + kernel wrapper check:
// the concat boundary is at a multiple of 32 inside the chunk), which may be the up-sampled one (nearest, x 2: source pixel
// (y >> 1, x >> 1) -- a big task loads four pixels and uses each twice, every offset is still (scaled tile origin) + (per-thread
// constant)).  X interior: wave 1 stages half 0, wave 2 half 1; halo pixels: a lane's task 0 is in half 0, task 1 in half 1 -- so the
// source of every load instruction is wave-uniform and its up-sampling a compile-time property of the wave's code copy.
// CO32 (<= 32 output channels): one 32-row co tile; the waves that would hold the second one split the sub-tile's two output rows
// instead (wave = (row ph, ci tile), 54 MFMAs per sub-tile) and each row writes its own partial slab, as in wgrad_halo64s_body.
template <bool CO32>
__device__ __forceinline__ void wgrad_halo64d_body(const WgradP& p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                   const float* __restrict__ x0, const float* __restrict__ x1,
                                                   const float* __restrict__ dz, float* __restrict__ part, unsigned short* lds16) {
    constexpr int TH = 2, TW = 16, XH = TH + 2, PIX = TH * TW, XROW = 32;
    constexpr int ZP = 3 * PIX + 8;                    // halfwords per dZ channel (104: 52 dwords, conflict-free 16-byte fragment reads)
    constexpr int XQ = XH * XROW, XP = 3 * XQ + 8;     // halfwords per X piece / per X channel (392: 196 dwords)
    constexpr int XS0 = 64 * ZP;                       // X rows start behind the dZ rows
    constexpr int BUF = 64 * (ZP + XP);               // halfwords per buffer: [64][ZP] dZ, [64][XP] X
    CODEPS_STAMP_BEGIN();
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, h = lane >> 5;
    const int wco = CO32 ? 0 : (wave & 1), wci = wave >> 1;
    const int role = __builtin_amdgcn_readfirstlane(wave);            // 0: dZ, 1 / 2: X interior, 3: halo pixels
    const int co_base = blockIdx.y * 64;
    const int chunk = blockIdx.x % ci_chunks, blk = blockIdx.x / ci_chunks;
    const int c_base = chunk * 64;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    const int NJ = 2 * (t_end - t_beg);                               // sub-tiles of this block (even)
    // X source of a half of the chunk (block-uniform)
    struct XSrc { const float* ptr; int cs, c0; bool up; size_t img; };
    auto xsrc_of = [&](int half) {
        const int ch = c_base + 32 * half;
        const bool s1 = ch >= p.C0;
        XSrc o;
        o.ptr = s1 ? x1 : x0; o.cs = s1 ? p.C1 : p.C0; o.c0 = s1 ? ch - p.C0 : ch; o.up = p.up0 && !s1;
        o.img = o.up ? (size_t)(p.H / 2) * (p.W / 2) * o.cs : (size_t)p.H * p.W * o.cs;
        return o;
    };
    const XSrc xs[2] = {xsrc_of(0), xsrc_of(1)};

    f32x16 acc[9];
#pragma unroll
    for (int t = 0; t < 9; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

    // per-thread constants.  Big task (quad's low two bits over four consecutive lanes, then the pixel group, then the quad's high
    // bits: see wgrad_halo64s_body): global byte offset from the sub-tile origin, the X row it reads, LDS halfword of its first store
    int b_off = 0, b_row = 0, b_dst = 0;
    bool b_ok = false;
    if (role == 0) {
        const int c4 = (lane & 3) | ((lane >> 4) << 2), grp = (lane >> 2) & 3;
        b_off = (((grp >> 1) * p.Wo + (grp & 1) * 8) * p.Co + co_base + c4 * 4) * 4;
        b_ok = co_base + c4 * 4 < p.Co;
        b_dst = (c4 * 4) * ZP + grp * 8;
    } else if (role < 3) {
        const XSrc& sx = xs[role - 1];
        const int t = tid - 64, c4 = (t & 3) | ((t >> 5) << 2), c4l = c4 & 7, grp = (t >> 2) & 7;      // wave 1: quads 0-7, wave 2: 8-15
        b_row = (grp >> 1) - 1;
        b_off = sx.up ? (((b_row >> 1) * (p.W / 2) + (grp & 1) * 4) * sx.cs + sx.c0 + c4l * 4) * 4
                      : ((b_row * p.W + (grp & 1) * 8) * sx.cs + sx.c0 + c4l * 4) * 4;
        b_ok = sx.c0 + c4l * 4 < sx.cs;
        b_dst = XS0 + (c4 * 4) * XP + (grp >> 1) * XROW + 8 + (grp & 1) * 8;
    }
    int s_off[2] = {0, 0}, s_row = 0, s_dstk[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    unsigned s_selk[4] = {0, 0, 0, 0};
    bool s_ok[2] = {false, false}, s_side = false;
    if (role == 3) {
        const int c4l = lane & 7, rs = lane >> 3;                    // task u: quad c4l + 8 u, (row, side) rs
        s_side = rs & 1;
        s_row = (rs >> 1) - 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const XSrc& sx = xs[u];
            s_off[u] = sx.up ? (((s_row >> 1) * (p.W / 2) + (s_side ? TW / 2 : -1)) * sx.cs + sx.c0 + c4l * 4) * 4
                             : ((s_row * p.W + (s_side ? TW : -1)) * sx.cs + sx.c0 + c4l * 4) * 4;
            s_ok[u] = sx.c0 + c4l * 4 < sx.cs;
            const int dst = XS0 + ((c4l + 8 * u) * 4) * XP + (rs >> 1) * XROW + (s_side ? 24 : 7);
#pragma unroll
            for (int k = 0; k < 4; ++k) s_dstk[u][k] = dst + ((k + (c4l >> 1)) & 3) * XP;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = (k + (c4l >> 1)) & 3;
            s_selk[k] = 0x0c0c0000u | (e == 0 ? 0x0504u : e == 1 ? 0x0706u : e == 2 ? 0x0100u : 0x0302u);
        }
    }
    const size_t zimg = (size_t)p.Ho * p.Wo * p.Co;
    // cfg of a wave's code copy: bits 0-1 role (0: dZ, 1: X interior, 3: halo pixels), bit 2: the wave's source (role 1) / the source of
    // half 0 (role 3) is up-sampled, bit 3: role 3, the source of half 1 is up-sampled, bit 4: CO32, the wave's output row
    // the loads of sub-tile j (role 0, 1: eight 16-byte loads, four from an up-sampled source; 3: two halo pixels); all lanes read
    // zeros when !valid (the sub-tile behind the last one), so the tile loop has no branch around its loads
    auto issue_loads = [&](auto cfg_c, int j, bool valid, f32x4 (&raw)[8], unsigned tok = 0) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3;
        constexpr bool UPA = (CFG >> 2) & 1, UPB = (CFG >> 3) & 1;
        const int tile = t_beg + (j >> 1);                                                     // (all scalar)
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * 4 + (j & 1) * TH, tx0 = (tr % tiles_x) * TW;
        if (ROLE == 0) {
            const __amdgpu_buffer_rsrc_t rsz = make_rsrc(dz + (size_t)b * zimg, zimg * 4);
            const int zorg = (ty0 * p.Wo + tx0) * p.Co * 4, zpix = p.Co * 4;
            const unsigned vo = (valid && b_ok) ? (unsigned)(zorg + b_off) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsz, vo, i * zpix, 0));
        } else if (ROLE == 1) {
            const XSrc& sx = xs[role - 1];
            const __amdgpu_buffer_rsrc_t rsx = make_rsrc(sx.ptr + (size_t)b * sx.img, sx.img * 4);
            const int xorg = UPA ? ((ty0 / 2) * (p.W / 2) + tx0 / 2) * sx.cs * 4 : (ty0 * p.W + tx0) * sx.cs * 4, xpix = sx.cs * 4;
            const unsigned vo = (valid && b_ok && (unsigned)(ty0 + b_row) < (unsigned)p.H) ? (unsigned)(xorg + b_off) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < (UPA ? 4 : 8); ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsx, vo, i * xpix, 0));
        } else {
            const bool okp = valid && (unsigned)(ty0 + s_row) < (unsigned)p.H && (s_side ? tx0 + TW < p.W : tx0 > 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const XSrc& sx = xs[u];
                const bool up = u == 0 ? UPA : UPB;
                const __amdgpu_buffer_rsrc_t rsx = make_rsrc(sx.ptr + (size_t)b * sx.img, sx.img * 4);
                const int xorg = up ? ((ty0 / 2) * (p.W / 2) + tx0 / 2) * sx.cs * 4 : (ty0 * p.W + tx0) * sx.cs * 4;
                raw[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsx, ((okp && s_ok[u]) ? (unsigned)(xorg + s_off[u]) : GATHER_OOB) + tok, 0, 0));
            }
        }
    };
    // channel e of the big task: 8 pixels -> three 16-byte rows (one per piece)
    auto store_big = [&](auto cfg_c, const f32x4 (&raw)[8], int e, unsigned short* buf) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3;
        constexpr bool UPA = (CFG >> 2) & 1;
        constexpr int cs = ROLE == 0 ? ZP : XP, qs = ROLE == 0 ? PIX : XQ;
        if (UPA && ROLE == 1) {                                     // four source pixels, each twice
            const f32x4 v4 = {raw[0][e], raw[1][e], raw[2][e], raw[3][e]};
            u16x4 pc[3];
            split_bf16<3>(v4, pc);
#pragma unroll
            for (int q = 0; q < 3; ++q)
                *reinterpret_cast<i32x4*>(buf + b_dst + e * cs + q * qs) =
                    pack8(u16x4{pc[q][0], pc[q][0], pc[q][1], pc[q][1]}, u16x4{pc[q][2], pc[q][2], pc[q][3], pc[q][3]});
            return;
        }
        const f32x4 lo4 = {raw[0][e], raw[1][e], raw[2][e], raw[3][e]};
        const f32x4 hi4 = {raw[4][e], raw[5][e], raw[6][e], raw[7][e]};
        u16x4 lo[3], hi[3];
        split_bf16<3>(lo4, lo);
        split_bf16<3>(hi4, hi);
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<i32x4*>(buf + b_dst + e * cs + q * qs) = pack8(lo[q], hi[q]);
    };
    // a halo pixel's 2-byte stores: a channel's row starts 196 dwords behind its neighbour's (= 4 mod 32: what the 16-byte fragment reads
    // want), so the halo slots of all rows and channels fall on 16 of the 32 write banks -- 4-way at best.  With all lanes storing the
    // SAME channel of their quad the 64 addresses would fall on four to eight banks; so lane's k-th store takes channel
    // (k + (quad >> 1)) & 3 of its quad: 4 lanes per bank.
    struct SmallPc { unsigned lo[3], hi[3]; };                      // a halo pixel's 4 channels x 3 pieces, two halfwords per dword
    auto split_small = [&](const f32x4 v) {
        u16x4 pc[3];
        split_bf16<3>(v, pc);
        SmallPc o;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            o.lo[q] = (unsigned)pc[q][0] | ((unsigned)pc[q][1] << 16);
            o.hi[q] = (unsigned)pc[q][2] | ((unsigned)pc[q][3] << 16);
        }
        return o;
    };
    auto store_small = [&](const SmallPc& pc, int u, unsigned short* buf) {
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k)                              // v_perm_b32: bytes 0-3 = hi, 4-7 = lo (selector = byte numbers of the wanted halfword)
                buf[s_dstk[u][k] + q * XQ] = (unsigned short)__builtin_amdgcn_perm(pc.lo[q], pc.hi[q], s_selk[k]);
    };
    auto store_all = [&](auto cfg_c, const f32x4 (&raw)[8], unsigned short* buf) {
        constexpr int ROLE = decltype(cfg_c)::value & 3;
        if (ROLE == 3) { store_small(split_small(raw[0]), 0, buf); store_small(split_small(raw[1]), 1, buf); }
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) store_big(cfg_c, raw, e, buf);
        }
    };

    const int zoff = (wco * 32 + l32) * ZP + h * 8, xoff = XS0 + (wci * 32 + l32) * XP + h * 8;
    // fragments a phase starts with: the dZ rows and X row 0 of its buffer.  They are read by the PREVIOUS phase, right behind the
    // barrier that phase places in front of its last row's MFMAs (row 3: registers only) -- the LDS latency at the start of a sub-tile
    // disappears under those MFMAs
    struct Frag { bf16x8 zf[TH][3]; i32x4 x0[3][3]; };
    auto prefetch = [&](const unsigned short* buf, Frag& f) {
        const unsigned short* zrow = buf + zoff;
        const unsigned short* xrow = buf + xoff;
#pragma unroll
        for (int py = 0; py < TH; ++py)
#pragma unroll
            for (int q = 0; q < 3; ++q) f.zf[py][q] = *reinterpret_cast<const bf16x8*>(zrow + q * PIX + py * TW);
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            const unsigned short* g0 = xrow + q * XQ;
            f.x0[q][0] = *reinterpret_cast<const i32x4*>(g0);
            f.x0[q][1] = *reinterpret_cast<const i32x4*>(g0 + 8);
            f.x0[q][2] = *reinterpret_cast<const i32x4*>(g0 + 16);
        }
    };
    // one sub-tile: its MFMAs out of `cur`, the staging of the next one (registers rs, loaded a phase ago) into `nxt`, the loads of the
    // one after that into rl.  One copy of this code per cfg: a wave runs ITS staging instructions between the MFMAs and nothing else,
    // in one basic block
    auto phase = [&](auto cfg_c, int j, const f32x4 (&rs)[8], f32x4 (&rl)[8], const unsigned short* cur, unsigned short* nxt, Frag& fr) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3, PH = (CFG >> 4) & 1;
        // (halo role: split BEFORE the next loads are issued -- with the two old and the two new loads in flight together the compiler's
        //  wait in front of the split, vmcnt(1), also waited for the first NEW load: a memory latency per sub-tile, stamped per wave)
        SmallPc pc0 = {}, pc1 = {};
        unsigned tok = 0;                                           // (zero; makes the loads' offsets depend on the split's results: program order alone did not hold)
        if (ROLE == 3) {
            pc0 = split_small(rs[0]);
            pc1 = split_small(rs[1]);
            asm volatile("" : "+v"(tok) : "v"(pc0.lo[0]), "v"(pc0.lo[1]), "v"(pc0.lo[2]), "v"(pc0.hi[0]), "v"(pc0.hi[1]), "v"(pc0.hi[2]),
                                          "v"(pc1.lo[0]), "v"(pc1.lo[1]), "v"(pc1.lo[2]), "v"(pc1.hi[0]), "v"(pc1.hi[1]), "v"(pc1.hi[2]));
        }
        issue_loads(cfg_c, min(j + 2, NJ - 1), j + 2 < NJ, rl, tok);
        const unsigned short* xrow = cur + xoff;
        bf16x8 zf[TH][3];
        i32x4 xraw[2][3][3];                                        // [row parity][piece][prev | cur | next]
#pragma unroll
        for (int q = 0; q < 3; ++q) {
#pragma unroll
            for (int py = 0; py < TH; ++py) zf[py][q] = fr.zf[py][q];
#pragma unroll
            for (int i = 0; i < 3; ++i) xraw[0][q][i] = fr.x0[q][i];
        }
        auto read_row = [&](int r) {
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const unsigned short* g0 = xrow + q * XQ + r * XROW;
                xraw[r & 1][q][0] = *reinterpret_cast<const i32x4*>(g0);
                xraw[r & 1][q][1] = *reinterpret_cast<const i32x4*>(g0 + 8);
                xraw[r & 1][q][2] = *reinterpret_cast<const i32x4*>(g0 + 16);
            }
        };
#pragma unroll
        for (int r = 0; r < XH; ++r) {
            if (r + 1 < XH) read_row(r + 1);
            else {
                __syncthreads();                                    // every wave has read `cur` (row 3 is in registers) and written its part of `nxt`
                prefetch(nxt, fr);
            }
            __builtin_amdgcn_sched_barrier(0);
            // staging of the next sub-tile under the MFMAs of the two middle rows
            if (ROLE == 3) {
                if (r == 1) store_small(pc0, 0, nxt);
                if (r == 2) store_small(pc1, 1, nxt);
            } else {
                if (r == 1) { store_big(cfg_c, rs, 0, nxt); store_big(cfg_c, rs, 1, nxt); }
                if (r == 2) { store_big(cfg_c, rs, 2, nxt); store_big(cfg_c, rs, 3, nxt); }
            }
            bf16x8 xf[3][3];                                         // [kx][piece]
#pragma unroll
            for (int q = 0; q < 3; ++q) {
                const i32x4 prev = xraw[r & 1][q][0], curv = xraw[r & 1][q][1], next = xraw[r & 1][q][2];
                i32x4 left, right;
                left[0] = (int)__builtin_amdgcn_alignbit((unsigned)curv[0], (unsigned)prev[3], 16);
                right[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)curv[3], 16);
#pragma unroll
                for (int i = 1; i < 4; ++i) left[i] = (int)__builtin_amdgcn_alignbit((unsigned)curv[i], (unsigned)curv[i - 1], 16);
#pragma unroll
                for (int i = 0; i < 3; ++i) right[i] = (int)__builtin_amdgcn_alignbit((unsigned)curv[i + 1], (unsigned)curv[i], 16);
                xf[0][q] = __builtin_bit_cast(bf16x8, left);
                xf[1][q] = __builtin_bit_cast(bf16x8, curv);
                xf[2][q] = __builtin_bit_cast(bf16x8, right);
            }
            int n_mfma = 0;
#pragma unroll
            for (int ky = 0; ky < 3; ++ky) {
                const int py = r - ky;
                if (py < 0 || py >= TH) continue;
                if (CO32 && py != PH) continue;
                n_mfma += 18;
#pragma unroll
                for (int kx = 0; kx < 3; ++kx)
#pragma unroll
                    for (int ord = 2; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa)
                            acc[ky * 3 + kx] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(zf[py][qa], xf[kx][ord - qa], acc[ky * 3 + kx], 0, 0, 0);
            }
            // one MFMA, then up to WG_FILL of the staging's vector / LDS-store instructions in the cycles it leaves free
#pragma unroll
            for (int i = 0; i < n_mfma; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x202, CO32 ? WG_FILL + 2 : WG_FILL, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto run = [&](auto cfg_c) {
        f32x4 ra[8], rb[8];
        unsigned short* buf0 = lds16;
        unsigned short* buf1 = lds16 + BUF;
        issue_loads(cfg_c, 0, true, ra);
        issue_loads(cfg_c, 1, true, rb);
        store_all(cfg_c, ra, buf0);
        __syncthreads();
        Frag fr;
        prefetch(buf0, fr);
        for (int j = 0; j < NJ; j += 2) {
            phase(cfg_c, j, rb, ra, buf0, buf1, fr);
            phase(cfg_c, j + 1, ra, rb, buf1, buf0, fr);
        }
    };
    if (NJ > 0) {
        // the wave's code copy.  CO32: output row ph = wave & 1
#define WG_RUN(CFG) run(std::integral_constant<int, (CFG)>{})
        constexpr int P1 = CO32 ? 16 : 0;                           // cfg bit 4 of the odd waves
        if (role == 0) WG_RUN(0);
        else if (role == 1) { if (xs[0].up) WG_RUN(1 | 4 | P1); else WG_RUN(1 | P1); }
        else if (role == 2) { if (xs[1].up) WG_RUN(1 | 4); else WG_RUN(1); }
        else if (xs[1].up) WG_RUN(3 | 4 | 8 | P1);
        else if (xs[0].up) WG_RUN(3 | 4 | P1);
        else WG_RUN(3 | P1);
#undef WG_RUN
    }
    // partial slab [blk][co][tap][ci]; C layout: column (ci) = lane & 31, row (co) = (reg & 3) + 8 * (reg >> 2) + 4 * (lane >> 5)
    float* dst = part + (size_t)(CO32 ? blk * 2 + (wave & 1) : blk) * p.Co * 9 * p.Ct;
    const int ci = c_base + wci * 32 + l32;
    if (ci < p.Ct) {
#pragma unroll
        for (int t = 0; t < 9; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int co = co_base + wco * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
                if (co < p.Co) dst[((size_t)co * 9 + t) * p.Ct + ci] = acc[t][r];
            }
    }
#ifdef CODEPS_WG_STAMP_WAVES
    CODEPS_STAMP_END_WAVES(conv);
#else
    CODEPS_STAMP_END(conv);
#endif
}

// wgrad_halo64d_body on TWO fp16 pieces (round 6, arithmetic 16; split_f16 has the arithmetic): three products per tap instead of six, 86 KB
// of LDS instead of 127.  Both operands are activations, so both carry a running block-local scale: a wave publishes the largest exponent
// of its share of sub-tile t (dZ: wave 0; X: waves 1-3) two phases before the sub-tile's MFMAs, every wave derives the same two scales from
// the four words, and when a scale grows the nine accumulator tiles are multiplied by the exact ratio at the phase boundary.  A sub-tile
// is loaded three phases ahead (three register sets) -- a phase is 54 MFMAs now, shorter than a load's latency under traffic.
template <bool CO32>
__device__ __forceinline__ void wgrad_halo64h_body(const WgradP& p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                   const float* __restrict__ x0, const float* __restrict__ x1,
                                                   const float* __restrict__ dz, float* __restrict__ part, unsigned short* lds16) {
    constexpr int TH = 2, TW = 16, XH = TH + 2, PIX = TH * TW, XROW = 32;
    constexpr int NP = 2, NPROD = 3;
    constexpr int ZP = NP * PIX + 8;                   // halfwords per dZ channel (72: 36 dwords = 9 slots of 16 bytes, odd: conflict-free fragment reads)
    constexpr int XQ = XH * XROW, XP = NP * XQ + 8;    // halfwords per X piece / per X channel (264: 132 dwords = 33 slots)
    constexpr int XS0 = 64 * ZP;                       // X rows start behind the dZ rows
    constexpr int BUF = 64 * (ZP + XP);               // halfwords per buffer: [64][ZP] dZ, [64][XP] X
    int* slots = reinterpret_cast<int*>(lds16 + 2 * BUF);               // [sub-tile parity][wave]: the largest exponent a wave found in its share
    CODEPS_STAMP_BEGIN();
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l32 = lane & 31, h = lane >> 5;
    const int wco = CO32 ? 0 : (wave & 1), wci = wave >> 1;
    const int role = __builtin_amdgcn_readfirstlane(wave);            // 0: dZ, 1 / 2: X interior, 3: halo pixels
    const int co_base = blockIdx.y * 64;
    const int chunk = blockIdx.x % ci_chunks, blk = blockIdx.x / ci_chunks;
    const int c_base = chunk * 64;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    const int NJ = 2 * (t_end - t_beg);                               // sub-tiles of this block (even)
    // X source of a half of the chunk (block-uniform)
    struct XSrc { const float* ptr; int cs, c0; bool up; size_t img; };
    auto xsrc_of = [&](int half) {
        const int ch = c_base + 32 * half;
        const bool s1 = ch >= p.C0;
        XSrc o;
        o.ptr = s1 ? x1 : x0; o.cs = s1 ? p.C1 : p.C0; o.c0 = s1 ? ch - p.C0 : ch; o.up = p.up0 && !s1;
        o.img = o.up ? (size_t)(p.H / 2) * (p.W / 2) * o.cs : (size_t)p.H * p.W * o.cs;
        return o;
    };
    const XSrc xs[2] = {xsrc_of(0), xsrc_of(1)};

    f32x16 acc[9];
#pragma unroll
    for (int t = 0; t < 9; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

    // per-thread constants.  Big task (quad's low two bits over four consecutive lanes, then the pixel group, then the quad's high
    // bits: see wgrad_halo64s_body): global byte offset from the sub-tile origin, the X row it reads, LDS halfword of its first store
    int b_off = 0, b_row = 0, b_dst = 0;
    bool b_ok = false;
    if (role == 0) {
        const int c4 = (lane & 3) | ((lane >> 4) << 2), grp = (lane >> 2) & 3;
        b_off = (((grp >> 1) * p.Wo + (grp & 1) * 8) * p.Co + co_base + c4 * 4) * 4;
        b_ok = co_base + c4 * 4 < p.Co;
        b_dst = (c4 * 4) * ZP + grp * 8;
    } else if (role < 3) {
        const XSrc& sx = xs[role - 1];
        const int t = tid - 64, c4 = (t & 3) | ((t >> 5) << 2), c4l = c4 & 7, grp = (t >> 2) & 7;      // wave 1: quads 0-7, wave 2: 8-15
        b_row = (grp >> 1) - 1;
        b_off = sx.up ? (((b_row >> 1) * (p.W / 2) + (grp & 1) * 4) * sx.cs + sx.c0 + c4l * 4) * 4
                      : ((b_row * p.W + (grp & 1) * 8) * sx.cs + sx.c0 + c4l * 4) * 4;
        b_ok = sx.c0 + c4l * 4 < sx.cs;
        b_dst = XS0 + (c4 * 4) * XP + (grp >> 1) * XROW + 8 + (grp & 1) * 8;
    }
    int s_off[2] = {0, 0}, s_row = 0, s_dstk[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    unsigned s_selk[4] = {0, 0, 0, 0};
    bool s_ok[2] = {false, false}, s_side = false;
    if (role == 3) {
        const int c4l = lane & 7, rs = lane >> 3;                    // task u: quad c4l + 8 u, (row, side) rs
        s_side = rs & 1;
        s_row = (rs >> 1) - 1;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const XSrc& sx = xs[u];
            s_off[u] = sx.up ? (((s_row >> 1) * (p.W / 2) + (s_side ? TW / 2 : -1)) * sx.cs + sx.c0 + c4l * 4) * 4
                             : ((s_row * p.W + (s_side ? TW : -1)) * sx.cs + sx.c0 + c4l * 4) * 4;
            s_ok[u] = sx.c0 + c4l * 4 < sx.cs;
            const int dst = XS0 + ((c4l + 8 * u) * 4) * XP + (rs >> 1) * XROW + (s_side ? 24 : 7);
#pragma unroll
            for (int k = 0; k < 4; ++k) s_dstk[u][k] = dst + ((k + (c4l >> 1)) & 3) * XP;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = (k + (c4l >> 1)) & 3;
            s_selk[k] = 0x0c0c0000u | (e == 0 ? 0x0504u : e == 1 ? 0x0706u : e == 2 ? 0x0100u : 0x0302u);
        }
    }
    const size_t zimg = (size_t)p.Ho * p.Wo * p.Co;
    // cfg of a wave's code copy: bits 0-1 role (0: dZ, 1: X interior, 3: halo pixels), bit 2: the wave's source (role 1) / the source of
    // half 0 (role 3) is up-sampled, bit 3: role 3, the source of half 1 is up-sampled, bit 4: CO32, the wave's output row
    // the loads of sub-tile j (role 0, 1: eight 16-byte loads, four from an up-sampled source; 3: two halo pixels); all lanes read
    // zeros when !valid (the sub-tile behind the last one), so the tile loop has no branch around its loads
    auto issue_loads = [&](auto cfg_c, int j, bool valid, f32x4 (&raw)[8], unsigned tok = 0) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3;
        constexpr bool UPA = (CFG >> 2) & 1, UPB = (CFG >> 3) & 1;
        const int tile = t_beg + (j >> 1);                                                     // (all scalar)
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * 4 + (j & 1) * TH, tx0 = (tr % tiles_x) * TW;
        if (ROLE == 0) {
            const __amdgpu_buffer_rsrc_t rsz = make_rsrc(dz + (size_t)b * zimg, zimg * 4);
            const int zorg = (ty0 * p.Wo + tx0) * p.Co * 4, zpix = p.Co * 4;
            const unsigned vo = (valid && b_ok) ? (unsigned)(zorg + b_off) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsz, vo, i * zpix, 0));
        } else if (ROLE == 1) {
            const XSrc& sx = xs[role - 1];
            const __amdgpu_buffer_rsrc_t rsx = make_rsrc(sx.ptr + (size_t)b * sx.img, sx.img * 4);
            const int xorg = UPA ? ((ty0 / 2) * (p.W / 2) + tx0 / 2) * sx.cs * 4 : (ty0 * p.W + tx0) * sx.cs * 4, xpix = sx.cs * 4;
            const unsigned vo = (valid && b_ok && (unsigned)(ty0 + b_row) < (unsigned)p.H) ? (unsigned)(xorg + b_off) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < (UPA ? 4 : 8); ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsx, vo, i * xpix, 0));
        } else {
            const bool okp = valid && (unsigned)(ty0 + s_row) < (unsigned)p.H && (s_side ? tx0 + TW < p.W : tx0 > 0);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const XSrc& sx = xs[u];
                const bool up = u == 0 ? UPA : UPB;
                const __amdgpu_buffer_rsrc_t rsx = make_rsrc(sx.ptr + (size_t)b * sx.img, sx.img * 4);
                const int xorg = up ? ((ty0 / 2) * (p.W / 2) + tx0 / 2) * sx.cs * 4 : (ty0 * p.W + tx0) * sx.cs * 4;
                raw[u] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsx, ((okp && s_ok[u]) ? (unsigned)(xorg + s_off[u]) : GATHER_OOB) + tok, 0, 0));
            }
        }
    };
    // channel e of the big task: 8 pixels -> three 16-byte rows (one per piece)
    auto store_big = [&](auto cfg_c, const f32x4 (&raw)[8], int e, unsigned short* buf, float sc) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3;
        constexpr bool UPA = (CFG >> 2) & 1;
        constexpr int cs = ROLE == 0 ? ZP : XP, qs = ROLE == 0 ? PIX : XQ;
        if (UPA && ROLE == 1) {                                     // four source pixels, each twice
            const f32x4 v4 = {raw[0][e], raw[1][e], raw[2][e], raw[3][e]};
            u16x4 pc[NP];
            split_f16(v4, sc, pc[0], pc[1]);
#pragma unroll
            for (int q = 0; q < NP; ++q)
                *reinterpret_cast<i32x4*>(buf + b_dst + e * cs + q * qs) =
                    pack8(u16x4{pc[q][0], pc[q][0], pc[q][1], pc[q][1]}, u16x4{pc[q][2], pc[q][2], pc[q][3], pc[q][3]});
            return;
        }
        const f32x4 lo4 = {raw[0][e], raw[1][e], raw[2][e], raw[3][e]};
        const f32x4 hi4 = {raw[4][e], raw[5][e], raw[6][e], raw[7][e]};
        u16x4 lo[NP], hi[NP];
        split_f16(lo4, sc, lo[0], lo[1]);
        split_f16(hi4, sc, hi[0], hi[1]);
#pragma unroll
        for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(buf + b_dst + e * cs + q * qs) = pack8(lo[q], hi[q]);
    };
    // a halo pixel's 2-byte stores: a channel's row starts 196 dwords behind its neighbour's (= 4 mod 32: what the 16-byte fragment reads
    // want), so the halo slots of all rows and channels fall on 16 of the 32 write banks -- 4-way at best.  With all lanes storing the
    // SAME channel of their quad the 64 addresses would fall on four to eight banks; so lane's k-th store takes channel
    // (k + (quad >> 1)) & 3 of its quad: 4 lanes per bank.
    struct SmallPc { unsigned lo[NP], hi[NP]; };                    // a halo pixel's 4 channels x 2 pieces, two halfwords per dword
    auto split_small = [&](const f32x4 v, float sc) {
        u16x4 pc[NP];
        split_f16(v, sc, pc[0], pc[1]);
        SmallPc o;
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            o.lo[q] = (unsigned)pc[q][0] | ((unsigned)pc[q][1] << 16);
            o.hi[q] = (unsigned)pc[q][2] | ((unsigned)pc[q][3] << 16);
        }
        return o;
    };
    auto store_small = [&](const SmallPc& pc, int u, unsigned short* buf) {
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k)                              // v_perm_b32: bytes 0-3 = hi, 4-7 = lo (selector = byte numbers of the wanted halfword)
                buf[s_dstk[u][k] + q * XQ] = (unsigned short)__builtin_amdgcn_perm(pc.lo[q], pc.hi[q], s_selk[k]);
    };
    auto store_all = [&](auto cfg_c, const f32x4 (&raw)[8], unsigned short* buf, float sc) {
        constexpr int ROLE = decltype(cfg_c)::value & 3;
        if (ROLE == 3) { store_small(split_small(raw[0], sc), 0, buf); store_small(split_small(raw[1], sc), 1, buf); }
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) store_big(cfg_c, raw, e, buf, sc);
        }
    };
    // the largest exponent in a wave's share of a sub-tile (the registers of its loads) -> slots[parity][wave]
    auto publish = [&](auto cfg_c, const f32x4 (&raw)[8], int parity) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3;
        constexpr bool UPA = (CFG >> 2) & 1;
        constexpr int NR = ROLE == 3 ? 2 : ((ROLE == 1 && UPA) ? 4 : 8);
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(raw[i][e]));
        const int ex = wave_max_exponent(m);
        if (lane == 0) slots[parity * 4 + wave] = ex;
    };
    // running exponents of the two operands (block-uniform: every wave derives them from the same slots)
    int ez_run = F16_EMIN, ex_run = F16_EMIN;
    auto next_exponents = [&](int parity, int& ez_n, int& ex_n) {
        const i32x4 pe = *reinterpret_cast<const i32x4*>(slots + parity * 4);
        ez_n = __builtin_amdgcn_readfirstlane(max(ez_run, pe[0]));
        ex_n = __builtin_amdgcn_readfirstlane(max(ex_run, max(pe[1], max(pe[2], pe[3]))));
    };

    const int zoff = (wco * 32 + l32) * ZP + h * 8, xoff = XS0 + (wci * 32 + l32) * XP + h * 8;
    // fragments a phase starts with: the dZ rows and X row 0 of its buffer.  They are read by the PREVIOUS phase, right behind the
    // barrier that phase places in front of its last row's MFMAs (row 3: registers only) -- the LDS latency at the start of a sub-tile
    // disappears under those MFMAs
    struct Frag { f16x8 zf[TH][NP]; i32x4 x0[NP][3]; };
    auto prefetch = [&](const unsigned short* buf, Frag& f) {
        const unsigned short* zrow = buf + zoff;
        const unsigned short* xrow = buf + xoff;
#pragma unroll
        for (int py = 0; py < TH; ++py)
#pragma unroll
            for (int q = 0; q < NP; ++q) f.zf[py][q] = *reinterpret_cast<const f16x8*>(zrow + q * PIX + py * TW);
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const unsigned short* g0 = xrow + q * XQ;
            f.x0[q][0] = *reinterpret_cast<const i32x4*>(g0);
            f.x0[q][1] = *reinterpret_cast<const i32x4*>(g0 + 8);
            f.x0[q][2] = *reinterpret_cast<const i32x4*>(g0 + 16);
        }
    };
    // one sub-tile: its MFMAs out of `cur`, the staging of the next one (registers rs, loaded a phase ago) into `nxt`, the loads of the
    // one after that into rl.  One copy of this code per cfg: a wave runs ITS staging instructions between the MFMAs and nothing else,
    // in one basic block
    // rs: sub-tile j + 1 (stored now), rp: sub-tile j + 2 (landed; its maximum is published in front of this phase's barrier, so the next
    // phase knows the scale of its stores), rl: sub-tile j + 3 (loads issued now): three register sets, because a phase is half as long as
    // with three pieces and a load needs more than one of them to land
    auto phase = [&](auto cfg_c, int j, const f32x4 (&rs)[8], const f32x4 (&rp)[8], f32x4 (&rl)[8], Frag& fr) {
        constexpr int CFG = decltype(cfg_c)::value, ROLE = CFG & 3, PH = (CFG >> 4) & 1;
        const unsigned short* cur = lds16 + (j & 1) * BUF;
        unsigned short* nxt = lds16 + ((j + 1) & 1) * BUF;
        int ez_n, ex_n;
        next_exponents((j + 1) & 1, ez_n, ex_n);
        const float sc = f16_scale_of(ROLE == 0 ? ez_n : ex_n);
        // (halo role: split BEFORE the next loads are issued -- with the two old and the two new loads in flight together the compiler's
        //  wait in front of the split, vmcnt(1), also waited for the first NEW load: a memory latency per sub-tile, stamped per wave)
        SmallPc pc0 = {}, pc1 = {};
        unsigned tok = 0;                                           // (zero; makes the loads' offsets depend on the split's results: program order alone did not hold)
        if (ROLE == 3) {
            pc0 = split_small(rs[0], sc);
            pc1 = split_small(rs[1], sc);
            asm volatile("" : "+v"(tok) : "v"(pc0.lo[0]), "v"(pc0.lo[1]), "v"(pc0.hi[0]), "v"(pc0.hi[1]),
                                          "v"(pc1.lo[0]), "v"(pc1.lo[1]), "v"(pc1.hi[0]), "v"(pc1.hi[1]));
        }
        issue_loads(cfg_c, min(j + 3, NJ - 1), j + 3 < NJ, rl, tok);
        const unsigned short* xrow = cur + xoff;
        f16x8 zf[TH][NP];
        i32x4 xraw[2][NP][3];                                       // [row parity][piece][prev | cur | next]
#pragma unroll
        for (int q = 0; q < NP; ++q) {
#pragma unroll
            for (int py = 0; py < TH; ++py) zf[py][q] = fr.zf[py][q];
#pragma unroll
            for (int i = 0; i < 3; ++i) xraw[0][q][i] = fr.x0[q][i];
        }
        auto read_row = [&](int r) {
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const unsigned short* g0 = xrow + q * XQ + r * XROW;
                xraw[r & 1][q][0] = *reinterpret_cast<const i32x4*>(g0);
                xraw[r & 1][q][1] = *reinterpret_cast<const i32x4*>(g0 + 8);
                xraw[r & 1][q][2] = *reinterpret_cast<const i32x4*>(g0 + 16);
            }
        };
#pragma unroll
        for (int r = 0; r < XH; ++r) {
            if (r + 1 < XH) read_row(r + 1);
            else {
                if (j + 2 < NJ) publish(cfg_c, rp, j & 1);          // sub-tile j + 2 (parity j: last read at this phase's start, by every wave before its stores)
                __syncthreads();                                    // every wave has read `cur` (row 3 is in registers) and written its part of `nxt`
                prefetch(nxt, fr);
            }
            __builtin_amdgcn_sched_barrier(0);
            // staging of the next sub-tile under the MFMAs of the two middle rows
            if (ROLE == 3) {
                if (r == 1) store_small(pc0, 0, nxt);
                if (r == 2) store_small(pc1, 1, nxt);
            } else {
                if (r == 1) { store_big(cfg_c, rs, 0, nxt, sc); store_big(cfg_c, rs, 1, nxt, sc); }
                if (r == 2) { store_big(cfg_c, rs, 2, nxt, sc); store_big(cfg_c, rs, 3, nxt, sc); }
            }
            f16x8 xf[3][NP];                                         // [kx][piece]
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const i32x4 prev = xraw[r & 1][q][0], curv = xraw[r & 1][q][1], next = xraw[r & 1][q][2];
                i32x4 left, right;
                left[0] = (int)__builtin_amdgcn_alignbit((unsigned)curv[0], (unsigned)prev[3], 16);
                right[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)curv[3], 16);
#pragma unroll
                for (int i = 1; i < 4; ++i) left[i] = (int)__builtin_amdgcn_alignbit((unsigned)curv[i], (unsigned)curv[i - 1], 16);
#pragma unroll
                for (int i = 0; i < 3; ++i) right[i] = (int)__builtin_amdgcn_alignbit((unsigned)curv[i + 1], (unsigned)curv[i], 16);
                xf[0][q] = __builtin_bit_cast(f16x8, left);
                xf[1][q] = __builtin_bit_cast(f16x8, curv);
                xf[2][q] = __builtin_bit_cast(f16x8, right);
            }
            int n_mfma = 0;
#pragma unroll
            for (int ky = 0; ky < 3; ++ky) {
                const int py = r - ky;
                if (py < 0 || py >= TH) continue;
                if (CO32 && py != PH) continue;
                n_mfma += 3 * NPROD;
#pragma unroll
                for (int kx = 0; kx < 3; ++kx)
#pragma unroll
                    for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa)
                            acc[ky * 3 + kx] = __builtin_amdgcn_mfma_f32_32x32x16_f16(zf[py][qa], xf[kx][ord - qa], acc[ky * 3 + kx], 0, 0, 0);
            }
            // one MFMA, then up to WG_FILL of the staging's vector / LDS-store instructions in the cycles it leaves free
#pragma unroll
            for (int i = 0; i < n_mfma; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x202, CO32 ? 2 * WG_FILL + 2 : 2 * WG_FILL, 0);      // (half the MFMAs for the same staging)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        // the next sub-tile was staged at (ez_n, ex_n): when that differs from this one's scale, re-base the sums (exact)
        if (ez_n + ex_n != ez_run + ex_run) {
            const float rb = f16_rebase(ez_run + ex_run, ez_n + ex_n);
#pragma unroll
            for (int t = 0; t < 9; ++t) acc[t] *= rb;
        }
        ez_run = ez_n; ex_run = ex_n;
    };
    auto run = [&](auto cfg_c) {
        constexpr int ROLE = decltype(cfg_c)::value & 3;
        f32x4 r0[8], r1[8], r2[8];                                  // sub-tile t lives in set t % 3
        issue_loads(cfg_c, 0, true, r0);
        issue_loads(cfg_c, 1, true, r1);                            // (NJ >= 2)
        issue_loads(cfg_c, min(2, NJ - 1), 2 < NJ, r2);
        publish(cfg_c, r0, 0);
        publish(cfg_c, r1, 1);
        __syncthreads();
        {
            int ez_n, ex_n;
            next_exponents(0, ez_n, ex_n);
            ez_run = ez_n; ex_run = ex_n;
            store_all(cfg_c, r0, lds16, f16_scale_of(ROLE == 0 ? ez_n : ex_n));
        }
        __syncthreads();
        Frag fr;
        prefetch(lds16, fr);
        for (int j = 0; j < NJ; j += 3) {
            phase(cfg_c, j, r1, r2, r0, fr);
            if (j + 1 < NJ) phase(cfg_c, j + 1, r2, r0, r1, fr);
            if (j + 2 < NJ) phase(cfg_c, j + 2, r0, r1, r2, fr);
        }
    };
    if (NJ > 0) {
        // the wave's code copy.  CO32: output row ph = wave & 1
#define WG_RUN(CFG) run(std::integral_constant<int, (CFG)>{})
        constexpr int P1 = CO32 ? 16 : 0;                           // cfg bit 4 of the odd waves
        if (role == 0) WG_RUN(0);
        else if (role == 1) { if (xs[0].up) WG_RUN(1 | 4 | P1); else WG_RUN(1 | P1); }
        else if (role == 2) { if (xs[1].up) WG_RUN(1 | 4); else WG_RUN(1); }
        else if (xs[1].up) WG_RUN(3 | 4 | 8 | P1);
        else if (xs[0].up) WG_RUN(3 | 4 | P1);
        else WG_RUN(3 | P1);
#undef WG_RUN
    }
    {                                                               // sums of (dZ 2^kz)(X 2^kx): back to the operands' units (exact)
        const float inv = f16_inv_scale_of(ez_run) * f16_inv_scale_of(ex_run);
#pragma unroll
        for (int t = 0; t < 9; ++t) acc[t] *= inv;
    }
    // partial slab [blk][co][tap][ci]; C layout: column (ci) = lane & 31, row (co) = (reg & 3) + 8 * (reg >> 2) + 4 * (lane >> 5)
    float* dst = part + (size_t)(CO32 ? blk * 2 + (wave & 1) : blk) * p.Co * 9 * p.Ct;
    const int ci = c_base + wci * 32 + l32;
    if (ci < p.Ct) {
#pragma unroll
        for (int t = 0; t < 9; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int co = co_base + wco * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
                if (co < p.Co) dst[((size_t)co * 9 + t) * p.Ct + ci] = acc[t][r];
            }
    }
#ifdef CODEPS_WG_STAMP_WAVES
    CODEPS_STAMP_END_WAVES(conv);
#else
    CODEPS_STAMP_END(conv);
#endif
}

template <bool CO32, int ARITH = 3>
__global__ __launch_bounds__(256) void wgrad_halo64s_kernel(WgradP p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                            const float* __restrict__ x0, const float* __restrict__ x1,
                                                            const float* __restrict__ dz, float* __restrict__ part) {
    extern __shared__ __attribute__((aligned(16))) unsigned short lds16[];
    const int c_base = (blockIdx.x % ci_chunks) * 64;
    const bool one_src = c_base >= p.C0 || p.C1 == 0 || c_base + 64 <= p.C0;
    // p.fast: the layer-wide conditions (host); per block: each 32-channel half of the chunk in one source -> the double-buffered body
    // (ARITH 16: on two fp16 pieces; the generic body keeps the three bf16 pieces under either arithmetic)
    if (p.fast && (one_src || c_base + 32 == p.C0)) {
        if constexpr (ARITH == 16) wgrad_halo64h_body<CO32>(p, ci_chunks, tiles_x, tiles_y, tiles_per_block, x0, x1, dz, part, lds16);
        else wgrad_halo64d_body<CO32>(p, ci_chunks, tiles_x, tiles_y, tiles_per_block, x0, x1, dz, part, lds16);
    } else wgrad_halo64s_body<CO32>(p, ci_chunks, tiles_x, tiles_y, tiles_per_block, x0, x1, dz, part, lds16);
}

// Weight gradient of the double-pixel stem (7 x 4 taps of 16 channels, stride (2, 1), 64 output channels) on the bf16 matrix
// cores, built like wgrad_halo64s_kernel: 4 x 16 output tiles, operands transposed to [channel][piece][pixel] while staged,
// x-shifted tap fragments made in registers from two aligned 8-pixel groups (kx = 2 is a pure register rotation).  N is only
// 16 channels, so the MFMA is v_mfma_f32_16x16x32_bf16 (16 co x 16 ci x 32 pixels); the four waves split the seven tap rows
// and each keeps all four 16-channel co tiles: 12 dZ + 24 X fragment reads for up to 384 MFMAs per wave and tile.
__global__ __launch_bounds__(256) void wgrad_stem74s_kernel(WgradP p, int tiles_x, int tiles_y, int tiles_per_block,
                                                            const float* __restrict__ x0, const float* __restrict__ dz, float* __restrict__ part) {
    constexpr int TH = 4, TW = 16, KH = 7, KW = 4, XH = (TH - 1) * 2 + KH, PIX = TH * TW, XROW = 24;
    constexpr int ZP = 3 * PIX + 8;                    // halfwords per dZ channel
    constexpr int XQ = XH * XROW, XP = 3 * XQ;         // halfwords per X piece / channel (468 dwords: odd multiple of 4 -> conflict-free)
    __shared__ __attribute__((aligned(16))) unsigned short dZs[64 * ZP];
    __shared__ __attribute__((aligned(16))) unsigned short Xs[16 * XP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, kg = lane >> 4;
    const int blk = blockIdx.x;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);

    f32x4 acc[4][2][KW];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int t = 0; t < KW; ++t) acc[a][b][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    // staging tasks of 8 pixels x 4 channels: 128 for dZ (16 channel quads x 8 groups), 156 for X (4 quads x 13 rows x 3 groups);
    // thread tid owns tasks tid and tid + 256 (< 284); quad index fastest over four lanes (64 contiguous bytes per pixel)
    f32x4 bigr[2][8];
    auto load_tile = [&](int tile) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int bt = tid + 256 * u;
            if (bt >= 284) break;
            if (bt < 128) {
                const int c4 = (bt & 3) | ((bt >> 5) << 2), grp = (bt >> 2) & 7;
                const int gy = ty0 + (grp >> 1), gx0 = tx0 + (grp & 1) * 8;
                const bool rowok = gy < p.Ho;
                const float* rowp = dz + (((size_t)b * p.Ho + gy) * p.Wo + gx0) * p.Co + c4 * 4;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    bigr[u][i] = (rowok && gx0 + i < p.Wo) ? *reinterpret_cast<const f32x4*>(rowp + (size_t)i * p.Co) : f32x4{0.f, 0.f, 0.f, 0.f};
            } else {
                const int t = bt - 128, c4 = t & 3, grp = t >> 2, row = grp / 3, g = grp % 3;
                const int iy = ty0 * 2 + row - p.pad, ix0 = tx0 + g * 8 - p.pad_w;
                const bool rowok = iy >= 0 && iy < p.H;
                const float* rowp = x0 + ((size_t)b * p.H + iy) * p.W * 16 + c4 * 4;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int ix = ix0 + i;
                    bigr[u][i] = (rowok && ix >= 0 && ix < p.W) ? *reinterpret_cast<const f32x4*>(rowp + (size_t)ix * 16) : f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
        }
    };
    auto store_tile = [&]() {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int bt = tid + 256 * u;
            if (bt >= 284) break;
            unsigned short* dst;
            int cstride, qstride;
            if (bt < 128) {
                const int c4 = (bt & 3) | ((bt >> 5) << 2), grp = (bt >> 2) & 7;
                dst = dZs + (c4 * 4) * ZP + grp * 8; cstride = ZP; qstride = PIX;
            } else {
                const int t = bt - 128, c4 = t & 3, grp = t >> 2, row = grp / 3, g = grp % 3;
                dst = Xs + (c4 * 4) * XP + row * XROW + g * 8; cstride = XP; qstride = XQ;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f32x4 lo4 = {bigr[u][0][e], bigr[u][1][e], bigr[u][2][e], bigr[u][3][e]};
                const f32x4 hi4 = {bigr[u][4][e], bigr[u][5][e], bigr[u][6][e], bigr[u][7][e]};
                u16x4 lo[3], hi[3];
                split_bf16<3>(lo4, lo);
                split_bf16<3>(hi4, hi);
#pragma unroll
                for (int q = 0; q < 3; ++q) *reinterpret_cast<i32x4*>(dst + e * cstride + q * qstride) = pack8(lo[q], hi[q]);
            }
        }
    };

    if (t_beg < t_end) load_tile(t_beg);
    for (int tile = t_beg; tile < t_end; ++tile) {
        __syncthreads();
        store_tile();
        __syncthreads();
        if (tile + 1 < t_end) load_tile(tile + 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {                           // K-step = 32 output pixels = tile rows 2 ks, 2 ks + 1
            bf16x8 zf[4][3];
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int q = 0; q < 3; ++q)
                    zf[a][q] = *reinterpret_cast<const bf16x8*>(dZs + (a * 16 + l16) * ZP + q * PIX + ks * 32 + kg * 8);
#pragma unroll
            for (int kyl = 0; kyl < 2; ++kyl) {
                const int ky = wave * 2 + kyl;
                if (ky >= KH) continue;
                const int r = 2 * (2 * ks + (kg >> 1)) + ky;       // input row of this lane's 8 pixels through tap row ky
                bf16x8 xf[KW][3];
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    const unsigned short* g0 = Xs + l16 * XP + q * XQ + r * XROW + (kg & 1) * 8;
                    const i32x4 cur = *reinterpret_cast<const i32x4*>(g0), next = *reinterpret_cast<const i32x4*>(g0 + 8);
                    i32x4 s1, s2, s3;
                    s2[0] = cur[1]; s2[1] = cur[2]; s2[2] = cur[3]; s2[3] = next[0];
#pragma unroll
                    for (int i = 0; i < 3; ++i) s1[i] = (int)__builtin_amdgcn_alignbit((unsigned)cur[i + 1], (unsigned)cur[i], 16);
                    s1[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)cur[3], 16);
                    s3[0] = (int)__builtin_amdgcn_alignbit((unsigned)cur[2], (unsigned)cur[1], 16);
                    s3[1] = (int)__builtin_amdgcn_alignbit((unsigned)cur[3], (unsigned)cur[2], 16);
                    s3[2] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)cur[3], 16);
                    s3[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[1], (unsigned)next[0], 16);
                    xf[0][q] = __builtin_bit_cast(bf16x8, cur);
                    xf[1][q] = __builtin_bit_cast(bf16x8, s1);
                    xf[2][q] = __builtin_bit_cast(bf16x8, s2);
                    xf[3][q] = __builtin_bit_cast(bf16x8, s3);
                }
#pragma unroll
                for (int kx = 0; kx < KW; ++kx)
#pragma unroll
                    for (int ord = 2; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                            for (int a = 0; a < 4; ++a)
                                acc[a][kyl][kx] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(zf[a][qa], xf[kx][ord - qa], acc[a][kyl][kx], 0, 0, 0);
            }
        }
    }
    // partial slab [blk][co][tap][ci]; C layout: column (ci) = lane & 15, row (co) = (lane >> 4) * 4 + reg
    float* dst = part + (size_t)blk * p.Co * (KH * KW) * p.Ct;
#pragma unroll
    for (int kyl = 0; kyl < 2; ++kyl) {
        const int ky = wave * 2 + kyl;
        if (ky >= KH) continue;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int kx = 0; kx < KW; ++kx)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int co = a * 16 + kg * 4 + r;
                    dst[((size_t)co * (KH * KW) + ky * KW + kx) * p.Ct + l16] = acc[a][kyl][kx][r];
                }
    }
}

// wgrad_stem74s_kernel, double-buffered like wgrad_halo64d_body (maps of whole 4 x 16 tiles, no x padding -- the double-pixel stem
// layout carries its zero columns): LDS holds two tiles (2 x 55 KB); while a wave runs the MFMAs of tile t it splits and stores tile
// t + 1 between them and then issues the loads of tile t + 2; addresses are (scalar tile origin) + (per-thread constant), row padding
// is the range check of the buffer resource.  Roles: waves 0, 1 stage dZ (128 tasks of 8 pixels x 4 channels), wave 2 the first 64 of
// the 156 X tasks; wave 3 -- tap row 6 only, half the MFMAs -- the other 92 (two per lane).  One code copy per role.
// ARITH 16 (round 6): two fp16 pieces, running block-local scales for dZ (waves 0, 1) and X (waves 2, 3), three register sets per task: a tile is
// loaded three phases ahead, its exponent published two ahead, stored one ahead -- as in wgrad_halo64h_body.
template <int ARITH = 3>
__global__ __launch_bounds__(256) void wgrad_stem74d_kernel(WgradP p, int tiles_x, int tiles_y, int tiles_per_block,
                                                            const float* __restrict__ x0, const float* __restrict__ dz, float* __restrict__ part) {
    constexpr int TH = 4, TW = 16, KH = 7, KW = 4, XH = (TH - 1) * 2 + KH, PIX = TH * TW, XROW = 24;
    constexpr int NP = ARITH == 16 ? 2 : 3;
    constexpr bool H16 = ARITH == 16;
    typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
    constexpr int ZP = NP * PIX + 8;                   // halfwords per dZ channel
    constexpr int XQ = XH * XROW, XP = NP * XQ + (H16 ? 8 : 0);      // halfwords per X piece / channel (468 / 316 dwords: odd multiples of 4 -> conflict-free)
    constexpr int XS0 = 64 * ZP, BUF = XS0 + 16 * XP;  // halfwords per buffer
    extern __shared__ __attribute__((aligned(16))) unsigned short lds16[];
    int* slots = reinterpret_cast<int*>(lds16 + 2 * BUF);           // ARITH 16: [tile parity][wave] largest exponents
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int blk = blockIdx.x;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    const int NT = t_end - t_beg;

    f32x4 acc[4][2][KW];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int t = 0; t < KW; ++t) acc[a][b][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    // per-thread constants of the (up to two) tasks: byte offset from the tile origin, the X row (relative to 2 ty0 - pad), LDS halfword
    int k_off[2] = {0, 0}, k_row[2] = {0, 0}, k_dst[2] = {0, 0};
    bool k_ok[2] = {false, false};
    if (wave < 2) {
        const int bt = tid, c4 = (bt & 3) | ((bt >> 5) << 2), grp = (bt >> 2) & 7;
        k_off[0] = (((grp >> 1) * p.Wo + (grp & 1) * 8) * p.Co + c4 * 4) * 4;
        k_ok[0] = true;
        k_dst[0] = (c4 * 4) * ZP + grp * 8;
    } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = (wave == 2 ? 0 : 64) + lane + 64 * u;
            if ((wave == 2 && u == 1) || t >= 156) continue;
            const int c4 = t & 3, grp = t >> 2, row = grp / 3, g = grp % 3;
            k_row[u] = row;
            k_off[u] = ((row * p.W + g * 8) * 16 + c4 * 4) * 4;
            k_ok[u] = true;
            k_dst[u] = XS0 + (c4 * 4) * XP + row * XROW + g * 8;
        }
        if (!k_ok[1]) k_dst[1] = k_dst[0];                          // (no second task: its zeros go where the first task's data follows)
    }
    const size_t zimg = (size_t)p.Ho * p.Wo * p.Co, ximg = (size_t)p.H * p.W * 16;
    // ROLE 0: dZ task, 1: one X task, 2: two X tasks (wave 3)
    auto issue_loads = [&](auto role_c, int u, int t, bool valid, f32x4 (&raw)[8]) {
        constexpr int ROLE = decltype(role_c)::value;
        const int tile = t_beg + t;                                                            // (all scalar)
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
        if (ROLE == 0) {
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(dz + (size_t)b * zimg, zimg * 4);
            const unsigned vo = valid ? (unsigned)((ty0 * p.Wo + tx0) * p.Co * 4 + k_off[0]) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, i * p.Co * 4, 0));
        } else {
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(x0 + (size_t)b * ximg, ximg * 4);
            const int iy0 = ty0 * 2 - p.pad;                        // rows above / below the image: zeros (the columns carry their own padding)
            const unsigned vo = (valid && k_ok[u] && (unsigned)(iy0 + k_row[u]) < (unsigned)p.H) ? (unsigned)((iy0 * p.W + tx0) * 64 + k_off[u]) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, i * 64, 0));
        }
    };
    auto store_big = [&](auto role_c, int u, const f32x4 (&raw)[8], int e, unsigned short* buf, float sc = 1.f) {
        constexpr int ROLE = decltype(role_c)::value;
        constexpr int cs = ROLE == 0 ? ZP : XP, qs = ROLE == 0 ? PIX : XQ;
        const f32x4 lo4 = {raw[0][e], raw[1][e], raw[2][e], raw[3][e]};
        const f32x4 hi4 = {raw[4][e], raw[5][e], raw[6][e], raw[7][e]};
        u16x4 lo[NP], hi[NP];
        if constexpr (H16) { split_f16(lo4, sc, lo[0], lo[1]); split_f16(hi4, sc, hi[0], hi[1]); }
        else { split_bf16<NP>(lo4, lo); split_bf16<NP>(hi4, hi); }
        // (lanes 28-63 of wave 3's second task have no task: they hold zeros and store them where the first task of the same lane
        //  stores -- before it, in program order -- so the slot ends with the real data)
#pragma unroll
        for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(buf + k_dst[u] + e * cs + q * qs) = pack8(lo[q], hi[q]);
    };
    const int ky0 = wave * 2;
    // one tile: its MFMAs out of `cur`; between them the staging of the next tile (registers r0 / r1, loaded a phase ago) into `nxt`,
    // then the loads of the tile after that
    // ARITH 16: exponents of the two operands (block-uniform: every wave derives them from the same slots)
    int ez_run = F16_EMIN, ex_run = F16_EMIN;
    auto publish = [&](auto role_c, const f32x4 (&a0)[8], const f32x4 (&a1)[8], int parity) {
        constexpr int ROLE = decltype(role_c)::value;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) { m = fmaxf(m, fabsf(a0[i][e])); if (ROLE == 2) m = fmaxf(m, fabsf(a1[i][e])); }
        const int ex = wave_max_exponent(m);
        if (lane == 0) slots[parity * 4 + wave] = ex;
    };
    auto next_exponents = [&](int parity, int& ez_n, int& ex_n) {
        const i32x4 pe = *reinterpret_cast<const i32x4*>(slots + parity * 4);
        ez_n = __builtin_amdgcn_readfirstlane(max(ez_run, max(pe[0], pe[1])));
        ex_n = __builtin_amdgcn_readfirstlane(max(ex_run, max(pe[2], pe[3])));
    };
    // ARITH 3: r0 / r1 hold tile t + 1 (stored in regions 0 / 1) and are re-loaded with tile t + 2 behind their stores (rp*, rl* unused).
    // ARITH 16: r0 / r1 = tile t + 1 (stored), rp0 / rp1 = tile t + 2 (published in front of the barrier), rl0 / rl1 = tile t + 3 (loads issued first).
    auto phase = [&](auto role_c, int t, f32x4 (&r0)[8], f32x4 (&r1)[8], const f32x4 (&rp0)[8], const f32x4 (&rp1)[8], f32x4 (&rl0)[8], f32x4 (&rl1)[8],
                     const unsigned short* cur, unsigned short* nxt) {
        constexpr int ROLE = decltype(role_c)::value, NKYL = ROLE == 2 ? 1 : 2;
        int ez_n = ez_run, ex_n = ex_run;
        float sc = 1.f;
        if constexpr (H16) {
            next_exponents((t + 1) & 1, ez_n, ex_n);
            sc = f16_scale_of(ROLE == 0 ? ez_n : ex_n);
            issue_loads(role_c, 0, min(t + 3, NT - 1), t + 3 < NT, rl0);
            if (ROLE == 2) issue_loads(role_c, 1, min(t + 3, NT - 1), t + 3 < NT, rl1);
        }
        const unsigned short* dZs = cur;
        const unsigned short* Xs = cur + XS0;
        i32x4 xraw[2][NP][2];                                       // [region parity][piece][cur | next]
        auto read_x = [&](int ks, int kyl, int par) {
            const int r = 2 * (2 * ks + (kg >> 1)) + ky0 + kyl;     // input row of this lane's 8 pixels through tap row ky
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const unsigned short* g0 = Xs + l16 * XP + q * XQ + r * XROW + (kg & 1) * 8;
                xraw[par][q][0] = *reinterpret_cast<const i32x4*>(g0);
                xraw[par][q][1] = *reinterpret_cast<const i32x4*>(g0 + 8);
            }
        };
        read_x(0, 0, 0);
        int region = 0;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {                           // K-step = 32 output pixels = tile rows 2 ks, 2 ks + 1
            frag_t zf[4][NP];
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int q = 0; q < NP; ++q)
                    zf[a][q] = *reinterpret_cast<const frag_t*>(dZs + (a * 16 + l16) * ZP + q * PIX + ks * 32 + kg * 8);
#pragma unroll
            for (int kyl = 0; kyl < NKYL; ++kyl, ++region) {
                const int par = region & 1;
                // the next region's X fragments, one region ahead
                if (kyl + 1 < NKYL) read_x(ks, kyl + 1, par ^ 1);
                else if (ks == 0) read_x(1, 0, par ^ 1);
                __builtin_amdgcn_sched_barrier(0);
                // staging: regions 0, 1 (wave 3: its two regions) split and store; the loads of the tile after the next follow the last split
                if (ROLE == 2) {
                    if (region == 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) store_big(role_c, 1, r1, e, nxt, sc);      // (second task first: see store_big)
                    } else {
                        if constexpr (!H16) issue_loads(role_c, 1, min(t + 2, NT - 1), t + 2 < NT, r1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) store_big(role_c, 0, r0, e, nxt, sc);
                    }
                } else {
                    if (region == 0) { store_big(role_c, 0, r0, 0, nxt, sc); store_big(role_c, 0, r0, 1, nxt, sc); }
                    if (region == 1) { store_big(role_c, 0, r0, 2, nxt, sc); store_big(role_c, 0, r0, 3, nxt, sc); }
                    if constexpr (!H16) { if (region == 2) issue_loads(role_c, 0, min(t + 2, NT - 1), t + 2 < NT, r0); }
                }
                frag_t xf[KW][NP];
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    const i32x4 cur4 = xraw[par][q][0], next = xraw[par][q][1];
                    i32x4 s1, s2, s3;
                    s2[0] = cur4[1]; s2[1] = cur4[2]; s2[2] = cur4[3]; s2[3] = next[0];
#pragma unroll
                    for (int i = 0; i < 3; ++i) s1[i] = (int)__builtin_amdgcn_alignbit((unsigned)cur4[i + 1], (unsigned)cur4[i], 16);
                    s1[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)cur4[3], 16);
                    s3[0] = (int)__builtin_amdgcn_alignbit((unsigned)cur4[2], (unsigned)cur4[1], 16);
                    s3[1] = (int)__builtin_amdgcn_alignbit((unsigned)cur4[3], (unsigned)cur4[2], 16);
                    s3[2] = (int)__builtin_amdgcn_alignbit((unsigned)next[0], (unsigned)cur4[3], 16);
                    s3[3] = (int)__builtin_amdgcn_alignbit((unsigned)next[1], (unsigned)next[0], 16);
                    xf[0][q] = __builtin_bit_cast(frag_t, cur4);
                    xf[1][q] = __builtin_bit_cast(frag_t, s1);
                    xf[2][q] = __builtin_bit_cast(frag_t, s2);
                    xf[3][q] = __builtin_bit_cast(frag_t, s3);
                }
#pragma unroll
                for (int kx = 0; kx < KW; ++kx)
#pragma unroll
                    for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                        for (int qa = 0; qa <= ord; ++qa)
#pragma unroll
                            for (int a = 0; a < 4; ++a) {
                                if constexpr (H16) acc[a][kyl][kx] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zf[a][qa], xf[kx][ord - qa], acc[a][kyl][kx], 0, 0, 0);
                                else acc[a][kyl][kx] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(zf[a][qa], xf[kx][ord - qa], acc[a][kyl][kx], 0, 0, 0);
                            }
                // 96 (48) MFMAs of 16 cycles: two of them, then up to three (six) of the staging's vector / LDS-store instructions
#pragma unroll
                for (int i = 0; i < (H16 ? 24 : 48); ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x202, (ROLE == 2 ? 5 : 3) * (H16 ? 2 : 1), 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (!H16) { if (ROLE == 2) issue_loads(role_c, 0, min(t + 2, NT - 1), t + 2 < NT, r0); }
        if constexpr (H16) {
            if (t + 2 < NT) publish(role_c, rp0, rp1, t & 1);      // tile t + 2 (parity t: read at this phase's start by every wave)
            if (ez_n + ex_n != ez_run + ex_run) {                   // the next tile was staged at a larger scale: re-base the sums (exact)
                const float rb = f16_rebase(ez_run + ex_run, ez_n + ex_n);
#pragma unroll
                for (int a = 0; a < 4; ++a)
#pragma unroll
                    for (int b2 = 0; b2 < 2; ++b2)
#pragma unroll
                        for (int x = 0; x < KW; ++x) acc[a][b2][x] *= rb;
            }
            ez_run = ez_n; ex_run = ex_n;
        }
        __syncthreads();                                            // `cur` is read, `nxt` is written
    };
    auto run_h = [&](auto role_c) {                                 // ARITH 16: tile t lives in register sets (a[t % 3], b[t % 3])
        constexpr int ROLE = decltype(role_c)::value;
        f32x4 a0[8], a1[8], a2[8], b0[8], b1[8], b2[8];
        auto buf_of = [&](int par) { return lds16 + (par & 1) * BUF; };
        issue_loads(role_c, 0, 0, true, a0);
        if (ROLE == 2) issue_loads(role_c, 1, 0, true, b0);
        issue_loads(role_c, 0, min(1, NT - 1), 1 < NT, a1);
        if (ROLE == 2) issue_loads(role_c, 1, min(1, NT - 1), 1 < NT, b1);
        issue_loads(role_c, 0, min(2, NT - 1), 2 < NT, a2);
        if (ROLE == 2) issue_loads(role_c, 1, min(2, NT - 1), 2 < NT, b2);
        publish(role_c, a0, b0, 0);
        publish(role_c, a1, b1, 1);
        __syncthreads();
        {
            int ez_n, ex_n;
            next_exponents(0, ez_n, ex_n);
            ez_run = ez_n; ex_run = ex_n;
            const float sc = f16_scale_of(ROLE == 0 ? ez_n : ex_n);
            if (ROLE == 2) {
#pragma unroll
                for (int e = 0; e < 4; ++e) store_big(role_c, 1, b0, e, lds16, sc);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) store_big(role_c, 0, a0, e, lds16, sc);
        }
        __syncthreads();
        for (int t = 0; t < NT; t += 3) {
            phase(role_c, t, a1, b1, a2, b2, a0, b0, buf_of(t), buf_of(t + 1));
            if (t + 1 < NT) phase(role_c, t + 1, a2, b2, a0, b0, a1, b1, buf_of(t + 1), buf_of(t));
            if (t + 2 < NT) phase(role_c, t + 2, a0, b0, a1, b1, a2, b2, buf_of(t), buf_of(t + 1));
        }
    };
    auto run = [&](auto role_c) {
        constexpr int ROLE = decltype(role_c)::value;
        f32x4 r0[8], r1[8];
        unsigned short* buf0 = lds16;
        unsigned short* buf1 = lds16 + BUF;
        issue_loads(role_c, 0, 0, true, r0);
        if (ROLE == 2) issue_loads(role_c, 1, 0, true, r1);
        if (ROLE == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) store_big(role_c, 1, r1, e, buf0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) store_big(role_c, 0, r0, e, buf0);
        issue_loads(role_c, 0, min(1, NT - 1), 1 < NT, r0);
        if (ROLE == 2) issue_loads(role_c, 1, min(1, NT - 1), 1 < NT, r1);
        __syncthreads();
        for (int t = 0; t < NT; t += 2) {
            phase(role_c, t, r0, r1, r0, r1, r0, r1, buf0, buf1);
            if (t + 1 < NT) phase(role_c, t + 1, r0, r1, r0, r1, r0, r1, buf1, buf0);
        }
    };
    if (NT > 0) {
        if constexpr (H16) {
            if (wave < 2) run_h(std::integral_constant<int, 0>{});
            else if (wave == 2) run_h(std::integral_constant<int, 1>{});
            else run_h(std::integral_constant<int, 2>{});
        } else {
            if (wave < 2) run(std::integral_constant<int, 0>{});
            else if (wave == 2) run(std::integral_constant<int, 1>{});
            else run(std::integral_constant<int, 2>{});
        }
    }
    if constexpr (H16) {                                            // back to the operands' units (exact)
        const float inv = f16_inv_scale_of(ez_run) * f16_inv_scale_of(ex_run);
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b2 = 0; b2 < 2; ++b2)
#pragma unroll
                for (int x = 0; x < KW; ++x) acc[a][b2][x] *= inv;
    }
    // partial slab [blk][co][tap][ci]; C layout: column (ci) = lane & 15, row (co) = (lane >> 4) * 4 + reg
    float* dst = part + (size_t)blk * p.Co * (KH * KW) * p.Ct;
#pragma unroll
    for (int kyl = 0; kyl < 2; ++kyl) {
        const int ky = wave * 2 + kyl;
        if (ky >= KH) continue;
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int kx = 0; kx < KW; ++kx)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int co = a * 16 + kg * 4 + r;
                    dst[((size_t)co * (KH * KW) + ky * KW + kx) * p.Ct + l16] = acc[a][kyl][kx][r];
                }
    }
}

// 3 x 3 / STRIDE 2 weight gradient (the first convolution of ResNet-18/34 stages 2-4: models/resnet_encoder.py:115-126 ->
// torchvision BasicBlock) on the bf16 matrix cores, double-buffered like wgrad_halo64d_body.  Through tap (ky, kx) output pixel
// (oy, ox) meets input pixel (2 oy + ky - 1, 2 ox + kx - 1): consecutive output pixels read every SECOND input column, so the input
// columns are de-interleaved by parity while they are staged -- an X row in LDS is [E: 16 even columns | O: halo, 16 odd columns] --
// and the 8-pixel fragment of tap kx is a contiguous 16-byte read again: kx = 1 reads E, kx = 2 reads O, kx = 0 reads O one slot to
// the left (v_alignbit with the preceding group, as in the stride-1 kernels).  A 2 x 16 output sub-tile needs 5 input rows of 33
// columns: with 64 input channels that is 79 KB per buffer, so a block takes 32 input channels x 64 output channels (two buffers of
// 52 KB) and its four waves are (co tile) x (output row of the sub-tile): 54 MFMAs per wave and sub-tile.  Staging roles: wave 0 dZ (64
// tasks of 8 pixels x 4 channels), waves 1-3 the 160 X tasks (8 input pixels x 4 channels: four even + four odd, two 8-byte stores per
// channel and piece), wave 3 also the 40 halo pixels (column -1).  Until this kernel these layers ran on the f32 MFMA at 84 TFLOP/s.
// ARITH 16 (round 6): two fp16 pieces, both operands with running block-local scales, three register sets -- as wgrad_halo64h_body.
template <int ARITH = 3>
__global__ __launch_bounds__(256) void wgrad_s2_halo_kernel(WgradP p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                            const float* __restrict__ x0, const float* __restrict__ dz, float* __restrict__ part) {
    constexpr int TH = 2, TW = 16, XR = 5, PIX = TH * TW, XROW = 40;
    constexpr int NP = ARITH == 16 ? 2 : 3, NPROD = NP * (NP + 1) / 2;
    constexpr bool H16 = ARITH == 16;
    typedef typename std::conditional<H16, f16x8, bf16x8>::type frag_t;
    constexpr int ZP = NP * PIX + 8;                   // halfwords per dZ channel (104 / 72)
    constexpr int XQ = XR * XROW, XP = NP * XQ + (H16 ? 24 : 16);    // halfwords per X piece / per X channel (616 / 424: 77 / 53 slots of 16 bytes, odd: conflict-free reads)
    constexpr int XS0 = 64 * ZP, BUF = XS0 + 32 * XP;  // halfwords per buffer: [64][ZP] dZ, [32][XP] X
    constexpr int OOFF = 16;                           // the O plane of a row starts here: slot OOFF + 7 = column -1, OOFF + 8 + i = column 2 i + 1
    extern __shared__ __attribute__((aligned(16))) unsigned short lds16[];
    int* slots = reinterpret_cast<int*>(lds16 + 2 * BUF);         // ARITH 16: [sub-tile parity][wave] largest exponents
    const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wco = wave & 1, ph = wave >> 1;          // this wave's 32-row co tile and output row of a sub-tile
    const int co_base = blockIdx.y * 64;
    const int chunk = blockIdx.x % ci_chunks, blk = blockIdx.x / ci_chunks;
    const int c_base = chunk * 32;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    const int NJ = 2 * (t_end - t_beg);
    const int xcs = p.C0;

    f32x16 acc[9];
#pragma unroll
    for (int t = 0; t < 9; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

    // per-thread constants of the big task (dZ: wave 0; X: waves 1-3, task t = 64 (wave - 1) + lane < 160) and of wave 3's halo task
    int b_off = 0, b_row = 0, b_dst = 0;
    bool b_ok = false;
    if (wave == 0) {
        const int c4 = (lane & 3) | ((lane >> 4) << 2), grp = (lane >> 2) & 3;
        b_off = (((grp >> 1) * p.Wo + (grp & 1) * 8) * p.Co + co_base + c4 * 4) * 4;
        b_ok = co_base + c4 * 4 < p.Co;
        b_dst = (c4 * 4) * ZP + grp * 8;
    } else {
        // (wave 3 holds tasks 128-159 only: its upper 32 lanes repeat the lower ones -- same loads, same stores, same data)
        const int t = wave == 3 ? 128 + (lane & 31) : 64 * (wave - 1) + lane, c4 = t & 7, g = (t >> 3) & 3, r = t >> 5;   // quad fastest: 128 contiguous bytes per pixel
        b_row = r - 1;
        b_off = ((b_row * p.W + g * 8) * xcs + c_base + c4 * 4) * 4;
        b_ok = c_base + c4 * 4 < xcs;
        b_dst = XS0 + (c4 * 4) * XP + r * XROW + g * 4;                                        // E slot of its four even pixels; O: + OOFF + 8
    }
    int s_off = 0, s_row = 0, s_dst = 0;
    bool s_ok = false;
    if (wave == 3) {
        const int sl = lane % 40, c4 = sl & 7, r = sl >> 3;          // 40 halo tasks; lanes 40-63 repeat lanes 0-23
        s_row = r - 1;
        s_off = ((s_row * p.W - 1) * xcs + c_base + c4 * 4) * 4;
        s_ok = c_base + c4 * 4 < xcs;
        s_dst = XS0 + (c4 * 4) * XP + r * XROW + OOFF + 7;
    }
    const size_t zimg = (size_t)p.Ho * p.Wo * p.Co, ximg = (size_t)p.H * p.W * xcs;
    // ROLE 0: dZ task; 1: X task; 3: X task + halo pixel (raw[8])
    auto issue_loads = [&](auto role_c, int j, bool valid, f32x4 (&raw)[9]) {
        constexpr int ROLE = decltype(role_c)::value;
        const int tile = t_beg + (j >> 1);                                                     // (all scalar)
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int oy0 = (tr / tiles_x) * 4 + (j & 1) * TH, ox0 = (tr % tiles_x) * TW;
        if (ROLE == 0) {
            const __amdgpu_buffer_rsrc_t rsz = make_rsrc(dz + (size_t)b * zimg, zimg * 4);
            const unsigned vo = (valid && b_ok) ? (unsigned)((oy0 * p.Wo + ox0) * p.Co * 4 + b_off) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsz, vo, i * p.Co * 4, 0));
        } else {
            const __amdgpu_buffer_rsrc_t rsx = make_rsrc(x0 + (size_t)b * ximg, ximg * 4);
            const int xorg = (2 * oy0 * p.W + 2 * ox0) * xcs * 4;
            const unsigned vo = (valid && b_ok && (unsigned)(2 * oy0 + b_row) < (unsigned)p.H) ? (unsigned)(xorg + b_off) : GATHER_OOB;
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsx, vo, i * xcs * 4, 0));
            if (ROLE == 3) {
                const bool ok = valid && s_ok && (unsigned)(2 * oy0 + s_row) < (unsigned)p.H && ox0 > 0;
                raw[8] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsx, ok ? (unsigned)(xorg + s_off) : GATHER_OOB, 0, 0));
            }
        }
    };
    // channel e of the big task.  dZ: 8 pixels -> one 16-byte row per piece.  X: pixels 0, 2, 4, 6 -> E, 1, 3, 5, 7 -> O, 8 bytes each
    auto split_np = [&](const f32x4 v, float sc, u16x4 (&pc)[NP]) {
        if constexpr (H16) split_f16(v, sc, pc[0], pc[1]);
        else split_bf16<NP>(v, pc);
    };
    auto store_big = [&](auto role_c, const f32x4 (&raw)[9], int e, unsigned short* buf, float sc) {
        constexpr int ROLE = decltype(role_c)::value;
        u16x4 lo[NP], hi[NP];
        if (ROLE == 0) {
            split_np(f32x4{raw[0][e], raw[1][e], raw[2][e], raw[3][e]}, sc, lo);
            split_np(f32x4{raw[4][e], raw[5][e], raw[6][e], raw[7][e]}, sc, hi);
#pragma unroll
            for (int q = 0; q < NP; ++q) *reinterpret_cast<i32x4*>(buf + b_dst + e * ZP + q * PIX) = pack8(lo[q], hi[q]);
        } else {
            split_np(f32x4{raw[0][e], raw[2][e], raw[4][e], raw[6][e]}, sc, lo);      // even columns
            split_np(f32x4{raw[1][e], raw[3][e], raw[5][e], raw[7][e]}, sc, hi);      // odd columns
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                *reinterpret_cast<u16x4*>(buf + b_dst + e * XP + q * XQ) = lo[q];
                *reinterpret_cast<u16x4*>(buf + b_dst + e * XP + q * XQ + OOFF + 8) = hi[q];
            }
        }
    };
    auto store_small = [&](const f32x4 v, unsigned short* buf, float sc) {
        u16x4 pc[NP];
        split_np(v, sc, pc);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int q = 0; q < NP; ++q) buf[s_dst + e * XP + q * XQ] = pc[q][e];
    };
    auto store_all = [&](auto role_c, const f32x4 (&raw)[9], unsigned short* buf, float sc) {
        constexpr int ROLE = decltype(role_c)::value;
#pragma unroll
        for (int e = 0; e < 4; ++e) store_big(role_c, raw, e, buf, sc);
        if (ROLE == 3) store_small(raw[8], buf, sc);
    };
    // ARITH 16: the largest exponent in a wave's share of a sub-tile -> slots[parity][wave]; every wave derives the same running exponents
    auto publish = [&](auto role_c, const f32x4 (&raw)[9], int parity) {
        constexpr int ROLE = decltype(role_c)::value;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < (ROLE == 3 ? 9 : 8); ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(raw[i][e]));
        const int ex = wave_max_exponent(m);
        if (lane == 0) slots[parity * 4 + wave] = ex;
    };
    int ez_run = F16_EMIN, ex_run = F16_EMIN;
    auto next_exponents = [&](int parity, int& ez_n, int& ex_n) {
        const i32x4 pe = *reinterpret_cast<const i32x4*>(slots + parity * 4);
        ez_n = __builtin_amdgcn_readfirstlane(max(ez_run, pe[0]));
        ex_n = __builtin_amdgcn_readfirstlane(max(ex_run, max(pe[1], max(pe[2], pe[3]))));
    };

    const int zoff = (wco * 32 + l32) * ZP + ph * TW + h * 8, xoff = XS0 + l32 * XP + (2 * ph) * XROW + h * 8;
    // fragments a phase starts with (read by the previous phase behind its barrier): this wave's dZ row and its first X row
    struct Frag { frag_t zf[NP]; i32x4 x0[NP][3]; };                // x0[piece][E | O | O's preceding group]
    auto read_row = [&](const unsigned short* xrow, int ky, i32x4 (&dst)[NP][3]) {
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            const unsigned short* g0 = xrow + q * XQ + ky * XROW;
            dst[q][0] = *reinterpret_cast<const i32x4*>(g0);
            dst[q][1] = *reinterpret_cast<const i32x4*>(g0 + OOFF + 8);
            dst[q][2] = *reinterpret_cast<const i32x4*>(g0 + OOFF);
        }
    };
    auto prefetch = [&](const unsigned short* buf, Frag& f) {
#pragma unroll
        for (int q = 0; q < NP; ++q) f.zf[q] = *reinterpret_cast<const frag_t*>(buf + zoff + q * PIX);
        read_row(buf + xoff, 0, f.x0);
    };
    // rs: sub-tile j + 1 (stored now); rp (ARITH 16): sub-tile j + 2, landed, its exponent published in front of this phase's barrier;
    // rl: the sub-tile whose loads are issued now (j + 2, or j + 3 with three register sets)
    auto phase = [&](auto role_c, int j, const f32x4 (&rs)[9], const f32x4 (&rp)[9], f32x4 (&rl)[9], Frag& fr) {
        constexpr int ROLE = decltype(role_c)::value;
        const unsigned short* cur = lds16 + (j & 1) * BUF;
        unsigned short* nxt = lds16 + ((j + 1) & 1) * BUF;
        int ez_n = ez_run, ex_n = ex_run;
        float sc = 1.f;
        if constexpr (H16) {
            next_exponents((j + 1) & 1, ez_n, ex_n);
            sc = f16_scale_of(ROLE == 0 ? ez_n : ex_n);
        }
        constexpr int AHEAD = H16 ? 3 : 2;
        issue_loads(role_c, min(j + AHEAD, NJ - 1), j + AHEAD < NJ, rl);
        const unsigned short* xrow = cur + xoff;
        frag_t zf[NP];
        i32x4 xraw[2][NP][3];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
            zf[q] = fr.zf[q];
#pragma unroll
            for (int i = 0; i < 3; ++i) xraw[0][q][i] = fr.x0[q][i];
        }
#pragma unroll
        for (int ky = 0; ky < 3; ++ky) {
            if (ky + 1 < 3) read_row(xrow, ky + 1, xraw[(ky + 1) & 1]);
            else {
                if constexpr (H16) { if (j + 2 < NJ) publish(role_c, rp, j & 1); }
                __syncthreads();                                    // every wave has read `cur` (its last row is in registers) and written its part of `nxt`
                prefetch(nxt, fr);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (ky == 0) { store_big(role_c, rs, 0, nxt, sc); store_big(role_c, rs, 1, nxt, sc); }
            if (ky == 1) { store_big(role_c, rs, 2, nxt, sc); store_big(role_c, rs, 3, nxt, sc); if (ROLE == 3) store_small(rs[8], nxt, sc); }
            frag_t xf[3][NP];                                        // [kx][piece]
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                const i32x4 ev = xraw[ky & 1][q][0], od = xraw[ky & 1][q][1], pv = xraw[ky & 1][q][2];
                i32x4 left;
                left[0] = (int)__builtin_amdgcn_alignbit((unsigned)od[0], (unsigned)pv[3], 16);
#pragma unroll
                for (int i = 1; i < 4; ++i) left[i] = (int)__builtin_amdgcn_alignbit((unsigned)od[i], (unsigned)od[i - 1], 16);
                xf[0][q] = __builtin_bit_cast(frag_t, left);
                xf[1][q] = __builtin_bit_cast(frag_t, ev);
                xf[2][q] = __builtin_bit_cast(frag_t, od);
            }
#pragma unroll
            for (int kx = 0; kx < 3; ++kx)
#pragma unroll
                for (int ord = NP - 1; ord >= 0; --ord)
#pragma unroll
                    for (int qa = 0; qa <= ord; ++qa) {
                        if constexpr (H16) acc[ky * 3 + kx] = __builtin_amdgcn_mfma_f32_32x32x16_f16(zf[qa], xf[kx][ord - qa], acc[ky * 3 + kx], 0, 0, 0);
                        else acc[ky * 3 + kx] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(zf[qa], xf[kx][ord - qa], acc[ky * 3 + kx], 0, 0, 0);
                    }
#pragma unroll
            for (int i = 0; i < 3 * NPROD; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x202, H16 ? 12 : 6, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (H16) {                                        // the next sub-tile was staged at (ez_n, ex_n): re-base the sums when that grew (exact)
            if (ez_n + ex_n != ez_run + ex_run) {
                const float rb = f16_rebase(ez_run + ex_run, ez_n + ex_n);
#pragma unroll
                for (int t = 0; t < 9; ++t) acc[t] *= rb;
            }
            ez_run = ez_n; ex_run = ex_n;
        }
    };
    auto run = [&](auto role_c) {
        constexpr int ROLE = decltype(role_c)::value;
        Frag fr;
        if constexpr (H16) {
            f32x4 r0[9], r1[9], r2[9];                              // sub-tile t lives in set t % 3
            issue_loads(role_c, 0, true, r0);
            issue_loads(role_c, 1, true, r1);                       // (NJ >= 2)
            issue_loads(role_c, min(2, NJ - 1), 2 < NJ, r2);
            publish(role_c, r0, 0);
            publish(role_c, r1, 1);
            __syncthreads();
            {
                int ez_n, ex_n;
                next_exponents(0, ez_n, ex_n);
                ez_run = ez_n; ex_run = ex_n;
                store_all(role_c, r0, lds16, f16_scale_of(ROLE == 0 ? ez_n : ex_n));
            }
            __syncthreads();
            prefetch(lds16, fr);
            for (int j = 0; j < NJ; j += 3) {
                phase(role_c, j, r1, r2, r0, fr);
                if (j + 1 < NJ) phase(role_c, j + 1, r2, r0, r1, fr);
                if (j + 2 < NJ) phase(role_c, j + 2, r0, r1, r2, fr);
            }
        } else {
            f32x4 ra[9], rb[9];
            issue_loads(role_c, 0, true, ra);
            issue_loads(role_c, 1, true, rb);
            store_all(role_c, ra, lds16, 1.f);
            __syncthreads();
            prefetch(lds16, fr);
            for (int j = 0; j < NJ; j += 2) {
                phase(role_c, j, rb, rb, ra, fr);
                phase(role_c, j + 1, ra, ra, rb, fr);
            }
        }
    };
    if (NJ > 0) {
        if (wave == 0) run(std::integral_constant<int, 0>{});
        else if (wave == 3) run(std::integral_constant<int, 3>{});
        else run(std::integral_constant<int, 1>{});
    }
    if constexpr (H16) {                                            // back to the operands' units (exact)
        const float inv = f16_inv_scale_of(ez_run) * f16_inv_scale_of(ex_run);
#pragma unroll
        for (int t = 0; t < 9; ++t) acc[t] *= inv;
    }
    // one partial slab per (block, output row of the sub-tiles): [2 blk + ph][co][tap][ci]
    float* dst = part + (size_t)(blk * 2 + ph) * p.Co * 9 * p.Ct;
    const int ci = c_base + l32;
    if (ci < p.Ct) {
#pragma unroll
        for (int t = 0; t < 9; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int co = co_base + wco * 32 + (r & 3) + 8 * (r >> 2) + 4 * h;
                if (co < p.Co) dst[((size_t)co * 9 + t) * p.Ct + ci] = acc[t][r];
            }
    }
}

// ---------------------------------------------------------------------------------- halo-tile wgrad, 64 x 64 channel tiles
// 3x3 / stride 1 weight gradient for layers with >= 48 channels on both sides.  A block owns a (64 output channels) x
// (64 input channels) tile of dW for all 9 taps and walks 4x16-pixel output tiles: the dZ tile and the X tile WITH its
// one-pixel halo are staged in LDS once and feed all 9 taps (the per-tap blocks of conv_wgrad_kernel load both operands 9
// times and spend more issue slots on gather arithmetic than on MFMAs).  The 4 waves split the CHANNELS, not the pixels:
// wave (wco, wci) accumulates its 32 x 32 quadrant x 9 taps in 144 accumulator registers over every pixel of the
// block's tiles, so there is no cross-wave reduction.  v_mfma_f32_16x16x4_f32, k = 4 pixels per step.
__global__ __launch_bounds__(256) void wgrad_halo64_kernel(WgradP p, int ci_chunks, int tiles_x, int tiles_y, int tiles_per_block,
                                                           const float* __restrict__ x0, const float* __restrict__ x1,
                                                           const float* __restrict__ dz, float* __restrict__ part) {
    constexpr int TH = 4, TW = 16, XH = TH + 2, XW = TW + 2, PIX = TH * TW, LD = 64 + 4;
    __shared__ __attribute__((aligned(16))) float dZs[PIX * LD];
    __shared__ __attribute__((aligned(16))) float Xs[XH * XW * LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, q = lane >> 4;
    const int wco = wave & 1, wci = wave >> 1;
    const int co_base = blockIdx.y * 64;
    const int chunk = blockIdx.x % ci_chunks, blk = blockIdx.x / ci_chunks;
    const int c_base = chunk * 64;
    const int total_tiles = p.B * tiles_y * tiles_x;
    const int t_beg = blk * tiles_per_block, t_end = min(t_beg + tiles_per_block, total_tiles);
    // source of this channel chunk (chunks never straddle the two concat sources: C0 % 64 == 0 or C1 == 0)
    const bool s1 = c_base >= p.C0;
    const float* src = s1 ? x1 : x0;
    const int cs = s1 ? p.C1 : p.C0, c_src = s1 ? c_base - p.C0 : c_base;
    const bool up = p.up0 && !s1;
    const int Hs = up ? p.H / 2 : p.H, Ws = up ? p.W / 2 : p.W;

    f32x4 acc[2][2][9];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int t = 0; t < 9; ++t) acc[a][b][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Software pipeline over tiles (as in wgrad_small_kernel): tile t + 1 is loaded into registers during the MFMAs of tile t.
    constexpr int NZ = PIX * 16 / 256, NX = (XH * XW * 16 + 255) / 256;
    f32x4 zr[NZ], xr_[NX];
    auto load_tile = [&](int tile) {
        const int b = tile / (tiles_y * tiles_x), tr = tile % (tiles_y * tiles_x);
        const int ty0 = (tr / tiles_x) * TH, tx0 = (tr % tiles_x) * TW;
#pragma unroll
        for (int u = 0; u < NZ; ++u) {                          // dZ tile: [pixel][64] as float4
            const int i = tid + 256 * u, pix = i >> 4, c4 = i & 15;
            const int gy = ty0 + pix / TW, gx = tx0 + pix % TW;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (gy < p.Ho && gx < p.Wo && co_base + c4 * 4 < p.Co)
                v = *reinterpret_cast<const f32x4*>(dz + (((size_t)b * p.Ho + gy) * p.Wo + gx) * p.Co + co_base + c4 * 4);
            zr[u] = v;
        }
#pragma unroll
        for (int u = 0; u < NX; ++u) {                          // X halo tile: [position][64] as float4
            const int i = tid + 256 * u;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (i < XH * XW * 16) {
                const int pos = i >> 4, c4 = i & 15;
                int iy = ty0 + pos / XW - 1, ix = tx0 + pos % XW - 1;
                if (p.pad_mode == 1) { iy = reflect_idx(iy, p.H); ix = reflect_idx(ix, p.W); }
                if (iy >= 0 && iy < p.H && ix >= 0 && ix < p.W && c_src + c4 * 4 < cs) {
                    if (up) { iy >>= 1; ix >>= 1; }
                    v = *reinterpret_cast<const f32x4*>(src + (((size_t)b * Hs + iy) * Ws + ix) * cs + c_src + c4 * 4);
                }
            }
            xr_[u] = v;
        }
    };
    if (t_beg < t_end) load_tile(t_beg);
    for (int tile = t_beg; tile < t_end; ++tile) {
        __syncthreads();                                        // previous tile's MFMAs are done with the LDS
#pragma unroll
        for (int u = 0; u < NZ; ++u) {
            const int i = tid + 256 * u;
            *reinterpret_cast<f32x4*>(dZs + (i >> 4) * LD + (i & 15) * 4) = zr[u];
        }
#pragma unroll
        for (int u = 0; u < NX; ++u) {
            const int i = tid + 256 * u;
            if (i < XH * XW * 16) *reinterpret_cast<f32x4*>(Xs + (i >> 4) * LD + (i & 15) * 4) = xr_[u];
        }
        __syncthreads();
        if (tile + 1 < t_end) load_tile(tile + 1);
#pragma unroll 2
        for (int j = 0; j < PIX / 4; ++j) {                     // k-steps of 4 pixels over the whole tile
            const int pix = j * 4 + q;
            const int py = pix / TW, px = pix % TW;
            float af[2];
#pragma unroll
            for (int a = 0; a < 2; ++a) af[a] = dZs[pix * LD + (wco * 2 + a) * 16 + l16];
#pragma unroll
            for (int ky = 0; ky < 3; ++ky)
#pragma unroll
                for (int kx = 0; kx < 3; ++kx) {
                    const float* xr = Xs + ((py + ky) * XW + px + kx) * LD + wci * 32 + l16;
#pragma unroll
                    for (int bb = 0; bb < 2; ++bb) {
                        const float bv = xr[bb * 16];
#pragma unroll
                        for (int a = 0; a < 2; ++a)
                            acc[a][bb][ky * 3 + kx] = __builtin_amdgcn_mfma_f32_16x16x4f32(af[a], bv, acc[a][bb][ky * 3 + kx], 0, 0, 0);
                    }
                }
        }
    }
    // partial slab [blk][co][tap][ci]; C layout: column (ci) = lane & 15, row (co) = (lane >> 4) * 4 + reg
    float* dst = part + (size_t)blk * p.Co * 9 * p.Ct;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int bb = 0; bb < 2; ++bb) {
            const int ci = c_base + (wci * 2 + bb) * 16 + l16;
            if (ci >= p.Ct) continue;
#pragma unroll
            for (int t = 0; t < 9; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int co = co_base + (wco * 2 + a) * 16 + q * 4 + r;
                    if (co < p.Co) dst[((size_t)co * 9 + t) * p.Ct + ci] = acc[a][bb][t][r];
                }
        }
}

struct SmallPlan { bool ok, stem, halo64, co32; int mt, nt, ci_chunks, co_groups, tiles_x, tiles_y, nblk, tiles_per_block, splits; };

// Halo-tile weight gradient on the bf16 matrix cores with 3-piece operands (wgrad_halo64s_kernel); CODEPS_WGRAD_SPLIT=0 or
// CODEPS_SPLIT != 3 selects the f32-MFMA kernel.
// Operand arithmetic of the conv engine: 3 (default) = exact 3-way bf16 split on the bf16 MFMA, 0 = f32 MFMA, 2 = two pieces
// (experiments only).  Initialised from CODEPS_SPLIT; codeps_conv2d_set_arith switches it at run time (A/B runs and the
// precision tests, which compare the split kernels with the f32-MFMA kernels on the same tensors in one process).
// Form of the halo-tile ring kernel: 0 (default) = the 256-thread kernel (conv_halo3r_kernel), 1 (CODEPS_HALO_WS=1) = producer /
// consumer waves (conv_halo3p_kernel).  Bit-identical results; codeps_conv2d_set_halo_ws switches at run time (the tests compare the
// two).  Round 4 measured the two within 1 % of each other on every layer and the step 0.4 % SLOWER with the producer form (33.78 vs
// 33.64 ms, alternating runs on one box): the consumers' 20 % fewer cycles per tap come back as a lower clock (2.13 vs 2.32 GHz in
// the kernel) -- DESIGN.md section 6c.
static int g_halo_ws = -1;
static int halo_ws_on() {
    if (g_halo_ws < 0) g_halo_ws = getenv("CODEPS_HALO_WS") ? (atoi(getenv("CODEPS_HALO_WS")) != 0) : 0;
    return g_halo_ws;
}

static int g_split_np = -1;
static int split_raw() {
    if (g_split_np < 0) g_split_np = getenv("CODEPS_SPLIT") ? atoi(getenv("CODEPS_SPLIT")) : 16;
    return g_split_np;
}
// 16 = two fp16 pieces in the kernels that have that form (f16_pairs()); every other kernel runs the three-bf16-piece arithmetic under it
static int split_pieces() { return split_raw() == 16 ? 3 : split_raw(); }
static bool f16_pairs() { return split_raw() == 16; }

static bool wgrad_split_on() {
    static const bool env_on = getenv("CODEPS_WGRAD_SPLIT") ? atoi(getenv("CODEPS_WGRAD_SPLIT")) != 0 : true;
    const bool on = env_on && split_pieces() == 3;
    return on;
}
// channel tiles (64 x 64) a layer must have for the halo kernel: the split kernel also takes single-tile 64 -> 64 layers
static int halo_min_tiles() {
    static const int env_v = getenv("CODEPS_HALO_MIN_TILES") ? atoi(getenv("CODEPS_HALO_MIN_TILES")) : 0;
    const int v = env_v ? env_v : (wgrad_split_on() ? 1 : 2);
    return v;
}

static SmallPlan wgrad_small_plan(const codeps_conv_desc* d) {
    SmallPlan s;
    memset(&s, 0, sizeof(s));
    const int Ct = d->c0 + d->c1;
    s.co_groups = 1;
    const bool stem77 = d->kh == 7 && d->kw == 7 && d->stride == 2 && d->stride_w == 2 && d->pad_w == d->pad;
    const bool stem74 = d->kh == 7 && d->kw == 4 && d->stride == 2 && d->stride_w == 1;          // double-pixel layout (functional.stem_conv2d)
    if ((stem77 || stem74) && Ct == 16 && d->c1 == 0 && !d->up0 && (d->out_c % 16) == 0 && d->pad_mode == 0) {
        // ResNet stem (7x7 / 2 on the 16-channel padded image, or its 7x4 double-pixel form): 4x16-pixel output tiles, one
        // 16-channel output group per block
        s.ok = s.stem = true;
        s.mt = 1; s.nt = 1; s.ci_chunks = 1; s.co_groups = d->out_c / 16;
        const bool stem_split = stem74 && d->out_c == 64 && wgrad_split_on() && !(getenv("CODEPS_STEM_SPLIT") && atoi(getenv("CODEPS_STEM_SPLIT")) == 0);
        if (stem_split) s.co_groups = 1;                          // wgrad_stem74s_kernel: all 64 output channels in one block
        s.tiles_x = cdiv(d->out_w, 16); s.tiles_y = cdiv(d->out_h, 4);
        const int total = d->batch * s.tiles_x * s.tiles_y;
        static const int stem_blocks = getenv("CODEPS_STEM_BLOCKS") ? atoi(getenv("CODEPS_STEM_BLOCKS")) : 768;   // env: tuning experiments only
        static const int stem_sblocks = getenv("CODEPS_STEM_SBLOCKS") ? atoi(getenv("CODEPS_STEM_SBLOCKS")) : 256;   // split kernel: 312 VGPRs -> 1 block / CU, one round
        s.tiles_per_block = std::max(8, cdiv(total, std::max(1, (stem_split ? stem_sblocks : stem_blocks) / s.co_groups)));
        s.nblk = cdiv(total, s.tiles_per_block);
        s.splits = s.nblk;
        return s;
    }
    static const int halo_off = getenv("CODEPS_NO_HALO64") ? 1 : 0;                                    // tuning experiments only
    // <= 32 output channels (the decoders' half-resolution stages, f32 MFMA until round 3): the split kernel's CO32 form
    static const int co32_on = getenv("CODEPS_WGRAD_CO32") ? atoi(getenv("CODEPS_WGRAD_CO32")) : 1;       // tuning experiments only
    const bool co32 = co32_on && wgrad_split_on() && d->out_c > 16 && d->out_c <= 32;
    if (!halo_off && d->kh == 3 && d->kw == 3 && d->stride == 1 && d->stride_w == 1 && d->pad == 1 && d->pad_w == 1 && (d->out_c >= 48 || co32) && Ct >= 48 &&
        (co32 || cdiv(Ct, 64) * cdiv(d->out_c, 64) >= halo_min_tiles()) && (d->c1 == 0 || d->c0 % 64 == 0 || wgrad_split_on()) &&
        d->out_h == d->in_h && d->out_w == d->in_w) {
        // 64 x 64 channel tiles over 4x16-pixel tiles with halo (wgrad_halo64_kernel); a single-tile 64 -> 64 layer would need
        // ~768 pixel blocks = 768 partial slabs, where the per-tap kernel measures faster
        s.ok = s.halo64 = true;
        s.ci_chunks = cdiv(Ct, 64); s.co_groups = cdiv(d->out_c, 64);
        s.tiles_x = cdiv(d->out_w, 16); s.tiles_y = cdiv(d->out_h, 4);
        const int total = d->batch * s.tiles_x * s.tiles_y;
        // f32 kernel: 228 VGPRs -> 2 blocks per CU: exactly one balanced round of <= 512 blocks (measured: 512 -> 54.8 ms/step,
        // 448 -> 55.7, 576 -> 56.8); split kernel: 82 KB of LDS -> 1 block per CU, one round of 256 (256 -> 45.9, 512 -> 46.2, 768 -> 46.9)
        static const int env_halo_blocks = getenv("CODEPS_HALO_BLOCKS") ? atoi(getenv("CODEPS_HALO_BLOCKS")) : 0;   // env: tuning experiments only
        const int halo_blocks = env_halo_blocks ? env_halo_blocks : (wgrad_split_on() ? 256 : 512);
        const int want = std::max(1, halo_blocks / (s.ci_chunks * s.co_groups));
        s.tiles_per_block = std::max(2, cdiv(total, want));
        s.nblk = cdiv(total, s.tiles_per_block);
        s.splits = co32 ? 2 * s.nblk : s.nblk;                   // CO32: one slab per pixel half
        s.co32 = co32;
        return s;
    }
    s.ok = d->stride == 1 && d->stride_w == 1 && d->pad_w == d->pad && d->kh == d->kw && (d->kh == 1 || d->kh == 3) && d->out_c <= 32 &&
           d->out_h == d->in_h && d->out_w == d->in_w;
    if (!s.ok) return s;
    s.mt = d->out_c > 16 ? 2 : 1;
    s.nt = (Ct % 32 == 0 && (d->c1 == 0 || d->c0 % 32 == 0)) ? 2 : 1;
    if (s.nt == 1 && d->c1 > 0 && d->c0 % 16 != 0) { s.ok = false; return s; }
    s.ci_chunks = cdiv(Ct, s.nt * 16);
    s.tiles_x = cdiv(d->out_w, 32); s.tiles_y = cdiv(d->out_h, 8);
    const int total = d->batch * s.tiles_x * s.tiles_y;
    static const int small_blocks = getenv("CODEPS_SMALL_BLOCKS") ? atoi(getenv("CODEPS_SMALL_BLOCKS")) : 512;   // env: tuning experiments only
    int want = std::max(1, small_blocks / s.ci_chunks);                // one balanced round of 2 blocks per CU
    s.tiles_per_block = std::max(4, cdiv(total, want));
    s.nblk = cdiv(total, s.tiles_per_block);
    s.splits = s.nblk;
    return s;
}

// 1 x 1 convolutions (any stride, no padding, one source) with >= 48 channels on both sides: wgrad_1x1s_kernel
struct W1Plan { bool ok, swap; int tb, tiles, splits, pps; };
static W1Plan wgrad_1x1_plan(const codeps_conv_desc* d) {
    W1Plan w;
    memset(&w, 0, sizeof(w));
    static const int on = getenv("CODEPS_WGRAD_1X1S") ? atoi(getenv("CODEPS_WGRAD_1X1S")) : 1;       // A/B switch
    const int P = d->batch * d->out_h * d->out_w;
    w.ok = on && wgrad_split_on() && d->kh == 1 && d->kw == 1 && d->pad == 0 && d->pad_w == 0 && d->c1 == 0 && !d->up0 && d->pad_mode == 0 &&
           d->pix_pitch == 0 && d->out_c >= 48 && d->c0 >= 48 && (d->out_c % 4) == 0 && (d->c0 % 4) == 0 && P >= 512 &&
           (d->out_h - 1) * d->stride < d->in_h && (d->out_w - 1) * d->stride_w < d->in_w &&
           (size_t)d->batch * d->in_h * d->in_w * d->c0 * 4 < (size_t)GATHER_OOB && (size_t)P * d->out_c * 4 < (size_t)GATHER_OOB;     // 32-bit byte offsets
    if (!w.ok) return w;
    w.swap = d->c0 > d->out_c;                                     // the wider operand takes the 256-channel side of the tile
    const int CA = w.swap ? d->c0 : d->out_c, CB = w.swap ? d->out_c : d->c0;
    w.tb = CB > 64 ? 2 : 1;                                        // B side: 128 channels, or 64 (two blocks per CU)
    w.tiles = cdiv(CA, 256) * cdiv(CB, 64 * w.tb);
    // one balanced round: ~256 blocks (512 for the 64-channel form), >= 4 K-steps of 32 pixels each
    const int s = std::max(1, std::min((w.tb == 1 ? 512 : 256) / w.tiles, P / 128));
    w.pps = (int)align_up((size_t)cdiv(P, s), 32);
    w.splits = cdiv(P, w.pps);
    return w;
}

// sum the split slabs and scatter into the OIHW gradient: dw[co][ci][ky][kx] (+= if accumulate).
// The slabs are [split][co][tap][ci] with ci padded to a multiple of 16: a thread owns four neighbouring ci of one (co, tap) and
// every SG-th slab (16-byte loads, four in flight), the SG partial sums of a column meet in LDS in a fixed order -- the layers
// with one 64 x 64 channel tile have 256 slabs of 36 864 elements, where one thread per element walked 256 slabs alone.
template <int SG>
__global__ __launch_bounds__(256) void wgrad_reduce_kernel(const f32x4* __restrict__ part, int splits, long long total4, int Ct,
                                                           int taps, int co_real, int ci_real, float* __restrict__ dw, int accumulate) {
    constexpr int IL = 256 / SG;                       // float4 columns per block
    __shared__ f32x4 red[SG][IL];
    const int il = threadIdx.x % IL, sg = threadIdx.x / IL;
    const long long i4 = (long long)blockIdx.x * IL + il;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    if (i4 < total4) {
#pragma unroll 4
        for (int s = sg; s < splits; s += SG) a += part[(size_t)s * total4 + i4];
    }
    red[sg][il] = a;
    __syncthreads();
    if (sg != 0 || i4 >= total4) return;
#pragma unroll
    for (int k = 1; k < SG; ++k) a += red[k][il];
    const long long i = i4 * 4;
    const int ci = (int)(i % Ct);
    const int tap = (int)((i / Ct) % taps);
    const int co = (int)(i / ((long long)Ct * taps));
    if (co >= co_real) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (ci + e >= ci_real) break;
        const size_t o = ((size_t)co * ci_real + ci + e) * taps + tap;
        dw[o] = accumulate ? dw[o] + a[e] : a[e];
    }
}

// 3x3 layers: one block per (output channel, 64 input channels) owns all nine taps, so that the OIHW scatter ([ci][tap]: a
// 36-byte stride per tap-major element) becomes one contiguous run of 576 floats through an LDS transpose.  Slab s goes to lane
// group s mod 16; the groups meet in LDS in a fixed order.
__global__ __launch_bounds__(256) void wgrad_reduce9_kernel(const f32x4* __restrict__ part, int splits, long long total4, int Ct, int n_chunks,
                                                            int co_real, int ci_real, float* __restrict__ dw, int accumulate) {
    __shared__ f32x4 red[16][9 * 16];
    __shared__ float outt[9 * 64 + 8];
    const int co = blockIdx.x / n_chunks, ci0 = (blockIdx.x % n_chunks) * 64;
    const int l = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int cw = min(64, Ct - ci0);                                 // padded channels of this chunk (a multiple of 16)
    if (co >= co_real) return;
    f32x4 acc[9];
#pragma unroll
    for (int t = 0; t < 9; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (l * 4 < cw) {
        const size_t base = ((size_t)co * 9 * Ct + ci0) / 4 + l;
        for (int sl = g; sl < splits; sl += 16) {
            const f32x4* ps = part + (size_t)sl * total4 + base;
#pragma unroll
            for (int t = 0; t < 9; ++t) acc[t] += ps[(size_t)t * (Ct / 4)];
        }
    }
#pragma unroll
    for (int t = 0; t < 9; ++t) red[g][t * 16 + l] = acc[t];
    __syncthreads();
    if (threadIdx.x < 9 * 16) {
        f32x4 a = red[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 16; ++k) a += red[k][threadIdx.x];
        const int t = threadIdx.x / 16, c4 = threadIdx.x % 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) outt[(c4 * 4 + e) * 9 + t] = a[e];   // [ci][tap]
    }
    __syncthreads();
    const int n_real = min(cw, ci_real - ci0);
    float* dst = dw + ((size_t)co * ci_real + ci0) * 9;
    for (int i = threadIdx.x; i < n_real * 9; i += 256) dst[i] = accumulate ? dst[i] + outt[i] : outt[i];
}

static void launch_wgrad_reduce(const float* part, int splits, int Co, int Ct, int taps, int co_real, int ci_real, float* dw, int accumulate,
                                hipStream_t st) {
    const long long total4 = (long long)Co * Ct * taps / 4;      // Ct is a multiple of 16
    static const int red9 = getenv("CODEPS_REDUCE9") ? atoi(getenv("CODEPS_REDUCE9")) : 1;
    if (red9 && taps == 9 && Ct >= 64 && ci_real > 0) {
        const int n_chunks = cdiv(Ct, 64);
        hipLaunchKernelGGL(wgrad_reduce9_kernel, dim3(Co * n_chunks), dim3(256), 0, st, reinterpret_cast<const f32x4*>(part), splits, total4, Ct,
                           n_chunks, co_real, ci_real, dw, accumulate);
        return;
    }
    // few columns and many slabs: 16 slab groups per block (16 columns), else 4 (64 columns)
    if (total4 / 64 < 1024 && splits >= 32)
        hipLaunchKernelGGL(wgrad_reduce_kernel<16>, dim3((int)((total4 + 15) / 16)), dim3(256), 0, st, reinterpret_cast<const f32x4*>(part), splits,
                           total4, Ct, taps, co_real, ci_real, dw, accumulate);
    else
        hipLaunchKernelGGL(wgrad_reduce_kernel<4>, dim3((int)((total4 + 63) / 64)), dim3(256), 0, st, reinterpret_cast<const f32x4*>(part), splits,
                           total4, Ct, taps, co_real, ci_real, dw, accumulate);
}

// OIHW -> forward pack [co][tap][ci] and dgrad pack [ci][tap][co]
__global__ __launch_bounds__(256) void pack_weights_kernel(const float* __restrict__ w, int co_real, int ci_real, int taps,
                                                           int Co, int Ci, float* __restrict__ wf, float* __restrict__ wd) {
    // enumerate the channel-padded index space; padding rows/columns are zero
    const long long total = (long long)Co * Ci * taps;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int tap = (int)(i % taps);
        const int ci = (int)((i / taps) % Ci);
        const int co = (int)(i / ((long long)taps * Ci));
        const float v = (co < co_real && ci < ci_real) ? w[((size_t)co * ci_real + ci) * taps + tap] : 0.f;
        if (wf) wf[((size_t)co * taps + tap) * Ci + ci] = v;
        if (wd) wd[((size_t)ci * taps + tap) * Co + co] = v;
    }
}

// fp32 pack [rows][wrow] -> [rows][wrow / 32][3 pieces][32] bf16 with the same split the kernel applies to activations
__global__ __launch_bounds__(256) void split_pack_kernel(const float* __restrict__ wq, long long n_chunks, unsigned short* __restrict__ out) {
    for (long long c = (long long)blockIdx.x * 256 + threadIdx.x; c < n_chunks; c += (long long)gridDim.x * 256) {     // chunk = 8 consecutive k
        const f32x4 a = *reinterpret_cast<const f32x4*>(wq + c * 8), b = *reinterpret_cast<const f32x4*>(wq + c * 8 + 4);
        u16x4 lo[3], hi[3];
        split_bf16<3>(a, lo);
        split_bf16<3>(b, hi);
        unsigned short* g = out + (c / 4) * 96 + (c % 4) * 8;
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<i32x4*>(g + q * 32) = pack8(lo[q], hi[q]);
    }
}

// All trainable weights of a step in ONE launch (instead of one pack + up to two split launches per layer and step): `items`
// is a device table, one entry per (parameter, pack kind).  Blocks find their item by bisection over the items' first
// work-group index.  A work group moves one SLAB through LDS so that both sides are coalesced (round 2 read the OIHW
// parameter with a stride of `taps` floats per thread: 10x its bytes from HBM by the counters):
//   forward pack  [co][tap][ci]: slab = one row co x up to `cbw` columns ci: ONE contiguous OIHW run of cbw * taps floats in,
//                                taps runs of cbw floats out;
//   dgrad pack    [ci][tap][co]: slab = `rb` rows ci x 64 columns co: per co one contiguous run of rb * taps floats in,
//                                rb * taps runs of 64 floats out.
// A thread then emits 8 consecutive k of a pack row -- the fp32 pack (32 bytes) and, when the row takes the split-operand
// kernel, its three bf16 pieces (3 x 16 bytes) -- exactly the bytes codeps_conv2d_pack_weights writes.
constexpr int PACK_SLAB = 4608;          // floats of LDS per work group (512 columns x 9 taps)
constexpr long long PACK_AMAX_INLINE = 32768;      // parameters up to this many elements: every pack group takes the maximum itself (128 loads per thread)
// Layout of a pack buffer in floats, `total` = rows x K extent (codeps_conv2d_packed_weight_floats):  [0, total) the fp32 pack;
// [total, 2.5 total) three bf16 pieces (6 bytes per element; written under arithmetic 3);  [2.5 total, 3.5 total) two fp16 pieces of w 2^kb
// (4 bytes per element; written under arithmetic 16);  [3.5 total, +4) the scale slot (2^-kb, 2^kb, max |w|, 0);  behind it one partial
// maximum per work group of the item.  A pack carries the pieces of the arithmetic it was made under (codeps_conv2d_set_arith: re-pack after a switch).
__host__ __device__ __forceinline__ long long pack_off_f16(long long total) { return total + (total * 6 + 3) / 4; }
__host__ __device__ __forceinline__ long long pack_off_scale(long long total) { return pack_off_f16(total) + total; }
struct PackItem {
    const float* w;              // OIHW parameter
    float* out;                  // fp32 pack [rows][taps * cols] (+ the split copy behind it when `split`)
    int co_real, ci_real, taps, rows, cols;      // rows x cols = padded (Co x Ci) for the forward pack, (Ci x Co) for the dgrad pack
    int dgrad, split;            // split: 0 fp32 only, 1 + the three bf16 pieces, 16 + the two fp16 pieces and their scale as well
    int cbw, rb;                 // slab shape: columns per slab (forward: <= 512; dgrad: 64), rows per slab (forward: 1)
    long long first_group, groups;               // work groups (slabs) of this item
};

// Per-tensor scale of the fp16 pieces, pass 1: work group u of an item takes the u-th share of the OIHW parameter and leaves the largest
// magnitude it saw behind the scale slot; the pack's groups (pass 2, the next launch) each reduce the item's partials -- no atomics, no
// zeroing, the same bits whatever the order of the groups.
__device__ __forceinline__ void pack_amax_body(const PackItem& it, long long g, float* red) {
    if (it.split != 16 || (long long)it.co_real * it.ci_real * it.taps <= PACK_AMAX_INLINE) return;
    const long long total = (long long)it.rows * it.taps * it.cols;
    const long long n = (long long)it.co_real * it.ci_real * it.taps;
    const int u = (int)(g - it.first_group);
    const long long per = (n + it.groups - 1) / it.groups;
    const long long i0 = (long long)u * per, i1 = min(n, i0 + per);
    float m = 0.f;
    for (long long i = i0 + threadIdx.x; i < i1; i += 256) m = fmaxf(m, fabsf(it.w[i]));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) it.out[pack_off_scale(total) + 4 + u] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

__device__ __forceinline__ void pack_item_body(const PackItem& it, long long g, float* slab) {
    const long long wrow = (long long)it.taps * it.cols;                   // k extent of a pack row
    const long long total = (long long)it.rows * wrow;
    const int u = (int)(g - it.first_group);
    float w_scale = 1.f;
    if (it.split == 16) {                                                  // every group of the item derives the same scale ...
        const float* part = it.out + pack_off_scale(total) + 4;
        const long long n_w = (long long)it.co_real * it.ci_real * it.taps;
        float m = 0.f;
        if (n_w <= PACK_AMAX_INLINE) {                                     // ... small tensors (re-laid-out stem / GUDA tap weights, packed one by one every step): from the parameter itself, no first pass
            for (long long i = threadIdx.x; i < n_w; i += 256) m = fmaxf(m, fabsf(it.w[i]));
        } else                                                             // ... from the partials of pack_amax_*_kernel
        for (long long i = threadIdx.x; i < it.groups; i += 256) m = fmaxf(m, part[i]);
        m = wave_max(m);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slab[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(slab[0], slab[1]), fmaxf(slab[2], slab[3]));
        __syncthreads();
        const int e = max((int)(__builtin_bit_cast(unsigned, m) >> 23), F16_EMIN);
        w_scale = f16_scale_of(e);
        if (u == 0 && threadIdx.x == 0) *reinterpret_cast<f32x4*>(it.out + pack_off_scale(total)) = f32x4{f16_inv_scale_of(e), w_scale, m, 0.f};
    }
    const int ncb = (it.cols + it.cbw - 1) / it.cbw;
    const int r0 = (u / ncb) * it.rb, c0 = (u % ncb) * it.cbw;
    const int ncol = min(it.cbw, it.cols - c0), nrow = min(it.rb, it.rows - r0);
    const int taps = it.taps;
    // ---- in: slab[(col * nrow + row) * taps + tap] (forward: nrow = 1 -> [col][tap], the OIHW order of one co)
    if (!it.dgrad) {
        const int n = ncol * taps;
        const int avail = (r0 < it.co_real) ? max(min(c0 + ncol, it.ci_real) - c0, 0) * taps : 0;
        const float* src = it.w + ((size_t)r0 * it.ci_real + c0) * taps;
        for (int i = threadIdx.x; i < n; i += 256) slab[i] = i < avail ? src[i] : 0.f;
    } else {
        const int run = nrow * taps, n = ncol * run;
        const int avail = max(min(r0 + nrow, it.ci_real) - r0, 0) * taps;       // floats of a run that exist (rows = ci)
        for (int i = threadIdx.x; i < n; i += 256) {
            const int col = i / run, k = i - col * run;
            const int co = c0 + col;
            slab[i] = (co < it.co_real && k < avail) ? it.w[((size_t)co * it.ci_real + r0) * taps + k] : 0.f;
        }
    }
    __syncthreads();
    // ---- out: chunks of 8 consecutive columns of one (row, tap)
    const int cpr = ncol / 8, nchunk = nrow * taps * cpr;
    for (int q = threadIdx.x; q < nchunk; q += 256) {
        const int jc = q % cpr, rt = q / cpr, tap = rt % taps, rr = rt / taps;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = slab[((jc * 8 + e) * nrow + rr) * taps + tap];
        const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
        const long long k = (long long)(r0 + rr) * wrow + (long long)tap * it.cols + c0 + jc * 8;     // first of the 8 k of this chunk
        const long long chunk = k / 8;
        float* dst = it.out + k;
        *reinterpret_cast<f32x4*>(dst) = a;
        *reinterpret_cast<f32x4*>(dst + 4) = b;
        if (it.split == 1) {                                               // (arithmetic 16 reads the fp16 pieces only: the pack skips the bf16 ones)
            u16x4 pl[3], ph[3];
            split_bf16<3>(a, pl);
            split_bf16<3>(b, ph);
            unsigned short* sp = reinterpret_cast<unsigned short*>(it.out + total) + (chunk / 4) * 96 + (chunk % 4) * 8;
#pragma unroll
            for (int qq = 0; qq < 3; ++qq) *reinterpret_cast<i32x4*>(sp + qq * 32) = pack8(pl[qq], ph[qq]);
        }
        if (it.split == 16) {
            u16x4 pl[2], ph[2];
            split_f16(a, w_scale, pl[0], pl[1]);
            split_f16(b, w_scale, ph[0], ph[1]);
            unsigned short* sp = reinterpret_cast<unsigned short*>(it.out + pack_off_f16(total)) + (chunk / 4) * 64 + (chunk % 4) * 8;
#pragma unroll
            for (int qq = 0; qq < 2; ++qq) *reinterpret_cast<i32x4*>(sp + qq * 32) = pack8(pl[qq], ph[qq]);
        }
    }
}

__global__ __launch_bounds__(256) void pack_amax_multi_kernel(const PackItem* __restrict__ items, int n_items) {
    __shared__ float red[4];
    int lo = 0, hi = n_items - 1;
    const long long g = blockIdx.x;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (items[mid].first_group <= g) lo = mid; else hi = mid - 1;
    }
    const PackItem it = items[lo];
    pack_amax_body(it, g, red);
}
__global__ __launch_bounds__(256) void pack_amax_pair_kernel(PackItem a, PackItem b) {
    __shared__ float red[4];
    if ((long long)blockIdx.x < a.groups) pack_amax_body(a, blockIdx.x, red);
    else pack_amax_body(b, blockIdx.x, red);
}

__global__ __launch_bounds__(256) void pack_weights_multi_kernel(const PackItem* __restrict__ items, int n_items) {
    __shared__ float slab[PACK_SLAB];
    int lo = 0, hi = n_items - 1;
    const long long g = blockIdx.x;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (items[mid].first_group <= g) lo = mid; else hi = mid - 1;
    }
    const PackItem it = items[lo];
    pack_item_body(it, g, slab);
}

// one parameter's forward and / or data-gradient pack (codeps_conv2d_pack_weights): the items travel as kernel arguments
__global__ __launch_bounds__(256) void pack_weights_pair_kernel(PackItem a, PackItem b) {
    __shared__ float slab[PACK_SLAB];
    if ((long long)blockIdx.x < a.groups) pack_item_body(a, blockIdx.x, slab);
    else pack_item_body(b, blockIdx.x, slab);
}

// ---------------------------------------------------------------------------------- host side
static int check_conv(const codeps_conv_desc* d, const char* who) {
    CODEPS_REQUIRE(d != nullptr, CODEPS_ERR_ARG, "%s: null descriptor", who);
    CODEPS_REQUIRE(d->batch > 0 && d->in_h > 0 && d->in_w > 0 && d->c0 > 0 && d->c1 >= 0 && d->out_c > 0, CODEPS_ERR_ARG,
                   "%s: bad shape", who);
    CODEPS_REQUIRE((d->stride == 1 || d->stride == 2) && (d->stride_w == 1 || d->stride_w == 2), CODEPS_ERR_ARG, "%s: stride (%d,%d) unsupported",
                   who, d->stride, d->stride_w);
    CODEPS_REQUIRE(d->pad >= 0 && d->pad_w >= 0 && d->kh > 0 && d->kw > 0, CODEPS_ERR_ARG, "%s: bad kernel / padding", who);
    const bool sym = d->stride_w == d->stride && d->pad_w == d->pad;
    CODEPS_REQUIRE(sym || (!d->up0 && d->pad_mode == 0 && d->out_c > 16), CODEPS_ERR_ARG,
                   "%s: per-dimension stride / padding needs zero padding, no fused upsample and out_c > 16", who);
    CODEPS_REQUIRE((d->c0 % 16) == 0 && (d->c1 % 16) == 0, CODEPS_ERR_ARG,
                   "%s: channel counts (%d,%d) must be multiples of 16 (pad the stem input)", who, d->c0, d->c1);
    CODEPS_REQUIRE(!d->up0 || ((d->in_h % 2) == 0 && (d->in_w % 2) == 0 && d->stride == 1 && d->stride_w == 1), CODEPS_ERR_ARG,
                   "%s: fused x2 upsample needs even size and stride 1", who);
    const int ho = (d->in_h + 2 * d->pad - d->kh) / d->stride + 1, wo = (d->in_w + 2 * d->pad_w - d->kw) / d->stride_w + 1;
    CODEPS_REQUIRE(ho == d->out_h && wo == d->out_w, CODEPS_ERR_ARG, "%s: output size %dx%d != expected %dx%d", who, d->out_h,
                   d->out_w, ho, wo);
    CODEPS_REQUIRE(d->pad_mode == 0 || (d->pad < d->in_h && d->pad < d->in_w), CODEPS_ERR_ARG, "%s: reflect pad too large", who);
    if (d->pix_pitch != 0) {
        CODEPS_REQUIRE(d->pix_pitch > 0 && d->pix_pitch % 4 == 0 && d->c0 >= d->pix_pitch && d->c1 == 0 && !d->up0 && d->kw == 1 && d->pad_w == 0 &&
                           d->stride_w == 1 && d->pad_mode == 0 && d->out_c > 16 &&
                           (long long)d->row_pitch * d->pix_pitch >= (long long)(d->in_w - 1) * d->pix_pitch + d->c0,
                       CODEPS_ERR_ARG, "%s: overlapping-pixel form needs pix_pitch %% 4 == 0, c0 >= pix_pitch, one source, kw 1, no horizontal "
                       "padding / stride, out_c > 16 and rows of >= (in_w - 1) * pix_pitch + c0 floats", who);
    }
    return CODEPS_OK;
}

// name of the kernel variant the last conv entry point launched (tests select variants by shape and check it)
static const char* volatile g_last_kernel = "";      // process-wide on purpose: autograd runs backward launches on its own thread
static const char* volatile g_last_finish = "";      // the finish pass of the last launch that was cut into K slices

static ConvP make_convp(const codeps_conv_desc* d) {
    ConvP p;
    memset(&p, 0, sizeof(p));
    p.B = d->batch; p.H = d->in_h; p.W = d->in_w; p.C0 = d->c0; p.C1 = d->c1; p.Ct = d->c0 + d->c1; p.up0 = d->up0;
    p.Co = d->out_c; p.Ho = d->out_h; p.Wo = d->out_w; p.KH = d->kh; p.KW = d->kw; p.stride = d->stride; p.pad = d->pad;
    p.stride_w = d->stride_w; p.pad_w = d->pad_w;
    p.pad_mode = d->pad_mode; p.act = d->act;
    p.pitch0 = d->pix_pitch; p.wrow0 = d->pix_pitch ? d->row_pitch : 0;
    return p;
}

// What the launches of the current entry-point call did with the requested epilogue extras (codeps_conv_epilogue's out fields)
struct EpiOut { int applied, n_seg, tile0[4], tpi[4], rows[4], tiles[4]; };
static thread_local EpiOut g_epi;

// Called by every launch site once the tile shape and the K split are known.  Statistics and the BatchNorm gate need every M tile
// inside one image; when that fails they are dropped together (the caller then runs the separate kernels on an UNGATED result:
// applied bit 0 stays clear).  With K slices the extras move into the finish pass (splitk_finish_ex_kernel; plain activation gates
// without statistics: splitk_finish_kernel).
constexpr int FIN_ROWS = 64;
static bool epi_plan(ConvP& p, int tile_rows, bool supported = true) {
    p.ex_fin = 0;
    if (!p.ex_gate_act && !p.ex_stat) return false;
    const bool bn = p.ex_gate_act == 3;
    int n_tiles = p.n_mt;
    if (p.ksplit > 1) {
        // K slices: the finish pass owns the epilogue.  Its extras form (splitk_finish_ex_kernel) works on 64-row tiles of the output
        // whatever GEMM kernel wrote the slices; plain activation gates without statistics stay on the simple finish kernel
        static const int fin_on = getenv("CODEPS_EPI_FINISH") ? atoi(getenv("CODEPS_EPI_FINISH")) : 1;      // A/B switch
        tile_rows = FIN_ROWS; n_tiles = cdiv(p.M, FIN_ROWS);
        const bool ok = fin_on && !p.par && p.N % 64 == 0 && (!(bn || p.ex_stat == 1) || (p.ex_img_rows > 0 && p.ex_img_rows % FIN_ROWS == 0));
        if (!ok) {
            if (bn) { p.ex_gate = nullptr; p.ex_gate_act = 0; }
            p.ex_stat = 0;
        }
        p.ex_fin = (bn || p.ex_stat) ? 1 : 0;
    } else {
        if (!supported) { p.ex_gate = nullptr; p.ex_gate_act = 0; p.ex_stat = 0; return false; }     // (a kernel form without the EX instantiation)
        if ((bn || p.ex_stat == 1) && (p.ex_img_rows <= 0 || p.ex_img_rows % tile_rows != 0)) {
            if (bn) { p.ex_gate = nullptr; p.ex_gate_act = 0; }
            p.ex_stat = 0;
        }
    }
    if (p.ex_gate_act) g_epi.applied |= 1;
    if (p.ex_stat) {
        g_epi.applied |= 2;
        for (int c = 0; c < (p.par == 2 ? 4 : 1) && g_epi.n_seg < 4; ++c) {          // (all parity classes in one launch: one segment each)
            const int k = g_epi.n_seg++;
            g_epi.tile0[k] = p.ex_tile0 + c * n_tiles; g_epi.rows[k] = tile_rows; g_epi.tiles[k] = n_tiles;
            g_epi.tpi[k] = p.ex_img_rows > 0 ? p.ex_img_rows / tile_rows : 0;
        }
    }
    return p.ksplit <= 1 && (p.ex_gate_act || p.ex_stat);          // true: launch the kernel's EX instantiation (K slices: the finish pass gates)
}

// K slices a launch of `blocks` tiles with `nsteps` K-steps is cut into (1 = no split-K); shared by the cost model and the launcher
static int splitk_slices(const ConvP& p, int blocks, int nsteps) {
    static const int sk_blocks = getenv("CODEPS_SPLITK_BLOCKS") ? atoi(getenv("CODEPS_SPLITK_BLOCKS")) : 192;   // env: tuning experiments only
    static const int sk_target = getenv("CODEPS_SPLITK_TARGET") ? atoi(getenv("CODEPS_SPLITK_TARGET")) : 512;
    if (!p.part || p.par || blocks >= sk_blocks || nsteps < 16) return 1;      // (the parity-class rows are not the output's rows: no K slices there)
    int ks = std::min(std::min(sk_target / blocks, nsteps / 8), 16);
    while (ks >= 2 && (size_t)ks * p.M * p.N * sizeof(float) > p.part_bytes) --ks;
    return std::max(ks, 1);
}

// K slices (over 32-channel chunks) of the halo-tile ring kernel for grids of fewer than 256 blocks (it runs one block per CU).
// Model in units of one chunk (nine taps, ~11.5 us): rounds x (chunks per slice + 1.5 for fill / epilogue) + the finish pass
// (a launch + (slices + 1) x M x N floats of traffic).  0 = leave the layer to the gather kernels (too few blocks and nothing
// to cut), 1 = the ring kernel without split, >= 2 = that many slices.
static int halo_splitk_slices(const ConvP& p, int blocks, int nchunks) {
    static const int on = getenv("CODEPS_HALO_SPLITK") ? atoi(getenv("CODEPS_HALO_SPLITK")) : 1;             // tuning experiments only
    if (!on || blocks >= 256) return 0;
    int best = blocks >= 128 ? 1 : 0;
    double best_t = blocks >= 128 ? nchunks + 1.5 : 1e300;
    if (p.part && nchunks >= 8)
        for (int ks = 2; ks <= 8 && nchunks / ks >= 4; ++ks) {
            if ((size_t)ks * p.M * p.N * sizeof(float) > p.part_bytes) break;
            const int per = cdiv(nchunks, ks), slices = cdiv(nchunks, per);
            const double finish = 0.35 + (double)p.M * p.N * 4.0 * (slices + 1) / 5e12 / 11.5e-6;
            const double t = (double)cdiv(blocks * slices, 256) * (per + 1.5) + finish;
            if (t < best_t - 1e-9) { best_t = t; best = slices; }
        }
    return best;
}

// split-K finish: out = act((sum_z part[z]) * scale + shift + residual), fixed summation order
__global__ __launch_bounds__(256) void splitk_finish_kernel(const float* __restrict__ part, int ksplit, long long MN, int N,
                                                            const float* __restrict__ scale, const float* __restrict__ shift,
                                                            const float* __restrict__ residual, int act, float* __restrict__ out,
                                                            const float* __restrict__ gate, int gate_act) {
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < MN; i += (long long)gridDim.x * 1024) {
        f32x4 v = *reinterpret_cast<const f32x4*>(part + i);
        for (int z = 1; z < ksplit; ++z) v += *reinterpret_cast<const f32x4*>(part + (size_t)z * MN + i);
        const int n = (int)(i % N);
        if (scale) v = v * *reinterpret_cast<const f32x4*>(scale + n);
        if (shift) v += *reinterpret_cast<const f32x4*>(shift + n);
        if (residual) v += *reinterpret_cast<const f32x4*>(residual + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = apply_act(v[e], act);
        if (gate) {                                               // ConvP.ex_gate_act 1 / 2 (epi_apply's product)
            const f32x4 g = *reinterpret_cast<const f32x4*>(gate + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= g[e] > 0.f ? 1.f : (gate_act == 2 ? g[e] + 1.f : 0.f);
        }
        *reinterpret_cast<f32x4*>(out + i) = v;
    }
}

// The same finish with the epilogue extras (ConvP.ex_*: gates 1-3, statistics 1-3): block = 64 rows x 64 columns of the output (small-M
// layers: M / 64 x N / 64 blocks fill the chip where 256-column blocks left half of it idle -- 28 us per launch against 9), a thread
// owns one column quad and every 16th row (epi_begin / epi_apply / epi_flush as in the GEMM kernels' epilogues), so the per-tile
// partial statistics come out in the layout codeps_bn_finalize_tiles / codeps_bn_bwd_tiles / codeps_colsum_finish read.
constexpr int FIN_COLS = 64;
__global__ __launch_bounds__(256) void splitk_finish_ex_kernel(ConvP p, const float* __restrict__ scale, const float* __restrict__ shift,
                                                               const float* __restrict__ residual, int act, float* __restrict__ out) {
    __shared__ __attribute__((aligned(16))) float red[2 * 256 * 4];
    constexpr int V4 = FIN_COLS / 4, RPASS = 256 / V4, NR = FIN_ROWS / RPASS;
    const int tid = threadIdx.x, c4 = tid % V4, k = tid / V4;
    const int tile = blockIdx.x, n = blockIdx.y * FIN_COLS + c4 * 4;          // (N is a multiple of 64: epi_plan)
    const long long MN = (long long)p.M * p.N;
    const int m0 = tile * FIN_ROWS;
    EpiCtx ec;
    epi_begin(p, ec, p.ex_img_rows ? m0 / p.ex_img_rows : 0, n);
    f32x4 sc = {1.f, 1.f, 1.f, 1.f}, sh = {0.f, 0.f, 0.f, 0.f};
    if (scale) sc = *reinterpret_cast<const f32x4*>(scale + n);
    if (shift) sh = *reinterpret_cast<const f32x4*>(shift + n);
    f32x4 v[NR];
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        const int m = m0 + k + u * RPASS;
        v[u] = m < p.M ? *reinterpret_cast<const f32x4*>(p.part + (size_t)m * p.N + n) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int z = 1; z < p.ksplit; ++z)
#pragma unroll
        for (int u = 0; u < NR; ++u) {
            const int m = m0 + k + u * RPASS;
            if (m < p.M) v[u] += *reinterpret_cast<const f32x4*>(p.part + (size_t)z * MN + (size_t)m * p.N + n);
        }
    if (p.ex_stat == 1) {                                  // the tile's first row = the statistics' shift
        const size_t i0 = (size_t)m0 * p.N + n;
        f32x4 f = *reinterpret_cast<const f32x4*>(p.part + i0);
        for (int z = 1; z < p.ksplit; ++z) f += *reinterpret_cast<const f32x4*>(p.part + (size_t)z * MN + i0);
        ec.sh = f * sc + sh;
    }
    f32x4 resv[NR];
    EpiPre pre[NR];                                            // (residual and the gates' tensors: all rows before the first store, see EpiPre)
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        const int m = m0 + k + u * RPASS;
        const size_t i = (size_t)(m < p.M ? m : 0) * p.N + n;
        resv[u] = (residual && m < p.M) ? *reinterpret_cast<const f32x4*>(residual + i) : f32x4{0.f, 0.f, 0.f, 0.f};
        pre[u] = epi_prefetch(p, i, m < p.M);
    }
#pragma unroll
    for (int u = 0; u < NR; ++u) {
        const int m = m0 + k + u * RPASS;
        if (m >= p.M) continue;
        const size_t i = (size_t)m * p.N + n;
        f32x4 r = v[u];
        if (scale) r = r * sc;
        if (shift) r += sh;
        if (residual) r += resv[u];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = apply_act(r[e], act);
        *reinterpret_cast<f32x4*>(out + i) = epi_apply(p, ec, r, pre[u]);
    }
    epi_flush(p, ec, red, tid, V4, RPASS, tile, n);
}

template <int MODE>
static void launch_splitk_finish(const ConvP& p, hipStream_t st, const float* scale, const float* shift, const float* residual, float* out) {
    const long long MN = (long long)p.M * p.N;
    const float* sc = MODE == MODE_FWD ? scale : nullptr;
    const float* sh = MODE == MODE_FWD ? shift : nullptr;
    const int act = MODE == MODE_FWD ? p.act : 0;
    g_last_finish = p.ex_fin ? "splitk_finish_ex_kernel" : "splitk_finish_kernel";
    if (p.ex_fin)
        hipLaunchKernelGGL(splitk_finish_ex_kernel, dim3(cdiv(p.M, FIN_ROWS), p.N / FIN_COLS), dim3(256), 0, st, p, sc, sh, residual, act, out);
    else
        hipLaunchKernelGGL(splitk_finish_kernel, dim3((int)std::min<long long>((MN / 4 + 255) / 256, 2048)), dim3(256), 0, st, p.part, p.ksplit, MN,
                           p.N, sc, sh, residual, act, out, p.ex_gate, p.ex_gate_act);
}

// 3x3 / stride 1 / zero padding layers the halo-tile kernels take (forward: also the decoder's concat + fused nearest-x2 input)
template <int MODE>
static bool halo3_shape_ok(const ConvP& p) {
    static const int halo3_up = getenv("CODEPS_HALO3_UP") ? atoi(getenv("CODEPS_HALO3_UP")) : 1;
    const int Hm_ = (MODE == MODE_FWD) ? p.Ho : p.H, Wm_ = (MODE == MODE_FWD) ? p.Wo : p.W;
    const bool plain = !p.up0 && p.C1 == 0;
    return p.KH == 3 && p.KW == 3 && p.stride == 1 && p.stride_w == 1 && p.pad == 1 && p.pad_w == 1 && p.pad_mode == 0 &&
           !p.par && p.Ho == p.H && p.Wo == p.W && Wm_ % 32 == 0 && Hm_ % 4 == 0 &&
           (MODE == MODE_FWD ? (plain || (halo3_up && p.C0 % 32 == 0 && p.C1 % 32 == 0 && (!p.up0 || (p.H % 2 == 0 && p.W % 2 == 0))))
                             : (plain && p.src == 0 && p.Cs == p.C0));
}

template <int MODE, int WM, int WN, int TM, int TN, int BK, int NBUF = 2, int NP = 0>
static void launch_igemm(ConvP p, const float* a0, const float* a1, const float* wq, const float* scale, const float* shift,
                         const float* residual, float* out, hipStream_t st) {
    constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
    p.n_mt = cdiv(p.M, BM); p.n_nt = cdiv(p.N, BN);
    // K-loop staging buffers + the gather table [sources][taps][BM] behind them; the epilogue tile reuses the front
    const int ntap = (MODE == MODE_DGRAD && p.par) ? p.nky * p.nkx : ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW);
    const int nsrc = (MODE == MODE_FWD && p.C1 > 0) ? 2 : 1;
    constexpr int LDKp = NP == 0 ? BK + 4 : (NP * BK + 8) / 2;   // LDS row in floats of the padded layouts (halo / ring / wave-specialised kernels)
    constexpr int LDKf = (CODEPS_IGEMM_SWZ && NP > 0 && BK == 32) ? NP * BK / 2 : LDKp;      // ... of conv_igemm_kernel (unpadded + swizzled at BK = 32)
    const size_t aff_b = (MODE == MODE_FWD && p.in_aff) ? 16 + (size_t)16 * p.Ct : 0;     // in_aff: the image's four BatchNorm vectors behind the gather table
    const size_t lds = std::max(((size_t)NBUF * (BM + BN) * LDKf + (size_t)nsrc * ntap * BM) * sizeof(float) + aff_b,
                                (size_t)WM * 32 * (BN + 4) * sizeof(float));
    if constexpr (NP == 3 && WM == 2 && WN == 2 && TM == 2 && BK == 32) {
        // 3x3 / stride 1 / zero padding, one source at full resolution: halo-tile kernel (activations staged once per channel chunk)
        static const int halo3 = getenv("CODEPS_HALO3") ? atoi(getenv("CODEPS_HALO3")) : 2;          // x 128 blocks: smaller grids keep split-K / the 256-thread kernel
        if (halo3 && halo3_shape_ok<MODE>(p) &&
            ((long long)p.n_mt * p.n_nt >= halo3 * 128 || (TN == 2 && halo_splitk_slices(p, p.n_mt * p.n_nt, ((MODE == MODE_FWD) ? p.Ct : p.Co) / BK) >= 1))) {
            constexpr size_t lds_h = std::max(((size_t)204 * (LDKp + (CODEPS_HALO_SWZ ? 4 : 0)) + (size_t)2 * BN * LDKp) * sizeof(float),
                                              (size_t)WM * 32 * (BN + 4) * sizeof(float));
            static const int halo_ring = getenv("CODEPS_HALO_RING") ? atoi(getenv("CODEPS_HALO_RING")) : 1;
            if constexpr (TN == 2) {
                const int nchunks_ = ((MODE == MODE_FWD) ? p.Ct : p.Co) / BK;
                const int hks = halo_splitk_slices(p, p.n_mt * p.n_nt, nchunks_);
                if (halo_ring || hks >= 2) {
                    constexpr size_t lds_r = ((size_t)205 * (LDKp + (CODEPS_HALO_SWZ ? 4 : 0)) + (size_t)4 * BN * LDKp) * sizeof(float);
                    // CODEPS_HALO_WS=1: the producer / consumer form of the ring kernel (bit-identical results); default 0: the 256-thread form
                    const bool h16 = f16_pairs();
                    const int halo_ws = h16 ? 0 : halo_ws_on();
                    auto kr = halo_ws ? conv_halo3p_kernel<MODE, TN> : (h16 ? conv_halo3r_kernel<MODE, TN, false, 16> : conv_halo3r_kernel<MODE, TN>);
                    codeps_allow_lds((const void*)kr, 160 * 1024, halo_ws ? "conv_halo3p_kernel" : "conv_halo3r_kernel");
                    p.ksplit = 1; p.ksteps = nchunks_;
                    // grids below one block per CU (the 1/16- and 1/32-resolution layers of the pose encoder and the decoders): cut the
                    // channel chunks into K slices so that the ring kernel (one block per CU) runs whole rounds of 256 blocks
                    if (hks >= 2) { p.ksteps = cdiv(nchunks_, hks); p.ksplit = cdiv(nchunks_, p.ksteps); }
                    const bool ex = epi_plan(p, 128, !halo_ws);
                    if (ex) {
                        kr = h16 ? conv_halo3r_kernel<MODE, TN, true, 16> : conv_halo3r_kernel<MODE, TN, true>;
                        codeps_allow_lds((const void*)kr, 160 * 1024, "conv_halo3r_kernel<ex>");
                    }
                    // fp16 form: eight waves on the tile (two per SIMD) -- CODEPS_RING8=0: the four-wave form
                    static const int ring8 = getenv("CODEPS_RING8") ? atoi(getenv("CODEPS_RING8")) : 1;
                    const bool w8 = h16 && ring8;
                    if (w8) {
                        kr = ex ? conv_halo3r_kernel<MODE, 1, true, 16, 8> : conv_halo3r_kernel<MODE, 1, false, 16, 8>;
                        codeps_allow_lds((const void*)kr, 160 * 1024, "conv_halo3r_kernel<8 waves>");
                    }
                    g_last_kernel = halo_ws ? (p.ksplit > 1 ? "conv_halo3p_kernel<splitk>" : "conv_halo3p_kernel")
                                            : h16 ? (p.ksplit > 1 ? "conv_halo3r_kernel<splitk,f16x2>" : "conv_halo3r_kernel<f16x2>")
                                            : (p.ksplit > 1 ? "conv_halo3r_kernel<splitk>" : "conv_halo3r_kernel");
                    constexpr size_t lds_r16 = ((size_t)(CODEPS_RING_ADB ? 2 : 1) * 205 * ((2 * BK + 8) / 2 + 4) + (size_t)4 * BN * ((2 * BK + 8) / 2)) * sizeof(float) + 16;
                    hipLaunchKernelGGL(kr, dim3(p.n_mt * p.n_nt, p.ksplit), dim3(halo_ws ? 384 : (w8 ? 512 : 256)), h16 ? lds_r16 + 16 : lds_r, st, p, a0, a1, scale, shift, residual, out);
                    if (p.ksplit > 1) launch_splitk_finish<MODE>(p, st, scale, shift, residual, out);
                    return;
                }
            }
            p.ksplit = 1;
            const bool h16 = f16_pairs();
            const bool ex = epi_plan(p, 128);
            auto kh = h16 ? (ex ? conv_halo3_kernel<MODE, TN, 2, 2, true, 16> : conv_halo3_kernel<MODE, TN, 2, 2, false, 16>)
                          : (ex ? conv_halo3_kernel<MODE, TN, 2, 2, true> : conv_halo3_kernel<MODE, TN>);
            codeps_allow_lds((const void*)kh, 160 * 1024, "kh");
            g_last_kernel = h16 ? "conv_halo3_kernel<f16x2>" : "conv_halo3_kernel";
            constexpr size_t lds_h16 = std::max(((size_t)204 * 40 + (size_t)2 * BN * 36) * sizeof(float) + 16, (size_t)WM * 32 * (BN + 4) * sizeof(float));
            hipLaunchKernelGGL(kh, dim3(p.n_mt * p.n_nt), dim3(256), h16 ? lds_h16 : lds_h, st, p, a0, a1, scale, shift, residual, out);
            return;
        }
        static const int ws_min = getenv("CODEPS_WS_MIN") ? atoi(getenv("CODEPS_WS_MIN")) : 32;      // K-steps from which the wave-specialised kernel runs
        const int ntap_ = (MODE == MODE_DGRAD && p.par) ? p.nky * p.nkx : ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW);
        const int Kc_ = (MODE == MODE_FWD) ? p.Ct : p.Co, nsteps_ = ntap_ * (Kc_ / BK);
        // ... and whose grid is a single round of one block per CU: the block owns the CU (111 KB of LDS), so a second round
        // would run without the co-resident blocks that hide the 256-thread kernel's prologue / epilogue
        static const int ws_blocks = getenv("CODEPS_WS_BLOCKS") ? atoi(getenv("CODEPS_WS_BLOCKS")) : 256;
        if (ws_min > 0 && nsteps_ >= ws_min && p.n_mt * p.n_nt * std::max(p.grid_mult, 1) <= ws_blocks && !(MODE == MODE_FWD && p.in_aff)) {
            const int nsrc_ = (MODE == MODE_FWD && p.C1 > 0) ? 2 : 1;
            const size_t lds_ws = std::max(((size_t)2 * (BM + BN) * LDKp + (size_t)nsrc_ * ntap_ * BM) * sizeof(float), (size_t)WM * 32 * (BN + 4) * sizeof(float));
            const int blocks_ = p.n_mt * p.n_nt;
            p.ksplit = 1; p.ksteps = nsteps_;
            const int ks_ = splitk_slices(p, blocks_, nsteps_);
            if (ks_ >= 2) { p.ksteps = cdiv(nsteps_, ks_); p.ksplit = cdiv(nsteps_, p.ksteps); }
            const bool h16 = f16_pairs(), ex = epi_plan(p, BM);
            auto kw = h16 ? (ex ? conv_igemm_ws_kernel<MODE, TN, true, 16> : conv_igemm_ws_kernel<MODE, TN, false, 16>)
                          : (ex ? conv_igemm_ws_kernel<MODE, TN, true> : conv_igemm_ws_kernel<MODE, TN>);
            codeps_allow_lds((const void*)kw, 160 * 1024, "kw");
            g_last_kernel = h16 ? "conv_igemm_ws_kernel<f16x2>" : "conv_igemm_ws_kernel";
            const size_t lds_ws16 = std::max(((size_t)2 * (BM + BN) * 36 + (size_t)nsrc_ * ntap_ * BM) * sizeof(float) + 32, (size_t)WM * 32 * (BN + 4) * sizeof(float));
            hipLaunchKernelGGL(kw, dim3(blocks_, p.ksplit, p.par == 2 ? 4 : 1), dim3(512), h16 ? lds_ws16 : lds_ws, st, p, a0, a1, scale, shift, residual, out);
            if (p.ksplit > 1) launch_splitk_finish<MODE>(p, st, scale, shift, residual, out);
            return;
        }
    }
    if constexpr (NP == 3 && WM == 4 && WN == 1 && TM == 2 && TN == 1 && BK == 32) {
        // <= 32 output columns, 3x3 / stride 1 / zero padding on whole 8 x 32 tiles: the halo-tile kernel in its 4 x 1 wave form
        static const int halo32 = getenv("CODEPS_HALO32") ? atoi(getenv("CODEPS_HALO32")) : 1;      // tuning experiments only
        const int Hm_ = (MODE == MODE_FWD) ? p.Ho : p.H;
        if (halo32 && halo3_shape_ok<MODE>(p) && Hm_ % 8 == 0 && (long long)p.n_mt * p.n_nt >= 256) {
            constexpr size_t lds_h = std::max(((size_t)340 * (LDKp + (CODEPS_HALO_SWZ ? 4 : 0)) + (size_t)2 * BN * LDKp) * sizeof(float),
                                              (size_t)WM * 32 * (BN + 4) * sizeof(float));
            p.ksplit = 1;
            const bool h16 = f16_pairs();
            const bool ex = epi_plan(p, 256);
            auto kh = h16 ? (ex ? conv_halo3_kernel<MODE, 1, 4, 1, true, 16> : conv_halo3_kernel<MODE, 1, 4, 1, false, 16>)
                          : (ex ? conv_halo3_kernel<MODE, 1, 4, 1, true> : conv_halo3_kernel<MODE, 1, 4, 1>);
            codeps_allow_lds((const void*)kh, 160 * 1024, "conv_halo3_kernel<4x1>");
            g_last_kernel = h16 ? "conv_halo3_kernel<32 columns,f16x2>" : "conv_halo3_kernel<32 columns>";
            constexpr size_t lds_h16 = std::max(((size_t)340 * 40 + (size_t)2 * BN * 36) * sizeof(float) + 16, (size_t)WM * 32 * (BN + 4) * sizeof(float));
            hipLaunchKernelGGL(kh, dim3(p.n_mt * p.n_nt), dim3(256), h16 ? lds_h16 : lds_h, st, p, a0, a1, scale, shift, residual, out);
            return;
        }
    }
    auto k = conv_igemm_kernel<MODE, WM, WN, TM, TN, BK, NBUF, NP>;
    // split-K when the tile grid cannot fill the chip and K is deep (B = 1 target inference, 1/32-resolution decoder inputs)
    const int blocks = p.n_mt * p.n_nt, Kc = (MODE == MODE_FWD) ? p.Ct : p.Co, nsteps = ntap * (Kc / BK);
    p.ksplit = 1; p.ksteps = nsteps;
    const int ks = splitk_slices(p, blocks, nsteps);
    if (ks >= 2) {
        p.ksteps = cdiv(nsteps, ks);
        p.ksplit = cdiv(nsteps, p.ksteps);
    }
    // (the extras exist in the default arithmetic's instantiations -- three bf16 pieces at 32-channel K steps -- and the f32 form the <= 64-column tiles fall back to)
    constexpr bool EXOK = (NP == 3 && BK == 32 && NBUF == 1) || (NP == 0 && BK == 16 && NBUF == 2);
    bool h16 = false;
    size_t lds_k = lds;
    if constexpr (NP == 3 && BK == 32 && NBUF == 1) {
        if (f16_pairs()) {                                   // two fp16 pieces (conv_igemm_kernel<.., NP = 2>): 128-byte LDS rows + the maxima slot
            h16 = true;
            k = epi_plan(p, BM) ? conv_igemm_kernel<MODE, WM, WN, TM, TN, BK, NBUF, 2, true> : conv_igemm_kernel<MODE, WM, WN, TM, TN, BK, NBUF, 2>;
            lds_k = std::max(((size_t)(BM + BN) * 32 + (size_t)nsrc * ntap * BM) * sizeof(float) + 16 + aff_b, (size_t)WM * 32 * (BN + 4) * sizeof(float));
        }
    }
    if (!h16) {
        if constexpr (EXOK) { if (epi_plan(p, BM)) k = conv_igemm_kernel<MODE, WM, WN, TM, TN, BK, NBUF, NP, true>; }
        else epi_plan(p, BM, false);
    }
    codeps_allow_lds((const void*)k, 160 * 1024, "k");
    g_last_kernel = h16 ? "conv_igemm_kernel<f16x2>" : NP == 3 ? (BK == 16 ? "conv_igemm_kernel<split3,bk16>" : "conv_igemm_kernel<split3>") : "conv_igemm_kernel<f32>";
    hipLaunchKernelGGL(k, dim3(blocks, p.ksplit, p.par == 2 ? 4 : 1), dim3(256), lds_k, st, p, a0, a1, wq, scale, shift, residual, out);
    if (p.ksplit > 1) launch_splitk_finish<MODE>(p, st, scale, shift, residual, out);
}

// Tile choice: estimated time ~ waves of blocks over the 256 CUs x tile area x a small-tile inefficiency factor.
// Big tiles win when the grid is large; per-key / deep-layer GEMMs with few rows need smaller tiles to fill the chip.
struct TileOpt { int bm, bn; float penalty; };

static int pick_tile(const ConvP& p, const TileOpt* opts, int n, int nsteps) {
    int best = 0;
    double best_t = 1e300;
    for (int i = 0; i < n; ++i) {
        const long long blocks = (long long)cdiv(p.M, opts[i].bm) * cdiv(p.N, opts[i].bn) * std::max(p.grid_mult, 1);
        const int ks = splitk_slices(p, (int)blocks, nsteps);
        const double t = (double)((blocks * ks + 255) / 256) * opts[i].bm * opts[i].bn / ks * opts[i].penalty * (ks > 1 ? 1.08 : 1.0);
        if (t < best_t) { best_t = t; best = i; }
    }
    return best;
}

// 3 x 3 / stride 1 / zero padding layers with 16 or 32 channels on either side (not 32 x 32: the 32-column halo kernel) on whole 8 x 32
// tiles: conv_halo3n16_kernel
template <int MODE>
static bool halo3n16_ok(const ConvP& p) {
    static const int on = getenv("CODEPS_HALO_N16") ? atoi(getenv("CODEPS_HALO_N16")) : 1;                // A/B switch
    const int kc = (MODE == MODE_FWD) ? p.Ct : p.Co, Hm = (MODE == MODE_FWD) ? p.Ho : p.H, Wm = (MODE == MODE_FWD) ? p.Wo : p.W;
    return on && split_pieces() == 3 && halo3_shape_ok<MODE>(p) && !p.up0 && p.C1 == 0 && p.pitch0 == 0 && Hm % 8 == 0 && (kc == 16 || kc == 32) &&
           (p.N == 16 || p.N == 32) && !(kc == 32 && p.N == 32) && (size_t)Hm * Wm * 32 * 4 < (size_t)GATHER_OOB;
}
template <int MODE>
static void launch_halo3n16(ConvP p, const float* a0, const float* wq, const float* scale, const float* shift, const float* residual, float* out,
                            hipStream_t st) {
    const int kc = (MODE == MODE_FWD) ? p.Ct : p.Co, Hm = (MODE == MODE_FWD) ? p.Ho : p.H, Wm = (MODE == MODE_FWD) ? p.Wo : p.W;
    const int tiles_x = Wm / 32, tiles_y = Hm / 8, total = p.B * tiles_x * tiles_y;
    const int nt = p.N / 16, kh = kc / 16;
    // persistent blocks: the weights are fetched and split once per block.  Two per CU; one for the 32-channel-input form, whose 120
    // registers of weight fragments + 44 of prefetched pixels spill at 256 registers
    const bool h16 = f16_pairs();                  // (two fp16 pieces, 32 input channels: 80 registers of weight fragments, and the form with the extras still spills at 256)
    const int tpb = std::max(1, cdiv(total, kh == 2 ? 256 : 512));
    p.n_mt = total; p.n_nt = 1; p.ksplit = 1;
    // extras of this kernel: the activation gates and the column sums (the decoder tail has no BatchNorm)
    const bool ex = epi_plan(p, 256, p.ex_gate_act != 3 && (p.ex_stat == 0 || p.ex_stat == 2));
    const size_t lds_x = (size_t)kh * 340 * (h16 ? 40 : 56) * 2, lds_c = (size_t)256 * (p.N + 4) * 4 + 2 * 256 * 16;
    const size_t lds = std::max(lds_x, lds_c);
    g_last_kernel = h16 ? "conv_halo3n16_kernel<f16x2>" : "conv_halo3n16_kernel";
#define N16_LAUNCH(NT_, KH_)                                                                                                   \
    do {                                                                                                                       \
        auto k = h16 ? (ex ? conv_halo3n16_kernel<MODE, NT_, KH_, true, 16> : conv_halo3n16_kernel<MODE, NT_, KH_, false, 16>)   \
                     : (ex ? conv_halo3n16_kernel<MODE, NT_, KH_, true> : conv_halo3n16_kernel<MODE, NT_, KH_, false>);         \
        codeps_allow_lds((const void*)k, 96 * 1024, "conv_halo3n16_kernel");      /* (+ 16 bytes of static LDS) */                \
        hipLaunchKernelGGL(k, dim3(cdiv(total, tpb)), dim3(256), lds, st, p, tiles_x, tiles_y, tpb, a0, wq, scale, shift, residual, out); \
    } while (0)
    if (nt == 1 && kh == 1) N16_LAUNCH(1, 1); else if (nt == 1) N16_LAUNCH(1, 2); else N16_LAUNCH(2, 1);
#undef N16_LAUNCH
}

template <int MODE>
static void dispatch_igemm(ConvP p, int kc_gran, const float* a0, const float* a1, const float* wq, const float* scale,
                           const float* shift, const float* residual, float* out, hipStream_t st) {
    static const int force_bk = getenv("CODEPS_FORCE_BK") ? atoi(getenv("CODEPS_FORCE_BK")) : 0;   // tuning experiments only
    const bool bk32 = (kc_gran % 32) == 0 && force_bk != 16;
    if (halo3n16_ok<MODE>(p)) { launch_halo3n16<MODE>(p, a0, wq, scale, shift, residual, out, st); return; }
    if (p.N <= 16) {
        p.n_mt = cdiv(p.M, 256); p.n_nt = 1;
        p.ksplit = 1;
        const bool ex = epi_plan(p, 256);
        const int kc = (MODE == MODE_FWD) ? p.Ct : p.Co;
        g_last_kernel = kc >= 96 ? "conv_igemm16_lds_kernel" : "conv_igemm16_kernel";
        if (kc >= 96) {                        // deep K per tap (GUDA 240 channels): LDS-staged flavour
            auto k16 = bk32 ? (ex ? conv_igemm16_lds_kernel<MODE, 32, true> : conv_igemm16_lds_kernel<MODE, 32>)
                            : (ex ? conv_igemm16_lds_kernel<MODE, 16, true> : conv_igemm16_lds_kernel<MODE, 16>);
            hipLaunchKernelGGL(k16, dim3(p.n_mt), dim3(256), 0, st, p, a0, a1, wq, scale, shift, residual, out);
        } else {
            const int ntap = (MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW;
            const size_t lds = (size_t)((MODE == MODE_FWD && p.C1 > 0) ? 2 : 1) * ntap * 256 * sizeof(unsigned);
            auto k16 = bk32 ? (ex ? conv_igemm16_kernel<MODE, 32, true> : conv_igemm16_kernel<MODE, 32>)
                            : (ex ? conv_igemm16_kernel<MODE, 16, true> : conv_igemm16_kernel<MODE, 16>);
            codeps_allow_lds((const void*)k16, 120 * 1024, "conv_igemm16_kernel");
            hipLaunchKernelGGL(k16, dim3(p.n_mt), dim3(256), lds, st, p, a0, a1, wq, scale, shift, residual, out);
        }
        return;
    }
    const int nsteps32 = ((MODE == MODE_DGRAD && p.par) ? p.nky * p.nkx : ((MODE == MODE_DGRAD && p.up0 && p.src == 0) ? 4 * p.KH * p.KW : p.KH * p.KW)) *
                         (((MODE == MODE_FWD) ? p.Ct : p.Co) / (bk32 ? 32 : 16));
    // Operand arithmetic of the main kernel.  3 (default): every fp32 operand is the exact sum of three bf16 pieces (8 + 8 + 8 =
    // 24 significand bits); the six piece products of order <= 2 run on v_mfma_f32_32x32x16_bf16 with fp32 accumulation --
    // product error ~6e-9 relative, below fp32 rounding (tools/split_precision_study.py), 192 instead of 512 MFMA cycles per
    // 16-deep chunk.  0: v_mfma_f32_32x32x2_f32.  2: two pieces / three products, ~4e-6 relative: faster still but NOT inside this
    // repo's parity bar (6 network / trunk tests fail) -- experiments only.
    const int split_np = split_pieces();
    static const int nbuf_env = getenv("CODEPS_NBUF") ? atoi(getenv("CODEPS_NBUF")) : 0;          // tuning experiments only
#define IG(WM, WN, TM, TN)                                                                          \
    do {                                                                                            \
        /* single LDS buffer (next stage in registers, up to 4 blocks / CU): measured faster than the double-buffered */ \
        /* form on the whole adapt step (63.3 vs 66.2 ms of conv time), so it is the default                          */ \
        const int nbuf = nbuf_env ? nbuf_env : 1;                                                    \
        if (bk32 && nbuf == 1 && split_np == 3) launch_igemm<MODE, WM, WN, TM, TN, 32, 1, 3>(p, a0, a1, wq, scale, shift, residual, out, st); \
        else if (bk32 && nbuf == 1) launch_igemm<MODE, WM, WN, TM, TN, 32, 1>(p, a0, a1, wq, scale, shift, residual, out, st); \
        else if (bk32) launch_igemm<MODE, WM, WN, TM, TN, 32>(p, a0, a1, wq, scale, shift, residual, out, st); \
        else if (MODE == MODE_FWD && split_np == 3 && !f16_pairs() && nbuf == 1 && p.Ct == 16 && p.C1 == 0 && (p.KH * p.KW * 16) % 32 == 0)   /* stem */ \
            launch_igemm<MODE, WM, WN, TM, TN, 16, 1, 3>(p, a0, a1, wq, scale, shift, residual, out, st); \
        else      launch_igemm<MODE, WM, WN, TM, TN, 16>(p, a0, a1, wq, scale, shift, residual, out, st); \
    } while (0)
    if (p.N > 64) {
        static const float pen1 = getenv("CODEPS_PEN1") ? atof(getenv("CODEPS_PEN1")) : 1.1f, pen2 = getenv("CODEPS_PEN2") ? atof(getenv("CODEPS_PEN2")) : 1.3f;   // tuning experiments only
        // short K (< 32 K-steps, the 1x1 layers): a single round of 128x128 blocks runs its prologue / epilogue phases in lock-step
        // on every CU; twice as many 128x64 blocks desynchronise and overlap them (measured -0.5 ms per step)
        static const float pens = getenv("CODEPS_PENS") ? atof(getenv("CODEPS_PENS")) : 0.5f;
        static const int shortk = getenv("CODEPS_SHORTK") ? atoi(getenv("CODEPS_SHORTK")) : 31;       // 32-step 1x1 layers (K = 1024, N = 256): one round of 128x128 blocks on the wave-specialised kernel, 57 vs 62 us
        const TileOpt o[3] = {{128, 128, 1.0f}, {128, 64, nsteps32 <= shortk ? pens : pen1}, {64, 64, pen2}};
        // 3x3 layers whose 128 x 128 grid is below one block per CU: the halo ring kernel (215 TFLOP/s class) on >= 128 CUs, or
        // with its channel chunks cut into K slices that make whole rounds of 256 blocks, instead of the gather kernels (140-160)
        static const int halo_sk_on = getenv("CODEPS_HALO_SK") ? atoi(getenv("CODEPS_HALO_SK")) : 1;     // tuning experiments only
        const bool halo_sk = halo_sk_on && bk32 && split_np == 3 && p.N % 128 == 0 && halo3_shape_ok<MODE>(p) &&
                             halo_splitk_slices(p, cdiv(p.M, 128) * cdiv(p.N, 128), ((MODE == MODE_FWD) ? p.Ct : p.Co) / 32) >= 1;
        switch (halo_sk ? 0 : pick_tile(p, o, 3, nsteps32)) {
            case 0: IG(2, 2, 2, 2); break;
            case 1: IG(2, 2, 2, 1); break;
            default: IG(2, 2, 1, 1); break;
        }
    } else if (p.N > 32) {
        static const TileOpt o[2] = {{128, 64, 1.0f}, {64, 64, 1.2f}};
        if (pick_tile(p, o, 2, nsteps32) == 0) IG(2, 2, 2, 1); else IG(2, 2, 1, 1);
    } else {
        static const TileOpt o[2] = {{256, 32, 1.0f}, {128, 32, 1.15f}};
        if (pick_tile(p, o, 2, nsteps32) == 0) IG(4, 1, 2, 1); else IG(4, 1, 1, 1);
    }
#undef IG
}

}  // namespace

CODEPS_STAMP_SETTER(conv)


// a pack row ([tap][channel]) gets a pre-split copy when the kernel that reads it can be the split-operand one: 32-channel K
// chunks, or 16-channel chunks (the stem) as long as the row is a whole number of 32-element groups
static bool split_tail_ok(int kc, int taps) { return kc % 32 == 0 || (kc == 16 && (taps * kc) % 32 == 0); }

// table entry of one pack (slab shape, work groups); false when the shape does not fit the slab kernel
static bool fill_pack_item(PackItem& it, const float* w_oihw, float* out, int out_c, int in_c, int kh, int kw, int out_c_pad, int in_c_pad,
                           int dgrad, long long first_group) {
    if ((out_c_pad % 8) != 0 || (in_c_pad % 8) != 0 || kh * kw * 64 > PACK_SLAB) return false;
    it.w = w_oihw; it.out = out; it.co_real = out_c; it.ci_real = in_c; it.taps = kh * kw; it.dgrad = dgrad ? 1 : 0;
    it.rows = dgrad ? in_c_pad : out_c_pad; it.cols = dgrad ? out_c_pad : in_c_pad;
    it.split = split_tail_ok(it.cols, it.taps) ? (f16_pairs() ? 16 : 1) : 0;
    it.first_group = first_group;
    if (!it.dgrad) {
        it.rb = 1;
        it.cbw = std::max(8, std::min(512, PACK_SLAB / it.taps / 8 * 8));
        it.groups = (long long)it.rows * cdiv(it.cols, it.cbw);
    } else {
        it.cbw = 64;
        it.rb = std::max(1, std::min(8, PACK_SLAB / (64 * it.taps)));
        it.groups = (long long)cdiv(it.rows, it.rb) * cdiv(it.cols, it.cbw);
    }
    return true;
}

extern "C" int codeps_conv2d_pack_weights(int out_c, int in_c, int kh, int kw, int out_c_pad, int in_c_pad,
                                          const float* w_oihw, float* w_fwd, float* w_dgrad, codeps_stream_t stream) {
    CODEPS_REQUIRE(out_c > 0 && in_c > 0 && kh > 0 && kw > 0 && out_c_pad >= out_c && in_c_pad >= in_c && w_oihw &&
                       (w_fwd || w_dgrad),
                   CODEPS_ERR_ARG, "conv2d_pack_weights: bad arguments");
    const long long total = (long long)out_c_pad * in_c_pad * kh * kw;
    {   // one launch through the LDS slab (coalesced both ways, pack + split copy together); odd shapes keep the kernels below
        PackItem a, b;
        memset(&a, 0, sizeof(a)); memset(&b, 0, sizeof(b));
        bool ok = true;
        long long groups = 0;
        PackItem* slot = &a;
        if (w_fwd) { ok = ok && fill_pack_item(*slot, w_oihw, w_fwd, out_c, in_c, kh, kw, out_c_pad, in_c_pad, 0, groups); groups += slot->groups; slot = &b; }
        if (w_dgrad) { ok = ok && fill_pack_item(*slot, w_oihw, w_dgrad, out_c, in_c, kh, kw, out_c_pad, in_c_pad, 1, groups); groups += slot->groups; }
        if (ok && groups > 0 && groups < (1ll << 31)) {
            const bool big_a = a.split == 16 && (long long)a.co_real * a.ci_real * a.taps > PACK_AMAX_INLINE;
            const bool big_b = b.split == 16 && (long long)b.co_real * b.ci_real * b.taps > PACK_AMAX_INLINE;
            if (big_a || big_b) hipLaunchKernelGGL(pack_amax_pair_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a, b);
            hipLaunchKernelGGL(pack_weights_pair_kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, a, b);
            CODEPS_CHECK_LAUNCH("pack_weights_pair_kernel");
            return CODEPS_OK;
        }
    }
    const int grid = (int)std::min<long long>((total + 255) / 256, 4096);
    hipLaunchKernelGGL(pack_weights_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, w_oihw, out_c, in_c, kh * kw,
                       out_c_pad, in_c_pad, w_fwd, w_dgrad);
    // pre-split copies behind the fp32 packs (rows whose K extent is a multiple of 32 channels: the 3-piece kernel's shapes)
    const int sgrid = (int)std::min<long long>((total / 8 + 255) / 256, 4096);
    if (w_fwd && split_tail_ok(in_c_pad, kh * kw))
        hipLaunchKernelGGL(split_pack_kernel, dim3(sgrid), dim3(256), 0, (hipStream_t)stream, w_fwd, total / 8, reinterpret_cast<unsigned short*>(w_fwd + total));
    if (w_dgrad && split_tail_ok(out_c_pad, kh * kw))
        hipLaunchKernelGGL(split_pack_kernel, dim3(sgrid), dim3(256), 0, (hipStream_t)stream, w_dgrad, total / 8, reinterpret_cast<unsigned short*>(w_dgrad + total));
    CODEPS_CHECK_LAUNCH("pack_weights_kernel");
    return CODEPS_OK;
}

extern "C" size_t codeps_pack_item_bytes(void) { return sizeof(PackItem); }

// Fills ONE host-side table entry (the caller copies the table to the device once and keeps it); returns the number of
// 256-thread work groups the entry needs, 0 on bad arguments.
extern "C" long long codeps_pack_item_fill(void* item, const float* w_oihw, float* out, int out_c, int in_c, int kh, int kw, int out_c_pad,
                                           int in_c_pad, int dgrad, long long first_group) {
    if (!item || !w_oihw || !out || out_c <= 0 || in_c <= 0 || kh <= 0 || kw <= 0 || out_c_pad < out_c || in_c_pad < in_c ||
        (out_c_pad % 8) != 0 || (in_c_pad % 8) != 0) {
        codeps_set_error("pack_item_fill: bad arguments");
        return 0;
    }
    PackItem it;
    memset(&it, 0, sizeof(it));
    if (!fill_pack_item(it, w_oihw, out, out_c, in_c, kh, kw, out_c_pad, in_c_pad, dgrad, first_group)) {
        codeps_set_error("pack_item_fill: %d taps exceed the slab", kh * kw);
        return 0;
    }
    memcpy(item, &it, sizeof(it));
    return it.groups;
}

extern "C" int codeps_conv2d_pack_weights_multi(const void* items_device, int n_items, long long total_groups, codeps_stream_t stream) {
    CODEPS_REQUIRE(items_device && n_items > 0 && total_groups > 0 && total_groups < (1ll << 31), CODEPS_ERR_ARG, "pack_weights_multi: bad arguments");
    // (the fp16 pieces need the tensors' largest magnitudes first; items filled under another arithmetic skip the pass)
    if (f16_pairs())
        hipLaunchKernelGGL(pack_amax_multi_kernel, dim3((unsigned)total_groups), dim3(256), 0, (hipStream_t)stream, (const PackItem*)items_device, n_items);
    hipLaunchKernelGGL(pack_weights_multi_kernel, dim3((unsigned)total_groups), dim3(256), 0, (hipStream_t)stream, (const PackItem*)items_device, n_items);
    CODEPS_CHECK_LAUNCH("pack_weights_multi_kernel");
    return CODEPS_OK;
}

// floats a w_fwd / w_dgrad buffer must hold: the fp32 pack, plus its pre-split copy (6 bytes per element) when the pack's K
// extent (in_c_pad for w_fwd, out_c_pad for w_dgrad) is a multiple of 32 channels
extern "C" size_t codeps_conv2d_packed_weight_floats(int out_c_pad, int in_c_pad, int kh, int kw, int dgrad) {
    if (out_c_pad <= 0 || in_c_pad <= 0 || kh <= 0 || kw <= 0) return 0;
    const size_t total = (size_t)out_c_pad * in_c_pad * kh * kw;
    const int kext = dgrad ? out_c_pad : in_c_pad;
    // (+ the two fp16 pieces, their scale slot and the partial maxima of the pack's work groups: see pack_off_f16 / pack_off_scale)
    return total + (split_tail_ok(kext, kh * kw) ? 3 * total + 16 : 0);
}

// Which arithmetic a launch of this shape uses: 3 / 2 = fp32 operands as 3 / 2 bf16 pieces on v_mfma_f32_32x32x16_bf16 (main
// kernel, K chunks of 32 channels), 0 = f32 MFMA (16-column kernels, 16-channel K chunks, CODEPS_SPLIT=0).  mode 0 = forward,
// 1 = data gradient w.r.t. `source`, 2 = weight gradient (3 for the halo-tile layers, else 0).  Used by bench.py to price each launch
// against the right peak.
// 3 x 3 / stride 2 weight gradient on wgrad_s2_halo_kernel: whole 4 x 16 output tiles, one source, 32-channel input chunks
struct S2Plan { bool ok; int ci_chunks, co_groups, tiles_x, tiles_y, nblk, tiles_per_block, splits; };
static S2Plan wgrad_s2_plan(const codeps_conv_desc* d) {
    S2Plan s;
    memset(&s, 0, sizeof(s));
    static const int s2_on = getenv("CODEPS_WGRAD_S2") ? atoi(getenv("CODEPS_WGRAD_S2")) : 1;                     // tuning experiments only
    s.ok = s2_on && wgrad_split_on() && d->kh == 3 && d->kw == 3 && d->stride == 2 && d->stride_w == 2 && d->pad == 1 && d->pad_w == 1 &&
           d->c1 == 0 && !d->up0 && d->pad_mode == 0 && d->pix_pitch == 0 && d->c0 >= 32 && d->c0 % 32 == 0 && d->out_c >= 48 && d->out_c % 4 == 0 &&
           d->in_h == 2 * d->out_h && d->in_w == 2 * d->out_w && d->out_h % 4 == 0 && d->out_w % 16 == 0 &&
           (size_t)d->in_h * d->in_w * std::max(d->c0, d->out_c) * 4 < ((size_t)1 << 31);
    if (!s.ok) return s;
    s.ci_chunks = d->c0 / 32; s.co_groups = cdiv(d->out_c, 64);
    s.tiles_x = d->out_w / 16; s.tiles_y = d->out_h / 4;
    const int total = d->batch * s.tiles_x * s.tiles_y;
    const int want = std::max(1, 256 / (s.ci_chunks * s.co_groups));      // one block per CU and round
    s.tiles_per_block = std::max(2, cdiv(total, want));
    s.nblk = cdiv(total, s.tiles_per_block);
    s.splits = 2 * s.nblk;                                                 // one slab per (block, output row of the sub-tiles)
    return s;
}

static int conv_arith(const codeps_conv_desc* d, int mode, int source) {
    const int split_np = split_pieces();
    static const int force_bk = getenv("CODEPS_FORCE_BK") ? atoi(getenv("CODEPS_FORCE_BK")) : 0;
    static const int nbuf_env = getenv("CODEPS_NBUF") ? atoi(getenv("CODEPS_NBUF")) : 0;
    if (split_np != 3) return 0;
    if (force_bk == 16 || (nbuf_env && nbuf_env != 1)) return 0;
    if (mode != 2 && split_np == 3) {
        // conv_halo3n16_kernel's shapes (halo3n16_ok on the descriptor; the same for the forward and the data gradient: stride 1, pad 1)
        static const int n16_on = getenv("CODEPS_HALO_N16") ? atoi(getenv("CODEPS_HALO_N16")) : 1;
        if (n16_on && d->kh == 3 && d->kw == 3 && d->stride == 1 && d->stride_w == 1 && d->pad == 1 && d->pad_w == 1 && d->pad_mode == 0 && d->c1 == 0 &&
            !d->up0 && d->pix_pitch == 0 && d->out_h == d->in_h && d->out_w == d->in_w && d->in_w % 32 == 0 && d->in_h % 8 == 0 &&
            (d->c0 == 16 || d->c0 == 32) && (d->out_c == 16 || d->out_c == 32) && !(d->c0 == 32 && d->out_c == 32))
            return 3;
    }
    if (mode == 0) {
        const int gran = (d->c1 == 0) ? d->c0 : ((d->c0 % 32 == 0 && d->c1 % 32 == 0) ? 32 : 16);
        if (d->out_c > 16 && gran == 16 && d->c1 == 0 && split_np == 3 && (d->kh * d->kw * 16) % 32 == 0) return 3;     // the stem
        return (d->out_c > 16 && gran % 32 == 0) ? split_np : 0;
    }
    if (mode == 2) {
        if (split_np != 3 || !wgrad_split_on()) return 0;
        if (wgrad_s2_plan(d).ok) return 3;                                             // stride-2 halo-tile kernel
        const SmallPlan sp = wgrad_small_plan(d);
        if (!sp.ok && wgrad_1x1_plan(d).ok) return 3;                                  // 1 x 1: wgrad_1x1s_kernel
        return (sp.ok && (sp.halo64 || (sp.stem && sp.co_groups == 1))) ? 3 : 0;       // halo-tile kernel / split stem kernel
    }
    const int n = source ? d->c1 : d->c0;
    return (n > 16 && d->out_c % 32 == 0) ? split_np : 0;
}
extern "C" int codeps_conv2d_arith(const codeps_conv_desc* d, int mode, int source) {
    if (check_conv(d, "conv2d_arith") != CODEPS_OK) return -1;
    return conv_arith(d, mode, source);
}

// Split-K workspace: launches whose tile grid cannot fill the chip (M <= 12288 rows) with a deep K are cut into up to 16
// K slices that write partial sums there; 0 = this shape never splits.
extern "C" size_t codeps_conv2d_fwd_workspace_bytes(const codeps_conv_desc* d) {
    if (check_conv(d, "conv2d_fwd_workspace_bytes") != CODEPS_OK) return 0;
    const long long M = (long long)d->batch * d->out_h * d->out_w;
    const long long K = (long long)d->kh * d->kw * (d->c0 + d->c1);
    static const long long sk_m = getenv("CODEPS_SPLITK_M") ? atoll(getenv("CODEPS_SPLITK_M")) : 12288;   // env: tuning experiments only
    if (d->out_c <= 16 || M > sk_m || K < 512) return 0;
    return (size_t)16 * M * d->out_c * sizeof(float);
}

static_assert(sizeof(codeps_conv_epilogue) == 184, "codeps_conv_epilogue: layout shared with the ctypes binding (_lib.ConvEpilogue)");
// codeps_conv_epilogue -> ConvP.ex_* (the request) and back (what the launches did)
static int epi_load(ConvP& p, const codeps_conv_epilogue* e, long long rows, const char* who) {
    memset(&g_epi, 0, sizeof(g_epi));
    if (!e) return CODEPS_OK;
    CODEPS_REQUIRE(e->gate_act >= 0 && e->gate_act <= 3 && e->stat_mode >= 0 && e->stat_mode <= 3, CODEPS_ERR_ARG, "%s: bad epilogue modes", who);
    CODEPS_REQUIRE((e->gate_act != 1 && e->gate_act != 2) || e->gate, CODEPS_ERR_ARG, "%s: activation gate without its tensor", who);
    CODEPS_REQUIRE(e->gate_act != 3 || (e->bn_x && e->bn_mean && e->bn_invstd && e->bn_groups >= 1 && e->bn_groups <= 8 &&
                                        (!e->bn_relu || e->gate || (e->bn_gamma && e->bn_beta))), CODEPS_ERR_ARG, "%s: BatchNorm gate: missing tensors / 1..8 groups", who);
    CODEPS_REQUIRE(e->stat_mode != 3 || e->gate_act == 3, CODEPS_ERR_ARG, "%s: statistics mode 3 belongs to the BatchNorm gate", who);
    const int srows = e->stat_mode == 1 ? 3 : (e->stat_mode == 2 ? 1 : 2);
    CODEPS_REQUIRE(!e->stat_mode || (e->stat_part && e->stat_part_bytes >= (size_t)(rows / 64 + 16) * srows * p.N * sizeof(float)),
                   CODEPS_ERR_WORKSPACE, "%s: statistics buffer too small (codeps_conv2d_epilogue_part_bytes)", who);
    p.ex_gate = e->gate; p.ex_gate_act = e->gate_act; p.ex_stat = e->stat_mode; p.ex_part = e->stat_part;
    p.ex_bn_x = e->bn_x; p.ex_bn_mean = e->bn_mean; p.ex_bn_invstd = e->bn_invstd; p.ex_bn_gamma = e->bn_gamma; p.ex_bn_beta = e->bn_beta;
    p.ex_bn_relu = e->bn_relu; p.ex_bn_ng = e->bn_groups;
    for (int i = 0; i < 8; ++i) p.ex_bn_b0[i] = i < e->bn_groups ? e->bn_group_b0[i] : 0;
    return CODEPS_OK;
}
static void epi_store(codeps_conv_epilogue* e) {
    if (!e) return;
    e->applied = g_epi.applied; e->n_seg = g_epi.n_seg;
    for (int i = 0; i < 4; ++i) {
        e->seg_tile0[i] = g_epi.tile0[i]; e->seg_tiles_per_image[i] = g_epi.tpi[i]; e->seg_tile_rows[i] = g_epi.rows[i]; e->seg_tiles[i] = g_epi.tiles[i];
    }
}

extern "C" size_t codeps_conv2d_epilogue_part_bytes(long long gemm_rows, int cols, int stat_mode) {
    const int srows = stat_mode == 1 ? 3 : (stat_mode == 2 ? 1 : 2);
    return (size_t)(gemm_rows / 64 + 16) * srows * cols * sizeof(float);
}

extern "C" int codeps_conv2d_fwd(const codeps_conv_desc* d, const float* x0, const float* x1, const float* w_fwd,
                                 const float* scale, const float* shift, const float* residual, float* y, void* workspace,
                                 size_t workspace_bytes, codeps_stream_t stream) {
    return codeps_conv2d_fwd_ex(d, x0, x1, w_fwd, scale, shift, residual, y, workspace, workspace_bytes, nullptr, stream);
}

// Shapes whose forward (which = 0) / weight gradient (which = 1) can take source 0 as the INPUT of a train-mode BatchNorm + ReLU and
// normalise it on the operand load: 1x1 / stride 1 / no padding, one dense source, > 16 output columns, M tiles inside one image.
extern "C" int codeps_conv2d_in_affine_ok(const codeps_conv_desc* d, int which) {
    if (check_conv(d, "conv2d_in_affine_ok") != CODEPS_OK) return 0;
    const int hw = d->out_h * d->out_w;
    if (d->kh != 1 || d->kw != 1 || d->stride != 1 || d->stride_w != 1 || d->pad != 0 || d->pad_w != 0 || d->c1 != 0 || d->up0 || d->pix_pitch != 0 ||
        d->pad_mode != 0 || d->c0 % 16 != 0 || d->c0 > 2048)
        return 0;
    if (which == 0) return d->out_c > 16 && hw % 256 == 0;
    const SmallPlan sp = wgrad_small_plan(d);
    if (sp.ok) return !sp.stem && !sp.halo64;                     // wgrad_small_kernel's 1x1 form (<= 32 output channels)
    const W1Plan w1 = wgrad_1x1_plan(d);
    return !wgrad_s2_plan(d).ok && w1.ok && hw % 32 == 0 && w1.pps % 32 == 0;
}

static int conv_fwd_impl(const codeps_conv_desc* d, const float* x0, const float* x1, const float* in_aff, const float* w_fwd,
                         const float* scale, const float* shift, const float* residual, float* y, void* workspace,
                         size_t workspace_bytes, codeps_conv_epilogue* epilogue, codeps_stream_t stream);

extern "C" int codeps_conv2d_fwd_ex(const codeps_conv_desc* d, const float* x0, const float* x1, const float* w_fwd,
                                    const float* scale, const float* shift, const float* residual, float* y, void* workspace,
                                    size_t workspace_bytes, codeps_conv_epilogue* epilogue, codeps_stream_t stream) {
    return conv_fwd_impl(d, x0, x1, nullptr, w_fwd, scale, shift, residual, y, workspace, workspace_bytes, epilogue, stream);
}

// codeps_conv2d_fwd_ex over relu(BatchNorm(x0)) without that tensor: x0 = the BatchNorm's input, in_affine [batch][mean | invstd | gamma |
// beta][c0] (codeps_bn_in_affine) -- shapes of codeps_conv2d_in_affine_ok(d, 0) only
extern "C" int codeps_conv2d_fwd_in(const codeps_conv_desc* d, const float* x0, const float* in_affine, const float* w_fwd,
                                    const float* scale, const float* shift, const float* residual, float* y, void* workspace,
                                    size_t workspace_bytes, codeps_conv_epilogue* epilogue, codeps_stream_t stream) {
    CODEPS_REQUIRE(in_affine && codeps_conv2d_in_affine_ok(d, 0), CODEPS_ERR_ARG, "conv2d_fwd_in: shape not served (codeps_conv2d_in_affine_ok)");
    return conv_fwd_impl(d, x0, nullptr, in_affine, w_fwd, scale, shift, residual, y, workspace, workspace_bytes, epilogue, stream);
}

static int conv_fwd_impl(const codeps_conv_desc* d, const float* x0, const float* x1, const float* in_aff, const float* w_fwd,
                         const float* scale, const float* shift, const float* residual, float* y, void* workspace,
                         size_t workspace_bytes, codeps_conv_epilogue* epilogue, codeps_stream_t stream) {
    int rc = check_conv(d, "conv2d_fwd");
    if (rc != CODEPS_OK) return rc;
    CODEPS_REQUIRE(x0 && w_fwd && y && (d->c1 == 0 || x1), CODEPS_ERR_ARG, "conv2d_fwd: null pointer");
    ConvP p = make_convp(d);
    p.in_aff = in_aff;
    p.M = d->batch * d->out_h * d->out_w; p.N = d->out_c;
    rc = epi_load(p, epilogue, p.M, "conv2d_fwd");
    if (rc != CODEPS_OK) return rc;
    p.ex_img_rows = d->out_h * d->out_w;
    if (workspace && codeps_conv2d_fwd_workspace_bytes(d) > 0) { p.part = (float*)workspace; p.part_bytes = workspace_bytes; }
    p.w3 = w_fwd + (size_t)d->out_c * d->kh * d->kw * (d->c0 + d->c1);         // behind the fp32 pack (codeps_conv2d_packed_weight_floats)
    {
        const long long total = (long long)d->out_c * d->kh * d->kw * (d->c0 + d->c1);
        p.w2 = w_fwd + pack_off_f16(total); p.w2s = w_fwd + pack_off_scale(total);
    }
    const int gran = (d->c1 == 0) ? d->c0 : ((d->c0 % 32 == 0 && d->c1 % 32 == 0) ? 32 : 16);
    static const int stem_halo = getenv("CODEPS_STEM_HALO") ? atoi(getenv("CODEPS_STEM_HALO")) : 1;                  // tuning experiments only
    if (stem_halo && d->kh == 7 && d->kw == 4 && d->stride == 2 && d->stride_w == 1 && d->pad == 3 && d->pad_w == 0 && d->c0 == 16 && d->c1 == 0 &&
        !d->up0 && d->out_c == 64 && d->pix_pitch == 0 && d->pad_mode == 0 && !residual && split_pieces() == 3 && d->out_h % 8 == 0 &&
        d->out_w % 32 == 0 && d->in_h == 2 * d->out_h && d->in_w >= d->out_w + 3 && (size_t)d->in_h * d->in_w * 64 < ((size_t)1 << 31)) {
        // the double-pixel stem (functional.stem_conv2d) on whole 8 x 32 tiles: the halo-tile kernel
        const int tiles_x = d->out_w / 32, tiles_y = d->out_h / 8, total = d->batch * tiles_x * tiles_y;
        const int tpb = std::max(1, cdiv(total, 256 * std::max(1, total / (256 * 12))));     // one block per CU and round, <= ~12 tiles each
        const bool h16 = f16_pairs();
        const size_t lds = ((size_t)21 * 35 * (h16 ? 40 : 56) + 2 * 64 * (h16 ? 136 : 200)) * 2 + (64 + 8 * 2 * 64) * sizeof(float);
        g_last_kernel = h16 ? "conv_stem74f_kernel<f16x2>" : "conv_stem74f_kernel";
        auto ks = h16 ? conv_stem74f_kernel<16> : conv_stem74f_kernel<3>;
        codeps_allow_lds((const void*)ks, 128 * 1024, "conv_stem74f_kernel");         // (+ 32 bytes of static LDS)
        // epilogue extras of this kernel: the forward statistics only (its 8 x 32 tiles lie inside one image by construction)
        const bool stem_stats = p.ex_stat == 1 && !p.ex_gate_act && !scale && !shift && d->act == 0;
        p.ex_gate = nullptr; p.ex_gate_act = 0;
        if (!stem_stats) p.ex_stat = 0;
        hipLaunchKernelGGL(ks, dim3(cdiv(total, tpb)), dim3(512), lds, (hipStream_t)stream, p, tiles_x, tiles_y, tpb, x0, scale, shift, y);
        CODEPS_CHECK_LAUNCH("conv_stem74f_kernel");
        if (stem_stats) {
            g_epi.applied = 2; g_epi.n_seg = 1;
            g_epi.tile0[0] = 0; g_epi.tpi[0] = tiles_x * tiles_y; g_epi.rows[0] = 256; g_epi.tiles[0] = total;
        }
        epi_store(epilogue);
        return CODEPS_OK;
    }
    dispatch_igemm<MODE_FWD>(p, gran, x0, x1, w_fwd, scale, shift, residual, y, (hipStream_t)stream);
    CODEPS_CHECK_LAUNCH("conv_igemm_kernel<fwd>");
    epi_store(epilogue);
    return CODEPS_OK;
}

// Split-K workspace of the data gradient (same rule as the forward's: small-M launches with a deep K); 0 = never splits.
extern "C" size_t codeps_conv2d_dgrad_workspace_bytes(const codeps_conv_desc* d, int source) {
    if (check_conv(d, "conv2d_dgrad_workspace_bytes") != CODEPS_OK) return 0;
    const bool up = d->up0 && source == 0;
    const long long M = (long long)d->batch * (up ? (d->in_h / 2) * (d->in_w / 2) : d->in_h * d->in_w);
    const long long K = (long long)d->kh * d->kw * d->out_c;
    const int n = source ? d->c1 : d->c0;
    static const long long sk_m = getenv("CODEPS_SPLITK_M") ? atoll(getenv("CODEPS_SPLITK_M")) : 12288;
    if (n <= 16 || M > sk_m || K < 512 || d->stride != 1) return 0;
    return (size_t)16 * M * n * sizeof(float);
}

extern "C" int codeps_conv2d_dgrad(const codeps_conv_desc* d, int source, const float* dz, const float* w_dgrad, float* dx,
                                   void* workspace, size_t workspace_bytes, codeps_stream_t stream) {
    return codeps_conv2d_dgrad_add(d, source, dz, w_dgrad, nullptr, dx, workspace, workspace_bytes, stream);
}

extern "C" int codeps_conv2d_dgrad_add(const codeps_conv_desc* d, int source, const float* dz, const float* w_dgrad, const float* add,
                                       float* dx, void* workspace, size_t workspace_bytes, codeps_stream_t stream) {
    return codeps_conv2d_dgrad_ex(d, source, dz, w_dgrad, add, dx, workspace, workspace_bytes, nullptr, stream);
}

extern "C" int codeps_conv2d_dgrad_ex(const codeps_conv_desc* d, int source, const float* dz, const float* w_dgrad, const float* add,
                                      float* dx, void* workspace, size_t workspace_bytes, codeps_conv_epilogue* epilogue,
                                      codeps_stream_t stream) {
    int rc = check_conv(d, "conv2d_dgrad");
    if (rc != CODEPS_OK) return rc;
    CODEPS_REQUIRE(dz && w_dgrad && dx && (source == 0 || (source == 1 && d->c1 > 0)), CODEPS_ERR_ARG, "conv2d_dgrad: bad arguments");
    CODEPS_REQUIRE(d->pad_mode == 0, CODEPS_ERR_ARG, "conv2d_dgrad: reflect padding has no dgrad path here");
    CODEPS_REQUIRE(d->pix_pitch == 0, CODEPS_ERR_ARG, "conv2d_dgrad: the overlapping-pixel form is forward only");
    CODEPS_REQUIRE(d->stride_w == d->stride && d->pad_w == d->pad, CODEPS_ERR_ARG, "conv2d_dgrad: per-dimension stride / padding has no dgrad path");
    CODEPS_REQUIRE((d->out_c % 16) == 0, CODEPS_ERR_ARG, "conv2d_dgrad: out_c %d must be a multiple of 16", d->out_c);
    ConvP p = make_convp(d);
    p.src = source;
    p.Cs = source ? d->c1 : d->c0;
    p.c_off = source ? d->c0 : 0;
    const bool up = d->up0 && source == 0;
    p.M = d->batch * (up ? (d->in_h / 2) * (d->in_w / 2) : d->in_h * d->in_w);
    p.N = p.Cs;
    rc = epi_load(p, epilogue, p.M, "conv2d_dgrad");
    if (rc != CODEPS_OK) return rc;
    p.ex_img_rows = up ? (d->in_h / 2) * (d->in_w / 2) : d->in_h * d->in_w;
    if (workspace && codeps_conv2d_dgrad_workspace_bytes(d, source) > 0) { p.part = (float*)workspace; p.part_bytes = workspace_bytes; }
    // weights of this source: rows [c_off, c_off + Cs) of the [ci][tap][co] pack
    const float* wsrc = w_dgrad + (size_t)p.c_off * d->kh * d->kw * d->out_c;
    p.w3 = reinterpret_cast<const char*>(w_dgrad + (size_t)(d->c0 + d->c1) * d->kh * d->kw * d->out_c) + (size_t)p.c_off * d->kh * d->kw * d->out_c * 6;
    {
        const long long total = (long long)(d->c0 + d->c1) * d->kh * d->kw * d->out_c;
        p.w2 = reinterpret_cast<const char*>(w_dgrad + pack_off_f16(total)) + (size_t)p.c_off * d->kh * d->kw * d->out_c * 4;
        p.w2s = w_dgrad + pack_off_scale(total);
    }
    if (d->stride == 2 && p.N > 16) {
        // one launch per input-parity class with only the taps that can reach it; classes without taps are zero
        bool need_zero = false;
        for (int c = 0; c < 4; ++c) {
            const int py = c >> 1, px = c & 1;
            const int ky0 = (py + d->pad) & 1, kx0 = (px + d->pad) & 1;
            if (ky0 >= d->kh || kx0 >= d->kw) need_zero = true;
        }
        // epilogue extras over the four class launches: all or nothing -- even sizes only (every class then has the same rows and the
        // same tile plan), and no class without taps (its pixels are a copy, not an epilogue)
        if (need_zero || (d->in_h & 1) || (d->in_w & 1)) { p.ex_gate = nullptr; p.ex_gate_act = 0; p.ex_stat = 0; }
        if (need_zero) {                                        // classes no tap reaches: zero, or the incoming gradient alone
            hipError_t e = add ? hipMemcpyAsync(dx, add, (size_t)p.M * p.N * sizeof(float), hipMemcpyDeviceToDevice, (hipStream_t)stream)
                               : hipMemsetAsync(dx, 0, (size_t)p.M * p.N * sizeof(float), (hipStream_t)stream);
            CODEPS_REQUIRE(e == hipSuccess, CODEPS_ERR_LAUNCH, "conv2d_dgrad: memset / copy failed: %s", hipGetErrorString(e));
        }
        static const int par_merge = getenv("CODEPS_PARITY_MERGE") ? atoi(getenv("CODEPS_PARITY_MERGE")) : 1;         // A/B: 0 = one launch per class
        if (par_merge && !need_zero && !(d->in_h & 1) && !(d->in_w & 1) && p.N > 16) {
            // every class has taps and the same rows: ONE launch, blockIdx.z = class (the K loop of a block walks its class's 1-4 taps)
            ConvP q = p;
            q.par = 2; q.grid_mult = 4;
            q.Hc = d->in_h / 2; q.Wc = d->in_w / 2;
            q.M = d->batch * q.Hc * q.Wc;
            q.ex_img_rows = q.Hc * q.Wc;
            q.nky = q.nkx = 0;
            for (int c = 0; c < 4; ++c) {
                const int py = c >> 1, px = c & 1, ky0 = (py + d->pad) & 1, kx0 = (px + d->pad) & 1;
                const int nky = (d->kh - ky0 + 1) / 2, nkx = (d->kw - kx0 + 1) / 2;
                q.pcls[c][0] = py; q.pcls[c][1] = px; q.pcls[c][2] = ky0; q.pcls[c][3] = kx0; q.pcls[c][4] = nky; q.pcls[c][5] = nkx;
                q.nky = std::max(q.nky, nky); q.nkx = std::max(q.nkx, nkx);          // (the host sizes the gather table for the largest class)
            }
            q.py = q.px = 0; q.ky0 = q.pcls[0][2]; q.kx0 = q.pcls[0][3];
            dispatch_igemm<MODE_DGRAD>(q, d->out_c, dz, nullptr, wsrc, nullptr, nullptr, add, dx, (hipStream_t)stream);
            CODEPS_CHECK_LAUNCH("conv_igemm_kernel<dgrad, parity classes in one launch>");
            epi_store(epilogue);
            return CODEPS_OK;
        }
        // one launch per class (the A/B switch, odd sizes, classes without taps): the classes differ in K (1 to 4 taps) and may get different
        // tile / K-slice plans, so the extras' all-or-nothing rule could not be kept across them -- they are dropped (the caller runs the passes)
        p.ex_gate = nullptr; p.ex_gate_act = 0; p.ex_stat = 0;
        int tile0 = 0;
        for (int c = 0; c < 4; ++c) {
            ConvP q = p;
            q.par = 1; q.py = c >> 1; q.px = c & 1;
            q.ky0 = (q.py + d->pad) & 1; q.kx0 = (q.px + d->pad) & 1;
            if (q.ky0 >= d->kh || q.kx0 >= d->kw) continue;
            q.nky = (d->kh - q.ky0 + 1) / 2; q.nkx = (d->kw - q.kx0 + 1) / 2;
            q.Hc = (d->in_h - q.py + 1) / 2; q.Wc = (d->in_w - q.px + 1) / 2;
            if (q.Hc <= 0 || q.Wc <= 0) continue;
            q.M = d->batch * q.Hc * q.Wc;
            q.ex_img_rows = q.Hc * q.Wc;
            q.ex_tile0 = tile0;
            const int seg_before = g_epi.n_seg;
            dispatch_igemm<MODE_DGRAD>(q, d->out_c, dz, nullptr, wsrc, nullptr, nullptr, add, dx, (hipStream_t)stream);
            if (g_epi.n_seg > seg_before) tile0 += g_epi.tiles[seg_before];        // the classes' tiles follow one another without gaps
        }
        CODEPS_CHECK_LAUNCH("conv_igemm_kernel<dgrad, parity classes>");
        epi_store(epilogue);
        return CODEPS_OK;
    }
    dispatch_igemm<MODE_DGRAD>(p, d->out_c, dz, nullptr, wsrc, nullptr, nullptr, add, dx, (hipStream_t)stream);
    CODEPS_CHECK_LAUNCH("conv_igemm_kernel<dgrad>");
    epi_store(epilogue);
    return CODEPS_OK;
}

static void wgrad_plan(const codeps_conv_desc* d, int& bm, int& bn, int& n_mt, int& n_nt, int& splits, int& pps) {
    const int Ct = d->c0 + d->c1;
    bm = d->out_c > 64 ? 128 : (d->out_c > 32 ? 64 : 32);
    bn = Ct > 64 ? 128 : (Ct > 32 ? 64 : 32);
    n_mt = cdiv(d->out_c, bm); n_nt = cdiv(Ct, bn);
    const long long tiles = (long long)n_mt * n_nt * d->kh * d->kw;
    const int P = d->batch * d->out_h * d->out_w;
    static const int wg_blocks = getenv("CODEPS_WG_BLOCKS") ? atoi(getenv("CODEPS_WG_BLOCKS")) : 256 * 6;   // tuning experiments only
    long long s = std::max<long long>(1, wg_blocks / tiles);
    s = std::min<long long>(s, std::max(1, P / 256));
    s = std::min<long long>(s, 512);
    pps = (int)align_up((size_t)cdiv(P, (int)s), 16);
    splits = cdiv(P, pps);
}

extern "C" size_t codeps_conv2d_wgrad_workspace_bytes(const codeps_conv_desc* d) {
    if (check_conv(d, "conv2d_wgrad_workspace_bytes") != CODEPS_OK) return 0;
    const S2Plan s2 = wgrad_s2_plan(d);
    if (s2.ok) return (size_t)s2.splits * d->out_c * d->c0 * 9 * sizeof(float);
    const SmallPlan sp = wgrad_small_plan(d);
    if (sp.ok) return (size_t)sp.splits * d->out_c * (d->c0 + d->c1) * d->kh * d->kw * sizeof(float);
    const W1Plan w1 = wgrad_1x1_plan(d);
    if (w1.ok) return (size_t)w1.splits * d->out_c * d->c0 * sizeof(float);
    int bm, bn, n_mt, n_nt, splits, pps;
    wgrad_plan(d, bm, bn, n_mt, n_nt, splits, pps);
    return (size_t)splits * d->out_c * (d->c0 + d->c1) * d->kh * d->kw * sizeof(float);
}

extern "C" const char* codeps_conv2d_last_kernel(void) { return g_last_kernel; }
extern "C" const char* codeps_conv2d_last_finish_kernel(void) { return g_last_finish; }

extern "C" int codeps_conv2d_set_halo_ws(int on) {
    const int prev = halo_ws_on();
    if (on == 0 || on == 1) g_halo_ws = on;
    return prev;
}

extern "C" int codeps_conv2d_set_arith(int pieces) {
    const int prev = split_raw();
    if (pieces == 0 || pieces == 3 || pieces == 16) g_split_np = pieces;
    return prev;
}

static int conv_wgrad_impl(const codeps_conv_desc* d, const float* x0, const float* x1, const float* in_aff, const float* dz, float* dw_oihw,
                           int out_c_real, int in_c_real, int accumulate, void* workspace, size_t workspace_bytes, codeps_stream_t stream);

extern "C" int codeps_conv2d_wgrad(const codeps_conv_desc* d, const float* x0, const float* x1, const float* dz, float* dw_oihw,
                                   int out_c_real, int in_c_real, int accumulate, void* workspace, size_t workspace_bytes,
                                   codeps_stream_t stream) {
    return conv_wgrad_impl(d, x0, x1, nullptr, dz, dw_oihw, out_c_real, in_c_real, accumulate, workspace, workspace_bytes, stream);
}

// codeps_conv2d_wgrad over relu(BatchNorm(x0)) without that tensor (see codeps_conv2d_fwd_in) -- shapes of codeps_conv2d_in_affine_ok(d, 1) only
extern "C" int codeps_conv2d_wgrad_in(const codeps_conv_desc* d, const float* x0, const float* in_affine, const float* dz, float* dw_oihw,
                                      int out_c_real, int in_c_real, int accumulate, void* workspace, size_t workspace_bytes,
                                      codeps_stream_t stream) {
    CODEPS_REQUIRE(in_affine && codeps_conv2d_in_affine_ok(d, 1), CODEPS_ERR_ARG, "conv2d_wgrad_in: shape not served (codeps_conv2d_in_affine_ok)");
    return conv_wgrad_impl(d, x0, nullptr, in_affine, dz, dw_oihw, out_c_real, in_c_real, accumulate, workspace, workspace_bytes, stream);
}

static int conv_wgrad_impl(const codeps_conv_desc* d, const float* x0, const float* x1, const float* in_aff, const float* dz, float* dw_oihw,
                           int out_c_real, int in_c_real, int accumulate, void* workspace, size_t workspace_bytes, codeps_stream_t stream) {
    int rc = check_conv(d, "conv2d_wgrad");
    if (rc != CODEPS_OK) return rc;
    CODEPS_REQUIRE(x0 && dz && dw_oihw && workspace && (d->c1 == 0 || x1), CODEPS_ERR_ARG, "conv2d_wgrad: null pointer");
    CODEPS_REQUIRE(out_c_real > 0 && out_c_real <= d->out_c && in_c_real > 0 && in_c_real <= d->c0 + d->c1, CODEPS_ERR_ARG,
                   "conv2d_wgrad: real channel counts exceed the padded ones");
    CODEPS_REQUIRE((d->out_c % 4) == 0, CODEPS_ERR_ARG, "conv2d_wgrad: out_c %d must be a multiple of 4", d->out_c);
    CODEPS_REQUIRE(d->pix_pitch == 0, CODEPS_ERR_ARG, "conv2d_wgrad: the overlapping-pixel form is forward only");
    int bm, bn, n_mt, n_nt, splits, pps;
    wgrad_plan(d, bm, bn, n_mt, n_nt, splits, pps);
    const SmallPlan sp = wgrad_small_plan(d);
    if (sp.ok) splits = sp.splits;
    const S2Plan s2 = wgrad_s2_plan(d);
    if (s2.ok) splits = s2.splits;
    const W1Plan w1 = (sp.ok || s2.ok) ? W1Plan{} : wgrad_1x1_plan(d);
    if (w1.ok) { splits = w1.splits; pps = w1.pps; }
    const size_t need = (size_t)splits * d->out_c * (d->c0 + d->c1) * d->kh * d->kw * sizeof(float);
    CODEPS_REQUIRE(workspace_bytes >= need, CODEPS_ERR_WORKSPACE, "conv2d_wgrad: workspace %zu < %zu", workspace_bytes, need);
    WgradP p;
    memset(&p, 0, sizeof(p));
    p.B = d->batch; p.H = d->in_h; p.W = d->in_w; p.C0 = d->c0; p.C1 = d->c1; p.Ct = d->c0 + d->c1; p.up0 = d->up0;
    p.Co = d->out_c; p.Ho = d->out_h; p.Wo = d->out_w; p.KH = d->kh; p.KW = d->kw; p.stride = d->stride; p.pad = d->pad;
    p.stride_w = d->stride_w; p.pad_w = d->pad_w;
    p.pad_mode = d->pad_mode; p.n_mt = n_mt; p.n_nt = n_nt; p.splits = splits; p.pix_per_split = pps;
    p.P = d->batch * d->out_h * d->out_w;
    p.in_aff = in_aff;
    static const int wg_fast = getenv("CODEPS_WGRAD_FAST") ? atoi(getenv("CODEPS_WGRAD_FAST")) : 1;                 // tuning experiments only
    p.fast = wg_fast && d->pad_mode == 0 && d->out_h % 4 == 0 && d->out_w % 16 == 0 && (d->c0 % 4) == 0 && (d->c1 % 4) == 0 &&
             (size_t)d->in_h * d->in_w * std::max(std::max(d->c0, d->c1), d->out_c) * 4 < ((size_t)1 << 31);
    const int grid = n_mt * n_nt * d->kh * d->kw * splits;
    hipStream_t st = (hipStream_t)stream;
    float* part = (float*)workspace;
    if (s2.ok) {
        const bool h16 = f16_pairs();
        const size_t lds = h16 ? (size_t)2 * (64 * (2 * 32 + 8) + 32 * (2 * 5 * 40 + 24)) * 2 + 32 : (size_t)2 * (64 * (3 * 32 + 8) + 32 * (3 * 5 * 40 + 16)) * 2;
        g_last_kernel = h16 ? "wgrad_s2_halo_kernel<f16x2>" : "wgrad_s2_halo_kernel";
        auto k2 = h16 ? wgrad_s2_halo_kernel<16> : wgrad_s2_halo_kernel<3>;
        codeps_allow_lds((const void*)k2, 160 * 1024, "wgrad_s2_halo_kernel");
        hipLaunchKernelGGL(k2, dim3(s2.nblk * s2.ci_chunks, s2.co_groups), dim3(256), lds, st, p, s2.ci_chunks, s2.tiles_x, s2.tiles_y,
                           s2.tiles_per_block, x0, dz, part);
        CODEPS_CHECK_LAUNCH("wgrad_s2_halo_kernel");
        launch_wgrad_reduce(part, splits, d->out_c, d->c0, 9, out_c_real, in_c_real, dw_oihw, accumulate, st);
        CODEPS_CHECK_LAUNCH("wgrad_reduce_kernel");
        return CODEPS_OK;
    }
    if (sp.ok) {
        const int g = sp.nblk * sp.ci_chunks;
#define WS_LAUNCH(MT, NT, KS) hipLaunchKernelGGL((wgrad_small_kernel<MT, NT, KS, KS, 1, 1, 8, 32>), dim3(g), dim3(256), 0, st, p, sp.ci_chunks, sp.tiles_x, \
                                                 sp.tiles_y, sp.tiles_per_block, x0, x1, dz, part)
        g_last_kernel = "wgrad_small_kernel";
        if (sp.halo64) {
            g_last_kernel = wgrad_split_on() ? "wgrad_halo64s_kernel" : "wgrad_halo64_kernel";
            if (wgrad_split_on()) {
                // 4 x 16 tiles: dZs + Xs (halfwords); the double-buffered body: two 2 x 16 sub-tiles
                constexpr size_t lds_s = (size_t)64 * ((3 * 64 + 8) + (3 * 6 * 32 + 8)) * 2, lds_d = (size_t)2 * (64 * ((3 * 32 + 8) + (3 * 4 * 32 + 8))) * 2;
                constexpr size_t lds_h = (size_t)2 * (64 * ((2 * 32 + 8) + (2 * 4 * 32 + 8))) * 2 + 32;       // two fp16 pieces + the exponent slots
                const bool h16 = f16_pairs();
                const size_t lds = h16 ? std::max(lds_s, lds_h) : std::max(lds_s, lds_d);
                auto kw = sp.co32 ? (h16 ? wgrad_halo64s_kernel<true, 16> : wgrad_halo64s_kernel<true>) : (h16 ? wgrad_halo64s_kernel<false, 16> : wgrad_halo64s_kernel<false>);
                g_last_kernel = sp.co32 ? (h16 ? "wgrad_halo64s_kernel<co32,f16x2>" : "wgrad_halo64s_kernel<co32>") : (h16 ? "wgrad_halo64s_kernel<f16x2>" : "wgrad_halo64s_kernel");
                codeps_allow_lds((const void*)kw, 160 * 1024, "wgrad_halo64s_kernel");
                hipLaunchKernelGGL(kw, dim3(g, sp.co_groups), dim3(256), lds, st, p, sp.ci_chunks, sp.tiles_x, sp.tiles_y, sp.tiles_per_block, x0, x1, dz, part);
            } else
            hipLaunchKernelGGL(wgrad_halo64_kernel, dim3(g, sp.co_groups), dim3(256), 0, st, p, sp.ci_chunks, sp.tiles_x, sp.tiles_y,
                               sp.tiles_per_block, x0, x1, dz, part);
        } else if (sp.stem) {
            if (d->kw == 7)
                hipLaunchKernelGGL((wgrad_small_kernel<1, 1, 7, 7, 2, 2, 4, 16>), dim3(g, sp.co_groups), dim3(256), 0, st, p, sp.ci_chunks,
                                   sp.tiles_x, sp.tiles_y, sp.tiles_per_block, x0, x1, dz, part);
            else if (sp.co_groups == 1) {              // ... on the bf16 matrix cores (3-piece operands)
                g_last_kernel = "wgrad_stem74s_kernel";
                static const int stem_dbuf = getenv("CODEPS_STEM_DBUF") ? atoi(getenv("CODEPS_STEM_DBUF")) : 1;        // tuning experiments only
                if (stem_dbuf && p.fast && d->pad_w == 0 && d->in_h == 2 * d->out_h) {          // whole tiles, rows padded by the range check
                    const bool h16 = f16_pairs();
                    const size_t lds = h16 ? (size_t)2 * (64 * (2 * 64 + 8) + 16 * (2 * 13 * 24 + 8)) * 2 + 32 : (size_t)2 * (64 * (3 * 64 + 8) + 16 * 3 * 13 * 24) * 2;
                    auto kst = h16 ? wgrad_stem74d_kernel<16> : wgrad_stem74d_kernel<3>;
                    if (h16) g_last_kernel = "wgrad_stem74s_kernel<f16x2>";
                    codeps_allow_lds((const void*)kst, 160 * 1024, "wgrad_stem74d_kernel");
                    hipLaunchKernelGGL(kst, dim3(g), dim3(256), lds, st, p, sp.tiles_x, sp.tiles_y, sp.tiles_per_block, x0, dz, part);
                } else
                hipLaunchKernelGGL(wgrad_stem74s_kernel, dim3(g), dim3(256), 0, st, p, sp.tiles_x, sp.tiles_y, sp.tiles_per_block, x0, dz, part);
            } else                                       // double-pixel stem: 7 x 4 taps of 16 (2 pixels x 8 channels), stride (2, 1)
                hipLaunchKernelGGL((wgrad_small_kernel<1, 1, 7, 4, 2, 1, 4, 16>), dim3(g, sp.co_groups), dim3(256), 0, st, p, sp.ci_chunks,
                                   sp.tiles_x, sp.tiles_y, sp.tiles_per_block, x0, x1, dz, part);
        } else if (d->kh == 3) {
            if (sp.mt == 1 && sp.nt == 1) WS_LAUNCH(1, 1, 3); else if (sp.mt == 1) WS_LAUNCH(1, 2, 3);
            else if (sp.nt == 1) WS_LAUNCH(2, 1, 3); else WS_LAUNCH(2, 2, 3);
        } else {
            if (sp.mt == 1 && sp.nt == 1) WS_LAUNCH(1, 1, 1); else if (sp.mt == 1) WS_LAUNCH(1, 2, 1);
            else if (sp.nt == 1) WS_LAUNCH(2, 1, 1); else WS_LAUNCH(2, 2, 1);
        }
#undef WS_LAUNCH
        CODEPS_CHECK_LAUNCH("wgrad_small_kernel");
        const long long total = (long long)d->out_c * (d->c0 + d->c1) * d->kh * d->kw;
        (void)total;
        launch_wgrad_reduce(part, splits, d->out_c, d->c0 + d->c1, d->kh * d->kw, out_c_real, in_c_real, dw_oihw, accumulate, st);
        CODEPS_CHECK_LAUNCH("wgrad_reduce_kernel");
        return CODEPS_OK;
    }
    if (w1.ok) {
        const bool h16 = f16_pairs();
        const size_t lds = (size_t)(256 + 64 * w1.tb) * ((h16 ? 2 : 3) * 32 + 8) * 2;
        g_last_kernel = h16 ? "wgrad_1x1s_kernel<f16x2>" : "wgrad_1x1s_kernel";
        auto k1 = h16 ? (w1.tb == 2 ? (w1.swap ? wgrad_1x1s_kernel<true, 2, 16> : wgrad_1x1s_kernel<false, 2, 16>)
                                    : (w1.swap ? wgrad_1x1s_kernel<true, 1, 16> : wgrad_1x1s_kernel<false, 1, 16>))
                      : (w1.tb == 2 ? (w1.swap ? wgrad_1x1s_kernel<true, 2> : wgrad_1x1s_kernel<false, 2>)
                                    : (w1.swap ? wgrad_1x1s_kernel<true, 1> : wgrad_1x1s_kernel<false, 1>));
        codeps_allow_lds((const void*)k1, 128 * 1024, "wgrad_1x1s_kernel");       // (+ 32 bytes of static LDS)
        hipLaunchKernelGGL(k1, dim3(w1.splits, w1.tiles), dim3(256), lds, st, p, x0, dz, part);
        CODEPS_CHECK_LAUNCH("wgrad_1x1s_kernel");
        launch_wgrad_reduce(part, splits, d->out_c, d->c0, 1, out_c_real, in_c_real, dw_oihw, accumulate, st);
        CODEPS_CHECK_LAUNCH("wgrad_reduce_kernel");
        return CODEPS_OK;
    }
#define WG_LAUNCH(WM, WN, TM, TN)                                                                              \
    do {                                                                                                       \
        constexpr int BM_ = 32 * WM * TM, BN_ = 32 * WN * TN, BKP_ = (4 / (WM * WN)) == 4 ? 32 : 16;           \
        const size_t lds = (size_t)2 * BKP_ * (BM_ + 4 + BN_ + 4) * sizeof(float);                             \
        hipLaunchKernelGGL((conv_wgrad_kernel<WM, WN, TM, TN>), dim3(grid), dim3(256), lds, st, p, x0, x1, dz, part); \
    } while (0)
    g_last_kernel = "conv_wgrad_kernel";
    if (bm == 128 && bn == 128) WG_LAUNCH(2, 2, 2, 2);
    else if (bm == 128 && bn == 64) WG_LAUNCH(2, 2, 2, 1);
    else if (bm == 128 && bn == 32) WG_LAUNCH(4, 1, 1, 1);
    else if (bm == 64 && bn == 128) WG_LAUNCH(2, 2, 1, 2);
    else if (bm == 64 && bn == 64) WG_LAUNCH(2, 2, 1, 1);
    else if (bm == 64 && bn == 32) WG_LAUNCH(2, 1, 1, 1);
    else if (bm == 32 && bn == 128) WG_LAUNCH(1, 4, 1, 1);
    else if (bm == 32 && bn == 64) WG_LAUNCH(1, 2, 1, 1);
    else WG_LAUNCH(1, 1, 1, 1);
#undef WG_LAUNCH
    CODEPS_CHECK_LAUNCH("conv_wgrad_kernel");
    const long long total = (long long)d->out_c * (d->c0 + d->c1) * d->kh * d->kw;
    (void)total;
    launch_wgrad_reduce(part, splits, d->out_c, d->c0 + d->c1, d->kh * d->kw, out_c_real, in_c_real, dw_oihw, accumulate, st);
    CODEPS_CHECK_LAUNCH("wgrad_reduce_kernel");
    return CODEPS_OK;
}
