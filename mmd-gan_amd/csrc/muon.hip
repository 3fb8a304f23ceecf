// Orthogonalised updates: O = the fifth (or any) iterate of the quintic  X <- a X + b (X X^T) X + c (X X^T)^2 X  started at
// X = U / ||U||_F, which takes every singular value of U to about 1 (0.7 .. 1.2), and the parameter update that applies it
// to a momentum matrix.  (a, b, c) = (3.4445, -4.7750, 2.0315) and the method are K. Jordan's (Muon, 2024); the step's factor
// 0.2 sqrt(max(rows, cols)), which gives every matrix an Adam update's size, is J. Liu et al.'s (2025).
// Matrices are row-major [rows, cols]; m = the shorter side, n = the longer one, X is [m, n].
//
// Mathematics used.  With A = X X^T the iterate is X' = Q X, Q = a I + b A + c A^2, and the next Gram matrix is
// A' = Q A Q: all of them are polynomials of one symmetric matrix, they commute, so up to three steps run on m x m
// matrices alone, P = Q3 Q2 Q1, before X is touched again: X <- P X, A = X X^T from the new X.  Rounding errors of A grow by Q^2
// (12 at the small end) per step on directions with tiny singular values; three steps between two true Gram matrices keep the
// result of four steps and more as near to the exact one as steps on X itself, five do not (six times the error on ill-conditioned U).  Work for five
// steps: two Gram matrices (m^2 n each, one triangle) and two products with X (2 m^2 n each) instead of five of both.
//
// Numerics.  Every m x n and m x m operand is held as TWO fp16 numbers, v * s = hi + lo with s a fixed power of two that keeps
// the largest possible entry (the norms are bounded: singular values <= 1.21, |Q| <= 3.45, |P| <= 41) below 65504: 22 bits, and
// 2^-25 / s absolute where lo underflows.  Products are hi hi + hi lo + lo hi in fp32 accumulators (lo lo is 2^-22 of the
// result): operands of 22 bits where fp32's have 24, at 16/3 of the fp32 matrix rate.  What comes out is about as near to 64 bits as fp32
// products on X: 4608x512 3.3e-6 against 5.7e-6, 129x1001 5.2e-6 and 5.5e-6; an update may be a tenth further off at other sizes.
//
// Layout ("packed"): an [R, K] operand is cut into 32 x 16 blocks, row blocks outermost; a block is 2 KB: the 64 lanes' 16-byte
// MFMA operands of the hi parts in lane order (lane = row % 32 + 32 * (k / 8 % 2), 8 halves along k), then those of the lo parts.
// Every operand load of a wave is one contiguous kilobyte, from L2 or from LDS, without bank conflicts or swizzles.  All sides are
// padded to 128 with zeros, so the products have no edges.  (Matrices with a side of 64 or less: muon_small.hip.)  Row blocks lie
// 4 KB further apart than their blocks fill: with m a power of two all workgroups of a product, at the same reduction step, would
// otherwise read addresses that are equal modulo 128 KB, from the same few memory channels.
//
// Measured (five steps; 21 launches): 4608x512 alone 147 us - thirteen m x m products of 5.5 us, latency, not work (24 us at the rate of
// a large fp16 product); the 64x64 images' discriminator (24 M parameters) 0.92 to 0.98 ms over several boxes: momentum and norm 92 us and
// the split 47 (HBM), two Gram matrices 91 + 20 each (0.6 of a large product's rate), thirteen m x m products of 20, two products with X
// 166 and 181 (0.67).
#include "muon_internal.h"

namespace mmdgan {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float mu_f4 __attribute__((ext_vector_type(4)));
typedef unsigned int mu_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMuPad = 128;
constexpr int kMuChain = 3;                  // steps between two true Gram matrices
// ... but three steps alone run as two and one: a chain of three is off by up to 3.3e-5 on a matrix of rank one (66x271), which the steps before
// or behind it make nothing of (five steps: 4.4e-5, on X itself 5.3e-5) and which three steps on X itself, 4.5e-6, do not have.
static int mu_chain(int done, int steps) { return steps == 3 && done == 0 ? 2 : steps - done < kMuChain ? steps - done : kMuChain; }
// X <- P X in tiles of 128 x 128; of 64 x 128 where a launch has fewer than 512 of the former (two on a CU at once): 129x1001
// alone 131 -> 119 us, 4608x512 171 -> 163 when this was taken (102 and 147 with what came later).  On a net's matrices together the
// finer tiles change nothing or cost: they read half as much again per product (64x64 images' discriminator 0.99 -> 1.00 ms).
constexpr int kMuApplyFine = 512;
constexpr float kScaleX = 4096.f, kScaleA = 4096.f, kScaleQ = 8192.f, kScaleP = 1024.f;

// halves from one row block to the next, of `kb` = K / 16 blocks
__host__ __device__ __forceinline__ size_t mu_strip(int kb) { return (size_t)kb * 1024 + 2048; }
// offset (in halves) of element (r, k)'s hi part; lo is 512 further
__device__ __forceinline__ size_t mu_off(int r, int k, int kb) {
    return (r >> 5) * mu_strip(kb) + (size_t)(k >> 4) * 1024 + ((r & 31) + ((k >> 3) & 1) * 32) * 8 + (k & 7);
}

__device__ __forceinline__ void mu_split(float v, f16 &hi, f16 &lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}
// eight values along k, the first at a multiple of 8, as one piece each of hi and lo
__device__ __forceinline__ void mu_put8(gptr<f16> o, size_t at, const float (&v)[8]) {
    f16x8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) { f16 h, l; mu_split(v[i], h, l); hi[i] = h; lo[i] = l; }
    *(gptr<f16x8>)(o + at) = hi;
    *(gptr<f16x8>)(o + at + 512) = lo;
}

// ---- the product of one tile -------------------------------------------------------------------------------------
// C[i, j] = sum_k A[i, k] B[j, k] for a tile of 64 TA x 128, four waves as 2 x 2 of 32 TA x 64.  Per 32-wide step the workgroup stages
// 2 TA row blocks of a and four of b (4 KB each, contiguous in memory) in LDS, double buffered.  a / b: the first block of the tile's
// first row block; sa / sb: halves from one row block to the next.
template <int TA> constexpr int kMuStage = (2 * TA + 4) * 4096;      // bytes of a stage
template <int TA>
__device__ __forceinline__ void mu_tile(gptr<const f16> a, size_t sa, gptr<const f16> b, size_t sb, int steps, char *lds, f32x16 (&acc)[TA][2]) {
    constexpr int STAGE = kMuStage<TA>;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    mu_u32x4 ga[2 * TA], gb[4];
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < 2 * TA) ga[i] = *(gptr<const mu_u32x4>)(a + i * sa + (size_t)s * 2048 + t * 8);
            gb[i] = *(gptr<const mu_u32x4>)(b + i * sb + (size_t)s * 2048 + t * 8);
        }
    };
    auto store = [&](char *buf) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < 2 * TA) *reinterpret_cast<mu_u32x4 *>(buf + i * 4096 + t * 16) = ga[i];
            *reinterpret_cast<mu_u32x4 *>(buf + (2 * TA + i) * 4096 + t * 16) = gb[i];
        }
    };
    f32x16 low[TA][2];                                      // hi lo + lo hi: 2^-11 of the sum, so their roundings do not count
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) { acc[i][j] = f32x16{}; low[i][j] = f32x16{}; }
    const int ar = (w >> 1) * TA * 4096 + lane * 16, br = (2 * TA + (w & 1) * 2) * 4096 + lane * 16;
    struct Frag { f16x8 ah[TA], al[TA], bh[2], bl[2]; } f0, f1;
    auto read = [&](Frag &f, const char *buf, int ks) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i < TA) {
                f.ah[i] = *reinterpret_cast<const f16x8 *>(buf + ar + i * 4096 + ks * 2048);
                f.al[i] = *reinterpret_cast<const f16x8 *>(buf + ar + i * 4096 + ks * 2048 + 1024);
            }
            f.bh[i] = *reinterpret_cast<const f16x8 *>(buf + br + i * 4096 + ks * 2048);
            f.bl[i] = *reinterpret_cast<const f16x8 *>(buf + br + i * 4096 + ks * 2048 + 1024);
        }
    };
    auto multiply = [&](const Frag &f) {                     // (an accumulator is touched every 2 TA-th product)
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[i], f.bl[j], low[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[i], f.bh[j], low[i][j], 0, 0, 0);
    };
    // Everything that a group of products needs was asked for one group earlier: operands of the second half of a stage are read from
    // LDS under the products of the first, those of the next stage's first half under the products of the second; global loads
    // run a stage and a half ahead (two and a half: 250 registers, and no faster).  The barrier publishes LDS only and leaves them
    // in flight.  No branch in the loop: past one the compiler waits for every load it has issued; the last two stages ask for
    // the last step again, and nobody reads it.
    const int last = steps - 1;
    fetch(0);
    store(lds);
    fetch(1);                                                // (steps >= 2)
    lds_barrier();
    read(f0, lds, 0);
    for (int s = 0; s < steps; ++s) {
        char *cur = lds + (s & 1) * STAGE, *nxt = lds + ((s + 1) & 1) * STAGE;
        read(f1, cur, 1);
        multiply(f0);
        store(nxt);                                          // (every wave has read the stage before last: the barrier below)
        lds_barrier();
        read(f0, nxt, 0);
        fetch(s + 2 < steps ? s + 2 : last);
        multiply(f1);
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] += low[i][j];
}
// C layout of the 32x32 MFMA: lane l, element e hold column l % 32, row 8 (e / 4) + 4 (l / 32) + e % 4
__device__ __forceinline__ int mu_row(int e) { return (e >> 2) * 8 + ((threadIdx.x & 63) >> 5) * 4 + (e & 3); }
__device__ __forceinline__ int mu_col() { return threadIdx.x & 31; }

// A wave's 64 x 64 result in 16 KB of LDS, eight-column groups of row r at group ^ (r & 7): rows are then read 16 bytes a lane by
// 32 lanes in 32 rows without bank conflicts, columns by neighbouring lanes.
__device__ __forceinline__ int mu_lds(int r, int c) { return r * 64 + (((c >> 3) ^ (r & 7)) << 3) + (c & 7); }

// lower-triangle tile number -> (ti, tj), ti >= tj
__device__ __forceinline__ void mu_tri(int t, int &ti, int &tj) {
    int r = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((r + 1) * (r + 2) / 2 <= t) ++r;
    while (r * (r + 1) / 2 > t) --r;
    ti = r;
    tj = t - r * (r + 1) / 2;
}

// Work item of a workgroup that is number b of its matrix, of n items on n rounded up to 8 workgroups: the eight XCDs take
// workgroups in turn and each has an L2 of its own - XCD x gets the x-th eighth of the matrix's items, neighbours, which share
// operands.  (An eighth of every matrix, not of the launch: the matrices' items differ in cost.)  -1: none.
__device__ __forceinline__ int mu_item(unsigned b, unsigned n) {
    const unsigned x = b & 7, per = n >> 3, rest = n & 7, i = b >> 3;
    return i < per + (x < rest ? 1u : 0u) ? (int)(x * per + (x < rest ? x : rest) + i) : -1;
}

// ---- momentum and norm -------------------------------------------------------------------------------------------
struct MuPrep {
    MuPtr<const float> grad, mom;    // mom null: U = grad
    MuPtr<float> mom_out, u;         // u: where U goes when it is neither grad nor mom_out (Nesterov), else null
    MuPtr<const float> dsigma, dot, sigma, scale;
    MuPtr<double> part;              // [blocks]
    long n;
    int vec;
    unsigned blocks;
};
struct MuPrepTable { MuFirst<kMuGroup> f; MuPrep j[kMuGroup]; float momentum, grad_scale; int nesterov; };
constexpr int kMuPrepPer = 4096;     // elements per workgroup and round
constexpr int kMuPrepMax = 1024;     // workgroups per matrix

__device__ __forceinline__ double mu_prep_one(const MuPrep &p, const MuPrepTable &t, long i, float g, float c0, float c1, float ds, float mom) {
    g *= c0;
    if (p.dsigma) g -= c1 * ds;
    float u = g;
    if (p.mom) {
        const float m = __builtin_fmaf(t.momentum, mom, g);
        p.mom_out[i] = m;
        u = t.nesterov ? __builtin_fmaf(t.momentum, m, g) : m;
        if (p.u) p.u[i] = u;
    }
    return (double)u * (double)u;
}
// U = g (+ momentum), its sum of squares by workgroup.  g = grad_scale * grad, or of a spectrally normalised kernel
// grad_scale * (scale * grad - (scale / sigma) <grad, W> dsigma/dW)  (Adam's read, elementwise.hip).  HBM-bound.
__global__ __launch_bounds__(256) void mu_prep_kernel(MuPrepTable t) {
    __shared__ double red[4];
    MuPrep p;
    unsigned start;
    mu_which(t.f, t.j, blockIdx.x, p, start);
    const unsigned nb = p.blocks, b = blockIdx.x - start;
    float c0 = t.grad_scale, c1 = 0.f;
    if (p.dsigma) { c0 = t.grad_scale * p.scale[0]; c1 = t.grad_scale * (p.scale[0] / p.sigma[0]) * p.dot[0]; }
    double ss = 0.0;
    if (p.vec) {                                             // every pointer 16-byte aligned: four float4 per tensor in flight
        const long n4 = p.n >> 2;
        constexpr int U = 4;
        for (long i0 = (long)b * 256 + threadIdx.x; i0 < n4; i0 += (long)nb * 256 * U) {
            mu_f4 g[U], d[U], m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long i = i0 + (long)u * nb * 256;
                if (i < n4) {
                    g[u] = p.grad.as<const mu_f4>()[i];
                    if (p.dsigma) d[u] = p.dsigma.as<const mu_f4>()[i];
                    if (p.mom) m[u] = p.mom.as<const mu_f4>()[i];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long i = i0 + (long)u * nb * 256;
                if (i >= n4) break;
                float gv[4] = {g[u].x, g[u].y, g[u].z, g[u].w}, mv[4] = {m[u].x, m[u].y, m[u].z, m[u].w};
                const float dv[4] = {d[u].x, d[u].y, d[u].z, d[u].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    gv[j] *= c0;
                    if (p.dsigma) gv[j] -= c1 * dv[j];
                    if (p.mom) {
                        mv[j] = __builtin_fmaf(t.momentum, mv[j], gv[j]);
                        gv[j] = t.nesterov ? __builtin_fmaf(t.momentum, mv[j], gv[j]) : mv[j];
                    }
                    ss += (double)gv[j] * (double)gv[j];
                }
                if (p.mom) {
                    p.mom_out.as<mu_f4>()[i] = mu_f4{mv[0], mv[1], mv[2], mv[3]};
                    if (p.u) p.u.as<mu_f4>()[i] = mu_f4{gv[0], gv[1], gv[2], gv[3]};
                }
            }
        }
    }
    for (long i = (p.vec ? p.n & ~3L : 0) + (long)b * 256 + threadIdx.x; i < p.n; i += (long)nb * 256)
        ss += mu_prep_one(p, t, i, p.grad[i], c0, c1, p.dsigma ? p.dsigma[i] : 0.f, p.mom ? p.mom[i] : 0.f);
    ss = wave_sum(ss);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    if (threadIdx.x == 0) p.part[b] = red[0] + red[1] + red[2] + red[3];
}

// ---- X = U / ||U|| as packed [m, n] and [n, m] --------------------------------------------------------------------
struct MuSplit {
    MuPtr<const float> u;            // [rows, cols]
    MuPtr<const double> part;
    int nparts;
    MuPtr<f16> x, xt;                     // [mp, np] and [np, mp]
    int rows, cols, mp, np, tall;    // tall: rows = n
};
struct MuSplitTable { MuFirst<kMuGroup> f; MuSplit j[kMuGroup]; };

// one 64 x 64 tile of the padded matrix; "natural" = the operand whose rows are U's rows
__global__ __launch_bounds__(256) void mu_split_kernel(MuSplitTable t) {
    __shared__ float tile[64][65];
    __shared__ double s_sum[4];
    MuSplit p;
    unsigned start;
    mu_which(t.f, t.j, blockIdx.x, p, start);
    const int b = blockIdx.x - start;
    const int prows = p.tall ? p.np : p.mp, pcols = p.tall ? p.mp : p.np;
    const int r0 = b / (pcols / 64) * 64, c0 = b % (pcols / 64) * 64;
    // everything asked for before anything is waited for: the partial sums, this thread's sixteen values (clamped, not skipped)
    const int tc = threadIdx.x & 63, tr = threadIdx.x >> 6, c = c0 + tc < p.cols ? c0 + tc : p.cols - 1;
    double d[kMuPrepMax / 256];
    float u[16];
#pragma unroll
    for (int i = 0; i < kMuPrepMax / 256; ++i) {
        const int at = threadIdx.x + 256 * i;
        d[i] = p.part[at < p.nparts ? at : 0];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + tr + 4 * i;
        u[i] = p.u[(size_t)(r < p.rows ? r : p.rows - 1) * p.cols + c];
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < kMuPrepMax / 256; ++i) ss += (int)threadIdx.x + 256 * i < p.nparts ? d[i] : 0.0;
    ss = wave_sum(ss);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = ss;
    const gptr<f16> nat = p.tall ? p.xt : p.x, tra = p.tall ? p.x : p.xt;
    __syncthreads();
    {
        const double s = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        const double inv = s > 0.0 ? (double)kScaleX / sqrt(s) : s == 0.0 ? 0.0 : s;                 // (NaN stays NaN)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            tile[tr + 4 * i][tc] = r0 + tr + 4 * i < p.rows && c0 + tc < p.cols ? (float)((double)u[i] * inv) : 0.f;
    }
    __syncthreads();
    // a lane writes 8 values along the operand's own k: lane = row % 32 + 32 * (k / 8 % 2), as the blocks are laid out
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int blk = w * 2 + i, r = (blk >> 2) * 32 + (lane & 31), k = (blk & 3) * 16 + (lane >> 5) * 8;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[r][k + e];
        mu_put8(nat, mu_off(r0 + r, c0 + k, pcols / 16), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[k + e][r];
        mu_put8(tra, mu_off(c0 + r, r0 + k, prows / 16), v);
    }
}

// ---- Gram matrix A = X X^T: one triangle of 128 x 128 tiles, the reduction over n split ----------------------------
struct MuGram {
    MuPtr<const f16> x;
    MuPtr<float> slab;               // [splits][tiles][128][128]
    MuPtr<f16> a;                    // [mp, mp]
    int mp, np, tiles, splits, steps_per;
};
struct MuGramTable { MuFirst<kMuGroup> f, r; MuGram j[kMuGroup]; };

__global__ __launch_bounds__(256, 2) void mu_gram_kernel(MuGramTable t) {
    __shared__ __attribute__((aligned(16))) char lds[2 * kMuStage<2>];
    MuGram p;
    unsigned start;
    mu_which(t.f, t.j, blockIdx.x, p, start);
    const int b = mu_item(blockIdx.x - start, p.tiles * p.splits);
    if (b < 0) return;
    const int split = b / p.tiles, tile = b % p.tiles;
    int ti, tj;
    mu_tri(tile, ti, tj);
    const int s0 = split * p.steps_per, all = p.np / 32;
    const int steps = s0 + p.steps_per < all ? p.steps_per : all - s0;
    f32x16 acc[2][2];
    const size_t sx = mu_strip(p.np / 16);
    mu_tile<2>(p.x + (size_t)ti * 4 * sx + (size_t)s0 * 2048, sx, p.x + (size_t)tj * 4 * sx + (size_t)s0 * 2048, sx, steps, lds, acc);
    const gptr<float> o = p.slab + ((size_t)split * p.tiles + tile) * 128 * 128;
    const int w = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                o[((w >> 1) * 64 + i * 32 + mu_row(e)) * 128 + (w & 1) * 64 + j * 32 + mu_col()] = acc[i][j][e];
}

// sums the splits of a 32 x 32 block in order, writes A packed, and its mirror image
__global__ __launch_bounds__(256) void mu_gram_reduce_kernel(MuGramTable t) {
    __shared__ float blk[32][33];
    MuGram p;
    unsigned start;
    mu_which(t.r, t.j, blockIdx.x, p, start);
    const int b = blockIdx.x - start, tile = b >> 4, sub = b & 15;
    int ti, tj;
    mu_tri(tile, ti, tj);
    const int r0 = (sub >> 2) * 32, c0 = (sub & 3) * 32, tc = (threadIdx.x & 7) * 4, tr = threadIdx.x >> 3;
    const double k = (double)kScaleA / ((double)kScaleX * kScaleX);
    const gptr<const float> s = p.slab + (size_t)tile * 128 * 128 + (r0 + tr) * 128 + c0 + tc;
    const size_t next = (size_t)p.tiles * 128 * 128;
    double v[4] = {0.0, 0.0, 0.0, 0.0};                      // (the splits' own sums are short: the long one is formed here)
    for (int z0 = 0; z0 < p.splits; z0 += 8) {
        mu_f4 f[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) f[z] = *(gptr<const mu_f4>)(s + (size_t)(z0 + z < p.splits ? z0 + z : z0) * next);
#pragma unroll
        for (int z = 0; z < 8; ++z)
            if (z0 + z < p.splits) { v[0] += f[z].x; v[1] += f[z].y; v[2] += f[z].z; v[3] += f[z].w; }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) blk[tr][tc + e] = (float)(v[e] * k);
    __syncthreads();
    // waves 0, 1: the block's two 16-column halves; waves 2, 3: its mirror image (a tile on the diagonal holds both halves)
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 31, kk = (w & 1) * 16 + (lane >> 5) * 8, R = ti * 128 + r0, K = tj * 128 + c0;
    float o[8];
    if (w < 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = blk[r][kk + e];
        mu_put8(p.a, mu_off(R + r, K + kk, p.mp / 16), o);
    } else if (ti != tj) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = blk[kk + e][r];
        mu_put8(p.a, mu_off(K + r, R + kk, p.mp / 16), o);
    }
}

// ---- m x m products of commuting symmetric matrices: one triangle of tiles --------------------------------
struct MuSquare {
    MuPtr<const f16> a, b;           // o = alpha a b  (packed, symmetric, [mp, mp])
    MuPtr<f16> o;
    MuPtr<const f16> z;              // polynomial form: o += zscale * z + diag on the diagonal; null: the plain product
    float alpha, zscale, diag;
    int mp, tiles;
};
struct MuSquareTable { MuFirst<2 * kMuGroup> f; MuSquare j[2 * kMuGroup]; };

// Latency-bound: no staging, tiles of 32 x 32 (136 workgroups from one matrix of m = 512), the four waves of a tile take the 32-wide
// reduction steps in turn, each straight from L2 into MFMA operands with kMuAhead steps in flight, and their sums meet in LDS.
// A launch at m = 512 takes 5.5 us (64 x 64 tiles on 36 workgroups: 9.8).  At m = 1024 the finer tiles read twice as much from L2 and
// still win, several workgroups to a CU covering each other's waits: 21 us for the products of the 64 x 64 images' discriminator, 270 MB
// of operands at 12.5 TB/s.
constexpr int kMuAhead = 2;

// tile number -> (ti, tj), ti >= tj, of a triangle of nb rows: in blocks of 4 x 4 tiles where nb allows, so that an XCD's run of
// neighbours needs few row blocks (that net's whole update without it 1.04 ms, with it 1.02, both at the time)
__device__ __forceinline__ void mu_tri_blocked(int t, int nb, int &ti, int &tj) {
    if (nb & 3) { mu_tri(t, ti, tj); return; }
    int si = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.125f);        // 8 si^2 + 2 si tiles before block row si
    while (8 * (si + 1) * (si + 1) + 2 * (si + 1) <= t) ++si;
    while (8 * si * si + 2 * si > t) --si;
    t -= 8 * si * si + 2 * si;
    if (t < 16 * si) { ti = si * 4 + ((t >> 2) & 3); tj = (t >> 4) * 4 + (t & 3); return; }
    mu_tri(t - 16 * si, ti, tj);
    ti += si * 4; tj += si * 4;
}
// a 32 x 32 sum in LDS, eight-column groups of row r at group ^ (r & 3)
__device__ __forceinline__ int mu_lds32(int r, int c) { return r * 32 + (((c >> 3) ^ (r & 3)) << 3) + (c & 7); }

__global__ __launch_bounds__(256, 2) void mu_square_kernel(MuSquareTable t) {
    __shared__ __attribute__((aligned(16))) float part[4][32 * 32];
    MuSquare p;
    unsigned start;
    mu_which(t.f, t.j, blockIdx.x, p, start);
    const int item = mu_item(blockIdx.x - start, p.tiles);
    if (item < 0) return;
    int ti, tj;
    mu_tri_blocked(item, p.mp / 32, ti, tj);
    const int kb = p.mp / 16, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const size_t sr = mu_strip(kb);
    const gptr<const f16> a = p.a + ti * sr + lane * 8, b = p.b + tj * sr + lane * 8;
    struct Step { f16x8 a[2][2], b[2][2]; } f[kMuAhead];     // [ks][hi, lo]
    auto fetch = [&](int s, Step &x) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x.a[ks][h] = *(gptr<const f16x8>)(a + (size_t)s * 2048 + ks * 1024 + h * 512);
                x.b[ks][h] = *(gptr<const f16x8>)(b + (size_t)s * 2048 + ks * 1024 + h * 512);
            }
    };
    const int steps = p.mp / 128;                            // of this wave: w, w + 4, ...
#pragma unroll
    for (int i = 0; i < kMuAhead; ++i)
        if (i < steps) fetch(w + 4 * i, f[i]);
    // the result goes out in pieces of 8 values of a row, 64 to a block of 32 rows and 16 columns in lane order: waves 0 and 1 write the
    // tile, waves 2 and 3 its mirror image.  Their pieces of z are asked for with the operands.
    const bool mirror = w >= 2;
    const int r = lane & 31, k = (w & 1) * 16 + (lane >> 5) * 8, R = (mirror ? tj : ti) * 32 + r, K = (mirror ? ti : tj) * 32 + k;
    const size_t o = mu_off(R, K, kb);
    f16x8 zh, zl;
    if (p.z) { zh = *(gptr<const f16x8>)(p.z + o); zl = *(gptr<const f16x8>)(p.z + o + 512); }
    f32x16 acc = {}, low = {};
    for (int s0 = 0; s0 < steps; s0 += kMuAhead) {
#pragma unroll
        for (int i = 0; i < kMuAhead; ++i) {
            if (s0 + i < steps) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i].a[ks][0], f[i].b[ks][0], acc, 0, 0, 0);
                    low = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i].a[ks][0], f[i].b[ks][1], low, 0, 0, 0);
                    low = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[i].a[ks][1], f[i].b[ks][0], low, 0, 0, 0);
                }
                if (s0 + i + kMuAhead < steps) fetch(w + 4 * (s0 + i + kMuAhead), f[i]);
            }
        }
    }
    acc += low;
#pragma unroll
    for (int e = 0; e < 16; ++e) part[w][mu_lds32(mu_row(e), mu_col())] = acc[e];
    __syncthreads();
    if (mirror && ti == tj) return;                          // (a tile on the diagonal holds both halves)
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int at = mirror ? mu_lds32(k + e, r) : mu_lds32(r, k) + e;
        v[e] = p.alpha * ((part[0][at] + part[1][at]) + (part[2][at] + part[3][at]));
    }
    if (p.z) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += p.zscale * ((float)zh[e] + (float)zl[e]) + (R == K + e ? p.diag : 0.f);
    }
    mu_put8(p.o, o, v);
}

// ---- X <- P X, between two chains (packed, both layouts) or as the result ------------------------------------------
struct MuApply {
    MuPtr<const f16> a, b;           // tile rows from a, tile columns from b, reduction over mp
    MuPtr<f16> x, xt;                // not last: packed [mp, np], [np, mp]
    MuPtr<const float> param;        // last, update form: out = keep * param - step * O; null: out = O
    MuPtr<float> out;                // last: [rows, cols]
    float alpha, keep, step;
    int mp, np, rows, cols, tiles_m, items, flip;
};
struct MuApplyTable { MuFirst<kMuGroup> f; MuApply j[kMuGroup]; };

template <bool LAST, int TA>
__global__ __launch_bounds__(256, 2) void mu_apply_kernel(MuApplyTable t) {
    __shared__ __attribute__((aligned(16))) char lds[2 * kMuStage<TA>];
    MuApply p;
    unsigned start;
    mu_which(t.f, t.j, blockIdx.x, p, start);
    const int b = mu_item(blockIdx.x - start, p.items), lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (b < 0) return;
    // the m side of the tile runs fastest: its operand (P, at most a few MB) stays in L2 while X streams through once
    const int tr = (LAST && p.flip ? b / p.tiles_m : b % p.tiles_m) * 64 * TA, tc = (LAST && p.flip ? b % p.tiles_m : b / p.tiles_m) * 128;
    const size_t sr = mu_strip(p.mp / 16);
    f32x16 acc[TA][2];
    mu_tile<TA>(p.a + (size_t)(tr / 32) * sr, sr, p.b + (size_t)(tc / 32) * sr, sr, p.mp / 32, lds, acc);
    const int r0 = tr + (w >> 1) * 32 * TA, c0 = tc + (w & 1) * 64;      // this wave's 32 TA x 64
    if (LAST) {
        // (every parameter is read before the first result is written: out may be param)
        float old[TA][2][16];
        if (p.param) {
#pragma unroll
            for (int i = 0; i < TA; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int r = r0 + i * 32 + mu_row(e), c = c0 + j * 32 + mu_col();
                        old[i][j][e] = r < p.rows && c < p.cols ? p.param[(size_t)r * p.cols + c] : 0.f;
                    }
        }
#pragma unroll
        for (int i = 0; i < TA; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int r = r0 + i * 32 + mu_row(e), c = c0 + j * 32 + mu_col();
                    const float v = p.alpha * acc[i][j][e];
                    if (r < p.rows && c < p.cols) p.out[(size_t)r * p.cols + c] = p.param ? p.keep * old[i][j][e] - p.step * v : v;
                }
        return;
    }
    // both layouts of the next X from the wave's own quarter of the staging buffers (mu_tile ends with a barrier)
    float *mine = reinterpret_cast<float *>(lds) + w * 2048 * TA;
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) mine[mu_lds(i * 32 + mu_row(e), j * 32 + mu_col())] = p.alpha * acc[i][j][e];
    __syncthreads();
#pragma unroll
    for (int blk = 0; blk < 4 * TA; ++blk) {
        float v[8];
        {
            const int r = (blk >> 2) * 32 + (lane & 31), k = (blk & 3) * 16 + (lane >> 5) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = mine[mu_lds(r, k) + e];
            mu_put8(p.x, mu_off(r0 + r, c0 + k, p.np / 16), v);
        }
        const int r = (blk / (2 * TA)) * 32 + (lane & 31), k = (blk % (2 * TA)) * 16 + (lane >> 5) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mine[mu_lds(k + e, r)];
        mu_put8(p.xt, mu_off(c0 + r, r0 + k, p.mp / 16), v);
    }
}

// ---- host side -----------------------------------------------------------------------------------------------------
static bool mu_aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }
struct MuMat {                       // a matrix's place in the workspace
    int rows, cols, mp, np, tall, nparts, tiles, splits, steps_per;
    size_t part, u, x, xt, xt2, a, qq, w, p0, p1, slab;      // byte offsets
    size_t end;
};
static MuMat mu_place(int rows, int cols, bool keep_u, int steps, size_t base) {
    MuMat m{};
    m.rows = rows; m.cols = cols; m.tall = rows >= cols;
    const int s = m.tall ? cols : rows, l = m.tall ? rows : cols;
    m.mp = (s + kMuPad - 1) / kMuPad * kMuPad;
    m.np = (int)(((long)l + kMuPad - 1) / kMuPad * kMuPad);
    const long n = (long)rows * cols, want = (n + kMuPrepPer - 1) / kMuPrepPer;
    m.nparts = (int)(want < kMuPrepMax ? want : kMuPrepMax);
    // one triangle of 128 x 128 tiles, the reduction in runs of 8 to 16 32-wide steps: 512 workgroups from one matrix where it has
    // them, and no run so short that its 64 KB of sums cost more than its 32 KB stages; up to 64 steps where 4096 workgroups
    // remain (4194304 x 511: 34.9 ms and 37 GB of scratch, with 16 steps 38.5 ms and 41 GB).  (A rule on the matrix alone:
    // what it gives does not depend on the others of a call.)
    const int tb = m.mp / 128, all = m.np / 32;
    m.tiles = tb * (tb + 1) / 2;
    long run = ((long)m.tiles * all + 511) / 512;
    run = run < 8 ? 8 : run > 16 ? 16 : run;
    const long far = (long)m.tiles * all / 4096;
    if (far > run) run = far < 64 ? far : 64;
    run = (run + 1) & ~1L;                                   // (even: mu_tile)
    m.steps_per = all < run ? all : (int)run;
    m.splits = (all + m.steps_per - 1) / m.steps_per;
    const size_t bx = m.mp / 32 * mu_strip(m.np / 16) * 2, bt = m.np / 32 * mu_strip(m.mp / 16) * 2, sq = m.mp / 32 * mu_strip(m.mp / 16) * 2;
    size_t o = mu_round(base);
    auto take = [&](size_t bytes) { const size_t at = o; o += mu_round(bytes); return at; };
    m.part = take((size_t)m.nparts * sizeof(double));
    m.u = keep_u ? take((size_t)n * 4) : 0;
    m.x = take(bx); m.xt = take(bt);
    m.xt2 = steps > mu_chain(0, steps) ? take(bt) : 0;
    m.a = take(sq); m.qq = take(sq); m.w = take(sq); m.p0 = take(sq); m.p1 = take(sq);
    m.slab = take((size_t)m.splits * m.tiles * 128 * 128 * 4);
    m.end = o;
    return m;
}

// the matrices with the longest products first: a launch ends with its short workgroups
static void mu_order(MuJob *j, int n) {
    auto before = [](const MuJob &a, const MuJob &b) {
        const int sa = a.rows < a.cols ? a.rows : a.cols, sb = b.rows < b.cols ? b.rows : b.cols;
        return sa != sb ? sa > sb : (long)a.rows * a.cols > (long)b.rows * b.cols;
    };
    for (int i = 1; i < n; ++i) {
        const MuJob x = j[i];
        int k = i;
        for (; k > 0 && before(x, j[k - 1]); --k) j[k] = j[k - 1];
        j[k] = x;
    }
}

// all matrices of one group, phase by phase
static void mu_run_group(const MuJob *jobs, int n, bool update, const MuStep &sp, char *ws, hipStream_t st) {
    MuMat m[kMuGroup];
    const int steps = sp.steps;
    const bool keep_u = update && sp.nesterov;
    size_t at = 0;
    for (int i = 0; i < n; ++i) { m[i] = mu_place(jobs[i].rows, jobs[i].cols, keep_u, steps, at); at = m[i].end; }
    {
        MuPrepTable t{};
        t.momentum = sp.momentum; t.grad_scale = sp.grad_scale; t.nesterov = sp.nesterov;
        unsigned blocks = 0;
        for (int i = 0; i < n; ++i) {
            MuPrep &p = t.j[i];
            p.grad = jobs[i].grad; p.mom = jobs[i].mom; p.mom_out = jobs[i].mom_out;
            p.u = keep_u ? (float *)(ws + m[i].u) : nullptr;
            p.dsigma = jobs[i].dsigma; p.dot = jobs[i].dot; p.sigma = jobs[i].sigma; p.scale = jobs[i].scale;
            p.part = (double *)(ws + m[i].part);
            p.n = (long)jobs[i].rows * jobs[i].cols;
            p.vec = mu_aligned(p.grad.p) && mu_aligned(p.mom.p) && mu_aligned(p.mom_out.p) && mu_aligned(p.dsigma.p);
            p.blocks = m[i].nparts;
            t.f.first[i] = blocks;
            blocks += m[i].nparts;
        }
        mu_close(t.f, n);
        hipLaunchKernelGGL(mu_prep_kernel, dim3(blocks), dim3(256), 0, st, t);
    }
    f16 *x[kMuGroup], *xt[kMuGroup], *xt_next[kMuGroup];
    {
        MuSplitTable t{};
        unsigned blocks = 0;
        for (int i = 0; i < n; ++i) {
            MuSplit &p = t.j[i];
            p.u = keep_u ? (const float *)(ws + m[i].u) : update ? jobs[i].mom_out.p : jobs[i].grad.p;
            p.part = (const double *)(ws + m[i].part); p.nparts = m[i].nparts;
            x[i] = (f16 *)(ws + m[i].x); xt[i] = (f16 *)(ws + m[i].xt); xt_next[i] = (f16 *)(ws + m[i].xt2);
            p.x = x[i]; p.xt = xt[i];
            p.rows = jobs[i].rows; p.cols = jobs[i].cols; p.mp = m[i].mp; p.np = m[i].np; p.tall = m[i].tall;
            t.f.first[i] = blocks;
            blocks += (unsigned)((long)m[i].mp / 64 * (m[i].np / 64));
        }
        mu_close(t.f, n);
        hipLaunchKernelGGL(mu_split_kernel, dim3(blocks), dim3(256), 0, st, t);
    }
    for (int done = 0; done < steps;) {
        const int chain = mu_chain(done, steps);
        {
            MuGramTable t{};
            unsigned blocks = 0, red = 0;
            for (int i = 0; i < n; ++i) {
                MuGram &p = t.j[i];
                p.x = x[i]; p.slab = (float *)(ws + m[i].slab); p.a = (f16 *)(ws + m[i].a);
                p.mp = m[i].mp; p.np = m[i].np; p.tiles = m[i].tiles; p.splits = m[i].splits; p.steps_per = m[i].steps_per;
                t.f.first[i] = blocks; t.r.first[i] = red;
                blocks += (p.tiles * p.splits + 7) & ~7; red += p.tiles * 16;
            }
            mu_close(t.f, n);
            mu_close(t.r, n);
            hipLaunchKernelGGL(mu_gram_kernel, dim3(blocks), dim3(256), 0, st, t);
            hipLaunchKernelGGL(mu_gram_reduce_kernel, dim3(red), dim3(256), 0, st, t);
        }
        // P: the product of the chain's polynomials so far, in p0 or p1; Q of the first step IS the first P
        bool in_p0 = true;
        for (int k = 0; k < chain; ++k) {
            const bool last = k == chain - 1;
            const float s_p = k == 1 ? kScaleQ : kScaleP;    // scale of the P that this step's Q multiplies
            MuSquareTable t{};
            unsigned blocks = 0;
            int nt = 0;
            auto add = [&](int i, size_t a, size_t b, size_t o, float alpha) -> MuSquare & {
                MuSquare &p = t.j[nt];
                p = MuSquare{};
                p.a = (const f16 *)(ws + a); p.b = (const f16 *)(ws + b); p.o = (f16 *)(ws + o); p.alpha = alpha;
                p.mp = m[i].mp;
                const int tb = p.mp / 32;
                p.tiles = tb * (tb + 1) / 2;
                t.f.first[nt++] = blocks;
                blocks += (p.tiles + 7) & ~7;
                return p;
            };
            auto go = [&]() {
                mu_close(t.f, nt);
                if (nt) hipLaunchKernelGGL(mu_square_kernel, dim3(blocks), dim3(256), 0, st, t);
                blocks = 0;
                nt = 0;
            };
            auto q_of = [&](int i) { return k == 0 ? m[i].p0 : m[i].qq; };
            for (int i = 0; i < n; ++i) {                    // Q = a I + b A + c A^2
                MuSquare &p = add(i, m[i].a, m[i].a, q_of(i), kMuC * kScaleQ / (kScaleA * kScaleA));
                p.z = p.a; p.zscale = kMuB * kScaleQ / kScaleA; p.diag = kMuA * kScaleQ;
            }
            go();
            for (int i = 0; i < n; ++i) {
                if (!last) add(i, q_of(i), m[i].a, m[i].w, 1.f / kScaleQ);                                     // W = Q A
                if (k > 0) add(i, m[i].qq, in_p0 ? m[i].p0 : m[i].p1, in_p0 ? m[i].p1 : m[i].p0, kScaleP / (kScaleQ * s_p));   // P = Q P
            }
            go();
            if (k > 0) in_p0 = !in_p0;
            if (!last) {
                for (int i = 0; i < n; ++i) add(i, m[i].w, q_of(i), m[i].a, 1.f / kScaleQ);                    // A = W Q
                go();
            }
        }
        done += chain;
        MuApplyTable t{};
        unsigned blocks = 0;
        long all = 0;
        for (int i = 0; i < n; ++i) all += (long)(m[i].mp / 128) * (m[i].np / 128);
        const int ta = all < kMuApplyFine ? 1 : 2;
        const float s_p = chain == 1 ? kScaleQ : kScaleP;
        for (int i = 0; i < n; ++i) {
            MuApply &p = t.j[i];
            const f16 *pp = (const f16 *)(ws + (in_p0 ? m[i].p0 : m[i].p1));
            const bool flip = done == steps && m[i].tall;    // the result in U's own layout: tile rows along its rows
            p.a = flip ? xt[i] : pp; p.b = flip ? pp : xt[i];
            p.mp = m[i].mp; p.np = m[i].np; p.rows = jobs[i].rows; p.cols = jobs[i].cols;
            p.flip = flip;
            p.tiles_m = flip ? m[i].mp / 128 : m[i].mp / (64 * ta);
            p.alpha = done == steps ? 1.f / (s_p * kScaleX) : 1.f / s_p;
            p.x = x[i]; p.xt = xt_next[i];
            p.param = update ? jobs[i].param.p : nullptr; p.out = jobs[i].out; p.keep = jobs[i].keep; p.step = jobs[i].step;
            t.f.first[i] = blocks;
            p.items = m[i].mp / 128 * (m[i].np / 128) * (2 / ta);
            blocks += (unsigned)(p.items + 7) & ~7u;
        }
        mu_close(t.f, n);
        if (ta == 1) {
            if (done == steps) hipLaunchKernelGGL((mu_apply_kernel<true, 1>), dim3(blocks), dim3(256), 0, st, t);
            else hipLaunchKernelGGL((mu_apply_kernel<false, 1>), dim3(blocks), dim3(256), 0, st, t);
        } else {
            if (done == steps) hipLaunchKernelGGL((mu_apply_kernel<true, 2>), dim3(blocks), dim3(256), 0, st, t);
            else hipLaunchKernelGGL((mu_apply_kernel<false, 2>), dim3(blocks), dim3(256), 0, st, t);
        }
        for (int i = 0; i < n; ++i) { f16 *s = xt[i]; xt[i] = xt_next[i]; xt_next[i] = s; }
    }
}

// The matrices of a call in groups of kMuGroup, small ones (muon_small.hip) and others each among themselves: calls
// f(indices, count, small) per group, in an order that depends on the sizes' kinds alone.
template <typename F> static void mu_groups(const mmdgan_muon_job *jobs, int n, F &&f) {
    for (int small = 0; small < 2; ++small) {
        int idx[kMuGroup], k = 0;
        for (int i = 0; i < n; ++i) {
            if (mu_is_small(jobs[i].rows, jobs[i].cols) != (small != 0)) continue;
            idx[k++] = i;
            if (k == kMuGroup) { f(idx, k, small != 0); k = 0; }
        }
        if (k) f(idx, k, small != 0);
    }
}
// groups run one after the other in the same scratch
static size_t mu_bytes(const mmdgan_muon_job *jobs, int n, int steps, bool keep_u) {
    size_t most = 256;
    mu_groups(jobs, n, [&](const int *idx, int k, bool small) {
        size_t at = 0;
        for (int i = 0; i < k; ++i) {
            const mmdgan_muon_job &j = jobs[idx[i]];
            at = small ? mu_round(at) + mu_small_bytes(j.rows, j.cols, keep_u, steps) : mu_place(j.rows, j.cols, keep_u, steps, at).end;
        }
        if (at > most) most = at;
    });
    return most;
}
static void mu_run(MuJob *j, int n, bool update, const MuStep &s, bool small, char *ws, hipStream_t st) {
    mu_order(j, n);
    if (small) mu_small_run(j, n, s, ws, st);
    else mu_run_group(j, n, update, s, ws, st);
}
static bool mu_sizes_ok(const mmdgan_muon_job *jobs, int n, int steps) {
    if (!jobs || n < 1 || steps < 1 || steps > 16) return false;
    for (int i = 0; i < n; ++i) {
        const long r = jobs[i].rows, c = jobs[i].cols, s = r < c ? r : c, l = r < c ? c : r;
        if (s < 1 || s > 8192 || l > (1L << 22) || r * c > (1L << 31) - 1) return false;
    }
    return true;
}
}  // namespace mmdgan

using namespace mmdgan;

extern "C" size_t mmdgan_muon_workspace_bytes(const mmdgan_muon_job *jobs, int n_jobs, int steps) {
    return mu_sizes_ok(jobs, n_jobs, steps) ? mu_bytes(jobs, n_jobs, steps, true) : 0;
}

static int mu_check(const mmdgan_muon_job *jobs, int n_jobs, int steps, bool update, void *workspace, const char *what) {
    MMDGAN_REQUIRE(jobs && n_jobs >= 1, "%s: no matrices", what);
    MMDGAN_REQUIRE(steps >= 1 && steps <= 16, "%s: %d steps, 1 to 16 are built", what, steps);
    MMDGAN_REQUIRE(mu_sizes_ok(jobs, n_jobs, steps), "%s: a matrix side is below 1, its shorter side above 8192 or its longer above 4194304", what);
    MMDGAN_REQUIRE(workspace && !((uintptr_t)workspace & 15), "%s: the workspace is null or not 16-byte aligned", what);
    for (int i = 0; i < n_jobs; ++i) {
        const mmdgan_muon_job &j = jobs[i];
        MMDGAN_REQUIRE(j.grad && j.out, "%s: matrix %d: null pointer", what, i);
        MMDGAN_REQUIRE(!update || (j.param && j.momentum && j.momentum_out), "%s: matrix %d: null pointer", what, i);
        MMDGAN_REQUIRE(!j.dsigma || (j.dot && j.sigma && j.scale), "%s: matrix %d: dsigma without dot, sigma and scale", what, i);
    }
    // what a matrix writes is its own: groups run one after the other, and a matrix's workgroups in no order
    for (int i = 0; i < n_jobs; ++i) {
        const mmdgan_muon_job &j = jobs[i];
        const size_t bytes = (size_t)j.rows * j.cols * 4;
        for (int k = 0; k < n_jobs; ++k) {
            const mmdgan_muon_job &o = jobs[k];
            const size_t ob = (size_t)o.rows * o.cols * 4;
            const bool same = i == k;
            bool meet = (same ? (update || j.out != o.grad) && spans_meet(j.out, bytes, o.grad, ob)
                              : spans_meet(j.out, bytes, o.grad, ob) || spans_meet(j.out, bytes, o.out, ob));
            if (update) {
                meet = meet || (!(same && j.out == o.param) && spans_meet(j.out, bytes, o.param, ob)) || spans_meet(j.out, bytes, o.momentum, ob) ||
                       spans_meet(j.out, bytes, o.momentum_out, ob) || spans_meet(j.out, bytes, o.dsigma, ob);
                meet = meet || spans_meet(j.momentum_out, bytes, o.grad, ob) || spans_meet(j.momentum_out, bytes, o.param, ob) ||
                       (!(same && j.momentum_out == o.momentum) && spans_meet(j.momentum_out, bytes, o.momentum, ob)) ||
                       (!same && spans_meet(j.momentum_out, bytes, o.momentum_out, ob)) || spans_meet(j.momentum_out, bytes, o.dsigma, ob);
            }
            MMDGAN_REQUIRE(!meet, "%s: an output of matrix %d overlaps a tensor of matrix %d", what, i, k);
        }
    }
    return MMDGAN_OK;
}

extern "C" int mmdgan_orthogonalize(const mmdgan_muon_job *jobs, int n_jobs, int steps, void *workspace, void *stream) {
    if (int rc = mu_check(jobs, n_jobs, steps, false, workspace, "orthogonalize")) return rc;
    const MuStep s{0.f, 1.f, 0, steps};
    mu_groups(jobs, n_jobs, [&](const int *idx, int n, bool small) {
        MuJob j[kMuGroup] = {};
        for (int i = 0; i < n; ++i) {
            const mmdgan_muon_job &q = jobs[idx[i]];
            j[i].rows = q.rows; j[i].cols = q.cols; j[i].grad = q.grad; j[i].out = q.out;
        }
        mu_run(j, n, false, s, small, (char *)workspace, (hipStream_t)stream);
    });
    return check_launch("orthogonalize");
}

extern "C" int mmdgan_muon_update(const mmdgan_muon_job *jobs, int n_jobs, float lr, float momentum, int nesterov, float weight_decay,
                                  float grad_scale, int apply_fixup, int steps, void *workspace, void *stream) {
    if (int rc = mu_check(jobs, n_jobs, steps, true, workspace, "muon_update")) return rc;
    const MuStep st{momentum, grad_scale, nesterov != 0, steps};
    mu_groups(jobs, n_jobs, [&](const int *idx, int n, bool small) {
        MuJob j[kMuGroup] = {};
        for (int i = 0; i < n; ++i) {
            const mmdgan_muon_job &q = jobs[idx[i]];
            MuJob &d = j[i];
            d.rows = q.rows; d.cols = q.cols; d.grad = q.grad; d.mom = q.momentum; d.mom_out = q.momentum_out; d.param = q.param; d.out = q.out;
            if (apply_fixup && q.dsigma) { d.dsigma = q.dsigma; d.dot = q.dot; d.sigma = q.sigma; d.scale = q.scale; }
            const int big = q.rows > q.cols ? q.rows : q.cols;
            d.keep = (float)(1.0 - (double)lr * weight_decay);
            d.step = (float)((double)lr * 0.2 * sqrt((double)big));
        }
        mu_run(j, n, true, st, small, (char *)workspace, (hipStream_t)stream);
    });
    return check_launch("muon_update");
}
