// Orthogonalised updates: O = the fifth (or any) iterate of the quintic  X <- a X + b (X X^T) X + c (X X^T)^2 X  started at
// X = U / ||U||_F, which takes every singular value of U to about 1 (0.7 .. 1.2), and the parameter update that applies it
// to a momentum matrix.  Matrices are row-major [rows, cols]; m = the shorter side, n = the longer one, X is [m, n].
//
// Mathematics used.  With A = X X^T the iterate is X' = Q X, Q = a I + b A + c A^2, and the next Gram matrix is
// A' = Q A Q: all of them are polynomials of one symmetric matrix, they commute, so up to three steps run on m x m
// matrices alone, P = Q3 Q2 Q1, before X is touched again: X <- P X, A = X X^T from the new X.  Rounding errors of A grow by Q^2
// (12 at the small end) per step on directions with tiny singular values; three steps between two true Gram matrices keep the
// result as near to the exact one as steps on X itself, five do not (six times the error on ill-conditioned U).  Work for five
// steps: two Gram matrices (m^2 n each, one triangle) and two products with X (2 m^2 n each) instead of five of both.
//
// Numerics.  Every m x n and m x m operand is held as TWO fp16 numbers, v * s = hi + lo with s a fixed power of two that keeps
// the largest possible entry (the norms are bounded: singular values <= 1.21, |Q| <= 3.45, |P| <= 41) below 65504: 22 bits, and
// 2^-25 / s absolute where lo underflows.  Products are hi hi + hi lo + lo hi in fp32 accumulators (lo lo is 2^-22 of the
// result): as good as fp32 operands at 16/3 of the fp32 matrix rate.
//
// Layout ("packed"): row r of an [R, K] operand is K / 32 groups of 128 bytes, 32 hi halves then 32 lo halves: a 128-byte line
// per row and 32-wide reduction step, and the MFMA operand of a lane (8 halves) is one 16-byte piece of it.  All sides are
// padded to 128 with zeros, so the products have no edges.
#include "common.h"

namespace mmdgan {

typedef _Float16 f16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int mu_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMuGroup = 16;                 // matrices per launch (the task tables travel by value)
constexpr int kMuPad = 128;
constexpr int kMuChain = 3;                  // steps between two true Gram matrices
constexpr float kMuA = 3.4445f, kMuB = -4.7750f, kMuC = 2.0315f;
constexpr float kScaleX = 4096.f, kScaleA = 4096.f, kScaleQ = 8192.f, kScaleP = 1024.f;

// offset (in halves) of element (r, k)'s hi part in a packed operand with `ld` = 2 * K halves per row; lo is 32 further
__host__ __device__ __forceinline__ size_t mu_off(size_t r, int k, int ld) { return r * ld + (size_t)(k >> 5) * 64 + (k & 31); }

__device__ __forceinline__ void mu_split(float v, f16 &hi, f16 &lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// ---- the product of one tile -------------------------------------------------------------------------------------
// C[i, j] = sum_k A[i, k] B[j, k] for a (64 TB) x (64 TB) tile, four waves as 2 x 2, each (32 TB) x (32 TB).  Per 32-wide step the
// workgroup stages 64 TB rows of each operand (128 bytes a row) in LDS, double buffered; 16-byte piece c of row r lies at
// piece c ^ (r & 7), which spreads the 8 rows that a ds_read_b128 serves per cycle over all banks.
template <int TB> struct MuTile {
    static constexpr int kRows = 64 * TB;
    static constexpr int kStage = 2 * kRows * 128;           // bytes
    static constexpr int kLds = 2 * kStage;
};
template <int TB>
__device__ __forceinline__ void mu_tile(const f16 *A, int lda, const f16 *B, int ldb, int steps, char *lds, f32x16 (&acc)[TB][TB]) {
    constexpr int R = MuTile<TB>::kRows, L = 2 * TB;         // 16-byte pieces per thread and operand: R * 8 / 256
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int pr = t >> 3, pc = t & 7;                       // this thread's piece of rows pr, pr + 32, ...
    mu_u32x4 ra[L], rb[L];
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
            ra[i] = *reinterpret_cast<const mu_u32x4 *>(A + (size_t)(pr + 32 * i) * lda + s * 64 + pc * 8);
            rb[i] = *reinterpret_cast<const mu_u32x4 *>(B + (size_t)(pr + 32 * i) * ldb + s * 64 + pc * 8);
        }
    };
    auto store = [&](char *buf) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int r = pr + 32 * i;
            *reinterpret_cast<mu_u32x4 *>(buf + r * 128 + ((pc ^ (r & 7)) << 4)) = ra[i];
            *reinterpret_cast<mu_u32x4 *>(buf + (R + r) * 128 + ((pc ^ (r & 7)) << 4)) = rb[i];
        }
    };
    f32x16 low[TB][TB];                                      // hi lo + lo hi: 2^-11 of the sum, so their roundings do not count
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) { acc[i][j] = f32x16{}; low[i][j] = f32x16{}; }
    const int ar = (w >> 1) * 32 * TB + (lane & 31), br = R + (w & 1) * 32 * TB + (lane & 31), half = lane >> 5;
    fetch(0);
    store(lds);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const char *buf = lds + (s & 1) * MuTile<TB>::kStage;
        if (s + 1 < steps) fetch(s + 1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            f16x8 ah[TB], al[TB], bh[TB], bl[TB];
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                const int r = ar + 32 * i, q = br + 32 * i, c = ks * 2 + half;
                ah[i] = *reinterpret_cast<const f16x8 *>(buf + r * 128 + ((c ^ (r & 7)) << 4));
                al[i] = *reinterpret_cast<const f16x8 *>(buf + r * 128 + (((c + 4) ^ (r & 7)) << 4));
                bh[i] = *reinterpret_cast<const f16x8 *>(buf + q * 128 + ((c ^ (q & 7)) << 4));
                bl[i] = *reinterpret_cast<const f16x8 *>(buf + q * 128 + (((c + 4) ^ (q & 7)) << 4));
            }
#pragma unroll
            for (int i = 0; i < TB; ++i)
#pragma unroll
                for (int j = 0; j < TB; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
                    low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], low[i][j], 0, 0, 0);
                    low[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], low[i][j], 0, 0, 0);
                }
        }
        if (s + 1 < steps) store(lds + ((s + 1) & 1) * MuTile<TB>::kStage);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j) acc[i][j] += low[i][j];
}
// row / column within the tile of accumulator element e of block (bi, bj): C layout of the 32x32 MFMA
template <int TB> __device__ __forceinline__ int mu_row(int bi, int e) {
    const int t = threadIdx.x;
    return ((t >> 7) & 1) * 32 * TB + 32 * bi + (e >> 2) * 8 + ((t & 63) >> 5) * 4 + (e & 3);
}
template <int TB> __device__ __forceinline__ int mu_col(int bj) {
    const int t = threadIdx.x;
    return ((t >> 6) & 1) * 32 * TB + 32 * bj + (t & 31);
}

// lower-triangle tile number -> (ti, tj), ti >= tj
__device__ __forceinline__ void mu_tri(int t, int &ti, int &tj) {
    int r = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while ((r + 1) * (r + 2) / 2 <= t) ++r;
    while (r * (r + 1) / 2 > t) --r;
    ti = r;
    tj = t - r * (r + 1) / 2;
}

// ---- momentum and norm -------------------------------------------------------------------------------------------
struct MuPrep {
    const float *grad, *mom;         // mom null: U = grad
    float *mom_out, *u;              // u: where U goes when it is neither grad nor mom_out (Nesterov), else null
    const float *dsigma, *dot, *sigma, *scale;
    double *part;                    // [blocks]
    long n;
    unsigned first_block;
};
struct MuPrepTable { MuPrep j[kMuGroup]; int n; float momentum, grad_scale; int nesterov; };
constexpr int kMuPrepPer = 4096;     // elements per workgroup and round
constexpr int kMuPrepMax = 256;      // workgroups per matrix

// U = g (+ momentum), its sum of squares by workgroup.  g = grad_scale * grad, or of a spectrally normalised kernel
// grad_scale * (scale * grad - (scale / sigma) <grad, W> dsigma/dW)  (Adam's read, elementwise.hip)
__global__ __launch_bounds__(256) void mu_prep_kernel(MuPrepTable t) {
    __shared__ double red[4];
    int q = 0;
    while (q + 1 < t.n && blockIdx.x >= t.j[q + 1].first_block) ++q;
    const MuPrep &p = t.j[q];
    const unsigned nb = (q + 1 < t.n ? t.j[q + 1].first_block : gridDim.x) - p.first_block, b = blockIdx.x - p.first_block;
    float c0 = t.grad_scale, c1 = 0.f;
    if (p.dsigma) { c0 = t.grad_scale * p.scale[0]; c1 = t.grad_scale * (p.scale[0] / p.sigma[0]) * p.dot[0]; }
    double ss = 0.0;
    for (long i = (long)b * 256 + threadIdx.x; i < p.n; i += (long)nb * 256) {
        float g = c0 * p.grad[i];
        if (p.dsigma) g -= c1 * p.dsigma[i];
        float u = g;
        if (p.mom) {
            const float m = __builtin_fmaf(t.momentum, p.mom[i], g);
            p.mom_out[i] = m;
            u = t.nesterov ? __builtin_fmaf(t.momentum, m, g) : m;
            if (p.u) p.u[i] = u;
        }
        ss += (double)u * (double)u;
    }
    ss = wave_sum(ss);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    if (threadIdx.x == 0) p.part[b] = red[0] + red[1] + red[2] + red[3];
}

// ---- X = U / ||U|| as packed [m, n] and [n, m] --------------------------------------------------------------------
struct MuSplit {
    const float *u;                  // [rows, cols]
    const double *part;
    int nparts;
    f16 *x, *xt;                     // [mp, np] and [np, mp]
    int rows, cols, mp, np, tall;    // tall: rows = n
    unsigned first_block;
};
struct MuSplitTable { MuSplit j[kMuGroup]; int n; };

// one 64 x 64 tile of the padded matrix; "natural" = the operand whose rows are U's rows
__global__ __launch_bounds__(256) void mu_split_kernel(MuSplitTable t) {
    __shared__ float tile[64][65];
    __shared__ double s_inv;
    int q = 0;
    while (q + 1 < t.n && blockIdx.x >= t.j[q + 1].first_block) ++q;
    const MuSplit &p = t.j[q];
    const int b = blockIdx.x - p.first_block;
    const int prows = p.tall ? p.np : p.mp, pcols = p.tall ? p.mp : p.np;
    const int r0 = b / (pcols / 64) * 64, c0 = b % (pcols / 64) * 64;
    if (threadIdx.x < 64) {
        double s = 0.0;
        for (int i = threadIdx.x; i < p.nparts; i += 64) s += p.part[i];
        s = wave_sum(s);
        if (threadIdx.x == 0) s_inv = s > 0.0 ? (double)kScaleX / sqrt(s) : s == 0.0 ? 0.0 : s;       // NaN stays NaN
    }
    __syncthreads();
    const double inv = s_inv;
    const int tc = threadIdx.x & 63, tr = threadIdx.x >> 6;
    f16 *nat = p.tall ? p.xt : p.x, *tra = p.tall ? p.x : p.xt;
    const int ldn = 2 * pcols, ldt = 2 * prows;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const int r = r0 + tr + 4 * i, c = c0 + tc;
        const float v = r < p.rows && c < p.cols ? (float)((double)p.u[(size_t)r * p.cols + c] * inv) : 0.f;
        tile[tr + 4 * i][tc] = v;
        f16 hi, lo;
        mu_split(v, hi, lo);
        const size_t o = mu_off(r, c, ldn);
        nat[o] = hi; nat[o + 32] = lo;
    }
    __syncthreads();
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
        const int c = tr + 4 * i;
        f16 hi, lo;
        mu_split(tile[tc][c], hi, lo);
        const size_t o = mu_off(c0 + c, r0 + tc, ldt);
        tra[o] = hi; tra[o + 32] = lo;
    }
}

// ---- Gram matrix A = X X^T: one triangle of 128 x 128 tiles, the reduction over n split ----------------------------
struct MuGram {
    const f16 *x;
    float *slab;                     // [splits][tiles][128][128]
    f16 *a;                          // [mp, mp]
    int mp, np, tiles, splits, steps_per;
    unsigned first_block, first_reduce;
};
struct MuGramTable { MuGram j[kMuGroup]; int n; };

__global__ __launch_bounds__(256, 2) void mu_gram_kernel(MuGramTable t) {
    __shared__ __attribute__((aligned(16))) char lds[MuTile<2>::kLds];
    int q = 0;
    while (q + 1 < t.n && blockIdx.x >= t.j[q + 1].first_block) ++q;
    const MuGram &p = t.j[q];
    const int b = blockIdx.x - p.first_block, split = b / p.tiles, tile = b % p.tiles;
    int ti, tj;
    mu_tri(tile, ti, tj);
    const int s0 = split * p.steps_per, all = p.np / 32;
    const int steps = s0 + p.steps_per < all ? p.steps_per : all - s0;
    f32x16 acc[2][2];
    mu_tile<2>(p.x + (size_t)ti * 128 * 2 * p.np + (size_t)s0 * 64, 2 * p.np, p.x + (size_t)tj * 128 * 2 * p.np + (size_t)s0 * 64, 2 * p.np,
               steps, lds, acc);
    float *o = p.slab + ((size_t)split * p.tiles + tile) * 128 * 128;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[mu_row<2>(i, e) * 128 + mu_col<2>(j)] = acc[i][j][e];
}

// sums the splits of a 32 x 32 block in order, writes A packed, and its mirror image
__global__ __launch_bounds__(256) void mu_gram_reduce_kernel(MuGramTable t) {
    __shared__ float blk[32][33];
    int q = 0;
    while (q + 1 < t.n && blockIdx.x >= t.j[q + 1].first_reduce) ++q;
    const MuGram &p = t.j[q];
    const int b = blockIdx.x - p.first_reduce, tile = b >> 4, sub = b & 15;
    int ti, tj;
    mu_tri(tile, ti, tj);
    const int r0 = (sub >> 2) * 32, c0 = (sub & 3) * 32, tc = threadIdx.x & 31, tr = threadIdx.x >> 5;
    const float k = kScaleA / (kScaleX * kScaleX);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = tr + 8 * i;
        const float *s = p.slab + (size_t)tile * 128 * 128 + (r0 + r) * 128 + c0 + tc;
        double sum = 0.0;                                    // (the splits' own sums are short: this is where the long one is formed)
        for (int z = 0; z < p.splits; ++z) sum += (double)s[(size_t)z * p.tiles * 128 * 128];
        const float v = (float)(sum * k);
        blk[r][tc] = v;
        f16 hi, lo;
        mu_split(v, hi, lo);
        const size_t o = mu_off(ti * 128 + r0 + r, tj * 128 + c0 + tc, 2 * p.mp);
        p.a[o] = hi; p.a[o + 32] = lo;
    }
    if (ti == tj) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = tr + 8 * i;
        f16 hi, lo;
        mu_split(blk[tc][c], hi, lo);
        const size_t o = mu_off(tj * 128 + c0 + c, ti * 128 + r0 + tc, 2 * p.mp);
        p.a[o] = hi; p.a[o + 32] = lo;
    }
}

// ---- m x m products of commuting symmetric matrices: one triangle of 64 x 64 tiles --------------------------------
struct MuSquare {
    const f16 *a, *b;                // o = alpha a b  (packed, symmetric, [mp, mp])
    f16 *o;
    const f16 *z;                    // polynomial form: o += zscale * z + diag on the diagonal; null: the plain product
    float alpha, zscale, diag;
    int mp, tiles;
    unsigned first_block;
};
struct MuSquareTable { MuSquare j[2 * kMuGroup]; int n; };

__global__ __launch_bounds__(256) void mu_square_kernel(MuSquareTable t) {
    __shared__ __attribute__((aligned(16))) char lds[MuTile<1>::kLds];
    int q = 0;
    while (q + 1 < t.n && blockIdx.x >= t.j[q + 1].first_block) ++q;
    const MuSquare &p = t.j[q];
    int ti, tj;
    mu_tri(blockIdx.x - p.first_block, ti, tj);
    const int ld = 2 * p.mp;
    f32x16 acc[1][1];
    mu_tile<1>(p.a + (size_t)ti * 64 * ld, ld, p.b + (size_t)tj * 64 * ld, ld, p.mp / 32, lds, acc);
    const int c = tj * 64 + mu_col<1>(0);
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
        f16x4 hi, lo;
        const int r = ti * 64 + mu_row<1>(0, e4 * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = p.alpha * acc[0][0][e4 * 4 + e];
            const size_t o = mu_off(r + e, c, ld);
            if (p.z) {
                v += p.zscale * ((float)p.z[o] + (float)p.z[o + 32]);
                if (r + e == c) v += p.diag;
            }
            f16 h, l;
            mu_split(v, h, l);
            p.o[o] = h; p.o[o + 32] = l;
            hi[e] = h; lo[e] = l;
        }
        if (ti != tj) {
            const size_t o = mu_off(c, r, ld);
            *reinterpret_cast<f16x4 *>(p.o + o) = hi;
            *reinterpret_cast<f16x4 *>(p.o + o + 32) = lo;
        }
    }
}

// ---- X <- P X, between two chains (packed, both layouts) or as the result ------------------------------------------
struct MuApply {
    const f16 *a, *b;                // tile rows from a, tile columns from b, reduction over mp
    f16 *x, *xt;                     // not last: packed [mp, np], [np, mp]
    const float *param;              // last, update form: out = keep * param - step * O; null: out = O
    float *out;                      // last: [rows, cols]
    float alpha, keep, step;
    int mp, np, rows, cols, tiles_c;
    unsigned first_block;
};
struct MuApplyTable { MuApply j[kMuGroup]; int n; };

template <bool LAST>
__global__ __launch_bounds__(256, 2) void mu_apply_kernel(MuApplyTable t) {
    __shared__ __attribute__((aligned(16))) char lds[MuTile<2>::kLds];
    int q = 0;
    while (q + 1 < t.n && blockIdx.x >= t.j[q + 1].first_block) ++q;
    const MuApply &p = t.j[q];
    const int b = blockIdx.x - p.first_block, r0 = b / p.tiles_c * 128, c0 = b % p.tiles_c * 128;
    f32x16 acc[2][2];
    mu_tile<2>(p.a + (size_t)r0 * 2 * p.mp, 2 * p.mp, p.b + (size_t)c0 * 2 * p.mp, 2 * p.mp, p.mp / 32, lds, acc);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int c = c0 + mu_col<2>(j);
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                f16x4 hi, lo;
                const int r = r0 + mu_row<2>(i, e4 * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = p.alpha * acc[i][j][e4 * 4 + e];
                    if (LAST) {
                        if (r + e < p.rows && c < p.cols) {
                            const size_t o = (size_t)(r + e) * p.cols + c;
                            p.out[o] = p.param ? p.keep * p.param[o] - p.step * v : v;
                        }
                    } else {
                        f16 h, l;
                        mu_split(v, h, l);
                        const size_t o = mu_off(r + e, c, 2 * p.np);
                        p.x[o] = h; p.x[o + 32] = l;
                        hi[e] = h; lo[e] = l;
                    }
                }
                if (!LAST) {
                    const size_t o = mu_off(c, r, 2 * p.mp);
                    *reinterpret_cast<f16x4 *>(p.xt + o) = hi;
                    *reinterpret_cast<f16x4 *>(p.xt + o + 32) = lo;
                }
            }
        }
}

// ---- host side -----------------------------------------------------------------------------------------------------
struct MuMat {                       // a matrix's place in the workspace
    int rows, cols, mp, np, tall, nparts, tiles, splits, steps_per;
    size_t part, u, x, xt, xt2, a, qq, w, p0, p1, slab;      // byte offsets
    size_t end;
};
static size_t mu_round(size_t v) { return (v + 255) & ~(size_t)255; }
static MuMat mu_place(int rows, int cols, bool keep_u, int steps, size_t base) {
    MuMat m{};
    m.rows = rows; m.cols = cols; m.tall = rows >= cols;
    const int s = m.tall ? cols : rows, l = m.tall ? rows : cols;
    m.mp = (s + kMuPad - 1) / kMuPad * kMuPad;
    m.np = (int)(((long)l + kMuPad - 1) / kMuPad * kMuPad);
    const long n = (long)rows * cols, want = (n + kMuPrepPer - 1) / kMuPrepPer;
    m.nparts = (int)(want < kMuPrepMax ? want : kMuPrepMax);
    // one triangle of 128 x 128 tiles; the reduction split so that a matrix alone gives about 512 workgroups, at least four
    // 32-wide steps each
    const int tb = m.mp / 128, all = m.np / 32;
    m.tiles = tb * (tb + 1) / 2;
    int splits = (512 + m.tiles - 1) / m.tiles;
    if (splits > all / 4) splits = all / 4;
    if (splits < 1) splits = 1;
    m.steps_per = (all + splits - 1) / splits;
    m.splits = (all + m.steps_per - 1) / m.steps_per;
    const size_t big = mu_round((size_t)m.mp * m.np * 4), sq = mu_round((size_t)m.mp * m.mp * 4);
    size_t o = mu_round(base);
    auto take = [&](size_t bytes) { const size_t at = o; o += mu_round(bytes); return at; };
    m.part = take((size_t)m.nparts * sizeof(double));
    m.u = keep_u ? take((size_t)n * 4) : 0;
    m.x = take(big); m.xt = take(big);
    m.xt2 = steps > kMuChain ? take(big) : 0;
    m.a = take(sq); m.qq = take(sq); m.w = take(sq); m.p0 = take(sq); m.p1 = take(sq);
    m.slab = take((size_t)m.splits * m.tiles * 128 * 128 * 4);
    m.end = o;
    return m;
}

struct MuJob {
    int rows, cols;
    const float *grad, *mom, *param;
    float *mom_out, *out;
    const float *dsigma, *dot, *sigma, *scale;
    float keep, step;
};

// all matrices of one group, phase by phase
static int mu_run_group(const MuJob *jobs, int n, bool update, float momentum, int nesterov, float grad_scale, int steps, char *ws,
                        hipStream_t st) {
    MuMat m[kMuGroup];
    const bool keep_u = update && nesterov;
    size_t at = 0;
    for (int i = 0; i < n; ++i) { m[i] = mu_place(jobs[i].rows, jobs[i].cols, keep_u, steps, at); at = m[i].end; }
    {
        MuPrepTable t{};
        t.n = n; t.momentum = momentum; t.grad_scale = grad_scale; t.nesterov = nesterov;
        unsigned blocks = 0;
        for (int i = 0; i < n; ++i) {
            MuPrep &p = t.j[i];
            p.grad = jobs[i].grad; p.mom = jobs[i].mom; p.mom_out = jobs[i].mom_out;
            p.u = keep_u ? (float *)(ws + m[i].u) : nullptr;
            p.dsigma = jobs[i].dsigma; p.dot = jobs[i].dot; p.sigma = jobs[i].sigma; p.scale = jobs[i].scale;
            p.part = (double *)(ws + m[i].part);
            p.n = (long)jobs[i].rows * jobs[i].cols;
            p.first_block = blocks;
            blocks += m[i].nparts;
        }
        hipLaunchKernelGGL(mu_prep_kernel, dim3(blocks), dim3(256), 0, st, t);
    }
    f16 *x[kMuGroup], *xt[kMuGroup], *xt_next[kMuGroup];
    {
        MuSplitTable t{};
        t.n = n;
        unsigned blocks = 0;
        for (int i = 0; i < n; ++i) {
            MuSplit &p = t.j[i];
            p.u = keep_u ? (const float *)(ws + m[i].u) : update ? jobs[i].mom_out : jobs[i].grad;
            p.part = (const double *)(ws + m[i].part); p.nparts = m[i].nparts;
            x[i] = (f16 *)(ws + m[i].x); xt[i] = (f16 *)(ws + m[i].xt); xt_next[i] = (f16 *)(ws + m[i].xt2);
            p.x = x[i]; p.xt = xt[i];
            p.rows = jobs[i].rows; p.cols = jobs[i].cols; p.mp = m[i].mp; p.np = m[i].np; p.tall = m[i].tall;
            p.first_block = blocks;
            blocks += (unsigned)((long)m[i].mp / 64 * (m[i].np / 64));
        }
        hipLaunchKernelGGL(mu_split_kernel, dim3(blocks), dim3(256), 0, st, t);
    }
    for (int done = 0; done < steps;) {
        const int chain = steps - done < kMuChain ? steps - done : kMuChain;
        {
            MuGramTable t{};
            t.n = n;
            unsigned blocks = 0, red = 0;
            for (int i = 0; i < n; ++i) {
                MuGram &p = t.j[i];
                p.x = x[i]; p.slab = (float *)(ws + m[i].slab); p.a = (f16 *)(ws + m[i].a);
                p.mp = m[i].mp; p.np = m[i].np; p.tiles = m[i].tiles; p.splits = m[i].splits; p.steps_per = m[i].steps_per;
                p.first_block = blocks; p.first_reduce = red;
                blocks += p.tiles * p.splits; red += p.tiles * 16;
            }
            hipLaunchKernelGGL(mu_gram_kernel, dim3(blocks), dim3(256), 0, st, t);
            hipLaunchKernelGGL(mu_gram_reduce_kernel, dim3(red), dim3(256), 0, st, t);
        }
        // P: the product of the chain's polynomials so far, in p0 or p1; Q of the first step IS the first P
        bool in_p0 = true;
        for (int k = 0; k < chain; ++k) {
            const bool last = k == chain - 1;
            const float sp = k == 1 ? kScaleQ : kScaleP;     // scale of the P that this step's Q multiplies
            MuSquareTable t{};
            unsigned blocks = 0;
            auto add = [&](int i, size_t a, size_t b, size_t o, float alpha) -> MuSquare & {
                MuSquare &p = t.j[t.n++];
                p.a = (const f16 *)(ws + a); p.b = (const f16 *)(ws + b); p.o = (f16 *)(ws + o); p.alpha = alpha;
                p.mp = m[i].mp;
                const int tb = p.mp / 64;
                p.tiles = tb * (tb + 1) / 2;
                p.first_block = blocks;
                blocks += p.tiles;
                return p;
            };
            auto go = [&]() {
                if (t.n) hipLaunchKernelGGL(mu_square_kernel, dim3(blocks), dim3(256), 0, st, t);
                t = MuSquareTable{};
                blocks = 0;
            };
            auto q_of = [&](int i) { return k == 0 ? m[i].p0 : m[i].qq; };
            for (int i = 0; i < n; ++i) {                    // Q = a I + b A + c A^2
                MuSquare &p = add(i, m[i].a, m[i].a, q_of(i), kMuC * kScaleQ / (kScaleA * kScaleA));
                p.z = p.a; p.zscale = kMuB * kScaleQ / kScaleA; p.diag = kMuA * kScaleQ;
            }
            go();
            for (int i = 0; i < n; ++i) {
                if (!last) add(i, q_of(i), m[i].a, m[i].w, 1.f / kScaleQ);                                     // W = Q A
                if (k > 0) add(i, m[i].qq, in_p0 ? m[i].p0 : m[i].p1, in_p0 ? m[i].p1 : m[i].p0, kScaleP / (kScaleQ * sp));   // P = Q P
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
        t.n = n;
        unsigned blocks = 0;
        const float sp = chain == 1 ? kScaleQ : kScaleP;
        for (int i = 0; i < n; ++i) {
            MuApply &p = t.j[i];
            const f16 *pp = (const f16 *)(ws + (in_p0 ? m[i].p0 : m[i].p1));
            const bool flip = done == steps && m[i].tall;    // the result in U's own layout: tile rows along its rows
            p.a = flip ? xt[i] : pp; p.b = flip ? pp : xt[i];
            p.mp = m[i].mp; p.np = m[i].np; p.rows = jobs[i].rows; p.cols = jobs[i].cols;
            p.tiles_c = (flip ? m[i].mp : m[i].np) / 128;
            p.alpha = done == steps ? 1.f / (sp * kScaleX) : 1.f / sp;
            p.x = x[i]; p.xt = xt_next[i];
            p.param = update ? jobs[i].param : nullptr; p.out = jobs[i].out; p.keep = jobs[i].keep; p.step = jobs[i].step;
            p.first_block = blocks;
            blocks += (unsigned)((long)m[i].mp / 128 * (m[i].np / 128));
        }
        if (done == steps) hipLaunchKernelGGL((mu_apply_kernel<true>), dim3(blocks), dim3(256), 0, st, t);
        else hipLaunchKernelGGL((mu_apply_kernel<false>), dim3(blocks), dim3(256), 0, st, t);
        for (int i = 0; i < n; ++i) { f16 *s = xt[i]; xt[i] = xt_next[i]; xt_next[i] = s; }
    }
    return check_launch(update ? "muon_update" : "orthogonalize");
}

static size_t mu_bytes(const mmdgan_muon_job *jobs, int n, int steps, bool keep_u) {
    size_t most = 0;
    for (int g = 0; g < n; g += kMuGroup) {
        size_t at = 0;
        for (int i = g; i < n && i < g + kMuGroup; ++i) at = mu_place(jobs[i].rows, jobs[i].cols, keep_u, steps, at).end;
        if (at > most) most = at;
    }
    return most;
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
    return MMDGAN_OK;
}

extern "C" int mmdgan_orthogonalize(const mmdgan_muon_job *jobs, int n_jobs, int steps, void *workspace, void *stream) {
    if (int rc = mu_check(jobs, n_jobs, steps, false, workspace, "orthogonalize")) return rc;
    for (int g = 0; g < n_jobs; g += kMuGroup) {
        MuJob j[kMuGroup] = {};
        int n = 0;
        for (int i = g; i < n_jobs && n < kMuGroup; ++i, ++n) {
            j[n].rows = jobs[i].rows; j[n].cols = jobs[i].cols; j[n].grad = jobs[i].grad; j[n].out = jobs[i].out;
        }
        if (int rc = mu_run_group(j, n, false, 0.f, 0, 1.f, steps, (char *)workspace, (hipStream_t)stream)) return rc;
    }
    return MMDGAN_OK;
}

extern "C" int mmdgan_muon_update(const mmdgan_muon_job *jobs, int n_jobs, float lr, float momentum, int nesterov, float weight_decay,
                                  float grad_scale, int apply_fixup, int steps, void *workspace, void *stream) {
    if (int rc = mu_check(jobs, n_jobs, steps, true, workspace, "muon_update")) return rc;
    for (int g = 0; g < n_jobs; g += kMuGroup) {
        MuJob j[kMuGroup] = {};
        int n = 0;
        for (int i = g; i < n_jobs && n < kMuGroup; ++i, ++n) {
            const mmdgan_muon_job &s = jobs[i];
            MuJob &d = j[n];
            d.rows = s.rows; d.cols = s.cols; d.grad = s.grad; d.mom = s.momentum; d.mom_out = s.momentum_out; d.param = s.param; d.out = s.out;
            if (apply_fixup && s.dsigma) { d.dsigma = s.dsigma; d.dot = s.dot; d.sigma = s.sigma; d.scale = s.scale; }
            const int big = s.rows > s.cols ? s.rows : s.cols;
            d.keep = (float)(1.0 - (double)lr * weight_decay);
            d.step = (float)((double)lr * 0.2 * sqrt((double)big));
        }
        if (int rc = mu_run_group(j, n, true, momentum, nesterov != 0, grad_scale, steps, (char *)workspace, (hipStream_t)stream)) return rc;
    }
    return MMDGAN_OK;
}
