// Orthogonalised updates (muon.hip) of matrices whose shorter side m is at most 64: three launches for up to eight steps, all
// products in 64 bits.
//
//   gram     U = g (+ momentum) read, U kept, partial sums of A = U U^T over pieces of the longer side n
//   chain    one workgroup per matrix: A / trace(A) (the trace is ||U||^2), up to eight steps of the polynomial on m x m matrices in
//            LDS, P = Q_steps ... Q_1 / ||U||
//   apply    out = P U, or the parameter update with it
//
// U is never normalised, so nothing is rounded before P U.  What the chain does to A's rounding errors bounds its length: along a
// direction that U hardly has, A's eigenvalue is noise, 2^-46 or so and of either sign, a step multiplies it by Q^2 <= 12, and once it
// reaches -0.1 Q grows with it and the chain diverges (32x288 of rank one, one Gram matrix for all steps: singular values up to 13 after
// 13 steps, 5e6 after 16).  Eight steps leave it at 12^8 2^-46 = 6e-6, which puts Q off by 1e-5 of itself along directions whose singular
// value is still below 3e-3: less than rounding X = P U to 32 bits does.  So X is formed, and the next eight steps start from its own
// Gram matrix.
// v_mfma_f64_16x16x4 runs at a quarter of the rate of the fp16 pairs of muon.hip per product, but these products are small: what
// counts is launches (3 instead of 21) and their latency.  The chain is one CU's work, 17 products of m^3 at 128 flop / cycle on one
// triangle's tiles with a barrier between each two: 34.7 us at m = 64, 11.6 at m = 27; beyond 64 it would grow eightfold, and the four m x m buffers would not fit LDS.  A 27x64 kernel alone takes 20 us,
// eight matrices of a width-8 net 54 (gram 9, chain 35, apply 10).
#include "muon_internal.h"

namespace mmdgan {

typedef double d4 __attribute__((ext_vector_type(4)));

constexpr int kSmRows = 64;                  // rows of n per LDS tile
constexpr int kSmPieces = 64;                // pieces of n at most: partial sums the chain adds up
constexpr int kSmChain = 8;                  // steps from one Gram matrix
constexpr int kSmGramStride = 80, kSmApplyStride = 68;   // floats: conflict-free for the operand reads of the two kernels

struct SmMat {
    MuJob j;
    MuPtr<float> u;                  // U where it is neither grad nor mom_out
    MuPtr<double> slab, p;                // [pieces][tiles][256]; [R][R]
    int m, n, mt, pieces, per;       // mt 16-wide tiles; per: rows of n in a piece (a multiple of kSmRows)
};
struct SmTable { MuFirst<kMuGroup> f; SmMat a[kMuGroup]; MuStep s; int norm; };          // norm: the Gram matrix is U's, not an iterate's
static_assert(sizeof(SmTable) <= 4096, "a launch's tables travel as kernel arguments");

__device__ __forceinline__ d4 sm_mfma(double a, double b, d4 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
// C layout of the 16 x 16 x 4 product: lane l, element i: row l / 16 + 4 i, column l % 16
__device__ __forceinline__ int sm_row(int i) { return ((threadIdx.x & 63) >> 4) + 4 * i; }
__device__ __forceinline__ int sm_col() { return threadIdx.x & 15; }

// tile number of a lower triangle -> (ti, tj)
__device__ __forceinline__ void sm_tri(int t, int &ti, int &tj) {
    ti = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
    tj = t - ti * (ti + 1) / 2;
}

// element e of rows [n0, n0 + kSmRows) of the [n, m] matrix: its index in memory (rows x cols), its place in the tile.  inv_m = 1 / m: the
// quotient is exact ((e + 1/2) / m is at least 1/128 from an integer, the product's error at most 2^-10 at e < 4096).
__device__ __forceinline__ bool sm_at(const SmMat &p, int n0, int e, float inv_m, size_t &at, int &r, int &c) {
    const bool tall = p.j.rows >= p.j.cols;
    if (tall) { r = (int)(((float)e + 0.5f) * inv_m); c = e - r * p.m; at = (size_t)n0 * p.m + e; }
    else { c = e >> 6; r = e & 63; at = (size_t)c * p.n + n0 + r; }
    return n0 + r < p.n;
}
// columns beyond m of a tile: zero (four threads a row)
template <int MT, int STRIDE> __device__ __forceinline__ void sm_clear(float (*tile)[STRIDE], int m) {
    for (int c = m + (threadIdx.x & 3); c < 16 * MT; c += 4) tile[threadIdx.x >> 2][c] = 0.f;
}

template <int MT>
__device__ void sm_gram(const SmMat &p, const MuStep &s, int piece, float (*tile)[kSmGramStride]) {
    constexpr int NT = MT * (MT + 1) / 2, PER = (NT + 3) / 4;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const int begin = piece * p.per, end = begin + p.per < p.n ? begin + p.per : p.n;
    float c0 = s.grad_scale, c1 = 0.f;
    if (p.j.dsigma) { c0 = s.grad_scale * p.j.scale[0]; c1 = s.grad_scale * (p.j.scale[0] / p.j.sigma[0]) * p.j.dot[0]; }
    d4 acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = d4{0.0, 0.0, 0.0, 0.0};
    const float inv_m = 1.f / (float)p.m;
    sm_clear<MT>(tile, p.m);                                 // (published with the first rows)
    for (int n0 = begin; n0 < end; n0 += kSmRows) {
        constexpr int L = MT * 4;                            // kSmRows * 16 MT / 256
        float g[L], d[L], m[L];
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int e = t + 256 * i;
            size_t at; int r, c;
            const bool ok = e < kSmRows * p.m && sm_at(p, n0, e, inv_m, at, r, c);
            g[i] = ok ? p.j.grad[at] : 0.f;
            d[i] = ok && p.j.dsigma ? p.j.dsigma[at] : 0.f;
            m[i] = ok && p.j.mom ? p.j.mom[at] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int e = t + 256 * i;
            size_t at; int r, c;
            if (e >= kSmRows * p.m) continue;
            const bool ok = sm_at(p, n0, e, inv_m, at, r, c);
            float u = c0 * g[i];
            if (p.j.dsigma) u -= c1 * d[i];
            if (p.j.mom) {
                const float q = __builtin_fmaf(s.momentum, m[i], u);
                u = s.nesterov ? __builtin_fmaf(s.momentum, q, u) : q;
                if (ok) { p.j.mom_out[at] = q; if (p.u) p.u[at] = u; }
            }
            tile[r][c] = ok ? u : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int q = w + 4 * i;
            if (q < NT) {
                int ti, tj;
                sm_tri(q, ti, tj);
#pragma unroll 4
                for (int k = 0; k < kSmRows; k += 4) {
                    const float *row = tile[k + (lane >> 4)];
                    acc[i] = sm_mfma((double)row[ti * 16 + (lane & 15)], (double)row[tj * 16 + (lane & 15)], acc[i]);
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int q = w + 4 * i;
        if (q < NT) *(gptr<d4>)(p.slab + ((size_t)piece * NT + q) * 256 + lane * 4) = acc[i];
    }
}
__global__ __launch_bounds__(256) void mu_small_gram_kernel(SmTable t) {
    __shared__ float tile[kSmRows][kSmGramStride];
    SmMat p;
    unsigned start;
    mu_which(t.f, t.a, blockIdx.x, p, start);
    const int piece = blockIdx.x - start;
    if (p.mt == 1) sm_gram<1>(p, t.s, piece, tile);
    else if (p.mt == 2) sm_gram<2>(p, t.s, piece, tile);
    else sm_gram<4>(p, t.s, piece, tile);
}

// x, y: symmetric [R][R + 2] in LDS (rows four banks apart: conflict-free operand reads); the product's tile (ti, tj)
template <int MT> __device__ __forceinline__ d4 sm_product(const double *x, const double *y, int ti, int tj) {
    constexpr int R = 16 * MT, ST = R + 2;
    const int lane = threadIdx.x & 63;
    const double *a = x + (ti * 16 + (lane & 15)) * ST + (lane >> 4), *b = y + (tj * 16 + (lane & 15)) * ST + (lane >> 4);
    d4 c = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int k = 0; k < R; k += 4) c = sm_mfma(a[k], b[k], c);
    return c;
}
template <int MT> __device__ __forceinline__ void sm_put(double *x, int ti, int tj, d4 v) {
    constexpr int ST = 16 * MT + 2;
    const int c = tj * 16 + sm_col();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ti * 16 + sm_row(i);
        x[r * ST + c] = v[i];
        if (ti != tj) x[c * ST + r] = v[i];
    }
}

template <int MT>
__device__ void sm_chain(const SmMat &p, int steps, bool norm, double *lds) {
    constexpr int R = 16 * MT, ST = R + 2, NT = MT * (MT + 1) / 2;
    double *A = lds, *Q = A + R * ST, *W = Q + R * ST, *P = W + R * ST;
    const int t = threadIdx.x, w = t >> 6, waves = 16;       // 1024 threads
    constexpr int PER_T = (NT * 256 + 1023) / 1024;
    double sum[PER_T];
#pragma unroll
    for (int i = 0; i < PER_T; ++i) sum[i] = 0.0;
    for (int z0 = 0; z0 < p.pieces; z0 += 8) {               // in order; eight pieces in flight
        double f[PER_T][8];
#pragma unroll
        for (int i = 0; i < PER_T; ++i)
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                const int e = t + 1024 * i;
                f[i][z] = e < NT * 256 && z0 + z < p.pieces ? p.slab[(size_t)(z0 + z) * NT * 256 + e] : 0.0;
            }
#pragma unroll
        for (int i = 0; i < PER_T; ++i)
#pragma unroll
            for (int z = 0; z < 8; ++z) sum[i] += f[i][z];
    }
#pragma unroll
    for (int i = 0; i < PER_T; ++i) {
        const int e = t + 1024 * i;
        if (e >= NT * 256) break;
        const double v = sum[i];
        int ti, tj;
        sm_tri(e >> 8, ti, tj);
        const int l = (e & 255) >> 2, r = ti * 16 + (l >> 4) + 4 * (e & 3), c = tj * 16 + (l & 15);
        A[r * ST + c] = v;
        if (ti != tj) A[c * ST + r] = v;
    }
    __syncthreads();
    double tr = (t & 63) < R ? A[(t & 63) * (ST + 1)] : 0.0;
    tr = wave_sum(tr);                                       // ||U||^2, the same in every wave
    const double inv = !norm ? 1.0 : tr > 0.0 ? 1.0 / tr : tr == 0.0 ? 0.0 : tr;
    const double psc = !norm ? 1.0 : tr > 0.0 ? 1.0 / sqrt(tr) : tr == 0.0 ? 0.0 : tr;       // (NaN stays NaN)
    __syncthreads();
    for (int e = t; e < R * R; e += blockDim.x) A[e / R * ST + e % R] *= inv;
    __syncthreads();
    for (int k = 0; k < steps; ++k) {
        const bool last = k == steps - 1;
        for (int q = w; q < NT; q += waves) {                // Q = a I + b A + c A^2 (the first one is P too)
            int ti, tj;
            sm_tri(q, ti, tj);
            d4 v = sm_product<MT>(A, A, ti, tj);
            const int c = tj * 16 + sm_col();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = ti * 16 + sm_row(i);
                v[i] = (double)kMuC * v[i] + (double)kMuB * A[r * ST + c] + (r == c ? (double)kMuA : 0.0);
            }
            sm_put<MT>(Q, ti, tj, v);
            if (k == 0) sm_put<MT>(P, ti, tj, v);
        }
        __syncthreads();
        // P = Q P waits in registers until every wave has read the old P; W = Q A goes straight to its buffer
        constexpr int PER = (2 * NT + 15) / 16;              // at 16 waves
        d4 keep[PER];
        const int nw = last ? 0 : NT, np = k > 0 ? NT : 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int q = w + waves * i;
            int ti, tj;
            if (q < np) {
                sm_tri(q, ti, tj);
                keep[i] = sm_product<MT>(Q, P, ti, tj);
            } else if (q < np + nw) {
                sm_tri(q - np, ti, tj);
                sm_put<MT>(W, ti, tj, sm_product<MT>(Q, A, ti, tj));
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int q = w + waves * i;
            if (q < np) {
                int ti, tj;
                sm_tri(q, ti, tj);
                sm_put<MT>(P, ti, tj, keep[i]);
            }
        }
        if (!last)
            for (int q = w; q < NT; q += waves) {            // A = W Q
                int ti, tj;
                sm_tri(q, ti, tj);
                sm_put<MT>(A, ti, tj, sm_product<MT>(W, Q, ti, tj));
            }
        __syncthreads();
    }
    for (int e = t; e < R * R; e += blockDim.x) p.p[e] = P[e / R * ST + e % R] * psc;
}
__global__ __launch_bounds__(1024) void mu_small_chain_kernel(SmTable t) {
    extern __shared__ double sm_lds[];
    const SmMat &p = t.a[blockIdx.x];
    if (p.mt == 1) sm_chain<1>(p, t.s.steps, t.norm, sm_lds);
    else if (p.mt == 2) sm_chain<2>(p, t.s.steps, t.norm, sm_lds);
    else sm_chain<4>(p, t.s.steps, t.norm, sm_lds);
}

template <int MT>
__device__ void sm_apply(const SmMat &p, gptr<const float> u, int n0, double *P, float (*tile)[kSmApplyStride]) {
    constexpr int R = 16 * MT, ST = R + 2, L = MT * 4;
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    const bool tall = p.j.rows >= p.j.cols;
    const float inv_m = 1.f / (float)p.m;
    float v[L];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int e = t + 256 * i;
        size_t at; int r, c;
        v[i] = e < kSmRows * p.m && sm_at(p, n0, e, inv_m, at, r, c) ? u[at] : 0.f;
    }
    double pv[R * R / 256];                                  // (every load of the workgroup in flight before the first is used)
#pragma unroll
    for (int i = 0; i < R * R / 256; ++i) pv[i] = p.p[t + 256 * i];
    sm_clear<MT>(tile, p.m);
    // this wave's 16 rows of n and all of m: (row, column) of the result in memory, its parameter before the products
    float old[MT][4];
    size_t at[MT][4];
    bool ok[MT][4];
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + w * 16 + (tall ? sm_row(i) : sm_col()), m = q * 16 + (tall ? sm_col() : sm_row(i));
            ok[q][i] = n < p.n && m < p.m;
            at[q][i] = tall ? (size_t)n * p.m + m : (size_t)m * p.n + n;
            old[q][i] = ok[q][i] && p.j.param ? p.j.param[at[q][i]] : 0.f;
        }
#pragma unroll
    for (int i = 0; i < R * R / 256; ++i) { const int e = t + 256 * i; P[e / R * ST + e % R] = pv[i]; }
#pragma unroll
    for (int i = 0; i < L; ++i) {
        const int e = t + 256 * i;
        size_t a; int r, c;
        if (e < kSmRows * p.m) { (void)sm_at(p, n0, e, inv_m, a, r, c); tile[r][c] = v[i]; }
    }
    __syncthreads();
    d4 acc[MT];
#pragma unroll
    for (int q = 0; q < MT; ++q) acc[q] = d4{0.0, 0.0, 0.0, 0.0};
#pragma unroll 2
    for (int k = 0; k < R; k += 4) {
        const double x = (double)tile[w * 16 + (lane & 15)][k + (lane >> 4)];
#pragma unroll
        for (int q = 0; q < MT; ++q) {
            const double y = P[(q * 16 + (lane & 15)) * ST + k + (lane >> 4)];
            acc[q] = tall ? sm_mfma(x, y, acc[q]) : sm_mfma(y, x, acc[q]);
        }
    }
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (ok[q][i]) p.j.out[at[q][i]] = p.j.param ? (float)((double)p.j.keep * old[q][i] - (double)p.j.step * acc[q][i]) : (float)acc[q][i];
}
__global__ __launch_bounds__(256) void mu_small_apply_kernel(SmTable t) {
    __shared__ double P[64 * 66];
    __shared__ float tile[kSmRows][kSmApplyStride];
    SmMat p;
    unsigned start;
    mu_which(t.f, t.a, blockIdx.x, p, start);
    const gptr<const float> u = p.u ? p.u.as<const float>() : p.j.mom ? p.j.mom_out.as<const float>() : (gptr<const float>)p.j.grad;
    const int n0 = (blockIdx.x - start) * kSmRows;
    if (p.mt == 1) sm_apply<1>(p, u, n0, P, tile);
    else if (p.mt == 2) sm_apply<2>(p, u, n0, P, tile);
    else sm_apply<4>(p, u, n0, P, tile);
}

// ---- host side -----------------------------------------------------------------------------------------------------
struct SmPlace { int m, n, mt, pieces, per; size_t slab, p, u, end; };
// scratch: U where it is kept, and X between two chains in the same place
static SmPlace sm_place(int rows, int cols, bool scratch, size_t base) {
    SmPlace s{};
    s.m = rows < cols ? rows : cols; s.n = rows < cols ? cols : rows;
    s.mt = s.m <= 16 ? 1 : s.m <= 32 ? 2 : 4;
    const int tiles = (s.n + kSmRows - 1) / kSmRows, most = tiles < kSmPieces ? tiles : kSmPieces;
    s.per = (tiles + most - 1) / most * kSmRows;
    s.pieces = (s.n + s.per - 1) / s.per;
    size_t o = mu_round(base);
    auto take = [&](size_t bytes) { const size_t at = o; o += mu_round(bytes); return at; };
    s.slab = take((size_t)s.pieces * (s.mt * (s.mt + 1) / 2) * 256 * sizeof(double));
    s.p = take((size_t)s.mt * s.mt * 256 * sizeof(double));
    s.u = scratch ? take((size_t)rows * cols * 4) : 0;
    s.end = o;
    return s;
}
size_t mu_small_bytes(int rows, int cols, bool keep_u, int steps) { return sm_place(rows, cols, keep_u || steps > kSmChain, 0).end; }

void mu_small_run(const MuJob *jobs, int n, const MuStep &s, char *ws, hipStream_t st) {
    SmTable t{};
    t.s = s;
    t.norm = 1;
    size_t at = 0;
    unsigned gram = 0, apply = 0, first_gram[kMuGroup] = {}, first_apply[kMuGroup] = {};
    float *x[kMuGroup];                                      // an iterate between two chains: in U's place, or where U would be
    int widest = 1;
    for (int i = 0; i < n; ++i) {
        const bool keep_u = jobs[i].mom.p && s.nesterov;
        const SmPlace pl = sm_place(jobs[i].rows, jobs[i].cols, keep_u || s.steps > kSmChain, at);
        at = pl.end;
        SmMat &p = t.a[i];
        p.j = jobs[i];
        x[i] = (float *)(ws + pl.u);
        p.u = keep_u ? x[i] : nullptr;
        p.slab = (double *)(ws + pl.slab); p.p = (double *)(ws + pl.p);
        p.m = pl.m; p.n = pl.n; p.mt = pl.mt; p.pieces = pl.pieces; p.per = pl.per;
        first_gram[i] = gram; first_apply[i] = apply;
        gram += pl.pieces; apply += (pl.n + kSmRows - 1) / kSmRows;
        if (pl.mt > widest) widest = pl.mt;
    }
    mu_close(t.f, n);
    const size_t lds = (size_t)4 * 16 * widest * (16 * widest + 2) * sizeof(double);         // up to 132 KB
    static const hipError_t allowed = hipFuncSetAttribute((const void *)mu_small_chain_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                          4 * 64 * 66 * (int)sizeof(double));
    (void)allowed;                                           // (a launch that it would have allowed reports the failure)
    for (int done = 0; done < s.steps; done += t.s.steps) {
        t.s.steps = s.steps - done < kSmChain ? s.steps - done : kSmChain;
        const bool last = done + t.s.steps == s.steps;
        for (int i = 0; i < n; ++i) t.f.first[i] = first_gram[i];
        hipLaunchKernelGGL(mu_small_gram_kernel, dim3(gram), dim3(256), 0, st, t);
        hipLaunchKernelGGL(mu_small_chain_kernel, dim3(n), dim3(1024), lds, st, t);
        for (int i = 0; i < n; ++i) {
            t.f.first[i] = first_apply[i];
            if (last) { t.a[i].j.out = jobs[i].out; t.a[i].j.param = jobs[i].param; }
            else { t.a[i].j.out = x[i]; t.a[i].j.param = nullptr; }
        }
        hipLaunchKernelGGL(mu_small_apply_kernel, dim3(apply), dim3(256), 0, st, t);
        // the next chain's U is X as it stands
        t.norm = 0;
        t.s.grad_scale = 1.f;
        for (int i = 0; i < n; ++i) {
            t.a[i].u = nullptr;
            t.a[i].j.grad = x[i]; t.a[i].j.mom = nullptr; t.a[i].j.dsigma = nullptr;
        }
    }
}
}  // namespace mmdgan
