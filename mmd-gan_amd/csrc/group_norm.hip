// Group normalisation over [N, HW, C] (NHWC), channels in G groups of D = C / G, with the following activation fused.
//
//   forward    mean, rstd = 1 / sqrt(var + eps) over the HW * D values of one image's group
//              z = (x - mean) * rstd * gamma[c] + beta[c],   y = act(z)
//   backward   dz = dy * act'(z),  xhat = (x - mean) * rstd,  M = HW * D
//              dbeta[c] = sum dz,  dgamma[c] = sum dz * xhat                        (over images and pixels)
//              dx = rstd * (gamma * dz - m1 - xhat * m2),  m1 = sum gamma dz / M,  m2 = sum gamma dz xhat / M    (per group)
//
// Bound by HBM: forward reads x and writes y, backward reads x and dy and writes dx.  What the kernels do about it:
//   gn_resident   one workgroup holds an image's channel slab (whole groups, all pixels) in registers between the sums and
//                 the apply, so every tensor moves once.  Needs C a multiple of 4, groups of a power of two up to 256 channels or of any
//                 number up to 64, and a slab of at most 256 KB (forward) / 128 KB per tensor (backward).
//   gn_partial + gn_apply   everything else: pixel chunks' sums to the workspace, then the apply pass reads x (and dy) again.
// Arithmetic on elements is in 64 bits, but for tanh and its slope: v_fma_f64 issues at the fp32 rate on this part, the kernels wait for
// memory either way, and with it the sign that relu / lrelu take is the one the exact value has and a group's own mean and variance
// cancel cleanly from dx, wherever the mean lies (kGnFar below).  The sums are formed in a fixed order, without atomics: equal inputs
// give equal bits.
#include <type_traits>
#include "common.h"

namespace mmdgan {

constexpr int kGnMaxThreads = 512;                   // 256 VGPRs per wave: at most half of them hold the slab
constexpr int kGnFwdRegs = 32, kGnBwdRegs = 16;      // float4 per thread and tensor
// ... and for slabs and groups that are no powers of two: half of it, 8 at most (ANY below)
constexpr int gn_any_regs(int regs) { return regs / 2 < 8 ? regs / 2 : 8; }
constexpr int kGnGrid = 1024;                        // workgroups of a launch: four per CU
constexpr int kGnSplitCh = 256;                      // channels of a slab in the two-pass form

struct GnArgs {
    const float *x, *dy, *gamma, *beta;
    double *stats;               // [N][G][2]: mean, rstd
    float *out;                  // y / dx
    double *part;                // backward: [rows][2][C] partial dbeta, dgamma (null: not wanted)
    double *gpart, *pivot;       // two-pass form: [N][G][P][2]; forward: [N][G]
    int N, x_batch, HW, C, G, D;
    float below;                 // the activation's slope below zero
    float eps;
    // resident: slab width, slabs, images per grid row count
    int S, slabs, rows;
    // two-pass: channels per slab, groups per slab, pieces a group is cut into, pixel chunks and pixels per chunk
    int SB, gps, pieces, chunks, chunk_px;
};

// The activation by its side below zero: 0 relu, 0.1 lrelu, 1 linear (common.h: act_fwd, the same value for every number; NaN stays NaN
// under relu too, so that an image whose statistics are spoiled shows in y as it does in dx); tanh is a template argument of the
// kernels - its code in every unrolled element costs registers the others need.
template <bool TANH> __device__ __forceinline__ float gn_act(float z, float below) {
    if (TANH) return tanhf(z);
    return !(z <= 0.f) ? z : below == 0.f ? 0.f : z * below;
}
template <bool TANH> __device__ __forceinline__ double gn_slope(double z, float below) {
    if (TANH) {
        // 1 - tanh^2 = 4 e / (1 + e)^2, e = exp(-2 |z|): one exponential and one reciprocal in 32 bits (both good to 2^-23).  In units of
        // 2^-24: 1 + e, the reciprocal and the products 8; e itself 2 + 6 |z| (z's, the constant's and the product's rounding), of
        // which tanh |z| counts: at most 9 of 1 in all, where 1 - t^2 from tanhf had 12.
        const float e = __builtin_amdgcn_exp2f(-2.88539008f * fabsf((float)z)), r = __builtin_amdgcn_rcpf(1.f + e);
        return (double)(4.f * e * r * r);
    }
    return z > 0.0 ? 1.0 : (double)below;
}
// A value that the compiler must treat as new: without it the 64-bit conversions and normalised values of the first pass over
// a thread's elements are kept across the barrier for the second (U * 16 more registers: spills from U = 8 on).
__device__ __forceinline__ void gn_fresh(float4 &v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
// Means far from zero.  E[x^2] - mean^2 in 64 bits loses (mean rstd)^2 2^-53 of the variance, nothing that counts while the mean is a
// few standard deviations, but 1e-4 at 10^6 of them and all of it for a constant group; and A x + B, below, is off by |mean| rstd 2^-53.
// - Statistics: around the group's first value k, whatever part of the group a workgroup sums, E[(x - k)^2] - E[x - k]^2 loses M 2^-53 at
//   most, k lying within sqrt(M) standard deviations of the mean.  The two-pass form always subtracts k; in the resident form that
//   subtraction shows (256x64x64x64 in groups of 4: 138 -> 142 us): it sums x itself and reads a slab once more, from L2, where a mean
//   turns out to be far (64x32x32x64 at a mean of 10^5 deviations: in groups of 8 10.0 -> 12.6 us, in groups of 2 11.6 -> 20.1).
// - Maps and the backward sums take x - c, c = the mean rounded to 32 bits where it is far, else 0.  The 32-bit difference is exact for
//   x within a factor of two of c; a value further out is sqrt(M) standard deviations away at most, and off by 2^-24 of that.
constexpr double kGnFar = 256.0;
__device__ __forceinline__ bool gn_far(double mean, double rstd) { return fabs(mean) * rstd > kGnFar; }
__device__ __forceinline__ float gn_centre(double mean, double rstd) { return gn_far(mean, rstd) ? (float)mean : 0.f; }
// (k: 0 if the first value is infinite or NaN, which then reaches mean and variance through the sums)
__device__ __forceinline__ float gn_finite(float k) { return fabsf(k) < __builtin_inff() ? k : 0.f; }
__device__ __forceinline__ void gn_subtract(float4 &v, float x, float y, float z, float w) { v.x -= x; v.y -= y; v.z -= z; v.w -= w; }
// image of x (and of stats) that output image n reads: the images beyond x_batch take the last ones again
__device__ __forceinline__ int gn_src(const GnArgs &a, int n) { return n < a.x_batch ? n : n - (a.N - a.x_batch); }

// ---- resident form ----------------------------------------------------------------------------------------------
// Thread t: float4 column t % CV of the slab, pixels t / CV, t / CV + RT, ...; CV = S / 4 and the thread count are powers of two.
// Per channel the maps are z = A x + B (A = rstd gamma, B = beta - mean A) and dx = A dz + L x + M (L = -rstd^2 m2, M = rstd (rstd mean
// m2 - m1), per group): three 64-bit multiply-adds and four registers' worth of constants per channel and group.  The backward
// sums are of dz and dz x, sum dz xhat = rstd (sum dz x - mean sum dz).
// GP: groups that a thread's four channels can belong to - 1 if D is a multiple of 4 (fewer registers, and the forward sums of the
// four are one), else 4.  An item of the reduction is a channel, or (forward, GP = 1) a column of four.
// ANY: slabs and groups that are no powers of two - columns dealt to the threads by division, those that are left over idle, sums
// through LDS from every thread instead of by shuffles.  64x8x8x320 in groups of 10: forward 6.3 us, backward 10.3 (in two passes 15.9 and
// 28.6), 64x32x32x96 in groups of 3: 15.6 and 27.7 (16.5 and 30.7); with 16 float4 per thread and more the two passes win
// (33x47x31x96: forward 14.5 us against 21.3).
// Forward, one thread of a group forms its mean and rstd, the others read them: the square roots and divisions of a thread's four
// groups, side by side, cost the registers that hold the slab (64x32x32x64 in groups of 2: 12.4 us, now 11.6).
// red: [row groups][NV][CV] doubles (ANY: [NV][T]), chan: [2][S] (backward: totals of this workgroup), stat: [2][S] (forward:
// mean and rstd, by group).
// Waves per SIMD that the registers are cut for: four where the slab's values leave room.  Four channels' own groups or tanh's slope
// beside 4 float4 of x and dy spilled (64x16x16x64 in groups of two, backward: 12.0 us with the spills, 9.2 on half of the waves).
// Forward with 8 float4 and four channels' own groups 14 to 20 registers spill; on half of the waves none do, and 256x16x16x96 in groups
// of 3 takes 15.9 us instead of 13.3 (64x32x32x64 in groups of 2: 11.6 either way).  A few more spill where the slab takes half of 256
// registers (32 float4 forward, 16 backward) and backward with 2 float4 and four channels' own groups.
constexpr int gn_waves(int U, bool bwd, bool tanh, int gp) { return (bwd ? U <= (tanh || gp == 4 ? 2 : 4) : U <= 8) ? 4 : 2; }
template <int U, bool BWD, bool TANH, int GP, bool ANY>
__global__ __launch_bounds__(kGnMaxThreads, gn_waves(U, BWD, TANH, GP)) void gn_resident_kernel(GnArgs a) {
    constexpr bool kByCol = !BWD && GP == 1;
    constexpr int NV = kByCol ? 2 : 8;
    constexpr bool kOnce = BWD && GP == 4;             // x - c kept from the sums: four c held through the barrier are too many
    extern __shared__ double gn_lds[];
    const int T = blockDim.x, t = threadIdx.x, lane = t & 63;
    const int S = a.S, CV = S >> 2, RT = T / CV, D = a.D, HW = a.HW;
    const int col = ANY ? t % CV : t & (CV - 1), row0 = !ANY || t < RT * CV ? t / CV : HW;
    const int wide = CV < 64 ? 64 : CV, RG = T / wide, rg = t / wide;
    double *red = gn_lds;
    double *chan = red + (ANY ? T * NV : RG * NV * CV);
    double *stat = chan + 2 * S;
    int *again = reinterpret_cast<int *>(chan);        // forward: whether the slab's sums are taken around its groups' first values
    // the slabs of an image share its cache lines: neighbours on one XCD (workgroups go to the eight XCDs in turn, each has its own
    // L2) and close in time - of every 8 images, slab fastest, an XCD takes an eighth
    const int group = blockIdx.x / (8 * a.slabs), in = blockIdx.x - group * 8 * a.slabs;
    const int count = (a.rows - group * 8 < 8 ? a.rows - group * 8 : 8) * a.slabs, xcd = in & 7, rest = count & 7;
    const int item = xcd * (count >> 3) + (xcd < rest ? xcd : rest) + (in >> 3);
    const int slab = item % a.slabs, row = group * 8 + item / a.slabs;
    const int c0 = slab * S + col * 4, g0 = slab * S / D;
    const int items = kByCol ? CV : S, per_group = kByCol ? D >> 2 : D;      // items, and items per group
    const int DW = ANY ? 1 : per_group < 64 ? per_group : 64;        // neighbours that one wave reduces by shuffles
    int LN = 64;                                       // ANY: lanes that share a channel (backward) or a group
    while (LN > 1 && (BWD ? S : S / D) * LN > T) LN >>= 1;
    const int per = per_group / DW;
    const float4 gv = *reinterpret_cast<const float4 *>(a.gamma + c0), bv = *reinterpret_cast<const float4 *>(a.beta + c0);
    const float ga[4] = {gv.x, gv.y, gv.z, gv.w}, be[4] = {bv.x, bv.y, bv.z, bv.w};
    const double inv_m = 1.0 / ((double)HW * D);
    if (BWD && a.part)
        for (int i = t; i < 2 * S; i += T) chan[i] = 0.0;

    for (int n = row; n < a.N; n += a.rows) {
        const int ns = gn_src(a, n);
        const float *px = a.x + (size_t)ns * HW * a.C + c0;
        const float *pd = BWD ? a.dy + (size_t)n * HW * a.C + c0 : nullptr;
        float4 vx[U], vd[BWD ? U : 1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = row0 + u * RT;
            const bool ok = r < HW;
            vx[u] = ok ? *reinterpret_cast<const float4 *>(px + (size_t)r * a.C) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (BWD) vd[u] = ok ? *reinterpret_cast<const float4 *>(pd + (size_t)r * a.C) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        double A[4], B[4], mean[GP], rstd[GP];             // mean: of x - cf
        float cf[GP];
        if (BWD) {
#pragma unroll
            for (int j = 0; j < GP; ++j) {
                const double *st = a.stats + 2 * ((size_t)ns * a.G + (c0 + j) / D);
                rstd[j] = st[1];
                cf[j] = gn_centre(st[0], rstd[j]);
                mean[j] = st[0] - (double)cf[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { A[j] = rstd[j % GP] * (double)ga[j]; B[j] = fma(-mean[j % GP], A[j], (double)be[j]); }
        }
        double s[NV], L[GP], M[GP];
#pragma unroll
        for (int k = 0; k < NV; ++k) s[k] = 0.0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float4 w = vx[u];
            if (BWD) gn_subtract(w, cf[0], cf[1 % GP], cf[2 % GP], cf[3 % GP]);
            if (kOnce) vx[u] = w;
            const float xv[4] = {w.x, w.y, w.z, w.w};
            float dv[4] = {0.f, 0.f, 0.f, 0.f};
            if (BWD) { dv[0] = vd[u].x; dv[1] = vd[u].y; dv[2] = vd[u].z; dv[3] = vd[u].w; }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = xv[j];
                if (!BWD) {
                    s[kByCol ? 0 : j] += v;
                    s[kByCol ? 1 : 4 + j] = fma(v, v, s[kByCol ? 1 : 4 + j]);
                } else {                                   // (a pixel beyond the image holds dy = 0: it adds nothing)
                    const double dz = (double)dv[j] * gn_slope<TANH>(fma(A[j], v, B[j]), a.below);
                    s[j] += dz;
                    s[(4 + j) % NV] = fma(dz, v, s[(4 + j) % NV]);
                }
            }
        }
        auto gather = [&](auto first) {                    // s to the groups' totals (forward: mean, rstd) in stat, through two barriers
            constexpr bool FIRST = decltype(first)::value;
            // lanes of a wave that hold the same column
            if (!ANY) {
                for (int o = 32; o >= CV; o >>= 1) {
#pragma unroll
                    for (int k = 0; k < NV; ++k) s[k] += __shfl_xor(s[k], o, 64);
                }
            }
            if (ANY) {
#pragma unroll
                for (int k = 0; k < NV; ++k) red[k * T + t] = s[k];
            } else if (CV >= 64 || lane < CV) {
#pragma unroll
                for (int k = 0; k < NV; ++k) red[(rg * NV + k) * CV + col] = s[k];
            }
            if (!BWD && FIRST && t == 0) *again = 0;
            __syncthreads();
            // group g of the slab, by one thread
            auto publish = [&](int g, double s1, double s2) {
                const double k = FIRST ? 0.0 : (double)gn_finite(px[g * D - col * 4]), m1 = s1 * inv_m, m2 = s2 * inv_m;
                double var = fma(-m1, m1, m2);
                if (var < 0.0) var = 0.0;
                const double rstd = 1.0 / sqrt(var + (double)a.eps);
                if (FIRST && gn_far(m1, rstd)) *again = 1;
                double *st = a.stats + 2 * ((size_t)n * a.G + g0 + g);
                st[0] = stat[g] = k + m1;
                st[1] = stat[S + g] = rstd;
            };
            if (ANY && !BWD) {                             // LN lanes share a group's RT x W values
                const int W = kByCol ? D >> 2 : D, second = kByCol ? T : 4 * T, step_r = LN / W, step_c = LN % W;
                for (int i0 = 0; i0 < S / D; i0 += T / LN) {
                    const int g = i0 + t / LN;
                    double s1 = 0.0, s2 = 0.0;
                    if (g < S / D)
                        for (int z = (t & (LN - 1)) / W, d = (t & (LN - 1)) % W; z < RT;) {
                            const int c = g * W + d, at = kByCol ? z * CV + c : (c & 3) * T + z * CV + (c >> 2);
                            s1 += red[at];
                            s2 += red[second + at];
                            z += step_r; d += step_c;
                            if (d >= W) { d -= W; ++z; }
                        }
                    for (int o = LN >> 1; o > 0; o >>= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
                    if (g < S / D && !(t & (LN - 1))) publish(g, s1, s2);
                }
            } else {
                // totals over the row groups, then over the group's items
                for (int i0 = 0; i0 < (ANY ? S : items); i0 += ANY ? T / LN : T) {
                    const int i = i0 + (ANY ? t / LN : t);
                    if (!ANY && i >= items) break;
                    const int k = kByCol ? 0 : i & 3, q = kByCol ? i : i >> 2;
                    double s1 = 0.0, s2 = 0.0;
                    if (ANY) {
                        if (i < S)
                            for (int z = t & (LN - 1); z < RT; z += LN) {
                                s1 += red[k * T + z * CV + q];
                                s2 += red[(4 + k) * T + z * CV + q];
                            }
                        for (int o = LN >> 1; o > 0; o >>= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
                        if (i >= S || (t & (LN - 1))) continue;
                    } else {
                        for (int z = 0; z < RG; ++z) {
                            s1 += red[(z * NV + k) * CV + q];
                            s2 += red[(z * NV + (kByCol ? 1 : 4) + k) * CV + q];
                        }
                    }
                    if (BWD) {
                        const double *st = a.stats + 2 * ((size_t)ns * a.G + (slab * S + i) / D);
                        s2 = st[1] * fma((double)gn_centre(st[0], st[1]) - st[0], s1, s2);
                        if (a.part && n < a.x_batch) { chan[i] += s1; chan[S + i] += s2; }
                        const double g = (double)a.gamma[slab * S + i];
                        s1 *= g; s2 *= g;
                    }
                    for (int o = DW >> 1; o > 0; o >>= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
                    if ((i & (DW - 1)) == 0) {
                        if (BWD) { stat[i / DW] = s1; stat[S + i / DW] = s2; }
                        else publish(i / DW, s1, s2);      // (forward: at most 64 items a group)
                    }
                }
            }
            __syncthreads();
        };
        gather(std::true_type());
        if (!BWD) {
            if (__builtin_expect(*again, 0)) {
                const float *p2 = px;
                int r2 = row0;
                asm volatile("" : "+v"(p2), "+v"(r2));     // (nothing computed for the first reads is kept for these)
                float pivot[GP];
#pragma unroll
                for (int j = 0; j < GP; ++j) pivot[j] = gn_finite(p2[(c0 + j) / D * D - c0]);
#pragma unroll
                for (int k = 0; k < NV; ++k) s[k] = 0.0;
                for (int r = r2; r < HW; r += RT) {
                    const float4 q = *reinterpret_cast<const float4 *>(p2 + (size_t)r * a.C);
                    const float xv[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const double d = xv[j] - (double)pivot[j % GP];
                        s[kByCol ? 0 : j] += d;
                        s[(kByCol ? 1 : 4 + j) % NV] = fma(d, d, s[(kByCol ? 1 : 4 + j) % NV]);
                    }
                }
                gather(std::false_type());
            }
#pragma unroll
            for (int j = 0; j < GP; ++j) {
                const int g = (col * 4 + j) / D;
                rstd[j] = stat[S + g];
                cf[j] = gn_centre(stat[g], rstd[j]);
                mean[j] = stat[g] - (double)cf[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { A[j] = rstd[j % GP] * (double)ga[j]; B[j] = fma(-mean[j % GP], A[j], (double)be[j]); }
        } else {
#pragma unroll
            for (int j = 0; j < GP; ++j) {
                const int g = (col * 4 + j) / D;
                if (ANY && j && g == (col * 4 + j - 1) / D) {    // (the same group as the channel before)
                    L[j] = L[j ? j - 1 : 0]; M[j] = M[j ? j - 1 : 0];
                    continue;
                }
                double s1 = 0.0, s2 = 0.0;
                for (int q = 0; q < per; ++q) { s1 += stat[g * per + q]; s2 += stat[S + g * per + q]; }
                s1 *= inv_m; s2 *= inv_m;
                L[j] = -rstd[j] * rstd[j] * s2;
                M[j] = -fma(L[j], mean[j], rstd[j] * s1);
            }
        }
        float *po = a.out + (size_t)n * HW * a.C + c0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = row0 + u * RT;
            gn_fresh(vx[u]);
            if (BWD) gn_fresh(vd[BWD ? u : 0]);
            if (!kOnce) gn_subtract(vx[u], cf[0], cf[1 % GP], cf[2 % GP], cf[3 % GP]);
            const float xv[4] = {vx[u].x, vx[u].y, vx[u].z, vx[u].w};
            float dv[4] = {0.f, 0.f, 0.f, 0.f}, o[4];
            if (BWD) { dv[0] = vd[u].x; dv[1] = vd[u].y; dv[2] = vd[u].z; dv[3] = vd[u].w; }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double v = xv[j], z = fma(A[j], v, B[j]);
                if (!BWD) o[j] = gn_act<TANH>((float)z, a.below);
                else o[j] = (float)fma(A[j], (double)dv[j] * gn_slope<TANH>(z, a.below), fma(L[j % GP], v, M[j % GP]));
            }
            if (r < HW) *reinterpret_cast<float4 *>(po + (size_t)r * a.C) = make_float4(o[0], o[1], o[2], o[3]);
        }
        if (n + a.rows < a.N) __syncthreads();         // red and stat are written again for the next image
    }
    if (BWD && a.part) {
        if (ANY) __syncthreads();
        for (int i = t; i < S; i += T) {               // (else the thread that owns item i wrote chan[i])
            double *p = a.part + (size_t)row * 2 * a.C + slab * S + i;
            p[0] = chan[i]; p[a.C] = chan[S + i];
        }
    }
}

// ---- two-pass form ----------------------------------------------------------------------------------------------
// slab: `gps` whole groups (D <= 256) or one piece of 256 channels of a group (D > 256)
struct GnSlab { int c0, width, g0, groups, piece; };
__device__ __forceinline__ GnSlab gn_slab(const GnArgs &a, int s) {
    GnSlab r;
    if (a.pieces == 1) {
        r.g0 = s * a.gps;
        r.groups = a.G - r.g0 < a.gps ? a.G - r.g0 : a.gps;
        r.c0 = r.g0 * a.D; r.width = r.groups * a.D; r.piece = 0;
    } else {
        r.g0 = s / a.pieces; r.piece = s % a.pieces; r.groups = 1;
        r.c0 = r.g0 * a.D + r.piece * kGnSplitCh;
        const int left = a.D - r.piece * kGnSplitCh;
        r.width = left < kGnSplitCh ? left : kGnSplitCh;
    }
    return r;
}

// lanes of a 256-thread workgroup that add up one of `groups` (at most 256) groups: a power of two up to a wave
__device__ __forceinline__ int gn_lanes(int groups) {
    int l = 64;
    while (l > 1 && groups * l > 256) l >>= 1;
    return l;
}
template <int VEC> __device__ __forceinline__ void gn_load(const float *p, float *v) {
    if (VEC == 4) {
        const float4 q = *reinterpret_cast<const float4 *>(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        v[0] = *p;
    }
}

template <int VEC, bool BWD, bool TANH>
__global__ __launch_bounds__(256) void gn_partial_kernel(GnArgs a) {
    constexpr int U = 4;
    __shared__ double red[2][256 * VEC];
    __shared__ double chan[2][kGnSplitCh];
    const int t = threadIdx.x;
    const int chunk = blockIdx.y, n = blockIdx.z, ns = gn_src(a, n);
    const GnSlab sl = gn_slab(a, blockIdx.x);
    const int CV = (sl.width + VEC - 1) / VEC, RT = 256 / CV, rl = t / CV, col = t % CV;
    const int p0 = chunk * a.chunk_px;                 // rows are counted from the chunk's first: p0 + chunk_px may pass an int
    const int rows = a.HW - p0 < a.chunk_px ? a.HW - p0 : a.chunk_px;
    double s1[VEC], s2[VEC], mean[VEC], rstd[VEC], ga[VEC], be[VEC];
    float pivot[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { s1[j] = 0.0; s2[j] = 0.0; }
    if (rl < RT) {
        const int c = sl.c0 + col * VEC;
        if (BWD) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const double *st = a.stats + 2 * ((size_t)ns * a.G + (c + j) / a.D);
                mean[j] = st[0]; rstd[j] = st[1]; ga[j] = a.gamma[c + j]; be[j] = a.beta[c + j];
            }
        }
        const float *px = a.x + ((size_t)ns * a.HW + p0) * a.C + c;
        if (BWD) {
            const float *pd = a.dy + ((size_t)n * a.HW + p0) * a.C + c;
            for (int r = rl; r < rows; r += RT * U) {
                float vx[U][VEC], vd[U][VEC];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int rr = r + u * RT;
                    const bool ok = rr < rows;
                    if (ok) gn_load<VEC>(px + (size_t)rr * a.C, vx[u]);
                    if (ok) gn_load<VEC>(pd + (size_t)rr * a.C, vd[u]);
                    if (!ok) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) { vx[u][j] = 0.f; vd[u][j] = 0.f; }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const double xh = ((double)vx[u][j] - mean[j]) * rstd[j];
                        const double dz = (double)vd[u][j] * gn_slope<TANH>(fma(xh, ga[j], be[j]), a.below);
                        s1[j] += dz; s2[j] = fma(dz, xh, s2[j]);
                    }
                }
            }
        } else {
            float vx[U][VEC];
            const int last = rows - 1;
            auto fetch = [&](int r) {                      // (a row beyond the chunk: its last row again)
#pragma unroll
                for (int u = 0; u < U; ++u) gn_load<VEC>(px + (size_t)(r + u * RT < last ? r + u * RT : last) * a.C, vx[u]);
            };
            int r = rl, g = sl.groups == 1 ? sl.g0 : c / a.D, f = g * a.D;     // the channel's group and that one's first channel
            fetch(r);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {                // (in flight beside the first rows)
                if (c + j == f + a.D) f += a.D;
                pivot[j] = a.x[(size_t)n * a.HW * a.C + f];
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) pivot[j] = gn_finite(pivot[j]);
            if (chunk == 0 && rl == 0) {                   // (kept for the second pass, which may write where x stands)
                f = g * a.D;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (c + j == f + a.D) { f += a.D; ++g; }
                    if (c + j == f) a.pivot[(size_t)n * a.G + g] = pivot[j];
                }
            }
            auto add = [&](int u) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const double d = (double)vx[u][j] - (double)pivot[j];
                    s1[j] += d; s2[j] = fma(d, d, s2[j]);
                }
            };
            while (r + (U - 1) * RT < rows) {
#pragma unroll
                for (int u = 0; u < U; ++u) add(u);
                r += RT * U;
                fetch(r);
            }
#pragma unroll
            for (int u = 0; u < U - 1; ++u)
                if (r + u * RT < rows) add(u);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            red[0][rl * CV * VEC + col * VEC + j] = s1[j];
            red[1][rl * CV * VEC + col * VEC + j] = s2[j];
        }
    }
    __syncthreads();
    for (int i = t; i < sl.width; i += 256) {
        double u1 = 0.0, u2 = 0.0;
        for (int q = 0; q < RT; ++q) { u1 += red[0][q * CV * VEC + i]; u2 += red[1][q * CV * VEC + i]; }
        if (BWD) {
            if (a.part && n < a.x_batch) {
                double *p = a.part + ((size_t)n * a.chunks + chunk) * 2 * a.C + sl.c0 + i;
                p[0] = u1; p[a.C] = u2;
            }
            const double g = (double)a.gamma[sl.c0 + i];
            u1 *= g; u2 *= g;
        }
        chan[0][i] = u1; chan[1][i] = u2;
    }
    __syncthreads();
    const int P = a.chunks * a.pieces, p = chunk * a.pieces + sl.piece;
    const int per = sl.groups == 1 ? sl.width : a.D;   // channels of a group in this slab
    const int lanes = gn_lanes(sl.groups), g = t / lanes, l = t & (lanes - 1);
    double u1 = 0.0, u2 = 0.0;
    if (g < sl.groups)
        for (int q = l; q < per; q += lanes) { u1 += chan[0][g * per + q]; u2 += chan[1][g * per + q]; }
    for (int o = lanes >> 1; o > 0; o >>= 1) { u1 += __shfl_xor(u1, o, 64); u2 += __shfl_xor(u2, o, 64); }
    if (g < sl.groups && l == 0) {
        double *o = a.gpart + (((size_t)n * a.G + sl.g0 + g) * P + p) * 2;
        o[0] = u1; o[1] = u2;
    }
}

template <int VEC, bool BWD, bool TANH>
__global__ __launch_bounds__(256) void gn_apply_kernel(GnArgs a) {
    constexpr int U = 4;
    __shared__ double stat[2][kGnSplitCh];             // per group of the slab: mean, rstd / m1, m2
    const int t = threadIdx.x;
    const int chunk = blockIdx.y, n = blockIdx.z, ns = gn_src(a, n);
    const GnSlab sl = gn_slab(a, blockIdx.x);
    const int CV = (sl.width + VEC - 1) / VEC, RT = 256 / CV, rl = t / CV, col = t % CV;
    const int p0 = chunk * a.chunk_px;                 // rows are counted from the chunk's first: p0 + chunk_px may pass an int
    const int rows = a.HW - p0 < a.chunk_px ? a.HW - p0 : a.chunk_px;
    const int P = a.chunks * a.pieces;
    const double inv_m = 1.0 / ((double)a.HW * a.D);
    auto publish = [&](int g, double u1, double u2, double pivot) {
        if (BWD) { stat[0][g] = u1 * inv_m; stat[1][g] = u2 * inv_m; return; }
        const double off = u1 * inv_m, mu = pivot + off;
        double var = fma(-off, off, u2 * inv_m);
        if (var < 0.0) var = 0.0;
        const double is = 1.0 / sqrt(var + (double)a.eps);
        stat[0][g] = mu; stat[1][g] = is;
        if (chunk == 0 && sl.piece == 0) {
            double *st = a.stats + 2 * ((size_t)n * a.G + sl.g0 + g);
            st[0] = mu; st[1] = is;
        }
    };
    const int c = sl.c0 + col * VEC;
    const float *px = a.x + ((size_t)ns * a.HW + p0) * a.C + c;
    const float *pd = BWD ? a.dy + ((size_t)n * a.HW + p0) * a.C + c : nullptr;
    float vx[U][VEC], vd[BWD ? U : 1][VEC];
    auto fetch = [&](int r) {                          // (a row beyond the chunk: its last row again, never used)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int rr = r + u * RT < rows ? r + u * RT : rows - 1;
            gn_load<VEC>(px + (size_t)rr * a.C, vx[u]);
            if (BWD) gn_load<VEC>(pd + (size_t)rr * a.C, vd[BWD ? u : 0]);
        }
    };
    fetch(rl);                                         // in flight while the statistics come together
    const int lanes = gn_lanes(sl.groups), mine = t / lanes, l = t & (lanes - 1);
    double u1 = 0.0, u2 = 0.0, pivot = 0.0;
    if (mine < sl.groups) {
        if (!BWD) pivot = a.pivot[(size_t)n * a.G + sl.g0 + mine];
        const double2 *q = reinterpret_cast<const double2 *>(a.gpart + ((size_t)n * a.G + sl.g0 + mine) * P * 2);
#pragma unroll 4
        for (int p = l; p < P; p += lanes) { const double2 v = q[p]; u1 += v.x; u2 += v.y; }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) { u1 += __shfl_xor(u1, o, 64); u2 += __shfl_xor(u2, o, 64); }
    if (mine < sl.groups && l == 0) publish(mine, u1, u2, pivot);
    __syncthreads();
    if (rl >= RT) return;
    double A[VEC], B[VEC], L[VEC], M[VEC];             // the maps of the resident form
    float cf[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int g = (c + j) / a.D - sl.g0;
        double mean, rstd;
        if (BWD) {
            const double *st = a.stats + 2 * ((size_t)ns * a.G + sl.g0 + g);
            mean = st[0]; rstd = st[1];
        } else {
            mean = stat[0][g]; rstd = stat[1][g];
        }
        cf[j] = gn_centre(mean, rstd);
        mean -= (double)cf[j];
        if (BWD) {
            L[j] = -rstd * rstd * stat[1][g];
            M[j] = -fma(L[j], mean, rstd * stat[0][g]);
        }
        A[j] = rstd * (double)a.gamma[c + j];
        B[j] = fma(-mean, A[j], (double)a.beta[c + j]);
    }
    float *po = a.out + ((size_t)n * a.HW + p0) * a.C + c;
    for (int r = rl; r < rows; r += RT * U) {
        if (r != rl) fetch(r);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int rr = r + u * RT;
            float o[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const double v = vx[u][j] - cf[j], z = fma(A[j], v, B[j]);
                if (!BWD) o[j] = gn_act<TANH>((float)z, a.below);
                else o[j] = (float)fma(A[j], (double)vd[BWD ? u : 0][j] * gn_slope<TANH>(z, a.below), fma(L[j], v, M[j]));
            }
            if (rr < rows) {
                if (VEC == 4) *reinterpret_cast<float4 *>(po + (size_t)rr * a.C) = make_float4(o[0], o[1 % VEC], o[2 % VEC], o[3 % VEC]);
                else po[(size_t)rr * a.C] = o[0];
            }
        }
    }
}

// dbeta[c] / dgamma[c] = sum of the partial rows, in row order per lane
__global__ __launch_bounds__(256) void gn_param_kernel(const double *part, long rows, int C, float *dgamma, float *dbeta) {
    __shared__ double red[2][32][9];
    const int cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
    const int c = blockIdx.x * 8 + cl;
    double s1 = 0.0, s2 = 0.0;
    if (c < C) {
#pragma unroll 4
        for (long r = rl; r < rows; r += 32) { s1 += part[r * 2 * C + c]; s2 += part[r * 2 * C + C + c]; }
    }
    red[0][rl][cl] = s1; red[1][rl][cl] = s2;
    __syncthreads();
    if (threadIdx.x < 16) {
        const int which = threadIdx.x >> 3, ch = blockIdx.x * 8 + cl;
        double v = 0.0;
        for (int q = 0; q < 32; ++q) v += red[which][q][cl];
        float *out = which == 0 ? dbeta : dgamma;
        if (ch < C && out) out[ch] = (float)v;
    }
}

// ---- host side --------------------------------------------------------------------------------------------------
static inline bool gn_pow2(long v) { return v > 0 && (v & (v - 1)) == 0; }

// How a geometry runs; the same for the workspace query and for the call (which may still fall back from the resident form
// when a pointer is not 16-byte aligned: the workspace covers both).
struct GnPlan {
    bool resident, any;
    int S, T, U;                 // resident: slab channels, threads, float4 per thread
    int SB, gps, pieces, slabs, chunks, chunk_px;     // two-pass
};
// regs: float4 per thread and tensor at most.  ANY form: whole groups and whole float4, multiples of `unit`, the widest of at most 64
// channels that occupies the CUs and fits.
static void gn_plan_any(long HW, int C, int D, long N, int regs, GnPlan &p) {
    const int unit = D % 4 == 0 ? D : D % 2 == 0 ? 2 * D : 4 * D, most = gn_any_regs(regs);
    p.resident = false;
    p.any = true;
    if (D > 64) return;
    for (int S = unit; S <= C && (S == unit || S <= 64); S += unit) {
        if (C % S) continue;
        long T = 64, U = 1;
        while (T < kGnMaxThreads && T * 4 < HW * (S / 4)) T *= 2;
        const long RT = T / (S / 4);
        while (U * RT < HW && U <= most) U *= 2;
        if (U > most || (p.resident && N * (C / S) < 256)) continue;
        p.resident = true;
        p.S = S; p.T = (int)T; p.U = (int)U;
    }
}
static void gn_plan_resident(long HW, int C, int D, long N, int regs, GnPlan &p) {
    p.resident = false;
    if ((C & 3) || D > kGnSplitCh) return;
    int top = 4;                                       // widest power-of-two slab that divides C
    while (top < kGnSplitCh && C % (top * 2) == 0) top *= 2;
    // ... of 4 or 8 channels reads 16 or 32 bytes of a pixel at a time: the other form's wider slabs first (64x16x16x200 in groups of one:
    // forward 12.5 -> 10.2 us, backward 27.9 -> 19.4)
    if (!gn_pow2(D) || (top < 16 && top < C)) {
        gn_plan_any(HW, C, D, N, regs, p);
        if (p.resident || !gn_pow2(D)) return;
    }
    p.any = false;
    if (top < D) return;
    const long cap = (long)kGnMaxThreads * regs;
    int least = D < 4 ? 4 : D;
    // a slab of 64 channels, down to 8 where it takes that to occupy the CUs or to hold the image (32x64x64x64 forward 28.1 us on
    // 16 channels and half of the CUs, 19.5 on 8; with 256 workgroups already, 64x32x32x64 takes 11.1 on 16 and 12.9 on 8)
    int S = top < 64 ? top : 64;
    if (S < least) S = least;
    while (S > least && S > 8 && (N * (C / S) < 256 || HW * (S / 4) > cap)) S >>= 1;
    if (HW * (S / 4) > cap) return;
    const long total = HW * (S / 4);
    long T = 64;
    while (T < S / 4) T *= 2;
    while (T < kGnMaxThreads && T * 4 < total) T *= 2;
    long U = 1;
    while (T * U < total) U *= 2;
    p.resident = true;
    p.S = S; p.T = (int)T; p.U = (int)U;
}
static void gn_plan_split(long HW, int C, int D, long N, GnPlan &p) {
    const int G = C / D;
    if (D <= kGnSplitCh) { p.gps = kGnSplitCh / D < G ? kGnSplitCh / D : G; p.pieces = 1; p.SB = p.gps * D; p.slabs = (G - 1) / p.gps + 1; }
    else { p.gps = 1; p.pieces = (D + kGnSplitCh - 1) / kGnSplitCh; p.SB = kGnSplitCh; p.slabs = G * p.pieces; }
    // pixel chunks: four workgroups per CU in all, at least 64 pixels each
    long want = (4L * 256 + N * p.slabs - 1) / (N * p.slabs), most = (HW + 63) / 64;
    if (want > most) want = most;
    if (want > 64) want = 64;
    if (want < 1) want = 1;
    p.chunk_px = (int)((HW + want - 1) / want);
    p.chunks = (int)((HW + p.chunk_px - 1) / p.chunk_px);
}
static long gn_resident_rows(long N, int slabs) {
    const long rows = kGnGrid / slabs > 1 ? kGnGrid / slabs : 1;
    return rows < N ? rows : N;
}
static size_t gn_bytes(long N, long HW, int C, int G) {
    GnPlan p;
    gn_plan_split(HW, C, C / G, N, p);
    const size_t gpart = (size_t)N * G * p.chunks * p.pieces * 2 * sizeof(double);
    const size_t part = (size_t)N * p.chunks * 2 * C * sizeof(double);      // (forward: N G first values in its place)
    return gpart + part + 256;
}

// the sizes that the entries take: an image's offsets fit an int, a batch a grid dimension
static bool gn_sizes_ok(int N, long HW, int C, int G) { return N >= 1 && HW >= 1 && C >= 1 && G >= 1 && C % G == 0 && N <= 65535 && HW <= 0x7fffffffL / C; }

static bool gn_aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <bool BWD, bool TANH, int GP, bool ANY>
static void gn_launch_resident(const GnArgs &a, const GnPlan &p, hipStream_t st) {
    const int CV = p.S / 4, wide = CV < 64 ? 64 : CV;
    const size_t lds = ((ANY ? (size_t)p.T * 8 : (size_t)(p.T / wide) * (!BWD && GP == 1 ? 2 : 8) * CV) + 4 * (size_t)p.S) * sizeof(double);
    const dim3 grid((unsigned)(a.rows * a.slabs)), block(p.T);
    constexpr int REGS = BWD ? kGnBwdRegs : kGnFwdRegs, MOST = ANY ? gn_any_regs(REGS) : REGS;      // U at most
    switch (p.U) {
        case 1: hipLaunchKernelGGL((gn_resident_kernel<1, BWD, TANH, GP, ANY>), grid, block, lds, st, a); break;
        case 2: hipLaunchKernelGGL((gn_resident_kernel<2, BWD, TANH, GP, ANY>), grid, block, lds, st, a); break;
        case 4: hipLaunchKernelGGL((gn_resident_kernel<4, BWD, TANH, GP, ANY>), grid, block, lds, st, a); break;
        case 8: if constexpr (MOST >= 8) hipLaunchKernelGGL((gn_resident_kernel<8, BWD, TANH, GP, ANY>), grid, block, lds, st, a); break;
        case 16: if constexpr (MOST >= 16) hipLaunchKernelGGL((gn_resident_kernel<16, BWD, TANH, GP, ANY>), grid, block, lds, st, a); break;
        case kGnFwdRegs: if constexpr (MOST >= kGnFwdRegs) hipLaunchKernelGGL((gn_resident_kernel<kGnFwdRegs, BWD, TANH, GP, ANY>), grid, block, lds, st, a); break;
    }
}

template <bool BWD, bool TANH>
static int gn_run(GnArgs &a, float *dgamma, float *dbeta, void *workspace, hipStream_t st, const char *what) {
    GnPlan p;
    gn_plan_resident(a.HW, a.C, a.D, a.N, BWD ? kGnBwdRegs : kGnFwdRegs, p);
    if (p.resident && !(gn_aligned(a.x) && gn_aligned(a.out) && gn_aligned(a.gamma) && gn_aligned(a.beta) && (!BWD || gn_aligned(a.dy))))
        p.resident = false;
    long part_rows;
    const bool params = BWD && (dgamma || dbeta);
    if (p.resident) {
        a.S = p.S; a.slabs = a.C / p.S;
        a.rows = (int)gn_resident_rows(a.N, a.slabs);
        part_rows = a.rows;
        a.part = params ? (double *)workspace : nullptr;
        if (p.any) {
            if constexpr (BWD) gn_launch_resident<true, TANH, 4, true>(a, p, st);            // (per channel: dgamma, dbeta)
            else if (a.D % 4 == 0) gn_launch_resident<false, TANH, 1, true>(a, p, st);
            else gn_launch_resident<false, TANH, 4, true>(a, p, st);
        } else if (a.D % 4 == 0) gn_launch_resident<BWD, TANH, 1, false>(a, p, st);
        else gn_launch_resident<BWD, TANH, 4, false>(a, p, st);
    } else {
        gn_plan_split(a.HW, a.C, a.D, a.N, p);
        a.SB = p.SB; a.gps = p.gps; a.pieces = p.pieces; a.slabs = p.slabs; a.chunks = p.chunks; a.chunk_px = p.chunk_px;
        a.gpart = (double *)workspace;
        part_rows = (long)a.x_batch * a.chunks;
        double *rest = a.gpart + (size_t)a.N * a.G * a.chunks * a.pieces * 2;
        a.pivot = BWD ? nullptr : rest;
        a.part = params ? rest : nullptr;
        const bool vec = !(a.C & 3) && (a.pieces == 1 ? !(a.SB & 3) : !(a.D & 3)) && gn_aligned(a.x) && gn_aligned(a.out) && (!BWD || gn_aligned(a.dy));
        const dim3 grid(p.slabs, p.chunks, a.N), block(256);
        if (vec) {
            hipLaunchKernelGGL((gn_partial_kernel<4, BWD, TANH>), grid, block, 0, st, a);
            hipLaunchKernelGGL((gn_apply_kernel<4, BWD, TANH>), grid, block, 0, st, a);
        } else {
            hipLaunchKernelGGL((gn_partial_kernel<1, BWD, TANH>), grid, block, 0, st, a);
            hipLaunchKernelGGL((gn_apply_kernel<1, BWD, TANH>), grid, block, 0, st, a);
        }
    }
    if (params) hipLaunchKernelGGL(gn_param_kernel, dim3((a.C - 1) / 8 + 1), dim3(256), 0, st, a.part, part_rows, a.C, dgamma, dbeta);
    return check_launch(what);
}
template <bool BWD>
static int gn_dispatch(GnArgs &a, int act, float *dgamma, float *dbeta, void *workspace, hipStream_t st, const char *what) {
    if (act == MMDGAN_ACT_TANH) return gn_run<BWD, true>(a, dgamma, dbeta, workspace, st, what);
    a.below = act == MMDGAN_ACT_RELU ? 0.f : act == MMDGAN_ACT_LRELU ? kLreluAlpha : 1.f;
    return gn_run<BWD, false>(a, dgamma, dbeta, workspace, st, what);
}
}  // namespace mmdgan

using namespace mmdgan;

#define GN_REQUIRE_GEOMETRY(what)                                                                                                    \
    MMDGAN_REQUIRE(N >= 1 && HW >= 1 && C >= 1 && G >= 1, what ": bad size N=%d HW=%ld C=%d G=%d", N, HW, C, G);                      \
    MMDGAN_REQUIRE(C % G == 0, what ": %d channels do not divide into %d groups", C, G);                                              \
    MMDGAN_REQUIRE(gn_sizes_ok(N, HW, C, G), what ": image of %ld pixels x %d channels or batch of %d is too large", HW, C, N); \
    MMDGAN_REQUIRE(!((uintptr_t)workspace & 15), what ": the workspace is not 16-byte aligned");                                       \
    MMDGAN_REQUIRE(act >= MMDGAN_ACT_LINEAR && act <= MMDGAN_ACT_TANH, what ": unknown activation %d", act)

extern "C" size_t mmdgan_gn_workspace_bytes(int N, long HW, int C, int G) {
    return gn_sizes_ok(N, HW, C, G) ? gn_bytes(N, HW, C, G) : 0;
}
extern "C" int mmdgan_gn_fwd(const float *x, int N, long HW, int C, int G, const float *gamma, const float *beta, float eps, int act,
                             float *y, double *stats, void *workspace, void *stream) {
    MMDGAN_REQUIRE(x && gamma && beta && y && stats && workspace, "gn_fwd: null pointer");
    GN_REQUIRE_GEOMETRY("gn_fwd");
    MMDGAN_REQUIRE(eps > 0.f, "gn_fwd: eps must be positive");
    const size_t bytes = (size_t)N * HW * C * 4;
    MMDGAN_REQUIRE(y == x || !spans_meet(y, bytes, x, bytes), "gn_fwd: y overlaps x without being x");
    GnArgs a{};
    a.x = x; a.gamma = gamma; a.beta = beta; a.stats = stats; a.out = y;
    a.N = a.x_batch = N; a.HW = (int)HW; a.C = C; a.G = G; a.D = C / G; a.eps = eps;
    return gn_dispatch<false>(a, act, nullptr, nullptr, workspace, (hipStream_t)stream, "gn_fwd");
}
extern "C" int mmdgan_gn_bwd(const float *x, const float *dy, int N, int x_batch, long HW, int C, int G, const float *gamma,
                             const float *beta, const double *stats, int act, float *dx, float *dgamma, float *dbeta,
                             void *workspace, void *stream) {
    MMDGAN_REQUIRE(x && dy && gamma && beta && stats && dx && workspace, "gn_bwd: null pointer");
    GN_REQUIRE_GEOMETRY("gn_bwd");
    if (x_batch == 0) x_batch = N;
    MMDGAN_REQUIRE(x_batch >= 1 && x_batch <= N && N - x_batch <= x_batch, "gn_bwd: x_batch %d for %d images", x_batch, N);
    MMDGAN_REQUIRE(dx != x || x_batch == N, "gn_bwd: dx must not be x when images of x are read twice");
    const size_t bytes = (size_t)N * HW * C * 4;
    MMDGAN_REQUIRE((dx == x || !spans_meet(dx, bytes, x, (size_t)x_batch * HW * C * 4)) && (dx == dy || !spans_meet(dx, bytes, dy, bytes)),
                   "gn_bwd: dx overlaps x or dy without being it");
    MMDGAN_REQUIRE(!dgamma || !dbeta || !spans_meet(dgamma, (size_t)C * 4, dbeta, (size_t)C * 4), "gn_bwd: dgamma overlaps dbeta");
    GnArgs a{};
    a.x = x; a.dy = dy; a.gamma = gamma; a.beta = beta; a.stats = const_cast<double *>(stats); a.out = dx;
    a.N = N; a.x_batch = x_batch; a.HW = (int)HW; a.C = C; a.G = G; a.D = C / G;
    return gn_dispatch<true>(a, act, dgamma, dbeta, workspace, (hipStream_t)stream, "gn_bwd");
}
