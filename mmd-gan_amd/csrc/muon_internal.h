// Shared by muon.hip and muon_small.hip: one matrix of an orthogonalised update, the polynomial, the tables of a launch.
#pragma once
#include "common.h"

namespace mmdgan {

constexpr int kMuGroup = 16;                 // matrices per launch (the task tables travel by value)
constexpr float kMuA = 3.4445f, kMuB = -4.7750f, kMuC = 2.0315f;

struct MuJob {
    int rows, cols;
    const float *grad, *mom, *param;         // mom, param null: orthogonalize
    float *mom_out, *out;
    const float *dsigma, *dot, *sigma, *scale;
    float keep, step;                        // out = keep * param - step * O
};
struct MuStep { float momentum, grad_scale; int nesterov, steps; };

// Which matrix of a launch a workgroup belongs to: `first` holds the matrices' first workgroups (entries beyond the last: none
// reaches them).  Kept apart from the jobs, in two cache lines at most: a search through the jobs themselves waited for one
// kernel-argument line after the other.
template <int N> struct MuFirst { unsigned first[N]; };
template <int N> __device__ __forceinline__ int mu_which(const MuFirst<N> &f, unsigned b) {
    int q = 0;
#pragma unroll
    for (int i = 1; i < N; ++i) q += b >= f.first[i] ? 1 : 0;
    return q;
}
template <int N> static void mu_close(MuFirst<N> &f, int n) {
    for (int i = n; i < N; ++i) f.first[i] = 0xffffffffu;
}

static inline size_t mu_round(size_t v) { return (v + 255) & ~(size_t)255; }

// muon_small.hip: matrices whose shorter side is at most kMuSmall
constexpr int kMuSmall = 64;
static inline bool mu_is_small(int rows, int cols) { return (rows < cols ? rows : cols) <= kMuSmall; }
size_t mu_small_bytes(int rows, int cols, bool keep_u);
void mu_small_run(const MuJob *jobs, int n, const MuStep &s, char *ws, hipStream_t st);

}  // namespace mmdgan
