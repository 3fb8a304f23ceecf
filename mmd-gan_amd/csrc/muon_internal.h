// Shared by muon.hip and muon_small.hip: one matrix of an orthogonalised update, the polynomial, the tables of a launch.
#pragma once
#include "common.h"

namespace mmdgan {

constexpr int kMuGroup = 16;                 // matrices per launch (the task tables travel by value)
constexpr float kMuA = 3.4445f, kMuB = -4.7750f, kMuC = 2.0315f;

// A pointer in a job.  Taken from a table by an index that is not a constant, a pointer may point anywhere as far as the compiler knows
// and is read through flat accesses, which count as LDS traffic too: every LDS wait would wait for them.
template <typename T> using gptr = __attribute__((address_space(1))) T *;
template <typename T> struct MuPtr {
    T *p;
    MuPtr &operator=(T *q) { p = q; return *this; }
    __device__ __forceinline__ operator gptr<T>() const { return (gptr<T>)p; }
    template <typename U> __device__ __forceinline__ gptr<U> as() const { return (gptr<U>)(gptr<T>)p; }
};

struct MuJob {
    int rows, cols;
    MuPtr<const float> grad, mom, param;     // mom, param null: orthogonalize
    MuPtr<float> mom_out, out;
    MuPtr<const float> dsigma, dot, sigma, scale;
    float keep, step;                        // out = keep * param - step * O
};
struct MuStep { float momentum, grad_scale; int nesterov, steps; };

// Which matrix of a launch a workgroup belongs to: `first` holds the matrices' first workgroups (entries beyond the last: none
// reaches them).  Kept apart from the jobs, in two cache lines at most: a search through the jobs themselves waited for one
// kernel-argument line after the other.
template <int N> struct MuFirst { unsigned first[N]; };
// The job of workgroup b: itself in `job`, its first workgroup in `start`.  `first` (a lane each) and job 0 (the largest matrix:
// the launch ends with it) are asked for together - a chain of scalar compares waited for kernel arguments three times before the
// first load of data, 0.8 us of a launch that is over in 5.
typedef unsigned mu_s16 __attribute__((ext_vector_type(16)));
template <typename T, int N, int M> __device__ __forceinline__ void mu_which(const MuFirst<N> &f, const T (&j)[M], unsigned b, T &job, unsigned &start) {
    typedef mu_s16 __attribute__((may_alias, aligned(4))) line;
    constexpr int W = (sizeof(T) + 63) / 64;
    static_assert(N <= 64 && W <= 3 && sizeof(T) * M >= 64 * W, "whole lines, inside the table");
    const unsigned mine = f.first[threadIdx.x & (N - 1)];
    const line *l = reinterpret_cast<const line *>(&j[0]);
    mu_s16 w[3] = {l[0], W > 1 ? l[1] : mu_s16{}, W > 2 ? l[2] : mu_s16{}};
    const int q = __popcll(__ballot(b >= mine) & (N == 64 ? ~0ull : (1ull << (N & 63)) - 1)) - 1;
    start = __builtin_amdgcn_readlane(mine, q);
    if (W == 1) asm volatile("" : "+s"(w[0]));
    else if (W == 2) asm volatile("" : "+s"(w[0]), "+s"(w[1]));
    else asm volatile("" : "+s"(w[0]), "+s"(w[1]), "+s"(w[2]));
    if (q) job = j[q];
    else __builtin_memcpy(&job, w, sizeof(T));
}
template <int N> static void mu_close(MuFirst<N> &f, int n) {
    for (int i = n; i < N; ++i) f.first[i] = 0xffffffffu;
}

static inline size_t mu_round(size_t v) { return (v + 255) & ~(size_t)255; }

// muon_small.hip: matrices whose shorter side is at most kMuSmall
constexpr int kMuSmall = 64;
static inline bool mu_is_small(int rows, int cols) { return (rows < cols ? rows : cols) <= kMuSmall; }
size_t mu_small_bytes(int rows, int cols, bool keep_u, int steps);
void mu_small_run(const MuJob *jobs, int n, const MuStep &s, char *ws, hipStream_t st);

}  // namespace mmdgan
