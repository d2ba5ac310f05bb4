// mx4_rows.cuh -- what the kernels of the 4-bit colours share: one thread per
// Gaussian, rows of floats passing through shared memory so that global
// accesses are contiguous, and the checks of their entry points.
#pragma once
#include <type_traits>

#include "engine.h"
#include "mx4.cuh"

namespace msp {

constexpr int kMxThreads = 128;

// Row stride in shared memory: odd, so that the threads of a warp, each on
// its own row, meet 32 different banks.
template <int DEG>
__host__ __device__ constexpr int mx4_pitch() { return (3 * mx4_rest(DEG)) | 1; }

// Copies `cnt` rows of E floats between global and (padded) shared rows.
template <int E, int PITCH>
__device__ __forceinline__ void rows_in(float* sm, const float* g, int cnt)
{
    for (int e = threadIdx.x; e < cnt * E; e += kMxThreads) {
        const int r = e / E;
        sm[r * PITCH + (e - r * E)] = g[e];
    }
}
template <int E, int PITCH>
__device__ __forceinline__ void rows_out(float* g, const float* sm, int cnt)
{
    for (int e = threadIdx.x; e < cnt * E; e += kMxThreads) {
        const int r = e / E;
        g[e] = sm[r * PITCH + (e - r * E)];
    }
}

inline unsigned mx4_blocks(int n) { return (unsigned)(((long long)n + kMxThreads - 1) / kMxThreads); }

// f(std::integral_constant) for a degree that was checked.
template <typename F>
inline void with_degree(int degree, F f)
{
    switch (degree) {
        case 0: f(std::integral_constant<int, 0>()); break;
        case 1: f(std::integral_constant<int, 1>()); break;
        case 2: f(std::integral_constant<int, 2>()); break;
        case 3: f(std::integral_constant<int, 3>()); break;
        default: f(std::integral_constant<int, 4>()); break;
    }
}

inline bool mx4_shape_ok(const char* who, int n, int degree)
{
    if (n < 0 || degree < 0 || degree > kMx4MaxDegree) {
        set_error("%s: invalid shape (%d Gaussians of SH degree %d; degrees 0 to %d)", who, n,
                  degree, kMx4MaxDegree);
        return false;
    }
    return true;
}

inline int mx4_null_pointer(const char* who)
{
    set_error("%s: null device pointer", who);
    return MSPLAT_ERR_ARG;
}

}  // namespace msp
