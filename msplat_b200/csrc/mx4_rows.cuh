// mx4_rows.cuh -- what the kernels of the 4-bit colours share: one thread per
// Gaussian, rows of floats passing through shared memory so that global
// accesses are contiguous, and the checks of their entry points.
#pragma once
#include <type_traits>

#include "engine.h"
#include "mx4.cuh"
#include "tma.cuh"

namespace msp {

constexpr int kMxThreads = 128;

// A block's rows of E floats in shared memory (E = 3 (dc), 9, 24, 45, 72).
// The stride keeps a warp whose threads each walk their own row off each
// other's banks: the rows as they are when E is odd (one float at a time, 32
// banks), and padded by one vector when E is a multiple of four (one vector
// at a time, an odd number of vectors apart).
__host__ __device__ constexpr int row_pitch(int e) { return e % 4 ? e : e + 4; }

// A block's `cnt` rows, one after another at g, into shared memory:
// asynchronous 16-byte copies when g is aligned, so that all of them are under
// way at once; else, and for the last floats of an odd count, plain loads.
// rows_wait() before the barrier that readers need.
template <int E>
__device__ __forceinline__ void rows_in(float* sm, const float* __restrict__ g, int cnt)
{
    constexpr int P = row_pitch(E), V = E % 4 ? 1 : E / 4;
    int done = 0;
    if (((uintptr_t)g & 15) == 0) {
        const int vecs = cnt * E / 4;
#pragma unroll 4
        for (int c = threadIdx.x; c < vecs; c += kMxThreads) {
            const int at = E % 4 ? 4 * c : (c / V) * P + 4 * (c % V);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                         :: "r"(smem_addr(sm + at)), "l"(g + 4 * c) : "memory");
        }
        done = 4 * vecs;
    }
#pragma unroll 8
    for (int e = done + threadIdx.x; e < cnt * E; e += kMxThreads) sm[(e / E) * P + e % E] = g[e];
}
__device__ __forceinline__ void rows_wait()
{
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// The rows back to g, after every thread has called rows_done() and a
// barrier.  Unpadded rows of a full block leave as one bulk copy, which one
// thread starts; rows_left() before the block's shared memory is given up.
__device__ __forceinline__ void rows_done()
{
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
template <int E>
__device__ __forceinline__ void rows_out(float* __restrict__ g, const float* sm, int cnt)
{
    constexpr int P = row_pitch(E), V = E % 4 ? 1 : E / 4;
    const bool aligned = ((uintptr_t)g & 15) == 0;
    if (E % 4 && aligned && cnt == kMxThreads) {
        if (threadIdx.x == 0)
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                         :: "l"(g), "r"(smem_addr(sm)), "r"(kMxThreads * E * 4) : "memory");
    } else if (E % 4 == 0 && aligned) {
#pragma unroll 4
        for (int c = threadIdx.x; c < cnt * V; c += kMxThreads)
            reinterpret_cast<float4*>(g)[c] =
                *reinterpret_cast<const float4*>(sm + (c / V) * P + 4 * (c % V));
    } else {
#pragma unroll 4
        for (int e = threadIdx.x; e < cnt * E; e += kMxThreads) g[e] = sm[(e / E) * P + e % E];
    }
}
__device__ __forceinline__ void rows_left()
{
    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
}

// A thread's own row.
template <int E>
__device__ __forceinline__ void row_get(const float* row, float* q)
{
    if constexpr (E % 4 == 0) {
#pragma unroll
        for (int k = 0; k < E / 4; k++) {
            const float4 v = reinterpret_cast<const float4*>(row)[k];
            q[4 * k] = v.x;
            q[4 * k + 1] = v.y;
            q[4 * k + 2] = v.z;
            q[4 * k + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < E; j++) q[j] = row[j];
    }
}
template <int E>
__device__ __forceinline__ void row_put(float* row, const float* q)
{
    if constexpr (E % 4 == 0) {
#pragma unroll
        for (int k = 0; k < E / 4; k++)
            reinterpret_cast<float4*>(row)[k] =
                make_float4(q[4 * k], q[4 * k + 1], q[4 * k + 2], q[4 * k + 3]);
    } else {
#pragma unroll
        for (int j = 0; j < E; j++) row[j] = q[j];
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
