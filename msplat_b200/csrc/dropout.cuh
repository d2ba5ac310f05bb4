// dropout.cuh -- the counter-based draws of dropout.  No mask is ever
// stored: whether element i is kept is a function of (seed, step, i), so the
// backward pass, another rank or another kernel recomputes it.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace msp {

// The ten round keys of a seed.  As a kernel argument they are operands of the
// rounds' logic instructions; stepping them in the kernel took 20 of the 144
// instructions of four elements.
struct PhiloxKeys {
    unsigned k[10][2];
};
__host__ __device__ inline PhiloxKeys philox_keys(unsigned long long seed)
{
    PhiloxKeys K;
    for (unsigned r = 0; r < 10; r++) {
        K.k[r][0] = (unsigned)seed + r * 0x9E3779B9u;
        K.k[r][1] = (unsigned)(seed >> 32) + r * 0xBB67AE85u;
    }
    return K;
}

// Philox4x32-10 of Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
// as easy as 1, 2, 3" (SC 2011): four 32-bit draws of counter
// (group, step) under the keys of the seed.
__device__ __forceinline__ uint4 philox4x32(unsigned long long group, unsigned long long step,
                                            const PhiloxKeys& K)
{
    unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32);
    unsigned c2 = (unsigned)step, c3 = (unsigned)(step >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned long long p = (unsigned long long)c0 * 0xD2511F53u;
        const unsigned long long q = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(q >> 32) ^ c1 ^ K.k[r][0];
        c1 = (unsigned)q;
        c2 = (unsigned)(p >> 32) ^ c3 ^ K.k[r][1];
        c3 = (unsigned)p;
    }
    return make_uint4(c0, c1, c2, c3);
}

// Draw i is word i mod 4 of group i / 4.
__device__ __forceinline__ unsigned dropout_draw(unsigned long long i, unsigned long long step,
                                                 unsigned long long seed)
{
    const uint4 d = philox4x32(i >> 2, step, philox_keys(seed));
    const unsigned k = (unsigned)i & 3u;
    return k == 0 ? d.x : k == 1 ? d.y : k == 2 ? d.z : d.w;
}

// A rate as the kernels use it: an element is dropped when its draw is
// below `threshold`, so that the rate in effect is threshold / 2^32 and the
// kept values' factor is one over the rest of it, exactly to one rounding.
struct DropoutRate {
    unsigned threshold;
    float scale;
};

// False for a rate outside [0, 1) (a NaN too) or one that rounds to 1.
inline bool dropout_rate(double rate, DropoutRate* out)
{
    if (!(rate >= 0.0 && rate < 1.0)) return false;
    const double t = __builtin_rint(rate * 4294967296.0);
    if (t >= 4294967296.0) return false;
    out->threshold = (unsigned)t;
    out->scale = (float)(4294967296.0 / (4294967296.0 - t));
    return true;
}

}  // namespace msp
