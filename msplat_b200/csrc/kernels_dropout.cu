// kernels_dropout.cu -- dropout of an array's rows or elements
// (msplat_dropout).  y = x * scale where kept, 0 where dropped; its backward
// pass is the same map on the gradient, under the same seed and step.
// A pass reads and writes four bytes per element, and one Philox block
// (about 60 integer operations) serves four draws.
#include <algorithm>

#include "dropout.cuh"
#include "engine.h"

namespace msp {
namespace {

constexpr int kDropThreads = 256;

struct DropArgs {
    const float* x;
    float* y;
    long long rows, x_stride, y_stride;
    int cols;
    unsigned threshold;
    float scale;
    unsigned long long seed, step;
};

// One draw per element.  A thread takes the four elements of one Philox
// group, which lie side by side in the array when it has no gaps (FLAT);
// VEC: 16-byte accesses.
template <bool FLAT, bool VEC>
__global__ void __launch_bounds__(kDropThreads)
dropout_elements_kernel(DropArgs a, long long total)
{
    const long long groups = (total + 3) >> 2;
    for (long long g = blockIdx.x * (long long)kDropThreads + threadIdx.x; g < groups;
         g += (long long)gridDim.x * kDropThreads) {
        const long long i0 = g << 2;
        const uint4 d = philox4x32((unsigned long long)g, a.step, a.seed);
        const unsigned u[4] = {d.x, d.y, d.z, d.w};
        if (VEC && i0 + 4 <= total) {
            float4 v = *reinterpret_cast<const float4*>(a.x + i0);
            v.x = u[0] >= a.threshold ? v.x * a.scale : 0.f;
            v.y = u[1] >= a.threshold ? v.y * a.scale : 0.f;
            v.z = u[2] >= a.threshold ? v.z * a.scale : 0.f;
            v.w = u[3] >= a.threshold ? v.w * a.scale : 0.f;
            *reinterpret_cast<float4*>(a.y + i0) = v;
            continue;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const long long i = i0 + k;
            if (i >= total) break;
            long long ix = i, iy = i;
            if (!FLAT) {
                const long long r = i / a.cols, c = i - r * a.cols;
                ix = r * a.x_stride + c;
                iy = r * a.y_stride + c;
            }
            a.y[iy] = u[k] >= a.threshold ? a.x[ix] * a.scale : 0.f;
        }
    }
}

// One draw per row.  A block draws for kDropRows rows, then streams them.
constexpr int kDropRows = 128;
__global__ void __launch_bounds__(kDropThreads)
dropout_rows_kernel(DropArgs a)
{
    __shared__ float s_scale[kDropRows];
    const long long chunks = (a.rows + kDropRows - 1) / kDropRows;
    for (long long ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const long long r0 = ch * kDropRows;
        const int cnt = (int)min((long long)kDropRows, a.rows - r0);
        __syncthreads();
        if (threadIdx.x < kDropRows / 4) {
            const uint4 d = philox4x32((unsigned long long)(r0 >> 2) + threadIdx.x, a.step, a.seed);
            s_scale[4 * threadIdx.x] = d.x >= a.threshold ? a.scale : 0.f;
            s_scale[4 * threadIdx.x + 1] = d.y >= a.threshold ? a.scale : 0.f;
            s_scale[4 * threadIdx.x + 2] = d.z >= a.threshold ? a.scale : 0.f;
            s_scale[4 * threadIdx.x + 3] = d.w >= a.threshold ? a.scale : 0.f;
        }
        __syncthreads();
        const long long total = (long long)cnt * a.cols;
        for (long long e = threadIdx.x; e < total; e += kDropThreads) {
            const int r = (int)(e / a.cols);
            const int c = (int)(e - (long long)r * a.cols);
            const float f = s_scale[r];   // a dropped value may be anything, a NaN too: no product
            a.y[(r0 + r) * a.y_stride + c] = f != 0.f ? a.x[(r0 + r) * a.x_stride + c] * f : 0.f;
        }
    }
}

}  // namespace
}  // namespace msp

using namespace msp;

extern "C" int msplat_dropout(long long rows, int cols, const float* x, long long x_stride,
                              float* y, long long y_stride, double rate, unsigned long long seed,
                              unsigned long long step, int whole_rows, void* cuda_stream)
{
    if (x_stride == 0) x_stride = cols;
    if (y_stride == 0) y_stride = cols;
    if (rows < 0 || cols < 1 || x_stride < cols || y_stride < cols ||
        rows > (1LL << 60) / std::max(x_stride, y_stride)) {
        set_error("msplat_dropout: invalid shape (%lld rows of %d, strides %lld and %lld)", rows,
                  cols, x_stride, y_stride);
        return MSPLAT_ERR_ARG;
    }
    DropoutRate dr;
    if (!dropout_rate(rate, &dr)) {
        set_error("msplat_dropout: the rate must be in [0, 1), not %g", rate);
        return MSPLAT_ERR_ARG;
    }
    if (rows == 0) return MSPLAT_OK;
    if (!x || !y || (x == y && x_stride != y_stride)) {
        set_error("msplat_dropout: %s", !x || !y ? "null device pointer"
                                                 : "in place needs the same row stride twice");
        return MSPLAT_ERR_ARG;
    }
    const DropArgs a{x, y, rows, x_stride, y_stride, cols, dr.threshold, dr.scale, seed, step};
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    if (whole_rows && cols > 1) {
        const long long chunks = (rows + kDropRows - 1) / kDropRows;
        dropout_rows_kernel<<<(unsigned)std::min<long long>(chunks, 1 << 20), kDropThreads, 0, st>>>(a);
    } else {
        const long long total = rows * cols;
        const bool flat = x_stride == cols && y_stride == cols;
        const bool vec = flat && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
        const unsigned blocks = (unsigned)std::min<long long>(
            ((total + 3) / 4 + kDropThreads - 1) / kDropThreads, 1 << 20);
        if (vec) dropout_elements_kernel<true, true><<<blocks, kDropThreads, 0, st>>>(a, total);
        else if (flat) dropout_elements_kernel<true, false><<<blocks, kDropThreads, 0, st>>>(a, total);
        else dropout_elements_kernel<false, false><<<blocks, kDropThreads, 0, st>>>(a, total);
    }
    return launched("msplat_dropout", 1);
}
