// kernels_dropout.cu -- dropout of an array's rows or elements
// (msplat_dropout).  y = x * scale where kept, 0 where dropped; its backward
// pass is the same map on the gradient, under the same seed and step.
// A pass reads and writes four bytes per element, and one Philox block (ten
// rounds of two wide multiplications and two three-way exclusive ors) serves
// four draws.
#include <algorithm>
#include <type_traits>

#include "dropout.cuh"
#include "engine.h"

namespace msp {
namespace {

constexpr int kDropThreads = 256;

struct DropArgs {
    const float* x;
    float* y;
    long long x_stride, y_stride;
    int cols;
    unsigned threshold;
    float scale;
    unsigned long long step;
    PhiloxKeys keys;
};

// A block takes a chunk of consecutive elements: one 64-bit division finds the
// chunk's first row, and an element's row and column in the chunk come from
// 32-bit arithmetic.  (Dividing each element's 64-bit index took 34 us a pass
// over 333,337 rows of 23, of which the traffic is 10.)
constexpr int kChunkElems = 8192;

// Row of place t = (column of the chunk's first element) + (element of the
// chunk), counted from the chunk's first row.  Exact: t < cols + 8192 and, by
// `magic` = ceil(2^32 / cols) for 2 <= cols <= 8192, t * cols < 2^32.  kNoGaps:
// an element's index is its place, and no row is needed.
enum RowRule { kOneColumn, kByMagic, kWideRows, kNoGaps };
template <RowRule RULE>
using Rule = std::integral_constant<RowRule, RULE>;
template <RowRule RULE>
__device__ __forceinline__ int local_row(unsigned t, int cols, unsigned magic)
{
    return RULE == kByMagic ? (int)__umulhi(t, magic)
         : RULE == kOneColumn ? (int)t : (int)(t >= (unsigned)cols);
}

// One draw per element, any strides and alignment.  A warp takes 256
// elements; each lane draws two groups' four, and ballots turn the draws into
// a bit per element, so that every access is of 32 neighbours and not of each
// lane's own four.  Offset: the type that holds a row offset in a chunk (32
// bits for all but the widest strides); YGAPS: y's rows are apart.  40M
// elements without gaps: 54 us (5.9 TB/s), at any alignment -- a vector an access
// is no faster.  With gaps it is bound by the pipe of the draws' wide
// multiplications, which is busy two thirds of the time that the
// multiprocessors are: 333,337 rows of 23 in rows of 27, 15.2 us a pass
// (4.0 TB/s).  48 registers: 18.1 us where 78 took 21.4.
// `magic64` = ceil(2^64 / cols) divides the chunk's first index exactly while
// index * cols < 2^64; 0: plain division.
constexpr int kElemsChunk = 256 * (kDropThreads / 32);

template <RowRule RULE, typename Offset, bool YGAPS, bool FULL>
__device__ __forceinline__ void dropout_chunk(const DropArgs& a, long long i0, int cnt,
                                              unsigned magic, unsigned long long magic64)
{
    const int lane = threadIdx.x & 31;
    const int e0 = 256 * (threadIdx.x >> 5) + lane;
    long long r0 = 0;
    unsigned c0 = 0;
    if (RULE != kNoGaps) {
        r0 = magic64 ? (long long)__umul64hi((unsigned long long)i0, magic64) : i0 / a.cols;
        c0 = (unsigned)(i0 - r0 * a.cols);
    }
    const float* x = RULE == kNoGaps ? a.x + i0 + e0 : a.x + r0 * a.x_stride;
    float* y = YGAPS ? a.y + r0 * a.y_stride : a.y + i0 + e0;
    float v[8];
    Offset to[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        Offset from = 32 * k;
        to[k] = 32 * k;
        if (RULE != kNoGaps) {
            const unsigned t = c0 + e0 + 32 * k;
            const int r = local_row<RULE>(t, a.cols, magic);
            const int c = (int)(t - (unsigned)r * (unsigned)a.cols);
            from = (Offset)r * (Offset)a.x_stride + c;
            if (YGAPS) to[k] = (Offset)r * (Offset)a.y_stride + c;
        }
        v[k] = 0.f;
        if (FULL || e0 + 32 * k < cnt) v[k] = x[from];   // in flight under the draws
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint4 d = philox4x32((unsigned long long)((i0 + e0 - lane) >> 2) + 32 * h + lane,
                                   a.step, a.keys);
        const unsigned b0 = __ballot_sync(0xffffffffu, d.x >= a.threshold);
        const unsigned b1 = __ballot_sync(0xffffffffu, d.y >= a.threshold);
        const unsigned b2 = __ballot_sync(0xffffffffu, d.z >= a.threshold);
        const unsigned b3 = __ballot_sync(0xffffffffu, d.w >= a.threshold);
        // element 32 k + lane: word lane & 3 of group 8 k + lane / 4
        const unsigned word = (lane & 2 ? (lane & 1 ? b3 : b2) : (lane & 1 ? b1 : b0)) >> (lane >> 2);
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (FULL || e0 + 128 * h + 32 * k < cnt)
                y[to[4 * h + k]] = (word >> (8 * k)) & 1u ? v[4 * h + k] * a.scale : 0.f;
    }
}

template <RowRule RULE, typename Offset, bool YGAPS>
__global__ void __launch_bounds__(kDropThreads, 5)
dropout_elements_kernel(DropArgs a, long long total, unsigned magic, unsigned long long magic64)
{
    const long long chunks = (total + kElemsChunk - 1) / kElemsChunk;
    for (long long ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const long long i0 = ch * kElemsChunk;
        if (i0 + kElemsChunk <= total)
            dropout_chunk<RULE, Offset, YGAPS, true>(a, i0, kElemsChunk, magic, magic64);
        else
            dropout_chunk<RULE, Offset, YGAPS, false>(a, i0, (int)(total - i0), magic, magic64);
    }
}

// One draw per row: a block draws for its chunk's rows into shared memory,
// then streams the elements; dropped ones are not read.
// VEC: rows side by side, 16-byte alignment -- four elements an access, of at
// most two rows (with two columns too: a chunk starts at a row then, so an
// access starts at one).  1M rows of 45 at rate 0.2, both directions: 106 us
// (6.8 TB/s of the bytes of all rows; the dropped fifth is not read), against
// 292 with an element an access.
// Otherwise eight accesses of an element each are under way at once; XGAPS and
// YGAPS say whose rows are apart, Offset as above.  800,000 rows of 45 off
// alignment: 54 us (5.4 TB/s), aligned 46.
template <RowRule RULE, bool VEC, typename Offset, bool XGAPS, bool YGAPS>
__global__ void __launch_bounds__(kDropThreads)
dropout_rows_kernel(DropArgs a, long long total, unsigned magic)
{
    __shared__ float s_scale[kChunkElems / 2 + 8];   // the rows of a chunk: at least 2 columns
    const long long chunks = (total + kChunkElems - 1) / kChunkElems;
    for (long long ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const long long i0 = ch * kChunkElems;
        const long long r0 = i0 / a.cols;
        const unsigned c0 = (unsigned)(i0 - r0 * a.cols);
        const int cnt = (int)min((long long)kChunkElems, total - i0);
        const long long g0 = r0 >> 2;
        const int skip = (int)(r0 & 3);   // s_scale starts at the row of the first group
        const int rows = skip + local_row<RULE>(c0 + cnt - 1, a.cols, magic) + 1;
        __syncthreads();
        for (int g = threadIdx.x; 4 * g < rows; g += kDropThreads) {
            const uint4 d = philox4x32((unsigned long long)(g0 + g), a.step, a.keys);
            s_scale[4 * g] = d.x >= a.threshold ? a.scale : 0.f;
            s_scale[4 * g + 1] = d.y >= a.threshold ? a.scale : 0.f;
            s_scale[4 * g + 2] = d.z >= a.threshold ? a.scale : 0.f;
            s_scale[4 * g + 3] = d.w >= a.threshold ? a.scale : 0.f;
        }
        __syncthreads();
        const float* scale = s_scale + skip;
        if (VEC) {
            const float* x = a.x + i0;
            float* y = a.y + i0;
            const int vecs = cnt >> 2;
            constexpr int kU = 4;
            for (int b = threadIdx.x; b < vecs; b += kDropThreads * kU) {
                float4 v[kU];
                float f0[kU], f1[kU];
                int edge[kU];
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    const int q = b + u * kDropThreads;
                    if (q >= vecs) continue;
                    const unsigned t = c0 + 4u * q;
                    const int r = local_row<RULE>(t, a.cols, magic);
                    edge[u] = (int)((unsigned)(r + 1) * (unsigned)a.cols - t);   // elements left of row r
                    f0[u] = scale[r];
                    f1[u] = edge[u] < 4 ? scale[r + 1] : f0[u];
                    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (f0[u] != 0.f || f1[u] != 0.f) v[u] = reinterpret_cast<const float4*>(x)[q];
                }
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    const int q = b + u * kDropThreads;
                    if (q >= vecs) continue;
                    const float g1 = edge[u] > 1 ? f0[u] : f1[u], g2 = edge[u] > 2 ? f0[u] : f1[u],
                                g3 = edge[u] > 3 ? f0[u] : f1[u];
                    // a dropped value may be anything, a NaN too: no product
                    v[u].x = f0[u] != 0.f ? v[u].x * f0[u] : 0.f;
                    v[u].y = g1 != 0.f ? v[u].y * g1 : 0.f;
                    v[u].z = g2 != 0.f ? v[u].z * g2 : 0.f;
                    v[u].w = g3 != 0.f ? v[u].w * g3 : 0.f;
                    reinterpret_cast<float4*>(y)[q] = v[u];
                }
            }
            const int e = 4 * vecs + threadIdx.x;
            if (e < cnt) {
                const float f = scale[local_row<RULE>(c0 + e, a.cols, magic)];
                y[e] = f != 0.f ? x[e] * f : 0.f;
            }
            continue;
        }
        const float* x = XGAPS ? a.x + r0 * a.x_stride : a.x + i0;
        float* y = YGAPS ? a.y + r0 * a.y_stride : a.y + i0;
        constexpr int kU = 8;
        for (int e0 = threadIdx.x; e0 < cnt; e0 += kDropThreads * kU) {
            float v[kU], f[kU];
            Offset to[kU];
#pragma unroll
            for (int u = 0; u < kU; u++) {
                const int e = e0 + u * kDropThreads;
                const unsigned t = c0 + e;
                const int r = local_row<RULE>(t, a.cols, magic);
                const int c = (int)(t - (unsigned)r * (unsigned)a.cols);
                to[u] = YGAPS ? (Offset)r * (Offset)a.y_stride + c : (Offset)e;
                f[u] = e < cnt ? scale[r] : 0.f;
                v[u] = 0.f;   // a dropped value may be anything, a NaN too: no product
                if (f[u] != 0.f) v[u] = x[XGAPS ? (Offset)r * (Offset)a.x_stride + c : (Offset)e];
            }
#pragma unroll
            for (int u = 0; u < kU; u++)
                if (e0 + u * kDropThreads < cnt) y[to[u]] = v[u] * f[u];
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
        rows > (1LL << 46) / std::max(x_stride, y_stride)) {
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
    const DropArgs a{x, y, x_stride, y_stride, cols, dr.threshold, dr.scale, step, philox_keys(seed)};
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const long long total = rows * cols;
    const bool xgaps = x_stride != cols, ygaps = y_stride != cols, flat = !xgaps && !ygaps;
    const bool aligned = flat && (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const unsigned magic =
        cols >= 2 && cols <= kChunkElems ? (unsigned)(((1ULL << 32) + cols - 1) / cols) : 0u;
    auto blocks = [&](long long per) {
        return (unsigned)std::min<long long>((total + per - 1) / per, 1 << 20);
    };
    // whether a row offset within a chunk fits 32 bits
    auto narrow = [&](long long per) {
        return (per / cols + 2) * std::max(x_stride, y_stride) < 1LL << 31;
    };
    static const char* const who = "msplat_dropout";
    int rc = MSPLAT_OK;
    if (whole_rows && cols > 1) {
        auto run = [&](auto kernel) {
            rc = launch(who, kernel, blocks(kChunkElems), kDropThreads, st, a, total, magic);
        };
        auto pick = [&](auto R) {
            constexpr RowRule rule = R.value;
            if (aligned) run(dropout_rows_kernel<rule, true, int, false, false>);
            else if (flat) run(dropout_rows_kernel<rule, false, int, false, false>);
            else if (narrow(kChunkElems))
                ygaps ? run(dropout_rows_kernel<rule, false, int, true, true>)
                      : run(dropout_rows_kernel<rule, false, int, true, false>);
            else
                ygaps ? run(dropout_rows_kernel<rule, false, long long, true, true>)
                      : run(dropout_rows_kernel<rule, false, long long, true, false>);
        };
        magic ? pick(Rule<kByMagic>()) : pick(Rule<kWideRows>());
    } else {
        const bool fits = cols > 1 && total < (1LL << 62) / cols;
        const unsigned long long magic64 = fits ? ~0ULL / (unsigned)cols + 1 : 0;
        auto run = [&](auto kernel) {
            rc = launch(who, kernel, blocks(kElemsChunk), kDropThreads, st, a, total, magic, magic64);
        };
        auto pick = [&](auto R) {
            constexpr RowRule rule = R.value;
            if (narrow(kElemsChunk))
                ygaps ? run(dropout_elements_kernel<rule, int, true>)
                      : run(dropout_elements_kernel<rule, int, false>);
            else
                ygaps ? run(dropout_elements_kernel<rule, long long, true>)
                      : run(dropout_elements_kernel<rule, long long, false>);
        };
        if (flat) run(dropout_elements_kernel<kNoGaps, int, false>);
        else if (cols == 1) pick(Rule<kOneColumn>());
        else magic ? pick(Rule<kByMagic>()) : pick(Rule<kWideRows>());
    }
    return rc;
}
