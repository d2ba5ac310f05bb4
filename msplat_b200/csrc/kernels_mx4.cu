// kernels_mx4.cu -- 4-bit colour records (format in mx4.cuh): pack, unpack,
// the colours of a batch of views from records, and the gradient of the
// coefficients.  Compiled with --fmad=false, as the projection is: a colour
// from a record has the bits that the projection computes from the unpacked
// coefficients.  One thread per Gaussian; rows of floats pass through
// shared memory so that global accesses are contiguous.
#include <type_traits>

#include "engine.h"
#include "mx4.cuh"

namespace msp {
namespace {

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

template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_pack_kernel(int n, const float* __restrict__ dc, const float* __restrict__ rest,
                void* __restrict__ records)
{
    constexpr int E = 3 * mx4_rest(DEG), PITCH = mx4_pitch<DEG>();
    __shared__ float s_dc[kMxThreads * 3];
    __shared__ float s_rest[E ? kMxThreads * PITCH : 1];
    const long long base = (long long)blockIdx.x * kMxThreads;
    const int cnt = (int)min((long long)kMxThreads, n - base);
    rows_in<3, 3>(s_dc, dc + base * 3, cnt);
    if constexpr (E > 0) rows_in<E, PITCH>(s_rest, rest + base * E, cnt);
    __syncthreads();
    if (threadIdx.x >= cnt) return;
    unsigned w[mx4_words(DEG)];
    mx4_encode<DEG>(s_dc + 3 * threadIdx.x, s_rest + threadIdx.x * (E ? PITCH : 0), w);
    mx4_store<DEG>(records, base + threadIdx.x, w);
}

template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_unpack_kernel(int n, const void* __restrict__ records, float* __restrict__ dc,
                  float* __restrict__ rest)
{
    constexpr int E = 3 * mx4_rest(DEG), PITCH = mx4_pitch<DEG>();
    __shared__ float s_dc[kMxThreads * 3];
    __shared__ float s_rest[E ? kMxThreads * PITCH : 1];
    const long long base = (long long)blockIdx.x * kMxThreads;
    const int cnt = (int)min((long long)kMxThreads, n - base);
    if (threadIdx.x < cnt) {
        unsigned w[mx4_words(DEG)];
        mx4_load<DEG>(records, base + threadIdx.x, w);
        mx4_dc(w, s_dc + 3 * threadIdx.x);
        if constexpr (E > 0) {
            float s[3];
            mx4_scales(w, s);
#pragma unroll
            for (int j = 0; j < E; j++)
                s_rest[threadIdx.x * PITCH + j] = mx4_code(w, j) * s[j % 3];
        }
    }
    __syncthreads();
    rows_out<3, 3>(dc + base * 3, s_dc, cnt);
    if constexpr (E > 0) rows_out<E, PITCH>(rest + base * E, s_rest, cnt);
}

// Views of `radii` that see Gaussian i, as bits; all of them without radii.
__device__ __forceinline__ unsigned long long views_of(const int* radii, long long i, long long n,
                                                       int views)
{
    unsigned long long seen = 0;
    for (int v = 0; v < views; v++)
        if (!radii || radii[v * n + i] > 0) seen |= 1ull << v;
    return seen;
}

template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_colors_kernel(int n, int use, const float* __restrict__ means,
                  const void* __restrict__ records, int views, const Mx4Cams cams,
                  const int* __restrict__ radii, float* __restrict__ colors)
{
    __shared__ float s_col[kMxThreads * 3];
    const int tid = threadIdx.x, lane = tid & 31, w0 = tid & ~31;
    const long long base = (long long)blockIdx.x * kMxThreads;
    const long long i = base + tid;
    const unsigned long long seen = i < n ? views_of(radii, i, n, views) : 0ull;
    float p[3] = {0.f, 0.f, 0.f}, dc[3], s[3] = {0.f, 0.f, 0.f};
    unsigned w[mx4_words(DEG)];
    if (seen) {
#pragma unroll
        for (int k = 0; k < 3; k++) p[k] = means[3 * i + k];
        mx4_load<DEG>(records, i, w);
        mx4_dc(w, dc);
        if constexpr (DEG > 0) mx4_scales(w, s);
    }
    for (int v = 0; v < views; v++) {
        const bool on = (seen >> v) & 1ull;
        if (on) {
            float d[3] = {0.f, 0.f, 0.f};
            if (use > 0) view_dir(cams.p[v], p, d);
            const ShDir D = sh_dir(d);
#pragma unroll
            for (int c = 0; c < 3; c++)
                s_col[3 * tid + c] = mx4_color<DEG>(
                    use, D, dc[c], s[c], [&](int k) { return mx4_code(w, 3 * k + c); });
        }
        const unsigned bal = __ballot_sync(0xffffffffu, on);
        __syncwarp();
        float* out = colors + (v * (long long)n + base + w0) * 3;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int e = 32 * k + lane;
            if ((bal >> (e / 3)) & 1u) out[e] = s_col[3 * w0 + e];
        }
        __syncwarp();
    }
}

// One view's colours of the visible Gaussians, into the renderer's buffer.
template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_rgb_kernel(int n, int use, const float* __restrict__ means,
               const void* __restrict__ records, float3 cam, const int* __restrict__ radii,
               float4* __restrict__ rgb)
{
    const long long i = (long long)blockIdx.x * kMxThreads + threadIdx.x;
    if (i >= n || radii[i] <= 0) return;
    const float cp[3] = {cam.x, cam.y, cam.z};
    float p[3], d[3], dc[3], s[3] = {0.f, 0.f, 0.f}, col[3];
#pragma unroll
    for (int k = 0; k < 3; k++) p[k] = means[3 * i + k];
    unsigned w[mx4_words(DEG)];
    mx4_load<DEG>(records, i, w);
    mx4_dc(w, dc);
    if constexpr (DEG > 0) mx4_scales(w, s);
    view_dir(cp, p, d);
    const ShDir D = sh_dir(d);
#pragma unroll
    for (int c = 0; c < 3; c++)
        col[c] = mx4_color<DEG>(use, D, dc[c], s[c], [&](int k) { return mx4_code(w, 3 * k + c); });
    rgb[i] = make_float4(col[0], col[1], col[2], 0.f);
}

template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_colors_backward_kernel(int n, int use, const float* __restrict__ means, int views,
                           const Mx4Cams cams, const int* __restrict__ radii,
                           const float* __restrict__ v_colors, float* __restrict__ v_dc,
                           float* __restrict__ v_rest)
{
    constexpr int B = mx4_rest(DEG), E = 3 * B, PITCH = mx4_pitch<DEG>();
    __shared__ float s_dc[kMxThreads * 3];
    __shared__ float s_rest[E ? kMxThreads * PITCH : 1];
    const long long base = (long long)blockIdx.x * kMxThreads;
    const long long i = base + threadIdx.x;
    const int cnt = (int)min((long long)kMxThreads, n - base);
    if (i < n) {
        const unsigned long long seen = views_of(radii, i, n, views);
        float gd[3] = {0.f, 0.f, 0.f}, gr[E ? E : 1];
#pragma unroll
        for (int e = 0; e < E; e++) gr[e] = 0.f;
        float p[3];
#pragma unroll
        for (int k = 0; k < 3; k++) p[k] = means[3 * i + k];
        for (int v = 0; v < views; v++) {
            if (!((seen >> v) & 1ull)) continue;
            float g[3];
#pragma unroll
            for (int c = 0; c < 3; c++) {
                g[c] = v_colors[(v * (long long)n + i) * 3 + c];
                gd[c] += g[c];
            }
            if constexpr (DEG > 0) {
                if (use > 0) {
                    float d[3], bs[24];
                    view_dir(cams.p[v], p, d);
                    sh_rest_basis(cams.p[v], p, bs);
                    sh_rest_basis4(sh_dir(d), bs + 15);
                    const int nb = mx4_rest(use);
#pragma unroll
                    for (int k = 0; k < B; k++)
                        if (k < nb)
#pragma unroll
                            for (int c = 0; c < 3; c++) gr[3 * k + c] += bs[k] * g[c];
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 3; c++) s_dc[3 * threadIdx.x + c] = MSP_SH_C0 * gd[c];
#pragma unroll
        for (int e = 0; e < E; e++) s_rest[threadIdx.x * PITCH + e] = gr[e];
    }
    __syncthreads();
    rows_out<3, 3>(v_dc + base * 3, s_dc, cnt);
    if constexpr (E > 0) rows_out<E, PITCH>(v_rest + base * E, s_rest, cnt);
}

unsigned blocks_for(int n) { return (unsigned)(((long long)n + kMxThreads - 1) / kMxThreads); }

// f(std::integral_constant) for a degree that was checked.
template <typename F>
void with_degree(int degree, F f)
{
    switch (degree) {
        case 0: f(std::integral_constant<int, 0>()); break;
        case 1: f(std::integral_constant<int, 1>()); break;
        case 2: f(std::integral_constant<int, 2>()); break;
        case 3: f(std::integral_constant<int, 3>()); break;
        default: f(std::integral_constant<int, 4>()); break;
    }
}

bool check_shape(const char* who, int n, int degree)
{
    if (n < 0 || degree < 0 || degree > kMx4MaxDegree) {
        set_error("%s: invalid shape (%d Gaussians of SH degree %d; degrees 0 to %d)", who, n,
                  degree, kMx4MaxDegree);
        return false;
    }
    return true;
}

bool check_views(const char* who, int degree, int degrees_to_use, int views, const float* cam_pos,
                 Mx4Cams* cams)
{
    if (degrees_to_use < 0 || degrees_to_use > degree || views < 0 || views > kMx4MaxViews ||
        (views > 0 && !cam_pos)) {
        set_error("%s: invalid arguments (degree %d in use of %d, %d views; up to %d views)", who,
                  degrees_to_use, degree, views, kMx4MaxViews);
        return false;
    }
    for (int v = 0; v < views; v++)
        for (int k = 0; k < 3; k++) cams->p[v][k] = cam_pos[3 * v + k];
    return true;
}

int null_pointer(const char* who)
{
    set_error("%s: null device pointer", who);
    return MSPLAT_ERR_ARG;
}

}  // namespace

bool mx4_records_ok(const char* who, const void* records, int degree)
{
    if (records && ((uintptr_t)records & (mx4_align(degree) - 1)) == 0) return true;
    set_error("%s: records of degree %d must be a %d-byte aligned device pointer", who, degree,
              mx4_align(degree));
    return false;
}

void launch_mx4_pack(int n, int degree, const float* dc, const float* rest, void* records,
                     cudaStream_t s)
{
    if (n <= 0) return;
    with_degree(degree, [&](auto D) {
        mx4_pack_kernel<D.value><<<blocks_for(n), kMxThreads, 0, s>>>(n, dc, rest, records);
    });
}

void launch_mx4_rgb(int n, int degree, int use, const float* means, const void* records,
                    const float* cam_pos, const int* radii, float4* rgb, cudaStream_t s)
{
    if (n <= 0) return;
    const float3 cam = make_float3(cam_pos[0], cam_pos[1], cam_pos[2]);
    with_degree(degree, [&](auto D) {
        mx4_rgb_kernel<D.value><<<blocks_for(n), kMxThreads, 0, s>>>(n, use, means, records, cam,
                                                                     radii, rgb);
    });
}

}  // namespace msp

using namespace msp;

extern "C" {

int msplat_mx4_record_bytes(int degree)
{
    if (!check_shape("msplat_mx4_record_bytes", 0, degree)) return MSPLAT_ERR_ARG;
    return 4 * mx4_words(degree);
}

int msplat_mx4_pack(int n, int degree, const float* features_dc, const float* features_rest,
                    void* records, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_pack";
    if (!check_shape(who, n, degree)) return MSPLAT_ERR_ARG;
    if (n == 0) return MSPLAT_OK;
    if (!features_dc || (degree > 0 && !features_rest)) return null_pointer(who);
    if (!mx4_records_ok(who, records, degree)) return MSPLAT_ERR_ARG;
    launch_mx4_pack(n, degree, features_dc, features_rest, records,
                    static_cast<cudaStream_t>(cuda_stream));
    return launched(who, 1);
}

int msplat_mx4_unpack(int n, int degree, const void* records, float* features_dc,
                      float* features_rest, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_unpack";
    if (!check_shape(who, n, degree)) return MSPLAT_ERR_ARG;
    if (n == 0) return MSPLAT_OK;
    if (!features_dc || (degree > 0 && !features_rest)) return null_pointer(who);
    if (!mx4_records_ok(who, records, degree)) return MSPLAT_ERR_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    with_degree(degree, [&](auto D) {
        mx4_unpack_kernel<D.value><<<blocks_for(n), kMxThreads, 0, st>>>(n, records, features_dc,
                                                                          features_rest);
    });
    return launched(who, 1);
}

int msplat_mx4_colors(int n, int degree, int degrees_to_use, const float* means3d,
                      const void* records, int num_views, const float* cam_pos,
                      const int32_t* radii, float* colors, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_colors";
    Mx4Cams cams;
    if (!check_shape(who, n, degree) ||
        !check_views(who, degree, degrees_to_use, num_views, cam_pos, &cams))
        return MSPLAT_ERR_ARG;
    if (n == 0 || num_views == 0) return MSPLAT_OK;
    if (!means3d || !colors) return null_pointer(who);
    if (!mx4_records_ok(who, records, degree)) return MSPLAT_ERR_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    with_degree(degree, [&](auto D) {
        mx4_colors_kernel<D.value><<<blocks_for(n), kMxThreads, 0, st>>>(
            n, degrees_to_use, means3d, records, num_views, cams, radii, colors);
    });
    return launched(who, 1);
}

int msplat_mx4_colors_backward(int n, int degree, int degrees_to_use, const float* means3d,
                               int num_views, const float* cam_pos, const int32_t* radii,
                               const float* v_colors, float* v_features_dc,
                               float* v_features_rest, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_colors_backward";
    Mx4Cams cams;
    if (!check_shape(who, n, degree) ||
        !check_views(who, degree, degrees_to_use, num_views, cam_pos, &cams))
        return MSPLAT_ERR_ARG;
    if (n == 0) return MSPLAT_OK;
    if (!means3d || (num_views > 0 && !v_colors) || !v_features_dc ||
        (degree > 0 && !v_features_rest))
        return null_pointer(who);
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    with_degree(degree, [&](auto D) {
        mx4_colors_backward_kernel<D.value><<<blocks_for(n), kMxThreads, 0, st>>>(
            n, degrees_to_use, means3d, num_views, cams, radii, v_colors, v_features_dc,
            v_features_rest);
    });
    return launched(who, 1);
}

}  // extern "C"
