// kernels_mx4.cu -- 4-bit colour records (format in mx4.cuh): pack and unpack.
#include "engine.h"
#include "mx4_rows.cuh"

namespace msp {
namespace {

// Pack and unpack move 224 bytes a Gaussian at degree 3 and are bound by
// memory: 6M Gaussians in 188 us (7.1 TB/s, reading mostly) and 201 us (6.7).
template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_pack_kernel(int n, const float* __restrict__ dc, const float* __restrict__ rest,
                void* __restrict__ records)
{
    constexpr int E = 3 * mx4_rest(DEG), P = row_pitch(E);
    __shared__ __align__(16) float s_dc[kMxThreads * 3];
    __shared__ __align__(16) float s_rest[E ? kMxThreads * P : 4];
    const long long base = (long long)blockIdx.x * kMxThreads;
    const int cnt = (int)min((long long)kMxThreads, n - base);
    if constexpr (E > 0) rows_in<E>(s_rest, rest + base * E, cnt);
    rows_in<3>(s_dc, dc + base * 3, cnt);
    rows_wait();
    __syncthreads();
    if (threadIdx.x >= cnt) return;
    float q[E + 1];
    if constexpr (E > 0) row_get<E>(s_rest + threadIdx.x * P, q);
    unsigned w[mx4_words(DEG)];
    mx4_encode<DEG>(s_dc + 3 * threadIdx.x, q, w);
    mx4_store<DEG>(records, base + threadIdx.x, w);
}

template <int DEG>
__global__ void __launch_bounds__(kMxThreads)
mx4_unpack_kernel(int n, const void* __restrict__ records, float* __restrict__ dc,
                  float* __restrict__ rest)
{
    constexpr int E = 3 * mx4_rest(DEG), P = row_pitch(E);
    __shared__ __align__(16) float s_dc[kMxThreads * 3];
    __shared__ __align__(16) float s_rest[E ? kMxThreads * P : 4];
    const long long base = (long long)blockIdx.x * kMxThreads;
    const int cnt = (int)min((long long)kMxThreads, n - base);
    if (threadIdx.x < cnt) {
        unsigned w[mx4_words(DEG)];
        mx4_load<DEG>(records, base + threadIdx.x, w);
        mx4_dc(w, s_dc + 3 * threadIdx.x);
        if constexpr (E > 0) {
            float s[3], q[E + 1];
            mx4_scales(w, s);
            mx4_codes<DEG>(w, q);
#pragma unroll
            for (int j = 0; j < E; j++) q[j] *= s[j % 3];
            row_put<E>(s_rest + threadIdx.x * P, q);
        }
    }
    rows_done();
    __syncthreads();
    if constexpr (E > 0) rows_out<E>(rest + base * E, s_rest, cnt);
    rows_out<3>(dc + base * 3, s_dc, cnt);
    rows_left();
}

}  // namespace

bool mx4_records_ok(const char* who, const void* records, int degree)
{
    if (records && ((uintptr_t)records & (mx4_align(degree) - 1)) == 0) return true;
    set_error("%s: records of degree %d must be a %d-byte aligned device pointer", who, degree,
              mx4_align(degree));
    return false;
}

}  // namespace msp

using namespace msp;

extern "C" {

int msplat_mx4_record_bytes(int degree)
{
    if (!mx4_shape_ok("msplat_mx4_record_bytes", 0, degree)) return MSPLAT_ERR_ARG;
    return 4 * mx4_words(degree);
}

int msplat_mx4_pack(int n, int degree, const float* features_dc, const float* features_rest,
                    void* records, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_pack";
    if (!mx4_shape_ok(who, n, degree)) return MSPLAT_ERR_ARG;
    if (n == 0) return MSPLAT_OK;
    if (!features_dc || (degree > 0 && !features_rest)) return mx4_null_pointer(who);
    if (!mx4_records_ok(who, records, degree)) return MSPLAT_ERR_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    int rc = MSPLAT_OK;
    with_degree(degree, [&](auto D) {
        rc = launch(who, mx4_pack_kernel<D.value>, mx4_blocks(n), kMxThreads, st, n, features_dc,
                    features_rest, records);
    });
    return rc;
}

int msplat_mx4_unpack(int n, int degree, const void* records, float* features_dc,
                      float* features_rest, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_unpack";
    if (!mx4_shape_ok(who, n, degree)) return MSPLAT_ERR_ARG;
    if (n == 0) return MSPLAT_OK;
    if (!features_dc || (degree > 0 && !features_rest)) return mx4_null_pointer(who);
    if (!mx4_records_ok(who, records, degree)) return MSPLAT_ERR_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    int rc = MSPLAT_OK;
    with_degree(degree, [&](auto D) {
        rc = launch(who, mx4_unpack_kernel<D.value>, mx4_blocks(n), kMxThreads, st, n, records,
                    features_dc, features_rest);
    });
    return rc;
}

}  // extern "C"
