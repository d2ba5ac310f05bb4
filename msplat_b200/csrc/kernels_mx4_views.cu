// kernels_mx4_views.cu -- the colours of a batch of views from 4-bit records
// (format in mx4.cuh) and the gradient of the coefficients.  Compiled with FMA
// contraction: a fused multiply-add per coefficient and view is what bounds
// many views.  (A rendered view's colours come from the projection, kernels_fwd.cu,
// and have its bits.)
#include <algorithm>

#include "mx4_rows.cuh"

namespace msp {
namespace {

// Unit direction from a camera to a mean: the hardware's reciprocal square
// root (2^-22.9) and one Newton step.  IEEE root and division, as the
// projection has them, are a third of a view's instructions.
__device__ __forceinline__ void unit_dir(const float* cam, const float p[3], float d[3])
{
    const float d0 = p[0] - cam[0], d1 = p[1] - cam[1], d2 = p[2] - cam[2];
    const float n = fmaf(d2, d2, fmaf(d1, d1, d0 * d0));
    float r;
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(n));
    r = fmaf(0.5f * r, fmaf(-(n * r), r, 1.f), r);
    d[0] = d0 * r;
    d[1] = d1 * r;
    d[2] = d2 * r;
}

// SH basis values beside dc of degrees 1 to DEG (sh_to_color's convention).
template <int DEG>
__device__ __forceinline__ void sh_basis(const float d[3], float* b)
{
    if constexpr (DEG == 0) return;
    const float x = d[0], y = d[1], z = d[2];
    b[0] = -MSP_SH_C1 * y;
    b[1] = MSP_SH_C1 * z;
    b[2] = -MSP_SH_C1 * x;
    if constexpr (DEG >= 2) {
        const float xx = x * x, yy = y * y, zz = z * z, xy = x * y, yz = y * z, xz = x * z;
        const float xmy = xx - yy;
        b[3] = kSH_C2[0] * xy;
        b[4] = kSH_C2[1] * yz;
        b[5] = kSH_C2[2] * (fmaf(2.f, zz, -xx) - yy);
        b[6] = kSH_C2[3] * xz;
        b[7] = kSH_C2[4] * xmy;
        if constexpr (DEG >= 3) {
            const float u = fmaf(3.f, xx, -yy), v = fmaf(-3.f, yy, xx), w = fmaf(4.f, zz, -xx) - yy;
            b[8] = kSH_C3[0] * y * u;
            b[9] = kSH_C3[1] * xy * z;
            b[10] = kSH_C3[2] * y * w;
            b[11] = kSH_C3[3] * z * fmaf(2.f, zz, -3.f * (xx + yy));
            b[12] = kSH_C3[4] * x * w;
            b[13] = kSH_C3[5] * z * xmy;
            b[14] = kSH_C3[6] * x * v;
            if constexpr (DEG >= 4) {
                const float s = fmaf(7.f, zz, -1.f), t = fmaf(7.f, zz, -3.f);
                b[15] = kSH_C4[0] * xy * xmy;
                b[16] = kSH_C4[1] * yz * u;
                b[17] = kSH_C4[2] * xy * s;
                b[18] = kSH_C4[3] * yz * t;
                b[19] = kSH_C4[4] * fmaf(zz, fmaf(35.f, zz, -30.f), 3.f);
                b[20] = kSH_C4[5] * xz * t;
                b[21] = kSH_C4[6] * xmy * s;
                b[22] = kSH_C4[7] * xz * v;
                b[23] = kSH_C4[8] * fmaf(xx, v, -(yy * u));
            }
        }
    }
}

// Views of `radii` that see Gaussian i, as bits; all of them without radii.
__device__ __forceinline__ unsigned long long views_of(const int* radii, long long i, long long n,
                                                       int views)
{
    if (!radii) return ~0ull >> (64 - views);
    unsigned long long seen = 0;
    for (int v0 = 0; v0 < views; v0 += 4) {
        int r[4];  // four loads under way at once
#pragma unroll
        for (int k = 0; k < 4; k++) r[k] = v0 + k < views ? radii[(v0 + k) * n + i] : 0;
#pragma unroll
        for (int k = 0; k < 4; k++) seen |= (unsigned long long)(r[k] > 0) << (v0 + k);
    }
    return seen;
}

// What a thread needs of one Gaussian, as it comes from memory.
template <int DEG>
struct RawGaussian {
    float p[3];
    unsigned w[mx4_words(DEG)];
    __device__ __forceinline__ void load(const float* means, const void* records, long long i)
    {
#pragma unroll
        for (int k = 0; k < 3; k++) p[k] = means[3 * i + k];
        mx4_load<DEG>(records, i, w);
    }
};

// The colour of one view.
template <int USE>
__device__ __forceinline__ void color_of(const float* cam, const float p[3], const float* q,
                                         const float s[3], const float dc[3], float col[3])
{
#pragma unroll
    for (int c = 0; c < 3; c++) col[c] = dc[c];
    if constexpr (USE > 0) {
        constexpr int B = mx4_rest(USE);
        float d[3], b[B];
        unit_dir(cam, p, d);
        sh_basis<USE>(d, b);
#pragma unroll
        for (int c = 0; c < 3; c++) {
            float sum = b[0] * q[c];
#pragma unroll
            for (int k = 1; k < B; k++) sum = fmaf(b[k], q[3 * k + c], sum);
            col[c] = fmaf(s[c], sum, dc[c]);
        }
    }
}

// The same, decoding the record as it goes: eight coefficients at a time are
// held and not all of them.
template <int DEG, int USE>
__device__ __forceinline__ void color_of_record(const float* cam, const RawGaussian<DEG>& g, float col[3])
{
    constexpr int B = mx4_rest(USE);
    mx4_dc(g.w, col);
#pragma unroll
    for (int c = 0; c < 3; c++) col[c] *= MSP_SH_C0;
    if constexpr (USE > 0) {
        float d[3], b[B], s[3], sum[3];
        mx4_scales(g.w, s);
        unit_dir(cam, g.p, d);
        sh_basis<USE>(d, b);
#pragma unroll
        for (int k = 2; k < mx4_words(DEG); k++) {
            float v[8];
            e2m1x8_floats(g.w[k], v);
#pragma unroll
            for (int h = 0; h < 8; h++) {
                const int j = 8 * k + h - 18;  // bytes 0-8 of the record are 18 codes' room
                if (j < 0 || j >= 3 * B) continue;
                sum[j % 3] = j < 3 ? b[0] * v[h] : fmaf(b[j / 3], v[h], sum[j % 3]);
            }
        }
#pragma unroll
        for (int c = 0; c < 3; c++) col[c] = fmaf(s[c], sum[c], col[c]);
    }
}

// One view.  Blocks stay and take every gridDim-th tile of kMxThreads
// Gaussians; a tile's records load while the one before is computed, and its
// radii, which say what of them to load, one tile earlier still.  1M Gaussians:
// 12.4 us, 60% of them visible 13.4 (a block per 256 Gaussians, all loads up
// front: 15.1; per 128: 17.5).  Colours are stored where they are computed, three
// floats a thread: whole lines by way of shared memory took longer (13.1; 8 views
// of 6M 232), the L2 joins the parts.  Degree 4 would spill at the other degrees' 64 registers.
constexpr int one_view_blocks(int deg) { return deg == 4 ? 6 : 8; }
// The B200's multiprocessors.  Blocks take tiles until none is left, so the number
// is a matter of speed only; asking the runtime for it took 0.1 us of a call's 8.
constexpr unsigned kSms = 148;
template <int DEG, int USE, bool MASKED>
__global__ void __launch_bounds__(kMxThreads, one_view_blocks(DEG))
mx4_colors_one_kernel(int n, const float* __restrict__ means, const void* __restrict__ records,
                      const Mx4Cam cam, const int* __restrict__ radii, float* __restrict__ colors)
{
    const long long step = (long long)gridDim.x * kMxThreads;
    long long i = (long long)blockIdx.x * kMxThreads + threadIdx.x;
    auto visible = [&](long long j) { return j < n && (!MASKED || radii[j] > 0); };
    bool on = visible(i), on_next = visible(i + step);
    RawGaussian<DEG> g{}, g_next{};  // set, as lanes that are off compute too
    if (on) g.load(means, records, i);
    for (; i < n; i += step) {
        const bool on_after = visible(i + 2 * step);
        if (on_next) g_next.load(means, records, i + step);
        float col[3];
        color_of_record<DEG, USE>(cam.p, g, col);
        if (on)
#pragma unroll
            for (int c = 0; c < 3; c++) colors[3 * i + c] = col[c];
        g = g_next;
        on = on_next;
        on_next = on_after;
    }
}

// Several views, one Gaussian a thread, its coefficients decoded once.  Bound
// by instructions (82% of the issue slots at degree 3): 135 a colour, of which
// direction, basis and product are about a hundred.  8 views of 6M Gaussians:
// 210 us (a pair of Gaussians a thread in the two-float
// instructions gained nothing, their rate is the same; nor did the basis'
// constants multiplied into the coefficients, 221).
template <int DEG, int USE, bool MASKED>
__global__ void __launch_bounds__(kMxThreads)
mx4_colors_kernel(int n, const float* __restrict__ means, const void* __restrict__ records,
                  int views, const Mx4Cams cams, const int* __restrict__ radii,
                  float* __restrict__ colors)
{
    const long long i = (long long)blockIdx.x * kMxThreads + threadIdx.x;
    if (i >= n) return;
    unsigned long long seen = 0;
    RawGaussian<DEG> g;
    g.load(means, records, i);  // most Gaussians have a view that sees them: no wait for the masks
    if (MASKED) seen = views_of(radii, i, n, views);
    float dc[3], s[3], q[3 * mx4_rest(DEG) + 1], col[3];
    mx4_dc(g.w, dc);
#pragma unroll
    for (int c = 0; c < 3; c++) dc[c] *= MSP_SH_C0;
    if constexpr (USE > 0) {
        mx4_scales(g.w, s);
        mx4_codes<DEG>(g.w, q);
    }
    for (int v = 0; v < views; v++) {
        if (MASKED && !((seen >> v) & 1ull)) continue;
        color_of<USE>(cams.p[v], g.p, q, s, dc, col);
        float* out = colors + 3 * (v * (long long)n + i);
#pragma unroll
        for (int c = 0; c < 3; c++) out[c] = col[c];
    }
}

// Gradient of the coefficients: 12 bytes a view in, 192 a Gaussian out at
// degree 3.  kU: views whose gradients are under way at once -- 1 for a single
// view (4 would cost it registers: 47.6 us against 38.7 on 1M Gaussians), 4 for
// several (200,003 in 8 views: 15.0 us, 18.8 with 1).
template <int DEG, int USE, int kU>
__global__ void __launch_bounds__(kMxThreads)
mx4_colors_backward_kernel(int n, const float* __restrict__ means, int views_arg, const Mx4Cams cams,
                           const int* __restrict__ radii, const float* __restrict__ v_colors,
                           float* __restrict__ v_dc, float* __restrict__ v_rest)
{
    constexpr int B = mx4_rest(USE), E = 3 * mx4_rest(DEG), P = row_pitch(E);
    const int views = kU == 1 ? 1 : views_arg;
    __shared__ __align__(16) float s_dc[kMxThreads * 3];
    __shared__ __align__(16) float s_rest[E ? kMxThreads * P : 4];
    const long long base = (long long)blockIdx.x * kMxThreads;
    const long long i = base + threadIdx.x;
    const int cnt = (int)min((long long)kMxThreads, n - base);
    if (i < n) {
        const unsigned long long seen = views > 0 ? views_of(radii, i, n, views) : 0ull;
        float gd[3] = {0.f, 0.f, 0.f}, gr[E + 1];  // rows of degrees not in use stay 0
#pragma unroll
        for (int e = 0; e < E; e++) gr[e] = 0.f;
        float p[3];
#pragma unroll
        for (int k = 0; k < 3; k++) p[k] = means[3 * i + k];
        for (int v0 = 0; v0 < views; v0 += kU) {
            float g[kU][3];
#pragma unroll
            for (int u = 0; u < kU; u++) {
                if (v0 + u >= views || !((seen >> (v0 + u)) & 1ull)) continue;
#pragma unroll
                for (int c = 0; c < 3; c++) g[u][c] = v_colors[((v0 + u) * (long long)n + i) * 3 + c];
            }
#pragma unroll
            for (int u = 0; u < kU; u++) {
                if (v0 + u >= views || !((seen >> (v0 + u)) & 1ull)) continue;
#pragma unroll
                for (int c = 0; c < 3; c++) gd[c] += g[u][c];
                if constexpr (USE > 0) {
                    float d[3], b[B];
                    unit_dir(cams.p[v0 + u], p, d);
                    sh_basis<USE>(d, b);
#pragma unroll
                    for (int k = 0; k < B; k++)
#pragma unroll
                        for (int c = 0; c < 3; c++) gr[3 * k + c] = fmaf(b[k], g[u][c], gr[3 * k + c]);
                }
            }
        }
#pragma unroll
        for (int c = 0; c < 3; c++) s_dc[3 * threadIdx.x + c] = MSP_SH_C0 * gd[c];
        if constexpr (E > 0) row_put<E>(s_rest + threadIdx.x * P, gr);
    }
    rows_done();
    __syncthreads();
    if constexpr (E > 0) rows_out<E>(v_rest + base * E, s_rest, cnt);
    rows_out<3>(v_dc + base * 3, s_dc, cnt);
    rows_left();
}

bool views_ok(const char* who, int degree, int degrees_to_use, int views, const float* cam_pos,
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

// f(degree, degrees in use), both checked, as std::integral_constants.
template <typename F>
void with_degrees(int degree, int use, F f)
{
    with_degree(degree, [&](auto D) {
        with_degree(use, [&](auto U) {
            if constexpr (U.value <= D.value) f(D, U);
        });
    });
}

}  // namespace
}  // namespace msp

using namespace msp;

extern "C" {

int msplat_mx4_colors(int n, int degree, int degrees_to_use, const float* means3d,
                      const void* records, int num_views, const float* cam_pos,
                      const int32_t* radii, float* colors, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_colors";
    Mx4Cams cams;
    if (!mx4_shape_ok(who, n, degree) ||
        !views_ok(who, degree, degrees_to_use, num_views, cam_pos, &cams))
        return MSPLAT_ERR_ARG;
    if (n == 0 || num_views == 0) return MSPLAT_OK;
    if (!means3d || !colors) return mx4_null_pointer(who);
    if (!mx4_records_ok(who, records, degree)) return MSPLAT_ERR_ARG;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    int rc = MSPLAT_OK;
    with_degrees(degree, degrees_to_use, [&](auto D, auto U) {
        constexpr int d = D.value, u = U.value;
        const unsigned tiles = mx4_blocks(n);
        auto one = [&](auto kernel) {
            const unsigned stay = std::min(tiles, kSms * one_view_blocks(d));
            const Mx4Cam cam = {{cam_pos[0], cam_pos[1], cam_pos[2]}};
            rc = launch(who, kernel, stay, kMxThreads, st, n, means3d, records, cam, radii, colors);
        };
        auto several = [&](auto kernel) {
            rc = launch(who, kernel, tiles, kMxThreads, st, n, means3d, records, num_views, cams,
                        radii, colors);
        };
        if (num_views == 1)
            radii ? one(mx4_colors_one_kernel<d, u, true>) : one(mx4_colors_one_kernel<d, u, false>);
        else
            radii ? several(mx4_colors_kernel<d, u, true>) : several(mx4_colors_kernel<d, u, false>);
    });
    return rc;
}

int msplat_mx4_colors_backward(int n, int degree, int degrees_to_use, const float* means3d,
                               int num_views, const float* cam_pos, const int32_t* radii,
                               const float* v_colors, float* v_features_dc,
                               float* v_features_rest, void* cuda_stream)
{
    static const char* const who = "msplat_mx4_colors_backward";
    Mx4Cams cams;
    if (!mx4_shape_ok(who, n, degree) ||
        !views_ok(who, degree, degrees_to_use, num_views, cam_pos, &cams))
        return MSPLAT_ERR_ARG;
    if (n == 0) return MSPLAT_OK;
    if (!means3d || (num_views > 0 && !v_colors) || !v_features_dc ||
        (degree > 0 && !v_features_rest))
        return mx4_null_pointer(who);
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    int rc = MSPLAT_OK;
    with_degrees(degree, degrees_to_use, [&](auto D, auto U) {
        auto run = [&](auto kernel) {
            rc = launch(who, kernel, mx4_blocks(n), kMxThreads, st, n, means3d, num_views, cams, radii,
                        v_colors, v_features_dc, v_features_rest);
        };
        num_views == 1 ? run(mx4_colors_backward_kernel<D.value, U.value, 1>)
                       : run(mx4_colors_backward_kernel<D.value, U.value, 4>);
    });
    return rc;
}

}  // extern "C"
