// mx4.cuh -- 4-bit colour records: a Gaussian's SH coefficients in one small
// aligned record, with the element and scale types of the OCP MX formats (e2m1
// under a power-of-two e8m0 scale), but a block per colour channel (3 to 24
// elements, not 32) and another choice of the scale (below).
//
// Record of SH degree D with B = (D+1)^2 - 1 rest coefficients per channel
// (8, 16, 24, 32, 48 bytes for D = 0..4; degree 3 is one 32-byte sector):
//   bytes 0-5   dc of r, g, b as IEEE half: its rounding (2^-11 relative)
//               moves a colour by at most 1.4e-4 |dc|, an eighth of an 8-bit
//               step of the image at |dc| = 3.5 -- 4 bits would show
//   bytes 6-8   scale byte of r, g, b (D >= 1): 2^(b - 127), 255 = NaN
//   from 9      e2m1 codes, two per byte, low nibble first; element
//               j = 3 k + c, the order of a features_rest row
// and zeros to its end.
//
// The scale of a channel is the power of two that puts its largest
// magnitude in [3.5, 7): at 7 and above e2m1 (largest value 6, the next
// would be 8) would be off by more than half a step, below 3.5 a finer
// grid would hold it.  So no element is off by more than half the spacing
// of the grid at its place.
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "msp_math.cuh"

namespace msp {

constexpr int kMx4MaxDegree = 4;
constexpr int kMx4MaxViews = 64;

__host__ __device__ constexpr int mx4_rest(int degree) { return (degree + 1) * (degree + 1) - 1; }
__host__ __device__ constexpr int mx4_words(int degree)
{
    return degree == 4 ? 12 : 2 * (degree + 1);
}
// Alignment of a record array: what its records keep among themselves.
__host__ __device__ constexpr int mx4_align(int degree) { return degree == 0 || degree == 2 ? 8 : 16; }

// The camera positions of one call, by value: no copy, so that a captured
// call keeps its own.
struct Mx4Cams {
    float p[kMx4MaxViews][3];
};
struct Mx4Cam {
    float p[3];
};

// Eight floats to e2m1, round to nearest even: v0 in the low nibble.
__device__ __forceinline__ unsigned e2m1x8(float v0, float v1, float v2, float v3, float v4,
                                           float v5, float v6, float v7)
{
    unsigned r;
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t"
        "}"
        : "=r"(r)
        : "f"(v0), "f"(v1), "f"(v2), "f"(v3), "f"(v4), "f"(v5), "f"(v6), "f"(v7));
    return r;
}

// Scale byte of a channel whose largest magnitude has the bits `amax`.  Above
// 252 a code's value could pass the largest float: magnitudes from 7 2^125 on
// saturate at 6 2^125 instead.
__device__ __forceinline__ int mx4_scale_byte(unsigned amax)
{
    if (amax >= 0x7f800000u) return 255;
    return min(252, max(0, (int)((amax + 0x200000u) >> 23) - 2));
}

// Encodes dc[3] and a row q of rest coefficients, which it scales in place.
template <int DEG>
__device__ __forceinline__ void mx4_encode(const float* dc, float (&q)[3 * mx4_rest(DEG) + 1],
                                           unsigned (&w)[mx4_words(DEG)])
{
    constexpr int E = 3 * mx4_rest(DEG), W = mx4_words(DEG);
    const unsigned h0 = __half_as_ushort(__float2half_rn(dc[0]));
    const unsigned h1 = __half_as_ushort(__float2half_rn(dc[1]));
    const unsigned h2 = __half_as_ushort(__float2half_rn(dc[2]));
    w[0] = h0 | h1 << 16;
    w[1] = h2;
    if constexpr (DEG > 0) {
        unsigned top[3] = {0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < E; j++)
            top[j % 3] = max(top[j % 3], __float_as_uint(q[j]) & 0x7fffffffu);
        int b[3];
        float inv[3];
#pragma unroll
        for (int c = 0; c < 3; c++) {
            b[c] = mx4_scale_byte(top[c]);
            inv[c] = __int_as_float((254 - b[c]) << 23);  // 2^(127 - b), exact; unused at 255
        }
#pragma unroll
        for (int j = 0; j < E; j++) q[j] = b[j % 3] == 255 ? 0.f : q[j] * inv[j % 3];
        auto at = [&](int j) { return j < E ? q[j < E ? j : 0] : 0.f; };
        w[1] |= (unsigned)b[0] << 16 | (unsigned)b[1] << 24;
        w[2] = (unsigned)b[2] | e2m1x8(0.f, 0.f, at(0), at(1), at(2), at(3), at(4), at(5));
#pragma unroll
        for (int k = 3; k < W; k++) {
            const int j = 6 + 8 * (k - 3);
            w[k] = e2m1x8(at(j), at(j + 1), at(j + 2), at(j + 3), at(j + 4), at(j + 5), at(j + 6),
                          at(j + 7));
        }
    }
}

// The codes of a record as floats, unscaled.  The conversion instruction takes
// a byte, two codes; by shifts and masks a pair takes eight instructions of the
// integer pipe and ran at less than half the rate.  The byte is masked out
// first and narrowed from 32 bits: with the word unpacked into four byte
// registers, or the byte narrowed from 16 bits, this compiler (12.9) reads the
// wrong byte where some of a word's bytes are not used.
// `byte` in 0..255.
__device__ __forceinline__ float2 e2m1x2_floats(unsigned byte)
{
    unsigned h;
    asm("{\n\t"
        ".reg .b8 a;\n\t"
        "cvt.u8.u32 a, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "}"
        : "=r"(h)
        : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ void e2m1x8_floats(unsigned word, float v[8])
{
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float2 f = e2m1x2_floats(__byte_perm(word, 0u, 0x4440u + k));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
    }
}

template <int DEG>
__device__ __forceinline__ void mx4_codes(const unsigned (&w)[mx4_words(DEG)],
                                          float (&q)[3 * mx4_rest(DEG) + 1])
{
    constexpr int E = 3 * mx4_rest(DEG), W = mx4_words(DEG);
    if constexpr (DEG > 0) {
        float v[8];
        e2m1x8_floats(w[2], v);
#pragma unroll
        for (int j = 0; j < 6; j++) q[j] = v[j + 2];  // byte 0 is a scale
#pragma unroll
        for (int k = 3; k < W; k++) {
            e2m1x8_floats(w[k], v);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (6 + 8 * (k - 3) + j < E) q[6 + 8 * (k - 3) + j] = v[j];
        }
    }
}

template <int W>
__device__ __forceinline__ void mx4_dc(const unsigned (&w)[W], float dc[3])
{
    dc[0] = __half2float(__ushort_as_half((unsigned short)w[0]));
    dc[1] = __half2float(__ushort_as_half((unsigned short)(w[0] >> 16)));
    dc[2] = __half2float(__ushort_as_half((unsigned short)w[1]));
}

// The scales 2^(b - 127) of r, g, b (b = 0: the subnormal 2^-127; 255: NaN):
// two bytes to two bf16, which are the upper halves of floats.
__device__ __forceinline__ float2 e8m0x2_floats(unsigned bytes)
{
    unsigned h;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(h) : "h"((unsigned short)bytes));
    return make_float2(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u));
}

template <int W>
__device__ __forceinline__ void mx4_scales(const unsigned (&w)[W], float s[3])
{
    const float2 rg = e8m0x2_floats(w[1] >> 16);
    s[0] = rg.x;
    s[1] = rg.y;
    s[2] = e8m0x2_floats(w[2] & 255u).x;
}

template <int DEG>
__device__ __forceinline__ void mx4_load(const void* records, long long i,
                                         unsigned (&w)[mx4_words(DEG)])
{
    constexpr int W = mx4_words(DEG);
    if constexpr (mx4_align(DEG) == 16) {
        const uint4* p = reinterpret_cast<const uint4*>(records) + i * (W / 4);
#pragma unroll
        for (int k = 0; k < W / 4; k++) {
            const uint4 v = p[k];
            w[4 * k] = v.x;
            w[4 * k + 1] = v.y;
            w[4 * k + 2] = v.z;
            w[4 * k + 3] = v.w;
        }
    } else {
        const uint2* p = reinterpret_cast<const uint2*>(records) + i * (W / 2);
#pragma unroll
        for (int k = 0; k < W / 2; k++) {
            const uint2 v = p[k];
            w[2 * k] = v.x;
            w[2 * k + 1] = v.y;
        }
    }
}

template <int DEG>
__device__ __forceinline__ void mx4_store(void* records, long long i,
                                          const unsigned (&w)[mx4_words(DEG)])
{
    constexpr int W = mx4_words(DEG);
    if constexpr (mx4_align(DEG) == 16) {
        uint4* p = reinterpret_cast<uint4*>(records) + i * (W / 4);
#pragma unroll
        for (int k = 0; k < W / 4; k++)
            p[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
    } else {
        uint2* p = reinterpret_cast<uint2*>(records) + i * (W / 2);
#pragma unroll
        for (int k = 0; k < W / 2; k++) p[k] = make_uint2(w[2 * k], w[2 * k + 1]);
    }
}

// A unit direction and the products of its components.
struct ShDir {
    float x, y, z, xx, xy, xz, yy, yz, zz;
};

__device__ __forceinline__ ShDir sh_dir(const float d[3])
{
    return {d[0], d[1], d[2], d[0] * d[0], d[0] * d[1], d[0] * d[2], d[1] * d[1], d[1] * d[2],
            d[2] * d[2]};
}

// Colour of one channel: dc and code sums per degree.  The products and
// sums are sh_to_color's (kernels_fwd.cu) in its order on the codes; the
// power-of-two scale commutes with every rounding (short of overflow and
// underflow), so a colour is bit for bit what the projection computes from
// the unpacked coefficients.
// `r(k)`: coefficient k of the channel, unscaled.
template <int DEG, typename R>
__device__ __forceinline__ float mx4_color(int use, const ShDir& D, float dc, float scale, R r)
{
    float v = MSP_SH_C0 * dc;
    const float x = D.x, y = D.y, z = D.z, xx = D.xx, xy = D.xy, xz = D.xz, yy = D.yy, yz = D.yz,
                zz = D.zz;
    if constexpr (DEG >= 1) {
        if (use < 1) return v;
        v += scale * (MSP_SH_C1 * ((-y * r(0) + z * r(1)) - x * r(2)));
    }
    if constexpr (DEG >= 2) {
        if (use < 2) return v;
        v += scale * ((((kSH_C2[0] * xy * r(3) + kSH_C2[1] * yz * r(4)) +
                        kSH_C2[2] * ((2.f * zz - xx) - yy) * r(5)) +
                       kSH_C2[3] * xz * r(6)) +
                      kSH_C2[4] * (xx - yy) * r(7));
    }
    if constexpr (DEG >= 3) {
        if (use < 3) return v;
        v += scale * ((((((kSH_C3[0] * y * (3.f * xx - yy) * r(8) + kSH_C3[1] * xy * z * r(9)) +
                          kSH_C3[2] * y * ((4.f * zz - xx) - yy) * r(10)) +
                         kSH_C3[3] * z * ((2.f * zz - 3.f * xx) - 3.f * yy) * r(11)) +
                        kSH_C3[4] * x * ((4.f * zz - xx) - yy) * r(12)) +
                       kSH_C3[5] * z * (xx - yy) * r(13)) +
                      kSH_C3[6] * x * (xx - 3.f * yy) * r(14));
    }
    if constexpr (DEG >= 4) {
        if (use < 4) return v;
        v += scale * ((((((((kSH_C4[0] * xy * (xx - yy) * r(15) +
                             kSH_C4[1] * yz * (3.f * xx - yy) * r(16)) +
                            kSH_C4[2] * xy * (7.f * zz - 1.f) * r(17)) +
                           kSH_C4[3] * yz * (7.f * zz - 3.f) * r(18)) +
                          kSH_C4[4] * (zz * (35.f * zz - 30.f) + 3.f) * r(19)) +
                         kSH_C4[5] * xz * (7.f * zz - 3.f) * r(20)) +
                        kSH_C4[6] * (xx - yy) * (7.f * zz - 1.f) * r(21)) +
                       kSH_C4[7] * xz * (xx - 3.f * yy) * r(22)) +
                      kSH_C4[8] * (xx * (xx - 3.f * yy) - yy * (3.f * xx - yy)) * r(23));
    }
    return v;
}

// A record's colour seen along the unit direction d.
template <int DEG>
__device__ __forceinline__ float4 mx4_view_color(int use, const float d[3],
                                                 const unsigned (&w)[mx4_words(DEG)])
{
    float dc[3], s[3] = {0.f, 0.f, 0.f}, col[3], q[3 * mx4_rest(DEG) + 1];
    mx4_dc(w, dc);
    if constexpr (DEG > 0) mx4_scales(w, s);
    mx4_codes<DEG>(w, q);
    const ShDir D = sh_dir(d);
#pragma unroll
    for (int c = 0; c < 3; c++)
        col[c] = mx4_color<DEG>(use, D, dc[c], s[c], [&](int k) { return q[3 * k + c]; });
    return make_float4(col[0], col[1], col[2], 0.f);
}

}  // namespace msp
