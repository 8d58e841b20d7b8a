// E4M3 quantisation shared by the kernels that write or read 8-bit values.
//
// A group of values v_i shares one F32 scale s = max(max |v_i| / 448, 2^-126)
// (448 is the largest E4M3 value), and its codes are E4M3(v_i / s): the
// quotient rounded to F32, then to the nearest E4M3 value, ties to even.  The
// quotient is the correctly rounded one: bf16 inputs meet E4M3 ties exactly
// (v / s is a short fraction for many scales), and a reciprocal product an
// ulp off would send them to the wrong side.  The lower bound of s keeps its
// reciprocal finite.  A group with a NaN or an infinity gets a NaN scale,
// which makes every code a NaN.
#pragma once

#include <cuda_fp8.h>

#include <cstdint>

#include "m3c_device.cuh"

namespace m3c {

constexpr float E4M3_LARGEST = 448.0f;
constexpr float E4M3_LARGEST_RECIPROCAL = 1.0f / 448.0f;
constexpr float E4M3_SMALLEST_SCALE = 0x1p-126f;
constexpr float E4M3_CERTAIN_SCALE = 0x1p119f;  // 448 times any below it is finite
// div_markstein's remainder v - q s is a multiple of ulp(q) ulp(s).  Quotients
// below 2^-10 have the code 0 however they round, and for the others the
// remainder is exact while 2^-33 * 2^-23 s >= 2^-149.
// Smaller scales and their values are lifted first, which is exact.
constexpr float E4M3_MARKSTEIN_SCALE = 0x1p-90f;
constexpr float E4M3_LIFT = 0x1p64f;

// The magnitude as an integer: ordered like |v|, with NaN above infinity, so a
// maximum of these keeps a NaN that a float maximum would drop.
__device__ __forceinline__ uint32_t magnitude_bits(float v)
{
    return as_bits(v) & 0x7fffffffu;
}

__device__ __forceinline__ float e4m3_scale(uint32_t largest_bits)
{
    if (largest_bits >= 0x7f800000u) return as_float(0x7fc00000u);
    const float a = as_float(largest_bits);
    const float lift = a < E4M3_MARKSTEIN_SCALE ? E4M3_LIFT : 1.0f;
    const float s = div_markstein(__fmul_rn(a, lift), E4M3_LARGEST, E4M3_LARGEST_RECIPROCAL);
    return fmaxf(lift == 1.0f ? s : __fmul_rn(s, 1.0f / E4M3_LIFT), E4M3_SMALLEST_SCALE);
}

// The divisor of one group: its scale, lifted by a power of two with the values
// where it is too small for div_markstein, and that number's rounded reciprocal.
struct e4m3_divisor {
    float scale;
    float lift;
    float lifted;
    float reciprocal;
};

__device__ __forceinline__ e4m3_divisor e4m3_divide_by(float scale)
{
    const float lift = scale < E4M3_MARKSTEIN_SCALE ? E4M3_LIFT : 1.0f;
    const float lifted = __fmul_rn(scale, lift);
    return {scale, lift, lifted, __frcp_rn(lifted)};
}

// The largest magnitude of N values, a NaN if one of them is a NaN.
template <int N>
__device__ __forceinline__ float largest_of(const float (&v)[N])
{
    static_assert(N % 2 == 0 || N == 1, "pairs");
    if constexpr (N == 1) {
        return fabsf(v[0]);
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(v[i]), "f"(v[i + 1]));
        }
        return m;
    }
}

// The codes of four quotients, the first in the lowest byte; NaN becomes 0x7f,
// magnitudes above 448 (a rounding step at most) become 448.
__device__ __forceinline__ uint32_t e4m3_four(const float *q)
{
    uint32_t codes;
    asm("{\n\t.reg .b16 low, high;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 low, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 high, %4, %3;\n\t"
        "mov.b32 %0, {low, high};\n\t}"
        : "=r"(codes)
        : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]));
    return codes;
}

// Store the codes of 16 or eight values (to a boundary of as many bytes) or of
// one: quotients by div_markstein's steps, two a packed instruction.
template <int N>
__device__ __forceinline__ void e4m3_store(uint8_t *to, const float (&v)[N], const e4m3_divisor &d)
{
    static_assert(N == 1 || N == 8 || N == 16, "one code, eight or 16");
    if constexpr (N == 1) {
        *to = __nv_cvt_float_to_fp8(div_markstein(__fmul_rn(v[0], d.lift), d.lifted, d.reciprocal), __NV_SATFINITE,
                                    __NV_E4M3);
    } else {
        float q[N];
        const uint64_t y = f2_splat(d.reciprocal);
        const uint64_t s = f2_splat(-d.lifted);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            uint64_t a = f2_pack(v[i], v[i + 1]);
            if (d.lift != 1.0f) a = f2_mul(a, f2_splat(d.lift));
            const uint64_t q0 = f2_mul(a, y);
            f2_unpack(f2_fma(f2_fma(q0, s, a), y, q0), q[i], q[i + 1]);
        }
        if constexpr (N == 16) {
            *reinterpret_cast<uint4 *>(to) =
                make_uint4(e4m3_four(q), e4m3_four(q + 4), e4m3_four(q + 8), e4m3_four(q + 12));
        } else {
            *reinterpret_cast<uint2 *>(to) = make_uint2(e4m3_four(q), e4m3_four(q + 4));
        }
    }
}

__device__ __forceinline__ float e4m3_value(uint8_t code)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

// N codes (eight or 16, at a boundary of as many bytes) and their exact values.
template <int N>
struct e4m3_codes {
    uint32_t w[N / 4];

    __device__ __forceinline__ void load(const uint8_t *from)
    {
        if constexpr (N == 16) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4 *>(from));
            w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
        } else {
            const uint2 q = __ldcs(reinterpret_cast<const uint2 *>(from));
            w[0] = q.x, w[1] = q.y;
        }
    }

    __device__ __forceinline__ void values(float (&x)[N]) const
    {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2(
                static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (i % 2 * 16)), __NV_E4M3);
            const float2 f = __half22float2(__half2(two));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};

// Element i of a float tensor, and its store.
__device__ __forceinline__ float load_element(const void *base, int dtype, uint64_t i)
{
    if (dtype == M3C_F32) return static_cast<const float *>(base)[i];
    return widen(dtype, static_cast<const uint16_t *>(base)[i]);
}

__device__ __forceinline__ void store_element(void *base, int dtype, uint64_t i, float v)
{
    if (dtype == M3C_F32) {
        static_cast<float *>(base)[i] = v;
    } else {
        static_cast<uint16_t *>(base)[i] = static_cast<uint16_t>(narrow(dtype, v));
    }
}

}  // namespace m3c
