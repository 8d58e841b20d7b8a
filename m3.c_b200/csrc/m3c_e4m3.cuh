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
constexpr float E4M3_SMALLEST_SCALE = 0x1p-126f;
// div_markstein's remainder v - q s is a multiple of ulp(q) ulp(s).  Quotients
// below 2^-10 have the code 0 however they round, and for the others the
// remainder is exact while 2^-33 * 2^-23 s >= 2^-149.
constexpr float E4M3_MARKSTEIN_SCALE = 0x1p-90f;

// The magnitude as an integer: ordered like |v|, with NaN above infinity, so a
// maximum of these keeps a NaN that a float maximum would drop.
__device__ __forceinline__ uint32_t magnitude_bits(float v)
{
    return as_bits(v) & 0x7fffffffu;
}

__device__ __forceinline__ float e4m3_scale(uint32_t largest_bits)
{
    if (largest_bits >= 0x7f800000u) return as_float(0x7fc00000u);
    return fmaxf(__fdiv_rn(as_float(largest_bits), E4M3_LARGEST), E4M3_SMALLEST_SCALE);
}

// The divisor of one group: its scale and the scale's rounded reciprocal, or a
// reciprocal of 0 where the scale is too small for div_markstein.
struct e4m3_divisor {
    float scale;
    float reciprocal;
};

__device__ __forceinline__ e4m3_divisor e4m3_divide_by(float scale)
{
    return {scale, scale < E4M3_MARKSTEIN_SCALE ? 0.0f : __frcp_rn(scale)};
}

__device__ __forceinline__ float e4m3_quotient(float v, const e4m3_divisor &d)
{
    return d.reciprocal == 0.0f ? __fdiv_rn(v, d.scale) : div_markstein(v, d.scale, d.reciprocal);
}

__device__ __forceinline__ uint8_t e4m3_code(float v, const e4m3_divisor &d)
{
    return __nv_cvt_float_to_fp8(e4m3_quotient(v, d), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float e4m3_value(uint8_t code)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

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
