// E4M3 outputs (sm_100a): the RMS norm with the residual's addition into codes
// and scales, and the paged key/value cache, quantised as it is written and
// read back.

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "m3c_device.cuh"
#include "m3c_e4m3.cuh"
#include "m3c_kernels.h"

namespace m3c {
namespace {

constexpr int QUANT_THREADS = 256;
constexpr int QUANT_WARPS = QUANT_THREADS / 32;
constexpr int NORM_THREADS = 128;                   // rows share a CTA up to these
constexpr uint64_t NORM_WIDEST = 16384;             // of the register kernel
constexpr uint64_t NORM_KEPT_BYTES = 200u * 1024u;  // of shared memory for a row
constexpr uint32_t NORM_CHAIN = 256;                // squares summed one by one

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}

__device__ __forceinline__ uint32_t warp_max(uint32_t v)
{
    return __reduce_max_sync(0xffffffffu, v);
}

// SMs of the current device.
int sm_count()
{
    static std::atomic<int> known[64];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 148;
    int sms = known[device].load(std::memory_order_relaxed);
    if (sms == 0) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 148;
        known[device].store(sms, std::memory_order_relaxed);
    }
    return sms;
}

unsigned capped_grid(uint64_t wanted, unsigned per_sm)
{
    const uint64_t cap = static_cast<uint64_t>(sm_count()) * per_sm;
    // at least one CTA: an empty launch still records the start of the run
    return static_cast<unsigned>(wanted == 0 ? 1 : (wanted < cap ? wanted : cap));
}

// ------------------------------------------------------------------- norm
//
//   h = x, or x + r rounded;  y_j = h_j w_j / sqrt(mean(h^2) + eps);
//   per group of y: scale, codes (m3c_e4m3.cuh).
//
// Bytes bound it: x and r in, h and the codes out, 7 bytes per element of a
// 16-bit residual stream.  16384 x 4096 bf16 with residual: 70.3 us, 6.7 TB/s,
// 1.02 of the measured copy rate (71.8 us in groups of 128, with a divisor per
// piece).  Without a residual, three bytes an element, the instructions weigh
// more: 43 us (0.71).  Both kernels below read a row once and keep h on the SM
// until its codes are out.

// The register kernel: `threads` threads (whole warps) own a row, each K pieces
// of VEC consecutive elements in registers, piece k of thread i being number
// k * threads + i of the row, so a warp reads consecutive memory: 32 bytes a lane
// where every row is aligned for it (VEC = 16 elements of 16 bits, 8 of F32), 16
// bytes (VEC = 8) or one element (VEC = 1) elsewhere: odd widths and addresses pay
// for it (8192 x 4099 bf16 87.6 us, 0.18 of the copy rate; with residual 140 us,
// 0.26).  z = h w is made before the row's sum is known, and the largest |y| is the
// largest |z| times the inverse root (rounding keeps order), so one exchange
// between a row's warps carries the sum of squares and the maximum.
//   GROUP_ROW    one group per row
//   GROUP_LANES  a group is 1, 2, 4, ... or 32 pieces: the lanes that own one
//                reduce among themselves
//   GROUP_WORDS  any other group of whole pieces: a word of shared memory per
//                group (integer maxima, so the order of the atomics is free)
enum { GROUP_ROW, GROUP_LANES, GROUP_WORDS };

// VEC elements as they are stored: h is a stored value already, so 16-bit rows
// stay packed.  A piece of 32 bytes is read and written by one access, to a
// 32-byte boundary: a sector at once.
template <int DT, int VEC>
struct Piece {
    static constexpr int BYTES = VEC * (DT == M3C_F32 ? 4 : 2);
    static constexpr int WORDS = BYTES < 4 ? 1 : BYTES / 4;
    uint32_t w[WORDS];
};

template <int DT, int VEC>
__device__ __forceinline__ Piece<DT, VEC> load_piece(const void *base, uint64_t element)
{
    Piece<DT, VEC> v;
    const char *from = static_cast<const char *>(base) + element * (DT == M3C_F32 ? 4u : 2u);
    if constexpr (Piece<DT, VEC>::BYTES == 2) {
        v.w[0] = __ldcs(reinterpret_cast<const unsigned short *>(from));
    } else if constexpr (Piece<DT, VEC>::BYTES == 4) {
        v.w[0] = __ldcs(reinterpret_cast<const unsigned *>(from));
    } else if constexpr (Piece<DT, VEC>::BYTES == 32) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]),
                       "=r"(v.w[6]), "=r"(v.w[7])
                     : "l"(from)
                     : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < Piece<DT, VEC>::WORDS / 4; ++i) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4 *>(from) + i);
            v.w[4 * i] = q.x;
            v.w[4 * i + 1] = q.y;
            v.w[4 * i + 2] = q.z;
            v.w[4 * i + 3] = q.w;
        }
    }
    return v;
}

template <int DT, int VEC>
__device__ __forceinline__ void store_piece(void *base, uint64_t element, const Piece<DT, VEC> &v)
{
    char *to = static_cast<char *>(base) + element * (DT == M3C_F32 ? 4u : 2u);
    if constexpr (Piece<DT, VEC>::BYTES == 2) {
        *reinterpret_cast<uint16_t *>(to) = static_cast<uint16_t>(v.w[0]);
    } else if constexpr (Piece<DT, VEC>::BYTES == 4) {
        *reinterpret_cast<uint32_t *>(to) = v.w[0];
    } else if constexpr (Piece<DT, VEC>::BYTES == 32) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v.w[0]), "r"(v.w[1]),
                     "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
                     : "memory");
    } else {
#pragma unroll
        for (int i = 0; i < Piece<DT, VEC>::WORDS / 4; ++i) {
            __stcs(reinterpret_cast<uint4 *>(to) + i,
                   make_uint4(v.w[4 * i], v.w[4 * i + 1], v.w[4 * i + 2], v.w[4 * i + 3]));
        }
    }
}

// Both 16-bit values of a word in F32 (the second is 0 where a piece is one
// element).
template <int DT>
__device__ __forceinline__ float2 widen_word(uint32_t w)
{
    if constexpr (DT == M3C_BF16) {
        return make_float2(as_float(w << 16), as_float(w & 0xffff0000u));
    } else {
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
}

template <int DT, int VEC>
__device__ __forceinline__ void widen_piece(const Piece<DT, VEC> &v, float (&x)[VEC])
{
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if constexpr (DT == M3C_F32) {
            x[i] = as_float(v.w[i]);
        } else {
            const float2 pair = widen_word<DT>(v.w[i / 2]);
            x[i] = i % 2 ? pair.y : pair.x;
        }
    }
}

// VEC F32 values as they are stored.
template <int DT, int VEC>
__device__ __forceinline__ Piece<DT, VEC> narrow_piece(const float (&x)[VEC])
{
    Piece<DT, VEC> v;
    if constexpr (DT == M3C_F32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v.w[i] = as_bits(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            if constexpr (DT == M3C_BF16) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                v.w[i] = *reinterpret_cast<const uint32_t *>(&two);
            } else {
                const __half2 two = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                v.w[i] = *reinterpret_cast<const uint32_t *>(&two);
            }
        }
    }
    return v;
}

// round(a + b) in place of a.  The packed 16-bit addition rounds the exact sum
// once; F32 holds at least 2 p + 2 bits of a p-bit format, so rounding the F32
// sum gives the same.
template <int DT, int VEC>
__device__ __forceinline__ void add_piece(Piece<DT, VEC> &a, const Piece<DT, VEC> &b)
{
#pragma unroll
    for (int i = 0; i < Piece<DT, VEC>::WORDS; ++i) {
        if constexpr (DT == M3C_F32) {
            a.w[i] = as_bits(__fadd_rn(as_float(a.w[i]), as_float(b.w[i])));
        } else if constexpr (DT == M3C_BF16) {
            const __nv_bfloat162 s = __hadd2_rn(*reinterpret_cast<const __nv_bfloat162 *>(&a.w[i]),
                                                *reinterpret_cast<const __nv_bfloat162 *>(&b.w[i]));
            a.w[i] = *reinterpret_cast<const uint32_t *>(&s);
        } else {
            const __half2 s = __hadd2_rn(*reinterpret_cast<const __half2 *>(&a.w[i]),
                                         *reinterpret_cast<const __half2 *>(&b.w[i]));
            a.w[i] = *reinterpret_cast<const uint32_t *>(&s);
        }
    }
}

// VEC weights; the same for every row, they stay in the caches.  They are read
// with the row, but for eight or more F32 ones, which take twice the registers
// and are read when used.
template <int VEC>
struct Weights {
    Piece<M3C_F16, VEC> early;

    __device__ __forceinline__ void load(const void *scale, int dtype, uint32_t element)
    {
        const uint16_t *from = static_cast<const uint16_t *>(scale) + element;
        if (dtype == M3C_F32) {
            if constexpr (VEC == 1) early.w[0] = __ldg(static_cast<const uint32_t *>(scale) + element);
        } else if constexpr (VEC >= 8) {
#pragma unroll
            for (int i = 0; i < VEC / 8; ++i) {
                const uint4 q = __ldg(reinterpret_cast<const uint4 *>(from) + i);
                early.w[4 * i] = q.x, early.w[4 * i + 1] = q.y, early.w[4 * i + 2] = q.z, early.w[4 * i + 3] = q.w;
            }
        } else {
            early.w[0] = __ldg(from);
        }
    }

    __device__ __forceinline__ void widen(const void *scale, int dtype, uint32_t element, float (&x)[VEC]) const
    {
        if (dtype == M3C_F32) {
            const float *from = static_cast<const float *>(scale) + element;
            if constexpr (VEC >= 8) {
#pragma unroll
                for (int i = 0; i < VEC / 4; ++i) {
                    const float4 a = __ldg(reinterpret_cast<const float4 *>(from) + i);
                    x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = a.z, x[4 * i + 3] = a.w;
                }
            } else {
                x[0] = as_float(early.w[0]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const uint32_t word = early.w[i / 2];
            const float2 pair = dtype == M3C_BF16 ? widen_word<M3C_BF16>(word) : widen_word<M3C_F16>(word);
            x[i] = i % 2 ? pair.y : pair.x;
        }
    }
};

// a[i] = a[i] * b[i] (b one number or as many); two a packed instruction, which
// rounds each as the scalar one does.
template <int N>
__device__ __forceinline__ void multiply(float (&a)[N], const float (&b)[N])
{
    if constexpr (N == 1) {
        a[0] = __fmul_rn(a[0], b[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            f2_unpack(f2_mul(f2_pack(a[i], a[i + 1]), f2_pack(b[i], b[i + 1])), a[i], a[i + 1]);
        }
    }
}

template <int N>
__device__ __forceinline__ void multiply(float (&a)[N], float b)
{
    float all[N];
#pragma unroll
    for (int i = 0; i < N; ++i) all[i] = b;
    multiply(a, all);
}

// The divisor of a group whose largest |z| is `most`.  A code is that of y / s =
// (z inverse) / s, and as s is the group's largest |y| / 448, that of z over the
// largest |z| / 448: the inverse root drops out, and with it two roundings.
// Where a scale is at its lower bound, not finite, or so large that the group's y
// may pass the F32 range, the quotient is taken of y itself (`normed`).  Where a z
// passed the range, or the largest is so small that others have lost bits below
// it, y is made `anew` from h.
struct norm_divisor {
    e4m3_divisor by;
    float scale;
    bool normed;
    bool anew;
};

// A z below 2^-126 is off by 2^-150 at most: nothing against the smallest code of
// a group whose largest z is not below 2^-102.  Where all z are 0, the y of none is
// above 2^-150 times the inverse root; below 2^-126 they may be 0, so that rows of
// zeros (padding) pass quickly under any epsilon above 2^-48: 16384 x 4096 bf16
// take 48 us, and 700 where they are made anew.
constexpr float NORM_LEAST_Z = 0x1p-102f;
constexpr float NORM_LEAST_SCALE = 0x1p-110f;  // of a group whose largest z is above it
constexpr float NORM_ZERO_INVERSE = 0x1p24f;

// Whether a group whose largest |z| is `most` is made anew.
__device__ __forceinline__ bool norm_left_range(float most, float inverse)
{
    // a NaN among the z, or in the row (its inverse root), is one of the group's y too
    return inverse == inverse && (magnitude_bits(most) == 0x7f800000u ||
                                  (most < NORM_LEAST_Z && !(most == 0.0f && inverse < NORM_ZERO_INVERSE)));
}

__device__ __forceinline__ norm_divisor divide_norm_by(float most, float inverse)
{
    norm_divisor d;
    const float of_z = e4m3_scale(magnitude_bits(most));
    d.scale = __fmul_rn(of_z, inverse);
    d.normed = !(of_z > NORM_LEAST_SCALE && d.scale > E4M3_SMALLEST_SCALE &&
                 d.scale < E4M3_CERTAIN_SCALE);  // a NaN too
    d.anew = false;
    if (d.normed) {
        d.anew = norm_left_range(most, inverse);
        d.scale = e4m3_scale(magnitude_bits(__fmul_rn(most, inverse)));
    }
    d.by = e4m3_divide_by(d.normed ? d.scale : of_z);
    return d;
}

// h as it was normed: the stored sum (which may lie in the input's memory by now),
// or the input.
__device__ __forceinline__ float norm_input(const m3c_norm_e4m3_params &p, uint64_t row, uint64_t j)
{
    if (p.sum_out != nullptr) return load_element(p.sum_out, p.dtype, row * p.sum_stride + j);
    const float x = load_element(p.x, p.dtype, row * p.x_stride + j);
    if (p.resid_b == nullptr) return x;
    return round_to(p.dtype, __fadd_rn(x, load_element(p.resid_b, p.dtype, row * p.resid_stride + j)));
}

// y from h: the root first, which brings h near 1 wherever its square was in range.
__device__ __forceinline__ float norm_anew(const m3c_norm_e4m3_params &p, float h, uint64_t j, float inverse)
{
    return __fmul_rn(__fmul_rn(h, inverse), load_element(p.scale, p.scale_dtype, j));
}

// A thread's codes of the register kernel once more, pieces of `run` elements: those
// of the groups that left the range, made anew from h.  Rare, so nothing is kept for
// it from the pass before, and each thread reads its groups for itself (the warps
// of a row that is one group share the reading).  The row's h, if it was stored, is
// visible to it: a barrier of the row's warps is behind the stores.  A function of its
// own, so that the quick path's registers stay as they are (the variants of 32
// registers spill 12 bytes for the call).
template <bool ROW>
__device__ __noinline__ void norm_anew_codes(const m3c_norm_e4m3_params &p, float inverse, uint32_t run)
{
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const uint32_t width = static_cast<uint32_t>(p.width);
    const uint32_t group = static_cast<uint32_t>(p.group);
    uint32_t known = width;  // the group whose divisor is known
    e4m3_divisor d = {};
    bool wanted = false;
#pragma unroll 1
    for (uint32_t at = threadIdx.x * run; ROW || at < width; at += blockDim.x * run) {
        const uint32_t g = ROW ? 0u : at / group;
        if (g != known) {
            known = g;
            uint32_t most_z = 0u;
            uint32_t most_y = 0u;
#pragma unroll 1
            for (uint32_t j = ROW ? threadIdx.x % 32u : 0u; j < group; j += ROW ? 32u : 1u) {
                const float h = norm_input(p, row, g * group + j);
                const uint32_t z = magnitude_bits(__fmul_rn(h, load_element(p.scale, p.scale_dtype, g * group + j)));
                const uint32_t y = magnitude_bits(norm_anew(p, h, g * group + j, inverse));
                most_z = z > most_z ? z : most_z;
                most_y = y > most_y ? y : most_y;
            }
            if (ROW) most_y = warp_max(most_y);
            wanted = ROW || norm_left_range(as_float(most_z), inverse);
            d = e4m3_divide_by(e4m3_scale(most_y));
        }
        if (at >= width) break;
        if (!wanted) continue;
        if (at == g * group) p.code_scales[row * (width / group) + g] = d.scale;
#pragma unroll 1
        for (uint32_t j = at; j < at + run; ++j) {
            const float y[1] = {norm_anew(p, norm_input(p, row, j), j, inverse)};
            e4m3_store<1>(static_cast<uint8_t *>(p.codes) + row * width + j, y, d);
        }
    }
}

// The most threads of a CTA of the register kernel, as norm_depth chooses K.
constexpr int norm_block(int vec, int k)
{
    return vec == 1 ? 1024 : vec == 16 ? (k == 4 ? 256 : 512) : k == 1 ? NORM_THREADS : k == 2 ? 512 : 256;
}

template <int DT, int MODE, int VEC, int K>
__global__ void __launch_bounds__(norm_block(VEC, K))
    norm_e4m3_kernel(const __grid_constant__ m3c_norm_e4m3_params p)
{
    extern __shared__ uint32_t words[];  // GROUP_WORDS: the groups' maxima of |z|, row by row
    __shared__ float part[32];
    __shared__ uint32_t top[32];
    if (p.status != nullptr) {
        // no launch that can fail runs beside this one: the same for all threads
        if (failed_before(p.status, p.skip_before)) return;
        if (p.first_of_run && blockIdx.x == 0 && threadIdx.x == 0 && threadIdx.y == 0) {
            atomicAdd(&p.status->runs_started, 1u);
        }
    }
    // a row's threads are the block's x, the row's place in the CTA its y
    const uint32_t threads = blockDim.x;
    const uint32_t tid = threadIdx.x;
    const int lane = static_cast<int>(tid % 32u);
    const int warps = static_cast<int>(threads / 32u);
    const int first = static_cast<int>(threadIdx.y) * warps;  // the row's first warp
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    const bool live = row < p.rows;
    const uint32_t width = static_cast<uint32_t>(p.width);
    const uint32_t group = static_cast<uint32_t>(p.group);
    const uint32_t groups = width / group;
    const uint32_t place = threadIdx.y * groups;  // of the row's words
    const uint32_t shift = 31u - __clz(group);    // GROUP_LANES: the group is a power of two
    auto group_of = [&](uint32_t at) { return MODE == GROUP_LANES ? at >> shift : at / group; };

    Piece<DT, VEC> h[K];
    Weights<VEC> weight[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t at = (k * threads + tid) * VEC;
        h[k] = {};
        if (live && at < width) h[k] = load_piece<DT, VEC>(p.x, row * p.x_stride + at);
    }
    auto load_weights = [&] {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const uint32_t at = (k * threads + tid) * VEC;
            weight[k] = {};
            if (at < width) weight[k].load(p.scale, p.scale_dtype, at);
        }
    };
    if (p.resid_b != nullptr) {
        Piece<DT, VEC> r[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const uint32_t at = (k * threads + tid) * VEC;
            r[k] = {};
            if (live && at < width) r[k] = load_piece<DT, VEC>(p.resid_b, row * p.resid_stride + at);
        }
        load_weights();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const uint32_t at = (k * threads + tid) * VEC;
            add_piece<DT, VEC>(h[k], r[k]);
            if (p.sum_out != nullptr && live && at < width) {
                store_piece<DT, VEC>(p.sum_out, row * p.sum_stride + at, h[k]);
            }
        }
    } else {
        load_weights();
    }
    if constexpr (MODE == GROUP_WORDS) {
        for (uint32_t g = tid; g < groups; g += threads) words[place + g] = 0u;
        __syncthreads();
    }
    float z[K][VEC];
    float most[K];           // the largest |z| of each piece, or of its group
    uint64_t pair = 0;       // the sums of squares of even and odd elements
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t at = (k * threads + tid) * VEC;
        float w[VEC] = {};
        widen_piece<DT, VEC>(h[k], z[k]);
        if (at < width) weight[k].widen(p.scale, p.scale_dtype, at, w);
        if constexpr (VEC == 1) {
            pair = f2_fma(f2_pack(z[k][0], 0.0f), f2_pack(z[k][0], 0.0f), pair);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i += 2) {
                const uint64_t two = f2_pack(z[k][i], z[k][i + 1]);
                pair = f2_fma(two, two, pair);
            }
        }
        multiply(z[k], w);
        most[k] = largest_of<VEC>(z[k]);
        if constexpr (MODE == GROUP_LANES) {
            // a group's lanes are consecutive, and all inside the row or none
            uint32_t m = as_bits(most[k]);
            for (uint32_t d = 1; d < group / VEC; d <<= 1) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, m, d);
                m = other > m ? other : m;
            }
            most[k] = as_float(m);
        }
        if constexpr (MODE == GROUP_WORDS) {
            if (at < width) atomicMax(&words[place + group_of(at)], as_bits(most[k]));
        }
    }
    float squares[2];
    f2_unpack(pair, squares[0], squares[1]);
    squares[0] = warp_sum(__fadd_rn(squares[0], squares[1]));
    uint32_t largest = 0u;
    if constexpr (MODE == GROUP_ROW) {
#pragma unroll
        for (int k = 0; k < K; ++k) largest = as_bits(most[k]) > largest ? as_bits(most[k]) : largest;
        largest = warp_max(largest);
    }
    if (warps > 1 || MODE == GROUP_WORDS) {
        if (lane == 0) {
            part[first + tid / 32u] = squares[0];
            top[first + tid / 32u] = largest;
        }
        __syncthreads();
        squares[0] = warp_sum(lane < warps ? part[first + lane] : 0.0f);
        if constexpr (MODE == GROUP_ROW) largest = warp_max(lane < warps ? top[first + lane] : 0u);
    }
    if (!live) return;
    const float inverse = __frsqrt_rn(__fadd_rn(__fmul_rn(squares[0], p.width_reciprocal), p.epsilon));
    norm_divisor d;
    if constexpr (MODE == GROUP_ROW) {
        d = divide_norm_by(as_float(largest), inverse);
        if (d.anew) {  // the same for the row's threads
            __syncwarp();
            norm_anew_codes<true>(p, inverse, VEC);
            return;
        }
        if (tid == 0) p.code_scales[row] = d.scale;
    }
    bool anew = false;
    uint8_t *codes = static_cast<uint8_t *>(p.codes) + row * width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t at = (k * threads + tid) * VEC;
        if (at >= width) continue;
        if constexpr (MODE != GROUP_ROW) {
            const uint32_t g = group_of(at);
            if constexpr (MODE == GROUP_WORDS) most[k] = as_float(words[place + g]);
            d = divide_norm_by(most[k], inverse);
            anew = anew || d.anew;
            if (at == g * group) p.code_scales[row * groups + g] = d.scale;
        }
        if (d.normed) multiply(z[k], inverse);
        e4m3_store<VEC>(codes + at, z[k], d.by);
    }
    if constexpr (MODE != GROUP_ROW) {
        __syncwarp();
        if (anew) norm_anew_codes<false>(p, inverse, VEC);
    }
}

// Any width, alignment and group: a CTA per row, one element per thread and
// step, h kept in shared memory as F32 where the row fits (`kept`), else read
// again from the caches.
__global__ void __launch_bounds__(QUANT_THREADS)
    norm_e4m3_any_kernel(const __grid_constant__ m3c_norm_e4m3_params p, int kept)
{
    extern __shared__ float held[];
    __shared__ float part[QUANT_WARPS];
    __shared__ uint32_t top[QUANT_WARPS];
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    if (p.status != nullptr) {
        // no launch that can fail runs beside this one: the same for all threads
        if (failed_before(p.status, p.skip_before)) return;
        if (p.first_of_run && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(&p.status->runs_started, 1u);
    }
    const uint64_t groups = p.width / p.group;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        // chains of at most NORM_CHAIN squares, whose sums join in 64 bits: a longer chain
        // of like squares drifts by its length in roundings
        float squares = 0.0f;
        double before = 0.0;
        uint32_t chain = 0;
        for (uint64_t j = threadIdx.x; j < p.width; j += QUANT_THREADS) {
            float h = load_element(p.x, p.dtype, row * p.x_stride + j);
            if (p.resid_b != nullptr) {
                h = round_to(p.dtype, __fadd_rn(h, load_element(p.resid_b, p.dtype, row * p.resid_stride + j)));
            }
            if (p.sum_out != nullptr) store_element(p.sum_out, p.dtype, row * p.sum_stride + j, h);
            if (kept) held[j] = h;
            if (chain == NORM_CHAIN) {
                before += static_cast<double>(squares);
                squares = 0.0f;
                chain = 0;
            }
            ++chain;
            squares = __fmaf_rn(h, h, squares);
        }
        squares = static_cast<float>(before + static_cast<double>(squares));
        squares = warp_sum(squares);
        if (lane == 0) part[warp] = squares;
        __syncthreads();
        squares = 0.0f;
        for (int w = 0; w < QUANT_WARPS; ++w) squares = __fadd_rn(squares, part[w]);
        const float inverse =
            __frsqrt_rn(__fadd_rn(__fmul_rn(squares, p.width_reciprocal), p.epsilon));
        auto input = [&](uint64_t j) { return kept ? held[j] : norm_input(p, row, j); };
        auto weighted = [&](uint64_t j) {
            return __fmul_rn(input(j), load_element(p.scale, p.scale_dtype, j));
        };
        uint8_t *codes = static_cast<uint8_t *>(p.codes) + row * p.width;
        // many groups: one warp each; few: the whole CTA one after another
        const bool alone = groups >= QUANT_WARPS;
        const uint64_t step = alone ? 32u : QUANT_THREADS;
        const uint32_t from = alone ? lane : threadIdx.x;
        for (uint64_t g = alone ? warp : 0; g < groups; g += alone ? QUANT_WARPS : 1) {
            const uint64_t g0 = g * p.group;
            // of what the threads that share a group found
            auto join = [&](uint32_t m) {
                m = warp_max(m);
                if (!alone) {
                    if (lane == 0) top[warp] = m;
                    __syncthreads();
                    for (int w = 0; w < QUANT_WARPS; ++w) m = top[w] > m ? top[w] : m;
                }
                return m;
            };
            uint32_t largest = 0u;
            for (uint64_t j = from; j < p.group; j += step) {
                const uint32_t m = magnitude_bits(weighted(g0 + j));
                largest = m > largest ? m : largest;
            }
            const norm_divisor d = divide_norm_by(as_float(join(largest)), inverse);
            if (!d.anew) {
                if (from == 0) p.code_scales[row * groups + g] = d.scale;
                for (uint64_t j = from; j < p.group; j += step) {
                    float z[1] = {weighted(g0 + j)};
                    if (d.normed) multiply(z, inverse);
                    e4m3_store<1>(codes + g0 + j, z, d.by);
                }
            } else {  // rare, and the same for all threads that share the group
                if (!alone) __syncthreads();
                largest = 0u;
#pragma unroll 1
                for (uint64_t j = from; j < p.group; j += step) {
                    const uint32_t m = magnitude_bits(norm_anew(p, input(g0 + j), g0 + j, inverse));
                    largest = m > largest ? m : largest;
                }
                const e4m3_divisor by = e4m3_divide_by(e4m3_scale(join(largest)));
                if (from == 0) p.code_scales[row * groups + g] = by.scale;
#pragma unroll 1
                for (uint64_t j = from; j < p.group; j += step) {
                    const float y[1] = {norm_anew(p, input(g0 + j), g0 + j, inverse)};
                    e4m3_store<1>(codes + g0 + j, y, by);
                }
            }
            if (!alone) __syncthreads();
        }
        __syncthreads();
    }
}

bool aligned_to(const void *p, unsigned bytes)
{
    return reinterpret_cast<uintptr_t>(p) % bytes == 0u;
}

template <int DT, int MODE, int VEC, int K>
int norm_launch(const m3c_norm_e4m3_params &p, cudaStream_t stream)
{
    const uint64_t pieces = (p.width + VEC - 1) / VEC;
    const int threads = static_cast<int>((pieces + 32u * K - 1) / (32u * K)) * 32;
    const int places = threads < NORM_THREADS ? NORM_THREADS / threads : 1;
    const size_t smem = MODE == GROUP_WORDS ? places * (p.width / p.group) * sizeof(uint32_t) : 0u;
    const uint64_t grid = p.rows == 0 ? 1 : (p.rows + places - 1) / places;
    if (grid > 0x7fffffffu) return static_cast<int>(cudaErrorInvalidValue);
    norm_e4m3_kernel<DT, MODE, VEC, K>
        <<<static_cast<unsigned>(grid), dim3(threads, places), smem, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

template <int DT, int MODE>
int norm_depth(const m3c_norm_e4m3_params &p, bool vectors, bool wide, cudaStream_t stream)
{
    // pieces per thread.  What a thread does once per row (the root, the divisor)
    // weighs on one piece: many rows of one group take two of 16 elements (16384 x
    // 4096 bf16 without residual: 43 us, 50 with one).  With a divisor per piece, or
    // too few rows to fill the SMs with a row's fewer threads, one is as fast or
    // faster.  Rows past 8192 elements need four
    const bool many = p.rows >= 2048u && MODE == GROUP_ROW;
    if constexpr (DT != M3C_F32) {
        const uint64_t pieces = p.width / 16u;
        if (wide && pieces > 512u) return norm_launch<DT, MODE, 16, 4>(p, stream);
        if constexpr (MODE == GROUP_ROW) {
            if (wide && many && pieces > 32u) return norm_launch<DT, MODE, 16, 2>(p, stream);
        }
        if (wide) return norm_launch<DT, MODE, 16, 1>(p, stream);
    }
    // single elements: 333 rows of 2051 F32 take 5.3 us with four per thread and
    // 5.9 with eight, which are for the widths that four leave past 1024 threads
    if (!vectors && p.width <= 4096u) return norm_launch<DT, MODE, 1, 4>(p, stream);
    if (!vectors) return norm_launch<DT, MODE, 1, 8>(p, stream);
    // the same in pieces of eight elements, of which F32's take as many registers
    // as 16 of the others (8192 x 4096 with residual: 66.6 us with two)
    const uint64_t pieces = p.width / 8u;
    if (pieces <= 32u) return norm_launch<DT, MODE, 8, 1>(p, stream);
    if (pieces > 1024u) return norm_launch<DT, MODE, 8, 8>(p, stream);
    if constexpr (DT != M3C_F32 && MODE == GROUP_ROW) {
        if (many && pieces > 64u) return norm_launch<DT, MODE, 8, 4>(p, stream);
    }
    return norm_launch<DT, MODE, 8, 2>(p, stream);
}

template <int DT>
int norm_mode(const m3c_norm_e4m3_params &p, bool vectors, bool wide, cudaStream_t stream)
{
    const uint64_t lanes = p.group / (wide ? 16u : vectors ? 8u : 1u);
    if (p.group == p.width) return norm_depth<DT, GROUP_ROW>(p, vectors, wide, stream);
    if (lanes <= 32u && (lanes & (lanes - 1)) == 0u) return norm_depth<DT, GROUP_LANES>(p, vectors, wide, stream);
    return norm_depth<DT, GROUP_WORDS>(p, vectors, wide, stream);
}

// ------------------------------------------------------------------ cache

// Where packed row t lies in the cache: the number of its slot's first vector
// (slot * heads), or -1 where it has none (not in a sequence, or skipped and
// recorded).  `s` is the last sequence that begins at or before t, if any does.
__device__ __forceinline__ int64_t slot_in_sequence(const m3c_cache_params &p, uint32_t t, uint32_t s)
{
    const int64_t row = t;
    const int64_t begin = p.offsets[s];
    if (row < begin || row >= p.offsets[s + 1]) return -1;
    const int64_t position = (p.starts != nullptr ? static_cast<int64_t>(p.starts[s]) : 0) + row - begin;
    uint32_t reason = M3C_CACHE_BAD_POSITION;
    // positions below 2^32 fit the 32-bit division; a negative first offset can give
    // greater ones
    if (position >= 0 && position <= UINT32_MAX) {
        const uint32_t at = static_cast<uint32_t>(position) / p.page_tokens;
        if (at < p.page_table_stride) {
            const int64_t page = p.page_table[s * p.page_table_stride + at];
            if (page >= 0 && static_cast<uint64_t>(page) < p.pages) {
                return (page * p.page_tokens + (static_cast<uint32_t>(position) - at * p.page_tokens)) * p.heads;
            }
            reason = M3C_CACHE_BAD_PAGE;
        }
    }
    atomicMin(p.first_skipped, static_cast<unsigned long long>(t) * 4u + reason);
    return -1;
}

// The slots (their first vectors) of `count` consecutive rows, by one warp: the sequence of the first
// by a 32-way search (a step for 32 sequences, two for 1024), the others' from
// there on.
__device__ __forceinline__ void find_slots(const m3c_cache_params &p, uint32_t first, uint32_t count, int64_t *slots)
{
    const uint32_t lane = threadIdx.x % 32u;
    uint32_t low = 0;                 // sequence `low` begins at or before `first`, or none does
    uint32_t high = p.sequences;      // `high` does not, or is the end
    while (high - low > 1u) {
        const uint32_t step = (high - low + 31u) / 32u;
        const uint32_t s = low + lane * step;
        const bool before = s < high && p.offsets[s] <= static_cast<int64_t>(first);
        const uint32_t begun = __popc(__ballot_sync(0xffffffffu, before));
        low = begun == 0u ? low : low + (begun - 1u) * step;
        high = min(low + step, high);
    }
    for (uint32_t r = lane; r < count; r += 32u) {
        const int64_t row = static_cast<int64_t>(first) + r;
        uint32_t s = low;
        if (s + 1u < p.sequences && p.offsets[s + 1u] <= row) {
            uint32_t end = p.sequences;
            ++s;
            while (end - s > 1u) {
                const uint32_t middle = s + (end - s) / 2u;
                if (p.offsets[middle] <= row) {
                    s = middle;
                } else {
                    end = middle;
                }
            }
        }
        slots[r] = slot_in_sequence(p, first + r, s);
    }
}

// The vector kernels: vectors of whole pieces of VEC elements, rows aligned for
// them.  `lanes` lanes (a power of two) own a vector, P pieces each, piece j of
// lane l being number j * lanes + l.  A thread
// keeps its place (keys or values, head, lane) for several rows; blockIdx.y
// takes over where a row's vectors do not fit a block.  The slots of a CTA's
// rows are found once, in shared memory.
//
// Bytes bound both directions: three per element of 16-bit rows, five of F32.
// 262144 rows of 8 heads of 128 in bf16 are read in 249 us (6.5 TB/s, 1.00 of the
// measured copy rate), 131072 in F32 in 207 us (0.99); 65536 in bf16 are written in
// 70.6 us (5.8 TB/s, 0.88), 16384 in 20.1 us (0.77), in F32 in 103 us (1.00) and
// 28.4 us (0.90).  Writing has some twelve instructions an element (the maximum over the vector,
// a correctly rounded quotient) and the dependent loads that find a slot.
struct cache_shape {
    uint32_t lane_shift;
    uint32_t vectors;       // of a row, in a block
    uint32_t rows;          // side by side in a block
    uint32_t steps;         // groups of such rows, one after another
};

constexpr int CACHE_THREADS = 512;    // at most; 256 where the shape allows
constexpr uint32_t CACHE_STEPS = 16;  // at most
constexpr uint32_t CACHE_SLOTS = 128 * CACHE_STEPS;  // 256 threads, one head of eight elements

// A thread's place in its block's rows.
struct cache_place {
    uint32_t lane;
    uint32_t lanes;
    uint32_t side;          // the row's place in the block
    uint32_t head;
    int kv;
    bool owner;             // of a vector at all
    uint32_t first;         // the block's rows
    uint32_t count;

    __device__ __forceinline__ cache_place(const m3c_cache_params &p, const cache_shape &shape)
    {
        lanes = 1u << shape.lane_shift;
        lane = threadIdx.x & (lanes - 1u);
        const uint32_t place = threadIdx.x >> shape.lane_shift;
        side = place / shape.vectors;
        const uint32_t vector = blockIdx.y * shape.vectors + place - side * shape.vectors;
        owner = side < shape.rows && vector < 2u * p.heads;
        kv = vector >= p.heads ? 1 : 0;
        head = vector - (kv ? p.heads : 0u);
        first = blockIdx.x * shape.rows * shape.steps;
        count = min(shape.rows * shape.steps, p.row_count - first);
    }
};

// Writing: the CTA walks over its rows, the next rows' loads on their way while
// one row's codes are made; the slots are found behind the first loads.  Two CTAs
// of 512 threads an SM leave 64 registers, of which three F32 pieces (heads of 96)
// spill seven: 65536 rows of 8 x 96 take 85 us (0.91).
template <int DT, int VEC, int P>
__global__ void __launch_bounds__(CACHE_THREADS, 2)
    cache_write_kernel(const __grid_constant__ m3c_cache_params p, const __grid_constant__ cache_shape shape)
{
    __shared__ int64_t slots[CACHE_SLOTS];
    const cache_place at(p, shape);
    const uint64_t token_stride = p.token_stride[at.kv];
    const char *base = static_cast<const char *>(p.rows[at.kv]) +
                       (at.first * token_stride + at.head * p.head_stride[at.kv] + at.lane * VEC) *
                           (DT == M3C_F32 ? 4u : 2u);
    uint8_t *const codes = p.codes[at.kv] + at.lane * VEC;
    float *const scales = p.scales[at.kv];
    bool inside[P];
#pragma unroll
    for (int j = 0; j < P; ++j) inside[j] = at.owner && (j * at.lanes + at.lane) * VEC < p.head_dim;
    // the thread's next row, and the way from row to row, in bytes
    const char *row = base + at.side * token_stride * (DT == M3C_F32 ? 4u : 2u);
    const uint64_t stride = shape.rows * token_stride * (DT == M3C_F32 ? 4u : 2u);
    auto load = [&](uint32_t r, Piece<DT, VEC> (&piece)[P]) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            piece[j] = {};
            if (inside[j] && r < at.count) piece[j] = load_piece<DT, VEC>(row, j * at.lanes * VEC);
        }
        row += stride;
    };
    Piece<DT, VEC> next[P];
    load(at.side, next);
    if (threadIdx.x < 32u) find_slots(p, at.first, at.count, slots);
    __syncthreads();
    // the loop's bounds are the block's, so that its shuffles are whole
    for (uint32_t r0 = 0; r0 < at.count; r0 += shape.rows) {
        const uint32_t r = r0 + at.side;
        float x[P][VEC];
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            widen_piece<DT, VEC>(next[j], x[j]);
            const float m = largest_of<VEC>(x[j]);
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(most) : "f"(most), "f"(m));
        }
        load(r + shape.rows, next);
        uint32_t largest = as_bits(most);
        for (uint32_t d = 1; d < at.lanes; d <<= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, largest, d);
            largest = other > largest ? other : largest;
        }
        const int64_t slot = at.owner && r < at.count ? slots[r] : -1;
        if (slot >= 0) {
            const e4m3_divisor d = e4m3_divide_by(e4m3_scale(largest));
            const uint64_t vector = static_cast<uint64_t>(slot) + at.head;
            if (at.lane == 0u) scales[vector] = d.scale;
#pragma unroll
            for (int j = 0; j < P; ++j) {
                if (inside[j]) e4m3_store<VEC>(codes + vector * p.head_dim + j * at.lanes * VEC, x[j], d);
            }
        }
    }
}

// Reading: the slots first, then STEPS rows of a thread at once, with stores of 32
// bytes a lane, which fill their sectors at once.
template <int DT, int VEC, int P, int STEPS>
__global__ void __launch_bounds__(CACHE_THREADS)
    cache_read_kernel(const __grid_constant__ m3c_cache_params p, const __grid_constant__ cache_shape shape)
{
    __shared__ int64_t slots[128 * STEPS];
    const cache_place at(p, shape);
    if (threadIdx.x < 32u) find_slots(p, at.first, at.count, slots);
    __syncthreads();
    if (!at.owner) return;
    const uint64_t token_stride = p.token_stride[at.kv];
    char *const base = static_cast<char *>(p.rows[at.kv]) +
                       (at.first * token_stride + at.head * p.head_stride[at.kv] + at.lane * VEC) *
                           (DT == M3C_F32 ? 4u : 2u);
    const uint8_t *const from = p.codes[at.kv] + at.lane * VEC;
    e4m3_codes<VEC> codes[STEPS][P];
    float scale[STEPS];
    bool live[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const uint32_t r = i * shape.rows + at.side;
        const int64_t slot = r < at.count ? slots[r] : -1;
        const uint64_t vector = static_cast<uint64_t>(slot) + at.head;
        live[i] = slot >= 0;
        scale[i] = live[i] ? p.scales[at.kv][vector] : 0.0f;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            codes[i][j] = {};
            if (live[i] && (j * at.lanes + at.lane) * VEC < p.head_dim) {
                codes[i][j].load(from + vector * p.head_dim + j * at.lanes * VEC);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const uint32_t r = i * shape.rows + at.side;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            float x[VEC];
            codes[i][j].values(x);
            multiply(x, scale[i]);
            if (live[i] && (j * at.lanes + at.lane) * VEC < p.head_dim) {
                store_piece<DT, VEC>(base, r * token_stride + j * at.lanes * VEC, narrow_piece<DT, VEC>(x));
            }
        }
    }
}

// Any shape, and keys and values of two types: one warp per (row, keys or values,
// head), one element a lane.  What bounds it is the search for the slot, once a
// vector, and the narrow accesses: 16384 rows of 8 x 60 bf16 are written in 95 us
// and read in 72 (0.08 and 0.10 of the copy rate).
template <bool WRITE>
__global__ void __launch_bounds__(QUANT_THREADS) cache_any_kernel(const __grid_constant__ m3c_cache_params p)
{
    __shared__ int64_t slots[QUANT_WARPS];
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const uint64_t vectors = static_cast<uint64_t>(p.row_count) * 2u * p.heads;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * QUANT_WARPS;
    for (uint64_t v = static_cast<uint64_t>(blockIdx.x) * QUANT_WARPS + threadIdx.x / 32; v < vectors; v += stride) {
        const uint32_t t = static_cast<uint32_t>(v / (2u * p.heads));
        const uint32_t rest = static_cast<uint32_t>(v % (2u * p.heads));
        const int kv = rest >= p.heads ? 1 : 0;
        const uint32_t head = rest - kv * p.heads;
        __syncwarp();
        find_slots(p, t, 1u, &slots[threadIdx.x / 32]);
        __syncwarp();
        const int64_t slot = slots[threadIdx.x / 32];
        if (slot < 0) continue;
        const uint64_t at = static_cast<uint64_t>(slot) + head;
        const uint64_t row = t * p.token_stride[kv] + head * p.head_stride[kv];
        uint8_t *codes = p.codes[kv] + at * p.head_dim;
        if constexpr (WRITE) {
            uint32_t largest = 0u;
            for (uint32_t j = lane; j < p.head_dim; j += 32) {
                const uint32_t m = magnitude_bits(load_element(p.rows[kv], p.dtype[kv], row + j));
                largest = m > largest ? m : largest;
            }
            const e4m3_divisor d = e4m3_divide_by(e4m3_scale(warp_max(largest)));
            if (lane == 0) p.scales[kv][at] = d.scale;
            for (uint32_t j = lane; j < p.head_dim; j += 32) {
                const float v[1] = {load_element(p.rows[kv], p.dtype[kv], row + j)};
                e4m3_store<1>(codes + j, v, d);
            }
        } else {
            const float scale = p.scales[kv][at];
            for (uint32_t j = lane; j < p.head_dim; j += 32) {
                store_element(p.rows[kv], p.dtype[kv], row + j, __fmul_rn(e4m3_value(codes[j]), scale));
            }
        }
    }
}

template <int DT, int VEC, bool WRITE, int P>
int launch_cache_vectors(const m3c_cache_params &p, cudaStream_t stream)
{
    cache_shape shape;
    shape.lane_shift = 0u;
    while ((static_cast<uint32_t>(VEC * P) << shape.lane_shift) < p.head_dim) ++shape.lane_shift;
    const uint32_t fit = CACHE_THREADS >> shape.lane_shift;
    const uint32_t all = 2u * p.heads;
    shape.vectors = all < fit ? all : fit;
    const uint32_t threads = shape.vectors << shape.lane_shift;
    shape.rows = threads < 256u ? 256u / threads : 1u;
    const uint32_t block = (shape.rows * threads + 31u) / 32u * 32u;
    const uint32_t chunks = (all - 1u) / shape.vectors + 1u;
    const uint64_t groups = static_cast<uint64_t>((p.row_count - 1u) / shape.rows + 1u) * chunks;
    const uint64_t resident = 4u * static_cast<uint64_t>(sm_count());  // CTAs at a time
    if constexpr (WRITE) {
        // whole waves of CTAs, each with as many steps as it may have
        const uint64_t waves = (groups - 1u) / resident + 1u;
        const uint64_t rounds = (waves - 1u) / CACHE_STEPS + 1u;
        shape.steps = static_cast<uint32_t>((waves - 1u) / rounds + 1u);
        const dim3 grid((p.row_count - 1u) / (shape.rows * shape.steps) + 1u, chunks);
        cache_write_kernel<DT, VEC, P><<<grid, block, 0, stream>>>(p, shape);
    } else {
        // the 262144 rows above take 297 us with one row at once; a small batch
        // takes one all the same, since the unrolled code's own fetch costs more
        // than it hides (500 rows of 4 x 64 F32: 2.8 us, 3.1 with four)
        constexpr int MANY = VEC * P == 8 ? 4 : 2;
        shape.steps = groups < MANY * resident ? 1u : MANY;
        const dim3 grid((p.row_count - 1u) / (shape.rows * shape.steps) + 1u, chunks);
        if (shape.steps == 1u) {
            cache_read_kernel<DT, VEC, P, 1><<<grid, block, 0, stream>>>(p, shape);
        } else {
            cache_read_kernel<DT, VEC, P, MANY><<<grid, block, 0, stream>>>(p, shape);
        }
    }
    return static_cast<int>(cudaGetLastError());
}

// The pieces per lane of a vector of `dim` elements in pieces of `vec`: as few
// idle lanes as can be (lanes a power of two, at most a warp), and of equals the
// more pieces, up to `preferred`.  `idle` becomes the elements that idle lanes
// would have.
int cache_pieces(uint32_t dim, uint32_t vec, int most, int preferred, uint32_t *idle)
{
    const uint32_t pieces = dim / vec;
    int best = 1;
    *idle = UINT32_MAX;
    for (int k = 1; k <= most; ++k) {
        uint32_t lanes = 1u;
        while (lanes * k < pieces) lanes <<= 1;
        const uint32_t rest = (lanes * k - pieces) * vec;
        if (lanes <= 32u && (rest < *idle || (rest == *idle && k <= preferred))) {
            *idle = rest;
            best = k;
        }
    }
    return best;
}

// Pieces of 32 bytes (`wide`: the rows are aligned for them) unless pieces of 16
// leave fewer lanes idle: one a lane up to 512 elements, for reading three beyond
// (two are never fewer idle lanes than one, or than three).  More than one to
// write leave too few threads on an SM.
template <int DT, bool WRITE>
int launch_cache_pieces(const m3c_cache_params &p, bool wide, cudaStream_t stream)
{
    uint32_t idle = 0;
    const int narrow = cache_pieces(p.head_dim, 8u, 3, 3, &idle);
    if constexpr (DT != M3C_F32) {
        uint32_t wide_idle = 0;
        const int k = cache_pieces(p.head_dim, 16u, WRITE ? 1 : 3, 1, &wide_idle);
        if (wide && wide_idle <= idle) {
            if constexpr (!WRITE) {
                if (k == 3) return launch_cache_vectors<DT, 16, WRITE, 3>(p, stream);
            }
            return launch_cache_vectors<DT, 16, WRITE, 1>(p, stream);
        }
    }
    if (narrow == 1) return launch_cache_vectors<DT, 8, WRITE, 1>(p, stream);
    if (narrow == 2) return launch_cache_vectors<DT, 8, WRITE, 2>(p, stream);
    return launch_cache_vectors<DT, 8, WRITE, 3>(p, stream);
}

// The first skipped row, and none from here on.
__global__ void cache_report_kernel(unsigned long long *first_skipped, unsigned long long *report)
{
    *report = atomicExch(first_skipped, ~0ull);
}

template <bool WRITE>
int launch_cache(const m3c_cache_params &p, cudaStream_t stream)
{
    const uint64_t vectors = static_cast<uint64_t>(p.row_count) * 2u * p.heads;
    // pieces of 32 bytes where the rows are aligned for them, else of 16; a
    // vector's lanes are at most a warp of three pieces each; the grid's y
    // counts heads
    const uint32_t size = p.dtype[0] == M3C_F32 ? 4u : 2u;
    bool fits = p.dtype[0] == p.dtype[1] && p.head_dim % 8u == 0u && p.head_dim <= 768u && p.heads <= 16384u;
    bool wide = p.head_dim % (32u / size) == 0u;
    for (int k = 0; k < 2; ++k) {
        const uint64_t address = reinterpret_cast<uintptr_t>(p.rows[k]) | p.token_stride[k] * size |
                                 p.head_stride[k] * size;
        fits = fits && address % 16u == 0u;
        wide = wide && address % 32u == 0u;
    }
    if (fits && (wide || p.dtype[0] != M3C_F32)) {
        switch (p.dtype[0]) {
        case M3C_F16: return launch_cache_pieces<M3C_F16, WRITE>(p, wide, stream);
        case M3C_BF16: return launch_cache_pieces<M3C_BF16, WRITE>(p, wide, stream);
        default: return launch_cache_pieces<M3C_F32, WRITE>(p, wide, stream);
        }
    }
    const unsigned grid = capped_grid((vectors + QUANT_WARPS - 1) / QUANT_WARPS, 32u);
    cache_any_kernel<WRITE><<<grid, QUANT_THREADS, 0, stream>>>(p);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace
}  // namespace m3c

extern "C" int m3c_launch_norm_e4m3(const m3c_norm_e4m3_params *params, void *stream)
{
    using namespace m3c;
    m3c_norm_e4m3_params p = *params;
    p.width_reciprocal = 1.0f / static_cast<float>(p.width);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    // eight elements are one access: 32 bytes of F32, 16 of the others
    const unsigned bytes = p.dtype == M3C_F32 ? 32u : 16u;
    const bool vectors = p.width % 8u == 0u && p.group % 8u == 0u && p.x_stride % 8u == 0u && aligned_to(p.x, bytes) &&
                         aligned_to(p.scale, 16) && aligned_to(p.codes, 8) &&
                         (p.resid_b == nullptr || (p.resid_stride % 8u == 0u && aligned_to(p.resid_b, bytes))) &&
                         (p.sum_out == nullptr || (p.sum_stride % 8u == 0u && aligned_to(p.sum_out, bytes)));
    // sixteen 16-bit ones 32, where they keep a warp's lanes busy
    const bool wide = vectors && p.dtype != M3C_F32 && p.width > 256u && p.width % 16u == 0u && p.group % 16u == 0u &&
                      p.x_stride % 16u == 0u && aligned_to(p.x, 32) && aligned_to(p.codes, 16) &&
                      (p.resid_b == nullptr || (p.resid_stride % 16u == 0u && aligned_to(p.resid_b, 32))) &&
                      (p.sum_out == nullptr || (p.sum_stride % 16u == 0u && aligned_to(p.sum_out, 32)));
    if (p.width <= (vectors ? NORM_WIDEST : NORM_WIDEST / 2u)) {
        switch (p.dtype) {
        case M3C_F16: return norm_mode<M3C_F16>(p, vectors, wide, s);
        case M3C_BF16: return norm_mode<M3C_BF16>(p, vectors, wide, s);
        default: return norm_mode<M3C_F32>(p, vectors, wide, s);
        }
    }
    const size_t row_bytes = p.width * sizeof(float);
    const bool kept = row_bytes <= NORM_KEPT_BYTES;
    if (kept) {
        // these rows begin at 32 KB; with the kernel's static shared memory they pass
        // the default of 48 KB below 12288 elements
        const cudaError_t code = cudaFuncSetAttribute(
            norm_e4m3_any_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(NORM_KEPT_BYTES));
        if (code != cudaSuccess) return static_cast<int>(code);
    }
    norm_e4m3_any_kernel<<<capped_grid(p.rows, 32u), QUANT_THREADS, kept ? row_bytes : 0u, s>>>(p, kept ? 1 : 0);
    return static_cast<int>(cudaGetLastError());
}

extern "C" int m3c_launch_cache_write(const m3c_cache_params *params, void *stream)
{
    return m3c::launch_cache<true>(*params, static_cast<cudaStream_t>(stream));
}

extern "C" int m3c_launch_cache_read(const m3c_cache_params *params, void *stream)
{
    return m3c::launch_cache<false>(*params, static_cast<cudaStream_t>(stream));
}

extern "C" int m3c_launch_cache_report(unsigned long long *first_skipped, unsigned long long *report, void *stream)
{
    m3c::cache_report_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(first_skipped, report);
    return static_cast<int>(cudaGetLastError());
}
