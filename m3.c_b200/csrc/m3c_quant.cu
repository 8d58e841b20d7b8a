// E4M3 outputs (sm_100a): the RMS norm with the residual's addition into codes
// and scales, and the paged key/value cache, quantised as it is written and
// read back.

#include <cuda_runtime.h>

#include <cstdint>

#include "m3c_device.cuh"
#include "m3c_e4m3.cuh"
#include "m3c_kernels.h"

extern "C" void m3c_fastdiv_init(m3c_fastdiv *fd, uint32_t divisor);

namespace m3c {
namespace {

constexpr int QUANT_THREADS = 256;
constexpr int QUANT_WARPS = QUANT_THREADS / 32;
#ifndef NORM_THREADS
#define NORM_THREADS 128
#endif
constexpr uint64_t NORM_WIDEST = 16384;             // of the register kernel
constexpr uint64_t NORM_KEPT_BYTES = 200u * 1024u;  // of shared memory for a row

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

unsigned capped_grid(uint64_t wanted, unsigned per_sm)
{
    int device = 0;
    int sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess) {
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    }
    const uint64_t cap = static_cast<uint64_t>(sms) * per_sm;
    // at least one CTA: an empty launch still records the start of the run
    return static_cast<unsigned>(wanted == 0 ? 1 : (wanted < cap ? wanted : cap));
}

// ------------------------------------------------------------------- norm
//
//   h = x, or x + r rounded;  y_j = h_j w_j / sqrt(mean(h^2) + eps);
//   per group of y: scale, codes (m3c_e4m3.cuh).
//
// Bytes bound it: x and r in, h and the codes out, 7 bytes per element of a
// 16-bit residual stream against some 14 instructions.  Both kernels below
// read a row once and keep h on the SM until its codes are out.

// The register kernel: `threads` threads (whole warps) own a row, each K pieces
// of VEC consecutive elements in registers, piece k of thread i being number
// k * threads + i of the row, so a warp reads consecutive memory: VEC = 8 (16
// bytes of a 16-bit row a lane) where every row is aligned for it, VEC = 1
// elsewhere.  z = h w is made before the row's sum is known, and the largest |y|
// is the largest |z| times the inverse root (rounding keeps order), so one
// exchange between a row's warps carries the sum of squares and the maximum.
//   GROUP_ROW    one group per row
//   GROUP_LANES  a group is 1, 2, 4, ... or 32 pieces: the lanes that own one
//                reduce among themselves
//   GROUP_WORDS  any other group of whole pieces: a word of shared memory per
//                group (integer maxima, so the order of the atomics is free)
enum { GROUP_ROW, GROUP_LANES, GROUP_WORDS };

// VEC elements as they are stored: h is a stored value already, so 16-bit rows
// stay packed.
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

// Eight F32 values as they are stored.
template <int DT>
__device__ __forceinline__ Piece<DT, 8> narrow_piece(const float (&x)[8])
{
    Piece<DT, 8> v;
    if constexpr (DT == M3C_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.w[i] = as_bits(x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
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

// VEC weights; the same for every row, they stay in the caches.  16-bit ones are
// read with the row, F32 ones, which take twice the registers, when used.
template <int VEC>
struct Weights {
    Piece<M3C_F16, VEC> early;

    __device__ __forceinline__ void load(const void *scale, int dtype, uint32_t element)
    {
        if (dtype == M3C_F32) return;
        const uint16_t *from = static_cast<const uint16_t *>(scale) + element;
        if constexpr (VEC == 8) {
            const uint4 q = __ldg(reinterpret_cast<const uint4 *>(from));
            early.w[0] = q.x, early.w[1] = q.y, early.w[2] = q.z, early.w[3] = q.w;
        } else {
            early.w[0] = __ldg(from);
        }
    }

    __device__ __forceinline__ void widen(const void *scale, int dtype, uint32_t element, float (&x)[VEC]) const
    {
        if (dtype == M3C_F32) {
            const float *from = static_cast<const float *>(scale) + element;
            if constexpr (VEC == 8) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(from));
                const float4 b = __ldg(reinterpret_cast<const float4 *>(from) + 1);
                x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
                x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
            } else {
                x[0] = __ldg(from);
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

template <int DT, int MODE, int VEC, int K>
__global__ void __launch_bounds__(K == 1 ? 1024 : 512, K == 4 && DT != M3C_F32 ? 2 : 1)
    norm_e4m3_kernel(const __grid_constant__ m3c_norm_e4m3_params p)
{
    extern __shared__ uint32_t words[];  // GROUP_WORDS: the groups' maxima of |z|, row by row
    __shared__ float part[32];
    __shared__ uint32_t top[32];
    if (p.status != nullptr) {
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
    const float inverse = __frsqrt_rn(__fadd_rn(__fdiv_rn(squares[0], static_cast<float>(width)), p.epsilon));
    e4m3_divisor d;
    if constexpr (MODE == GROUP_ROW) {
        d = e4m3_divide_by(e4m3_scale(magnitude_bits(__fmul_rn(as_float(largest), inverse))));
        if (tid == 0) p.code_scales[row] = d.scale;
    }
    uint8_t *codes = static_cast<uint8_t *>(p.codes) + row * width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t at = (k * threads + tid) * VEC;
        if (at >= width) continue;
        if constexpr (MODE != GROUP_ROW) {
            if constexpr (MODE == GROUP_WORDS) most[k] = as_float(words[place + group_of(at)]);
            d = e4m3_divide_by(e4m3_scale(magnitude_bits(__fmul_rn(most[k], inverse))));
            const uint32_t g = group_of(at);
            if (at == g * group) p.code_scales[row * groups + g] = d.scale;
        }
        multiply(z[k], inverse);
        e4m3_store<VEC>(codes + at, z[k], d);
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
        if (failed_before(p.status, p.skip_before)) return;
        if (p.first_of_run && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(&p.status->runs_started, 1u);
    }
    const uint64_t groups = p.width / p.group;
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const uint64_t x0 = row * p.x_stride;
        const uint64_t r0 = row * p.resid_stride;
        const uint64_t s0 = row * p.sum_stride;
        auto read = [&](uint64_t j) {
            float h = load_element(p.x, p.dtype, x0 + j);
            if (p.resid_b != nullptr) h = round_to(p.dtype, __fadd_rn(h, load_element(p.resid_b, p.dtype, r0 + j)));
            return h;
        };
        float squares = 0.0f;
        for (uint64_t j = threadIdx.x; j < p.width; j += QUANT_THREADS) {
            const float h = read(j);
            if (p.sum_out != nullptr) store_element(p.sum_out, p.dtype, s0 + j, h);
            if (kept) held[j] = h;
            squares = __fmaf_rn(h, h, squares);
        }
        squares = warp_sum(squares);
        if (lane == 0) part[warp] = squares;
        __syncthreads();
        squares = 0.0f;
        for (int w = 0; w < QUANT_WARPS; ++w) squares = __fadd_rn(squares, part[w]);
        const float inverse =
            __frsqrt_rn(__fadd_rn(__fdiv_rn(squares, static_cast<float>(p.width)), p.epsilon));
        auto normed = [&](uint64_t j) {
            // the stored sum is h (and may be the input's own storage by now)
            const float h = kept                   ? held[j]
                            : p.sum_out != nullptr ? load_element(p.sum_out, p.dtype, s0 + j)
                                                   : read(j);
            return __fmul_rn(__fmul_rn(h, load_element(p.scale, p.scale_dtype, j)), inverse);
        };
        uint8_t *codes = static_cast<uint8_t *>(p.codes) + row * p.width;
        // many groups: one warp each; few: the whole CTA one after another
        const bool alone = groups >= QUANT_WARPS;
        const uint64_t step = alone ? 32u : QUANT_THREADS;
        const uint32_t from = alone ? lane : threadIdx.x;
        for (uint64_t g = alone ? warp : 0; g < groups; g += alone ? QUANT_WARPS : 1) {
            const uint64_t g0 = g * p.group;
            uint32_t largest = 0u;
            for (uint64_t j = from; j < p.group; j += step) {
                const uint32_t m = magnitude_bits(normed(g0 + j));
                largest = m > largest ? m : largest;
            }
            largest = warp_max(largest);
            if (!alone) {
                if (lane == 0) top[warp] = largest;
                __syncthreads();
                for (int w = 0; w < QUANT_WARPS; ++w) largest = top[w] > largest ? top[w] : largest;
            }
            const e4m3_divisor d = e4m3_divide_by(e4m3_scale(largest));
            if (from == 0) p.code_scales[row * groups + g] = d.scale;
            for (uint64_t j = from; j < p.group; j += step) codes[g0 + j] = e4m3_code(normed(g0 + j), d);
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
int norm_depth(const m3c_norm_e4m3_params &p, bool vectors, cudaStream_t stream)
{
    if (!vectors) return norm_launch<DT, MODE, 1, 16>(p, stream);
    // pieces per thread: two keep a row of 4096 elements in 256 threads; wider
    // rows take four, unless there are too few rows to fill the SMs with
    // their fewer threads
    const uint64_t pieces = p.width / 8u;
    const int k = pieces <= 32u ? 1 : pieces <= 512u || (pieces <= 1024u && p.rows < 2048u) ? 2 : 4;
    if (k == 1) return norm_launch<DT, MODE, 8, 1>(p, stream);
    if (k == 2) return norm_launch<DT, MODE, 8, 2>(p, stream);
    return norm_launch<DT, MODE, 8, 4>(p, stream);
}

template <int DT>
int norm_mode(const m3c_norm_e4m3_params &p, bool vectors, cudaStream_t stream)
{
    if (p.group == p.width) return norm_depth<DT, GROUP_ROW>(p, vectors, stream);
    const uint64_t lanes = vectors ? p.group / 8u : p.group;
    if (lanes <= 32u && (lanes & (lanes - 1)) == 0u) return norm_depth<DT, GROUP_LANES>(p, vectors, stream);
    return norm_depth<DT, GROUP_WORDS>(p, vectors, stream);
}

// ------------------------------------------------------------------ cache

// Where packed row t lies in the cache: its slot, or -1 where it has none (not
// in a sequence, or skipped and recorded).
__device__ int64_t cache_slot(const m3c_cache_params &p, uint32_t t)
{
    // the last sequence that begins at or before t
    if (static_cast<int64_t>(t) < p.offsets[0]) return -1;
    uint32_t low = 0;
    uint32_t high = p.sequences;
    while (high - low > 1) {
        const uint32_t middle = low + (high - low) / 2;
        if (p.offsets[middle] <= static_cast<int64_t>(t)) {
            low = middle;
        } else {
            high = middle;
        }
    }
    if (static_cast<int64_t>(t) >= p.offsets[low + 1]) return -1;
    const int64_t position =
        (p.starts != nullptr ? static_cast<int64_t>(p.starts[low]) : 0) + t - p.offsets[low];
    uint32_t reason = 0u;
    int64_t slot = -1;
    if (position < 0 || static_cast<uint64_t>(position) / p.page_tokens >= p.page_table_stride) {
        reason = M3C_CACHE_BAD_POSITION;
    } else {
        const uint64_t at = static_cast<uint64_t>(position) / p.page_tokens;
        const int64_t page = p.page_table[low * p.page_table_stride + at];
        if (page < 0 || static_cast<uint64_t>(page) >= p.pages) {
            reason = M3C_CACHE_BAD_PAGE;
        } else {
            slot = page * p.page_tokens + static_cast<int64_t>(static_cast<uint64_t>(position) % p.page_tokens);
        }
    }
    if (reason != 0u) atomicMin(p.first_skipped, static_cast<unsigned long long>(t) * 4u + reason);
    return slot;
}

// The vector kernel: vectors of a multiple of eight elements up to 256, rows
// aligned for 16-byte accesses.  A vector belongs to `lanes` lanes (a power of
// two), eight elements each; a CTA takes DEPTH * 256 / lanes consecutive
// vectors, those of a row (keys, then values, head by head) beside one
// another, and finds the slots of their rows once, in shared memory.  Bytes
// bound both directions: three per element of 16-bit rows.
#ifndef DW
#define DW 4
#endif
#ifndef DR
#define DR 4
#endif
constexpr int CACHE_DEPTH_WRITE = DW;
constexpr int CACHE_DEPTH_READ = DR;
constexpr int CACHE_DEPTH = CACHE_DEPTH_READ > CACHE_DEPTH_WRITE ? CACHE_DEPTH_READ : CACHE_DEPTH_WRITE;
constexpr uint32_t CACHE_MOST_ROWS = QUANT_THREADS * CACHE_DEPTH / 2 + 2;  // of a CTA: one head, eight elements

struct cache_shape {
    m3c_fastdiv of_row;     // vectors of a row
    uint32_t vectors;       // of the batch
    uint32_t lanes;         // of a vector
    uint32_t lane_shift;
};

template <int DT, bool WRITE>
__global__ void __launch_bounds__(QUANT_THREADS)
    cache_kernel(const __grid_constant__ m3c_cache_params p, const __grid_constant__ cache_shape shape)
{
    constexpr int DEPTH = WRITE ? CACHE_DEPTH_WRITE : CACHE_DEPTH_READ;
    __shared__ int64_t slots[CACHE_MOST_ROWS];
    const uint32_t per_pass = QUANT_THREADS >> shape.lane_shift;
    const uint32_t first = blockIdx.x * per_pass * DEPTH;
    const uint32_t first_row = fastdiv(first, shape.of_row);
    const uint32_t last = min(first + per_pass * DEPTH, shape.vectors) - 1u;
    const uint32_t rows = fastdiv(last, shape.of_row) - first_row + 1u;
    const uint32_t element = (threadIdx.x & (shape.lanes - 1u)) * 8u;
    const bool inside = element < p.head_dim;
    uint32_t row[DEPTH];
    uint32_t head[DEPTH];
    int kv[DEPTH];
    bool live[DEPTH];
    uint64_t at[DEPTH];      // the lane's place among the rows' elements
    Piece<DT, 8> piece[DEPTH];
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
        const uint32_t v = first + i * per_pass + (threadIdx.x >> shape.lane_shift);
        live[i] = v <= last;
        row[i] = live[i] ? fastdiv(v, shape.of_row) : first_row;
        const uint32_t rest = live[i] ? v - row[i] * shape.of_row.divisor : 0u;
        kv[i] = rest >= p.heads ? 1 : 0;
        head[i] = rest - (kv[i] ? p.heads : 0u);
        at[i] = row[i] * p.token_stride[kv[i]] + head[i] * p.head_stride[kv[i]] + element;
        piece[i] = {};
        if (WRITE && live[i] && inside) piece[i] = load_piece<DT, 8>(p.rows[kv[i]], at[i]);
    }
    for (uint32_t r = threadIdx.x; r < rows; r += QUANT_THREADS) slots[r] = cache_slot(p, first_row + r);
    __syncthreads();
    if constexpr (WRITE) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            float x[8];
            widen_piece<DT, 8>(piece[i], x);
            uint32_t largest = as_bits(largest_of<8>(x));
            for (uint32_t d = 1; d < shape.lanes; d <<= 1) {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, largest, d);
                largest = other > largest ? other : largest;
            }
            const int64_t slot = slots[row[i] - first_row];
            if (!live[i] || slot < 0) continue;
            const e4m3_divisor d = e4m3_divide_by(e4m3_scale(largest));
            const uint64_t vector = static_cast<uint64_t>(slot) * p.heads + head[i];
            if (element == 0u) p.scales[kv[i]][vector] = d.scale;
            if (inside) e4m3_store<8>(p.codes[kv[i]] + vector * p.head_dim + element, x, d);
        }
    } else {
        uint2 codes[DEPTH];
        float scale[DEPTH];
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            const int64_t slot = slots[row[i] - first_row];
            live[i] = live[i] && slot >= 0 && inside;
            codes[i] = {};
            scale[i] = 0.0f;
            if (live[i]) {
                const uint64_t vector = static_cast<uint64_t>(slot) * p.heads + head[i];
                codes[i] = __ldcs(reinterpret_cast<const uint2 *>(p.codes[kv[i]] + vector * p.head_dim + element));
                scale[i] = p.scales[kv[i]][vector];
            }
        }
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) {
            float x[8];
            e4m3_values(codes[i], x);
            multiply(x, scale[i]);
            if (live[i]) store_piece<DT, 8>(p.rows[kv[i]], at[i], narrow_piece<DT>(x));
        }
    }
}

// Any shape: one warp per (row, keys or values, head).
template <bool WRITE>
__global__ void __launch_bounds__(QUANT_THREADS) cache_any_kernel(const __grid_constant__ m3c_cache_params p)
{
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const uint64_t vectors = static_cast<uint64_t>(p.row_count) * 2u * p.heads;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * QUANT_WARPS;
    for (uint64_t v = static_cast<uint64_t>(blockIdx.x) * QUANT_WARPS + threadIdx.x / 32; v < vectors; v += stride) {
        const uint32_t t = static_cast<uint32_t>(v / (2u * p.heads));
        const uint32_t rest = static_cast<uint32_t>(v % (2u * p.heads));
        const int kv = rest >= p.heads ? 1 : 0;
        const uint32_t head = rest - kv * p.heads;
        int64_t slot = lane == 0 ? cache_slot(p, t) : 0;
        slot = __shfl_sync(0xffffffffu, slot, 0);
        if (slot < 0) continue;
        const uint64_t at = static_cast<uint64_t>(slot) * p.heads + head;
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
                codes[j] = e4m3_code(load_element(p.rows[kv], p.dtype[kv], row + j), d);
            }
        } else {
            const float scale = p.scales[kv][at];
            for (uint32_t j = lane; j < p.head_dim; j += 32) {
                store_element(p.rows[kv], p.dtype[kv], row + j, __fmul_rn(e4m3_value(codes[j]), scale));
            }
        }
    }
}

template <int DT, bool WRITE>
int launch_cache_vectors(const m3c_cache_params &p, const cache_shape &shape, cudaStream_t stream)
{
    const uint32_t each = (QUANT_THREADS >> shape.lane_shift) * (WRITE ? CACHE_DEPTH_WRITE : CACHE_DEPTH_READ);
    cache_kernel<DT, WRITE><<<(shape.vectors - 1u) / each + 1u, QUANT_THREADS, 0, stream>>>(p, shape);
    return static_cast<int>(cudaGetLastError());
}

template <bool WRITE>
int launch_cache(const m3c_cache_params &p, cudaStream_t stream)
{
    const uint64_t vectors = static_cast<uint64_t>(p.row_count) * 2u * p.heads;
    const uint64_t step = p.dtype[0] == M3C_F32 ? 4u : 8u;  // elements of 16 bytes
    bool fits = p.dtype[0] == p.dtype[1] && p.head_dim % 8u == 0u && p.head_dim <= 256u && vectors < (1ull << 31);
    for (int k = 0; k < 2; ++k) {
        fits = fits && aligned_to(p.rows[k], 16) && p.token_stride[k] % step == 0u && p.head_stride[k] % step == 0u;
    }
    if (fits) {
        cache_shape shape;
        m3c_fastdiv_init(&shape.of_row, 2u * p.heads);
        shape.vectors = static_cast<uint32_t>(vectors);
        shape.lane_shift = 0u;
        while ((8u << shape.lane_shift) < p.head_dim) ++shape.lane_shift;
        shape.lanes = 1u << shape.lane_shift;
        switch (p.dtype[0]) {
        case M3C_F16: return launch_cache_vectors<M3C_F16, WRITE>(p, shape, stream);
        case M3C_BF16: return launch_cache_vectors<M3C_BF16, WRITE>(p, shape, stream);
        default: return launch_cache_vectors<M3C_F32, WRITE>(p, shape, stream);
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
    const m3c_norm_e4m3_params &p = *params;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const uint64_t step = p.dtype == M3C_F32 ? 4u : 8u;  // elements of 16 bytes
    const bool vectors = p.width % 8u == 0u && p.group % 8u == 0u && p.x_stride % step == 0u && aligned_to(p.x, 16) &&
                         aligned_to(p.scale, 16) && aligned_to(p.codes, 8) &&
                         (p.resid_b == nullptr || (p.resid_stride % step == 0u && aligned_to(p.resid_b, 16))) &&
                         (p.sum_out == nullptr || (p.sum_stride % step == 0u && aligned_to(p.sum_out, 16)));
    if (p.width <= (vectors ? NORM_WIDEST : NORM_WIDEST / 2u)) {
        switch (p.dtype) {
        case M3C_F16: return norm_mode<M3C_F16>(p, vectors, s);
        case M3C_BF16: return norm_mode<M3C_BF16>(p, vectors, s);
        default: return norm_mode<M3C_F32>(p, vectors, s);
        }
    }
    const size_t row_bytes = p.width * sizeof(float);
    const bool kept = row_bytes <= NORM_KEPT_BYTES;
    if (kept && row_bytes > 48u * 1024u) {
        cudaFuncSetAttribute(norm_e4m3_any_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(NORM_KEPT_BYTES));
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
