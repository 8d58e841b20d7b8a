// E4M3 outputs (sm_100a): the RMS norm with the residual's addition into codes
// and scales, and the paged key/value cache, quantised as it is written and
// read back.

#include <cuda_runtime.h>

#include <cstdint>

#include "m3c_device.cuh"
#include "m3c_e4m3.cuh"
#include "m3c_kernels.h"

namespace m3c {
namespace {

constexpr int QUANT_THREADS = 256;
constexpr int QUANT_WARPS = QUANT_THREADS / 32;

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
// Any shape: one CTA per row, three passes over the row (the sum of squares,
// which stores the residual sum; per group the largest |y|; the codes).  The
// second and third read the row from the caches.
__global__ void __launch_bounds__(QUANT_THREADS)
    norm_e4m3_any_kernel(const __grid_constant__ m3c_norm_e4m3_params p)
{
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
        float squares = 0.0f;
        for (uint64_t j = threadIdx.x; j < p.width; j += QUANT_THREADS) {
            float h = load_element(p.x, p.dtype, x0 + j);
            if (p.resid_b != nullptr) {
                h = round_to(p.dtype, __fadd_rn(h, load_element(p.resid_b, p.dtype, r0 + j)));
                if (p.sum_out != nullptr) store_element(p.sum_out, p.dtype, s0 + j, h);
            }
            squares = __fmaf_rn(h, h, squares);
        }
        squares = warp_sum(squares);
        if (lane == 0) part[warp] = squares;
        __syncthreads();
        squares = 0.0f;
        for (int w = 0; w < QUANT_WARPS; ++w) squares = __fadd_rn(squares, part[w]);
        const float inverse =
            __frsqrt_rn(__fadd_rn(__fdiv_rn(squares, static_cast<float>(p.width)), p.epsilon));
        // the stored sum is h (and may be the input's own storage by now)
        const bool stored = p.sum_out != nullptr;
        auto normed = [&](uint64_t j) {
            float h = stored ? load_element(p.sum_out, p.dtype, s0 + j) : load_element(p.x, p.dtype, x0 + j);
            if (!stored && p.resid_b != nullptr) {
                h = round_to(p.dtype, __fadd_rn(h, load_element(p.resid_b, p.dtype, r0 + j)));
            }
            return __fmul_rn(__fmul_rn(h, inverse), load_element(p.scale, p.scale_dtype, j));
        };
        uint8_t *codes = static_cast<uint8_t *>(p.codes) + row * p.width;
        if (groups >= QUANT_WARPS) {
            for (uint64_t g = warp; g < groups; g += QUANT_WARPS) {
                uint32_t largest = 0u;
                for (uint64_t j = lane; j < p.group; j += 32) {
                    const uint32_t m = magnitude_bits(normed(g * p.group + j));
                    largest = m > largest ? m : largest;
                }
                const e4m3_divisor d = e4m3_divide_by(e4m3_scale(warp_max(largest)));
                if (lane == 0) p.code_scales[row * groups + g] = d.scale;
                for (uint64_t j = lane; j < p.group; j += 32) {
                    codes[g * p.group + j] = e4m3_code(normed(g * p.group + j), d);
                }
            }
        } else {
            for (uint64_t g = 0; g < groups; ++g) {
                uint32_t largest = 0u;
                for (uint64_t j = threadIdx.x; j < p.group; j += QUANT_THREADS) {
                    const uint32_t m = magnitude_bits(normed(g * p.group + j));
                    largest = m > largest ? m : largest;
                }
                largest = warp_max(largest);
                if (lane == 0) top[warp] = largest;
                __syncthreads();
                for (int w = 0; w < QUANT_WARPS; ++w) largest = top[w] > largest ? top[w] : largest;
                const e4m3_divisor d = e4m3_divide_by(e4m3_scale(largest));
                if (threadIdx.x == 0) p.code_scales[row * groups + g] = d.scale;
                for (uint64_t j = threadIdx.x; j < p.group; j += QUANT_THREADS) {
                    codes[g * p.group + j] = e4m3_code(normed(g * p.group + j), d);
                }
                __syncthreads();
            }
        }
        __syncthreads();
    }
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

template <bool WRITE>
int launch_cache(const m3c_cache_params &p, void *stream)
{
    const uint64_t vectors = static_cast<uint64_t>(p.row_count) * 2u * p.heads;
    const unsigned grid = capped_grid((vectors + QUANT_WARPS - 1) / QUANT_WARPS, 32u);
    cache_any_kernel<WRITE><<<grid, QUANT_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace
}  // namespace m3c

extern "C" int m3c_launch_norm_e4m3(const m3c_norm_e4m3_params *params, void *stream)
{
    const unsigned grid = m3c::capped_grid(params->rows, 32u);
    m3c::norm_e4m3_any_kernel<<<grid, m3c::QUANT_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*params);
    return static_cast<int>(cudaGetLastError());
}

extern "C" int m3c_launch_cache_write(const m3c_cache_params *params, void *stream)
{
    return m3c::launch_cache<true>(*params, stream);
}

extern "C" int m3c_launch_cache_read(const m3c_cache_params *params, void *stream)
{
    return m3c::launch_cache<false>(*params, stream);
}
