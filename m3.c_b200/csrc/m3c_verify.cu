// Verification of drafted tokens (sm_100a).
//
// Draft i of a sequence is accepted while u_i q_i(d_i) < p_i(d_i); behind the m
// accepted ones a token is drawn from the weights
//   w_j = max(p_m(j) - q_m(j), 0)   after a rejection (p_m(j) if all are zero),
//   w_j = p_m(j)                    where every draft was accepted,
// as the first j whose running sum exceeds u_n * total.  The product of two
// F32 numbers is exact in 64 bits, and so are the comparisons that accept; the
// running sums are 64-bit sums, since a vocabulary of 10^5 tokens puts F32
// rounding errors of a sum past whole tokens' probabilities.

#include <cuda_runtime.h>

#include <cstdint>

#include "m3c_device.cuh"
#include "m3c_e4m3.cuh"
#include "m3c_kernels.h"

namespace m3c {
namespace {

constexpr int VERIFY_THREADS = 256;

__device__ __forceinline__ bool valid_probability(float p)
{
    return p >= 0.0f && p < as_float(0x7f800000u);  // false for a NaN
}

// A CTA per sequence.
__global__ void __launch_bounds__(VERIFY_THREADS) verify_kernel(const __grid_constant__ m3c_verify_params p)
{
    __shared__ int accepted;         // -1: the sequence is bad
    __shared__ int rejected;         // a draft was rejected behind them
    __shared__ double sums[2][VERIFY_THREADS];
    __shared__ unsigned found;
    __shared__ unsigned last_positive;
    __shared__ int bad;
    if (p.status != nullptr) {
        if (failed_before(p.status, p.skip_before)) return;
        if (p.first_of_run && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(&p.status->runs_started, 1u);
    }
    const uint32_t tid = threadIdx.x;
    for (uint64_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int32_t *tokens = p.tokens + b * (p.drafts + 1);
        const int32_t *drafted = p.draft_tokens + b * p.drafts;
        const float *uniforms = p.uniforms + b * (p.drafts + 1);
        if (tid == 0) {
            const int64_t length = p.lengths != nullptr ? p.lengths[b] : static_cast<int64_t>(p.drafts);
            int m = 0;
            int no = 0;
            if (length < 0 || length > static_cast<int64_t>(p.drafts)) m = -1;
            while (m >= 0 && m < length) {
                const int64_t d = drafted[m];
                const float u = uniforms[m];
                if (d < 0 || d >= p.vocabulary || !(u >= 0.0f && u < 1.0f)) {
                    m = -1;
                    break;
                }
                const float t = load_element(p.target, p.dtype, (b * (p.drafts + 1) + m) * p.target_stride + d);
                const float q =
                    p.draft != nullptr ? load_element(p.draft, p.dtype, (b * p.drafts + m) * p.draft_stride + d) : 1.0f;
                if (!valid_probability(t) || !valid_probability(q)) {
                    m = -1;
                    break;
                }
                if (!(static_cast<double>(u) * static_cast<double>(q) < static_cast<double>(t))) {
                    no = 1;
                    break;
                }
                ++m;
            }
            const float u = uniforms[p.drafts];
            if (!(u >= 0.0f && u < 1.0f)) m = -1;
            accepted = m;
            rejected = no;
            found = 0xffffffffu;
            last_positive = 0u;
            bad = 0;
        }
        __syncthreads();
        const int m = accepted;
        if (m >= 0) {
            const uint64_t target = (b * (p.drafts + 1) + m) * p.target_stride;
            const uint64_t draft = (b * p.drafts + m) * p.draft_stride;
            const int64_t given = rejected && p.draft == nullptr ? drafted[m] : -1;
            // thread i owns a contiguous part of the vocabulary
            const uint32_t part = (p.vocabulary + VERIFY_THREADS - 1) / VERIFY_THREADS;
            const uint32_t from = min(tid * part, p.vocabulary);
            const uint32_t to = min(from + part, p.vocabulary);
            auto weight = [&](uint32_t j, bool residual, bool &ok) {
                const float t = load_element(p.target, p.dtype, target + j);
                ok = ok && valid_probability(t);
                double w = static_cast<double>(t);
                if (residual && p.draft != nullptr) {
                    const float q = load_element(p.draft, p.dtype, draft + j);
                    ok = ok && valid_probability(q);
                    w = fmax(w - static_cast<double>(q), 0.0);
                } else if (residual && j == given) {
                    w = 0.0;
                }
                return w;
            };
            bool ok = true;
            double whole = 0.0;
            double rest = 0.0;
            for (uint32_t j = from; j < to; ++j) {
                whole += weight(j, false, ok);
                rest += weight(j, rejected != 0, ok);
            }
            sums[0][tid] = rest;
            sums[1][tid] = whole;
            if (!ok) bad = 1;
            __syncthreads();
            if (!bad) {
                double total[2] = {0.0, 0.0};
                double before[2] = {0.0, 0.0};
                for (uint32_t i = 0; i < VERIFY_THREADS; ++i) {
                    if (i == tid) {
                        before[0] = total[0];
                        before[1] = total[1];
                    }
                    total[0] += sums[0][i];
                    total[1] += sums[1][i];
                }
                const int which = total[0] > 0.0 ? 0 : 1;
                const double aim = static_cast<double>(uniforms[p.drafts]) * total[which];
                double running = before[which];
                if (!(total[which] > 0.0)) {
                    bad = 1;
                } else if (running + sums[which][tid] > aim) {
                    for (uint32_t j = from; j < to; ++j) {
                        const double w = weight(j, which == 0 && rejected != 0, ok);
                        running += w;
                        if (w > 0.0) atomicMax(&last_positive, j);
                        if (w > 0.0 && running > aim) {
                            atomicMin(&found, j);
                            break;
                        }
                    }
                }
            }
        }
        __syncthreads();
        const bool fine = m >= 0 && !bad;
        for (uint64_t i = tid; i <= p.drafts; i += VERIFY_THREADS) {
            int32_t token = -1;
            if (fine && i < static_cast<uint64_t>(m)) token = drafted[i];
            if (fine && i == static_cast<uint64_t>(m)) {
                token = static_cast<int32_t>(found != 0xffffffffu ? found : last_positive);
            }
            tokens[i] = token;
        }
        if (tid == 0) p.accepted[b] = fine ? m : -1;
        __syncthreads();
    }
}

}  // namespace
}  // namespace m3c

extern "C" int m3c_launch_verify(const m3c_verify_params *params, void *stream)
{
    const unsigned grid = static_cast<unsigned>(params->batch == 0 ? 1 : (params->batch < 65536u ? params->batch : 65536u));
    m3c::verify_kernel<<<grid, m3c::VERIFY_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(*params);
    return static_cast<int>(cudaGetLastError());
}
