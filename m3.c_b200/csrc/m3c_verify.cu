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
//
// Bytes bound large batches in F32 (one row of each model per sequence), latency
// small ones: 128 sequences over 131072 tokens in F32 take 29.0 us (4.6 TB/s, 0.70
// of the measured copy rate), one over 32000 takes 6.6 us, nearly all of it loads
// that wait for one another.  16-bit rows take as long for half the bytes (27.7 us,
// 0.37; 256 sequences over 32000 tokens 17.9 us, 0.28): a lane has one load per
// model on its way and then 16 numbers to widen, convert and add.  Rows aligned
// for no vector are read by single elements (131073 tokens in F32: 37.8 us, 0.54).
// A cluster of CTAs takes a sequence, its warps one
// contiguous part of the vocabulary each.  One pass over the rows sums the
// parts; the parts' sums go round through the CTAs' shared memory, and the CTA
// that owns the part in which the running sum passes the aim looks for the token
// there, in a few KB that are still in the L2.

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "m3c_device.cuh"
#include "m3c_e4m3.cuh"
#include "m3c_kernels.h"

namespace cg = cooperative_groups;

namespace m3c {
namespace {

constexpr int VERIFY_THREADS = 512;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int VERIFY_MOST_CTAS = 8;  // of a cluster

__device__ __forceinline__ bool valid_probability(float p)
{
    return p >= 0.0f && p < as_float(0x7f800000u);  // false for a NaN
}

// VEC consecutive probabilities as they are stored.
template <int DT, int VEC>
struct Stored {
    static constexpr int WORDS = VEC == 1 ? 1 : 4;
    uint32_t w[WORDS];

    __device__ __forceinline__ void load(const void *base, uint64_t element)
    {
        if constexpr (VEC > 1) {
            const uint4 q = __ldg(reinterpret_cast<const uint4 *>(static_cast<const char *>(base) +
                                                                  element * (DT == M3C_F32 ? 4u : 2u)));
            w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
        } else if constexpr (DT == M3C_F32) {
            w[0] = __ldg(static_cast<const uint32_t *>(base) + element);
        } else {
            w[0] = __ldg(static_cast<const uint16_t *>(base) + element);
        }
    }

    __device__ __forceinline__ void widen(float (&x)[VEC]) const
    {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if constexpr (DT == M3C_F32) {
                x[i] = as_float(w[i]);
            } else if constexpr (DT == M3C_BF16) {
                x[i] = as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
            } else {
                const float2 two = __half22float2(*reinterpret_cast<const __half2 *>(&w[i / 2]));
                x[i] = i % 2 ? two.y : two.x;
            }
        }
    }
};

// The drafts' fate, found by one warp: how many are accepted, -1 for a bad
// sequence; `rejected` where one was refused behind them.
__device__ __forceinline__ int accepted_drafts(const m3c_verify_params &p, uint64_t b, bool &rejected)
{
    const uint32_t lane = threadIdx.x % 32u;
    const int64_t most = static_cast<int64_t>(p.drafts);
    const float *uniforms = p.uniforms + b * (p.drafts + 1u);
    // read together: a draft's probabilities wait for its token alone
    const int64_t length = p.lengths != nullptr ? p.lengths[b] : most;
    const float last = uniforms[most];
    bool bad_sequence = length < 0 || length > most || !(last >= 0.0f && last < 1.0f);
    rejected = false;
    for (int64_t i0 = 0; i0 < most; i0 += 32) {
        const int64_t i = i0 + lane;
        bool bad = false;
        bool refused = false;
        if (i < most) {
            const int64_t d = p.draft_tokens[b * p.drafts + i];
            const float u = uniforms[i];
            // behind the sequence's drafts nothing counts, and no row is read
            if (i < length) {
                bad = d < 0 || d >= p.vocabulary || !(u >= 0.0f && u < 1.0f);
                if (!bad) {
                    const float t = load_element(p.target, p.dtype, (b * (p.drafts + 1u) + i) * p.target_stride + d);
                    const float q = p.draft == nullptr
                                        ? 1.0f
                                        : load_element(p.draft, p.dtype, (b * p.drafts + i) * p.draft_stride + d);
                    bad = !valid_probability(t) || !valid_probability(q);
                    refused = !(static_cast<double>(u) * static_cast<double>(q) < static_cast<double>(t));
                }
            }
        }
        if (bad_sequence || i0 >= length) break;
        const uint32_t stop = __ballot_sync(0xffffffffu, bad || refused);
        const uint32_t bads = __ballot_sync(0xffffffffu, bad);
        if (stop != 0u) {
            const int at = __ffs(static_cast<int>(stop)) - 1;
            if ((bads >> at) & 1u) return -1;
            rejected = true;
            return static_cast<int>(i0) + at;
        }
    }
    return bad_sequence ? -1 : static_cast<int>(length);
}

// The rows a token is drawn from.
struct weights_of {
    const void *target;
    const void *draft;      // NULL: none to subtract
    uint64_t target_at;
    uint64_t draft_at;
    int64_t given;          // the token without weight, or -1
};

// The largest of `largest` and VEC probabilities as integers.  Adding +0 makes a
// +0 of a -0, and then the integers of all valid probabilities are below that
// of the infinity, those of negative ones and NaN above it.
template <int VEC>
__device__ __forceinline__ uint32_t largest_word(uint32_t largest, const float (&x)[VEC])
{
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const uint32_t word = as_bits(__fadd_rn(x[i], 0.0f));
        largest = word > largest ? word : largest;
    }
    return largest;
}

__device__ __forceinline__ double weight(float t, float q)
{
    return t > q ? static_cast<double>(t) - static_cast<double>(q) : 0.0;
}

// The sum of weights on its way: max(t - q, 0) is the F32 number d = max(t, q) -
// q and what its rounding lost, which F32 holds exactly (T. J. Dekker, "A
// floating-point technique for extending the available precision", Numer. Math.
// 18, 1971: |max(t, q)| >= |q|).  The d are summed in 64 bits, with one
// conversion each instead of two; what was lost is below 2^-24 of that, and is
// summed in F32 for some eight numbers before it joins them, off by less than
// 2^-45 of their sum.
struct running_sum {
    double high = 0.0;
    float low = 0.0f;

    __device__ __forceinline__ void add(float t, float q)
    {
        const float more = fmaxf(t, q);
        const float d = __fsub_rn(more, q);
        low = __fadd_rn(low, __fsub_rn(__fsub_rn(more, d), q));
        high += static_cast<double>(d);
    }

    __device__ __forceinline__ void join()
    {
        high += static_cast<double>(low);
        low = 0.0f;
    }
};

__device__ __forceinline__ double shuffle_up(double v, int d)
{
    return __shfl_up_sync(0xffffffffu, v, d);
}

// VEC elements (16 bytes) a load where both models' rows are aligned for it,
// else one.  `part` elements per warp, a multiple of VEC.
template <int DT, int VEC>
__global__ void __launch_bounds__(VERIFY_THREADS, 1024 / VERIFY_THREADS)
    verify_kernel(const __grid_constant__ m3c_verify_params p, uint32_t part)
{
    constexpr int LOADS = VEC == 1 ? 8 : VEC == 4 ? 4 : 1;  // on their way per lane and model
    constexpr int PARTS = VERIFY_MOST_CTAS * VERIFY_WARPS;
    __shared__ double mine[2][VERIFY_WARPS];    // the sums of this CTA's parts, per round
    __shared__ double parts[PARTS];
    __shared__ double scan[VERIFY_WARPS];
    __shared__ double total;
    __shared__ double before;                   // the sum of the parts before `chosen`
    __shared__ int chosen;
    __shared__ int fate;                        // accepted drafts, or -1
    __shared__ int refused;
    __shared__ uint32_t found;
    __shared__ uint32_t last_positive;
    if (p.status != nullptr) {
        // the same for all threads of a cluster: a session runs launches side by
        // side only where none of them can fail, so the status does not change
        // meanwhile
        if (failed_before(p.status, p.skip_before)) return;
        if (p.first_of_run && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(&p.status->runs_started, 1u);
    }
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks();
    const uint32_t rank = cluster.block_rank();
    const uint64_t b = blockIdx.x / ctas;
    if (b >= p.batch) return;  // the whole cluster
    const uint32_t tid = threadIdx.x;
    const uint32_t lane = tid % 32u;
    const uint32_t warp = tid / 32u;
    if (warp == 0u) {
        bool rejected;
        const int m = accepted_drafts(p, b, rejected);
        if (lane == 0u) {
            fate = m;
            refused = rejected ? 1 : 0;
            found = 0xffffffffu;
            last_positive = 0u;
        }
    }
    __syncthreads();
    const int m = fate;
    bool fine = m >= 0;
    bool rejected = refused != 0;
    const int32_t *drafted = p.draft_tokens + b * p.drafts;
    uint32_t owner = 0;
    if (fine) {
        weights_of from;
        from.target = p.target;
        from.target_at = (b * (p.drafts + 1u) + m) * p.target_stride;
        from.draft_at = (b * p.drafts + m) * p.draft_stride;
        for (int round = 0;; ++round) {
            from.draft = rejected ? p.draft : nullptr;
            from.given = rejected && p.draft == nullptr ? drafted[m] : -1;
            const uint64_t begin = static_cast<uint64_t>(rank * VERIFY_WARPS + warp) * part;
            const uint32_t start = static_cast<uint32_t>(begin < p.vocabulary ? begin : p.vocabulary);
            const uint32_t end = static_cast<uint32_t>(begin + part < p.vocabulary ? begin + part : p.vocabulary);
            running_sum run[2];
            uint32_t largest = 0u;
            auto add = [&](uint32_t j, const Stored<DT, VEC> &target, const Stored<DT, VEC> &draft) {
                float t[VEC];
                float q[VEC];
                target.widen(t);
                largest = largest_word(largest, t);
                if (from.draft != nullptr) {
                    draft.widen(q);
                    largest = largest_word(largest, q);
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    if (from.draft == nullptr) q[i] = 0.0f;
                    if (j + i == from.given) t[i] = 0.0f;
                    run[i % 2].add(t[i], q[i]);
                }
            };
            uint32_t j = start + lane * VEC;
            for (; j + (LOADS - 1) * 32u * VEC + VEC <= end; j += LOADS * 32u * VEC) {
                Stored<DT, VEC> target[LOADS];
                Stored<DT, VEC> draft[LOADS];
#pragma unroll
                for (int l = 0; l < LOADS; ++l) target[l].load(from.target, from.target_at + j + l * 32u * VEC);
                if (from.draft != nullptr) {
#pragma unroll
                    for (int l = 0; l < LOADS; ++l) draft[l].load(from.draft, from.draft_at + j + l * 32u * VEC);
                }
#pragma unroll
                for (int l = 0; l < LOADS; ++l) add(j + l * 32u * VEC, target[l], draft[l]);
                run[0].join();
                run[1].join();
            }
            for (; j + VEC <= end; j += 32u * VEC) {
                Stored<DT, VEC> target;
                Stored<DT, VEC> draft;
                target.load(from.target, from.target_at + j);
                if (from.draft != nullptr) draft.load(from.draft, from.draft_at + j);
                add(j, target, draft);
            }
            for (; j < end; ++j) {  // less than VEC elements, at the vocabulary's end
                float t[1] = {load_element(from.target, DT, from.target_at + j)};
                float q[1] = {from.draft != nullptr ? load_element(from.draft, DT, from.draft_at + j) : 0.0f};
                largest = largest_word(largest_word(largest, t), q);
                run[0].add(j == from.given ? 0.0f : t[0], q[0]);
            }
            run[0].join();
            run[1].join();
            double sum = run[0].high + run[1].high;
            const bool valid = largest < 0x7f800000u;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            // an invalid probability makes every sum that holds it a NaN
            if (!__all_sync(0xffffffffu, valid)) sum = __longlong_as_double(0x7ff8000000000000ll);
            if (lane == 0u) mine[round][warp] = sum;
            cluster.sync();
            if (tid < ctas * VERIFY_WARPS) {
                parts[tid] = *cluster.map_shared_rank(&mine[round][tid % VERIFY_WARPS], tid / VERIFY_WARPS);
            }
            __syncthreads();
            if (warp == 0u) {
                // four parts per lane, their running sums in the order of the
                // vocabulary
                double own[PARTS / 32];
                double run = 0.0;
#pragma unroll
                for (int k = 0; k < PARTS / 32; ++k) {
                    const uint32_t at = lane * (PARTS / 32) + k;
                    own[k] = at < ctas * VERIFY_WARPS ? parts[at] : 0.0;
                    run += own[k];
                }
                double up = run;
                for (int d = 1; d < 32; d <<= 1) {
                    const double other = shuffle_up(up, d);
                    if (lane >= static_cast<uint32_t>(d)) up += other;
                }
                const double all = __shfl_sync(0xffffffffu, up, 31);
                run = shuffle_up(up, 1);
                if (lane == 0u) run = 0.0;
                const double aim = static_cast<double>(p.uniforms[b * (p.drafts + 1u) + p.drafts]) * all;
                // the first part that passes the aim; where rounding leaves
                // none, the last with any weight
                int passes = PARTS;
                int heavy = -1;
                double base = 0.0;
                double heavy_base = 0.0;
#pragma unroll
                for (int k = 0; k < PARTS / 32; ++k) {
                    const int at = static_cast<int>(lane) * (PARTS / 32) + k;
                    if (own[k] > 0.0) {
                        heavy = at;
                        heavy_base = run;
                        if (passes == PARTS && run + own[k] > aim) {
                            passes = at;
                            base = run;
                        }
                    }
                    run += own[k];
                }
                const int first = __reduce_min_sync(0xffffffffu, passes);
                const int heaviest = __reduce_max_sync(0xffffffffu, heavy);
                const int pick = first < PARTS ? first : heaviest;
                if (pick >= 0 && static_cast<int>(lane) == pick / (PARTS / 32)) {
                    chosen = pick;
                    before = first < PARTS ? base : heavy_base;
                }
                if (lane == 0u) total = all;
            }
            __syncthreads();
            fine = total > 0.0;  // false for a NaN
            if (fine || !(total == 0.0) || !rejected) break;
            rejected = false;  // nothing is left of the target: draw from all of it
        }
        // no CTA leaves before the others have read its sums
        cg::this_cluster().barrier_arrive();
        owner = fine ? static_cast<uint32_t>(chosen) / VERIFY_WARPS : 0u;
        if (fine && rank == owner) {
            const double aim = static_cast<double>(p.uniforms[b * (p.drafts + 1u) + p.drafts]) * total;
            const uint32_t start = static_cast<uint32_t>(chosen) * part;
            const uint32_t end = static_cast<uint32_t>(
                static_cast<uint64_t>(start) + part < p.vocabulary ? start + part : p.vocabulary);
            double run = before;
            for (uint32_t j0 = start; j0 < end; j0 += VERIFY_THREADS * VEC) {
                const uint32_t j = j0 + tid * VEC;
                double w[VEC];
                double sum = 0.0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) w[i] = 0.0;
                if (j + VEC <= end) {
                    Stored<DT, VEC> target;
                    Stored<DT, VEC> draft;
                    float t[VEC];
                    float q[VEC] = {};
                    target.load(from.target, from.target_at + j);
                    target.widen(t);
                    if (from.draft != nullptr) {
                        draft.load(from.draft, from.draft_at + j);
                        draft.widen(q);
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) w[i] = j + i == from.given ? 0.0 : weight(t[i], q[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        if (j + i < end && j + i != from.given) {
                            const float t = load_element(from.target, DT, from.target_at + j + i);
                            const float q =
                                from.draft != nullptr ? load_element(from.draft, DT, from.draft_at + j + i) : 0.0f;
                            w[i] = weight(t, q);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum += w[i];
                double up = sum;
                for (int d = 1; d < 32; d <<= 1) {
                    const double other = shuffle_up(up, d);
                    if (lane >= static_cast<uint32_t>(d)) up += other;
                }
                if (lane == 31u) scan[warp] = up;
                __syncthreads();
                double mark = run;
                for (uint32_t k = 0; k < VERIFY_WARPS; ++k) {
                    if (k < warp) mark += scan[k];
                    run += scan[k];
                }
                const double lower = shuffle_up(up, 1);
                if (lane > 0u) mark += lower;
                uint32_t positive = 0u;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    mark += w[i];
                    if (w[i] > 0.0) {
                        positive = j + i;
                        if (mark > aim) {
                            atomicMin(&found, j + i);
                            break;
                        }
                    }
                }
                if (positive != 0u) atomicMax(&last_positive, positive);
                __syncthreads();
                if (found != 0xffffffffu) break;
            }
        }
    }
    if (rank == owner) {
        for (uint64_t i = tid; i <= p.drafts; i += VERIFY_THREADS) {
            int32_t token = -1;
            if (fine && i < static_cast<uint64_t>(m)) token = drafted[i];
            // where rounding leaves no sum past the aim, the last token with
            // any weight
            if (fine && i == static_cast<uint64_t>(m)) {
                token = static_cast<int32_t>(found != 0xffffffffu ? found : last_positive);
            }
            p.tokens[b * (p.drafts + 1u) + i] = token;
        }
        if (tid == 0u) p.accepted[b] = fine ? m : -1;
    }
    if (m >= 0) cg::this_cluster().barrier_wait();
}

template <int DT, int VEC>
int launch_verify(const m3c_verify_params &p, cudaStream_t stream)
{
    int device = 0;
    int sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess) {
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    }
    // as many CTAs for a sequence as run at the same time (two per SM), while
    // each keeps some elements per thread.  128 sequences over 131072 tokens
    // in F32: 29.0 us with 2 CTAs each, 31.8 with 4, 33.2 with 1
    uint32_t ctas = VERIFY_MOST_CTAS;
    while (ctas > 1u && (p.batch * ctas > 2u * static_cast<uint64_t>(sms) ||
                         p.vocabulary < ctas * static_cast<uint32_t>(VERIFY_THREADS))) {
        ctas >>= 1;
    }
    const uint32_t warps = ctas * VERIFY_WARPS;
    const uint32_t part = ((p.vocabulary + warps - 1u) / warps + VEC - 1u) / VEC * VEC;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = ctas;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    config.gridDim = dim3(static_cast<unsigned>(p.batch == 0 ? ctas : p.batch * ctas));
    config.blockDim = dim3(VERIFY_THREADS);
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    const cudaError_t code = cudaLaunchKernelEx(&config, verify_kernel<DT, VEC>, p, part);
    if (code != cudaSuccess) return static_cast<int>(code);
    return static_cast<int>(cudaGetLastError());
}

template <int DT>
int verify_vectors(const m3c_verify_params &p, cudaStream_t stream)
{
    constexpr int VEC = DT == M3C_F32 ? 4 : 8;
    const bool aligned = reinterpret_cast<uintptr_t>(p.target) % 16u == 0u && p.target_stride % VEC == 0u &&
                         (p.draft == nullptr ||
                          (reinterpret_cast<uintptr_t>(p.draft) % 16u == 0u && p.draft_stride % VEC == 0u));
    return aligned ? launch_verify<DT, VEC>(p, stream) : launch_verify<DT, 1>(p, stream);
}

}  // namespace
}  // namespace m3c

extern "C" int m3c_launch_verify(const m3c_verify_params *params, void *stream)
{
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (params->dtype) {
    case M3C_F16: return m3c::verify_vectors<M3C_F16>(*params, s);
    case M3C_BF16: return m3c::verify_vectors<M3C_BF16>(*params, s);
    default: return m3c::verify_vectors<M3C_F32>(*params, s);
    }
}
