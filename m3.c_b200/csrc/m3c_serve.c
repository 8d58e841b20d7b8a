/* The serving operators' host side: argument checks, the device they run on,
 * and the paged E4M3 cache object (include/m3_cuda.h, "Serving operators").
 * The kernels are in m3c_quant.cu and m3c_verify.cu. */

#include "m3c_internal.h"

#include <cuda_runtime_api.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>

struct m3_cuda_cache {
    m3_cuda_cache_options options;
    int device;
    unsigned char *arena;
    size_t arena_bytes;
    uint8_t *codes[2];
    float *scales[2];
    unsigned long long *first_skipped;   /* device; the word behind it holds
                                            a synchronise's copy */
    unsigned long long *seen;            /* pinned */
};

static m3_status cuda_failure(m3_error *error, cudaError_t code,
                              const char *what)
{
    (void)cudaGetLastError();
    return m3c_error_set(error,
                         code == cudaErrorMemoryAllocation
                             ? M3_STATUS_OUT_OF_MEMORY
                             : M3_STATUS_INTERNAL,
                         "%s: %s", what, cudaGetErrorString(code));
}

/* Make `device` current; `previous` is what leave_device restores. */
static m3_status enter_device(int device, int *previous, m3_error *error)
{
    cudaError_t code = cudaGetDevice(previous);

    if (code == cudaErrorNoDevice || code == cudaErrorInsufficientDriver) {
        (void)cudaGetLastError();
        return m3c_error_set(error, M3_STATUS_UNSUPPORTED,
                             "no CUDA device is available");
    }
    if (code == cudaSuccess && *previous != device) {
        code = cudaSetDevice(device);
        if (code == cudaErrorInvalidDevice) {
            (void)cudaGetLastError();
            return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                                 "CUDA device %d is not available", device);
        }
    }
    return code == cudaSuccess
               ? M3_STATUS_OK
               : cuda_failure(error, code, "cannot select device");
}

static void leave_device(int device, int previous)
{
    if (previous != device) {
        (void)cudaSetDevice(previous);
    }
}

static m3_status launched(int code, m3_error *error)
{
    if (code != 0) {
        (void)cudaGetLastError();
        return m3c_error_set(error, M3_STATUS_INTERNAL,
                             "kernel launch failed: %s",
                             m3c_cuda_error_string(code));
    }
    m3_error_reset(error);
    return M3_STATUS_OK;
}

/* ------------------------------------------------- checks of arguments */

/* A strided tensor of rows: [rows, extent], `stride` elements from row to
 * row.  The byte span [begin, end) is what the overlap checks compare. */
typedef struct {
    const char *name;
    uintptr_t begin;
    uintptr_t end;
    uint64_t stride;
} span;

static m3_status rows_span(span *s, const char *name, const void *data,
                           uint64_t rows, uint64_t extent, uint64_t stride,
                           uint64_t element, m3_error *error)
{
    uint64_t count;

    s->name = name;
    s->begin = (uintptr_t)data;
    s->end = s->begin;
    s->stride = stride == 0U ? extent : stride;
    if (rows == 0U || extent == 0U) {
        return M3_STATUS_OK;
    }
    if (data == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "%s is required", name);
    }
    if (s->begin % element != 0U) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "%s is not aligned to its element size", name);
    }
    if (s->stride < extent) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "%s stride is less than its row", name);
    }
    if (rows - 1U > (UINT64_MAX / 8U - extent) / s->stride) {
        return m3c_error_set(error, M3_STATUS_OVERFLOW, "%s size overflows",
                             name);
    }
    count = (rows - 1U) * s->stride + extent;
    if (count > (UINTPTR_MAX - s->begin) / element) {
        return m3c_error_set(error, M3_STATUS_OVERFLOW, "%s size overflows",
                             name);
    }
    s->end = s->begin + count * element;
    return M3_STATUS_OK;
}

static bool overlapping(const span *a, const span *b)
{
    return a->begin < b->end && b->begin < a->end;
}

static m3_status check_apart(const span *output, const span *other,
                             m3_error *error)
{
    if (!overlapping(output, other)) {
        return M3_STATUS_OK;
    }
    return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT, "%s overlaps %s",
                         output->name, other->name);
}

static m3_status check_float(m3_dtype dtype, const char *name, m3_error *error)
{
    if (m3c_dtype_float(dtype)) {
        return M3_STATUS_OK;
    }
    return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                         "%s must be F32, F16 or BF16", name);
}

/* ------------------------------------------------------ RMS norm in E4M3 */

void m3_cuda_rms_norm_e4m3_args_init(m3_cuda_rms_norm_e4m3_args *args)
{
    if (args != NULL) {
        memset(args, 0, sizeof(*args));
        args->epsilon = 1e-6F;
    }
}

m3_status m3_cuda_rms_norm_e4m3(int device, void *stream,
                                const m3_cuda_rms_norm_e4m3_args *args,
                                m3_error *error)
{
    enum { INPUT, RESIDUAL, SUM, SCALE, CODES, CODE_SCALES, SPANS };
    span s[SPANS];
    m3c_norm_e4m3_params p;
    uint64_t group;
    uint64_t element;
    m3_status status;
    int previous;
    int out;
    int k;

    if (args == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "norm arguments are required");
    }
    status = check_float(args->dtype, "norm input", error);
    if (status == M3_STATUS_OK) {
        status = check_float(args->scale_dtype, "norm scale", error);
    }
    if (status != M3_STATUS_OK) {
        return status;
    }
    group = args->group == 0U ? args->width : args->group;
    if (args->width == 0U || args->width > (uint64_t)INT32_MAX ||
        args->width % group != 0U || !isfinite(args->epsilon) ||
        args->epsilon <= 0.0F) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "norm width, group or epsilon is invalid");
    }
    if (args->sum != NULL && args->residual == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "norm sum needs a residual");
    }
    element = m3c_dtype_size(args->dtype);
    memset(s, 0, sizeof(s));
    status = rows_span(&s[INPUT], "norm input", args->input, args->rows,
                       args->width, args->input_stride, element, error);
    if (status == M3_STATUS_OK && args->residual != NULL) {
        status = rows_span(&s[RESIDUAL], "norm residual", args->residual,
                           args->rows, args->width, args->residual_stride,
                           element, error);
    }
    if (status == M3_STATUS_OK && args->sum != NULL) {
        status = rows_span(&s[SUM], "norm sum", args->sum, args->rows,
                           args->width, args->sum_stride, element, error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[SCALE], "norm scale", args->scale,
                           args->rows == 0U ? 0U : 1U, args->width, 0U,
                           m3c_dtype_size(args->scale_dtype), error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[CODES], "norm codes", args->codes, args->rows,
                           args->width, 0U, 1U, error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[CODE_SCALES], "norm code scales",
                           args->code_scales, args->rows, args->width / group,
                           0U, sizeof(float), error);
    }
    for (out = SUM; status == M3_STATUS_OK && out < SPANS; ++out) {
        for (k = 0; status == M3_STATUS_OK && k < out; ++k) {
            if (out == SCALE) {
                /* an input: only the sum is written before it in the list */
                if (k == SUM) {
                    status = check_apart(&s[SUM], &s[SCALE], error);
                }
            } else if (out != SUM || s[k].begin != s[SUM].begin ||
                       (s[k].stride != s[SUM].stride && args->rows > 1U)) {
                status = check_apart(&s[out], &s[k], error);
            }
        }
    }
    if (status != M3_STATUS_OK) {
        return status;
    }
    memset(&p, 0, sizeof(p));
    p.x = args->input;
    p.resid_b = args->residual;
    p.sum_out = args->sum;
    p.x_stride = s[INPUT].stride;
    p.resid_stride = s[RESIDUAL].stride;
    p.sum_stride = s[SUM].stride;
    p.scale = args->scale;
    p.codes = args->codes;
    p.code_scales = args->code_scales;
    p.rows = args->rows;
    p.width = args->width;
    p.group = group;
    p.dtype = (int32_t)args->dtype;
    p.scale_dtype = (int32_t)args->scale_dtype;
    p.epsilon = args->epsilon;
    status = enter_device(device, &previous, error);
    if (status != M3_STATUS_OK) {
        return status;
    }
    status = launched(args->rows == 0U ? 0 : m3c_launch_norm_e4m3(&p, stream),
                      error);
    leave_device(device, previous);
    return status;
}

/* ---------------------------------------------------------------- cache */

#define CACHE_CLEAN (~0ULL)
#define CACHE_PART_LIMIT ((uint64_t)1 << 20)

void m3_cuda_cache_options_init(m3_cuda_cache_options *options)
{
    if (options != NULL) {
        memset(options, 0, sizeof(*options));
        options->device = M3_CUDA_DEVICE_CURRENT;
        options->page_tokens = 16U;
    }
}

static uint64_t align_up(uint64_t bytes)
{
    return (bytes + M3C_ARENA_ALIGNMENT - 1U) &
           ~(uint64_t)(M3C_ARENA_ALIGNMENT - 1U);
}

m3_status m3_cuda_cache_create(m3_cuda_cache **cache,
                               const m3_cuda_cache_options *options,
                               m3_error *error)
{
    static const unsigned long long clean = CACHE_CLEAN;
    m3_cuda_cache *c;
    uint64_t vectors;
    uint64_t code_bytes;
    uint64_t scale_bytes;
    cudaError_t code;
    int devices = 0;
    int previous = 0;
    m3_status status;

    if (cache == NULL || *cache != NULL || options == NULL) {
        return m3c_error_set(
            error, M3_STATUS_INVALID_ARGUMENT,
            "cache output must be empty and options are required");
    }
    if (options->pages == 0U || options->pages > (uint64_t)INT32_MAX ||
        options->page_tokens == 0U || options->heads == 0U ||
        options->head_dim == 0U || options->page_tokens > CACHE_PART_LIMIT ||
        options->heads > CACHE_PART_LIMIT ||
        options->head_dim > CACHE_PART_LIMIT ||
        (uint64_t)options->heads * options->head_dim > CACHE_PART_LIMIT) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "cache pages, page tokens, heads or head "
                             "dimension is out of range");
    }
    /* pages < 2^31, tokens * heads * dim <= 2^40: no product overflows until
     * the last, which is checked */
    vectors = (uint64_t)options->page_tokens * options->heads;
    if (options->pages >
        (uint64_t)INT64_MAX / 16U / (vectors * options->head_dim + 4U * vectors)) {
        return m3c_error_set(error, M3_STATUS_OVERFLOW,
                             "cache size overflows");
    }
    vectors *= options->pages;
    code_bytes = align_up(vectors * options->head_dim);
    scale_bytes = align_up(vectors * sizeof(float));
    if (cudaGetDeviceCount(&devices) != cudaSuccess || devices == 0) {
        (void)cudaGetLastError();
        return m3c_error_set(error, M3_STATUS_UNSUPPORTED,
                             "no CUDA device is available");
    }
    c = calloc(1U, sizeof(*c));
    if (c == NULL) {
        return m3c_error_set(error, M3_STATUS_OUT_OF_MEMORY,
                             "cannot allocate cache");
    }
    c->options = *options;
    code = cudaGetDevice(&previous);
    c->device = options->device == M3_CUDA_DEVICE_CURRENT ? previous
                                                          : options->device;
    status = code == cudaSuccess
                 ? enter_device(c->device, &previous, error)
                 : cuda_failure(error, code, "cannot read the current device");
    if (status != M3_STATUS_OK) {
        free(c);
        return status;
    }
    c->arena_bytes = 2U * (code_bytes + scale_bytes) + M3C_ARENA_ALIGNMENT;
    code = cudaMalloc((void **)&c->arena, c->arena_bytes);
    if (code == cudaSuccess) {
        c->codes[0] = c->arena;
        c->codes[1] = c->codes[0] + code_bytes;
        c->scales[0] = (float *)(c->codes[1] + code_bytes);
        c->scales[1] = (float *)((unsigned char *)c->scales[0] + scale_bytes);
        c->first_skipped =
            (unsigned long long *)((unsigned char *)c->scales[1] + scale_bytes);
        code = cudaMallocHost((void **)&c->seen, sizeof(*c->seen));
    }
    if (code == cudaSuccess) {
        code = cudaMemset(c->arena, 0, 2U * (code_bytes + scale_bytes));
    }
    if (code == cudaSuccess) {
        code = cudaMemcpy(c->first_skipped, &clean, sizeof(clean),
                          cudaMemcpyHostToDevice);
    }
    if (code == cudaSuccess) {
        /* the fill runs on the legacy default stream, which non-blocking
         * streams do not wait for */
        code = cudaStreamSynchronize(NULL);
    }
    if (code != cudaSuccess) {
        status = cuda_failure(error, code, "cannot allocate the cache");
    }
    leave_device(c->device, previous);
    if (status != M3_STATUS_OK) {
        m3_cuda_cache_free(c);
        return status;
    }
    *cache = c;
    m3_error_reset(error);
    return M3_STATUS_OK;
}

void m3_cuda_cache_free(m3_cuda_cache *cache)
{
    int previous = 0;

    if (cache == NULL) {
        return;
    }
    if (enter_device(cache->device, &previous, NULL) == M3_STATUS_OK) {
        if (cache->arena != NULL) {
            (void)cudaFree(cache->arena);     /* waits for the device */
        }
        if (cache->seen != NULL) {
            (void)cudaFreeHost(cache->seen);
        }
        (void)cudaGetLastError();
        leave_device(cache->device, previous);
    }
    free(cache);
}

m3_status m3_cuda_cache_device_pointers(const m3_cuda_cache *cache,
                                        void **key_codes, float **key_scales,
                                        void **value_codes,
                                        float **value_scales, m3_error *error)
{
    if (cache == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "cache is null");
    }
    if (key_codes != NULL) *key_codes = cache->codes[0];
    if (key_scales != NULL) *key_scales = cache->scales[0];
    if (value_codes != NULL) *value_codes = cache->codes[1];
    if (value_scales != NULL) *value_scales = cache->scales[1];
    m3_error_reset(error);
    return M3_STATUS_OK;
}

/* The span of a batch's keys or values, and their strides: `vectors` steps from
 * head to head, `tokens` from token to token.  Either may be the outer one. */
static m3_status cache_span(const m3_cuda_cache *cache,
                            const m3_cuda_cache_rows *r, const char *name,
                            uint64_t rows, span *tokens, span *vectors,
                            m3_error *error)
{
    uint64_t heads = rows == 0U ? 0U : cache->options.heads;
    uint64_t dim = cache->options.head_dim;
    uint64_t size;
    uint64_t other_heads;
    m3_status status = check_float(r->dtype, name, error);

    if (status != M3_STATUS_OK) {
        return status;
    }
    size = m3c_dtype_size(r->dtype);
    status = rows_span(vectors, name, r->data, heads, dim, r->head_stride,
                       size, error);
    if (status == M3_STATUS_OK) {
        status = rows_span(tokens, name, r->data, rows, dim,
                           r->token_stride == 0U
                               ? cache->options.heads * dim
                               : r->token_stride,
                           size, error);
    }
    if (status != M3_STATUS_OK || rows == 0U) {
        return status;
    }
    /* from the last token's first vector to its last */
    other_heads = vectors->end - vectors->begin - dim * size;
    if (other_heads > UINTPTR_MAX - tokens->end) {
        return m3c_error_set(error, M3_STATUS_OVERFLOW, "%s size overflows",
                             name);
    }
    tokens->end += other_heads;
    return M3_STATUS_OK;
}

/* The launch block of one write, or read (`into_rows`), checked. */
static m3_status cache_params(const m3_cuda_cache *cache,
                              const m3_cuda_cache_batch *batch,
                              const m3_cuda_cache_rows *const rows[2],
                              bool into_rows, m3c_cache_params *p,
                              m3_error *error)
{
    enum { KEYS, VALUES, PAGE_TABLE, OFFSETS, STARTS, SPANS };
    static const char *const names[SPANS] = {
        "cache keys", "cache values", "cache page table", "cache offsets",
        "cache starts"};
    span s[SPANS];
    span memory;
    m3_status status = M3_STATUS_OK;
    int k;
    int other;

    if (cache == NULL || batch == NULL || rows[0] == NULL || rows[1] == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "cache, batch, keys and values are required");
    }
    if (batch->rows > (uint64_t)INT32_MAX ||
        batch->sequences > (uint64_t)INT32_MAX ||
        batch->page_table_stride > (uint64_t)INT32_MAX) {
        return m3c_error_set(error, M3_STATUS_OUT_OF_RANGE,
                             "cache batch has too many rows, sequences or "
                             "pages");
    }
    memset(p, 0, sizeof(*p));
    memset(s, 0, sizeof(s));
    for (k = KEYS; k <= VALUES; ++k) {
        span vectors;

        status = cache_span(cache, rows[k], names[k], batch->rows, &s[k],
                            &vectors, error);
        if (status != M3_STATUS_OK) {
            return status;
        }
        p->codes[k] = cache->codes[k];
        p->scales[k] = cache->scales[k];
        p->rows[k] = rows[k]->data;
        p->dtype[k] = (int32_t)rows[k]->dtype;
        p->token_stride[k] = s[k].stride;
        p->head_stride[k] = vectors.stride;
    }
    if (batch->rows != 0U && batch->sequences != 0U) {
        const void *data[SPANS] = {NULL, NULL, batch->page_table,
                                   batch->offsets, batch->starts};
        const uint64_t count[SPANS] = {
            0U, 0U, batch->sequences * batch->page_table_stride,
            batch->sequences + 1U, batch->starts == NULL ? 0U : batch->sequences};

        memory.name = "the cache's memory";
        memory.begin = (uintptr_t)cache->arena;
        memory.end = memory.begin + cache->arena_bytes;
        for (k = PAGE_TABLE; k < SPANS; ++k) {
            if ((data[k] == NULL && count[k] != 0U) ||
                (uintptr_t)data[k] % sizeof(int32_t) != 0U) {
                return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                                     "%s is absent or not aligned", names[k]);
            }
            status = rows_span(&s[k], names[k], data[k], 1U, count[k], 0U,
                               sizeof(int32_t), error);
            if (status != M3_STATUS_OK) {
                return status;
            }
        }
        for (k = KEYS; status == M3_STATUS_OK && k < SPANS; ++k) {
            status = check_apart(&s[k], &memory, error);
            for (other = PAGE_TABLE; status == M3_STATUS_OK && into_rows &&
                                     k <= VALUES && other < SPANS; ++other) {
                status = check_apart(&s[k], &s[other], error);
            }
        }
        if (status != M3_STATUS_OK) {
            return status;
        }
    }
    p->page_table = batch->page_table;
    p->offsets = batch->offsets;
    p->starts = batch->starts;
    p->page_table_stride = batch->page_table_stride;
    p->pages = cache->options.pages;
    p->sequences = (uint32_t)batch->sequences;
    p->row_count = (uint32_t)batch->rows;
    p->page_tokens = cache->options.page_tokens;
    p->heads = cache->options.heads;
    p->head_dim = cache->options.head_dim;
    p->first_skipped = cache->first_skipped;
    return M3_STATUS_OK;
}

static m3_status cache_move(m3_cuda_cache *cache, void *stream,
                            const m3_cuda_cache_batch *batch,
                            const m3_cuda_cache_rows *keys,
                            const m3_cuda_cache_rows *values,
                            bool into_rows, m3_error *error)
{
    const m3_cuda_cache_rows *rows[2];
    m3c_cache_params p;
    m3_status status;
    int previous;

    rows[0] = keys;
    rows[1] = values;
    status = cache_params(cache, batch, rows, into_rows, &p, error);
    if (status != M3_STATUS_OK) {
        return status;
    }
    if (p.row_count == 0U || p.sequences == 0U) {
        m3_error_reset(error);
        return M3_STATUS_OK;
    }
    status = enter_device(cache->device, &previous, error);
    if (status != M3_STATUS_OK) {
        return status;
    }
    status = launched(into_rows ? m3c_launch_cache_read(&p, stream)
                                : m3c_launch_cache_write(&p, stream),
                      error);
    leave_device(cache->device, previous);
    return status;
}

m3_status m3_cuda_cache_write(m3_cuda_cache *cache, void *stream,
                              const m3_cuda_cache_batch *batch,
                              const m3_cuda_cache_rows *keys,
                              const m3_cuda_cache_rows *values,
                              m3_error *error)
{
    return cache_move(cache, stream, batch, keys, values, false, error);
}

m3_status m3_cuda_cache_read(m3_cuda_cache *cache, void *stream,
                             const m3_cuda_cache_batch *batch,
                             const m3_cuda_cache_rows *keys,
                             const m3_cuda_cache_rows *values,
                             m3_error *error)
{
    return cache_move(cache, stream, batch, keys, values, true, error);
}

m3_status m3_cuda_cache_synchronize(m3_cuda_cache *cache, void *stream,
                                    m3_error *error)
{
    cudaStream_t s = (cudaStream_t)stream;
    unsigned long long seen = CACHE_CLEAN;
    cudaError_t code;
    int previous;
    m3_status status;

    if (cache == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "cache is null");
    }
    status = enter_device(cache->device, &previous, error);
    if (status != M3_STATUS_OK) {
        return status;
    }
    code = (cudaError_t)m3c_launch_cache_report(cache->first_skipped,
                                                cache->first_skipped + 1, s);
    if (code == cudaSuccess) {
        code = cudaMemcpyAsync(cache->seen, cache->first_skipped + 1,
                               sizeof(seen), cudaMemcpyDeviceToHost, s);
    }
    if (code == cudaSuccess) {
        code = cudaStreamSynchronize(s);
    }
    if (code == cudaSuccess) {
        seen = *cache->seen;
    }
    if (code != cudaSuccess) {
        status = cuda_failure(error, code, "cache synchronise failed");
    } else if (seen != CACHE_CLEAN) {
        status = m3c_error_set(
            error, M3_STATUS_OUT_OF_RANGE, "cache row %llu was skipped: %s",
            seen / 4U,
            seen % 4U == M3C_CACHE_BAD_PAGE
                ? "its page is outside the cache"
                : "its position is outside the page table");
    } else {
        m3_error_reset(error);
    }
    leave_device(cache->device, previous);
    return status;
}

/* -------------------------------------------------- draft verification */

void m3_cuda_verify_draft_args_init(m3_cuda_verify_draft_args *args)
{
    if (args != NULL) {
        memset(args, 0, sizeof(*args));
    }
}

m3_status m3_cuda_verify_draft(int device, void *stream,
                               const m3_cuda_verify_draft_args *args,
                               m3_error *error)
{
    enum { TARGET, DRAFT, DRAFT_TOKENS, LENGTHS, UNIFORMS, TOKENS, ACCEPTED,
           SPANS };
    span s[SPANS];
    m3c_verify_params p;
    uint64_t element;
    uint64_t places;
    m3_status status;
    int previous;
    int out;
    int k;

    if (args == NULL) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "verification arguments are required");
    }
    status = check_float(args->dtype, "verified probabilities", error);
    if (status != M3_STATUS_OK) {
        return status;
    }
    if (args->vocabulary == 0U || args->vocabulary > (uint64_t)INT32_MAX ||
        args->batch > (uint64_t)INT32_MAX || args->drafts >= (uint64_t)INT32_MAX) {
        return m3c_error_set(error, M3_STATUS_INVALID_ARGUMENT,
                             "verification batch, drafts or vocabulary is "
                             "out of range");
    }
    element = m3c_dtype_size(args->dtype);
    places = args->drafts + 1U;
    memset(s, 0, sizeof(s));
    status = rows_span(&s[TARGET], "target probabilities", args->target,
                       args->batch * places, args->vocabulary,
                       args->target_stride, element, error);
    if (status == M3_STATUS_OK && args->draft != NULL) {
        status = rows_span(&s[DRAFT], "draft probabilities", args->draft,
                           args->batch * args->drafts, args->vocabulary,
                           args->draft_stride, element, error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[DRAFT_TOKENS], "drafted tokens",
                           args->draft_tokens, args->batch, args->drafts, 0U,
                           sizeof(int32_t), error);
    }
    if (status == M3_STATUS_OK && args->lengths != NULL) {
        status = rows_span(&s[LENGTHS], "draft lengths", args->lengths,
                           args->batch, 1U, 0U, sizeof(int32_t), error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[UNIFORMS], "verification uniforms",
                           args->uniforms, args->batch, places, 0U,
                           sizeof(float), error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[TOKENS], "verified tokens", args->tokens,
                           args->batch, places, 0U, sizeof(int32_t), error);
    }
    if (status == M3_STATUS_OK) {
        status = rows_span(&s[ACCEPTED], "accepted counts", args->accepted,
                           args->batch, 1U, 0U, sizeof(int32_t), error);
    }
    for (out = TOKENS; status == M3_STATUS_OK && out < SPANS; ++out) {
        for (k = 0; status == M3_STATUS_OK && k < out; ++k) {
            status = check_apart(&s[out], &s[k], error);
        }
    }
    if (status != M3_STATUS_OK) {
        return status;
    }
    memset(&p, 0, sizeof(p));
    p.target = args->target;
    p.draft = args->draft;
    p.target_stride = s[TARGET].stride;
    p.draft_stride = s[DRAFT].stride;
    p.draft_tokens = args->draft_tokens;
    p.lengths = args->lengths;
    p.uniforms = args->uniforms;
    p.tokens = args->tokens;
    p.accepted = args->accepted;
    p.batch = args->batch;
    p.drafts = args->drafts;
    p.vocabulary = (uint32_t)args->vocabulary;
    p.dtype = (int32_t)args->dtype;
    status = enter_device(device, &previous, error);
    if (status != M3_STATUS_OK) {
        return status;
    }
    status = launched(args->batch == 0U ? 0 : m3c_launch_verify(&p, stream),
                      error);
    leave_device(device, previous);
    return status;
}
