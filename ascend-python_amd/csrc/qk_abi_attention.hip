// extern "C" entry points of the attention and cache functions (declared in include/qk_abi.h): the checks of their plain
// arguments, and the kernels' launches on the caller's stream.  Nothing here allocates or synchronises.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "kernels/attention.h"

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return qk::abi_error(code, buf);
}

int launched(hipError_t e, const char* op) {
    if (e != hipSuccess) return fail(QK_ERR_LAUNCH, "%s: kernel launch failed: %s", op, hipGetErrorString(e));
    return QK_OK;
}

constexpr int64_t kInt31 = ((int64_t)1 << 31) - 1;
constexpr int64_t kMaxHeads = 65535;
// Tokens of a sequence: the kernels count up to some hundreds past the last in 32 bits.
constexpr int64_t kMaxTokens = kInt31 - 1024;

bool is_half(int dt) { return dt == QK_F16 || dt == QK_BF16; }

// A window, and its first tokens that stay visible, as the kernels and their plans take them: past 31 bits is without end.
int32_t cut31(int64_t v) { return (int32_t)(v > kInt31 ? kInt31 : v); }

int check_workspace(const char* op, size_t need, const void* workspace, size_t workspace_bytes) {
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(QK_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", op, need, workspace_bytes);
    if (need > 0 && (uintptr_t)workspace % 256 != 0)
        return fail(QK_ERR_WORKSPACE, "%s: the workspace must be 256-byte aligned", op);
    return QK_OK;
}

// A cache's sizes and types; `dtype`: of the tensors beside it.
int check_cache_sizes(const char* op, const qk_kv_cache* c, int dtype) {
    if (!is_half(dtype)) return fail(QK_ERR_ARG, "%s: tensors must be float16 or bfloat16 (got dtype %d)", op, dtype);
    if (!c) return fail(QK_ERR_ARG, "%s: null cache", op);
    if (c->dtype != QK_I8 && c->dtype != dtype)
        return fail(QK_ERR_ARG, "%s: the cache must be int8 or of the tensors' dtype %d (got %d)", op, dtype, c->dtype);
    const int piece = c->dtype == QK_I8 ? 16 : 8;
    if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % piece != 0)
        return fail(QK_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of %d up to 256 (got %lld)", op, piece,
                    (long long)c->head_dim);
    if (c->num_pages < 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->kv_heads > kMaxHeads)
        return fail(QK_ERR_ARG, "%s: need num_pages >= 0, page_size > 0 and kv_heads in 1..%lld (got %lld, %lld, %lld)", op,
                    (long long)kMaxHeads, (long long)c->num_pages, (long long)c->page_size, (long long)c->kv_heads);
    if (c->num_pages > kInt31 || c->page_size > kInt31 || c->num_pages > kInt31 / c->page_size)
        return fail(QK_ERR_UNSUPPORTED, "%s: a cache of %lld pages of %lld tokens has slots past 31 bits", op,
                    (long long)c->num_pages, (long long)c->page_size);
    return QK_OK;
}

// ... and its pointers and strides (a cache that is read or written)
int check_cache_data(const char* op, const qk_kv_cache* c) {
    if (!c->key || !c->value) return fail(QK_ERR_ARG, "%s: null pointer in the cache", op);
    const int size = c->dtype == QK_I8 ? 1 : 2;
    const int64_t bytes[] = {c->key_page_stride * size, c->key_token_stride * size, c->key_head_stride * size,
                             c->value_page_stride * size, c->value_token_stride * size, c->value_head_stride * size};
    for (int64_t b : bytes) {
        if (b < 0) return fail(QK_ERR_ARG, "%s: negative stride in the cache", op);
        if (b % 16 != 0) return fail(QK_ERR_ARG, "%s: the cache's strides must be multiples of 16 bytes (got %lld)", op, (long long)b);
    }
    if ((uintptr_t)c->key % 16 != 0 || (uintptr_t)c->value % 16 != 0)
        return fail(QK_ERR_ARG, "%s: the cache must be 16-byte aligned", op);
    if (c->dtype == QK_I8) {
        if (!c->key_scale || !c->value_scale) return fail(QK_ERR_ARG, "%s: an int8 cache needs key_scale and value_scale", op);
        const int64_t s[] = {c->key_scale_page_stride, c->key_scale_token_stride, c->key_scale_head_stride,
                             c->value_scale_page_stride, c->value_scale_token_stride, c->value_scale_head_stride};
        for (int64_t b : s)
            if (b < 0) return fail(QK_ERR_ARG, "%s: negative stride in the scales", op);
    }
    return QK_OK;
}

int check_heads(const char* op, int64_t q_heads, const qk_kv_cache* c) {
    if (q_heads <= 0 || q_heads > kMaxHeads || q_heads % c->kv_heads != 0)
        return fail(QK_ERR_ARG, "%s: q_heads must be a positive multiple of kv_heads (got %lld and %lld)", op,
                    (long long)q_heads, (long long)c->kv_heads);
    return QK_OK;
}

int check_attention_sizes(const char* op, int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache* c, int dtype,
                          int64_t table_width, int64_t window, int64_t sinks) {
    if (int rc = check_cache_sizes(op, c, dtype)) return rc;
    if (int rc = check_heads(op, q_heads, c)) return rc;
    if (tokens < 0 || batch < 0 || table_width < 0 || window < 0 || sinks < 0)
        return fail(QK_ERR_ARG, "%s: negative size tokens=%lld batch=%lld table_width=%lld window=%lld sinks=%lld", op,
                    (long long)tokens, (long long)batch, (long long)table_width, (long long)window, (long long)sinks);
    if (tokens > kInt31 || batch > kInt31 || tokens > kInt31 / q_heads || batch > kInt31 / q_heads)
        return fail(QK_ERR_UNSUPPORTED, "%s: %lld rows of %lld heads exceed the launch limit", op,
                    (long long)(tokens > batch ? tokens : batch), (long long)q_heads);
    if (c->page_size > kMaxTokens || table_width > kMaxTokens / c->page_size)
        return fail(QK_ERR_UNSUPPORTED, "%s: a table of %lld pages of %lld tokens exceeds 31 bits", op,
                    (long long)table_width, (long long)c->page_size);
    return QK_OK;
}

int check_query(const char* op, const void* query, int64_t token_stride, int64_t head_stride, const void* out) {
    if (!query || !out) return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (token_stride < 0 || head_stride < 0 || token_stride % 8 != 0 || head_stride % 8 != 0)
        return fail(QK_ERR_ARG, "%s: the query's strides must be multiples of 8 elements (got %lld and %lld)", op,
                    (long long)token_stride, (long long)head_stride);
    if ((uintptr_t)query % 16 != 0 || (uintptr_t)out % 16 != 0)
        return fail(QK_ERR_ARG, "%s: query and out must be 16-byte aligned", op);
    return QK_OK;
}

// The kernels hold the scale times log2 e.
int check_scale(const char* op, float scale) {
    if (!std::isfinite(scale * (float)M_LOG2E)) return fail(QK_ERR_ARG, "%s: scale must be finite, and at most 2.3e38 (got %g)", op, scale);
    return QK_OK;
}

qk::AttnArgs attention_args(const void* query, int dtype, int64_t tokens, int64_t batch, int64_t q_heads,
                            int64_t q_token_stride, int64_t q_head_stride, const qk_kv_cache* cache,
                            const int32_t* table, int64_t table_width, int64_t table_stride, const int32_t* lens,
                            float scale, int64_t window, int64_t sinks, void* out, float* lse) {
    qk::AttnArgs a = {};
    a.q = query;
    a.dtype = dtype;
    a.tokens = tokens;
    a.batch = batch;
    a.q_heads = q_heads;
    a.q_token_stride = q_token_stride;
    a.q_head_stride = q_head_stride;
    a.kv.c = *cache;
    a.kv.table = table;
    a.kv.table_width = table_width;
    a.kv.table_stride = table_stride;
    a.kv.lens = lens;
    a.kv.page_div = qk::div31((uint32_t)cache->page_size);
    a.scale = scale;
    a.window = cut31(window);
    a.sinks = window ? cut31(sinks) : 0;
    a.out = out;
    a.lse = lse;
    return a;
}

int check_pool(const char* op, int64_t num_pages, int64_t page_size, const void* table, int64_t max_seqs,
               int64_t table_width, int64_t table_stride, const void* lens, const void* count) {
    if (num_pages < 0 || page_size <= 0 || max_seqs < 0 || table_width < 0)
        return fail(QK_ERR_ARG, "%s: need sizes >= 0 and page_size > 0 (num_pages=%lld page_size=%lld max_seqs=%lld table_width=%lld)",
                    op, (long long)num_pages, (long long)page_size, (long long)max_seqs, (long long)table_width);
    if (num_pages > kInt31 / page_size || table_width > kInt31 / page_size || max_seqs > kInt31)
        return fail(QK_ERR_UNSUPPORTED, "%s: sizes past 31 bits", op);
    if (max_seqs > 1 && table_stride < table_width)
        return fail(QK_ERR_ARG, "%s: table rows overlap (stride %lld, width %lld)", op, (long long)table_stride,
                    (long long)table_width);
    if ((max_seqs > 0 && (!lens || (table_width > 0 && !table))) || (num_pages > 0 && !count))
        return fail(QK_ERR_ARG, "%s: null pointer", op);
    return QK_OK;
}

int check_page_list(const char* op, const qk_pages* pages, int64_t tensors) {
    if (tensors < 0 || tensors > (1 << 20)) return fail(QK_ERR_ARG, "%s: invalid number of tensors %lld", op, (long long)tensors);
    if (tensors > 0 && !pages) return fail(QK_ERR_ARG, "%s: null pointer", op);
    for (int64_t i = 0; i < tensors; ++i) {
        const qk_pages& p = pages[i];
        if (p.page_bytes < 0 || (p.page_bytes > 0 && (!p.base || p.page_stride < p.page_bytes)))
            return fail(QK_ERR_ARG, "%s: tensor %lld: pages of %lld bytes, %lld apart", op, (long long)i,
                        (long long)p.page_bytes, (long long)p.page_stride);
    }
    return QK_OK;
}

int check_seqs(const char* op, int64_t n) {
    if (n < 0 || n > QK_MAX_SEQS)
        return fail(n < 0 ? QK_ERR_ARG : QK_ERR_UNSUPPORTED, "%s: %lld sequences (at most %d a call)", op, (long long)n, QK_MAX_SEQS);
    return QK_OK;
}

}  // namespace

extern "C" {

int qk_paged_attention_workspace_size(int64_t batch, int64_t q_heads, const qk_kv_cache* cache, int64_t table_width,
                                      int64_t window, int64_t sinks, size_t* bytes) {
    qk::abi_begin();
    const char* op = "npu_paged_attention";
    if (!bytes) return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (int rc = check_attention_sizes(op, batch, batch, q_heads, cache, cache && cache->dtype != QK_I8 ? cache->dtype : QK_BF16,
                                       table_width, window, sinks))
        return rc;
    *bytes = qk::attention_decode_workspace(batch, q_heads, *cache, table_width, cut31(window), cut31(sinks));
    return QK_OK;
}

int qk_paged_attention(const void* query, int dtype, int64_t batch, int64_t q_heads, int64_t q_token_stride,
                       int64_t q_head_stride, const qk_kv_cache* cache, const int32_t* block_table,
                       int64_t table_width, int64_t table_stride, const int32_t* context_lens, float scale,
                       int64_t window, int64_t sinks, void* out, float* lse, void* workspace, size_t workspace_bytes,
                       qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_paged_attention";
    if (int rc = check_attention_sizes(op, batch, batch, q_heads, cache, dtype, table_width, window, sinks)) return rc;
    if (batch == 0) return QK_OK;
    if (int rc = check_query(op, query, q_token_stride, q_head_stride, out)) return rc;
    if (int rc = check_scale(op, scale)) return rc;
    if (cache->num_pages > 0)
        if (int rc = check_cache_data(op, cache)) return rc;
    if (!context_lens || (table_width > 0 && !block_table)) return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (table_stride < 0) return fail(QK_ERR_ARG, "%s: negative stride of the table", op);
    static const int32_t no_table = 0;  // a table without columns: marks the paged form, never read
    const qk::AttnArgs a = attention_args(query, dtype, batch, batch, q_heads, q_token_stride, q_head_stride, cache,
                                          block_table ? block_table : &no_table, table_width, table_stride, context_lens,
                                          scale, window, sinks, out, lse);
    size_t need = 0;
    if (int rc = qk_paged_attention_workspace_size(batch, q_heads, cache, table_width, window, sinks, &need)) return rc;
    if (int rc = check_workspace(op, need, workspace, workspace_bytes)) return rc;
    return launched(qk::launch_attention_decode(a, workspace, (hipStream_t)stream), op);
}

int qk_prompt_attention_workspace_size(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache* cache,
                                       int64_t table_width, int64_t window, int64_t sinks, size_t* bytes) {
    qk::abi_begin();
    const char* op = "npu_prompt_attention";
    if (!bytes) return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (int rc = check_attention_sizes(op, tokens, batch, q_heads, cache, cache && cache->dtype != QK_I8 ? cache->dtype : QK_BF16,
                                       table_width, window, sinks))
        return rc;
    *bytes = qk::attention_prompt_workspace(tokens, batch, q_heads, *cache, table_width, cut31(window), cut31(sinks));
    return QK_OK;
}

int qk_prompt_attention(const void* query, int dtype, int64_t tokens, int64_t batch, int64_t q_heads,
                        int64_t q_token_stride, int64_t q_head_stride, const int32_t* cu_seqlens_q,
                        const qk_kv_cache* cache, const int32_t* cu_seqlens_k, const int32_t* block_table,
                        int64_t table_width, int64_t table_stride, const int32_t* kv_lens, float scale, int64_t window,
                        int64_t sinks, void* out, float* lse, void* workspace, size_t workspace_bytes,
                        qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_prompt_attention";
    if (int rc = check_attention_sizes(op, tokens, batch, q_heads, cache, dtype, table_width, window, sinks)) return rc;
    if (tokens == 0) return QK_OK;
    if (int rc = check_query(op, query, q_token_stride, q_head_stride, out)) return rc;
    if (int rc = check_scale(op, scale)) return rc;
    if (!cu_seqlens_q) return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (batch == 0) return fail(QK_ERR_ARG, "%s: rows without a sequence", op);
    static const int32_t no_table = 0;
    const int32_t* table = block_table;
    if (kv_lens) {
        if (cu_seqlens_k) return fail(QK_ERR_ARG, "%s: keys are either paged (kv_lens) or contiguous (cu_seqlens_k)", op);
        if (table_width > 0 && !block_table) return fail(QK_ERR_ARG, "%s: null pointer", op);
        if (table_stride < 0) return fail(QK_ERR_ARG, "%s: negative stride of the table", op);
        if (!table) table = &no_table;
    } else {
        if (block_table || !cu_seqlens_k) return fail(QK_ERR_ARG, "%s: contiguous keys need cu_seqlens_k and no table", op);
        if (cache->num_pages > 1) return fail(QK_ERR_ARG, "%s: contiguous keys are one page", op);
    }
    if (cache->num_pages > 0)
        if (int rc = check_cache_data(op, cache)) return rc;
    qk::AttnArgs a = attention_args(query, dtype, tokens, batch, q_heads, q_token_stride, q_head_stride, cache, table,
                                    table_width, table_stride, kv_lens, scale, window, sinks, out, lse);
    a.cu_q = cu_seqlens_q;
    a.kv.cu_k = cu_seqlens_k;
    size_t need = 0;
    if (int rc = qk_prompt_attention_workspace_size(tokens, batch, q_heads, cache, table_width, window, sinks, &need)) return rc;
    if (int rc = check_workspace(op, need, workspace, workspace_bytes)) return rc;
    return launched(qk::launch_attention_prompt(a, workspace, (hipStream_t)stream), op);
}

int qk_mrope(const void* query, const void* key, const void* value, int dtype, int64_t tokens, int64_t q_heads,
             int64_t kv_heads, int64_t head_dim, int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
             int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const int32_t* positions,
             int64_t axes, int64_t position_stride, const int64_t* sections, const void* cos_sin, int cos_sin_dtype,
             int64_t table_rows, int64_t rotary_dim, int interleave, void* out_query, void* out_key,
             const qk_kv_cache* cache, const int32_t* slots, qk_stream_t stream) {
    qk::abi_begin();
    const char* op = cache ? "npu_mrope_scatter_kv" : "npu_mrope";
    if (!is_half(dtype)) return fail(QK_ERR_ARG, "%s: tensors must be float16 or bfloat16 (got dtype %d)", op, dtype);
    if (cos_sin_dtype != QK_F32 && cos_sin_dtype != dtype)
        return fail(QK_ERR_ARG, "%s: cos_sin must be float32 or of the tensors' dtype (got dtype %d)", op, cos_sin_dtype);
    if (tokens < 0 || q_heads < 0 || kv_heads < 0 || table_rows < 0 || q_heads > kMaxHeads || kv_heads > kMaxHeads)
        return fail(QK_ERR_ARG, "%s: invalid size tokens=%lld q_heads=%lld kv_heads=%lld table_rows=%lld", op,
                    (long long)tokens, (long long)q_heads, (long long)kv_heads, (long long)table_rows);
    if (tokens > kInt31 || table_rows > kInt31) return fail(QK_ERR_UNSUPPORTED, "%s: sizes past 31 bits", op);
    if (head_dim <= 0 || head_dim > 256) return fail(QK_ERR_UNSUPPORTED, "%s: head_dim must be 1..256 (got %lld)", op, (long long)head_dim);
    if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
        return fail(QK_ERR_ARG, "%s: rotary_dim must be even, 2..head_dim=%lld (got %lld)", op, (long long)head_dim, (long long)rotary_dim);
    if (axes < 1 || axes > 4) return fail(QK_ERR_ARG, "%s: positions of 1 to 4 axes (got %lld)", op, (long long)axes);
    if (axes > 1 && !sections) return fail(QK_ERR_ARG, "%s: %lld axes need sections", op, (long long)axes);
    qk::MropeArgs a = {};
    int64_t end = 0;
    for (int64_t k = 0; k < axes; ++k) {
        const int64_t n = sections ? sections[k] : rotary_dim / 2;
        if (n < 0 || n > rotary_dim / 2) return fail(QK_ERR_ARG, "%s: invalid section %lld", op, (long long)n);
        a.section_end[k] = (int32_t)(end += n);
    }
    if (end != rotary_dim / 2)
        return fail(QK_ERR_ARG, "%s: sections must sum to rotary_dim / 2 = %lld (got %lld)", op, (long long)rotary_dim / 2, (long long)end);
    if (cache) {
        if (int rc = check_cache_sizes(op, cache, dtype)) return rc;
        if (cache->head_dim != head_dim || cache->kv_heads != kv_heads)
            return fail(QK_ERR_ARG, "%s: the cache has %lld heads of %lld, the keys %lld of %lld", op, (long long)cache->kv_heads,
                        (long long)cache->head_dim, (long long)kv_heads, (long long)head_dim);
    }
    if (tokens == 0 || q_heads + kv_heads == 0) return QK_OK;
    const int64_t strides[] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride};
    for (int64_t s : strides)
        if (s < 0) return fail(QK_ERR_ARG, "%s: negative stride", op);
    if ((q_heads > 0 && !query) || (kv_heads > 0 && !key) || !positions || !cos_sin)
        return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (cache && cache->num_pages > 0) {
        if (!slots) return fail(QK_ERR_ARG, "%s: null pointer", op);
        if (int rc = check_cache_data(op, cache)) return rc;
    }
    a.q = query;
    a.k = key;
    a.v = cache ? value : nullptr;
    a.dtype = dtype;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.q_token_stride = q_token_stride;
    a.q_head_stride = q_head_stride;
    a.k_token_stride = k_token_stride;
    a.k_head_stride = k_head_stride;
    a.v_token_stride = v_token_stride;
    a.v_head_stride = v_head_stride;
    a.positions = positions;
    a.axes = (int)axes;
    a.position_stride = position_stride;
    a.cos_sin = cos_sin;
    a.cos_sin_dtype = cos_sin_dtype;
    a.table_rows = table_rows;
    a.rotary_dim = rotary_dim;
    a.interleave = interleave != 0;
    a.out_q = out_query;
    a.out_k = out_key;
    if (cache && cache->num_pages > 0) {
        a.cached = true;
        a.c = *cache;
        a.slots = slots;
        a.page_div = qk::div31((uint32_t)cache->page_size);
    }
    return launched(qk::launch_mrope(a, (hipStream_t)stream), op);
}

int qk_kv_copy_pages(const qk_pages* pages, int64_t tensors, int64_t num_pages, const int32_t* src, const int32_t* dst,
                     int64_t n, qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_kv_copy_pages";
    if (int rc = check_page_list(op, pages, tensors)) return rc;
    if (num_pages < 0 || n < 0 || n > kInt31) return fail(QK_ERR_ARG, "%s: invalid size num_pages=%lld n=%lld", op, (long long)num_pages, (long long)n);
    if (n == 0 || tensors == 0) return QK_OK;
    if (!src || !dst) return fail(QK_ERR_ARG, "%s: null pointer", op);
    return launched(qk::launch_kv_copy_pages(pages, tensors, num_pages, src, dst, n, (hipStream_t)stream), op);
}

int qk_kv_fork_workspace_size(int64_t n, size_t* bytes) {
    qk::abi_begin();
    if (!bytes) return fail(QK_ERR_ARG, "npu_kv_fork: null pointer");
    if (int rc = check_seqs("npu_kv_fork", n)) return rc;
    *bytes = qk::kv_fork_workspace(n);
    return QK_OK;
}

int qk_kv_fork(const qk_pages* pages, int64_t tensors, int64_t num_pages, int64_t page_size, int32_t* block_table,
               int64_t max_seqs, int64_t table_width, int64_t table_stride, int32_t* context_lens, int32_t* ref_count,
               const int32_t* parents, const int32_t* children, int64_t n, int32_t* missing, void* workspace,
               size_t workspace_bytes, qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_kv_fork";
    if (int rc = check_pool(op, num_pages, page_size, block_table, max_seqs, table_width, table_stride, context_lens, ref_count)) return rc;
    if (int rc = check_page_list(op, pages, tensors)) return rc;
    if (int rc = check_seqs(op, n)) return rc;
    if (!missing || (n > 0 && (!parents || !children))) return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (int rc = check_workspace(op, qk::kv_fork_workspace(n), workspace, workspace_bytes)) return rc;
    const qk::PoolArgs p = {num_pages, page_size, block_table, max_seqs, table_width, table_stride, context_lens, ref_count};
    return launched(qk::launch_kv_fork(pages, tensors, p, parents, children, n, missing, workspace, (hipStream_t)stream), op);
}

int qk_kv_free(int64_t num_pages, int64_t page_size, int32_t* block_table, int64_t max_seqs, int64_t table_width,
               int64_t table_stride, int32_t* context_lens, int32_t* ref_count, const int32_t* seqs, int64_t n,
               qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_kv_free";
    if (int rc = check_pool(op, num_pages, page_size, block_table, max_seqs, table_width, table_stride, context_lens, ref_count)) return rc;
    if (int rc = check_seqs(op, n)) return rc;
    if (n == 0) return QK_OK;
    if (!seqs) return fail(QK_ERR_ARG, "%s: null pointer", op);
    const qk::PoolArgs p = {num_pages, page_size, block_table, max_seqs, table_width, table_stride, context_lens, ref_count};
    return launched(qk::launch_kv_free(p, seqs, n, (hipStream_t)stream), op);
}

int qk_kv_extend_workspace_size(int64_t n, int64_t num_pages, size_t* bytes) {
    qk::abi_begin();
    if (!bytes) return fail(QK_ERR_ARG, "npu_kv_extend: null pointer");
    if (int rc = check_seqs("npu_kv_extend", n)) return rc;
    if (num_pages < 0) return fail(QK_ERR_ARG, "npu_kv_extend: negative size num_pages=%lld", (long long)num_pages);
    *bytes = qk::kv_extend_workspace(n, num_pages);
    return QK_OK;
}

int qk_kv_extend(int64_t num_pages, int64_t page_size, int32_t* block_table, int64_t max_seqs, int64_t table_width,
                 int64_t table_stride, int32_t* context_lens, int32_t* ref_count, const int32_t* seqs,
                 const int32_t* cu_tokens, int64_t n, int64_t total, int32_t* slots, int32_t* positions,
                 int32_t* missing, void* workspace, size_t workspace_bytes, qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_kv_extend";
    if (int rc = check_pool(op, num_pages, page_size, block_table, max_seqs, table_width, table_stride, context_lens, ref_count)) return rc;
    if (int rc = check_seqs(op, n)) return rc;
    if (total < 0 || total > kInt31) return fail(QK_ERR_ARG, "%s: invalid number of tokens %lld", op, (long long)total);
    if (!missing || (n > 0 && (!seqs || !cu_tokens)) || (total > 0 && (!slots || !positions)))
        return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (int rc = check_workspace(op, qk::kv_extend_workspace(n, num_pages), workspace, workspace_bytes)) return rc;
    const qk::PoolArgs p = {num_pages, page_size, block_table, max_seqs, table_width, table_stride, context_lens, ref_count};
    return launched(qk::launch_kv_extend(p, seqs, cu_tokens, n, total, slots, positions, missing, workspace, (hipStream_t)stream), op);
}

int qk_kv_compact_workspace_size(int64_t num_pages, size_t* bytes) {
    qk::abi_begin();
    if (!bytes) return fail(QK_ERR_ARG, "npu_kv_compact: null pointer");
    if (num_pages < 0 || num_pages > kInt31) return fail(QK_ERR_ARG, "npu_kv_compact: invalid size num_pages=%lld", (long long)num_pages);
    *bytes = qk::kv_compact_workspace(num_pages);
    return QK_OK;
}

int qk_kv_compact(const qk_pages* pages, int64_t tensors, int64_t num_pages, const int32_t* block_table,
                  int64_t max_seqs, int64_t table_width, int64_t table_stride, const int32_t* ref_count,
                  int32_t* new_table, int32_t* new_count, int32_t* moved, void* workspace, size_t workspace_bytes,
                  qk_stream_t stream) {
    qk::abi_begin();
    const char* op = "npu_kv_compact";
    if (int rc = check_pool(op, num_pages, 1, block_table, max_seqs, table_width, table_stride, ref_count ? (const void*)ref_count : moved, ref_count)) return rc;
    if (int rc = check_page_list(op, pages, tensors)) return rc;
    if (!moved || (num_pages > 0 && !new_count) || (max_seqs > 0 && table_width > 0 && !new_table))
        return fail(QK_ERR_ARG, "%s: null pointer", op);
    if (int rc = check_workspace(op, qk::kv_compact_workspace(num_pages), workspace, workspace_bytes)) return rc;
    const qk::PoolArgs p = {num_pages, 1, const_cast<int32_t*>(block_table), max_seqs, table_width, table_stride, nullptr,
                            const_cast<int32_t*>(ref_count)};
    return launched(qk::launch_kv_compact(pages, tensors, p, new_table, new_count, moved, workspace, (hipStream_t)stream), op);
}

}  // extern "C"
