// torch.ops.npu.* registration of attention over a paged key-value cache: the two attention ops, rotary positions with the
// cache write, and the pages' own ops.
//
// As npu_quant_ops.cpp: each host function checks shapes, types and devices with TORCH_CHECK, allocates the outputs and
// the workspace (uninitialised, from the caching allocator) and launches through the C ABI on the current stream; a
// non-zero return becomes a TORCH_CHECK failure with qk_last_error().  Registered for the CUDA key (HIP tensors) and for
// Meta, which runs the same checks without launching.  Index tensors are int32.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cmath>
#include <limits>
#include <optional>
#include <tuple>
#include <vector>

#include "../../../include/qk_abi.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

int qk_dtype_of(at::ScalarType t) {
    switch (t) {
    case at::kHalf: return QK_F16;
    case at::kBFloat16: return QK_BF16;
    case at::kFloat: return QK_F32;
    case at::kChar: return QK_I8;
    default: return 0;
    }
}

qk_stream_t current_stream(const at::Tensor& t) {
    return reinterpret_cast<qk_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

void check_rc(int rc, const char* op) {
    TORCH_CHECK(rc == QK_OK, "call ", op, " failed, detail:", qk_last_error());
}

at::Tensor workspace_for(const at::Tensor& like, size_t bytes) {
    return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

bool is_half(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

void check_device(const char* op, const char* name, const at::Tensor& t, const at::Tensor& like) {
    TORCH_CHECK(t.device() == like.device(), op, ": ", name, " must be on ", like.device(), ", got ", t.device());
}

// An int32 index tensor of `dims` dimensions on the device of `like`.
void check_index(const char* op, const char* name, const at::Tensor& t, int64_t dims, const at::Tensor& like) {
    TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
    TORCH_CHECK(t.dim() == dims, op, ": ", name, " must have ", dims, " dimension(s), got ", t.sizes());
    check_device(op, name, t, like);
}

const int32_t* index_data(const at::Tensor& t) { return t.numel() ? t.const_data_ptr<int32_t>() : nullptr; }

// The stride of a dimension that has one.
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

bool last_is_dense(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

// t, or a copy of it where its rows are not dense, 16-byte aligned pieces.
at::Tensor whole_rows(const at::Tensor& t) {
    if (!last_is_dense(t)) return t.contiguous();
    bool ok = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && stride_of(t, d) * t.element_size() % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// The cache's shape and types.  key, value: [pages, page_size, heads, D], or [tokens, heads, D] as one page.
qk_kv_cache cache_shape(const char* op, const at::Tensor& key, const at::Tensor& value, const OptTensor& key_scale,
                        const OptTensor& value_scale, const at::Tensor& like, bool paged) {
    const int64_t dims = paged ? 4 : 3;
    const char* shape = paged ? "[pages, page_size, heads, head_dim]" : "[tokens, heads, head_dim]";
    TORCH_CHECK(key.dim() == dims && value.dim() == dims, op, ": keys and values must be ", shape, ", got ", key.sizes(),
                " and ", value.sizes());
    TORCH_CHECK(key.sizes() == value.sizes(), op, ": keys and values must have one shape, got ", key.sizes(), " and ",
                value.sizes());
    TORCH_CHECK(key.scalar_type() == value.scalar_type(), op, ": keys and values must have one dtype, got ",
                key.scalar_type(), " and ", value.scalar_type());
    TORCH_CHECK(key.scalar_type() == like.scalar_type() || key.scalar_type() == at::kChar, op,
                ": keys and values must be int8 or ", like.scalar_type(), ", got ", key.scalar_type());
    check_device(op, "keys", key, like);
    check_device(op, "values", value, like);
    TORCH_CHECK(last_is_dense(key) && last_is_dense(value), op, ": the last dimension of keys and values must be dense");
    const bool quant = key.scalar_type() == at::kChar;
    TORCH_CHECK(quant == key_scale.has_value() && quant == value_scale.has_value(), op,
                ": key_scale and value_scale go with int8 keys and values");
    qk_kv_cache c = {};
    c.dtype = qk_dtype_of(key.scalar_type());
    const int64_t o = paged ? 1 : 0;
    c.num_pages = paged ? key.size(0) : 1;
    c.page_size = key.size(o);
    c.kv_heads = key.size(o + 1);
    c.head_dim = key.size(o + 2);
    c.key_page_stride = paged ? stride_of(key, 0) : 0;
    c.key_token_stride = stride_of(key, o);
    c.key_head_stride = stride_of(key, o + 1);
    c.value_page_stride = paged ? stride_of(value, 0) : 0;
    c.value_token_stride = stride_of(value, o);
    c.value_head_stride = stride_of(value, o + 1);
    if (quant) {
        for (const at::Tensor* s : {&*key_scale, &*value_scale}) {
            TORCH_CHECK(s->scalar_type() == at::kFloat && s->sizes() == key.sizes().slice(0, dims - 1), op,
                        ": key_scale and value_scale must be float32 ", key.sizes().slice(0, dims - 1), ", got ",
                        s->scalar_type(), " ", s->sizes());
            check_device(op, "the scales", *s, like);
        }
        c.key_scale_page_stride = paged ? stride_of(*key_scale, 0) : 0;
        c.key_scale_token_stride = stride_of(*key_scale, o);
        c.key_scale_head_stride = stride_of(*key_scale, o + 1);
        c.value_scale_page_stride = paged ? stride_of(*value_scale, 0) : 0;
        c.value_scale_token_stride = stride_of(*value_scale, o);
        c.value_scale_head_stride = stride_of(*value_scale, o + 1);
    }
    TORCH_CHECK(c.page_size > 0 || !paged, op, ": pages must hold at least one token, got ", key.sizes());
    if (c.page_size == 0) {  // contiguous keys without a token
        c.num_pages = 0;
        c.page_size = 1;
    }
    return c;
}

void cache_data(qk_kv_cache& c, const at::Tensor& key, const at::Tensor& value, const OptTensor& key_scale,
                const OptTensor& value_scale) {
    c.key = const_cast<void*>(key.const_data_ptr());
    c.value = const_cast<void*>(value.const_data_ptr());
    c.key_scale = key_scale.has_value() ? const_cast<float*>(key_scale->const_data_ptr<float>()) : nullptr;
    c.value_scale = value_scale.has_value() ? const_cast<float*>(value_scale->const_data_ptr<float>()) : nullptr;
}

// What the C ABI refuses of a cache, for Meta calls, which do not reach it.  paged: read or written where it lies (contiguous
// keys are copied where their rows are not whole pieces).
void check_cache_limits(const char* op, const qk_kv_cache& c, const at::Tensor& key, const at::Tensor& value, bool paged) {
    const int64_t piece = c.dtype == QK_I8 ? 16 : 8, int31 = std::numeric_limits<int32_t>::max();
    TORCH_CHECK(c.head_dim > 0 && c.head_dim <= 256 && c.head_dim % piece == 0, op, ": head_dim must be a multiple of ", piece,
                " up to 256 (got ", c.head_dim, ")");
    TORCH_CHECK(c.kv_heads > 0 && c.kv_heads <= 65535, op, ": need kv_heads in 1..65535 (got ", c.kv_heads, ")");
    TORCH_CHECK(c.page_size <= int31 && c.num_pages <= int31 / c.page_size, op, ": a cache of ", c.num_pages, " pages of ",
                c.page_size, " tokens has slots past 31 bits");
    if (!paged || c.num_pages == 0) return;
    for (const at::Tensor* t : {&key, &value}) {
        for (int64_t d = 0; d + 1 < t->dim(); ++d)
            TORCH_CHECK(stride_of(*t, d) * t->element_size() % 16 == 0, op,
                        ": the cache's strides must be multiples of 16 bytes (got ", stride_of(*t, d) * t->element_size(), ")");
        TORCH_CHECK(t->storage_offset() * t->element_size() % 16 == 0, op, ": the cache must be 16-byte aligned");
    }
}

void check_query(const char* op, const at::Tensor& q, const qk_kv_cache* c) {
    TORCH_CHECK(is_half(q), op, ": query must be float16 or bfloat16, got ", q.scalar_type());
    TORCH_CHECK(q.dim() == 3, op, ": query must be [tokens, heads, head_dim], got ", q.sizes());
    if (!c) return;
    TORCH_CHECK(q.size(2) == c->head_dim, op, ": query and keys must have one head_dim, got ", q.size(2), " and ", c->head_dim);
    TORCH_CHECK(c->kv_heads > 0 && q.size(1) > 0 && q.size(1) % c->kv_heads == 0, op,
                ": the query's heads must be a multiple of the keys', got ", q.size(1), " and ", c->kv_heads);
}

double scale_or_default(const char* op, std::optional<double> scale, int64_t head_dim) {
    const double s = scale.value_or(1.0 / std::sqrt((double)head_dim));
    // the kernels hold it, times log2 e, in 32 bits
    TORCH_CHECK(std::isfinite((float)s * (float)M_LOG2E), op, ": scale must be finite, and at most 2.3e38, got ", s);
    return s;
}

void check_window(const char* op, int64_t window, int64_t sinks) {
    TORCH_CHECK(window >= 0 && sinks >= 0, op, ": window and sinks must not be negative, got ", window, " and ", sinks);
}

std::tuple<at::Tensor, at::Tensor> attention_outputs(const at::Tensor& q) {
    return {at::empty(q.sizes(), q.options()), at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat))};
}

// ---------------------------------------------------------------- npu_paged_attention

qk_kv_cache paged_attention_check(const char* op, const at::Tensor& q, const at::Tensor& key, const at::Tensor& value,
                                  const at::Tensor& table, const at::Tensor& lens, const OptTensor& key_scale,
                                  const OptTensor& value_scale, int64_t window, int64_t sinks) {
    check_query(op, q, nullptr);
    qk_kv_cache c = cache_shape(op, key, value, key_scale, value_scale, q, true);
    check_query(op, q, &c);
    check_index(op, "block_table", table, 2, q);
    check_index(op, "context_lens", lens, 1, q);
    TORCH_CHECK(table.size(0) == q.size(0) && lens.size(0) == q.size(0), op,
                ": block_table and context_lens must have one row per query, got ", table.sizes(), ", ", lens.sizes(),
                " and ", q.sizes());
    check_window(op, window, sinks);
    return c;
}

at::Tensor dense_table(const at::Tensor& table) { return last_is_dense(table) ? table : table.contiguous(); }

std::tuple<at::Tensor, at::Tensor> npu_paged_attention(const at::Tensor& query, const at::Tensor& key_cache,
                                                       const at::Tensor& value_cache, const at::Tensor& block_table,
                                                       const at::Tensor& context_lens, const OptTensor& key_scale,
                                                       const OptTensor& value_scale, std::optional<double> scale,
                                                       int64_t window, int64_t sinks) {
    const char* op = "npu_paged_attention";
    qk_kv_cache c = paged_attention_check(op, query, key_cache, value_cache, block_table, context_lens, key_scale,
                                          value_scale, window, sinks);
    const double s = scale_or_default(op, scale, c.head_dim);
    const c10::DeviceGuard guard(query.device());
    const auto q = whole_rows(query);
    const auto table = dense_table(block_table), lens = context_lens.contiguous();
    cache_data(c, key_cache, value_cache, key_scale, value_scale);
    auto [out, lse] = attention_outputs(q);
    const int64_t width = table.size(1);
    size_t ws_bytes = 0;
    check_rc(qk_paged_attention_workspace_size(q.size(0), q.size(1), &c, width, window, sinks, &ws_bytes), op);
    const auto ws = workspace_for(q, ws_bytes);
    check_rc(qk_paged_attention(q.const_data_ptr(), qk_dtype_of(q.scalar_type()), q.size(0), q.size(1), stride_of(q, 0),
                                stride_of(q, 1), &c, index_data(table), width, stride_of(table, 0), index_data(lens),
                                (float)s, window, sinks, out.data_ptr(), lse.data_ptr<float>(), ws.data_ptr(), ws_bytes,
                                current_stream(q)),
             op);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> npu_paged_attention_meta(const at::Tensor& query, const at::Tensor& key_cache,
                                                            const at::Tensor& value_cache, const at::Tensor& block_table,
                                                            const at::Tensor& context_lens, const OptTensor& key_scale,
                                                            const OptTensor& value_scale, std::optional<double> scale,
                                                            int64_t window, int64_t sinks) {
    const char* op = "npu_paged_attention";
    const qk_kv_cache c = paged_attention_check(op, query, key_cache, value_cache, block_table, context_lens, key_scale,
                                                value_scale, window, sinks);
    scale_or_default(op, scale, c.head_dim);
    check_cache_limits(op, c, key_cache, value_cache, true);
    size_t ws_bytes = 0;  // the query looks at the sizes as the launch does
    check_rc(qk_paged_attention_workspace_size(query.size(0), query.size(1), &c, block_table.size(1), window, sinks, &ws_bytes), op);
    return attention_outputs(query);
}

// ---------------------------------------------------------------- npu_prompt_attention

qk_kv_cache prompt_attention_check(const char* op, const at::Tensor& q, const at::Tensor& key, const at::Tensor& value,
                                   const at::Tensor& cu_q, const OptTensor& cu_k, const OptTensor& table,
                                   const OptTensor& lens, const OptTensor& key_scale, const OptTensor& value_scale,
                                   int64_t window, int64_t sinks) {
    check_query(op, q, nullptr);
    TORCH_CHECK(table.has_value() == lens.has_value(), op, ": block_table and context_lens go together");
    TORCH_CHECK(!(table.has_value() && cu_k.has_value()), op, ": keys are either paged (block_table) or contiguous (cu_seqlens_k)");
    qk_kv_cache c = cache_shape(op, key, value, key_scale, value_scale, q, table.has_value());
    check_query(op, q, &c);
    check_index(op, "cu_seqlens_q", cu_q, 1, q);
    TORCH_CHECK(cu_q.size(0) >= 1, op, ": cu_seqlens_q must have batch + 1 values");
    TORCH_CHECK(cu_q.size(0) > 1 || q.size(0) == 0, op, ": rows without a sequence");
    if (cu_k.has_value()) {
        check_index(op, "cu_seqlens_k", *cu_k, 1, q);
        TORCH_CHECK(cu_k->sizes() == cu_q.sizes(), op, ": cu_seqlens_k must be ", cu_q.sizes(), ", got ", cu_k->sizes());
    } else if (table.has_value()) {
        check_index(op, "block_table", *table, 2, q);
        check_index(op, "context_lens", *lens, 1, q);
        TORCH_CHECK(table->size(0) == cu_q.size(0) - 1 && lens->size(0) == cu_q.size(0) - 1, op,
                    ": block_table and context_lens must have one row per sequence, got ", table->sizes(), ", ",
                    lens->sizes(), " and ", cu_q.size(0) - 1);
    }
    check_window(op, window, sinks);
    return c;
}

std::tuple<at::Tensor, at::Tensor> npu_prompt_attention(const at::Tensor& query, const at::Tensor& key_in,
                                                        const at::Tensor& value_in, const at::Tensor& cu_seqlens_q,
                                                        const OptTensor& cu_seqlens_k, const OptTensor& block_table,
                                                        const OptTensor& context_lens, const OptTensor& key_scale,
                                                        const OptTensor& value_scale, std::optional<double> scale,
                                                        int64_t window, int64_t sinks) {
    const char* op = "npu_prompt_attention";
    const bool paged = block_table.has_value();
    const c10::DeviceGuard guard(query.device());
    // contiguous keys and values are inputs like the query, and copied where their rows are not whole pieces; a cache is not
    const auto fit = [&](const at::Tensor& t) { return paged || t.dim() != 3 ? t : whole_rows(t); };
    const auto key = fit(key_in), value = fit(value_in);
    qk_kv_cache c = prompt_attention_check(op, query, key, value, cu_seqlens_q, cu_seqlens_k, block_table, context_lens,
                                           key_scale, value_scale, window, sinks);
    const double s = scale_or_default(op, scale, c.head_dim);
    const auto q = whole_rows(query);
    const auto cu_q = cu_seqlens_q.contiguous();
    at::Tensor cu_k, table, lens;
    if (paged) {
        table = dense_table(*block_table);
        lens = context_lens->contiguous();
    } else {
        cu_k = cu_seqlens_k.has_value() ? cu_seqlens_k->contiguous() : cu_q;
    }
    cache_data(c, key, value, key_scale, value_scale);
    auto [out, lse] = attention_outputs(q);
    if (q.size(0) == 0) return {out, lse};
    const int64_t width = paged ? table.size(1) : 0, batch = cu_q.size(0) - 1;
    size_t ws_bytes = 0;
    check_rc(qk_prompt_attention_workspace_size(q.size(0), batch, q.size(1), &c, width, window, sinks, &ws_bytes), op);
    const auto ws = workspace_for(q, ws_bytes);
    check_rc(qk_prompt_attention(q.const_data_ptr(), qk_dtype_of(q.scalar_type()), q.size(0), batch, q.size(1),
                                 stride_of(q, 0), stride_of(q, 1), index_data(cu_q), &c, paged ? nullptr : index_data(cu_k),
                                 paged ? index_data(table) : nullptr, width, paged ? stride_of(table, 0) : 0,
                                 paged ? index_data(lens) : nullptr, (float)s, window, sinks, out.data_ptr(),
                                 lse.data_ptr<float>(), ws.data_ptr(), ws_bytes, current_stream(q)),
             op);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> npu_prompt_attention_meta(const at::Tensor& query, const at::Tensor& key,
                                                             const at::Tensor& value, const at::Tensor& cu_seqlens_q,
                                                             const OptTensor& cu_seqlens_k, const OptTensor& block_table,
                                                             const OptTensor& context_lens, const OptTensor& key_scale,
                                                             const OptTensor& value_scale, std::optional<double> scale,
                                                             int64_t window, int64_t sinks) {
    const char* op = "npu_prompt_attention";
    const bool paged = block_table.has_value();
    const auto fit = [&](const at::Tensor& t) { return paged || t.dim() != 3 || last_is_dense(t) ? t : t.contiguous(); };
    const qk_kv_cache c = prompt_attention_check(op, query, fit(key), fit(value), cu_seqlens_q, cu_seqlens_k, block_table,
                                                 context_lens, key_scale, value_scale, window, sinks);
    scale_or_default(op, scale, c.head_dim);
    if (query.size(0) > 0) {
        check_cache_limits(op, c, key, value, paged);
        size_t ws_bytes = 0;
        check_rc(qk_prompt_attention_workspace_size(query.size(0), cu_seqlens_q.size(0) - 1, query.size(1), &c,
                                                    paged ? block_table->size(1) : 0, window, sinks, &ws_bytes),
                 op);
    }
    return attention_outputs(query);
}

// ---------------------------------------------------------------- npu_mrope, npu_mrope_scatter_kv

struct Mrope {
    std::vector<int64_t> sections;
    int64_t axes = 1;
    bool interleave = false;
};

Mrope mrope_check(const char* op, const at::Tensor& positions, const at::Tensor& q, const at::Tensor& k,
                  const at::Tensor& cos_sin, const at::OptionalIntArrayRef& section, c10::string_view mode) {
    check_query(op, q, nullptr);
    TORCH_CHECK(k.dim() == 3 && k.scalar_type() == q.scalar_type() && k.size(0) == q.size(0) && k.size(2) == q.size(2), op,
                ": key must be [tokens, heads, head_dim] of the query's tokens, head_dim and dtype, got ", k.scalar_type(),
                " ", k.sizes(), " beside ", q.scalar_type(), " ", q.sizes());
    check_device(op, "key", k, q);
    TORCH_CHECK(cos_sin.dim() == 2 && (cos_sin.scalar_type() == at::kFloat || cos_sin.scalar_type() == q.scalar_type()), op,
                ": cos_sin_cache must be [positions, rotary_dim] in float32 or ", q.scalar_type(), ", got ",
                cos_sin.scalar_type(), " ", cos_sin.sizes());
    check_device(op, "cos_sin_cache", cos_sin, q);
    const int64_t R = cos_sin.size(1);
    TORCH_CHECK(R >= 2 && R % 2 == 0 && R <= q.size(2), op, ": rotary_dim must be even and at most head_dim ", q.size(2),
                ", got ", R);
    TORCH_CHECK(mode == "half" || mode == "interleave", op, ": rotary_mode must be 'half' or 'interleave', got '", mode, "'");
    TORCH_CHECK(positions.dim() == 1 || positions.dim() == 2, op, ": positions must be [tokens] or [axes, tokens], got ",
                positions.sizes());
    check_index(op, "positions", positions, positions.dim(), q);
    TORCH_CHECK(positions.size(-1) == q.size(0), op, ": positions must have one column per token, got ", positions.sizes(),
                " for ", q.size(0), " tokens");
    Mrope m;
    m.interleave = mode == "interleave";
    m.axes = positions.dim() == 2 ? positions.size(0) : 1;
    TORCH_CHECK(m.axes >= 1 && m.axes <= 4, op, ": positions of 1 to 4 axes, got ", m.axes);
    if (section.has_value()) m.sections = section->vec();
    TORCH_CHECK(section.has_value() || m.axes == 1, op, ": ", m.axes, " axes need mrope_section");
    if (section.has_value()) {
        TORCH_CHECK((int64_t)m.sections.size() == m.axes, op, ": mrope_section must have ", m.axes, " values, got ", m.sections);
        int64_t sum = 0;
        for (int64_t n : m.sections) {
            TORCH_CHECK(n >= 0, op, ": mrope_section must not be negative, got ", m.sections);
            sum += n;
        }
        TORCH_CHECK(sum == R / 2, op, ": mrope_section must sum to rotary_dim / 2 = ", R / 2, ", got ", m.sections);
    }
    return m;
}

// What the C ABI refuses of the heads, for Meta calls.
void check_mrope_limits(const char* op, const at::Tensor& q, const at::Tensor& k) {
    TORCH_CHECK(q.size(2) <= 256, op, ": head_dim must be 1..256 (got ", q.size(2), ")");
    TORCH_CHECK(q.size(1) <= 65535 && k.size(1) <= 65535, op, ": invalid size q_heads=", q.size(1), " kv_heads=", k.size(1));
}

void mrope_launch(const char* op, const Mrope& m, const at::Tensor& positions_in, const at::Tensor& q_in,
                  const at::Tensor& k_in, const at::Tensor* v_in, const at::Tensor& cos_sin_in, const at::Tensor& out_q,
                  const at::Tensor* out_k, const qk_kv_cache* c, const int32_t* slots) {
    const auto dense = [](const at::Tensor& t) { return last_is_dense(t) ? t : t.contiguous(); };
    const auto q = dense(q_in), k = dense(k_in), v = v_in ? dense(*v_in) : at::Tensor();
    const auto positions = dense(positions_in), cos_sin = cos_sin_in.contiguous();
    check_rc(qk_mrope(q.const_data_ptr(), k.const_data_ptr(), v_in ? v.const_data_ptr() : nullptr,
                      qk_dtype_of(q.scalar_type()), q.size(0), q.size(1), k.size(1), q.size(2), stride_of(q, 0),
                      stride_of(q, 1), stride_of(k, 0), stride_of(k, 1), v_in ? stride_of(v, 0) : 0,
                      v_in ? stride_of(v, 1) : 0, index_data(positions), m.axes,
                      positions.dim() == 2 ? stride_of(positions, 0) : 0, m.sections.empty() ? nullptr : m.sections.data(),
                      cos_sin.const_data_ptr(), qk_dtype_of(cos_sin.scalar_type()), cos_sin.size(0), cos_sin.size(1),
                      m.interleave, out_q.data_ptr(), out_k ? out_k->data_ptr() : nullptr, c, slots, current_stream(q)),
             op);
}

std::tuple<at::Tensor, at::Tensor> npu_mrope(const at::Tensor& positions, const at::Tensor& query, const at::Tensor& key,
                                             const at::Tensor& cos_sin_cache, at::OptionalIntArrayRef mrope_section,
                                             c10::string_view rotary_mode) {
    const char* op = "npu_mrope";
    const Mrope m = mrope_check(op, positions, query, key, cos_sin_cache, mrope_section, rotary_mode);
    const c10::DeviceGuard guard(query.device());
    auto out_q = at::empty(query.sizes(), query.options()), out_k = at::empty(key.sizes(), key.options());
    if (query.size(0) > 0)
        mrope_launch(op, m, positions, query, key, nullptr, cos_sin_cache, out_q, &out_k, nullptr, nullptr);
    return {out_q, out_k};
}

std::tuple<at::Tensor, at::Tensor> npu_mrope_meta(const at::Tensor& positions, const at::Tensor& query,
                                                  const at::Tensor& key, const at::Tensor& cos_sin_cache,
                                                  at::OptionalIntArrayRef mrope_section, c10::string_view rotary_mode) {
    mrope_check("npu_mrope", positions, query, key, cos_sin_cache, mrope_section, rotary_mode);
    if (query.size(0) > 0) check_mrope_limits("npu_mrope", query, key);
    return {at::empty(query.sizes(), query.options()), at::empty(key.sizes(), key.options())};
}

qk_kv_cache scatter_check(const char* op, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                          const at::Tensor& key_cache, const at::Tensor& value_cache, const at::Tensor& slots,
                          const OptTensor& key_scale, const OptTensor& value_scale) {
    TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), op, ": value must be as key, got ",
                v.scalar_type(), " ", v.sizes(), " and ", k.scalar_type(), " ", k.sizes());
    check_device(op, "value", v, q);
    const qk_kv_cache c = cache_shape(op, key_cache, value_cache, key_scale, value_scale, q, true);
    TORCH_CHECK(c.kv_heads == k.size(1) && c.head_dim == k.size(2), op, ": the cache must have the key's heads and head_dim, got ",
                key_cache.sizes(), " and ", k.sizes());
    check_index(op, "slot_mapping", slots, 1, q);
    TORCH_CHECK(slots.size(0) == q.size(0), op, ": slot_mapping must have one slot per token, got ", slots.sizes());
    return c;
}

at::Tensor npu_mrope_scatter_kv(const at::Tensor& positions, const at::Tensor& query, const at::Tensor& key,
                                const at::Tensor& value, const at::Tensor& cos_sin_cache, const at::Tensor& key_cache,
                                const at::Tensor& value_cache, const at::Tensor& slot_mapping, const OptTensor& key_scale,
                                const OptTensor& value_scale, at::OptionalIntArrayRef mrope_section,
                                c10::string_view rotary_mode) {
    const char* op = "npu_mrope_scatter_kv";
    const Mrope m = mrope_check(op, positions, query, key, cos_sin_cache, mrope_section, rotary_mode);
    qk_kv_cache c = scatter_check(op, query, key, value, key_cache, value_cache, slot_mapping, key_scale, value_scale);
    const c10::DeviceGuard guard(query.device());
    cache_data(c, key_cache, value_cache, key_scale, value_scale);
    auto out_q = at::empty(query.sizes(), query.options());
    if (query.size(0) == 0) return out_q;
    const auto slots = slot_mapping.contiguous();
    mrope_launch(op, m, positions, query, key, &value, cos_sin_cache, out_q, nullptr, &c, index_data(slots));
    return out_q;
}

at::Tensor npu_mrope_scatter_kv_meta(const at::Tensor& positions, const at::Tensor& query, const at::Tensor& key,
                                     const at::Tensor& value, const at::Tensor& cos_sin_cache, const at::Tensor& key_cache,
                                     const at::Tensor& value_cache, const at::Tensor& slot_mapping,
                                     const OptTensor& key_scale, const OptTensor& value_scale,
                                     at::OptionalIntArrayRef mrope_section, c10::string_view rotary_mode) {
    const char* op = "npu_mrope_scatter_kv";
    mrope_check(op, positions, query, key, cos_sin_cache, mrope_section, rotary_mode);
    const qk_kv_cache c = scatter_check(op, query, key, value, key_cache, value_cache, slot_mapping, key_scale, value_scale);
    if (query.size(0) > 0) {
        check_mrope_limits(op, query, key);
        check_cache_limits(op, c, key_cache, value_cache, true);
    }
    return at::empty(query.sizes(), query.options());
}

// ---------------------------------------------------------------- pages

// A page (the dimensions behind the first) fills its bytes, in whatever order.  From the sizes and strides alone: a view per tensor
// would cost more than the launch.
bool page_is_dense(const at::Tensor& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t next = 1;
    uint64_t done = 0;
    for (int64_t left = t.dim() - 1; left > 0; --left) {
        int64_t found = 0;  // the dimension whose stride is the product of those before it
        for (int64_t d = 1; d < t.dim() && !found; ++d)
            if (!(done >> d & 1) && (sizes[d] == 1 || strides[d] == next)) found = d;
        if (!found) return false;
        done |= (uint64_t)1 << found;
        next *= sizes[found];
    }
    return true;
}

std::vector<qk_pages> page_list(const char* op, at::TensorList caches, int64_t num_pages, const at::Tensor& like) {
    std::vector<qk_pages> list;
    list.reserve(caches.size());
    for (const at::Tensor& t : caches) {
        TORCH_CHECK(t.dim() >= 1 && t.dim() <= 64 && t.size(0) == num_pages, op, ": every cache tensor must have ", num_pages,
                    " pages in its first dimension, got ", t.sizes());
        check_device(op, "a cache tensor", t, like);
        if (t.numel() == 0) continue;
        TORCH_CHECK(page_is_dense(t), op, ": a page of a cache tensor must be dense, got sizes ",
                    t.sizes(), " and strides ", t.strides());
        const int64_t bytes = t.numel() / num_pages * t.element_size();
        TORCH_CHECK(num_pages == 1 || t.stride(0) * t.element_size() >= bytes, op, ": pages of a cache tensor overlap");
        list.push_back({t.is_meta() ? nullptr : t.data_ptr(), num_pages == 1 ? bytes : t.stride(0) * t.element_size(), bytes});
    }
    return list;
}

void check_seqs(const char* op, const at::Tensor& seqs) {
    TORCH_CHECK(seqs.numel() <= QK_MAX_SEQS, op, ": ", seqs.numel(), " sequences (at most ", QK_MAX_SEQS, " a call)");
}

void check_slots(const char* op, const at::Tensor& table, const at::Tensor& count, int64_t page_size) {
    const int64_t most = std::numeric_limits<int32_t>::max() / page_size;
    TORCH_CHECK(count.size(0) <= most && table.size(1) <= most, op, ": sizes past 31 bits");
}

void check_pool(const char* op, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count) {
    check_index(op, "block_table", table, 2, table);
    check_index(op, "context_lens", lens, 1, table);
    check_index(op, "ref_count", count, 1, table);
    TORCH_CHECK(lens.size(0) == table.size(0), op, ": context_lens must have one length per row of block_table, got ",
                lens.sizes(), " and ", table.sizes());
    TORCH_CHECK(last_is_dense(table) && lens.is_contiguous() && count.is_contiguous() &&
                    (table.size(0) <= 1 || table.stride(0) >= table.size(1)),
                op, ": block_table's rows, context_lens and ref_count must be contiguous");
}

int32_t* written(const at::Tensor& t) { return t.numel() ? t.data_ptr<int32_t>() : nullptr; }

void copy_check(const char* op, at::TensorList caches, const at::Tensor& src, const at::Tensor& dst) {
    check_index(op, "src", src, 1, src);
    check_index(op, "dst", dst, 1, src);
    TORCH_CHECK(src.sizes() == dst.sizes(), op, ": src and dst must have one length, got ", src.sizes(), " and ", dst.sizes());
    TORCH_CHECK(caches.empty() || caches[0].dim() >= 1, op, ": a cache tensor needs a dimension of pages");
}

void npu_kv_copy_pages(at::TensorList caches, const at::Tensor& src_in, const at::Tensor& dst_in) {
    const char* op = "npu_kv_copy_pages";
    copy_check(op, caches, src_in, dst_in);
    if (caches.empty()) return;
    const c10::DeviceGuard guard(src_in.device());
    const int64_t num_pages = caches[0].size(0);
    const auto list = page_list(op, caches, num_pages, src_in);
    const auto src = src_in.contiguous(), dst = dst_in.contiguous();
    check_rc(qk_kv_copy_pages(list.data(), (int64_t)list.size(), num_pages, index_data(src), index_data(dst), src.numel(),
                              current_stream(src)),
             op);
}

void npu_kv_copy_pages_meta(at::TensorList caches, const at::Tensor& src, const at::Tensor& dst) {
    copy_check("npu_kv_copy_pages", caches, src, dst);
    if (!caches.empty()) page_list("npu_kv_copy_pages", caches, caches[0].size(0), src);
}

void fork_check(const char* op, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count,
                const at::Tensor& parents, const at::Tensor& children, int64_t page_size) {
    check_pool(op, table, lens, count);
    check_index(op, "parents", parents, 1, table);
    check_index(op, "children", children, 1, table);
    TORCH_CHECK(parents.sizes() == children.sizes(), op, ": parents and children must have one length, got ",
                parents.sizes(), " and ", children.sizes());
    TORCH_CHECK(page_size > 0, op, ": page_size must be positive, got ", page_size);
    check_seqs(op, parents);
    check_slots(op, table, count, page_size);
}

at::Tensor npu_kv_fork(at::TensorList caches, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count,
                       const at::Tensor& parents_in, const at::Tensor& children_in, int64_t page_size) {
    const char* op = "npu_kv_fork";
    fork_check(op, table, lens, count, parents_in, children_in, page_size);
    const c10::DeviceGuard guard(table.device());
    const auto list = page_list(op, caches, count.size(0), table);
    const auto parents = parents_in.contiguous(), children = children_in.contiguous();
    auto missing = at::empty({1}, table.options());
    size_t ws_bytes = 0;
    check_rc(qk_kv_fork_workspace_size(parents.numel(), &ws_bytes), op);
    const auto ws = workspace_for(table, ws_bytes);
    check_rc(qk_kv_fork(list.data(), (int64_t)list.size(), count.size(0), page_size, written(table), table.size(0),
                        table.size(1), stride_of(table, 0), written(lens), written(count), index_data(parents),
                        index_data(children), parents.numel(), missing.data_ptr<int32_t>(), ws.data_ptr(), ws_bytes,
                        current_stream(table)),
             op);
    return missing;
}

at::Tensor npu_kv_fork_meta(at::TensorList caches, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count,
                            const at::Tensor& parents, const at::Tensor& children, int64_t page_size) {
    fork_check("npu_kv_fork", table, lens, count, parents, children, page_size);
    page_list("npu_kv_fork", caches, count.size(0), table);
    return at::empty({1}, table.options());
}

void free_check(const char* op, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count,
                const at::Tensor& seqs, int64_t page_size) {
    check_pool(op, table, lens, count);
    check_index(op, "seqs", seqs, 1, table);
    TORCH_CHECK(page_size > 0, op, ": page_size must be positive, got ", page_size);
    check_seqs(op, seqs);
    check_slots(op, table, count, page_size);
}

void npu_kv_free(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count, const at::Tensor& seqs_in,
                 int64_t page_size) {
    const char* op = "npu_kv_free";
    free_check(op, table, lens, count, seqs_in, page_size);
    const c10::DeviceGuard guard(table.device());
    const auto seqs = seqs_in.contiguous();
    check_rc(qk_kv_free(count.size(0), page_size, written(table), table.size(0), table.size(1), stride_of(table, 0),
                        written(lens), written(count), index_data(seqs), seqs.numel(), current_stream(table)),
             op);
}

void npu_kv_free_meta(const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count, const at::Tensor& seqs,
                      int64_t page_size) {
    free_check("npu_kv_free", table, lens, count, seqs, page_size);
}

void extend_check(const char* op, const at::Tensor& table, const at::Tensor& lens, const at::Tensor& count,
                  const at::Tensor& seqs, const at::Tensor& cu, int64_t total, int64_t page_size) {
    free_check(op, table, lens, count, seqs, page_size);
    check_index(op, "cu_tokens", cu, 1, table);
    TORCH_CHECK(cu.size(0) == seqs.size(0) + 1, op, ": cu_tokens must have one value more than seqs, got ", cu.sizes(),
                " and ", seqs.sizes());
    TORCH_CHECK(total >= 0, op, ": total_tokens must not be negative, got ", total);
    TORCH_CHECK(total <= std::numeric_limits<int32_t>::max(), op, ": invalid number of tokens ", total);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> npu_kv_extend(const at::Tensor& table, const at::Tensor& lens,
                                                             const at::Tensor& count, const at::Tensor& seqs_in,
                                                             const at::Tensor& cu_in, int64_t total, int64_t page_size) {
    const char* op = "npu_kv_extend";
    extend_check(op, table, lens, count, seqs_in, cu_in, total, page_size);
    const c10::DeviceGuard guard(table.device());
    const auto seqs = seqs_in.contiguous(), cu = cu_in.contiguous();
    auto slots = at::empty({total}, table.options()), positions = at::empty({total}, table.options());
    auto missing = at::empty({1}, table.options());
    size_t ws_bytes = 0;
    check_rc(qk_kv_extend_workspace_size(seqs.numel(), count.size(0), &ws_bytes), op);
    const auto ws = workspace_for(table, ws_bytes);
    check_rc(qk_kv_extend(count.size(0), page_size, written(table), table.size(0), table.size(1), stride_of(table, 0),
                          written(lens), written(count), index_data(seqs), index_data(cu), seqs.numel(), total,
                          written(slots), written(positions), missing.data_ptr<int32_t>(), ws.data_ptr(), ws_bytes,
                          current_stream(table)),
             op);
    return {slots, positions, missing};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> npu_kv_extend_meta(const at::Tensor& table, const at::Tensor& lens,
                                                                  const at::Tensor& count, const at::Tensor& seqs,
                                                                  const at::Tensor& cu, int64_t total, int64_t page_size) {
    extend_check("npu_kv_extend", table, lens, count, seqs, cu, total, page_size);
    return {at::empty({total}, table.options()), at::empty({total}, table.options()), at::empty({1}, table.options())};
}

void compact_check(const char* op, const at::Tensor& table, const at::Tensor& count) {
    check_index(op, "block_table", table, 2, table);
    check_index(op, "ref_count", count, 1, table);
    check_slots(op, table, count, 1);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> npu_kv_compact(at::TensorList caches, const at::Tensor& table_in,
                                                              const at::Tensor& count_in) {
    const char* op = "npu_kv_compact";
    compact_check(op, table_in, count_in);
    const c10::DeviceGuard guard(table_in.device());
    const auto list = page_list(op, caches, count_in.size(0), table_in);
    const auto table = table_in.contiguous(), count = count_in.contiguous();
    auto new_table = at::empty(table.sizes(), table.options()), new_count = at::empty(count.sizes(), table.options());
    auto moved = at::empty({1}, table.options());
    size_t ws_bytes = 0;
    check_rc(qk_kv_compact_workspace_size(count.size(0), &ws_bytes), op);
    const auto ws = workspace_for(table, ws_bytes);
    check_rc(qk_kv_compact(list.data(), (int64_t)list.size(), count.size(0), index_data(table), table.size(0),
                           table.size(1), table.size(1), index_data(count), written(new_table), written(new_count),
                           moved.data_ptr<int32_t>(), ws.data_ptr(), ws_bytes, current_stream(table)),
             op);
    return {new_table, new_count, moved};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> npu_kv_compact_meta(at::TensorList caches, const at::Tensor& table,
                                                                   const at::Tensor& count) {
    compact_check("npu_kv_compact", table, count);
    page_list("npu_kv_compact", caches, count.size(0), table);
    return {at::empty(table.sizes(), table.options()), at::empty(count.sizes(), table.options()),
            at::empty({1}, table.options())};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(npu, m) {
    m.def("npu_paged_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
          "Tensor context_lens, *, Tensor? key_scale=None, Tensor? value_scale=None, float? scale=None, int window=0, "
          "int sinks=0) -> (Tensor, Tensor)");
    m.def("npu_prompt_attention(Tensor query, Tensor key, Tensor value, Tensor cu_seqlens_q, *, Tensor? cu_seqlens_k=None, "
          "Tensor? block_table=None, Tensor? context_lens=None, Tensor? key_scale=None, Tensor? value_scale=None, "
          "float? scale=None, int window=0, int sinks=0) -> (Tensor, Tensor)");
    m.def("npu_mrope(Tensor positions, Tensor query, Tensor key, Tensor cos_sin_cache, *, int[]? mrope_section=None, "
          "str rotary_mode='half') -> (Tensor, Tensor)");
    m.def("npu_mrope_scatter_kv(Tensor positions, Tensor query, Tensor key, Tensor value, Tensor cos_sin_cache, "
          "Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slot_mapping, *, Tensor(c!)? key_scale=None, "
          "Tensor(d!)? value_scale=None, int[]? mrope_section=None, str rotary_mode='half') -> Tensor");
    m.def("npu_kv_copy_pages(Tensor(a!)[] caches, Tensor src, Tensor dst) -> ()");
    m.def("npu_kv_fork(Tensor(a!)[] caches, Tensor(b!) block_table, Tensor(c!) context_lens, Tensor(d!) ref_count, "
          "Tensor parents, Tensor children, int page_size) -> Tensor");
    m.def("npu_kv_free(Tensor(a!) block_table, Tensor(b!) context_lens, Tensor(c!) ref_count, Tensor seqs, "
          "int page_size) -> ()");
    m.def("npu_kv_extend(Tensor(a!) block_table, Tensor(b!) context_lens, Tensor(c!) ref_count, Tensor seqs, "
          "Tensor cu_tokens, int total_tokens, int page_size) -> (Tensor, Tensor, Tensor)");
    m.def("npu_kv_compact(Tensor(a!)[] caches, Tensor block_table, Tensor ref_count) -> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) {
    m.impl("npu_paged_attention", &npu_paged_attention);
    m.impl("npu_prompt_attention", &npu_prompt_attention);
    m.impl("npu_mrope", &npu_mrope);
    m.impl("npu_mrope_scatter_kv", &npu_mrope_scatter_kv);
    m.impl("npu_kv_copy_pages", &npu_kv_copy_pages);
    m.impl("npu_kv_fork", &npu_kv_fork);
    m.impl("npu_kv_free", &npu_kv_free);
    m.impl("npu_kv_extend", &npu_kv_extend);
    m.impl("npu_kv_compact", &npu_kv_compact);
}

TORCH_LIBRARY_IMPL(npu, Meta, m) {
    m.impl("npu_paged_attention", &npu_paged_attention_meta);
    m.impl("npu_prompt_attention", &npu_prompt_attention_meta);
    m.impl("npu_mrope", &npu_mrope_meta);
    m.impl("npu_mrope_scatter_kv", &npu_mrope_scatter_kv_meta);
    m.impl("npu_kv_copy_pages", &npu_kv_copy_pages_meta);
    m.impl("npu_kv_fork", &npu_kv_fork_meta);
    m.impl("npu_kv_free", &npu_kv_free_meta);
    m.impl("npu_kv_extend", &npu_kv_extend_meta);
    m.impl("npu_kv_compact", &npu_kv_compact_meta);
}
