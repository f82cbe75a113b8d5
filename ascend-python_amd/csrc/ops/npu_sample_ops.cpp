// torch.ops.npu.npu_sample: a token per row of logits.  As the other ops: shapes, types and devices are checked with TORCH_CHECK,
// outputs and workspace allocated, the launch goes through the C ABI on the current stream.  Registered for the CUDA key (HIP
// tensors) and for Meta, which runs the same checks without launching.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../../include/qk_abi.h"

namespace {

using OptTensor = std::optional<at::Tensor>;
constexpr const char* kOp = "npu_sample";

void check_rc(int rc) { TORCH_CHECK(rc == QK_OK, "call ", kOp, " failed, detail:", qk_last_error()); }

int qk_dtype_of(at::ScalarType t) { return t == at::kHalf ? QK_F16 : t == at::kBFloat16 ? QK_BF16 : QK_F32; }

void check_setting(const char* name, const at::Tensor& t, at::ScalarType type, const at::Tensor& x) {
    TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.size(0) == x.size(0), kOp, ": ", name, " must be ", type, " [", x.size(0),
                "], got ", t.scalar_type(), " ", t.sizes());
    TORCH_CHECK(t.device() == x.device(), kOp, ": ", name, " must be on ", x.device(), ", got ", t.device());
}

void sample_check(const at::Tensor& x, const at::Tensor& uniform, const OptTensor& temperature, const OptTensor& top_k,
                  const OptTensor& top_p, const OptTensor& min_p) {
    TORCH_CHECK(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, kOp,
                ": logits must be float16, bfloat16 or float32, got ", x.scalar_type());
    TORCH_CHECK(x.dim() == 2, kOp, ": logits must be [rows, vocabulary], got ", x.sizes());
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= QK_MAX_VOCAB, kOp, ": a vocabulary of 1 to ", QK_MAX_VOCAB, " tokens, got ", x.size(1));
    TORCH_CHECK(x.size(0) <= QK_MAX_SAMPLE_ROWS, kOp, ": invalid number of rows ", x.size(0), ", at most ", QK_MAX_SAMPLE_ROWS);
    check_setting("uniform", uniform, at::kFloat, x);
    if (temperature.has_value()) check_setting("temperature", *temperature, at::kFloat, x);
    if (top_k.has_value()) check_setting("top_k", *top_k, at::kInt, x);
    if (top_p.has_value()) check_setting("top_p", *top_p, at::kFloat, x);
    if (min_p.has_value()) check_setting("min_p", *min_p, at::kFloat, x);
}

std::tuple<at::Tensor, at::Tensor> outputs(const at::Tensor& x) {
    return {at::empty({x.size(0)}, x.options().dtype(at::kInt)), at::empty({x.size(0)}, x.options().dtype(at::kFloat))};
}

std::tuple<at::Tensor, at::Tensor> npu_sample(const at::Tensor& logits, const at::Tensor& uniform_in, const OptTensor& temperature,
                                              const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p) {
    sample_check(logits, uniform_in, temperature, top_k, top_p, min_p);
    const c10::DeviceGuard guard(logits.device());
    auto [tokens, logprobs] = outputs(logits);
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    if (rows == 0) return {tokens, logprobs};
    const auto x = vocab == 1 || logits.stride(1) == 1 ? logits : logits.contiguous();
    const auto uniform = uniform_in.contiguous();
    at::Tensor held[4];
    const auto setting = [&](int i, const OptTensor& t) { return t.has_value() ? (held[i] = t->contiguous()).const_data_ptr() : nullptr; };
    const auto* t = (const float*)setting(0, temperature);
    const auto* k = (const int32_t*)setting(1, top_k);
    const auto *p = (const float*)setting(2, top_p), *m = (const float*)setting(3, min_p);
    const int dtype = qk_dtype_of(x.scalar_type());
    size_t ws_bytes = 0;
    check_rc(qk_sample_workspace_size(rows, vocab, dtype, &ws_bytes));
    const auto ws = at::empty({(int64_t)ws_bytes}, x.options().dtype(at::kByte));
    check_rc(qk_sample(x.const_data_ptr(), dtype, rows, vocab, rows > 1 ? x.stride(0) : 0, uniform.const_data_ptr<float>(), t, k, p, m,
                       tokens.data_ptr<int32_t>(), logprobs.data_ptr<float>(), ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                       reinterpret_cast<qk_stream_t>(c10::hip::getCurrentHIPStream(x.device().index()).stream())));
    return {tokens, logprobs};
}

std::tuple<at::Tensor, at::Tensor> npu_sample_meta(const at::Tensor& logits, const at::Tensor& uniform, const OptTensor& temperature,
                                                   const OptTensor& top_k, const OptTensor& top_p, const OptTensor& min_p) {
    sample_check(logits, uniform, temperature, top_k, top_p, min_p);
    return outputs(logits);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(npu, m) {
    m.def("npu_sample(Tensor logits, Tensor uniform, *, Tensor? temperature=None, Tensor? top_k=None, Tensor? top_p=None, "
          "Tensor? min_p=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(npu, CUDA, m) { m.impl("npu_sample", &npu_sample); }

TORCH_LIBRARY_IMPL(npu, Meta, m) { m.impl("npu_sample", &npu_sample_meta); }
