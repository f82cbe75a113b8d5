// extern "C" entry points of sampling (declared in include/qk_abi.h): the checks of its plain arguments and the launch on the caller's
// stream.  Nothing here allocates or synchronises.
#include <cstdarg>
#include <cstdio>

#include "kernels/attention.h"
#include "kernels/sample.h"

namespace {

constexpr const char* kOp = "npu_sample";

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return qk::abi_error(code, buf);
}

int check_sizes(int64_t rows, int64_t vocab, int dtype) {
    if (dtype != QK_F16 && dtype != QK_BF16 && dtype != QK_F32)
        return fail(QK_ERR_ARG, "%s: logits must be float16, bfloat16 or float32 (got dtype %d)", kOp, dtype);
    // a launch holds less than 2^32 threads
    if (rows < 0 || rows > QK_MAX_SAMPLE_ROWS)
        return fail(QK_ERR_ARG, "%s: invalid number of rows %lld (at most %d)", kOp, (long long)rows, QK_MAX_SAMPLE_ROWS);
    if (vocab < 1 || vocab > QK_MAX_VOCAB)
        return fail(QK_ERR_UNSUPPORTED, "%s: a vocabulary of 1 to %d tokens (got %lld)", kOp, QK_MAX_VOCAB, (long long)vocab);
    return QK_OK;
}

}  // namespace

extern "C" {

int qk_sample_workspace_size(int64_t rows, int64_t vocab, int dtype, size_t* bytes) {
    qk::abi_begin();
    if (!bytes) return fail(QK_ERR_ARG, "%s: null pointer", kOp);
    if (int rc = check_sizes(rows, vocab, dtype)) return rc;
    *bytes = qk::sample_workspace(rows, vocab, dtype);
    return QK_OK;
}

int qk_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, const float* uniform,
              const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
              float* logprobs, void* workspace, size_t workspace_bytes, qk_stream_t stream) {
    qk::abi_begin();
    if (int rc = check_sizes(rows, vocab, dtype)) return rc;
    if (rows == 0) return QK_OK;
    if (!logits || !uniform || !tokens || !logprobs) return fail(QK_ERR_ARG, "%s: null pointer", kOp);
    if (row_stride < 0) return fail(QK_ERR_ARG, "%s: negative stride", kOp);
    if ((uintptr_t)logits % (dtype == QK_F32 ? 4 : 2) != 0) return fail(QK_ERR_ARG, "%s: logits that are not whole elements", kOp);
    const qk::SampleArgs a = {logits, dtype, rows, vocab, row_stride, uniform, temperature, top_k, top_p, min_p, tokens, logprobs};
    const size_t need = qk::sample_workspace(rows, vocab, dtype);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(QK_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", kOp, need, workspace_bytes);
    if (need > 0 && (uintptr_t)workspace % 256 != 0) return fail(QK_ERR_WORKSPACE, "%s: the workspace must be 256-byte aligned", kOp);
    const hipError_t e = qk::launch_sample(a, workspace, (hipStream_t)stream);
    if (e != hipSuccess) return fail(QK_ERR_LAUNCH, "%s: kernel launch failed: %s", kOp, hipGetErrorString(e));
    return QK_OK;
}

}  // extern "C"
