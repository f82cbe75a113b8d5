/*
 * qk_abi.h -- C ABI of libqk_hip.so, the MI355X (gfx950) kernels of the
 * quantized-inference hot path: npu_dynamic_quant, npu_quant_matmul (W8A8)
 * and npu_weight_quant_batchmatmul (W4A16 / W8A16).
 *
 * This is the layer the reference reaches through EXEC_NPU_CMD
 * (op_plugin/utils/op_api_common.h:520-570): a two-phase C call,
 * "<op>GetWorkspaceSize" then "<op>(workspace, size, executor, stream)",
 * resolved by dlsym from libcust_opapi.so / libopapi.so
 * (op_plugin/utils/op_api_common.h:80-123).  Here the two phases are
 * qk_*_workspace_size() and the op call itself; operands are plain device
 * pointers, sizes and strides instead of aclTensor descriptors, so no torch
 * or vendor type appears in a signature.
 *
 * Contract, as in the reference boundary:
 *   - the caller allocates every output and the workspace
 *     (op_plugin/ops/base_ops/opapi/MmKernelNpuOpApi.cpp:27-30,
 *      op_plugin/utils/op_api_common.h:547-551); the library allocates nothing;
 *   - work is enqueued on `stream` and never synchronised
 *     (op_plugin/utils/op_api_common.h:530, 563-566);
 *   - a non-zero return is an error and qk_last_error() gives a thread-local
 *     message (the reference's aclGetRecentErrMsg(),
 *     op_plugin/utils/op_api_common.h:546, 555).
 * All functions are thread-safe; calls on one stream execute in order.
 *
 * Workspaces, as the reference's per-call scratch
 * (op_plugin/utils/op_api_common.h:547-551, unsafe_empty_workspace): the
 * caller passes at least *_workspace_size() bytes, 256-byte aligned, of any
 * contents -- uninitialised memory is fine.  A non-empty workspace begins with
 * QK_SPLIT_COUNTER_BYTES of split-K arrival counters, followed by the partial
 * sums (split-K shapes) or by the activations' per-group sums (weight-quant
 * matmul at large M; where a row-major weight is cast per call -- from M = 17
 * on an int4 weight where that is faster, from M = 33 on an int8 weight -- the
 * weight cast to NZ, K*N/2 (int4) or K*N
 * (int8) bytes rounded to 256, comes first, then the sums or the fp32 partial
 * tiles of the mid-M kernel's K splits (none where the NZ decode kernel runs);
 * where the NZ prefill kernel runs stream-K, (P - 1) x 128 KB of fp32 partial slots follow
 * the sums, P being the current device's CU count).  Each arrival adds D = tag * 2^16 + 1 to its
 * counter (a 48-bit tag drawn per call, never 0 or all ones), so a counter of
 * this call holds j * D after j arrivals; a zero word is empty (the last
 * arrival leaves zero behind), and any other word that is not such a multiple
 * -- what another user left there, a 0xFF fill -- is recognised as stale and
 * replaced.  The one exception is memory whose counter words happen to hold a
 * small multiple of this call's D (odds below 2^-48 per counter word for
 * random contents, zero for zero- or 0xFF-filled memory).  The workgroup that completes a tile's splits
 * adds them up itself, so no second kernel runs.  Calls that may be in flight
 * at the same time need distinct workspaces.
 */
#ifndef QK_ABI_H
#define QK_ABI_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same type as hipStream_t; NULL is the default (null) stream. */
typedef struct ihipStream_t* qk_stream_t;

/* Element types.  F16 = IEEE binary16, BF16 = bfloat16. */
typedef enum {
    QK_F16 = 1,
    QK_BF16 = 2,
    QK_F32 = 3,
    QK_I8 = 4,
    QK_I32 = 5,
    QK_U8 = 6,
    /* weight codes of qk_weight_quant_bmm for weights in the MFMA-tiled NZ
     * layouts that qk_weight_format_cast writes: int4, int32 [N/16][K/128][64][4];
     * int8, int8 [N/16][K/64][64][16] */
    QK_I4_NZ = 16,
    QK_I8_NZ = 17,
    /* weight code of qk_weight_quant_bmm for an int8 weight stored [N, K] (row n
     * holds column n's K values: the nn.Linear layout, which the op receives as
     * the transposed view [K, N] of that tensor); read in place, as the reference
     * flags a transposed mat2 instead of copying it
     * (op_plugin/ops/base_ops/aclops/MmKernelNpu.cpp:40-53,
     * op_plugin/ops/base_ops/aclops/LinearKernelNpu.cpp:39-40) */
    QK_I8_NK = 18
} qk_dtype;

/* Weight storage formats: the reference's aclFormat numbers for ND and
 * FRACTAL_NZ (op_plugin/third_party/acl/inc/graph/types.h:111, 138). */
#define QK_FORMAT_ND 2
#define QK_FORMAT_FRACTAL_NZ 29

/* Return codes. */
enum {
    QK_OK = 0,
    QK_ERR_ARG = -1,          /* invalid argument (shape, dtype, pointer, alignment) */
    QK_ERR_UNSUPPORTED = -2,  /* valid request this build does not implement */
    QK_ERR_WORKSPACE = -3,    /* workspace missing or smaller than *_workspace_size() */
    QK_ERR_LAUNCH = -4        /* the HIP runtime refused a launch */
};

/* Thread-local description of the last failure on this thread ("" if none). */
const char* qk_last_error(void);

/* ABI revision; bumped on any incompatible signature or contract change
 * (2: the split-K counters at the head of a workspace; 3: the counters are
 * tagged per call, so a workspace needs no initialisation; 4: NZ weights,
 * qk_weight_format_cast, static quantization; 5: the [N, K] int8 weight code
 * QK_I8_NK, int8 NZ weights with K % 64 == 0 in qk_weight_quant_bmm; 6: qk_quant_matmul_swiglu,
 * qk_quant_matmul_swiglu_quant). */
int qk_abi_version(void);

/* Debug and test hook, no counterpart in the reference: forces kernel choices
 * of the planners (spec grammar in csrc/kernels/common.h, "PlanOverride"; NULL
 * or "" restores the planners' own choices).  The library reads the
 * QK_DEBUG_PLAN environment variable once at first use; this call replaces
 * that for the rest of the process.  Not meant for production callers.
 * Returns QK_ERR_ARG (override unchanged) for a spec it does not understand. */
int qk_debug_set_plan(const char* spec);

/* Bytes of split-K counters at the start of every non-empty workspace. */
#define QK_SPLIT_COUNTER_BYTES 4096

/*
 * npu_dynamic_quant -- replaces aclnnDynamicQuant behind EXEC_NPU_CMD
 * (op_plugin/utils/op_api_common.h:520-570); the nearest reference op is the
 * static quantize_per_channel (op_plugin/ops/base_ops/aclops/QuantizePerChannelKernelNpu.cpp:69-92).
 * x: [rows, K] fp16/bf16, row-major.  smooth_scales: [K] fp32 or NULL.
 * y: [rows, K] int8.  scale: [rows] fp32.
 * Per row: s = max|x*smooth| / 127 (fp32 division), y = clamp(rint(x*smooth / s)),
 * ties to even; an all-zero row gives s = 0, y = 0.  No workspace.
 */
int qk_dynamic_quant(const void* x, int x_dtype, int64_t rows, int64_t K,
                     const float* smooth_scales, int8_t* y, float* scale, qk_stream_t stream);

/*
 * npu_quant_matmul (W8A8), phase 1 -- replaces aclnnQuantMatmul*GetWorkspaceSize
 * (op_plugin/utils/op_api_common.h:543-546).  Writes the workspace bytes the
 * call with the same shape needs (0 when none) to *bytes.
 */
int qk_quant_matmul_workspace_size(int64_t M, int64_t N, int64_t K, int out_dtype, size_t* bytes);

/*
 * npu_quant_matmul (W8A8), phase 2 -- replaces aclnnQuantMatmul* behind
 * EXEC_NPU_CMD (op_plugin/utils/op_api_common.h:552-566); shape/bias rules
 * follow mm / addmm (op_plugin/ops/base_ops/opapi/MmKernelNpuOpApi.cpp:24-32,
 * op_plugin/ops/base_ops/opapi/AddmmKernelNpuOpApi.cpp:24-55).
 * x1: int8 [M,K], row stride ldx1.  x2: int8 [K,N] addressed as
 * x2[k*x2_stride_k + n*x2_stride_n]; exactly one stride must be 1
 * ([K,N]-contiguous: (N',1); transposed view of [N,K]: (1,K')), as the
 * reference flags a transposed mat2 instead of copying it
 * (op_plugin/ops/base_ops/aclops/MmKernelNpu.cpp:40-53).
 * acc = sum_k x1*x2 in int32, exact: K above 131071 is refused (QK_ERR_UNSUPPORTED).
 * scale: fp32 [scale_len], scale_len 1 or N.  offset (int8 output only): fp32 [1|N] or NULL.
 * pertoken_scale: fp32 [M] or NULL.  bias: [N] of bias_dtype
 * (QK_I32: added to acc; QK_BF16/QK_F16/QK_F32: added after scaling) or NULL.
 * out: [M,N] row-major of out_dtype:
 *   QK_BF16/QK_F16: cast(fmaf(float(acc) [* pertoken[m]], scale[n], bias[n]))
 *   QK_I8:          clamp(rint(fmaf(float(acc), scale[n], offset[n])))
 *   QK_I32:         acc (+ int32 bias)
 */
int qk_quant_matmul(const int8_t* x1, int64_t ldx1,
                    const int8_t* x2, int64_t x2_stride_k, int64_t x2_stride_n,
                    int64_t M, int64_t N, int64_t K,
                    const float* scale, int64_t scale_len,
                    const float* offset, int64_t offset_len,
                    const float* pertoken_scale,
                    const void* bias, int bias_dtype,
                    void* out, int out_dtype,
                    void* workspace, size_t workspace_bytes, qk_stream_t stream);

/*
 * npu_quant_matmul (W8A8) on an int8 weight in the NZ layout, phase 1: the
 * workspace bytes qk_quant_matmul_nz needs for this shape (0 when none).
 */
int qk_quant_matmul_nz_workspace_size(int64_t M, int64_t N, int64_t K, int out_dtype, size_t* bytes);

/*
 * npu_quant_matmul (W8A8) on an int8 weight in the NZ layout, phase 2 -- the
 * same op as qk_quant_matmul with x2 already cast to the device-native tiled
 * format, as the reference casts matmul weights to FRACTAL_NZ before its
 * matmuls (op_plugin/ops/base_ops/aclops/MmKernelNpu.cpp:303-316,
 * op_plugin/ops/base_ops/aclops/LinearKernelNpu.cpp:103-107) and hands
 * aclnnQuantMatmul* the NZ tensor behind EXEC_NPU_CMD
 * (op_plugin/utils/op_api_common.h:552-566).
 * x2_nz: int8 [N/16][K/64][64][16] as qk_weight_format_cast writes it from
 * an int8 [K,N] weight (K % 64 == 0, N % 16 == 0).  x1, x2_nz and out must be
 * 16-byte aligned, ldx1 a multiple of 16 below 2^24.  Every other argument,
 * the arithmetic and the result are those of qk_quant_matmul (bit-identical
 * outputs for the same weight in either layout).
 */
int qk_quant_matmul_nz(const int8_t* x1, int64_t ldx1, const int8_t* x2_nz,
                       int64_t M, int64_t N, int64_t K,
                       const float* scale, int64_t scale_len,
                       const float* offset, int64_t offset_len,
                       const float* pertoken_scale,
                       const void* bias, int bias_dtype,
                       void* out, int out_dtype,
                       void* workspace, size_t workspace_bytes, qk_stream_t stream);

/*
 * npu_weight_quant_batchmatmul, phase 1 (see qk_quant_matmul_workspace_size).
 */
int qk_weight_quant_bmm_workspace_size(int64_t M, int64_t N, int64_t K, int weight_dtype,
                                       int64_t group_size, size_t* bytes);

/*
 * npu_weight_quant_batchmatmul (W4A16 / W8A16), phase 2 -- replaces
 * aclnnWeightQuantBatchMatmul* behind EXEC_NPU_CMD; the nearest reference op
 * is bmm (op_plugin/ops/base_ops/opapi/BmmKernelNpuOpApi.cpp:24-52).
 * x: [M,K] fp16/bf16 row-major.  weight: QK_I32 -> int4 packed [K, N/8]
 * (nibble i of word j is column 8j+i, two's complement); QK_I8 -> int8 [K,N];
 * QK_I8_NK -> int8 stored [N,K] (element (k, n) at weight[n*K + k]); QK_I4_NZ /
 * QK_I8_NZ -> int4 / int8 in the NZ layouts of qk_weight_format_cast
 * (N % 16 == 0; K % 128 == 0 for int4, K % 64 == 0 for int8).
 * antiquant_scale / antiquant_offset: [K/group, N] (group_size > 0) or [N]
 * (group_size == 0, per channel), of scale_dtype (fp16/bf16); offset may be NULL.
 * bias: [N] or NULL.  out: [M,N] of out_dtype (fp16/bf16).
 * out = sum_k x[m,k] * (w[k,n] + offset[g,n]) * scale[g,n] + bias[n], g = k/group,
 * with fp32 accumulation; the dequantized weight is never rounded to 16 bits.
 * The pointers need no more than their element's alignment; x, weight (NZ and
 * [N, K]), antiquant_scale, antiquant_offset and out that are not 16-byte
 * aligned may run a general kernel, at a fraction of the speed (the torch op
 * copies such operands first).
 */
int qk_weight_quant_bmm(const void* x, int x_dtype,
                        const void* weight, int weight_dtype,
                        const void* antiquant_scale, const void* antiquant_offset, int scale_dtype,
                        int64_t M, int64_t N, int64_t K, int64_t group_size,
                        const void* bias, int bias_dtype,
                        void* out, int out_dtype,
                        void* workspace, size_t workspace_bytes, qk_stream_t stream);

/* Bytes of the library-held scratch that qk_weight_quant_bmm_noalloc uses on each GPU. */
#define QK_NOALLOC_SCRATCH_BYTES (16 << 20)

/*
 * npu_weight_quant_batchmatmul without a workspace argument.  No counterpart
 * in the reference (whose calls always take caller-allocated scratch): this
 * entry point is for callers that cannot allocate device memory -- code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc.
 * Arguments and results are those of qk_weight_quant_bmm; the scratch the
 * call needs (split-K partials, group sums) lives in a library-owned device
 * array of QK_NOALLOC_SCRATCH_BYTES per GPU, held until the process ends, and
 * the call allocates nothing.  Where the workspace qk_weight_quant_bmm_workspace_size
 * reports fits in that array, the call runs exactly the kernels qk_weight_quant_bmm
 * runs (the same bits).  Where only the NZ prefill kernel's stream-K partial
 * slots do not fit, it runs that kernel with whole tiles per workgroup (the
 * same bits again); where the mid-M kernel's K splits do not fit, the kernels
 * without it (within 1e-2).  Otherwise, for a row-major int4 weight at M >= 17
 * or int8 weight at M >= 33 whose cast to NZ is what does not fit, it runs the
 * row-major kernels without the cast (within the same 1e-2 bar; for int4 on
 * cfg3's shape, N = 11008, K = 4096, 128-row groups, at M = 1024 and 2048 the
 * same bits); a shape whose scratch exceeds
 * QK_NOALLOC_SCRATCH_BYTES even so is refused with QK_ERR_UNSUPPORTED.  The call uses the array of the current device, so
 * `stream` must belong to it.  All calls on one GPU share that array: calls
 * that may run at the same time on one GPU (several streams or threads) race
 * on it and give wrong results, so serialise them (e.g. one stream).
 */
int qk_weight_quant_bmm_noalloc(const void* x, int x_dtype,
                                const void* weight, int weight_dtype,
                                const void* antiquant_scale, const void* antiquant_offset, int scale_dtype,
                                int64_t M, int64_t N, int64_t K, int64_t group_size,
                                const void* bias, int bias_dtype,
                                void* out, int out_dtype, qk_stream_t stream);

/*
 * npu_format_cast for a matmul weight -- the MI355X counterpart of the
 * FRACTAL_NZ casts the reference applies to matmul operands
 * (op_plugin/ops/base_ops/aclops/MmKernelNpu.cpp:303-316,
 * op_plugin/ops/base_ops/aclops/LinearKernelNpu.cpp:103-107), done once when
 * weights are loaded.  src_format -> dst_format is QK_FORMAT_ND ->
 * QK_FORMAT_FRACTAL_NZ or back; N % 16 == 0; src and dst must not overlap and
 * must be 16-byte aligned.
 * weight_dtype QK_I32 (int4 packed, [K, N/8] in ND; K % 128 == 0): NZ is int32
 * [N/16][K/128][64][4]; element (k, n) is in word
 *   ((n/16 * (K/128) + k/128) * 64 + lane) * 4 + j,
 *   c = (k%128)/8, lane = n%16 + 16*(c%4), j = c/4,
 * at nibble i/2 for even i = k%8 and 4 + i/2 for odd i (two's complement).
 * weight_dtype QK_I8 ([K, N] in ND; K % 64 == 0): NZ is int8 [N/16][K/64][64][16];
 * element (k, n) is byte ((n/16 * (K/64) + k/64) * 64 + n%16 + 16*((k%64)/16)) * 16 + k%16.
 * Either way a 1 KB block (16 columns) is read by a wave as one 16-byte load
 * per lane, each lane's bytes being its MFMA B operands.  No workspace.
 */
int qk_weight_format_cast(const void* src, int src_format, void* dst, int dst_format, int weight_dtype,
                          int64_t K, int64_t N, qk_stream_t stream);

/*
 * npu_convert_weight_to_int4pack -- packs int4 values held one per element
 * (int8 or int32 [K,N], values in [-8,7]) into int32 [K, N/8] in the layout
 * qk_weight_quant_bmm reads.  No counterpart exists in the reference snapshot
 * (int4 is disabled there: op_plugin/third_party/acl/inc/graph/types.h:57).
 */
int qk_int4_pack(const void* w, int w_dtype, int64_t K, int64_t N, int32_t* packed,
                 qk_stream_t stream);

/*
 * quantize_per_tensor -- replaces the CANN Quantize call of
 * op_plugin/ops/base_ops/aclops/QuantizePerTensorKernelNpu.cpp:50-82 (schema
 * op_plugin/config/v2r2/op_plugin_functions.yaml:1233).  x: n elements,
 * fp32/fp16/bf16.  q: n elements of q_dtype QK_I8 (qint8), QK_U8 (quint8) or
 * QK_I32 (qint32), the plain integer tensor the reference returns (dtype map
 * :60-67).  Per element: q = clamp(RN(rint(x * RN(1/scale)) + float(zero_point)),
 * qmin, qmax), ties to even, the zero point added in float32 (torch's affine
 * quantizer); NaN gives qmin.  scale must be a positive finite float.
 */
int qk_quantize_per_tensor(const void* x, int x_dtype, int64_t n, float scale, int64_t zero_point, void* q,
                           int q_dtype, qk_stream_t stream);

/*
 * quantize_per_channel -- replaces the CANN Quantize call of
 * op_plugin/ops/base_ops/aclops/QuantizePerChannelKernelNpu.cpp:69-92 (schema
 * op_plugin/config/v2r2/op_plugin_functions.yaml:1231).  x is viewed as
 * [outer][C][inner] with C the quantized axis; scales: fp32 [C] (device);
 * zero_points: int64 [C] (device).  Element rule as qk_quantize_per_tensor with
 * the channel's scale and zero point.
 */
int qk_quantize_per_channel(const void* x, int x_dtype, int64_t outer, int64_t C, int64_t inner, const float* scales,
                            const int64_t* zero_points, void* q, int q_dtype, qk_stream_t stream);

/*
 * dequantize -- the reference's op_plugin/ops/v1r11/opapi/DequantizeKernelNpuOpApi.cpp:22-24
 * (schema op_plugin/config/v1r11/op_plugin_functions.yaml:127): the integers of
 * q (QK_I8, QK_U8 or QK_I32, n elements) cast to float32 (round to nearest even
 * past 2^24).
 */
int qk_dequantize(const void* q, int q_dtype, int64_t n, float* out, qk_stream_t stream);

/*
 * npu_rms_norm -- replaces aclnnRmsNorm behind EXEC_NPU_CMD
 * (op_plugin/ops/base_ops/opapi/RmsNormKernelOpApi.cpp:24-35: y has the dtype
 * of x, :31; rstd is fp32, :32; schema op_plugin/config/v2r2/op_plugin_functions.yaml:2047).
 * x: [rows, D] fp16/bf16/fp32 (fp32 is the reference's golden case).  gamma:
 * [D], same dtype.  y: [rows, D], x's dtype.
 * rstd: [rows] fp32 or NULL.  rstd = 1/sqrt(mean(x^2) + eps); y = x * rstd * gamma
 * (golden test/test_custom_ops/test_npu_rms_norm.py:10-17), fp32 arithmetic.
 */
int qk_rms_norm(const void* x, int x_dtype, const void* gamma, int64_t rows, int64_t D, float eps,
                void* y, float* rstd, qk_stream_t stream);

/*
 * RMSNorm followed by npu_dynamic_quant of its 16-bit output, in one pass
 * (the first two steps of the quantized MLP block).  No single reference op:
 * the unfused chain is qk_rms_norm then qk_dynamic_quant, and q / scale are
 * bit-identical to it.  x: fp16/bf16 only (npu_dynamic_quant takes no fp32).
 * q: [rows, D] int8.  scale: [rows] fp32.  rstd as above.
 */
int qk_rms_norm_quant(const void* x, int x_dtype, const void* gamma, int64_t rows, int64_t D, float eps,
                      int8_t* q, float* scale, float* rstd, qk_stream_t stream);

/*
 * npu_swiglu (dim = -1) -- silu(a) * b with a, b = h.chunk(2, -1), the first
 * half the gate; the gated halving follows npu_geglu
 * (op_plugin/ops/v1r11/opapi/GeGluKernelNpuOpApi.cpp:23-40), silu follows
 * op_plugin/ops/base_ops/opapi/SiluKernelNpuOpApi.cpp:22-43.
 * h: [rows, 2*I] fp16/bf16.  y: [rows, I], same dtype.  fp32 arithmetic.
 */
int qk_swiglu(const void* h, int dtype, int64_t rows, int64_t I, void* y, qk_stream_t stream);

/*
 * SwiGLU followed by npu_dynamic_quant of its 16-bit output, in one pass (the
 * activation step of the quantized MLP block); bit-identical to qk_swiglu then
 * qk_dynamic_quant.  q: [rows, I] int8.  scale: [rows] fp32.
 */
int qk_swiglu_quant(const void* h, int dtype, int64_t rows, int64_t I, int8_t* q, float* scale,
                    qk_stream_t stream);

/*
 * The quantized MLP block's gate-up projection with the SwiGLU fused into the
 * GEMM's epilogue.  No single reference op: the unfused chain is
 * qk_quant_matmul (x1 [M,K] int8 x x2 [K,2I] int8, per-channel or per-tensor
 * scale of 2I or 1 elements, optional pertoken_scale [M], no bias, 16-bit
 * output) then qk_swiglu, and h [M, I] (out_dtype QK_BF16 or QK_F16, rows of
 * I elements) is bit-identical to it: the gate and up outputs are rounded to
 * out_dtype as the GEMM rounds them, and silu(gate) * up as qk_swiglu rounds
 * it.  Quantizing h with qk_dynamic_quant gives qk_swiglu_quant's q and scale.
 * x2: x2_format QK_FORMAT_FRACTAL_NZ (the NZ blocks npu_format_cast writes) or
 * QK_FORMAT_ND ([K, 2I] rows of x2_stride_k >= 2I bytes).  Runs where
 * I % 128 == 0, K % 256 == 0, ldx1 % 16 == 0 (< 2^24), x1 / x2 / out 16-byte
 * aligned and every offset fits 32 bits; other requests return
 * QK_ERR_UNSUPPORTED (the caller composes the two calls instead).  No
 * workspace.
 */
int qk_quant_matmul_swiglu(const int8_t* x1, int64_t ldx1, const int8_t* x2, int x2_format, int64_t x2_stride_k,
                           int64_t M, int64_t I, int64_t K, const float* scale, int64_t scale_len,
                           const float* pertoken_scale, void* out, int out_dtype, qk_stream_t stream);

/*
 * The same projection followed by qk_dynamic_quant of h, as the quantized MLP
 * block uses it: q [M, I] int8 (rows of I bytes, 8-byte aligned) and q_scale
 * [M] fp32 equal qk_dynamic_quant(h) bit for bit, h [M, I] being
 * qk_quant_matmul_swiglu's output rounded to h_dtype (QK_BF16 / QK_F16).  h
 * lives in the workspace, and the GEMM's epilogue also stores each row's
 * largest |h| per 128-column slice there, so the quantizer needs no row
 * reduction.  No single reference op: the chain npu_quant_matmul ->
 * npu_swiglu -> npu_dynamic_quant.  Workspace: the bytes
 * qk_quant_matmul_swiglu_quant_workspace_size gives (h plus M * I / 128
 * floats), 256-byte aligned, any contents.  The shapes
 * qk_quant_matmul_swiglu takes (I % 128 == 0, K % 256 == 0, ...); others
 * return QK_ERR_UNSUPPORTED (the caller composes the calls).
 */
int qk_quant_matmul_swiglu_quant_workspace_size(int64_t M, int64_t I, size_t* bytes);
int qk_quant_matmul_swiglu_quant(const int8_t* x1, int64_t ldx1, const int8_t* x2, int x2_format,
                                 int64_t x2_stride_k, int64_t M, int64_t I, int64_t K, const float* scale,
                                 int64_t scale_len, const float* pertoken_scale, int h_dtype, int8_t* q,
                                 float* q_scale, void* workspace, size_t workspace_bytes, qk_stream_t stream);

/* ------------------------------------------------------------------ attention over a key-value cache
 *
 * The other half of a decoder layer in serving: rotary positions, a key-value
 * cache in pages, attention over it.  The reference reaches fused attention
 * through npu_prompt_flash_attention and npu_incre_flash_attention
 * (op_plugin/ops/v2r2/opapi/FlashAttentionKernelNpuOpApi.cpp:361-408); the ops
 * below keep its two phases (prompt, one token) and add the page table.
 *
 * Indexes (page tables, lengths, slots, positions, counts) are int32 on the
 * device.  They are checked where they are used: an index outside its array is
 * never followed, with the effect stated at each function.
 */

/* Keys and values of one layer.  key / value: [num_pages][page_size][kv_heads][head_dim] elements of `dtype`
 * (QK_F16, QK_BF16 or QK_I8), read through strides in elements (head_dim contiguous): any order of the axes.  Rows of
 * a head start at multiples of 16 bytes.  QK_I8 holds round(x / scale): key_scale / value_scale, fp32
 * [num_pages][page_size][kv_heads] through strides of their own, one scale per token and head, as npu_dynamic_quant
 * gives them.  head_dim: a multiple of 8 (QK_I8: of 16), at most 256.  Where a function takes contiguous keys
 * [tokens][kv_heads][head_dim], they are one page: num_pages = 1, page_size = tokens. */
typedef struct qk_kv_cache {
    void* key;
    void* value;
    float* key_scale;
    float* value_scale;
    int64_t num_pages, page_size, kv_heads, head_dim;
    int64_t key_page_stride, key_token_stride, key_head_stride;
    int64_t value_page_stride, value_token_stride, value_head_stride;
    int64_t key_scale_page_stride, key_scale_token_stride, key_scale_head_stride;
    int64_t value_scale_page_stride, value_scale_token_stride, value_scale_head_stride;
    int dtype;
} qk_kv_cache;

/*
 * npu_paged_attention -- attention of one new token per sequence over its pages (the op of one token,
 * npu_incre_flash_attention, op_plugin/ops/v2r2/opapi/FlashAttentionKernelNpuOpApi.cpp:385-408; golden
 * test/test_custom_ops/test_incre_flash_attention.py:15-23).  query: [batch][q_heads][head_dim] of dtype (QK_F16 /
 * QK_BF16; a 16-bit cache has the same), through strides in elements (multiples of 8).  q_heads is a multiple of
 * cache->kv_heads: head h reads key-value head h / (q_heads / kv_heads).  Sequence b holds context_lens[b] tokens, the
 * newest included, token j in slot j % page_size of page block_table[b * table_stride + j / page_size].  The query
 * stands at the last of them, p, and sees the keys j <= p with p - j < window (window 0: all) or j < sinks.
 *   s_j = scale * q . k_j,  out = sum exp(s_j - m) v_j / sum exp(s_j - m),  lse = m + ln sum exp(s_j - m)
 * in fp32, m the largest s_j, scale finite and at most 2.3e38; out: [batch][q_heads][head_dim] of dtype, lse:
 * [batch][q_heads] fp32 or NULL.  A sequence without a visible key (length 0) gives out = 0 and lse = -inf.  Lengths are
 * cut to table_width * page_size; a token whose page id is outside [0, num_pages) is not seen.  Workspace: partial
 * results where the keys of a sequence are split over workgroups.
 */
int qk_paged_attention_workspace_size(int64_t batch, int64_t q_heads, const qk_kv_cache* cache, int64_t table_width,
                                      int64_t window, int64_t sinks, size_t* bytes);
int qk_paged_attention(const void* query, int dtype, int64_t batch, int64_t q_heads, int64_t q_token_stride,
                       int64_t q_head_stride, const qk_kv_cache* cache, const int32_t* block_table,
                       int64_t table_width, int64_t table_stride, const int32_t* context_lens, float scale,
                       int64_t window, int64_t sinks, void* out, float* lse, void* workspace, size_t workspace_bytes,
                       qk_stream_t stream);

/*
 * npu_prompt_attention -- causal attention of ragged prompts or prompt chunks (the op of whole prompts,
 * npu_prompt_flash_attention, op_plugin/ops/v2r2/opapi/FlashAttentionKernelNpuOpApi.cpp:361-383; golden
 * test/test_custom_ops/test_prompt_flash_attention.py:15-21).  query: [tokens][q_heads][head_dim]; sequence b's rows
 * are cu_seqlens_q[b] .. cu_seqlens_q[b + 1] (batch + 1 values, the first 0, none falling).  Its keys: with
 * block_table, kv_lens[b] tokens in pages, as above; without (NULL, cache->num_pages 1), rows cu_seqlens_k[b] ..
 * cu_seqlens_k[b + 1] of the contiguous keys.  Query i of n, of a sequence with m keys, stands at p = m - n + i and sees
 * the keys j <= p with p - j < window (window 0: all) or j < sinks.  Same formula, outputs and rules as
 * qk_paged_attention; a row that sees no key, and a row past the last sequence, gives out = 0 and lse = -inf.
 */
int qk_prompt_attention_workspace_size(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache* cache,
                                       int64_t table_width, int64_t window, int64_t sinks, size_t* bytes);
int qk_prompt_attention(const void* query, int dtype, int64_t tokens, int64_t batch, int64_t q_heads,
                        int64_t q_token_stride, int64_t q_head_stride, const int32_t* cu_seqlens_q,
                        const qk_kv_cache* cache, const int32_t* cu_seqlens_k, const int32_t* block_table,
                        int64_t table_width, int64_t table_stride, const int32_t* kv_lens, float scale, int64_t window,
                        int64_t sinks, void* out, float* lse, void* workspace, size_t workspace_bytes,
                        qk_stream_t stream);

/*
 * npu_tree_attention -- attention of drafted tokens, a tree of them per sequence, over its pages (decoding with drafts: a
 * third phase between the two of the reference's fused attention, several rows of which no two need see each other).
 * query: [tokens][q_heads][head_dim], sequence b's rows cu_seqlens_q[b] .. cu_seqlens_q[b + 1] as above.  Sequence b holds
 * context_lens[b] tokens in pages, the last n of them the rows' own, n being their number; before them x =
 * context_lens[b] - n.  Row t sees the keys j < x, and key x + k for every k < n whose bit, k % 64 of
 * tree_mask[t * mask_stride + k / 64], is set (itself only if its own bit is; past mask_words words there are none).  With
 * a window it sees of the keys j < x those with p - j < window or j < sinks, p = x - 1 + the number of its bits set below n, so that
 * a row whose bits are its ancestors and itself stands at its depth; the tree's own keys go by the mask alone.  Same formula, outputs and
 * rules as qk_paged_attention; a row that sees no key, and a row past the last sequence, gives out = 0 and lse = -inf.
 */
int qk_tree_attention_workspace_size(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache* cache,
                                     int64_t table_width, int64_t window, int64_t sinks, size_t* bytes);
int qk_tree_attention(const void* query, int dtype, int64_t tokens, int64_t batch, int64_t q_heads, int64_t q_token_stride,
                      int64_t q_head_stride, const int32_t* cu_seqlens_q, const qk_kv_cache* cache,
                      const int32_t* block_table, int64_t table_width, int64_t table_stride, const int32_t* context_lens,
                      const int64_t* tree_mask, int64_t mask_words, int64_t mask_stride, float scale, int64_t window,
                      int64_t sinks, void* out, float* lse, void* workspace, size_t workspace_bytes, qk_stream_t stream);

/*
 * npu_mrope, npu_mrope_scatter_kv -- rotary positions of one to four axes (time, height, width of an image's or a
 * video's tokens), alone or with the write of the new keys and values into the cache.  query: [tokens][q_heads]
 * [head_dim], key, value: [tokens][kv_heads][head_dim] of dtype (QK_F16 / QK_BF16) through strides in elements.
 * positions: axes rows of `tokens` int32, position_stride apart.  cos_sin: [table_rows][rotary_dim] fp32 or of dtype,
 * each row rotary_dim / 2 cosines, then as many sines; rotary_dim even, at most head_dim.  Pair i < rotary_dim / 2
 * takes its row at positions[a][t], a being the section that i lies in (sections[axes], summing to rotary_dim / 2).
 * interleave 0: pair (x_i, x_{i + rotary_dim/2}); 1: (x_2i, x_2i+1).
 *   y0 = x0 * cos - x1 * sin,  y1 = x1 * cos + x0 * sin  (fp32, each product rounded; one rounding to dtype)
 * Dimensions past rotary_dim are copied.  A position outside the table makes its pairs NaN.  out_query, out_key
 * (contiguous, either may be NULL).  With cache: token t's rotated key and its value (NULL: not written) go to slot
 * slots[t] = page * page_size + token; a slot outside the cache (a padding token's -1) is not written.  An int8 cache takes
 * each 16-bit row through npu_dynamic_quant: scale = absmax / 127, the values rint(y / scale).  No workspace.
 */
int qk_mrope(const void* query, const void* key, const void* value, int dtype, int64_t tokens, int64_t q_heads,
             int64_t kv_heads, int64_t head_dim, int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
             int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, const int32_t* positions,
             int64_t axes, int64_t position_stride, const int64_t* sections, const void* cos_sin, int cos_sin_dtype,
             int64_t table_rows, int64_t rotary_dim, int interleave, void* out_query, void* out_key,
             const qk_kv_cache* cache, const int32_t* slots, qk_stream_t stream);

/* ------------------------------------------------------------------ pages of a cache
 *
 * State of a pool: block_table [max_seqs][table_width] (rows table_stride apart, -1 past a sequence's pages),
 * context_lens [max_seqs], ref_count [num_pages], the number of sequences that hold a page.  A page with count 0 is free,
 * and a page is allocated from the lowest free one upwards: no free list is kept, and the same calls give the same
 * pages.  A cache tensor is described by qk_pages: page p's page_bytes bytes begin at base + p * page_stride.
 * Sequence numbers outside [0, max_seqs) are passed over.  At most QK_MAX_SEQS sequences a call.
 */
typedef struct qk_pages {
    void* base;
    int64_t page_stride; /* bytes */
    int64_t page_bytes;
} qk_pages;
#define QK_MAX_SEQS 65536

/* npu_kv_copy_pages: for every i < n, page src[i] to page dst[i], in each of the tensors; a pair with an id outside
 * [0, num_pages) is passed over.  No page may be the destination of two pairs, or of one and the source of another. */
int qk_kv_copy_pages(const qk_pages* pages, int64_t tensors, int64_t num_pages, const int32_t* src,
                     const int32_t* dst, int64_t n, qk_stream_t stream);

/* npu_kv_fork: sequence children[i] becomes a copy of parents[i].  Whole pages are shared (count + 1); a last page that
 * is not full goes to a new page (count 1), whose bytes are copied in each of the tensors, so no writable page is
 * shared.  A child's former pages are not released (qk_kv_free does that before); no child may be a parent or occur
 * twice.  missing[0] = how many free pages are missing: 0, or nothing but missing[0] is written.  Workspace: see the
 * query. */
int qk_kv_fork_workspace_size(int64_t n, size_t* bytes);
int qk_kv_fork(const qk_pages* pages, int64_t tensors, int64_t num_pages, int64_t page_size, int32_t* block_table,
               int64_t max_seqs, int64_t table_width, int64_t table_stride, int32_t* context_lens, int32_t* ref_count,
               const int32_t* parents, const int32_t* children, int64_t n, int32_t* missing, void* workspace,
               size_t workspace_bytes, qk_stream_t stream);

/* npu_kv_free: the pages of sequences seqs[i] lose a count, their table rows become -1, their lengths 0.  A sequence
 * named twice is freed once. */
int qk_kv_free(int64_t num_pages, int64_t page_size, int32_t* block_table, int64_t max_seqs, int64_t table_width,
               int64_t table_stride, int32_t* context_lens, int32_t* ref_count, const int32_t* seqs, int64_t n,
               qk_stream_t stream);

/* npu_kv_extend: sequence seqs[i] (none twice) grows by cu_tokens[i + 1] - cu_tokens[i] tokens.  Pages are allocated in
 * the order of i; slots[t] and positions[t], t < total, are the cache slot and the position of each new token (-1
 * past cu_tokens[n], and for a sequence number that is passed over).  missing[0] = how many free pages, or table columns,
 * are missing (at most 2^31 - 1): 0, or slots and positions are -1 and nothing else is written.  Workspace: see the query. */
int qk_kv_extend_workspace_size(int64_t n, int64_t num_pages, size_t* bytes);
int qk_kv_extend(int64_t num_pages, int64_t page_size, int32_t* block_table, int64_t max_seqs, int64_t table_width,
                 int64_t table_stride, int32_t* context_lens, int32_t* ref_count, const int32_t* seqs,
                 const int32_t* cu_tokens, int64_t n, int64_t total, int32_t* slots, int32_t* positions,
                 int32_t* missing, void* workspace, size_t workspace_bytes, qk_stream_t stream);

/* npu_kv_compact: with L pages in use (count > 0), the k-th page in use of number >= L is copied to the k-th free page of
 * number < L, in each of the tensors.  new_table [max_seqs][table_width] (contiguous) and new_count [num_pages] are the
 * table and the counts with the pages at their new places; the old ones, and the pages moved from, stay as they were.
 * moved[0] = how many pages moved.  Workspace: see the query. */
int qk_kv_compact_workspace_size(int64_t num_pages, size_t* bytes);
int qk_kv_compact(const qk_pages* pages, int64_t tensors, int64_t num_pages, const int32_t* block_table,
                  int64_t max_seqs, int64_t table_width, int64_t table_stride, const int32_t* ref_count,
                  int32_t* new_table, int32_t* new_count, int32_t* moved, void* workspace, size_t workspace_bytes,
                  qk_stream_t stream);

/* npu_kv_accept: the end of a step of decoding with drafts.  Sequence seqs[i] (none twice) ends in the tokens of a tree, rows
 * first = cu_tokens[i] .. cu_tokens[i + 1] of tokens, parents and sampled: n of them, as qk_kv_extend placed them, behind
 * x = context_lens[seq] - n others.  Row 0 is the root, the token drawn last; the others are drafted, parents[first + k] < k
 * being the row of the tree that row k follows (rows without such a parent are reached by none).  sampled[first + k] is the
 * token that was drawn at row k.  From the root the way goes to the lowest of a row's children whose token (not negative) is the one
 * drawn at the row, until there is none: kept rows 0 = r_0 < r_1 < ... < r_{a-1}.  path[first + j] = first + r_j for j < a, -1
 * behind; accepted[i] = a (at least 1); next[i] = sampled[first + r_{a-1}], the token that the next tree begins with.
 * In every tensor the cache's row of token x + r_j moves to x + j (a page id outside [0, num_pages) is not followed); then
 * context_lens[seq] = x + a, and the pages behind it lose a count and their table entries become -1.  The tree's pages
 * must not be shared.  A sequence number outside [0, max_seqs), an empty tree, and one larger than the sequence are passed over:
 * accepted 0, next and path -1.  path [total], accepted and next [n].
 * A cache tensor is described by qk_rows: the row of the token at place s of page p is `pieces` pieces of piece_bytes bytes,
 * piece_stride apart, from base + p * page_stride + s * token_stride on (all in bytes); no two tensors share bytes.  Workspace: see the query. */
typedef struct qk_rows {
    void* base;
    int64_t page_stride, token_stride, piece_stride;
    int64_t pieces, piece_bytes;
} qk_rows;
int qk_kv_accept_workspace_size(int64_t n, size_t* bytes);
int qk_kv_accept(const qk_rows* rows, int64_t tensors, int64_t num_pages, int64_t page_size, int32_t* block_table,
                 int64_t max_seqs, int64_t table_width, int64_t table_stride, int32_t* context_lens, int32_t* ref_count,
                 const int32_t* seqs, const int32_t* cu_tokens, int64_t n, int64_t total, const int32_t* tokens,
                 const int32_t* parents, const int32_t* sampled, int32_t* path, int32_t* accepted, int32_t* next,
                 void* workspace, size_t workspace_bytes, qk_stream_t stream);

/* ------------------------------------------------------------------ a token per row of logits
 *
 * npu_sample -- temperature, top-k, top-p and min-p, and a draw from a given uniform number (the reference leaves sampling
 * to the framework's own sort, cumsum and multinomial).  logits: [rows][vocab] QK_F16, QK_BF16 or QK_F32, rows row_stride
 * elements apart, vocab 1 .. QK_MAX_VOCAB, rows up to QK_MAX_SAMPLE_ROWS.  The others are [rows] on the device; all but uniform may be NULL.
 *   w_i = exp((x_i - max x) / temperature[r])       (NULL: 1)
 * The row's tokens in order of x, falling, ties by index.  top_k[r] > 0 keeps the first so many.  top_p[r] < 1 keeps of
 * those the ones before which less than top_p of their sum of w lies.  min_p[r] > 0 keeps those with w_i >= min_p (above 1:
 * as 1).  The first is always kept.  S = the sum of the kept w; tokens[r] is the lowest kept i at which the kept w up to and
 * including i sum to more than uniform[r] * S (uniform cut to [0, 1)), logprobs[r] = ln(w_i / S).  A temperature that is
 * not above 0 takes the first, logprob 0.  A logit -inf or NaN is never drawn; a row without another gives token -1, logprob
 * -inf.  Among infinite logits all weight is theirs, in equal parts.  Weights are multiples of 2^-F of the largest, F = 62 -
 * ceil(log2 vocab), at most 50, and sums of them exact: the result does not depend on how the work is split.
 */
#define QK_MAX_VOCAB (1 << 24)
#define QK_MAX_SAMPLE_ROWS ((1 << 22) - 1)
int qk_sample_workspace_size(int64_t rows, int64_t vocab, int dtype, size_t* bytes);
int qk_sample(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, const float* uniform,
              const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
              float* logprobs, void* workspace, size_t workspace_bytes, qk_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* QK_ABI_H */
