// Arguments of the attention and cache kernels (validated by the C ABI) and what their files share.
#pragma once

#include "common.h"

namespace qk {

// The thread's error message (qk_last_error): cleared where an entry point begins, set where it refuses.
void abi_begin();
int abi_error(int code, const char* message);

// q = j / d for 0 <= j < 2^31 and a divisor fixed per launch (a page's size), by multiplication (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994): (j * m) >> s with m = ceil(2^s / d),
// s = 31 + ceil(log2 d).  The error of m, below d, adds j * d / (d * 2^s) < 1 / d to the quotient, too little to reach the
// next whole number; m < 2^32 as d > 2^(s - 32).
struct Div31 {
    uint32_t m, s;
};
inline Div31 div31(uint32_t d) {
    uint32_t c = 0;
    while (((uint64_t)1 << c) < d) ++c;
    const uint32_t s = 31 + c;
    return {(uint32_t)((((uint64_t)1 << s) + d - 1) / d), s};
}
__device__ __forceinline__ int32_t div31(int32_t j, Div31 d) { return (int32_t)(((uint64_t)(uint32_t)j * d.m) >> d.s); }

// Keys, values and where a sequence's tokens lie.  table != nullptr: token j of sequence b is in slot j % page_size of
// page table[b * table_stride + j / page_size]; else row cu_k[b] + j of the only page.
struct KvArgs {
    qk_kv_cache c;
    const int32_t* table;
    int64_t table_width, table_stride;
    const int32_t* lens;  // [batch] with table
    const int32_t* cu_k;  // [batch + 1] without
    Div31 page_div;
};

struct AttnArgs {
    const void* q;
    int dtype;
    int64_t tokens;  // rows of q (decode: the batch)
    int64_t batch, q_heads;
    int64_t q_token_stride, q_head_stride;
    const int32_t* cu_q;  // nullptr: one row per sequence
    KvArgs kv;
    float scale;
    int32_t window, sinks;
    void* out;
    float* lse;
};

// One token per sequence (cu_q == nullptr), keys in pages.
size_t attention_decode_workspace(int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width, int64_t window,
                                  int64_t sinks);
hipError_t launch_attention_decode(const AttnArgs& a, void* workspace, hipStream_t stream);

// Ragged prompts (cu_q != nullptr).
size_t attention_prompt_workspace(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width,
                                  int64_t window, int64_t sinks);
hipError_t launch_attention_prompt(const AttnArgs& a, void* workspace, hipStream_t stream);

struct MropeArgs {
    const void *q, *k, *v;
    int dtype;
    int64_t tokens, q_heads, kv_heads, head_dim;
    int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    const int32_t* positions;
    int axes;
    int64_t position_stride;
    int32_t section_end[4];  // first pair past each axis's section
    const void* cos_sin;
    int cos_sin_dtype;
    int64_t table_rows, rotary_dim;
    int interleave;
    void *out_q, *out_k;
    bool cached;
    qk_kv_cache c;
    const int32_t* slots;
    Div31 page_div;
};
hipError_t launch_mrope(const MropeArgs& a, hipStream_t stream);

// The pool's state, as the page kernels take it.
struct PoolArgs {
    int64_t num_pages, page_size;
    int32_t* table;
    int64_t max_seqs, table_width, table_stride;
    int32_t* lens;
    int32_t* count;
};
hipError_t launch_kv_copy_pages(const qk_pages* pages, int64_t tensors, int64_t num_pages, const int32_t* src,
                                const int32_t* dst, int64_t n, hipStream_t stream);
hipError_t launch_kv_fork(const qk_pages* pages, int64_t tensors, const PoolArgs& p, const int32_t* parents,
                          const int32_t* children, int64_t n, int32_t* missing, void* ws, hipStream_t stream);
hipError_t launch_kv_free(const PoolArgs& p, const int32_t* seqs, int64_t n, hipStream_t stream);
hipError_t launch_kv_extend(const PoolArgs& p, const int32_t* seqs, const int32_t* cu, int64_t n, int64_t total,
                            int32_t* slots, int32_t* positions, int32_t* missing, void* ws, hipStream_t stream);
hipError_t launch_kv_compact(const qk_pages* pages, int64_t tensors, const PoolArgs& p, int32_t* new_table,
                             int32_t* new_count, int32_t* moved, void* ws, hipStream_t stream);
size_t kv_fork_workspace(int64_t n);
size_t kv_extend_workspace(int64_t n, int64_t num_pages);
size_t kv_compact_workspace(int64_t num_pages);

}  // namespace qk
