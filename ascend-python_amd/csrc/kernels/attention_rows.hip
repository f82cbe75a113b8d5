// Attention, the plainest kernel that takes every case: one wave per query row and head walks the keys that the row sees,
// one at a time, each lane holding every 64th element of the head, with the running maximum and sum of a softmax.
//   m' = max(m, s),  l = l * e^(m - m') + e^(s - m'),  acc = acc * e^(m - m') + e^(s - m') * v
// All in fp32, one rounding of acc / l at the end.  Bound by its instructions: some 40 per key and wave.
#include "attention_device.h"

namespace qk {
namespace {


constexpr int kPer = 4;  // elements per lane: head_dim <= 256

__device__ __forceinline__ float load_elem(const void* p, int64_t i, int dtype) {
    if (dtype == QK_I8) return (float)((const int8_t*)p)[i];
    return load_half_bits(((const uint16_t*)p)[i], dtype);
}

__global__ __launch_bounds__(256) void attention_rows(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= a.tokens * a.q_heads) return;
    const int64_t t = id / a.q_heads;
    const int h = (int)(id % a.q_heads);
    const qk_kv_cache& c = a.kv.c;
    const int g = (int)(h / (a.q_heads / c.kv_heads));
    const int D = (int)c.head_dim;

    // the sequence of this row, its keys and the row's position among them
    int64_t b = t, first = t, n_q = 1;
    if (a.cu_q) {
        int64_t lo = 0, hi = a.batch;  // the last b with cu_q[b] <= t
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (a.cu_q[mid] <= t) lo = mid;
            else hi = mid;
        }
        b = lo;
        first = b == 0 ? 0 : a.cu_q[b];
        n_q = a.cu_q[b + 1] - first;
    }
    int64_t keys = 0, start = 0;
    if (t < first + n_q) {
        if (a.kv.table) {
            keys = a.kv.lens[b];
            if (keys > a.kv.table_width * c.page_size) keys = a.kv.table_width * c.page_size;
        } else {
            start = b == 0 ? 0 : a.kv.cu_k[b];
            const int64_t end = a.kv.cu_k[b + 1] < c.page_size ? a.kv.cu_k[b + 1] : c.page_size;
            if (start < 0) start = 0;
            keys = end - start;
        }
    }
    const int64_t p = t < first + n_q ? keys - n_q + (t - first) : -1;  // rows past the last sequence see nothing

    float q[kPer], acc[kPer] = {};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = lane + 64 * i;
        q[i] = d < D ? load_elem(a.q, t * a.q_token_stride + h * a.q_head_stride + d, a.dtype) : 0.0f;
    }
    float m = -__builtin_inff(), l = 0.0f;
    bool any = false;
    int64_t j = 0;
    if (a.window && p - a.window + 1 > a.sinks && a.sinks == 0) j = p - a.window + 1;
    for (; j <= p; ++j) {
        if (a.window && p - j >= a.window && j >= a.sinks) {
            j = p - a.window;
            continue;
        }
        int64_t page = 0, slot = start + j;
        if (a.kv.table) {
            const int32_t at = div31((int32_t)j, a.kv.page_div);
            page = a.kv.table[b * a.kv.table_stride + at];
            slot = j - at * c.page_size;
            if (page < 0 || page >= c.num_pages) continue;
        }
        const int64_t kr = page * c.key_page_stride + slot * c.key_token_stride + g * c.key_head_stride;
        const int64_t vr = page * c.value_page_stride + slot * c.value_token_stride + g * c.value_head_stride;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (lane + 64 * i < D) s = __builtin_fmaf(q[i], load_elem(c.key, kr + lane + 64 * i, c.dtype), s);
        s = wave_sum(s) * a.scale;
        float vs = 1.0f;
        if (c.dtype == QK_I8) {
            s *= c.key_scale[page * c.key_scale_page_stride + slot * c.key_scale_token_stride + g * c.key_scale_head_stride];
            vs = c.value_scale[page * c.value_scale_page_stride + slot * c.value_scale_token_stride +
                               g * c.value_scale_head_stride];
        }
        any = true;
        const float m2 = fmaxf(m, s);
        const float base = m2 == -__builtin_inff() ? 0.0f : m2;
        const float keep = __builtin_amdgcn_exp2f((m - base) * kLog2e), w = __builtin_amdgcn_exp2f((s - base) * kLog2e);
        m = m2;
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (lane + 64 * i < D) acc[i] = acc[i] * keep + (w * vs) * load_elem(c.value, vr + lane + 64 * i, c.dtype);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int d = lane + 64 * i;
        if (d >= D) continue;
        const float o = any ? acc[i] / l : 0.0f;
        ((uint16_t*)a.out)[id * D + d] = (uint16_t)(a.dtype == QK_BF16 ? f32_to_bf16_bits(o) : f32_to_f16_bits(o));
    }
    if (a.lse && lane == 0) a.lse[id] = any ? m + __builtin_amdgcn_logf(l) * kLn2 : -__builtin_inff();
}

}  // namespace

hipError_t launch_attention_rows(const AttnArgs& a, hipStream_t stream) {
    const int64_t blocks = (a.tokens * a.q_heads + 3) / 4;
    attention_rows<<<dim3((unsigned)blocks), 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace qk
