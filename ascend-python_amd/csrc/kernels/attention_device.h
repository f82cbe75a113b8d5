// Device code shared by the attention kernels: operands of the 16-bit matrix instructions and where a token's rows lie.
#pragma once

#include "attention.h"

namespace qk {

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
// The running maximum (of scores times log2 e) before any key: finite, so that no difference with it is NaN.
constexpr float kLowest = -3.0e38f;
// A running maximum stays until a score passes it by this much: weights reach 2^8, which neither 16-bit type nor the fp32
// sums mind, and most tiles rescale nothing.
constexpr float kSlack = 8.0f;
// Weights are rounded once to 16 bits, half a step each: the second product's matrix instruction takes operands of one 16-bit
// type, and a second one for what the rounding leaves would be half as much matrix work again, for an error of the size that
// V's own 16 bits have.  bf16 keeps its relative step whatever the weight; float16 (DT: the weights' type) loses bits below
// 2^-14 and everything below 2^-25, while the weights' fp32 sum does not, and 100000 small weights can be a share of the
// result that shows.  So the running "maximum" lies 7 below the largest score there: weights reach 2^(7 + 8), still finite,
// keep all their bits down to 2^-21 of the largest, and are rounded to multiples of 2^-31 of it below that.
template <int DT>
constexpr float kBelow = DT == QK_F16 ? 7.0f : 0.0f;

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int16_t i16x4 __attribute__((ext_vector_type(4)));

// Two fp32 values as 16-bit ones, each rounded to nearest.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == QK_BF16) return __builtin_bit_cast(uint32_t, (bf16x2){(__bf16)a, (__bf16)b});
    else return __builtin_bit_cast(uint32_t, (f16x2){(_Float16)a, (_Float16)b});
}

// A read of LDS that transposes: in a group of 16 lanes, lanes 4r .. 4r + 3 address the 16 elements of row r (8 bytes each),
// and lane i gets column i of the four rows.
__device__ __forceinline__ u32x2 lds_tr16(const void* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) i16x4*)(uintptr_t)(uint32_t)(uintptr_t)p));
}

// Eight int8 as fp16: x + 128 in the low byte of 0x6400 is the number 1152 + x, exactly; 1152 is taken off in fp16, exactly.
__device__ __forceinline__ u32x4 i8_to_f16(uint32_t lo, uint32_t hi) {
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    const f16x2 base = {(_Float16)1152.0f, (_Float16)1152.0f};
    u32x4 r;
    const uint32_t w[2] = {lo, hi};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t m = __builtin_amdgcn_perm(0x64646464u, w[i >> 1], i & 1 ? 0x04030402u : 0x04010400u);
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, m) - base);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ u32x4 i8_to_half(uint32_t lo, uint32_t hi) {
    if constexpr (DT == QK_F16) return i8_to_f16(lo, hi);
    else return i8_operand<QK_BF16>(lo, hi);
}

// What a row of the cache that is not seen reads instead: zeros.
__device__ const uint32_t kZeroRow[256] __attribute__((aligned(16))) = {};

// An address known to lie in global memory, so that loads through a choice of such addresses do not take the flat path.
typedef const __attribute__((address_space(1))) char* Global;
__device__ __forceinline__ Global global_address(const void* p) { return (Global)(uintptr_t)p; }
template <typename T>
__device__ __forceinline__ T load_global(Global p) {
    return *(const __attribute__((address_space(1))) T*)p;
}

// Largest value, and sum, over the four lanes that share lane & 15.
__device__ __forceinline__ float quad_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (uint64_t)hi << 32 | lo;
}

// Sum over the lanes up to this one, by moves within rows of 16 lanes and from a row's last lane to those behind.
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);
    return v;
}

// Work along a line of `total` units, of which each of `workers` takes an equal part.
// n / d for n >= 0, d > 0: by 32 bits where they fit, as they all but always do
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
    return (uint64_t)(n | d) >> 32 ? n / d : (int64_t)((uint32_t)n / (uint32_t)d);
}
__device__ __forceinline__ int64_t line_begin(int64_t total, int64_t workers, int64_t i) { return quotient(total * i, workers); }
// The worker whose part holds unit u
__device__ __forceinline__ int64_t worker_of(int64_t total, int64_t workers, int64_t u) {
    return quotient((u + 1) * workers + total - 1, total) - 1;
}

// Rows of tokens and keys of sequence b (b == batch: the rows past the last sequence, which see nothing)
struct Sequence {
    int32_t first, tokens;
};
__device__ __forceinline__ Sequence sequence_of(const AttnArgs& a, int64_t b) {
    const int32_t T = (int32_t)a.tokens;
    int32_t first = b == 0 ? 0 : a.cu_q[b], end = b == a.batch ? T : a.cu_q[b + 1];
    first = first < 0 ? 0 : first > T ? T : first;
    end = end > T ? T : end;
    return {first, end > first ? end - first : 0};
}

template <int DT>
__device__ __forceinline__ constexpr uint32_t exponent_of() {
    return DT == QK_BF16 ? 0x7f80u : 0x7c00u;
}
template <int DT>
__device__ __forceinline__ bool not_finite(u32x4 w) {
    constexpr uint32_t E = exponent_of<DT>(), H = E << 16;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (w[i] & E) == E || (w[i] & H) == H;
    return any;
}
// The finite values, and zero for the others.
template <int DT>
__device__ __forceinline__ u32x4 finite_only(u32x4 w) {
    constexpr uint32_t E = exponent_of<DT>(), H = E << 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= ((w[i] & E) == E ? 0u : 0xffffu) | ((w[i] & H) == H ? 0u : 0xffff0000u);
    return w;
}

// Tokens of sequence b in the cache.
__device__ __forceinline__ int32_t cached_tokens(const AttnArgs& a, int64_t b) {
    const int64_t most = a.kv.table_width * a.kv.c.page_size, n = a.kv.lens[b];
    return (int32_t)(n < 0 ? 0 : n > most ? most : n);
}

// The keys that a position sees, without a gap: the first `sinks` of them, then those from `low` on.
struct Seen {
    int32_t count, sinks, gap;
};
__device__ __forceinline__ Seen seen_by(int32_t p, int32_t window, int32_t sinks) {
    Seen s = {p + 1, 0, 0};
    if (window && p - window + 1 > 0) {
        const int32_t low = p - window + 1;
        s.sinks = sinks < low ? sinks : low;
        s.gap = low - s.sinks;
        s.count = p + 1 - s.gap;
    }
    return s;
}

}  // namespace qk
