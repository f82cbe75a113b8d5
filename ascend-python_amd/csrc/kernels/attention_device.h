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
