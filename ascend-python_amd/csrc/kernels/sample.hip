// A token per row of logits: w_i = e^((x_i - max) / temperature), the kept tokens a head of the row sorted by x (falling, then by
// index), and the first kept one, by index, at which the kept weights' sum passes uniform * their whole sum.
//
// Weights are whole numbers, multiples of 2^-F of the largest, in 64 bits: their sums are exact and do not depend on the order in
// which they are made, so the same call gives the same token however the work is split.  F = 62 - log2(vocab), at most 50: what is
// rounded away is below 2^-(F + 1) of the largest weight each.
//
// One workgroup per row: the largest logit, then the border of each filter found in the logits' bits, eleven at a time: a
// histogram of counts and weights, the bin in which the count or the sum passes the border, and on into that bin.
#include "sample.h"

namespace qk {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;

// Logits as whole numbers in their order; both zeros are one, NaN lies below -inf.
constexpr uint32_t kLeast = 0x00800000u;  // the lowest finite one: what lies below is never drawn
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return 0;
    if (u == 0x80000000u) return u;
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }

template <int DT>
__device__ __forceinline__ uint32_t load_key(const void* row, int64_t i) {
    if constexpr (DT == QK_F32) return key_of(((const float*)row)[i]);
    else return key_of(load_half_bits(((const uint16_t*)row)[i], DT));
}

// 2^t for -64 <= t <= 0: 2^n times the Taylor series of e^(f ln 2), |f| <= 1/2, whose terms past the 13th are below 2^-56.
__device__ __forceinline__ double pow2(double t) {
    const double n = __builtin_rint(t), z = (t - n) * 0.693147180559945309417;
    double p = 1.0 / 479001600.0;
    p = __builtin_fma(p, z, 1.0 / 39916800.0);
    p = __builtin_fma(p, z, 1.0 / 3628800.0);
    p = __builtin_fma(p, z, 1.0 / 362880.0);
    p = __builtin_fma(p, z, 1.0 / 40320.0);
    p = __builtin_fma(p, z, 1.0 / 5040.0);
    p = __builtin_fma(p, z, 1.0 / 720.0);
    p = __builtin_fma(p, z, 1.0 / 120.0);
    p = __builtin_fma(p, z, 1.0 / 24.0);
    p = __builtin_fma(p, z, 1.0 / 6.0);
    p = __builtin_fma(p, z, 0.5);
    p = __builtin_fma(p, z, 1.0);
    p = __builtin_fma(p, z, 1.0);
    return __builtin_ldexp(p, (int)n);
}

// Weights of a row whose largest logit is `top`.
struct Weights {
    double top, factor;  // log2 e / temperature
    double one;          // 2^F, the largest weight
    uint32_t top_key;

    // log2 of the weight
    __device__ __forceinline__ double log2_of(uint32_t key) const {
        if (key < kLeast) return -__builtin_inf();
        if (top == __builtin_inf()) return key == top_key ? 0.0 : -__builtin_inf();
        return ((double)value_of(key) - top) * factor;
    }
    __device__ __forceinline__ uint64_t of(uint32_t key) const {
        const double t = log2_of(key);
        if (!(t >= -60.0)) return 0;
        // rounded to a whole number by adding 2^52, in whose last bits it then stands
        return __builtin_bit_cast(uint64_t, pow2(t) * one + 0x1p52) & 0xfffffffffffffull;
    }
};

struct Sums {
    uint32_t count;
    uint64_t weight;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    return (uint64_t)__shfl_up((uint32_t)(v >> 32), d) << 32 | __shfl_up((uint32_t)v, d);
}

struct Shared {
    uint64_t weight[kBins];
    uint32_t count[kBins];
    uint64_t wave_weight[kWaves];
    uint32_t wave_count[kWaves];
    uint64_t found_weight;
    uint32_t found_count, found_bin, found_in_bin;
};

// Sums over the threads before this one, and over all.
__device__ __forceinline__ Sums scan_before(Sums v, Sums& all, Shared& sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums in = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t w = shfl_up64(in.weight, d);
        const uint32_t c = __shfl_up(in.count, d);
        if (lane >= d) {
            in.weight += w;
            in.count += c;
        }
    }
    __syncthreads();  // what an earlier call left has been read
    if (lane == 63) {
        sh.wave_weight[wave] = in.weight;
        sh.wave_count[wave] = in.count;
    }
    __syncthreads();
    Sums before = {in.count - v.count, in.weight - v.weight};
    all = {0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) {
            before.weight += sh.wave_weight[w];
            before.count += sh.wave_count[w];
        }
        all.weight += sh.wave_weight[w];
        all.count += sh.wave_count[w];
    }
    return before;
}

// A border in the sorted row: what lies above `key` is inside, and `ties` of those equal to it.
struct Border {
    uint32_t key, ties, equal;  // equal: how many there are
    uint64_t above;             // weight of what lies above
};

// Where the count (by_weight: the weight) of the sorted row reaches `goal`, which all of it does reach.
template <int DT>
__device__ Border find_border(const void* row, int64_t n, const Weights& w, bool by_weight, uint64_t goal, Shared& sh) {
    uint32_t prefix = 0, count_above = 0, equal = 0;
    uint64_t weight_above = 0;
    for (int level = 0; level < 3; ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            sh.weight[i] = 0;
            sh.count[i] = 0;
        }
        __syncthreads();
        for (int64_t i = threadIdx.x; i < n; i += kThreads) {
            const uint32_t key = load_key<DT>(row, i);
            if (key < kLeast || (level > 0 && key >> (shift + bits) != prefix)) continue;
            const uint32_t bin = key >> shift & ((1u << bits) - 1);
            atomicAdd(&sh.count[bin], 1u);
            atomicAdd((unsigned long long*)&sh.weight[bin], (unsigned long long)w.of(key));
        }
        __syncthreads();
        // a thread has two bins, the highest first
        const int hi = kBins - 1 - 2 * threadIdx.x, lo = hi - 1;
        const Sums a = {sh.count[hi], sh.weight[hi]}, b = {sh.count[lo], sh.weight[lo]};
        Sums all;
        Sums before = scan_before({a.count + b.count, a.weight + b.weight}, all, sh);
        before.count += count_above;
        before.weight += weight_above;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Sums& bin = k ? b : a;
            const uint64_t from = by_weight ? before.weight : before.count, to = from + (by_weight ? bin.weight : bin.count);
            if (from < goal && goal <= to) {
                sh.found_bin = k ? lo : hi;
                sh.found_count = before.count;
                sh.found_weight = before.weight;
                sh.found_in_bin = bin.count;
            }
            before.count += bin.count;
            before.weight += bin.weight;
        }
        __syncthreads();
        prefix = prefix << bits | sh.found_bin;
        count_above = sh.found_count;
        weight_above = sh.found_weight;
        equal = sh.found_in_bin;
        __syncthreads();
    }
    Border r = {prefix, 0, equal, weight_above};
    if (by_weight) {
        const uint64_t each = w.of(prefix);  // not 0: the weight reaches the goal here
        r.ties = (uint32_t)((goal - weight_above + each - 1) / each);
    } else {
        r.ties = (uint32_t)(goal - count_above);
    }
    return r;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a, int bits) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = blockIdx.x, n = a.vocab;
    const void* const row = (const char*)a.x + r * a.row_stride * (DT == QK_F32 ? 4 : 2);

    uint32_t top = 0;
    for (int64_t i = tid; i < n; i += kThreads) {
        const uint32_t key = load_key<DT>(row, i);
        top = key > top ? key : top;
    }
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_xor(top, d);
        top = o > top ? o : top;
    }
    if (lane == 0) sh.wave_count[wave] = top;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) top = sh.wave_count[w] > top ? sh.wave_count[w] : top;
    if (top < kLeast) {
        if (tid == 0) {
            a.tokens[r] = -1;
            a.logprobs[r] = -__builtin_inff();
        }
        return;
    }

    const float temperature = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    const Weights w = {(double)value_of(top), greedy ? 0.0 : 1.44269504088896340736 / (double)temperature, __builtin_ldexp(1.0, bits), top};
    // the kept: down to `border`, of whose ties those up to index `last`, and of those the ones of log2 weight `least` and more
    Border border = {kLeast, 0, 0, 0};
    bool cut = false;
    double least = -__builtin_inf();
    if (greedy) {
        border = {top, 1, 2, 0};
        cut = true;
    } else {
        const int32_t k = a.top_k ? a.top_k[r] : 0;
        const float p = a.top_p ? a.top_p[r] : 1.0f, m = a.min_p ? a.min_p[r] : 0.0f;
        if (m > 0.0f) least = ::log2((double)(m < 1.0f ? m : 1.0f));
        Sums all, mine = {0, 0};
        if ((k > 0 && k < n) || p < 1.0f) {
            for (int64_t i = tid; i < n; i += kThreads) {
                const uint32_t key = load_key<DT>(row, i);
                mine.count += key >= kLeast;
                mine.weight += w.of(key);
            }
            scan_before(mine, all, sh);
            uint64_t total = all.weight;
            if (k > 0 && (uint32_t)k < all.count) {
                border = find_border<DT>(row, n, w, false, (uint64_t)k, sh);
                cut = true;
                total = border.above + border.ties * w.of(border.key);
            }
            if (p < 1.0f) {
                const double goal = __builtin_ceil((double)p * (double)total);
                border = find_border<DT>(row, n, w, true, goal >= 1.0 ? (uint64_t)goal : 1, sh);
                cut = true;
            }
        }
    }

    // index of the last tie that is kept
    int64_t last = n - 1;
    if (cut && border.ties < border.equal) {
        uint32_t seen = 0;
        for (int64_t base = 0; base < n; base += kThreads) {
            const int64_t i = base + tid;
            const bool tie = i < n && load_key<DT>(row, i) == border.key;
            Sums all;
            const Sums before = scan_before({tie, 0}, all, sh);
            if (tie && seen + before.count == border.ties - 1) sh.found_weight = (uint64_t)i;
            seen += all.count;
            if (seen >= border.ties) break;
        }
        __syncthreads();
        last = (int64_t)sh.found_weight;
    }
    auto kept = [&](int64_t i, uint32_t key) -> uint64_t {
        if (key < border.key || (key == border.key && i > last) || w.log2_of(key) < least) return 0;
        return w.of(key);
    };

    Sums all, mine = {0, 0};
    for (int64_t i = tid; i < n; i += kThreads) mine.weight += kept(i, load_key<DT>(row, i));
    scan_before(mine, all, sh);
    const float u = fminf(fmaxf(a.uniform[r], 0.0f), 1.0f - 0x1p-24f);
    const uint64_t total = all.weight, goal = (uint64_t)((double)u * (double)total) + 1;  // at most total
    uint64_t passed = 0;
    for (int64_t base = 0; base < n; base += kThreads) {
        const int64_t i = base + tid;
        const uint32_t key = i < n ? load_key<DT>(row, i) : 0;
        const uint64_t v = i < n ? kept(i, key) : 0;
        const Sums before = scan_before({0, v}, all, sh);
        const uint64_t from = passed + before.weight;
        if (from < goal && goal <= from + v) {
            a.tokens[r] = (int32_t)i;
            a.logprobs[r] = greedy ? 0.0f : (float)((w.log2_of(key) + (double)bits - ::log2((double)total)) * 0.693147180559945309417);
        }
        passed += all.weight;
        if (passed >= goal) break;
    }
}

// F of the weights: the sum of `vocab` of them stays below 2^63.
int weight_bits(int64_t vocab) {
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    return 62 - bits < 50 ? 62 - bits : 50;
}

}  // namespace

size_t sample_workspace(int64_t rows, int64_t vocab, int dtype, bool filters) { return 0; }

hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream) {
    const int bits = weight_bits(a.vocab);
    const dim3 grid((unsigned)a.rows);
    if (a.dtype == QK_F32) sample_rows<QK_F32><<<grid, kThreads, 0, stream>>>(a, bits);
    else if (a.dtype == QK_BF16) sample_rows<QK_BF16><<<grid, kThreads, 0, stream>>>(a, bits);
    else sample_rows<QK_F16><<<grid, kThreads, 0, stream>>>(a, bits);
    return hipGetLastError();
}

}  // namespace qk
