// A token per row of logits: w_i = e^((x_i - max) / temperature), the kept tokens a head of the row sorted by x (falling, then by
// index), and the first kept one, by index, at which the kept weights' sum passes uniform * their whole sum.
//
// Weights are whole numbers, multiples of 2^-F of the largest, in 64 bits: their sums are exact and do not depend on the order in
// which they are made, so the same call gives the same token however the work is split.  F = 62 - log2(vocab), at most 50: what is
// rounded away is below 2^-(F + 1) of the largest weight each.
//
// Bound by HBM for many rows (each logit is read from it once), by latency for few.  No row is sorted.  A row is cut into segments of 256
// 16-byte vectors, a wave's step, and the segments dealt to workgroups; what one knows of its part goes to the last of the row's
// to arrive:
//   look   the largest logit; where a filter cuts, a histogram of the logits in bins of 1/64 of the temperature below the part's
//          largest, counts and weights (near enough: in units of the bin's upper end).  The last one joins them and finds the
//          bins in which the border of the kept tokens lies: counts are exact, and a border in the weights is bracketed.
//   draw   exact sums of the bins above those, by segment, and a list of the tokens in them.  The last one sorts the
//          list, finds the border in exact sums, the segment in which the drawn number falls, and the token there.
// A row whose list would be too long, or whose border is not where the histogram put it, is done by one workgroup that finds each border
// in the logits' bits, eleven at a time.  Rows that fill the card by themselves go through both steps in one launch.
#include "sample.h"

namespace qk {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;      // of the histograms
constexpr int kPerUnit = 64;     // bins per temperature
constexpr int kList = 4096;      // tokens in the border's bins
constexpr int kSegmentVectors = 256;
constexpr int kSegments = 1024;  // of a row at most
constexpr int64_t kMostTokens = 1 << 20;  // of a row that is split: a bin's count and weight share 64 bits

// Logits as whole numbers in their order; both zeros are one, NaN lies below -inf.
constexpr uint32_t kLeast = 0x00800000u;  // the lowest finite one: what lies below is never drawn
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return 0;
    if (u == 0x80000000u) return u;
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }
// A token in the sorted row: what comes earlier is smaller.
__device__ __forceinline__ uint64_t place_of(uint32_t key, uint32_t i) { return (uint64_t)~key << 32 | i; }

template <int DT>
__device__ __forceinline__ float load_logit(const void* row, int64_t i) {
    if constexpr (DT == QK_F32) return ((const float*)row)[i];
    else return load_half_bits(((const uint16_t*)row)[i], DT);
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
    bool infinite;       // top is: equal weights for its like, none for the others

    // log2 of the weight of a logit that is not below the lowest finite one
    __device__ __forceinline__ double log2_of(float x) const {
        if (infinite) return x == __builtin_inff() ? 0.0 : -__builtin_inf();
        return ((double)x - top) * factor;
    }
    __device__ __forceinline__ uint64_t of_log2(double t) const {
        if (!(t >= -60.0)) return 0;
        // rounded to a whole number by adding 2^52, in whose last bits it then stands
        return __builtin_bit_cast(uint64_t, pow2(t) * one + 0x1p52) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ uint64_t of(uint32_t key) const { return key < kLeast ? 0 : of_log2(log2_of(value_of(key))); }
};

// ---------------------------------------------------------------- sums over a workgroup

struct Sums {
    uint32_t count;
    uint64_t weight;
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    return (uint64_t)__shfl_up((uint32_t)(v >> 32), d) << 32 | __shfl_up((uint32_t)v, d);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
    for (int d = 1; d < 64; d <<= 1) v += (uint64_t)__shfl_xor((uint32_t)(v >> 32), d) << 32 | __shfl_xor((uint32_t)v, d);
    return v;
}

struct Scan {
    uint64_t weight[kWaves];
    uint32_t count[kWaves];
};

// Sums over the threads before this one, and over all.
__device__ __forceinline__ Sums scan_before(Sums v, Sums& all, Scan& sh) {
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
        sh.weight[wave] = in.weight;
        sh.count[wave] = in.count;
    }
    __syncthreads();
    Sums before = {in.count - v.count, in.weight - v.weight};
    all = {0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) {
            before.weight += sh.weight[w];
            before.count += sh.count[w];
        }
        all.weight += sh.weight[w];
        all.count += sh.count[w];
    }
    return before;
}

__device__ __forceinline__ float block_max(float v, Scan& sh) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.count[threadIdx.x >> 6] = __float_as_uint(v);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = fmaxf(v, __uint_as_float(sh.count[w]));
    return v;
}
__device__ __forceinline__ uint32_t block_min(uint32_t v, Scan& sh) {
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_xor(v, d);
        v = o < v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.count[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v = sh.count[w] < v ? sh.count[w] : v;
    return v;
}

// ---------------------------------------------------------------- what a row is asked for

struct Settings {
    float temperature, top_p, min_p, uniform;
    int32_t top_k;
    bool greedy;
};
__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int64_t r) {
    Settings s;
    s.temperature = a.temperature ? a.temperature[r] : 1.0f;
    s.top_k = a.top_k ? a.top_k[r] : 0;
    s.top_p = a.top_p ? a.top_p[r] : 1.0f;
    s.min_p = a.min_p ? a.min_p[r] : 0.0f;
    s.uniform = fminf(fmaxf(a.uniform[r], 0.0f), 1.0f - 0x1p-24f);
    s.greedy = !(s.temperature > 0.0f);
    return s;
}
__device__ __forceinline__ Weights weights_of(const Settings& s, float top, int bits) {
    return {(double)top, s.greedy ? 0.0 : 1.44269504088896340736 / (double)s.temperature, __builtin_ldexp(1.0, bits),
            top == __builtin_inff()};
}
// The least log2 of a weight that min_p keeps
__device__ __forceinline__ double least_of(const Settings& s) {
    return s.min_p > 0.0f ? ::log2((double)(s.min_p < 1.0f ? s.min_p : 1.0f)) : -__builtin_inf();
}
// The weight that the kept ones reach first, of a whole of `total`: at least 1, so that the first token stays
__device__ __forceinline__ uint64_t top_p_goal(const Settings& s, uint64_t total) {
    const double goal = __builtin_ceil((double)s.top_p * (double)total);
    return goal >= 1.0 ? (uint64_t)goal : 1;
}
__device__ __forceinline__ void write_token(const SampleArgs& a, int64_t r, int64_t i, float x, const Weights& w, int bits, uint64_t total) {
    a.tokens[r] = (int32_t)i;
    a.logprobs[r] = (float)((w.log2_of(x) + (double)bits - ::log2((double)total)) * 0.693147180559945309417);
}

// ---------------------------------------------------------------- one workgroup, border by border

struct Digits {
    uint64_t weight[kBins];
    uint32_t count[kBins];
    uint64_t found_weight;
    uint32_t found_count, found_bin, found_in_bin;
};

// A border in the sorted row: what lies above `key` is inside, and `ties` of those equal to it.
struct Border {
    uint32_t key, ties, equal;  // equal: how many there are
    uint64_t above;             // weight of what lies above
};

// Where the count (by_weight: the weight) of the sorted row reaches `goal`, which all of it does reach.
template <int DT>
__device__ Border find_border(const void* row, int64_t n, const Weights& w, bool by_weight, uint64_t goal, Digits& sh, Scan& scan) {
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
            const uint32_t key = key_of(load_logit<DT>(row, i));
            if (key < kLeast || (level > 0 && key >> (shift + bits) != prefix)) continue;
            const uint32_t bin = key >> shift & ((1u << bits) - 1);
            atomicAdd(&sh.count[bin], 1u);
            atomicAdd((unsigned long long*)&sh.weight[bin], (unsigned long long)w.of(key));
        }
        __syncthreads();
        // a thread has some bins, the highest first
        constexpr int kOwn = kBins / kThreads;
        const int hi = kBins - 1 - kOwn * (int)threadIdx.x;
        Sums own = {0, 0}, all;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            own.count += sh.count[hi - k];
            own.weight += sh.weight[hi - k];
        }
        Sums before = scan_before(own, all, scan);
        before.count += count_above;
        before.weight += weight_above;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const Sums bin = {sh.count[hi - k], sh.weight[hi - k]};
            const uint64_t from = by_weight ? before.weight : before.count, to = from + (by_weight ? bin.weight : bin.count);
            if (from < goal && goal <= to) {
                sh.found_bin = hi - k;
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

// A row whose largest logit is `top`, above -inf.
template <int DT>
__device__ void draw_alone(const SampleArgs& a, int64_t r, const void* row, const Settings& s, float top, int bits, Digits& sh, Scan& scan) {
    const int tid = threadIdx.x;
    const int64_t n = a.vocab;
    const Weights w = weights_of(s, top, bits);
    const double least = least_of(s);
    // the kept: down to `border`, of whose ties those up to index `last`, and of those the ones of log2 weight `least` and more
    Border border = {kLeast, 0, 0, 0};
    bool cut = false;
    Sums all, mine = {0, 0};
    if ((s.top_k > 0 && s.top_k < n) || s.top_p < 1.0f) {
        for (int64_t i = tid; i < n; i += kThreads) {
            const uint32_t key = key_of(load_logit<DT>(row, i));
            mine.count += key >= kLeast;
            mine.weight += w.of(key);
        }
        scan_before(mine, all, scan);
        uint64_t total = all.weight;
        if (s.top_k > 0 && (uint32_t)s.top_k < all.count) {
            border = find_border<DT>(row, n, w, false, (uint64_t)s.top_k, sh, scan);
            cut = true;
            total = border.above + border.ties * w.of(border.key);
        }
        if (s.top_p < 1.0f) {
            border = find_border<DT>(row, n, w, true, top_p_goal(s, total), sh, scan);
            cut = true;
        }
    }
    int64_t last = n - 1;
    if (cut && border.ties < border.equal) {
        uint32_t seen = 0;
        for (int64_t base = 0; base < n && seen < border.ties; base += kThreads) {
            const int64_t i = base + tid;
            const bool tie = i < n && key_of(load_logit<DT>(row, i)) == border.key;
            const Sums before = scan_before({tie, 0}, all, scan);
            if (tie && seen + before.count == border.ties - 1) sh.found_weight = (uint64_t)i;
            seen += all.count;
        }
        __syncthreads();
        last = (int64_t)sh.found_weight;
    }
    auto kept = [&](int64_t i) -> uint64_t {
        if (i >= n) return 0;
        const uint32_t key = key_of(load_logit<DT>(row, i));
        if (key < border.key || (key == border.key && i > last) || key < kLeast || w.log2_of(value_of(key)) < least) return 0;
        return w.of(key);
    };
    mine = {0, 0};
    for (int64_t i = tid; i < n; i += kThreads) mine.weight += kept(i);
    scan_before(mine, all, scan);
    const uint64_t total = all.weight, goal = (uint64_t)((double)s.uniform * (double)total) + 1;  // at most total
    uint64_t passed = 0;
    for (int64_t base = 0; base < n && passed < goal; base += kThreads) {
        const uint64_t v = kept(base + tid);
        const uint64_t from = passed + scan_before({0, v}, all, scan).weight;
        if (from < goal && goal <= from + v) write_token(a, r, base + tid, load_logit<DT>(row, base + tid), w, bits, total);
        passed += all.weight;
    }
}

// ---------------------------------------------------------------- look and draw

// A row as vectors of 16 aligned bytes: token i is element i + offset of them.  (Elements of the first and the last vector that are
// not the row's are read, and not used: a vector with one byte of a row lies in memory as a whole.)
template <int DT>
struct Row {
    static constexpr int kPer = DT == QK_F32 ? 4 : 8;
    static constexpr int kSteps = kSegmentVectors / 64;
    const u32x4* vectors;
    int32_t offset, n, count;  // count: of vectors

    __device__ __forceinline__ const void* start() const {
        return (const char*)vectors + offset * (DT == QK_F32 ? 4 : 2);
    }

    __device__ __forceinline__ Row(const SampleArgs& a, int64_t r) {
        constexpr int kSize = DT == QK_F32 ? 4 : 2;
        const uintptr_t at = (uintptr_t)a.x + r * a.row_stride * kSize;
        vectors = (const u32x4*)(at & ~(uintptr_t)15);
        offset = (int32_t)(at & 15) / kSize;
        n = (int32_t)a.vocab;
        count = (n + offset + kPer - 1) / kPer;
    }
    // A lane's vectors of a segment (past the row: of what comes first, not used)
    __device__ __forceinline__ void load(int32_t segment, int lane, u32x4 (&v)[kSteps]) const {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int32_t at = segment * kSegmentVectors + k * 64 + lane;
            v[k] = vectors[at < count ? at : 0];
        }
    }
    // f(token, logit) for its elements, -inf past the row's
    template <typename F>
    __device__ __forceinline__ void each(int32_t segment, int lane, const u32x4 (&v)[kSteps], F f) const {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int32_t first = (segment * kSegmentVectors + k * 64 + lane) * kPer - offset;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                float x;
                if constexpr (DT == QK_F32) x = __uint_as_float(v[k][e]);
                else x = load_half_bits(v[k][e >> 1] >> (16 * (e & 1)) & 0xffffu, DT);
                f(first + e, (uint32_t)(first + e) < (uint32_t)n ? x : -__builtin_inff());
            }
        }
    }
    __device__ __forceinline__ int32_t segment_of(uint32_t token) const { return (int32_t)(token + offset) / (kPer * kSegmentVectors); }
};

// The bin of a logit: below the one of `top` by so many.  Falls where the logit rises, as every step of it does.
__device__ __forceinline__ int32_t bin_at(float x, float per_bin) {
    return (int32_t)__builtin_floorf(fminf(fmaxf(x * per_bin, -0x1p29f), 0x1p29f));
}

// What the look at a row found: it is done (greedy, or nothing to draw), it is done by one workgroup, no filter cuts it, or the border of
// the kept tokens lies in bins low .. high, counted from the one of `top` (kBins: all past the histogram), `above` tokens before
// them; top_k: 0 where that does not cut.
constexpr int kDone = 0, kAlone = 1, kWhole = 2, kCut = 3;
struct Plan {
    int32_t mode;
    float top;
    int32_t top_bin, low, high, top_k;
    uint32_t above;
};
// What a workgroup's look at its part found: the largest logit, the first token that has it (greedy rows), how many could be drawn
// (rows with a histogram).
struct Part {
    float top;
    uint32_t first, valid;
};

struct Look {
    uint64_t bins[kBins];  // count << 40 | weight
    int32_t shift[kThreads];
    int32_t found[3];      // bins: the borders in the weights, from below and from above, and in the count
    uint64_t weight[2];
    uint32_t above, upto;
};
struct Draw {
    uint64_t list[kList];
    uint64_t kept[kSegments];
    uint64_t found_weight;
    uint32_t listed, base;
    int32_t found_k, found_p, segment;
};
union Space {
    Look look;
    Draw draw;
    Digits digits;
};

// A part of a row: its largest logit and, where a filter cuts, its histogram.  The weight of a logit in units of that of its bin's upper
// end, 1 - z + z^2 / 2 for e^-z below 1/64: it only has to lead to the border.
template <int DT>
__device__ Part look_at(const Row<DT>& row, const Settings& s, bool histogram, int32_t seg0, int32_t seg1, Look& sh, Scan& scan) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u32x4 v[Row<DT>::kSteps];
    Part part = {-__builtin_inff(), 0xffffffffu, 0};
    for (int32_t g = seg0 + wave; g < seg1; g += kWaves) {
        row.load(g, lane, v);
        row.each(g, lane, v, [&](int32_t, float x) { part.top = fmaxf(part.top, x); });
    }
    if (histogram)
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    part.top = block_max(part.top, scan);
    if (s.greedy) {
        for (int32_t g = seg0 + wave; g < seg1; g += kWaves) {
            row.load(g, lane, v);
            row.each(g, lane, v, [&](int32_t i, float x) { part.first = x == part.top && (uint32_t)i < part.first ? (uint32_t)i : part.first; });
        }
        part.first = block_min(part.first, scan);
    }
    if (histogram) {
        const float per_bin = (float)kPerUnit / s.temperature;
        const int32_t top_bin = bin_at(part.top, per_bin);
        for (int32_t g = seg0 + wave; g < seg1; g += kWaves) {
            row.load(g, lane, v);
            row.each(g, lane, v, [&](int32_t, float x) {
                if (x > -__builtin_inff()) {
                    ++part.valid;
                    const int32_t at = bin_at(x, per_bin), bin = top_bin - at;
                    const float z = fminf(fmaxf((float)at + 1.0f - x * per_bin, 0.0f), 1.0f) * (1.0f / kPerUnit);
                    if (bin < kBins)
                        atomicAdd((unsigned long long*)&sh.bins[bin], 1ull << 40 | (uint32_t)((1.0f - z + 0.5f * z * z) * 0x1p20f));
                }
            });
        }
        Sums all;
        scan_before({part.valid, 0}, all, scan);  // (its barriers: the histogram is whole behind them)
        part.valid = all.count;
    }
    return part;
}

// The border's bins of a row; bin(b, count, weight) gives the histogram's bin b, its weight in units of its own upper end.
template <typename F>
__device__ Plan plan_row(const Settings& s, float top, uint32_t valid, Look& sh, Scan& scan, F bin) {
    constexpr int kOwn = kBins / kThreads;
    const int first = kOwn * threadIdx.x;
    Sums own[kOwn], sum = {0, 0}, all;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        float weight;
        bin(first + k, own[k].count, weight);
        // in units of 2^-24 of the top bin's upper end
        own[k].weight = (uint64_t)(weight * __builtin_amdgcn_exp2f((float)(first + k) * (-1.44269504f / kPerUnit)) * 0x1p24f);
        sum.count += own[k].count;
        sum.weight += own[k].weight;
    }
    const Sums before = scan_before(sum, all, scan);
    const bool cuts = s.top_k > 0 && (uint32_t)s.top_k < valid;
    if (threadIdx.x == 0) {
        sh.found[0] = sh.found[1] = sh.found[2] = kBins;
        sh.weight[0] = sh.weight[1] = all.weight;
        sh.above = all.count;
        sh.upto = valid;
    }
    __syncthreads();
    // visit(b, sums before the bin, the bin's): this thread's bins
    auto each = [&](auto visit) {
        Sums at = before;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            visit(first + k, at, own[k]);
            at.count += own[k].count;
            at.weight += own[k].weight;
        }
    };
    if (cuts)
        each([&](int b, const Sums& at, const Sums& in) {
            if (at.count < (uint32_t)s.top_k && (uint32_t)s.top_k <= at.count + in.count) {
                sh.found[2] = b;
                sh.weight[0] = at.weight;
                sh.weight[1] = at.weight + in.weight;
            }
        });
    __syncthreads();
    if (s.top_p < 1.0f) {
        // the weights here are within 2^-13 of the exact ones by far; what does not hold in the end is found out then
        const double p = s.top_p > 0.0f ? (double)s.top_p : 0.0;
        const uint64_t from = (uint64_t)(p * (double)sh.weight[0] * (1.0 - 0x1p-13)) + 1, to = (uint64_t)(p * (double)sh.weight[1] * (1.0 + 0x1p-13)) + 1;
        each([&](int b, const Sums& at, const Sums& in) {
            if (at.weight < from && from <= at.weight + in.weight) sh.found[0] = b;
            if (at.weight < to && to <= at.weight + in.weight) sh.found[1] = b;
        });
    }
    __syncthreads();
    Plan p = {kCut, top, bin_at(top, (float)kPerUnit / s.temperature), 0, 0, cuts ? s.top_k : 0, 0};
    p.low = s.top_p < 1.0f && sh.found[0] < sh.found[2] ? sh.found[0] : sh.found[2];
    p.high = cuts ? sh.found[2] : sh.found[1];
    if (p.high < p.low) p.high = p.low;
    each([&](int b, const Sums& at, const Sums& in) {
        if (b == p.low) sh.above = at.count;
        if (b == p.high) sh.upto = at.count + in.count;
    });
    __syncthreads();
    p.above = sh.above;
    if (!cuts && !(s.top_p < 1.0f)) p.mode = kWhole;
    else if (sh.upto - sh.above > (uint32_t)kList) p.mode = kAlone;
    return p;
}

// A part of a row: exact sums of the weights above the border's bins (`all`: of all weights), by segment of those that min_p keeps,
// and the tokens in the border's bins, in any order.
struct Drawn {
    uint64_t all, above;
};
template <int DT, typename F>
__device__ Drawn draw_part(const Row<DT>& row, const Settings& s, const Weights& w, const Plan& p, int32_t seg0, int32_t seg1, Draw& sh,
                           Scan& scan, F segment_sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const bool cut = p.mode == kCut, whole_sum = cut && s.top_p < 1.0f && p.top_k == 0;
    const float per_bin = cut ? (float)kPerUnit / s.temperature : 0.0f;
    const double least = least_of(s);
    u32x4 v[Row<DT>::kSteps];
    Drawn d = {0, 0};
    for (int32_t g = seg0 + wave; g < seg1; g += kWaves) {
        uint64_t kept = 0;
        row.load(g, lane, v);
        row.each(g, lane, v, [&](int32_t i, float x) {
            if (x > -__builtin_inff()) {
                int32_t bin = cut ? p.top_bin - bin_at(x, per_bin) : -1;
                bin = bin < kBins ? bin : kBins;
                const bool above = !cut || bin < p.low;
                if (above || whole_sum) {
                    const double t = w.log2_of(x);
                    const uint64_t weight = w.of_log2(t);
                    d.all += weight;
                    if (above) {
                        d.above += weight;
                        kept += t >= least ? weight : 0;
                    }
                }
                if (!above && bin <= p.high) {
                    const uint32_t at = atomicAdd(&sh.listed, 1u);
                    if (at < (uint32_t)kList) sh.list[at] = place_of(key_of(x), (uint32_t)i);
                }
            }
        });
        kept = wave_sum64(kept);
        if (lane == 0) segment_sum(g, kept);
    }
    Sums all;
    scan_before({0, d.all}, all, scan);
    d.all = all.weight;
    scan_before({0, d.above}, all, scan);
    d.above = all.weight;
    return d;
}

// The token of a row whose parts are together: sh.list holds `listed` tokens, sh.kept the segments' sums.
template <int DT>
__device__ void draw_row(const SampleArgs& a, int64_t r, const Row<DT>& row, const Settings& s, const Weights& w, int bits, const Plan& p,
                         const Drawn& d, int32_t segments, uint32_t listed, Space& space, Scan& scan) {
    Draw& sh = space.draw;
    const int tid = threadIdx.x;
    const double least = least_of(s);
    uint64_t border = ~0ull;  // the last kept token in the sorted row
    if (p.mode == kCut) {
        // the list in order: a bitonic sort
        uint32_t size = 2;
        while (size < listed) size *= 2;
        for (uint32_t i = listed + tid; i < size; i += kThreads) sh.list[i] = ~0ull;
        for (uint32_t run = 2; run <= size; run *= 2)
            for (uint32_t step = run / 2; step > 0; step /= 2) {
                __syncthreads();
                for (uint32_t i = tid; i < size / 2; i += kThreads) {
                    const uint32_t x = 2 * i - (i & (step - 1)), y = x + step;
                    const uint64_t l = sh.list[x], h = sh.list[y];
                    if ((l > h) == ((x & run) == 0)) {
                        sh.list[x] = h;
                        sh.list[y] = l;
                    }
                }
            }
        if (tid == 0) {
            sh.found_k = sh.found_p = -1;
            sh.found_weight = d.all;
        }
        __syncthreads();
        constexpr int kOwn = kList / kThreads;
        uint64_t own[kOwn], sum = 0;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const uint32_t i = tid * kOwn + k;
            own[k] = i < listed ? w.of(~(uint32_t)(sh.list[i] >> 32)) : 0;
            sum += own[k];
        }
        Sums all;
        const uint64_t before = d.above + scan_before({0, sum}, all, scan).weight;
        if (p.top_k) {
            uint64_t at = before;
#pragma unroll
            for (int k = 0; k < kOwn; ++k) {
                const uint32_t i = tid * kOwn + k;
                at += own[k];
                if (i < listed && p.above + i + 1 == (uint32_t)p.top_k) {
                    sh.found_k = (int32_t)i;
                    sh.found_weight = at;
                }
            }
        }
        __syncthreads();
        int32_t last = p.top_k ? sh.found_k : (int32_t)listed - 1;
        bool held = last >= 0;
        if (s.top_p < 1.0f) {
            const uint64_t goal = top_p_goal(s, sh.found_weight);
            uint64_t at = before;
#pragma unroll
            for (int k = 0; k < kOwn; ++k) {
                if (at < goal && goal <= at + own[k]) sh.found_p = tid * kOwn + k;
                at += own[k];
            }
            __syncthreads();
            held = held && sh.found_p >= 0;
            last = sh.found_p < last ? sh.found_p : last;
        }
        if (!held) {  // the border is not in these bins
            __syncthreads();
            draw_alone<DT>(a, r, row.start(), s, p.top, bits, space.digits, scan);
            return;
        }
        border = sh.list[last];
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            const uint32_t i = tid * kOwn + k;
            if ((int32_t)i <= last && w.log2_of(value_of(~(uint32_t)(sh.list[i] >> 32))) >= least)
                atomicAdd((unsigned long long*)&sh.kept[row.segment_of((uint32_t)sh.list[i])], (unsigned long long)own[k]);
        }
    }
    __syncthreads();
    // the segment in which the drawn number falls
    constexpr int kOwn = kSegments / kThreads;
    uint64_t own[kOwn], sum = 0;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        const int32_t g = tid * kOwn + k;
        own[k] = g < segments ? sh.kept[g] : 0;
        sum += own[k];
    }
    Sums all;
    uint64_t at = scan_before({0, sum}, all, scan).weight;
    const uint64_t total = all.weight, goal = (uint64_t)((double)s.uniform * (double)total) + 1;  // at most total
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        if (at < goal && goal <= at + own[k]) {
            sh.segment = tid * kOwn + k;
            sh.found_weight = at;
        }
        at += own[k];
    }
    __syncthreads();
    // and the token there
    constexpr int kEach = kSegmentVectors * Row<DT>::kPer / kThreads;
    const int32_t first = sh.segment * kSegmentVectors * Row<DT>::kPer + tid * kEach - row.offset;
    float x[kEach];
    uint64_t weight[kEach];
    sum = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int32_t i = first + k;
        x[k] = i >= 0 && i < row.n ? load_logit<DT>(row.start(), i) : -__builtin_inff();
        weight[k] = 0;
        if (x[k] > -__builtin_inff() && place_of(key_of(x[k]), (uint32_t)i) <= border) {
            const double t = w.log2_of(x[k]);
            if (t >= least) weight[k] = w.of_log2(t);
        }
        sum += weight[k];
    }
    at = sh.found_weight;
    at += scan_before({0, sum}, all, scan).weight;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        if (at < goal && goal <= at + weight[k]) write_token(a, r, first + k, x[k], w, bits, total);
        at += weight[k];
    }
}

__device__ __forceinline__ void write_plain(const SampleArgs& a, int64_t r, int32_t token) {
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        a.logprobs[r] = token < 0 ? -__builtin_inff() : 0.0f;
    }
}
__device__ __forceinline__ bool cuts(const Settings& s, int64_t vocab) {
    return !s.greedy && ((s.top_k > 0 && s.top_k < vocab) || s.top_p < 1.0f);
}

// ---------------------------------------------------------------- kernels

// A workgroup a row, nothing kept between its steps but in LDS.
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_rows(SampleArgs a, int bits, int32_t segments) {
    __shared__ Space space;
    __shared__ Scan scan;
    const int64_t r = blockIdx.x;
    const Row<DT> row(a, r);
    const Settings s = settings_of(a, r);
    const bool histogram = cuts(s, a.vocab) && segments > 0;
    const Part part = look_at<DT>(row, s, histogram, 0, (row.count + kSegmentVectors - 1) / kSegmentVectors, space.look, scan);
    if (part.top == -__builtin_inff()) return write_plain(a, r, -1);
    if (s.greedy) return write_plain(a, r, (int32_t)part.first);
    Plan p = {kWhole, part.top, 0, 0, 0, 0, 0};
    if (part.top == __builtin_inff() || segments == 0) p.mode = kAlone;
    else if (histogram)
        p = plan_row(s, part.top, part.valid, space.look, scan, [&](int b, uint32_t& count, float& weight) {
            const uint64_t v = space.look.bins[b];
            count = (uint32_t)(v >> 40);
            weight = (float)(v & ((1ull << 40) - 1)) * 0x1p-20f;
        });
    __syncthreads();  // of the histogram
    if (p.mode == kAlone) return draw_alone<DT>(a, r, row.start(), s, p.top, bits, space.digits, scan);
    const Weights w = weights_of(s, p.top, bits);
    const Drawn d = draw_part<DT>(row, s, w, p, 0, segments, space.draw, scan, [&](int32_t g, uint64_t sum) { space.draw.kept[g] = sum; });
    draw_row<DT>(a, r, row, s, w, bits, p, d, segments, space.draw.listed, space, scan);
}

struct SplitArgs {
    SampleArgs a;
    int bits;
    int32_t segments, per_group, groups;  // of a row; of a workgroup; workgroups of a row
    uint64_t tag;
    uint64_t *look_arrivals, *draw_arrivals;  // [rows]
    Plan* plans;       // [rows]
    uint32_t* listed;  // [rows]
    Part* parts;       // [rows][groups]
    uint64_t* bins;    // [rows][groups][kBins]
    Drawn* sums;       // [rows][groups]
    uint64_t* kept;    // [rows][segments]
    uint64_t* list;    // [rows][kList]
};

// What other workgroups wrote in the same launch, or will read there.
template <typename T>
__device__ __forceinline__ void put(T* p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T get(const T* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_look(SplitArgs g) {
    __shared__ Look sh;
    __shared__ Scan scan;
    const SampleArgs& a = g.a;
    const int64_t r = blockIdx.x / (uint32_t)g.groups;
    const int group = (int)(blockIdx.x % (uint32_t)g.groups), tid = threadIdx.x;
    const Row<DT> row(a, r);
    const Settings s = settings_of(a, r);
    const bool histogram = cuts(s, a.vocab);
    const int32_t seg0 = group * g.per_group, seg1 = seg0 + g.per_group < g.segments ? seg0 + g.per_group : g.segments;
    const Part part = look_at<DT>(row, s, histogram, seg0, seg1, sh, scan);
    Part* const parts = g.parts + r * g.groups;
    uint64_t* const bins = g.bins + r * g.groups * kBins;
    if (tid == 0) {
        put(&parts[group].top, part.top);
        put(&parts[group].first, part.first);
        put(&parts[group].valid, part.valid);
    }
    if (histogram)
        for (int i = tid; i < kBins; i += kThreads) put(bins + (int64_t)group * kBins + i, sh.bins[i]);
    if (!splitk_last(g.look_arrivals + r, (uint32_t)g.groups, g.tag)) return;

    // groups: at most a workgroup's threads
    const float own = tid < g.groups ? get(&parts[tid].top) : -__builtin_inff();
    const float top = block_max(own, scan);
    Plan p = {kDone, top, 0, 0, 0, 0, 0};
    if (top == -__builtin_inff()) {
        write_plain(a, r, -1);
    } else if (s.greedy) {
        write_plain(a, r, (int32_t)block_min(own == top ? get(&parts[tid < g.groups ? tid : 0].first) : 0xffffffffu, scan));
    } else if (top == __builtin_inff()) {
        p.mode = kAlone;
    } else if (!histogram) {
        p.mode = kWhole;
    } else {
        const float per_bin = (float)kPerUnit / s.temperature;
        // how far a part's histogram lies below the row's (one without a logit: past it)
        if (tid < g.groups) sh.shift[tid] = own > -__builtin_inff() ? bin_at(top, per_bin) - bin_at(own, per_bin) : kBins;
        Sums all;
        scan_before({tid < g.groups ? get(&parts[tid].valid) : 0, 0}, all, scan);
        p = plan_row(s, top, all.count, sh, scan, [&](int b, uint32_t& count, float& weight) {
            count = 0;
            weight = 0.0f;
            for (int c = 0; c < g.groups; ++c) {
                const int32_t at = b - sh.shift[c];
                if (at < 0) continue;
                const uint64_t v = get(bins + (int64_t)c * kBins + at);
                count += (uint32_t)(v >> 40);
                weight += (float)(v & ((1ull << 40) - 1)) * 0x1p-20f;
            }
        });
    }
    if (tid == 0) {
        g.plans[r] = p;
        g.listed[r] = 0;
    }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_draw(SplitArgs g) {
    __shared__ Space space;
    __shared__ Scan scan;
    Draw& sh = space.draw;
    const SampleArgs& a = g.a;
    const int64_t r = blockIdx.x / (uint32_t)g.groups;
    const int group = (int)(blockIdx.x % (uint32_t)g.groups), tid = threadIdx.x;
    const Plan p = g.plans[r];
    if (p.mode == kDone || (p.mode == kAlone && group > 0)) return;
    const Row<DT> row(a, r);
    const Settings s = settings_of(a, r);
    if (p.mode == kAlone) return draw_alone<DT>(a, r, row.start(), s, p.top, g.bits, space.digits, scan);
    const Weights w = weights_of(s, p.top, g.bits);
    const int32_t seg0 = group * g.per_group, seg1 = seg0 + g.per_group < g.segments ? seg0 + g.per_group : g.segments;
    uint64_t* const kept = g.kept + r * g.segments;
    uint64_t* const list = g.list + r * kList;
    Drawn* const sums = g.sums + r * g.groups;
    Drawn d = draw_part<DT>(row, s, w, p, seg0, seg1, sh, scan, [&](int32_t at, uint64_t sum) { put(kept + at, sum); });
    const uint32_t own = sh.listed < (uint32_t)kList ? sh.listed : kList;
    if (tid == 0) {
        put(&sums[group].all, d.all);
        put(&sums[group].above, d.above);
        sh.base = own ? __hip_atomic_fetch_add(g.listed + r, own, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < own; i += kThreads)
        if (sh.base + i < (uint32_t)kList) put(list + sh.base + i, sh.list[i]);
    if (!splitk_last(g.draw_arrivals + r, (uint32_t)g.groups, g.tag)) return;

    uint32_t listed = get(g.listed + r);
    listed = listed < (uint32_t)kList ? listed : kList;
    for (uint32_t i = tid; i < listed; i += kThreads) sh.list[i] = get(list + i);
    for (int32_t i = tid; i < g.segments; i += kThreads) sh.kept[i] = get(kept + i);
    Sums all;
    scan_before({0, tid < g.groups ? get(&sums[tid].all) : 0}, all, scan);
    d.all = all.weight;
    scan_before({0, tid < g.groups ? get(&sums[tid].above) : 0}, all, scan);
    d.above = all.weight;
    draw_row<DT>(a, r, row, s, w, g.bits, p, d, g.segments, listed, space, scan);
}

// ---------------------------------------------------------------- host

// F of the weights: the sum of `vocab` of them stays below 2^63.
int weight_bits(int64_t vocab) {
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    return 62 - bits < 50 ? 62 - bits : 50;
}

// Workgroups that a call should have: rows are cut until there are so many.
constexpr int64_t kWanted = 512;

struct Split {
    int32_t segments, per_group;
    int64_t groups;
    int64_t arrivals, plans, listed, parts, bins, sums, kept, list, bytes;  // offsets in the workspace
};
Split split(int64_t rows, int64_t vocab, int dtype) {
    Split p = {};
    const int64_t per = dtype == QK_F32 ? 4 : 8;
    const int64_t most = (vocab + per - 1 + per - 1) / per;  // vectors of a row that begins with the last element of one
    if (vocab > kMostTokens - 8) {
        p.groups = 1;
        return p;
    }
    p.segments = (int32_t)((most + kSegmentVectors - 1) / kSegmentVectors);
    const int64_t steps = (p.segments + kWaves - 1) / kWaves;  // of a workgroup that has all
    int64_t groups = (kWanted + rows - 1) / rows;
    groups = groups < steps ? groups : steps;
    p.per_group = (int32_t)((steps + groups - 1) / groups) * kWaves;
    p.groups = (p.segments + p.per_group - 1) / p.per_group;
    if (p.groups == 1) return p;
    auto take = [&](int64_t bytes) {
        const int64_t at = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    p.arrivals = take(rows * 16);
    p.plans = take(rows * (int64_t)sizeof(Plan));
    p.listed = take(rows * 4);
    p.parts = take(rows * p.groups * (int64_t)sizeof(Part));
    p.sums = take(rows * p.groups * (int64_t)sizeof(Drawn));
    p.kept = take(rows * p.segments * 8);
    p.bins = take(rows * p.groups * kBins * 8);
    p.list = take(rows * kList * 8);
    return p;
}

template <int DT>
hipError_t launch(const SampleArgs& a, void* workspace, hipStream_t stream) {
    const Split p = split(a.rows, a.vocab, a.dtype);
    const int bits = weight_bits(a.vocab);
    if (p.groups == 1) {
        sample_rows<DT><<<dim3((unsigned)a.rows), kThreads, 0, stream>>>(a, bits, p.segments);
        return hipGetLastError();
    }
    char* const ws = (char*)workspace;
    SplitArgs g = {};
    g.a = a;
    g.bits = bits;
    g.segments = p.segments;
    g.per_group = p.per_group;
    g.groups = (int)p.groups;
    g.tag = next_split_tag();
    g.look_arrivals = (uint64_t*)(ws + p.arrivals);
    g.draw_arrivals = g.look_arrivals + a.rows;
    g.plans = (Plan*)(ws + p.plans);
    g.listed = (uint32_t*)(ws + p.listed);
    g.parts = (Part*)(ws + p.parts);
    g.bins = (uint64_t*)(ws + p.bins);
    g.sums = (Drawn*)(ws + p.sums);
    g.kept = (uint64_t*)(ws + p.kept);
    g.list = (uint64_t*)(ws + p.list);
    const dim3 grid((unsigned)(a.rows * p.groups));
    sample_look<DT><<<grid, kThreads, 0, stream>>>(g);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    sample_draw<DT><<<grid, kThreads, 0, stream>>>(g);
    return hipGetLastError();
}

}  // namespace

size_t sample_workspace(int64_t rows, int64_t vocab, int dtype) { return rows > 0 ? (size_t)split(rows, vocab, dtype).bytes : 0; }

hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream) {
    if (a.dtype == QK_F32) return launch<QK_F32>(a, workspace, stream);
    if (a.dtype == QK_BF16) return launch<QK_BF16>(a, workspace, stream);
    return launch<QK_F16>(a, workspace, stream);
}

}  // namespace qk
