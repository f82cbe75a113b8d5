// A token per row of logits: w_i = e^((x_i - max) / temperature), the kept tokens a head of the row sorted by x (falling, then by
// index), and the first kept one, by index, at which the kept weights' sum passes uniform * their whole sum.
//
// Weights are whole numbers, multiples of 2^-F of the largest, in 64 bits: their sums are exact and do not depend on the order in
// which they are made, so the same call gives the same token however the work is split.  F = 62 - log2(vocab), at most 50: what is
// rounded away is below 2^-(F + 1) of the largest weight each.
//
// Each logit is read from HBM once, and once or twice more from the caches; no row is sorted.  A row is cut into segments of one
// 16-byte vector a lane of a wave (four where there would be more than 1024 of them), and the segments dealt to workgroups; what one
// knows of its part goes to the last of the row's to arrive:
//   look   the largest logit; where a filter cuts, a histogram of the logits in bins of 1/64 of the temperature below the part's
//          largest, counts and weights (near enough: in units of the bin's upper end).  The last one joins them and finds the
//          bins in which the border of the kept tokens lies: counts are exact, and a border in the weights is bracketed.
//   draw   exact sums of the bins above those, by segment, and a list of the tokens in them.  The last one sorts the
//          list, finds the border in exact sums, the segment in which the drawn number falls, and the token there.
// A row whose list would be too long, or whose border is not where the histogram put it, is done by one workgroup that finds each border
// in the logits' bits, eleven at a time.  Rows that fill the card by themselves, and short ones, go through both steps in one workgroup; in
// rows whose look is little beside their draw each workgroup looks at the whole row, and one launch does (way_of).
//
// What bounds it: one row, the chain of steps (passes over the row, thresholds searched among the logits, a sort, scans): a row of
// 65536 takes 10 us without filters and 37 with all three, and twice the tokens 12 and 37.  Many rows, the vector units: an exact
// weight is 21 instructions in 64 bits, which a nucleus asks of every logit (its goal is a part of the exact sum), and the histogram an
// atomic in LDS each.  Measured on one MI355X: 96 rows of 65536 without filters 18.6 us (0.68 TB/s); 256 rows of 131072 under nuclei
// and min_p 94 us, of which the first pass takes 11, the histogram 17, the exact weights 45; 48 of 128257 in 32 bits under all three
// 46 us; one row of 32001 29 us.
#include "sample.h"

namespace qk {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;      // of the histograms
constexpr int kPerUnit = 64;     // bins per temperature
constexpr float kSlope = 0.0155038f;  // 1 - e^(-1 / 64): what a weight falls in a bin
constexpr int kList = 4096;      // tokens in the border's bins
constexpr int kAhead = 4;        // parts' histograms that are read at a time
constexpr int kBatch = 4;        // 16-byte vectors that a lane asks for at a time
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

// a * b + c with c in scalar registers: by itself the compiler copies such a c into the result's registers first, once per product.
__device__ __forceinline__ double fma_scalar(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}
// 2^t + unit, unit being the power of two 2^(52 - bits): the last bits of it are then 2^t times 2^bits as a whole number, 0 where t is
// below -60 or NaN (t <= 0).  2^n times a polynomial in f = t - n, |f| <= 1/2, that meets 2^f in the 11 Chebyshev nodes and stays
// within 2^-51 of it; n is found by an addition whose last bits it is, and goes to the exponent as a whole number.
__device__ __forceinline__ uint64_t raw_weight(double t, double unit) {
    double c, p;
    asm("v_max_f64 %0, %1, %2" : "=v"(c) : "v"(t), "s"(-60.0));
    const double n = __builtin_rint(c), f = c - n;
    p = fma_scalar(0x1.e6063f7217bc6p-28, f, 0x1.b675bca4eeebbp-24);
    p = fma_scalar(p, f, 0x1.62bfd47773353p-20);
    p = fma_scalar(p, f, 0x1.ffcb54062e698p-17);
    p = fma_scalar(p, f, 0x1.430913096fd9fp-13);
    p = fma_scalar(p, f, 0x1.5d87fe9d7a584p-10);
    p = fma_scalar(p, f, 0x1.3b2ab6fba1ddap-7);
    p = fma_scalar(p, f, 0x1.c6b08d703ce49p-5);
    p = fma_scalar(p, f, 0x1.ebfbdff82c598p-3);
    p = fma_scalar(p, f, 0x1.62e42fefa3a19p-1);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_bit_cast(uint64_t, __builtin_ldexp(p, (int)n) + unit);
}

// Weights of a row whose largest logit is `top`.
struct Weights {
    double top, factor;  // log2 e / temperature
    int bits;            // F: the largest weight is 2^F
    bool infinite;       // top is: equal weights for its like, none for the others
    double unit;         // 2^(52 - bits)

    // log2 of a logit's weight in a row without an infinite one (-inf: -inf, or NaN where the temperature is infinite)
    __device__ __forceinline__ double finite_log2(float x) const { return ((double)x - top) * factor; }
    __device__ __forceinline__ uint64_t whole(uint64_t raw) const { return raw & 0xfffffffffffffull; }
    __device__ __forceinline__ uint64_t raw(float x) const { return raw_weight(finite_log2(x), unit); }  // with the bits of `unit` on top
    __device__ __forceinline__ uint64_t finite(float x) const { return whole(raw(x)); }
    // ... in any row
    __device__ __forceinline__ double log2_of(float x) const {
        if (infinite) return x == __builtin_inff() ? 0.0 : -__builtin_inf();
        return finite_log2(x);
    }
    __device__ __forceinline__ uint64_t of(uint32_t key) const { return key < kLeast ? 0 : whole(raw_weight(log2_of(value_of(key)), unit)); }
};

// ---------------------------------------------------------------- sums over a workgroup

// v of the lane that the move `DPP` names, 0 where there is none
template <int DPP, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, DPP, ROWS, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), DPP, ROWS, 0xf, true);
    return (uint64_t)hi << 32 | lo;
}
// Sum over the lanes up to this one: within rows of 16 lanes, then from a row's last lane to those behind.
__device__ __forceinline__ uint64_t wave_upto(uint64_t v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);
    v += moved<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}

// Sums, maxima and minima over the workgroup, each with one barrier: calls take the two halves of the space in turn, so that
// one may write while the one before is still read.
struct Group {
    struct Space {
        uint64_t of[2][kWaves];
    };
    Space& sh;
    int turn = 0;

    __device__ __forceinline__ const uint64_t* exchange(uint64_t of_wave, bool writes) {
        turn ^= 1;
        if (writes) sh.of[turn][threadIdx.x >> 6] = of_wave;
        __syncthreads();
        return sh.of[turn];
    }
    // Sum over the threads before this one, and over all.
    __device__ __forceinline__ uint64_t before(uint64_t v, uint64_t& all) {
        const int wave = threadIdx.x >> 6;
        const uint64_t upto = wave_upto(v);
        const uint64_t* const of = exchange(upto, (threadIdx.x & 63) == 63);
        uint64_t sum = upto - v;
        all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            sum += w < wave ? of[w] : 0;
            all += of[w];
        }
        return sum;
    }
    __device__ __forceinline__ uint64_t sum(uint64_t v) {
        const uint64_t* const of = exchange(last_lane(wave_upto(v)), (threadIdx.x & 63) == 0);
        uint64_t all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) all += of[w];
        return all;
    }
    __device__ __forceinline__ float max(float v) {
        const uint64_t* const of = exchange(__float_as_uint(wave_max(v)), (threadIdx.x & 63) == 0);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v = fmaxf(v, __uint_as_float((uint32_t)of[w]));
        return v;
    }
    __device__ __forceinline__ uint32_t min(uint32_t v) {
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_xor(v, d);
            v = o < v ? o : v;
        }
        const uint64_t* const of = exchange(v, (threadIdx.x & 63) == 0);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v = (uint32_t)of[w] < v ? (uint32_t)of[w] : v;
        return v;
    }
};

// (one of it in a kernel, not one at each use)
__device__ __attribute__((noinline)) double log2_of_double(double v) { return ::log2(v); }

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
    return {(double)top, s.greedy ? 0.0 : 1.44269504088896340736 / (double)s.temperature, bits, top == __builtin_inff(), __builtin_ldexp(1.0, 52 - bits)};
}
// The least log2 of a weight that min_p keeps
__device__ __forceinline__ double least_of(const Settings& s) {
    return s.min_p > 0.0f ? log2_of_double((double)(s.min_p < 1.0f ? s.min_p : 1.0f)) : -__builtin_inf();
}
// The weight that the kept ones reach first, of a whole of `total`: at least 1, so that the first token stays
__device__ __forceinline__ uint64_t top_p_goal(const Settings& s, uint64_t total) {
    const double goal = __builtin_ceil((double)s.top_p * (double)total);
    return goal >= 1.0 ? (uint64_t)goal : 1;
}
__device__ __forceinline__ void write_token(const SampleArgs& a, int64_t r, int64_t i, float x, const Weights& w, int bits, uint64_t total) {
    a.tokens[r] = (int32_t)i;
    a.logprobs[r] = (float)((w.log2_of(x) + (double)bits - log2_of_double((double)total)) * 0.693147180559945309417);
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
__device__ Border find_border(const void* row, int64_t n, const Weights& w, bool by_weight, uint64_t goal, Digits& sh, Group& group) {
    uint32_t prefix = 0, count_above = 0, equal = 0;
    uint64_t weight_above = 0;
#pragma nounroll
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
        uint64_t count = 0, weight = 0, all;
        for (int k = 0; k < kOwn; ++k) {
            count += sh.count[hi - k];
            weight += sh.weight[hi - k];
        }
        count = count_above + group.before(count, all);
        weight = weight_above + group.before(weight, all);
        for (int k = 0; k < kOwn; ++k) {
            const uint64_t from = by_weight ? weight : count, to = from + (by_weight ? sh.weight[hi - k] : sh.count[hi - k]);
            if (from < goal && goal <= to) {
                sh.found_bin = hi - k;
                sh.found_count = (uint32_t)count;
                sh.found_weight = weight;
                sh.found_in_bin = sh.count[hi - k];
            }
            count += sh.count[hi - k];
            weight += sh.weight[hi - k];
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
__device__ __forceinline__ void draw_alone(const SampleArgs& a, int64_t r, const void* row, const Settings& s, float top, int bits, Digits& sh,
                                           Group& group) {
    const int tid = threadIdx.x;
    const int64_t n = a.vocab;
    const Weights w = weights_of(s, top, bits);
    const double least = least_of(s);
    __syncthreads();  // what the space held has been read
    // the kept: down to `border`, of whose ties those up to index `last`, and of those the ones of log2 weight `least` and more
    Border border = {kLeast, 0, 0, 0};
    bool cut = false;
    if ((s.top_k > 0 && s.top_k < n) || s.top_p < 1.0f) {
        uint64_t count = 0, total = 0;
        for (int64_t i = tid; i < n; i += kThreads) {
            const uint32_t key = key_of(load_logit<DT>(row, i));
            count += key >= kLeast;
            total += w.of(key);
        }
        count = group.sum(count);
        total = group.sum(total);
        if (s.top_k > 0 && (uint64_t)s.top_k < count) {
            border = find_border<DT>(row, n, w, false, (uint64_t)s.top_k, sh, group);
            cut = true;
            total = border.above + border.ties * w.of(border.key);
        }
        if (s.top_p < 1.0f) {
            border = find_border<DT>(row, n, w, true, top_p_goal(s, total), sh, group);
            cut = true;
        }
    }
    int64_t last = n - 1;
    if (cut && border.ties < border.equal) {
        uint64_t seen = 0, all;
        for (int64_t base = 0; base < n && seen < border.ties; base += kThreads) {
            const int64_t i = base + tid;
            const bool tie = i < n && key_of(load_logit<DT>(row, i)) == border.key;
            const uint64_t before = group.before(tie, all);
            if (tie && seen + before == border.ties - 1) sh.found_weight = (uint64_t)i;
            seen += all;
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
    uint64_t total = 0;
    for (int64_t i = tid; i < n; i += kThreads) total += kept(i);
    total = group.sum(total);
    const uint64_t goal = (uint64_t)((double)s.uniform * (double)total) + 1;  // at most total
    uint64_t passed = 0, all;
    for (int64_t base = 0; base < n && passed < goal; base += kThreads) {
        const uint64_t v = kept(base + tid), from = passed + group.before(v, all);
        if (from < goal && goal <= from + v) write_token(a, r, base + tid, load_logit<DT>(row, base + tid), w, bits, total);
        passed += all;
    }
}

// ---------------------------------------------------------------- look and draw

// A row as vectors of 16 aligned bytes: token i is element i + offset of them.  (Elements of the first and the last vector that are
// not the row's are read, and not used: a vector with one byte of a row lies in memory as a whole.)  A segment is STEPS vectors of
// each lane of a wave: what one sum is kept of.
template <int DT, int STEPS>
struct Row {
    static constexpr int kType = DT, kSize = DT == QK_F32 ? 4 : 2, kPer = 16 / kSize;
    static constexpr int kSegment = STEPS * 64 * kPer;  // elements
    const u32x4* vectors;
    int32_t offset, n, count;  // count: of vectors

    __device__ __forceinline__ Row(const SampleArgs& a, int64_t r) {
        const uintptr_t at = (uintptr_t)a.x + r * a.row_stride * kSize;
        vectors = (const u32x4*)(at & ~(uintptr_t)15);
        offset = (int32_t)(at & 15) / kSize;
        n = (int32_t)a.vocab;
        count = (n + offset + kPer - 1) / kPer;
    }
    __device__ __forceinline__ const void* start() const { return (const char*)vectors + offset * kSize; }
    __device__ __forceinline__ int32_t segments() const { return (count + STEPS * 64 - 1) / (STEPS * 64); }
    __device__ __forceinline__ int32_t segment_of(uint32_t token) const { return (int32_t)(token + offset) / kSegment; }

    // This wave's segments of those from seg0 on: f(first token, logits) for each of a lane's vectors, -inf for what is not the row's, and
    // end(segment) behind each segment.  The next vectors are on their way while some are worked on; the loop over those is not
    // written out, as a workgroup runs it a few times only and fetching its code would cost more.
    template <typename F, typename E>
    __device__ __forceinline__ void each(int32_t seg0, int32_t seg1, F f, E end) const {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int32_t steps = (seg1 - seg0 - wave + kWaves - 1) / kWaves * STEPS;
        auto segment = [&](int32_t q) { return seg0 + wave + kWaves * (q / STEPS); };
        auto vector = [&](int32_t q) { return (segment(q) * STEPS + q % STEPS) * 64 + lane; };
        auto load = [&](int32_t q, u32x4 (&v)[kBatch]) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int32_t at = vector(q + k);
                v[k] = vectors[q + k < steps && at < count ? at : 0];
            }
        };
        u32x4 v[kBatch], next[kBatch];
        load(0, next);
        for (int32_t q0 = 0; q0 < steps; q0 += kBatch) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) v[k] = next[k];
            if (q0 + kBatch < steps) load(q0 + kBatch, next);
#pragma nounroll
            for (int32_t q = q0; q < q0 + kBatch && q < steps; ++q) {
                const int32_t at = vector(q), first = at * kPer - offset, g = segment(q);
                float x[kPer];
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    if constexpr (DT == QK_F32) x[e] = __uint_as_float(v[0][e]);
                    else x[e] = load_half_bits(v[0][e >> 1] >> (16 * (e & 1)) & 0xffffu, DT);
                }
#pragma unroll
                for (int k = 1; k < kBatch; ++k) v[k - 1] = v[k];
                if (!(g * kSegment >= offset && (g + 1) * kSegment - offset <= n)) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) x[e] = (uint32_t)(first + e) < (uint32_t)n ? x[e] : -__builtin_inff();
                }
                f(first, x);
                if (q % STEPS == STEPS - 1) end(g);
            }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(int32_t seg0, int32_t seg1, F f) const {
        each(seg0, seg1, f, [](int32_t) {});
    }
};

// The number of a logit's bin, cut to 32 bits: it rises with the logit, as every step of it does.
__device__ __forceinline__ int32_t bin_at(float x, float per_bin) {
    int32_t at;
    asm("v_cvt_flr_i32_f32 %0, %1" : "=v"(at) : "v"(x * per_bin));
    return at;
}
// The least logit for which `is` holds, which holds for all above it; +inf where it holds for no finite one.  A wave's lanes
// try 64 at a time, first those around `guess`.
template <typename F>
__device__ __forceinline__ float least_logit(float guess, F is) {
    constexpr uint32_t kMost = 0xff800000u;  // +inf
    uint32_t low = kLeast, high = kMost, at = key_of(guess);
    if (at >= kLeast + 64 && at <= kMost - 64) {
        at = at - 32 + (threadIdx.x & 63);
        const uint64_t held = __builtin_amdgcn_ballot_w64(is(value_of(at)));
        at = __builtin_amdgcn_readfirstlane((int)at);
        const int first = held ? __builtin_ctzll(held) : 64;
        if (first > 0) low = at + first;
        if (first < 64) high = at + first;
    }
    while (low < high) {
        const uint32_t step = (high - low + 63) / 64;
        at = low + (threadIdx.x & 63) * step;
        at = at < high ? at : high;
        const uint64_t held = __builtin_amdgcn_ballot_w64(at == high || is(value_of(at)));
        const int first = held ? __builtin_ctzll(held) : 64;
        const uint32_t next = low + first * step;
        if (first > 0) low = next - step + 1;
        if (first < 64 && next < high) high = next;
    }
    return value_of(__builtin_amdgcn_readfirstlane((int)low));
}
// Bins per unit of a logit (near enough to 64 / temperature; the same wherever it is asked for)
__device__ __forceinline__ float bins_per_logit(const Settings& s) { return (float)kPerUnit * __builtin_amdgcn_rcpf(s.temperature); }

// What the look at a row found: it is done (greedy, or nothing to draw), it is done by one workgroup, no filter cuts it, or the border of
// the kept tokens lies among the logits from `listed` to `above`, at which those begin that are kept for certain, `count` of them;
// top_k: 0 where that does not cut; keep: the least logit that min_p keeps.
constexpr int kDone = 0, kAlone = 1, kWhole = 2, kCut = 3;
struct Plan {
    int32_t mode, top_k;
    uint32_t count;
    float top, above, listed, keep;
};
// What a workgroup's look at its part found: the largest logit, the first token that has it (greedy rows), how many could be drawn
// (rows with a histogram).
struct Part {
    float top;
    uint32_t first, valid;
};

struct Look {
    uint64_t bins[kBins + 64];  // count << 40 | weight; behind them, a place for each lane: of what has no bin
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

// A part of a row: its largest logit and, where a filter cuts, its histogram.  Weights there are in units of that of the bin's upper
// end, and near enough: they only have to lead to the border.
template <typename R>
__device__ __forceinline__ Part look_at(const R& row, const Settings& s, bool histogram, int32_t seg0, int32_t seg1, Look& sh, Group& group) {
    constexpr int kPer = R::kPer;
    Part part = {-__builtin_inff(), 0xffffffffu, 0};
    row.each(seg0, seg1, [&](int32_t, const float (&x)[kPer]) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) part.top = fmaxf(part.top, x[e]);
    });
    if (histogram)
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    part.top = group.max(part.top);
    if (s.greedy) {
        row.each(seg0, seg1, [&](int32_t first, const float (&x)[kPer]) {
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (x[e] == part.top && (uint32_t)(first + e) < part.first) part.first = first + e;
        });
        part.first = group.min(part.first);
    }
    if (histogram) {
        const float per_bin = bins_per_logit(s);
        const int32_t top_bin = bin_at(part.top, per_bin);
        const uint32_t past = kBins + (threadIdx.x & 63);
        uint32_t seen = 0, none = 0;  // of this wave
        row.each(seg0, seg1, [&](int32_t, const float (&x)[kPer]) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                // (-inf and NaN come to the least number there is)
                const float v = fmaxf(x[e], -__builtin_inff());
                none += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v == -__builtin_inff()));
                const uint32_t below = (uint32_t)top_bin - (uint32_t)bin_at(v, per_bin), bin = below < past ? below : past;
                // e^-z, z = (1 - f) / 64: on the line that passes it by 2^-15 at most
                const float f = __builtin_amdgcn_fractf(v * per_bin);
                atomicAdd((unsigned long long*)&sh.bins[bin], 1ull << 40 | (uint32_t)__builtin_fmaf(f, 0x1p20f * kSlope, 0x1p20f * (0.99998f - kSlope)));
            }
            seen += 64 * kPer;
        });
        // (the barrier: the histogram is whole behind it)
        part.valid = (uint32_t)group.sum((threadIdx.x & 63) == 0 ? seen - none : 0);
    }
    return part;
}

// The plan of a row that no filter but min_p cuts.
__device__ __forceinline__ Plan plan_of(const Settings& s, float top, int bits) {
    Plan p = {kWhole, 0, 0, top, value_of(kLeast), value_of(kLeast), value_of(kLeast)};
    if (s.min_p > 0.0f) {
        const Weights w = weights_of(s, top, bits);
        const double least = least_of(s);
        p.keep = least_logit(top + s.temperature * (float)least * 0.693147181f, [&](float x) { return w.finite_log2(x) >= least; });
    }
    return p;
}

// The border's bins of a row; bin(b, count, weight) gives the histogram's bin b, its weight in units of its own upper end.
template <typename F>
__device__ Plan plan_row(const Settings& s, float top, int bits, uint32_t valid, Look& sh, Group& group, F bin) {
    constexpr int kOwn = kBins / kThreads;
    const int first = kOwn * threadIdx.x;
    // counts, and weights in units of 2^-22 of the top bin's upper end, as count << 43 | weight
    constexpr int kCount = 43;
    struct Sums {
        uint32_t count;
        uint64_t weight;
    };
    auto apart = [](uint64_t v) { return Sums{(uint32_t)(v >> kCount), v & (((uint64_t)1 << kCount) - 1)}; };
    uint64_t own[kOwn], sum = 0, all;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        uint32_t count;
        float weight;
        bin(first + k, count, weight);
        weight *= __builtin_amdgcn_exp2f((float)(first + k) * (-1.44269504f / kPerUnit)) * 0x1p22f;
        own[k] = (uint64_t)count << kCount | (uint64_t)weight;
        sum += own[k];
    }
    const uint64_t before = group.before(sum, all);
    const bool cuts = s.top_k > 0 && (uint32_t)s.top_k < valid;
    if (threadIdx.x == 0) {
        sh.found[0] = sh.found[1] = sh.found[2] = kBins;
        sh.weight[0] = sh.weight[1] = apart(all).weight;
        sh.above = apart(all).count;
        sh.upto = valid;
    }
    __syncthreads();
    // visit(b, sums before the bin, the bin's): this thread's bins
    auto each = [&](auto visit) {
        uint64_t at = before;
#pragma unroll
        for (int k = 0; k < kOwn; ++k) {
            visit(first + k, apart(at), apart(own[k]));
            at += own[k];
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
    const int32_t low = s.top_p < 1.0f && sh.found[0] < sh.found[2] ? sh.found[0] : sh.found[2];
    int32_t high = cuts ? sh.found[2] : sh.found[1];
    if (high < low) high = low;
    each([&](int b, const Sums& at, const Sums& in) {
        if (b == low) sh.above = at.count;
        if (b == high) sh.upto = at.count + in.count;
    });
    __syncthreads();
    Plan p = plan_of(s, top, bits);
    if (!cuts && !(s.top_p < 1.0f)) return p;
    // (at the end of the numbers there is, -inf shares a bin with logits)
    const float per_bin = bins_per_logit(s);
    const int64_t top_bin = bin_at(top, per_bin);
    p.mode = sh.upto - sh.above > (uint32_t)kList || top_bin < -(1 << 30) ? kAlone : kCut;
    p.top_k = cuts ? s.top_k : 0;
    p.count = sh.above;
    // bins as logits (a bin's number below the top one's by so many; there is none below the last of the 32 bits)
    const float per = s.temperature * (1.0f / kPerUnit);
    p.above = least_logit((float)(top_bin - low + 1) * per, [&](float x) { return bin_at(x, per_bin) > top_bin - low; });
    p.listed = high == kBins ? value_of(kLeast)
                             : least_logit((float)(top_bin - high) * per, [&](float x) { return bin_at(x, per_bin) >= top_bin - high; });
    return p;
}

// A part of a row: exact sums of the weights from `above` on (`all`: of all weights, where top_p asks for them), by segment of those that
// min_p keeps, and the tokens from `listed` up to there, in any order.
struct Drawn {
    uint64_t all, above;
};
template <typename R, typename F>
__device__ __forceinline__ Drawn draw_part(const R& row, const Settings& s, const Weights& w, const Plan& p, int32_t seg0, int32_t seg1, Draw& sh,
                                           Group& group, F segment_sum) {
    constexpr int kPer = R::kPer;
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    const bool cut = p.mode == kCut, min_p = s.min_p > 0.0f;
    const bool whole_sum = cut && s.top_p < 1.0f && p.top_k == 0;
    const bool plain = !cut && !min_p;                   // every logit counts (-inf and NaN: weight 0)
    const float keep = fmaxf(p.keep, p.above), from = cut ? p.above : keep;
    const uint64_t unit = __builtin_bit_cast(uint64_t, w.unit);
    Drawn d = {0, 0};
    uint64_t sum = 0, above = 0, kept = 0;  // sum: with `added` units on top
    uint32_t added = 0;
    row.each(
        seg0, seg1,
        [&](int32_t first, const float (&x)[kPer]) {
            float top = x[0];
#pragma unroll
            for (int e = 1; e < kPer; ++e) top = fmaxf(top, x[e]);
            const bool some = !plain && __builtin_amdgcn_ballot_w64(top >= from);
            auto add = [&](float v, uint64_t raw) {
                above += v >= p.above ? w.whole(raw) : 0;
                if (min_p) kept += v >= keep ? w.whole(raw) : 0;
            };
            if (whole_sum || plain) {
                uint64_t raw[kPer];
#pragma unroll
                for (int e = 0; e < kPer; ++e) raw[e] = w.raw(x[e]);
#pragma unroll
                for (int e = 0; e < kPer; ++e) sum += raw[e];
                added += kPer;
                if (some) {
#pragma unroll
                    for (int e = 0; e < kPer; ++e) add(x[e], raw[e]);
                }
            } else if (some) {
                // a few hundred of a row's tokens: most elements of a vector have none
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (__builtin_amdgcn_ballot_w64(x[e] >= from)) add(x[e], w.raw(x[e]));
            }
            if (cut && top >= p.listed) {
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (x[e] < p.above && x[e] >= p.listed) {
                        const uint32_t at = atomicAdd(&sh.listed, 1u);
                        if (at < (uint32_t)kList) sh.list[at] = place_of(key_of(x[e]), (uint32_t)(first + e));
                    }
            }
        },
        [&](int32_t g) {
            if (plain) {
                above = sum - added * unit;
                sum = 0;
                added = 0;
            }
            const uint64_t of_segment = last_lane(wave_upto(min_p ? kept : above));
            if ((threadIdx.x & 63) == 0) segment_sum(g, of_segment);
            d.above += above;
            above = kept = 0;
        });
    if (cut) {
        d.all = whole_sum ? group.sum(sum - added * unit) : 0;
        d.above = group.sum(d.above);
    } else {
        __syncthreads();
    }
    return d;
}

// v of lane ^ M
template <int M>
__device__ __forceinline__ uint32_t across(uint32_t v) {
    if constexpr (M == 32) {
        const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x & 32) ? a[0] : a[1];
    } else if constexpr (M == 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (threadIdx.x & 16) ? a[0] : a[1];
    } else if constexpr (M == 8) {
        return __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false);
    } else if constexpr (M == 4) {  // lane ^ 7, then ^ 3
        return __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false), 0x1b, 0xf, 0xf, false);
    } else {
        return __builtin_amdgcn_update_dpp(0, (int)v, M == 2 ? 0x4e : 0xb1, 0xf, 0xf, false);
    }
}
// A step of a bitonic sort between lanes: the lower of the pair gets the smaller value where `up`.
template <int M>
__device__ __forceinline__ void sort_step(uint64_t& v, bool up) {
    const uint64_t o = (uint64_t)across<M>((uint32_t)(v >> 32)) << 32 | across<M>((uint32_t)v);
    const bool smaller = ((threadIdx.x & M) == 0) == up;
    v = (o < v) == smaller ? o : v;
}
// Sorts list[0 .. n), n up to N * kThreads: value k of a thread is k * kThreads + its number.  Steps between lanes and between a thread's
// own values are made in registers, those between waves through the list; what lies between n and the next power of two is overwritten.
template <int N>
__device__ __forceinline__ void sort_values(uint64_t* list, uint32_t n) {
    const uint32_t tid = threadIdx.x;
    uint32_t size = 2;
    while (size < n) size *= 2;
    uint64_t v[N];
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k * kThreads + tid < n ? list[k * kThreads + tid] : ~0ull;
    for (uint32_t run = 2; run <= size; run *= 2) {
        auto up = [&](int k) { return ((k * kThreads + tid) & run) == 0; };
#pragma unroll
        for (int apart = N / 2; apart > 0; apart /= 2)
            if (run >= 2u * apart * kThreads) {
#pragma unroll
                for (int k = 0; k < N; ++k)
                    if (!(k & apart)) {
                        const uint64_t a = v[k], b = v[k + apart];
                        const bool swap = (b < a) == up(k);
                        v[k] = swap ? b : a;
                        v[k + apart] = swap ? a : b;
                    }
            }
#pragma nounroll
        for (uint32_t step = run / 2 < kThreads / 2 ? run / 2 : kThreads / 2; step >= 64; step /= 2) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (tid < size) list[k * kThreads + tid] = v[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (tid < size) {
                    const uint64_t o = list[k * kThreads + (tid ^ step)];
                    v[k] = (o < v[k]) == (((tid & step) == 0) == up(k)) ? o : v[k];
                }
        }
        if ((tid & ~63u) >= size) continue;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (run >= 64) sort_step<32>(v[k], up(k));
            if (run >= 32) sort_step<16>(v[k], up(k));
            if (run >= 16) sort_step<8>(v[k], up(k));
            if (run >= 8) sort_step<4>(v[k], up(k));
            if (run >= 4) sort_step<2>(v[k], up(k));
            sort_step<1>(v[k], up(k));
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (tid < size) list[k * kThreads + tid] = v[k];
    __syncthreads();
}
__device__ __forceinline__ void sort_list(uint64_t* list, uint32_t n) {
    static_assert(kList == 4 * kThreads, "");
    if (n <= (uint32_t)kThreads) sort_values<1>(list, n);
    else if (n <= 2u * kThreads) sort_values<2>(list, n);
    else sort_values<4>(list, n);
}

// The token of a row whose parts are together: sh.list holds `listed` tokens, sh.kept the segments' sums.  False: the border is not in
// its bins.
template <typename R>
__device__ __forceinline__ bool draw_row(const SampleArgs& a, int64_t r, const R& row, const Settings& s, const Weights& w, int bits, const Plan& p,
                         const Drawn& d, int32_t segments, uint32_t listed, Draw& sh, Group& group) {
    const int tid = threadIdx.x;
    uint64_t border = ~0ull;  // the last kept token in the sorted row
    if (p.mode == kCut) {
        sort_list(sh.list, listed);
        if (tid == 0) {
            sh.found_k = sh.found_p = -1;
            sh.found_weight = d.all;
        }
        __syncthreads();
        auto weight_at = [&](uint32_t i) { return i < listed ? w.finite(value_of(~(uint32_t)(sh.list[i] >> 32))) : 0; };
        uint64_t all;
        if (p.top_k) {  // the sum of the first top_k
            const uint32_t length = (uint32_t)p.top_k - p.count;
            uint64_t at = 0;
            for (uint32_t i = tid; i < length; i += kThreads) at += weight_at(i);
            at = group.sum(at);
            if (tid == 0 && length > 0 && length <= listed) {
                sh.found_k = (int32_t)length - 1;
                sh.found_weight = d.above + at;
            }
            __syncthreads();
        }
        int32_t last = p.top_k ? sh.found_k : (int32_t)listed - 1;
        bool held = last >= 0;
        if (s.top_p < 1.0f) {
            const uint64_t goal = top_p_goal(s, sh.found_weight);
            uint64_t passed = d.above;
#pragma nounroll
            for (uint32_t base = 0; base < listed; base += kThreads) {
                const uint64_t v = weight_at(base + tid), at = passed + group.before(v, all);
                if (at < goal && goal <= at + v) sh.found_p = base + tid;
                passed += all;
            }
            __syncthreads();
            held = held && sh.found_p >= 0;
            last = sh.found_p < last ? sh.found_p : last;
        }
        if (!held) return false;
        border = sh.list[last];
        for (uint32_t i = tid; (int32_t)i <= last; i += kThreads) {
            const uint64_t v = weight_at(i);
            if (value_of(~(uint32_t)(sh.list[i] >> 32)) >= p.keep)
                atomicAdd((unsigned long long*)&sh.kept[row.segment_of((uint32_t)sh.list[i])], (unsigned long long)v);
        }
    }
    __syncthreads();
    // the segment in which the drawn number falls
    constexpr int kOwn = kSegments / kThreads;
    uint64_t own[kOwn], sum = 0, total;
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
        const int32_t g = tid * kOwn + k;
        own[k] = g < segments ? sh.kept[g] : 0;
        sum += own[k];
    }
    uint64_t at = group.before(sum, total);
    const uint64_t goal = (uint64_t)((double)s.uniform * (double)total) + 1;  // at most total
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
    constexpr int kEach = R::kSegment < kThreads ? 1 : R::kSegment / kThreads;
    const int32_t first = tid * kEach < R::kSegment ? sh.segment * R::kSegment + tid * kEach - row.offset : row.n;
    float x[kEach];
    uint64_t weight[kEach];
    sum = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int32_t i = first + k;
        x[k] = i >= 0 && i < row.n ? load_logit<R::kType>(row.start(), i) : -__builtin_inff();
        weight[k] = x[k] >= p.keep && place_of(key_of(x[k]), (uint32_t)i) <= border ? w.finite(x[k]) : 0;
        sum += weight[k];
    }
    uint64_t in_segment;
    at = sh.found_weight + group.before(sum, in_segment);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        if (at < goal && goal <= at + weight[k]) write_token(a, r, first + k, x[k], w, bits, total);
        at += weight[k];
    }
    return true;
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
template <int DT, int STEPS>
__global__ __launch_bounds__(kThreads, 4) void sample_rows(SampleArgs a, int bits, int32_t segments) {
    __shared__ Space space;
    __shared__ Group::Space shared;
    Group group = {shared};
    const int64_t r = blockIdx.x;
    const Row<DT, STEPS> row(a, r);
    const Settings s = settings_of(a, r);
    const bool histogram = cuts(s, a.vocab) && segments > 0;
    const Part part = look_at(row, s, histogram, 0, row.segments(), space.look, group);
    if (part.top == -__builtin_inff()) return write_plain(a, r, -1);
    if (s.greedy) return write_plain(a, r, (int32_t)part.first);
    Plan p = {kAlone, 0, 0, part.top, 0.0f, 0.0f, 0.0f};
    if (part.top == __builtin_inff() || segments == 0) {
    } else if (!histogram) {
        p = plan_of(s, part.top, bits);
    } else {
        p = plan_row(s, part.top, bits, part.valid, space.look, group, [&](int b, uint32_t& count, float& weight) {
            const uint64_t v = space.look.bins[b];
            count = (uint32_t)(v >> 40);
            weight = (float)(v & ((1ull << 40) - 1)) * 0x1p-20f;
        });
    }
    __syncthreads();  // of the histogram
    bool alone = p.mode == kAlone;
    if (!alone) {
        const Weights w = weights_of(s, p.top, bits);
        const Drawn d = draw_part(row, s, w, p, 0, segments, space.draw, group, [&](int32_t g, uint64_t sum) { space.draw.kept[g] = sum; });
        alone = !draw_row(a, r, row, s, w, bits, p, d, segments, space.draw.listed, space.draw, group);
    }
    if (alone) draw_alone<DT>(a, r, row.start(), s, p.top, bits, space.digits, group);
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

template <int DT, int STEPS>
__global__ __launch_bounds__(kThreads) void sample_look(SplitArgs g) {
    __shared__ Look sh;
    __shared__ Group::Space shared;
    Group group = {shared};
    const SampleArgs& a = g.a;
    const int64_t r = blockIdx.x / (uint32_t)g.groups;
    const int which = (int)(blockIdx.x % (uint32_t)g.groups), tid = threadIdx.x;
    const Row<DT, STEPS> row(a, r);
    const Settings s = settings_of(a, r);
    const bool histogram = cuts(s, a.vocab);
    const int32_t seg0 = which * g.per_group, seg1 = seg0 + g.per_group < g.segments ? seg0 + g.per_group : g.segments;
    const Part part = look_at(row, s, histogram, seg0, seg1, sh, group);
    Part* const parts = g.parts + r * g.groups;
    uint64_t* const bins = g.bins + r * g.groups * kBins;
    if (tid == 0) {
        put(&parts[which].top, part.top);
        put(&parts[which].first, part.first);
        put(&parts[which].valid, part.valid);
    }
    if (histogram)
        for (int i = tid; i < kBins; i += kThreads) put(bins + (int64_t)which * kBins + i, sh.bins[i]);
    if (!splitk_last(g.look_arrivals + r, (uint32_t)g.groups, g.tag)) return;

    // groups: at most a workgroup's threads
    const float own = tid < g.groups ? get(&parts[tid].top) : -__builtin_inff();
    const float top = group.max(own);
    Plan p = {kDone, 0, 0, top, 0.0f, 0.0f, 0.0f};
    if (top == -__builtin_inff()) {
        write_plain(a, r, -1);
    } else if (s.greedy) {
        write_plain(a, r, (int32_t)group.min(own == top ? get(&parts[tid < g.groups ? tid : 0].first) : 0xffffffffu));
    } else if (top == __builtin_inff()) {
        p.mode = kAlone;
    } else if (!histogram) {
        p = plan_of(s, top, g.bits);
    } else {
        const float per_bin = bins_per_logit(s);
        // how far a part's histogram lies below the row's (one without a logit: past it)
        if (tid < g.groups) {
            const uint32_t lower = (uint32_t)bin_at(top, per_bin) - (uint32_t)bin_at(own, per_bin);
            sh.shift[tid] = own > -__builtin_inff() && lower < (uint32_t)kBins ? (int32_t)lower : kBins;
        }
        const uint32_t valid = (uint32_t)group.sum(tid < g.groups ? get(&parts[tid].valid) : 0);  // (its barrier: the shifts are there)
        p = plan_row(s, top, g.bits, valid, sh, group, [&](int b, uint32_t& count, float& weight) {
            count = 0;
            weight = 0.0f;
            for (int c0 = 0; c0 < g.groups; c0 += kAhead) {
                uint64_t v[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int c = c0 + k < g.groups ? c0 + k : c0;
                    const int32_t at = c0 + k < g.groups ? b - sh.shift[c] : -1;
                    v[k] = get(bins + (int64_t)c * kBins + (at < 0 ? 0 : at));
                    if (at < 0) v[k] = 0;
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    count += (uint32_t)(v[k] >> 40);
                    weight += (float)(v[k] & ((1ull << 40) - 1)) * 0x1p-20f;
                }
            }
        });
    }
    if (tid == 0) {
        g.plans[r] = p;
        g.listed[r] = 0;
    }
}

template <int DT, int STEPS>
__global__ __launch_bounds__(kThreads, 4) void sample_draw(SplitArgs g) {
    __shared__ Space space;
    __shared__ Group::Space shared;
    Group group = {shared};
    Draw& sh = space.draw;
    const SampleArgs& a = g.a;
    const int64_t r = blockIdx.x / (uint32_t)g.groups;
    const int which = (int)(blockIdx.x % (uint32_t)g.groups), tid = threadIdx.x;
    const Plan p = g.plans[r];
    if (p.mode == kDone || (p.mode == kAlone && which > 0)) return;
    const Row<DT, STEPS> row(a, r);
    const Settings s = settings_of(a, r);
    bool alone = p.mode == kAlone;
    if (!alone) {
        const Weights w = weights_of(s, p.top, g.bits);
        const int32_t seg0 = which * g.per_group, seg1 = seg0 + g.per_group < g.segments ? seg0 + g.per_group : g.segments;
        uint64_t* const kept = g.kept + r * g.segments;
        uint64_t* const list = g.list + r * kList;
        Drawn* const sums = g.sums + r * g.groups;
        Drawn d = draw_part(row, s, w, p, seg0, seg1, sh, group, [&](int32_t at, uint64_t sum) { put(kept + at, sum); });
        const uint32_t own = sh.listed < (uint32_t)kList ? sh.listed : kList;
        if (tid == 0) {
            put(&sums[which].all, d.all);
            put(&sums[which].above, d.above);
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
        d.all = group.sum(tid < g.groups ? get(&sums[tid].all) : 0);
        d.above = group.sum(tid < g.groups ? get(&sums[tid].above) : 0);
        alone = !draw_row(a, r, row, s, w, g.bits, p, d, g.segments, listed, sh, group);
    }
    if (alone) draw_alone<DT>(a, r, row.start(), s, p.top, g.bits, space.digits, group);
}

// Rows that are looked at as a whole by each of their workgroups, which draw from a part: one launch.  CUT: there may be a top_k or a top_p.
template <int DT, int STEPS, bool CUT>
__global__ __launch_bounds__(kThreads, 4) void sample_parts(SplitArgs g) {
    __shared__ Space space;
    __shared__ Group::Space shared;
    Group group = {shared};
    Draw& sh = space.draw;
    const SampleArgs& a = g.a;
    const int64_t r = blockIdx.x / (uint32_t)g.groups;
    const int which = (int)(blockIdx.x % (uint32_t)g.groups), tid = threadIdx.x;
    const Row<DT, STEPS> row(a, r);
    const Settings s = settings_of(a, r);
    if (s.greedy && which > 0) return;
    const bool histogram = CUT && cuts(s, a.vocab);
    const Part part = look_at(row, s, histogram, 0, g.segments, space.look, group);
    Plan p = {kAlone, 0, 0, part.top, 0.0f, 0.0f, 0.0f};
    if (part.top == -__builtin_inff()) {
        p.mode = kDone;
    } else if (part.top == __builtin_inff()) {
    } else if (!histogram) {
        p = plan_of(s, part.top, g.bits);
    } else {
        p = plan_row(s, part.top, g.bits, part.valid, space.look, group, [&](int b, uint32_t& count, float& weight) {
            const uint64_t v = space.look.bins[b];
            count = (uint32_t)(v >> 40);
            weight = (float)(v & ((1ull << 40) - 1)) * 0x1p-20f;
        });
    }
    // (the same in all of the row's workgroups)
    if (which > 0 && (p.mode == kDone || p.mode == kAlone)) return;
    if (p.mode == kDone) return write_plain(a, r, -1);
    if (s.greedy) return write_plain(a, r, (int32_t)part.first);
    __syncthreads();  // of the histogram
    bool alone = p.mode == kAlone;
    if (!alone) {
        const Weights w = weights_of(s, p.top, g.bits);
        const int32_t seg0 = which * g.per_group, seg1 = seg0 + g.per_group < g.segments ? seg0 + g.per_group : g.segments;
        uint64_t* const kept = g.kept + r * g.segments;
        uint64_t* const list = g.list + r * g.groups * kList;
        Part* const parts = g.parts + r * g.groups;
        Drawn* const sums = g.sums + r * g.groups;
        Drawn d = draw_part(row, s, w, p, seg0, seg1, sh, group, [&](int32_t at, uint64_t sum) { put(kept + at, sum); });
        if (CUT && p.mode == kCut) {
            const uint32_t own = sh.listed < (uint32_t)kList ? sh.listed : kList;
            if (tid == 0) {
                put(&sums[which].all, d.all);
                put(&sums[which].above, d.above);
                put(&parts[which].valid, own);
            }
            for (uint32_t i = tid; i < own; i += kThreads) put(list + (int64_t)which * kList + i, sh.list[i]);
        }
        if (!splitk_last(g.draw_arrivals + r, (uint32_t)g.groups, g.tag)) return;

        uint32_t listed = 0;
        if (CUT && p.mode == kCut) {
            for (int c = 0; c < g.groups; ++c) {
                const uint32_t n = get(&parts[c].valid);
                for (uint32_t i = tid; i < n; i += kThreads)
                    if (listed + i < (uint32_t)kList) sh.list[listed + i] = get(list + (int64_t)c * kList + i);
                listed = listed + n < (uint32_t)kList ? listed + n : kList;
            }
            d.all = group.sum(tid < g.groups ? get(&sums[tid].all) : 0);
            d.above = group.sum(tid < g.groups ? get(&sums[tid].above) : 0);
        }
        for (int32_t i = tid; i < g.segments; i += kThreads) sh.kept[i] = get(kept + i);
        if (!CUT) p.mode = kWhole;  // (it is: told to the compiler)
        alone = !draw_row(a, r, row, s, w, g.bits, p, d, g.segments, listed, sh, group);
    }
    if (alone) draw_alone<DT>(a, r, row.start(), s, p.top, g.bits, space.digits, group);
}

// ---------------------------------------------------------------- host

// F of the weights: the sum of `vocab` of them stays below 2^63.
int weight_bits(int64_t vocab) {
    int bits = 0;
    while (((int64_t)1 << bits) < vocab) ++bits;
    return 62 - bits < 50 ? 62 - bits : 50;
}

// A row is split over workgroups where the parts fill the card once, at most 24 of them (one row of 200000 under all filters: up to 24
// parts 38.8 us, 32 40.0, one for every segment of a wave 47), in one of two ways:
//   apart  look and draw are both dealt, two launches with a join each.  It takes three parts (120 rows of 131072 without filters in two
//          49.0 us, in one launch without parts 43.2), and long rows.
//   whole  one launch, every workgroup looks at the whole row and draws from its part.
// Without top_k and top_p a look is a pass for the largest logit, little beside the exact weights: whole up to 131072 tokens (one row of
// 65536 10.3 us, apart 14.8; of 131072 12.0 and 15.4; of 260000 16.7 and 16.9, in 32 bits 21.1 and 16.4), and where there are two parts (96
// rows of 65536 18.7, in one part 22.1; 128 of 260000 51 and 71); shorter rows than 16384 are done faster in one part (10000: 7.9 and 8.2).
// With them it is a histogram: whole from 28672 to 49152 tokens (48 rows of 32001 under all filters 32.9, in one part 34.7; one 28.6 and
// 29.8; of 20000 26.4 and 24.5; of 65536 39.9, apart 37.2), and in two parts past 98304 (128 rows of 131072 70 and 79; 100 of 65536 51.8 and
// 49.3).
constexpr int64_t kWanted = 256, kLeastApart = 3, kMostGroups = 24;
enum class Way { one, whole, apart };
Way way_of(int64_t rows, int64_t vocab, bool cut) {
    const int64_t groups = kWanted / rows;
    if (vocab > kMostTokens - 8 || groups < 2 || vocab < (cut ? 28672 : 16384)) return Way::one;
    if (vocab <= (cut ? 49152 : 1 << 17)) return Way::whole;
    if (groups >= kLeastApart) return Way::apart;
    return !cut || vocab > 98304 ? Way::whole : Way::one;
}

struct Split {
    // Segments of one vector a lane: few vectors spread over more waves and workgroups (one row of 65536 without filters 15 us, with
    // segments of four 21; of 20000 in one launch 10.7 and 12.6; rows that fill the card alike).
    bool fine;
    int32_t segments, per_group;
    int64_t groups;
    int64_t arrivals, plans, listed, parts, bins, sums, kept, list, bytes;  // offsets in the workspace
};
Split split(int64_t rows, int64_t vocab, int dtype, Way way) {
    Split p = {};
    p.groups = 1;
    if (vocab > kMostTokens - 8) return p;
    const int64_t per = dtype == QK_F32 ? 4 : 8;
    const int64_t most = (vocab + per - 1 + per - 1) / per;  // vectors of a row that begins with the last element of one
    p.fine = most <= 64 * kSegments;
    const int64_t segment = 64 * (p.fine ? 1 : kBatch);
    p.segments = (int32_t)((most + segment - 1) / segment);
    if (way == Way::one) return p;
    const int64_t steps = (p.segments + kWaves - 1) / kWaves;  // of a workgroup that has all
    int64_t groups = kWanted / rows;
    groups = groups < kMostGroups ? groups : kMostGroups;
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
    p.kept = take(rows * p.segments * 8);
    p.parts = take(rows * p.groups * (int64_t)sizeof(Part));
    p.sums = take(rows * p.groups * (int64_t)sizeof(Drawn));
    p.list = take(rows * (way == Way::whole ? p.groups : 1) * kList * 8);
    if (way == Way::whole) return p;
    p.plans = take(rows * (int64_t)sizeof(Plan));
    p.listed = take(rows * 4);
    p.bins = take(rows * p.groups * kBins * 8);
    return p;
}

template <int DT, int STEPS>
hipError_t launch_steps(const SampleArgs& a, const Split& p, Way way, void* workspace, hipStream_t stream) {
    const int bits = weight_bits(a.vocab);
    if (p.groups == 1) {
        sample_rows<DT, STEPS><<<dim3((unsigned)a.rows), kThreads, 0, stream>>>(a, bits, p.segments);
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
    if (way == Way::whole) {
        if (a.top_k || a.top_p) sample_parts<DT, STEPS, true><<<grid, kThreads, 0, stream>>>(g);
        else sample_parts<DT, STEPS, false><<<grid, kThreads, 0, stream>>>(g);
        return hipGetLastError();
    }
    sample_look<DT, STEPS><<<grid, kThreads, 0, stream>>>(g);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    sample_draw<DT, STEPS><<<grid, kThreads, 0, stream>>>(g);
    return hipGetLastError();
}
template <int DT>
hipError_t launch(const SampleArgs& a, void* workspace, hipStream_t stream) {
    const Way way = way_of(a.rows, a.vocab, a.top_k || a.top_p);
    const Split p = split(a.rows, a.vocab, a.dtype, way);
    return p.fine ? launch_steps<DT, 1>(a, p, way, workspace, stream) : launch_steps<DT, kBatch>(a, p, way, workspace, stream);
}

}  // namespace

size_t sample_workspace(int64_t rows, int64_t vocab, int dtype) {
    if (rows == 0) return 0;
    // (which filters there are is not known here)
    const int64_t cut = split(rows, vocab, dtype, way_of(rows, vocab, true)).bytes;
    const int64_t whole = split(rows, vocab, dtype, way_of(rows, vocab, false)).bytes;
    return (size_t)(cut > whole ? cut : whole);
}

hipError_t launch_sample(const SampleArgs& a, void* workspace, hipStream_t stream) {
    if (a.dtype == QK_F32) return launch<QK_F32>(a, workspace, stream);
    if (a.dtype == QK_BF16) return launch<QK_BF16>(a, workspace, stream);
    return launch<QK_F16>(a, workspace, stream);
}

}  // namespace qk
