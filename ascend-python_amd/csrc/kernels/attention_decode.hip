// Attention of one new token per sequence over its pages: s_j = scale * q . k_j, out = sum e^(s_j - m) v_j / sum e^(s_j - m).
//
// Bound by HBM: each visible key and value is read once, 4 * head_dim bytes of a 16-bit cache per token and head for
// 4 * head_dim * (q_heads / kv_heads) operations.  So a workgroup takes all query heads of one key-value head (up to 16: the
// columns of a matrix instruction; more are blocks of their own), and the work is cut along the caches' lengths: the visible
// keys of all sequences and heads, in units of 32, are one line, of which every workgroup takes an equal part, whatever
// the lengths.  They are known on the device only, so each workgroup finds its part from the lengths itself.  A part that ends inside a
// sequence leaves (max, sum, sum of values) in the workspace, and the last of a sequence's workgroups to arrive joins them
// in the order of their parts, so the result does not depend on which it is.
//
// A wave takes 32 keys at a time.  Scores: K (16 keys are the rows) times Q^T (16 heads are the columns), 16x16x32; the
// lane holds four keys of one head, so the running maximum and sum need no exchange between lanes until the end, and the
// weights are, as they lie, the right operand of V^T (rows: 16 elements of the head) times P^T.  V goes through LDS, private to the
// wave, for a transposing read; K comes in the operand's layout from memory.  The next 32 rows and the pages after them are in flight
// while a tile is worked on.
//
// An int8 cache: scores take key_scale as a factor; values are exact in fp16, and the weights take value_scale.  The running
// maximum is that of score plus log2 value_scale, so that the weights with their scales stay in fp16's range.
//
// Measured on one MI355X, inputs that change: 4 x 131072 keys under 64 heads on 8 (2.1 GB) 402 us, 5.3 TB/s; 48 sequences up to
// 8191 (227 MB) 63 us, 3.6 TB/s; 96 on an int8 cache with a window of 4096 (159 MB) 53 us; 997 keys of one sequence 12 us.
#include "attention_device.h"

namespace qk {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kTile = 32;                // keys per wave and step
constexpr int kRound = kWaves * kTile;   // keys that the waves take at a time
// What a sequence costs besides its keys (finding its rows, the join, the output), in units: the first of its stretch of the
// line, which hold no keys (ragged batch: 0 units 111 us, 4 67.2, 8 68.5, 14 70.1).
constexpr int kSegment = 4;
// Parts joined at a time, where there are more than twice as many (8 x 30000 keys of width 256, 32 parts each and more: one join
// of all 83 us, by groups 65; 2 x 20000 keys under 48 heads of one key-value head 162 and 30.6).
constexpr int kGroup = 16;
constexpr int kMostParts = 64;  // and at most: workgroups of a launch / kGroup + 1
constexpr int kMinUnits = kRound / kTile; // units (of kTile keys) per workgroup at least: less is not worth a part of its own
constexpr int kHeads = 16;               // query heads per workgroup

struct DecodeArgs {
    AttnArgs a;
    int blocks_per_group;  // ceil(q_heads / kv_heads / 16)
    bool small;            // the line of units fits 31 bits, and the batch a wave
    uint64_t tag;
    uint64_t* arrivals;    // [batch * kv_heads * blocks_per_group]
    uint64_t* group_arrivals;  // [gridDim][2]
    float* parts;          // [gridDim][2][16 * (width + 2)]
    uint32_t part_bytes;
};

// A workgroup's place in the line of units.
struct Line {
    int64_t total;  // units, of 32 keys, of all sequences and heads
    int64_t begin, end;
    int32_t workers;
};
__device__ __forceinline__ int32_t length_of(const AttnArgs& a, int64_t b) {
    const int64_t most = a.kv.table_width * a.kv.c.page_size, n = a.kv.lens[b];
    return (int32_t)(n < 0 ? 0 : n > most ? most : n);
}
__device__ __forceinline__ int32_t units_of(const AttnArgs& a, int64_t b) {
    const int32_t n = seen_by(length_of(a, b) - 1, a.window, a.sinks).count;
    return kSegment + (n <= 0 ? 1 : (n - 1) / kTile + 1);
}

// KS: 32-wide steps over head_dim; WHOLE: head_dim == 32 * KS; Q8: int8 cache (KS even)
template <int KS, int DT, bool Q8, bool WHOLE>
__global__ __launch_bounds__(kThreads, KS <= 4 ? 3 : KS <= 6 ? 2 : 1) void attention_decode(DecodeArgs g) {
    constexpr int DP = 32 * KS;               // head_dim, padded
    constexpr int NB = DP / 16;               // 16-row blocks of V^T
    constexpr int VROW = DP * 2 + 16;         // bytes of a row of V in LDS
    constexpr int LOADS = Q8 ? KS / 2 : KS;   // 16-byte pieces per lane and row
    constexpr int PV = Q8 ? QK_F16 : DT;      // type of weights and values in the second product
    constexpr int VTILE = kTile * VROW + (Q8 ? 384 : 0);
    constexpr int JOIN = kHeads * DP * 4;     // bytes of a wave's sums when they are joined
    constexpr int WAVE_LDS = VTILE > JOIN ? VTILE : JOIN;
    __shared__ __attribute__((aligned(16))) char lds[kWaves * WAVE_LDS];
    __shared__ float join_m[kWaves][kHeads], join_l[kWaves][kHeads];

    const AttnArgs& a = g.a;
    const qk_kv_cache& c = a.kv.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = lane & 15, kg = lane >> 4;
    const int D = (int)c.head_dim, G = (int)(a.q_heads / c.kv_heads);
    const int64_t head_rows = c.kv_heads * g.blocks_per_group;

    // ---- this workgroup's part of the line, and the sequence that it begins in
    Line line;
    int64_t b, b_start;
    auto part_of = [&](int64_t total) {
        line.total = total;
        const int64_t most = (total + kMinUnits - 1) / kMinUnits;
        line.workers = (int32_t)(most < gridDim.x ? most : gridDim.x);
        line.begin = line_begin(total, line.workers, blockIdx.x);
        line.end = line_begin(total, line.workers, (int64_t)blockIdx.x + 1);
    };
    if (g.small) {  // a lane per sequence, each wave for itself
        const int32_t n = lane < a.batch ? units_of(a, lane) * (int32_t)head_rows : 0;
        const int32_t upto = wave_scan(n);
        part_of(__builtin_amdgcn_readlane(upto, 63));
        if ((int)blockIdx.x >= line.workers) return;
        b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(line.begin < upto));
        b_start = __builtin_amdgcn_readlane(upto - n, (int)b);
    } else {
        __shared__ int64_t scan[kWaves];
        __shared__ int64_t found[2];
        const int64_t per = (a.batch + kThreads - 1) / kThreads;
        const int64_t b_first = tid * per, b_last = b_first + per < a.batch ? b_first + per : a.batch;
        int64_t mine = 0;
        for (int64_t i = b_first; i < b_last; ++i) mine += units_of(a, i);
        int64_t in = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        if (lane == 63) scan[wave] = in;
        __syncthreads();
        for (int w = 0; w < wave; ++w) in += scan[w];
        part_of((int64_t)uniform64(scan[0] + scan[1] + scan[2] + scan[3]) * head_rows);
        if ((int)blockIdx.x >= line.workers) return;
        int64_t at = (in - mine) * head_rows;
        for (int64_t i = b_first; i < b_last; ++i) {
            const int64_t n = units_of(a, i) * head_rows;
            if (at <= line.begin && line.begin < at + n) {
                found[0] = i;
                found[1] = at;
            }
            at += n;
        }
        __syncthreads();
        b = (int64_t)uniform64(found[0]);
        b_start = (int64_t)uniform64(found[1]);
    }

    char* const v_lds = lds + wave * WAVE_LDS;
    float* const s_lds = (float*)(v_lds + kTile * VROW);  // 32 key scales (with the scores' factor), value scales, their log2
    const float factor = a.scale * kLog2e;
    // What finds the rows reads its arguments from memory again each time: some thirty scalar registers, which would otherwise be
    // kept in lanes of vector registers and moved through the vector unit.
    auto args = []() {
        const __attribute__((address_space(4))) DecodeArgs* from =
            (const __attribute__((address_space(4))) DecodeArgs*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(from));
        return from;
    };
    const Global zeros = global_address(kZeroRow);

    for (int64_t u0 = line.begin; u0 < line.end;) {
        int32_t seq_units = units_of(a, b);
        while (u0 >= b_start + seq_units * head_rows) {
            b_start += seq_units * head_rows;
            seq_units = units_of(a, ++b);
        }
        const int64_t hr = quotient(u0 - b_start, seq_units);
        const int64_t first_unit = b_start + hr * seq_units, last_unit = first_unit + seq_units;
        const int64_t u1 = last_unit < line.end ? last_unit : line.end;
        const int kvh = (int)(hr / g.blocks_per_group), blk = (int)(hr % g.blocks_per_group);
        const int heads = G - blk * kHeads < kHeads ? G - blk * kHeads : kHeads;
        const int64_t head0 = (int64_t)kvh * G + blk * kHeads;
        const Seen seen = seen_by(length_of(a, b) - 1, a.window, a.sinks);
        // the stretch begins with units without keys; a workgroup with no others has no part in the sequence
        const int64_t key_unit = first_unit + kSegment;
        if (u1 <= key_unit) {
            u0 = u1;
            continue;
        }
        const int32_t v_begin = u0 <= key_unit ? 0 : (int32_t)(u0 - key_unit) * kTile;
        const int32_t v_end = u1 == last_unit ? seen.count : (int32_t)(u1 - key_unit) * kTile;

        // ---- the query: column `row` of Q^T, elements in the order of K's pieces
        u32x4 q[KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = Q8 ? 64 * (s >> 1) + 16 * kg + 8 * (s & 1) : 32 * s + 8 * kg;
            q[s] = (u32x4){0, 0, 0, 0};
            if (row < heads && (WHOLE || d < D))
                q[s] = *(const u32x4*)((const uint16_t*)a.q + b * a.q_token_stride + (head0 + row) * a.q_head_stride + d);
        }

        f32x4 acc[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = (f32x4){0, 0, 0, 0};
        float m = kLowest, l = 0.0f;
        bool any = false;

        const int32_t* const table = a.kv.table + b * a.kv.table_stride;
        constexpr int ES = Q8 ? 1 : 2;

        // page of this lane's key of each half tile (-1: none), and the key's slot
        auto pages_of = [&](int32_t v0, int32_t (&page)[2], int32_t (&slot)[2]) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int32_t v = v0 + 16 * t + row;
                page[t] = -1;
                slot[t] = 0;
                if (v < v_end) {
                    const int32_t j = v < seen.sinks ? v : v + seen.gap;
                    const int32_t at = div31(j, a.kv.page_div);
                    slot[t] = j - at * (int32_t)c.page_size;
                    page[t] = table[at];
                }
            }
        };
        u32x4 kr[2][LOADS], vr[2][LOADS];
        float ksc[2], vsc[2];
        uint32_t ok[2];  // which of the tile's keys are seen: 16 bits each
        auto load_tile = [&](const int32_t (&page)[2], const int32_t (&slot)[2]) __attribute__((always_inline)) {
            const auto* g = args();
            const auto& c = g->a.kv.c;
            const Global k_base = global_address(c.key) + kvh * c.key_head_stride * ES + 16 * kg;
            const Global v_base = global_address(c.value) + kvh * c.value_head_stride * ES + 16 * kg;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bool valid = page[t] >= 0 && page[t] < c.num_pages;
                ok[t] = (uint32_t)__builtin_amdgcn_ballot_w64(valid) & 0xffffu;
                Global kp = zeros, vp = zeros;
                if (valid) {
                    kp = k_base + (page[t] * c.key_page_stride + slot[t] * c.key_token_stride) * ES;
                    vp = v_base + (page[t] * c.value_page_stride + slot[t] * c.value_token_stride) * ES;
                }
#pragma unroll
                for (int s = 0; s < LOADS; ++s) {
                    Global k1 = kp + 64 * s;
                    Global v1 = vp + 64 * s;
                    if (!WHOLE && 64 * s + 16 * kg >= D * ES) k1 = v1 = zeros;
                    kr[t][s] = load_global<u32x4>(k1);
                    vr[t][s] = load_global<u32x4>(v1);
                }
                if constexpr (Q8) {
                    Global kz = zeros, vz = zeros;
                    if (valid) {
                        kz = global_address(c.key_scale + page[t] * c.key_scale_page_stride + slot[t] * c.key_scale_token_stride +
                                            kvh * c.key_scale_head_stride);
                        vz = global_address(c.value_scale + page[t] * c.value_scale_page_stride + slot[t] * c.value_scale_token_stride +
                                            kvh * c.value_scale_head_stride);
                    }
                    ksc[t] = load_global<float>(kz);
                    vsc[t] = load_global<float>(vz);
                }
            }
        };

        int32_t v0 = v_begin + wave * kTile;
        int32_t page[2], slot[2];
        if (v0 < v_end) {
            pages_of(v0, page, slot);
            load_tile(page, slot);
            pages_of(v0 + kRound, page, slot);
        }
        for (; v0 < v_end; v0 += kRound) {
            int32_t page2[2], slot2[2];
            pages_of(v0 + 2 * kRound, page2, slot2);
            // V to LDS, row-major
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < LOADS; ++s) {
                    char* to = v_lds + (16 * t + row) * VROW;
                    if constexpr (Q8) {
                        const u32x4 w = vr[t][s];
                        *(u32x4*)(to + 128 * s + 32 * kg) = i8_to_f16(w[0], w[1]);
                        *(u32x4*)(to + 128 * s + 32 * kg + 16) = i8_to_f16(w[2], w[3]);
                    } else {
                        *(u32x4*)(to + 64 * s + 16 * kg) = vr[t][s];
                    }
                }
            if constexpr (Q8)
                if (kg == 0) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        s_lds[16 * t + row] = ksc[t] * factor;
                        s_lds[32 + 16 * t + row] = vsc[t];
                        s_lds[64 + 16 * t + row] = __builtin_amdgcn_logf(fmaxf(fabsf(vsc[t]), 0x1p-60f));
                    }
                }
            // scores: lane (head, kg) holds keys 16 t + 4 kg + r
            f32x4 x[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                x[t] = (f32x4){0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 k;
                    if constexpr (Q8) k = i8_to_half<DT>(kr[t][s >> 1][2 * (s & 1)], kr[t][s >> 1][2 * (s & 1) + 1]);
                    else k = kr[t][s];
                    x[t] = Mfma<DT>::mma(k, q[s], x[t]);
                }
            }
            const uint32_t ok0 = ok[0], ok1 = ok[1];
            if (v0 + kRound < v_end) load_tile(page, slot);  // the next tile's rows
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                page[t] = page2[t];
                slot[t] = slot2[t];
            }
            __builtin_amdgcn_sched_barrier(0);
            any |= (ok0 | ok1) != 0;
            f32x4 y[2];  // int8: scores plus log2 of the values' scales: what the running maximum is of
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if constexpr (Q8) {
                    const f32x4 ks = *(const f32x4*)(s_lds + 16 * t + 4 * kg), ls = *(const f32x4*)(s_lds + 64 + 16 * t + 4 * kg);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[t][r] *= ks[r];
                        y[t][r] = x[t][r] + ls[r];
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[t][r] *= factor;
                }
            }
            if ((ok0 & ok1) != 0xffffu) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (!(ok0 >> (4 * kg + r) & 1)) x[0][r] = y[0][r] = -__builtin_inff();
                    if (!(ok1 >> (4 * kg + r) & 1)) x[1][r] = y[1][r] = -__builtin_inff();
                }
            }
            if constexpr (!Q8) {
                y[0] = x[0];
                y[1] = x[1];
            }
            const float top = fmaxf(fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[0][2], y[0][3])),
                                    fmaxf(fmaxf(y[1][0], y[1][1]), fmaxf(y[1][2], y[1][3])));
            if (__builtin_amdgcn_ballot_w64(top > m + (kBelow<PV> + kSlack))) {
                const float m2 = fmaxf(m, quad_max(top) - kBelow<PV>);
                const float keep = __builtin_amdgcn_exp2f(m - m2);
                m = m2;
                l *= keep;
#pragma unroll
                for (int i = 0; i < NB; ++i) acc[i] *= keep;
            }
            // weights, as they lie the right operand of the second product: slot (kg, 4 t + r)
            u32x4 p;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 w, vs;
                if constexpr (Q8) vs = *(const f32x4*)(s_lds + 32 + 16 * t + 4 * kg);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    w[r] = __builtin_amdgcn_exp2f(x[t][r] - m);
                    l += w[r];
                    if constexpr (Q8) w[r] *= vs[r];
                }
                p[2 * t] = pack2<PV>(w[0], w[1]);
                p[2 * t + 1] = pack2<PV>(w[2], w[3]);
            }
            const char* const from = v_lds + (4 * kg + (row >> 2)) * VROW + (row & 3) * 8;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const u32x2 lo = lds_tr16(from + 32 * i), hi = lds_tr16(from + 16 * VROW + 32 * i);
                acc[i] = Mfma<PV>::mma((u32x4){lo[0], lo[1], hi[0], hi[1]}, p, acc[i]);
            }
        }

        // ---- the four waves' results: lane (head = row, kg) holds elements 16 i + 4 kg + r
        l = quad_sum(l);
        if (!any) m = -__builtin_inff();
        __syncthreads();  // the waves are done with V; the sums of the part before have been read
        if (kg == 0) {
            join_m[wave][row] = m;
            join_l[wave][row] = l;
        }
        __syncthreads();
        {
            const float top = fmaxf(fmaxf(join_m[0][row], join_m[1][row]), fmaxf(join_m[2][row], join_m[3][row]));
            const float f = any ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
            if (row < heads) {
#pragma unroll
                for (int i = 0; i < NB; ++i) *(f32x4*)(lds + wave * JOIN + (row * DP + 16 * i + 4 * kg) * 4) = acc[i] * f;
            }
        }
        __syncthreads();
        const bool alone = u0 <= key_unit && u1 == last_unit;
        const int quads = D / 4;
        // max and sum of a head over the waves (max -inf: no key)
        auto joined = [&](int h, float& top, float& sum) {
            top = fmaxf(fmaxf(join_m[0][h], join_m[1][h]), fmaxf(join_m[2][h], join_m[3][h]));
            sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                if (join_m[w][h] != -__builtin_inff()) sum += join_l[w][h] * __builtin_amdgcn_exp2f(join_m[w][h] - top);
        };
        auto sums_at = [&](int h, int d4) {
            f32x4 s = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s += *(const f32x4*)(lds + w * JOIN + (h * DP + 4 * d4) * 4);
            return s;
        };
        auto write_out = [&](int h, int d4, f32x4 s, float top, float sum) {
            const bool none = top == -__builtin_inff();
            const float inv = 1.0f / sum;
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = none ? 0.0f : s[r] * inv;
            const int64_t o = b * a.q_heads + head0 + h;
            *(u32x2*)((uint16_t*)a.out + o * D + 4 * d4) = (u32x2){pack2<DT>(s[0], s[1]), pack2<DT>(s[2], s[3])};
            if (d4 == 0 && a.lse) a.lse[o] = none ? top : (top + __builtin_amdgcn_logf(sum)) * kLn2;
        };
        if (alone) {
            for (int i = tid; i < heads * quads; i += kThreads) {
                const int h = i / quads, d4 = i % quads;
                float top, sum;
                joined(h, top, sum);
                write_out(h, d4, sums_at(h, d4), top, sum);
            }
        } else {
            constexpr uint32_t SLOT = kHeads * (DP + 2) * 4;  // sums, then max and sum of each head
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(g.parts, g.part_bytes);
            const uint32_t mine_at = (2 * blockIdx.x + (first_unit > line.begin)) * SLOT;
            for (int i = tid; i < heads * quads; i += kThreads) {
                const int h = i / quads, d4 = i % quads;
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sums_at(h, d4)), rs, mine_at + (h * DP + 4 * d4) * 4, 0, kCoherent);
            }
            if (tid < heads) {
                float top, sum;
                joined(tid, top, sum);
                __builtin_amdgcn_raw_buffer_store_b64((u32x2){__float_as_uint(top), __float_as_uint(sum)}, rs,
                                                      mine_at + (kHeads * DP + 2 * tid) * 4, 0, kCoherent);
            }
            const int64_t w0 = worker_of(line.total, line.workers, key_unit);
            const int n = (int)(worker_of(line.total, line.workers, last_unit - 1) - w0 + 1);
            // where the parts are: the first may be the second slot of its worker
            const uint32_t slot0 = 2 * (uint32_t)w0 + (line_begin(line.total, line.workers, w0) < first_unit);
            auto slot_of = [&](int k) { return k == 0 ? slot0 : 2 * ((uint32_t)w0 + k); };
            // Joins `count` of them, every `step`-th from `first` on, in their order.  emit(head, quad, sums, max, sum).
            auto join = [&](int first, int count, int step, auto emit) {
                float* const pm = (float*)lds;  // [count][kHeads] maxima, then as many sums
                float* const pl = pm + kMostParts * kHeads;
                __syncthreads();
                for (int i = tid; i < count * kHeads; i += kThreads) {
                    const u32x2 ml = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(
                                                                   rs, slot_of(first + i / kHeads * step) * SLOT + (kHeads * DP + 2 * (i % kHeads)) * 4, 0, kCoherent));
                    pm[i] = __uint_as_float(ml[0]);
                    pl[i] = __uint_as_float(ml[1]);
                }
                __syncthreads();
                for (int i = tid; i < heads * quads; i += kThreads) {
                    const int h = i / quads, d4 = i % quads;
                    float top = -__builtin_inff(), sum = 0.0f;
                    for (int k = 0; k < count; ++k) top = fmaxf(top, pm[k * kHeads + h]);
                    f32x4 s = {0, 0, 0, 0};
                    for (int k0 = 0; k0 < count; k0 += 8) {
                        f32x4 v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (k0 + k < count)
                                v[k] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                                                     rs, slot_of(first + (k0 + k) * step) * SLOT + (h * DP + 4 * d4) * 4, 0, kCoherent));
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (k0 + k < count) {
                                const float m1 = pm[(k0 + k) * kHeads + h];
                                if (m1 == -__builtin_inff()) continue;
                                const float f = __builtin_amdgcn_exp2f(m1 - top);
                                sum += pl[(k0 + k) * kHeads + h] * f;
                                s += v[k] * f;
                            }
                    }
                    emit(h, d4, s, top, sum);
                }
            };
            if (n <= 2 * kGroup) {
                if (splitk_last(g.arrivals + b * head_rows + hr, (uint32_t)n, g.tag)) join(0, n, 1, write_out);
            } else {
                // in two steps: the last of a group of parts leaves their join in the group's first, the last group joins those
                const int mine = (int)(blockIdx.x - w0) / kGroup, members = n - mine * kGroup < kGroup ? n - mine * kGroup : kGroup;
                if (splitk_last(g.group_arrivals + slot_of(mine * kGroup), (uint32_t)members, g.tag)) {
                    const uint32_t at = slot_of(mine * kGroup) * SLOT;
                    join(mine * kGroup, members, 1, [&](int h, int d4, f32x4 s, float top, float sum) {
                        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, s), rs, at + (h * DP + 4 * d4) * 4, 0, kCoherent);
                        if (d4 == 0)
                            __builtin_amdgcn_raw_buffer_store_b64((u32x2){__float_as_uint(top), __float_as_uint(sum)}, rs,
                                                                  at + (kHeads * DP + 2 * h) * 4, 0, kCoherent);
                    });
                    const int groups = (n + kGroup - 1) / kGroup;
                    if (splitk_last(g.arrivals + b * head_rows + hr, (uint32_t)groups, g.tag)) join(0, groups, kGroup, write_out);
                }
            }
        }
        u0 = u1;
        __syncthreads();  // the sums in LDS have been read
    }
}

struct Plan {
    int64_t grid, arrivals_bytes, part_bytes;
    int blocks_per_group, ks;
    bool small;
};

// Padded widths that have a kernel, in 32-wide steps
int steps_of(const qk_kv_cache& c) {
    const int n = (int)((c.head_dim + 31) / 32);
    if (n <= 2) return 2;
    if (n <= 4) return n == 3 && c.dtype != QK_I8 ? 3 : 4;
    return n <= 6 ? 6 : 8;
}

Plan plan(int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width, int64_t window, int64_t sinks) {
    Plan p = {};
    const int64_t group = q_heads / c.kv_heads;
    p.blocks_per_group = (int)((group + kHeads - 1) / kHeads);
    p.ks = steps_of(c);
    int64_t most = table_width * c.page_size;
    if (window && most > window && most - window > sinks) most = window + sinks;
    const int64_t units = kSegment + (most < 1 ? 1 : (most + kTile - 1) / kTile);
    const int64_t rows = batch * c.kv_heads * p.blocks_per_group;
    // as many workgroups as are resident at once: three per CU, two of wide heads, one of the widest (twice as many: 4 x 131072
    // keys 401 -> 438 us, the ragged batch 64 -> 73; two per CU: 424 and 65, int8 54 -> 63)
    const int64_t resident = 256 * (p.ks <= 4 ? 3 : p.ks <= 6 ? 2 : 1);
    // no more than the line can occupy
    const int64_t parts = units > (resident * kMinUnits) / rows ? resident : (units * rows + kMinUnits - 1) / kMinUnits;
    p.grid = parts < resident ? parts : resident;
    p.small = batch <= 64 && units < ((int64_t)1 << 31) / (rows + 1);
    p.arrivals_bytes = ((rows + 2 * p.grid) * 8 + 255) / 256 * 256;
    p.part_bytes = p.grid * 2 * kHeads * (32 * p.ks + 2) * 4;
    return p;
}

template <int KS, int DT, bool Q8>
void launch_width(const DecodeArgs& g, int64_t grid, hipStream_t stream) {
    if (g.a.kv.c.head_dim == 32 * KS) attention_decode<KS, DT, Q8, true><<<dim3((unsigned)grid), kThreads, 0, stream>>>(g);
    else attention_decode<KS, DT, Q8, false><<<dim3((unsigned)grid), kThreads, 0, stream>>>(g);
}
template <int DT, bool Q8>
void launch_type(const DecodeArgs& g, const Plan& p, hipStream_t stream) {
    switch (p.ks) {
    case 2: return launch_width<2, DT, Q8>(g, p.grid, stream);
    case 3:
        if constexpr (!Q8) return launch_width<3, DT, Q8>(g, p.grid, stream);
        return;
    case 4: return launch_width<4, DT, Q8>(g, p.grid, stream);
    case 6: return launch_width<6, DT, Q8>(g, p.grid, stream);
    default: return launch_width<8, DT, Q8>(g, p.grid, stream);
    }
}

}  // namespace

size_t attention_decode_workspace(int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width, int64_t window,
                                  int64_t sinks) {
    if (batch == 0) return 0;
    const Plan p = plan(batch, q_heads, c, table_width, window, sinks);
    return (size_t)(p.arrivals_bytes + p.part_bytes);
}

hipError_t launch_attention_decode(const AttnArgs& a, void* workspace, hipStream_t stream) {
    const Plan p = plan(a.batch, a.q_heads, a.kv.c, a.kv.table_width, a.window, a.sinks);
    DecodeArgs g = {};
    g.a = a;
    g.blocks_per_group = p.blocks_per_group;
    g.small = p.small;
    g.tag = next_split_tag();
    g.arrivals = (uint64_t*)workspace;
    g.group_arrivals = g.arrivals + a.batch * a.kv.c.kv_heads * p.blocks_per_group;
    g.parts = (float*)((char*)workspace + p.arrivals_bytes);
    g.part_bytes = (uint32_t)p.part_bytes;
    const bool q8 = a.kv.c.dtype == QK_I8;
    if (a.dtype == QK_BF16) {
        if (q8) launch_type<QK_BF16, true>(g, p, stream);
        else launch_type<QK_BF16, false>(g, p, stream);
    } else {
        if (q8) launch_type<QK_F16, true>(g, p, stream);
        else launch_type<QK_F16, false>(g, p, stream);
    }
    return hipGetLastError();
}

}  // namespace qk
