// Rotary positions of one to four axes, with the write of the new keys and values into the paged cache, on gfx950.
//
// For pair i of a head: y0 = x0 c - x1 s, y1 = x1 c + x0 s, c and s from row positions[a(i)][t] of the table.  The table
// holds the cosines themselves, so a far position loses nothing here.  Arithmetic is fp32, every product and sum rounded
// by itself; one rounding to 16 bits.  An int8 cache quantizes that 16-bit row as npu_dynamic_quant would, so the chain
// of ops and this kernel give the same bits.
//
// Bound by HBM: 2 bytes read and 2 written per element of q, k and v.  A lane owns eight pairs of a head (two 16-byte
// pieces, rotary_dim / 2 apart; interleaved: one piece of four pairs), so a head of 128 is eight lanes and a wave
// instruction covers whole 128-byte lines.  The cosines depend on the token and the pair alone: a workgroup takes
// one token, loads its 16 factors per lane once and walks the heads with them.  In a decode batch there are few tokens, so
// the heads of a token are spread over workgroups too (one pass each).
#include "attention.h"

namespace qk {
namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float table_at(const MropeArgs& a, int64_t i) {
    return a.cos_sin_dtype == QK_F32 ? ((const float*)a.cos_sin)[i] : load_half_bits(((const uint16_t*)a.cos_sin)[i], a.dtype);
}

// cos and sin of pair i at token t; NaN where the position lies outside the table
__device__ __forceinline__ void turn_of(const MropeArgs& a, int64_t t, int i, float& c, float& s) {
    int ax = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k) ax += k + 1 < a.axes && i >= a.section_end[k];
    const int32_t p = a.positions[ax * a.position_stride + t];
    c = s = __builtin_nanf("");
    if (p >= 0 && p < a.table_rows) {
        c = table_at(a, p * a.rotary_dim + i);
        s = table_at(a, p * a.rotary_dim + a.rotary_dim / 2 + i);
    }
}

// cos and sin of N pairs from `first` on (N a multiple of 4 that divides it): two runs of the table's row where they lie in one
// section, as they all but always do.  `whole`: the table is fp32, its rows whole 16-byte pieces.
template <int N>
__device__ __forceinline__ void turns_of(const MropeArgs& a, int64_t t, int first, bool whole, float (&c)[N], float (&s)[N]) {
    int ax = 0, last = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        ax += k + 1 < a.axes && first >= a.section_end[k];
        last += k + 1 < a.axes && first + N - 1 >= a.section_end[k];
    }
    if (whole && ax == last) {
        const int32_t p = a.positions[ax * a.position_stride + t];
        if (p >= 0 && p < a.table_rows) {
            const float* const row = (const float*)a.cos_sin + p * a.rotary_dim + first;
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const f32x4 vc = *(const f32x4*)(row + i), vs = *(const f32x4*)(row + a.rotary_dim / 2 + i);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    c[i + k] = vc[k];
                    s[i + k] = vs[k];
                }
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) turn_of(a, t, first + i, c[i], s[i]);
}

__device__ __forceinline__ uint32_t to_bits(float v, int dtype) {
    return dtype == QK_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
}

// Where a head of a token goes: the out tensors, and for keys and values their slot of the cache (or none).
struct Place {
    int64_t page, slot;
    bool cached;
};
__device__ __forceinline__ Place place_of(const MropeArgs& a, int64_t t) {
    Place p = {0, 0, false};
    if (a.cached) {
        const int32_t s = a.slots[t];
        if (s >= 0 && s < a.c.num_pages * a.c.page_size) {
            const int32_t page = div31(s, a.page_div);
            p = {page, s - page * a.c.page_size, true};
        }
    }
    return p;
}

// Where head h is read: the query's heads, then the keys', then the values'.
__device__ __forceinline__ const uint16_t* source_of(const MropeArgs& a, int64_t t, int h) {
    const int Hq = (int)a.q_heads, Hkv = (int)a.kv_heads;
    if (h < Hq) return (const uint16_t*)a.q + t * a.q_token_stride + h * a.q_head_stride;
    if (h < Hq + Hkv) return (const uint16_t*)a.k + t * a.k_token_stride + (h - Hq) * a.k_head_stride;
    return (const uint16_t*)a.v + t * a.v_token_stride + (h - Hq - Hkv) * a.v_head_stride;
}
// ... and where it goes
struct Head {
    uint16_t* out;       // 16-bit result, or null
    uint16_t* out2;      // a second one (the key's own tensor beside a 16-bit cache), or null
    int8_t* quant;       // int8 cache row, or null
    float* quant_scale;
};
__device__ __forceinline__ Head head_of(const MropeArgs& a, int64_t t, int h, const Place& p) {
    const int Hq = (int)a.q_heads, Hkv = (int)a.kv_heads;
    Head r = {};
    if (h < Hq) {
        r.out = a.out_q ? (uint16_t*)a.out_q + (t * Hq + h) * a.head_dim : nullptr;
        return r;
    }
    const bool key = h < Hq + Hkv;
    const int g = h - Hq - (key ? 0 : Hkv);
    if (key && a.out_k) r.out = (uint16_t*)a.out_k + (t * Hkv + g) * a.head_dim;
    if (p.cached) {
        const qk_kv_cache& c = a.c;
        const int64_t row = key ? p.page * c.key_page_stride + p.slot * c.key_token_stride + g * c.key_head_stride
                                : p.page * c.value_page_stride + p.slot * c.value_token_stride + g * c.value_head_stride;
        if (c.dtype == QK_I8) {
            r.quant = (int8_t*)(key ? c.key : c.value) + row;
            r.quant_scale = key ? c.key_scale + p.page * c.key_scale_page_stride + p.slot * c.key_scale_token_stride +
                                      g * c.key_scale_head_stride
                                : c.value_scale + p.page * c.value_scale_page_stride +
                                      p.slot * c.value_scale_token_stride + g * c.value_scale_head_stride;
        } else {
            (r.out ? r.out2 : r.out) = (uint16_t*)(key ? c.key : c.value) + row;
        }
    }
    return r;
}

// Eight 16-bit values <-> fp32
__device__ __forceinline__ void unpack8(u32x4 w, int dtype, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = load_half_bits(w[i] & 0xffffu, dtype);
        v[2 * i + 1] = load_half_bits(w[i] >> 16, dtype);
    }
}
__device__ __forceinline__ u32x4 pack8(const float (&v)[8], int dtype) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = to_bits(v[2 * i], dtype) | (to_bits(v[2 * i + 1], dtype) << 16);
    return w;
}

// Pieces of 16 bytes: a unit is two pieces of the first rotary_dim elements (interleaved: one), then one piece of the
// rest.  `lanes` (a power of two, at most 32) lanes hold a head.  The first pass's rows are asked for before the
// factors, whose addresses wait for the positions; more passes ahead cost registers, and with them waves (4099 tokens with
// three axes: none ahead but the first 22.0 us, 4.6 TB/s; two 24.0; four 25.9).
template <bool INTER>
__global__ __launch_bounds__(kThreads) void mrope_vec(MropeArgs a, int lanes, int units, int heads, int passes, bool whole) {
    constexpr int N = INTER ? 4 : 8;  // pairs of a lane
    const int64_t t = blockIdx.x;
    const int u = threadIdx.x & (lanes - 1), per = kThreads / lanes;
    const int half = (int)a.rotary_dim / 2;
    const int turning = half / N;
    const bool two = !INTER && u < turning;
    const int first = u < turning ? 8 * u : (int)a.rotary_dim + 8 * (u - turning);
    const int second = first + half;  // read only where `two`
    const int per_pass = per * gridDim.y, h0 = blockIdx.y * per + threadIdx.x / lanes;

    u32x4 in0, in1;
    auto ask = [&](int h) {
        in0 = in1 = (u32x4){0, 0, 0, 0};
        if (h < heads && u < units) {
            const uint16_t* const from = source_of(a, t, h);
            in0 = *(const u32x4*)(from + first);
            if (two) in1 = *(const u32x4*)(from + second);
        }
    };
    ask(h0);
    const Place place = place_of(a, t);
    float c[N], s[N];
    if (u < turning) turns_of<N>(a, t, N * u, whole, c, s);

    for (int pass = 0; pass < passes; ++pass) {
        const int h = h0 + pass * per_pass;
        if (pass) ask(h);
        const bool on = h < heads && u < units;
        Head hd = {};
        float x[8] = {}, y[8] = {};
        u32x4 w0 = in0, w1 = in1;
        if (on) {
            hd = head_of(a, t, h, place);
            if (h < a.q_heads + a.kv_heads && u < turning) {
                unpack8(w0, a.dtype, x);
                if constexpr (!INTER) {
                    unpack8(w1, a.dtype, y);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float x0 = x[i], x1 = y[i];
                        x[i] = x0 * c[i] - x1 * s[i];
                        y[i] = x1 * c[i] + x0 * s[i];
                    }
                    w1 = pack8(y, a.dtype);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x0 = x[2 * i], x1 = x[2 * i + 1];
                        x[2 * i] = x0 * c[i] - x1 * s[i];
                        x[2 * i + 1] = x1 * c[i] + x0 * s[i];
                    }
                }
                w0 = pack8(x, a.dtype);
            }
            if (hd.out) {
                *(u32x4*)(hd.out + first) = w0;
                if (two) *(u32x4*)(hd.out + second) = w1;
            }
            if (hd.out2) {
                *(u32x4*)(hd.out2 + first) = w0;
                if (two) *(u32x4*)(hd.out2 + second) = w1;
            }
        }
        if (a.cached && a.c.dtype == QK_I8) {
            float amax = 0.0f;
            if (hd.quant) {
                unpack8(w0, a.dtype, x);
                unpack8(w1, a.dtype, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(x[i]), two ? fabsf(y[i]) : 0.0f));
            }
            for (int d = 1; d < lanes; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
            if (hd.quant) {
                const RowQuant rq = row_quant(amax / 127.0f);
                *(u32x2*)(hd.quant + first) = quant8(x, rq);
                if (two) *(u32x2*)(hd.quant + second) = quant8(y, rq);
                if (u == 0) *hd.quant_scale = rq.s;
            }
        }
    }
}

// Any rotary_dim and alignment: a wave per head, a lane per pair (or per element past rotary_dim).
__global__ __launch_bounds__(kThreads) void mrope_any(MropeArgs a, int heads) {
    const int lane = threadIdx.x & 63;
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6);
    if (h >= heads) return;
    const Head hd = head_of(a, t, h, place_of(a, t));
    const uint16_t* const from = source_of(a, t, h);
    const bool rotate = h < a.q_heads + a.kv_heads;
    const int D = (int)a.head_dim, R = (int)a.rotary_dim, half = R / 2;
    const int units = half + D - R;
    uint32_t b0[4], b1[4];
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int u = lane + 64 * i;
        b0[i] = b1[i] = 0;
        if (u >= units) continue;
        const bool pair = u < half;
        const int e0 = !pair ? R + u - half : a.interleave ? 2 * u : u, e1 = a.interleave ? e0 + 1 : e0 + half;
        b0[i] = from[e0];
        if (pair) b1[i] = from[e1];
        if (pair && rotate) {
            float c, s;
            turn_of(a, t, u, c, s);
            const float x0 = load_half_bits(b0[i], a.dtype), x1 = load_half_bits(b1[i], a.dtype);
            b0[i] = to_bits(x0 * c - x1 * s, a.dtype);
            b1[i] = to_bits(x1 * c + x0 * s, a.dtype);
        }
        amax = fmaxf(amax, fmaxf(fabsf(load_half_bits(b0[i], a.dtype)), fabsf(load_half_bits(b1[i], a.dtype))));
    }
    amax = wave_max(amax);
    const RowQuant rq = row_quant(amax / 127.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int u = lane + 64 * i;
        if (u >= units) continue;
        const bool pair = u < half;
        const int e0 = !pair ? R + u - half : a.interleave ? 2 * u : u, e1 = a.interleave ? e0 + 1 : e0 + half;
        if (hd.out) {
            hd.out[e0] = (uint16_t)b0[i];
            if (pair) hd.out[e1] = (uint16_t)b1[i];
        }
        if (hd.out2) {
            hd.out2[e0] = (uint16_t)b0[i];
            if (pair) hd.out2[e1] = (uint16_t)b1[i];
        }
        if (hd.quant) {
            hd.quant[e0] = (int8_t)quant_row(load_half_bits(b0[i], a.dtype), rq);
            if (pair) hd.quant[e1] = (int8_t)quant_row(load_half_bits(b1[i], a.dtype), rq);
        }
    }
    if (hd.quant && lane == 0) *hd.quant_scale = rq.s;
}

bool whole_pieces(const void* p, int64_t token_stride, int64_t head_stride) {
    return !p || ((uintptr_t)p % 16 == 0 && token_stride % 8 == 0 && head_stride % 8 == 0);
}

}  // namespace

hipError_t launch_mrope(const MropeArgs& a, hipStream_t stream) {
    const int heads = (int)(a.q_heads + a.kv_heads * (a.v ? 2 : 1));
    const int D = (int)a.head_dim, R = (int)a.rotary_dim;
    const bool vec = D % 8 == 0 && R % (a.interleave ? 8 : 16) == 0 && whole_pieces(a.q, a.q_token_stride, a.q_head_stride) &&
                     whole_pieces(a.k, a.k_token_stride, a.k_head_stride) &&
                     whole_pieces(a.v, a.v_token_stride, a.v_head_stride) && whole_pieces(a.out_q, 0, 0) &&
                     whole_pieces(a.out_k, 0, 0);
    if (!vec) {
        mrope_any<<<dim3((unsigned)a.tokens, (unsigned)((heads + 1) / 2)), kThreads, 0, stream>>>(a, heads);
        return hipGetLastError();
    }
    const int units = (a.interleave ? R / 8 : R / 16) + (D - R) / 8;
    int lanes = 1;
    while (lanes < units) lanes *= 2;
    const int per = kThreads / lanes;
    int passes = (heads + per - 1) / per, spread = 1;
    // two workgroups per CU at least, as long as there are heads to spread
    while (passes > 1 && a.tokens * spread < 512) {
        ++spread;
        passes = (heads + per * spread - 1) / (per * spread);
    }
    const bool whole = a.cos_sin_dtype == QK_F32 && (uintptr_t)a.cos_sin % 16 == 0;
    const dim3 grid((unsigned)a.tokens, (unsigned)spread);
    if (a.interleave) mrope_vec<true><<<grid, kThreads, 0, stream>>>(a, lanes, units, heads, passes, whole);
    else mrope_vec<false><<<grid, kThreads, 0, stream>>>(a, lanes, units, heads, passes, whole);
    return hipGetLastError();
}

}  // namespace qk
