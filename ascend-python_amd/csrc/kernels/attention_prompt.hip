// Causal attention of ragged prompts: s_j = scale * q . k_j over the keys that a row sees, out = sum e^(s_j - m) v_j / sum e^(s_j - m).
//
// Bound by the matrix cores: 4 * head_dim operations per visible pair and query head.  A workgroup takes 128 rows of one
// key-value head and sequence, a row being a (token, query head of the group) pair, token first: so a tile of a group of four
// spans 32 tokens, its causal edge is short, and every key read serves the whole group.  It walks the keys that any of
// its rows sees 64 at a time, each of the four waves with 32 rows.
//
// Scores: K (32 keys are the rows) times Q^T (32 rows are the columns), 32x32x16: the lane holds 16 keys of one row, so
// maximum and sum need one exchange between lane pairs, and the weights as they lie are the right operand of V^T times P^T.
// K and V go straight from memory into two LDS buffers (an int8 cache through registers, where it becomes 16-bit), the 16-byte
// pieces of a row exchanged so that neither the reads of K nor the transposing reads of V meet in a bank.  One barrier per
// 64 keys: the next rows are on their way while these are worked on.  Where the rows of the cache lie is found for four
// tiles at a time, ahead of them.
//
// The next tile's scores are made between the exponentials of this one, so that a wave keeps both pipes busy.  The running
// maximum moves only where a score lies far above it: most tiles rescale nothing and need no exchange between lanes.
//
// Measured on one MI355X: 8192 tokens under 32 heads on 8 540 us, 1.0 PFLOP/s (on random data the card is held back by its power:
// 500 us on zeros); 2048 tokens 54 us; six chunks up to 1023 tokens over 12000 with a window of 2048 56 us; 4 tokens over
// 12000 33 us; 77 tokens 10 us.
//
// A masked weight is 0, but 0 times a NaN or an infinity in V is NaN: tiles that are masked for some rows look for such
// values once they are staged, and the values are added apart, for the rows that see them, with the weight that the products
// would take: an infinity whose weight rounds to 0 gives NaN in every tile.
#include <type_traits>

#include "attention_device.h"

namespace qk {
namespace {

// The parts of the kernel are lambdas, some of them used in several places: none may become a function.
#define INLINE __attribute__((always_inline))

constexpr int kThreads = 256;
constexpr int kRows = 128;   // query rows per workgroup
constexpr int kKeys = 64;    // keys per tile
// A tile's keys are cut, where there are few tiles, into parts of at least so many steps: a part costs its write and its
// share of the join (4 tokens over 12000: parts of eight steps 33.6 us, of four 36.8).
constexpr int kSplitTiles = 8;
// Workgroups that the card holds, two per CU; cutting up to 768 or 1024 takes longer where tiles are nearly enough (1500
// tokens 41.5 -> 46.9 us, chunks with a window 64 -> 69).
constexpr int64_t kResident = 512;
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    typedef typename Mfma<DT>::v8 v8;
    if constexpr (DT == QK_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

// 16 bytes from LDS address `at` + offset; and 8 of them as lds_tr16
__device__ __forceinline__ u32x4 lds_load(uint32_t at, int offset) {
    return *(const __attribute__((address_space(3))) u32x4*)((const __attribute__((address_space(3))) char*)(uintptr_t)at + offset);
}
__device__ __forceinline__ u32x2 lds_tr16(uint32_t at, int offset) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) i16x4*)((__attribute__((address_space(3))) char*)(uintptr_t)at + offset)));
}

// v, as a value that is made here: what follows from it is not computed ahead of the loop, where it would hold registers.
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// 16 bytes per lane from memory into LDS bytes [lds + 16 * lane, +16); the kernel waits on vmcnt itself (as dma16).
__device__ __forceinline__ void global_to_lds(Global from, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(from), "{m0}"(lds));
}

struct PromptArgs {
    AttnArgs a;
    Div31 group_div;  // q_heads / kv_heads
    int splits;       // at most: parts that a tile's keys are cut into
    uint64_t tag;
    uint64_t* arrivals;   // a counter for every tile and key-value head
    float* parts;         // [tile and head][splits][kRows * (DP + 2)], in the order of the registers
    int64_t part_bytes;   // of one of them
};

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

// Largest value, and sum, over lanes l and l ^ 32.
__device__ __forceinline__ float pair_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

__device__ __forceinline__ float largest(const f32x16 (&x)[2]) {
    float top = x[0][0];
#pragma unroll
    for (int e = 1; e < 16; ++e) top = __builtin_elementwise_maximum(top, x[0][e]);
#pragma unroll
    for (int e = 0; e < 16; ++e) top = __builtin_elementwise_maximum(top, x[1][e]);
    return top;
}

// DP: head_dim padded to 32s; WHOLE: head_dim == DP; Q8: int8 cache
template <int DP, int DT, bool Q8, bool WHOLE>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void attention_prompt(PromptArgs g) {
    constexpr int KS = DP / 16;                  // steps of the first product
    constexpr int NB = DP / 32;                  // 32-row blocks of V^T
    constexpr int LS = DP <= 64 ? 128 : DP <= 128 ? 256 : 512;  // bytes of a row in LDS
    constexpr int CHL = LS / 16;                 // 16-byte pieces of it
    constexpr int ES = Q8 ? 1 : 2;
    constexpr int CH = DP * ES / 16;             // 16-byte pieces of a cache row
    constexpr int PIECES = Q8 ? kKeys * CH / kThreads : 1;  // int8: per thread
    constexpr int DMAS = CHL / 4;                // 16-bit: 1 KB loads per wave for K, and for V
    constexpr int PV = Q8 ? QK_F16 : DT;
    static_assert(!Q8 || kKeys * CH % kThreads == 0, "");
    constexpr int TILE = kKeys * LS;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];  // buffer 0: K, V; buffer 1: K, V
    __shared__ __attribute__((aligned(16))) uint64_t info[8][kKeys][2];  // addresses of a key's and a value's row (none: of zeros)
    __shared__ uint64_t info_ok[8];              // which keys of the tile exist
    __shared__ uint64_t bad[3];                  // which rows of V hold a NaN or an infinity
    __shared__ float scales[8][3][kKeys];         // int8: of the scores (with log2 e), of the values, and the latter's log2
    __shared__ int64_t found[2];

    const AttnArgs& a = g.a;
    const qk_kv_cache& c = a.kv.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, kg = lane >> 5;
    const int D = (int)c.head_dim, G = (int)(a.q_heads / c.kv_heads);
    const int kvh = (int)(blockIdx.x % (uint32_t)c.kv_heads);

    // ---- which tile: those of all sequences in a line, the last first (the longest of a prompt come first)
    {
        const int64_t per = (a.batch + 1 + kThreads - 1) / kThreads;
        const int64_t b0 = tid * per, b1 = b0 + per < a.batch + 1 ? b0 + per : a.batch + 1;
        int64_t mine = 0;
        for (int64_t b = b0; b < b1; ++b) mine += ((int64_t)sequence_of(a, b).tokens * G + kRows - 1) / kRows;
        int64_t* const sums = (int64_t*)&info[0][0][0];
        int64_t in = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up(in, d);
            if (lane >= d) in += o;
        }
        if (lane == 63) sums[wave] = in;
        __syncthreads();
        for (int w = 0; w < wave; ++w) in += sums[w];
        const int64_t total = sums[0] + sums[1] + sums[2] + sums[3];
        const int64_t rank = total - 1 - blockIdx.x / (uint32_t)(c.kv_heads * g.splits);
        if (rank < 0) return;
        int64_t at = in - mine;
        for (int64_t b = b0; b < b1; ++b) {
            const int64_t n = ((int64_t)sequence_of(a, b).tokens * G + kRows - 1) / kRows;
            if (at <= rank && rank < at + n) {
                found[0] = b;
                found[1] = rank - at;
            }
            at += n;
        }
        if (tid < 3) bad[tid] = 0;
        __syncthreads();
    }
    const int32_t b = __builtin_amdgcn_readfirstlane((int32_t)found[0]);
    const int32_t row0 = __builtin_amdgcn_readfirstlane((int32_t)found[1]) * kRows;
    const Sequence seq = sequence_of(a, b);
    const int32_t rows = (int32_t)((int64_t)seq.tokens * G - row0 < kRows ? (int64_t)seq.tokens * G - row0 : kRows);

    // keys of the sequence, and the row of the first where they are contiguous
    int32_t keys = 0, key0 = 0;
    if (b < a.batch) {
        if (a.kv.table) {
            const int64_t most = a.kv.table_width * c.page_size;
            keys = a.kv.lens[b];
            keys = keys < 0 ? 0 : keys > most ? (int32_t)most : keys;
        } else {
            const int32_t all = c.num_pages ? (int32_t)c.page_size : 0;
            key0 = b == 0 ? 0 : a.kv.cu_k[b];
            key0 = key0 < 0 ? 0 : key0;
            const int32_t end = a.kv.cu_k[b + 1] < all ? a.kv.cu_k[b + 1] : all;
            keys = end > key0 ? end - key0 : 0;
        }
    }
    const int32_t past = keys - seq.tokens;  // position of the first token (negative: it stands before the first key)
    const int32_t p_first = past + div31(row0, g.group_div), p_last = past + div31(row0 + rows - 1, g.group_div);

    // this lane's row (past the last: as the last)
    const int32_t mine = row0 + (wave * 32 + col < rows ? wave * 32 + col : rows - 1);
    const int32_t token = div31(mine, g.group_div);
    const int64_t t = seq.first + token;
    const int h = kvh * G + (mine - token * G);
    const int32_t p = past + token;
    
    // the keys that any row sees, without a gap: key j is place j or, past the sinks, j - gap
    int32_t low = 0, sinks = 0;
    if (a.window && p_first >= a.window) {  // (a tile may begin before the first key: a difference could pass 32 bits)
        low = p_first - a.window + 1;
        sinks = a.sinks < low ? a.sinks : low;
    }
    const int32_t gap = low - sinks;
    const int32_t places = p_last < 0 ? 0 : p_last + 1 - gap;
    const int all_tiles = (places + kKeys - 1) / kKeys;
    // this workgroup's part of them
    const int split = (int)(blockIdx.x / (uint32_t)c.kv_heads % (uint32_t)g.splits);
    int splits = (all_tiles + kSplitTiles - 1) / kSplitTiles;
    splits = splits < 1 ? 1 : splits < g.splits ? splits : g.splits;
    if (split >= splits) return;
    const int tile0 = (int)((int64_t)all_tiles * split / splits), tiles = (int)((int64_t)all_tiles * (split + 1) / splits);

    // the largest score is found before the scale is applied: a negative scale's sign goes to the query
    const uint32_t turned = !Q8 && a.scale < 0.0f ? 0x80008000u : 0u;
    u32x4 q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int d = 16 * s + 8 * kg;
        q[s] = (u32x4){0, 0, 0, 0};
        if (WHOLE || d < D) q[s] = *(const u32x4*)((const uint16_t*)a.q + t * a.q_token_stride + h * a.q_head_stride + d);
        q[s] ^= turned;
    }
    f32x16 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
    float m = kLowest, l = 0.0f;
    bool any = false;
    // (a scale of 0 becomes one that leaves every product 0: -inf, a masked score, must stay what it is)
    const float factor = Q8 ? 1.0f : __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(fmaxf(fabsf(a.scale) * kLog2e, 0x1p-120f))));

    const bool paged = a.kv.table != nullptr;
    const Global zeros = global_address(kZeroRow);
    // What finds the rows' places reads its arguments from memory again each time: they would hold scalar registers that the
    // loop has better use for.
    auto args = []() INLINE {
        const __attribute__((address_space(4))) PromptArgs* from =
            (const __attribute__((address_space(4))) PromptArgs*)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(from));
        return from;
    };
    // Each wave finds its 16 rows of four tiles at a time, a lane per row: the page, then the place in memory and the scales.
    auto place = [&](int tile) INLINE {
        const int32_t v = (tile + kg * 2 + (col >> 4)) * kKeys + wave * 16 + (lane & 15);
        return v < places ? (v < sinks ? v : v + gap) : -1;
    };
    auto page_of = [&](int tile) INLINE {
        const int32_t j = place(tile);
        if (!paged || j < 0) return (int32_t)-1;
        const auto* g = args();
        const Global table = global_address(g->a.kv.table + b * g->a.kv.table_stride);
        return load_global<int32_t>(table + (int64_t)div31(j, (Div31){g->a.kv.page_div.m, g->a.kv.page_div.s}) * 4);
    };
    float ks_next = 0.0f, vs_next = 0.0f;
    auto put_info = [&](int tile, int32_t page) INLINE {
        const auto* g = args();
        const auto& c = g->a.kv.c;
        const int32_t j = place(tile);
        int32_t slot = key0 + j;
        bool valid = j >= 0;
        if (paged) {
            slot = j - div31(j, (Div31){g->a.kv.page_div.m, g->a.kv.page_div.s}) * (int32_t)c.page_size;
            valid = valid && page >= 0 && page < c.num_pages;
        } else {
            page = 0;
        }
        Global kp = zeros, vp = zeros;
        if (valid) {
            kp = global_address(c.key) + (page * c.key_page_stride + slot * c.key_token_stride + kvh * c.key_head_stride) * ES;
            vp = global_address(c.value) + (page * c.value_page_stride + slot * c.value_token_stride + kvh * c.value_head_stride) * ES;
        }
        uint64_t* const to = info[tile + (lane >> 4) & 7][wave * 16 + (lane & 15)];
        to[0] = (uint64_t)(uintptr_t)kp;
        to[1] = (uint64_t)(uintptr_t)vp;
        const uint64_t ok = __builtin_amdgcn_ballot_w64(valid);
        if ((lane & 15) == 0) ((uint16_t*)info_ok)[(tile + (lane >> 4) & 7) * 4 + wave] = (uint16_t)(ok >> lane);
        if constexpr (Q8) {
            Global kz = zeros, vz = zeros;
            if (valid) {
                kz = global_address(c.key_scale + page * c.key_scale_page_stride + slot * c.key_scale_token_stride +
                                    kvh * c.key_scale_head_stride);
                vz = global_address(c.value_scale + page * c.value_scale_page_stride + slot * c.value_scale_token_stride +
                                    kvh * c.value_scale_head_stride);
            }
            ks_next = load_global<float>(kz);
            vs_next = load_global<float>(vz);
        }
    };
    auto put_scales = [&](int tile) INLINE {
        if constexpr (Q8) {
            float* const to = &scales[tile + (lane >> 4) & 7][0][wave * 16 + (lane & 15)];
            to[0] = ks_next * (a.scale * kLog2e);
            to[kKeys] = vs_next;
            to[2 * kKeys] = __builtin_amdgcn_logf(fmaxf(fabsf(vs_next), 0x1p-60f));
        }
    };

    // the place of piece ch of row r in LDS
    auto k_turn = [](int r) INLINE { return CHL == 8 ? r >> 1 & 7 : r & 15; };
    auto v_turn = [](int r) INLINE { return CHL == 8 ? (r >> 1 & 3) << 1 : (r & 7) << 1; };
    u32x4 kr[PIECES], vr[PIECES];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    const int k_piece = (lane % CHL ^ k_turn(lane / CHL)) << 4, v_piece = (lane % CHL ^ v_turn(lane / CHL)) << 4;
    const int lane_rows = (wave * 16 + lane / CHL) * 2;
    // Addresses of this lane's pieces of K (which 0) or V (1) of a tile, and piece i on its way to LDS buffer tile & 1.
    // Load i of the wave fills rows i * R + lane / CHL of its 16; the turn of a sum of rows is the turns' exclusive or.
    constexpr int R = 64 / CHL;
    auto address = [&](int tile, int which, int i) INLINE {
        const int ch = (which ? v_piece : k_piece) ^ (which ? v_turn(i * R) : k_turn(i * R)) << 4;
        Global from = (Global)(uintptr_t)(&info[tile & 7][0][which] + lane_rows)[i * R * 2] + ch;
        if (!WHOLE || DP * 2 < LS) {
            if (ch >= D * 2) from = zeros;
        }
        return from;
    };
    auto send = [&](int tile, int which, int i, Global from) INLINE {
        global_to_lds(from, lds0 + (2 * (tile & 1) + which) * TILE + (wave * DMAS + i) * 1024);
    };
    // the whole of it; int8: into registers
    auto load_tile = [&](int tile, int which) INLINE {
        if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int at = tid + i * kThreads, r = at / CH, ch = at % CH;
                Global from = (Global)(uintptr_t)info[tile & 7][r][which] + ch * 16;
                if (!WHOLE && ch * 16 >= D) from = zeros;
                (which ? vr : kr)[i] = load_global<u32x4>(from);
            }
        } else {
#pragma unroll
            for (int i = 0; i < DMAS; ++i) send(tile, which, i, address(tile, which, i));
        }
    };
    // int8: K or V of a tile from the registers, as 16-bit values
    auto store_tile = [&](int tile, int which) INLINE {
        if constexpr (Q8) {
            char* const buffer = lds + (2 * (tile & 1) + which) * TILE;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int at = tid + i * kThreads, r = at / CH, ch = 2 * (at % CH), turn = which ? v_turn(r) : k_turn(r);
                const u32x4 w = (which ? vr : kr)[i];
                *(u32x4*)(buffer + r * LS + ((ch ^ turn) << 4)) = which ? i8_to_f16(w[0], w[1]) : i8_to_half<DT>(w[0], w[1]);
                *(u32x4*)(buffer + r * LS + ((ch + 1 ^ turn) << 4)) = which ? i8_to_f16(w[2], w[3]) : i8_to_half<DT>(w[2], w[3]);
            }
        }
    };

    const bool no_rows = wave * 32 >= rows;  // for this wave
    if (tile0 < tiles) {
        int32_t page = page_of(tile0);
        put_info(tile0, page);
        page = page_of(tile0 + 4);
        put_scales(tile0);
        __syncthreads();
        load_tile(tile0, 0);
        if constexpr (Q8) {
            store_tile(tile0, 0);
            load_tile(tile0 + 1, 0);
            load_tile(tile0, 1);
        } else {
            load_tile(tile0 + 1, 0);
            load_tile(tile0, 1);
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        }
        __syncthreads();

        const int k_at = col * LS + ((kg ^ k_turn(col)) << 4);
        const int v_row = 4 * kg + (lane >> 2 & 3);
        const int v_at = v_row * LS + (((lane >> 4 & 1) << 1 | (lane >> 1 & 1)) ^ v_turn(v_row)) * 16 + 8 * (lane & 1);
        // scores of a tile: lane (row, kg) holds keys 32 n + 8 (e / 4) + 4 kg + e % 4
        auto scores = [&](int tile, f32x16 (&x)[2]) INLINE {
            const char* const kb = lds + 2 * (tile & 1) * TILE;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) x[n][e] = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int n = 0; n < 2; ++n) x[n] = mma32<DT>(*(const u32x4*)(kb + (k_at ^ s << 5) + 32 * n * LS), q[s], x[n]);
        };

        uint64_t mine = ~0ull;  // the tile's keys that this lane's row sees, from the lane's first on: bit 32 n + 8 (e / 4) + e % 4
        bool edge = false;  // some row of the workgroup does not see some key of the tile at hand
        int32_t j0 = 0;     // the tile's first key
        uint64_t ok = 0;    // which of its keys exist
        auto look = [&](int tile, uint64_t which) INLINE {
            ok = uniform64(which);
            const int32_t last = tile * kKeys + kKeys - 1, j1 = last + (last < sinks ? 0 : gap);
            j0 = tile * kKeys + (tile * kKeys < sinks ? 0 : gap);
            edge = ~ok != 0 || j1 > p_first || (a.window && j1 >= a.sinks && p_last - j0 >= a.window);
        };
        // Moves the maximum where a score lies far above it; `top` is a lane's largest score (a NaN does not matter).
        auto raise = [&](float top) INLINE {
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(top * factor > m + (kBelow<PV> + kSlack)) != 0, 0)) {
                const float m2 = fmaxf(m, pair_max(top * factor) - kBelow<PV>);
                const float keep = __builtin_amdgcn_exp2f(m - m2);
                m = m2;
                l *= keep;
#pragma unroll
                for (int i = 0; i < NB; ++i) acc[i] *= keep;
            }
        };
        // int8: scores times the keys' scales, in units of log2; the largest of them, each with its value's scale: what the weight that
        // goes into the product is held against.  Keys that are hidden are not looked at.
        auto scale_scores = [&](int tile, f32x16 (&x)[2], auto hide) INLINE {
            float top = -__builtin_inff();
            const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    __builtin_amdgcn_sched_barrier(0);  // few of them in registers at a time
                    const f32x4 k4 = *(const f32x4*)&scales[tile & 7][0][32 * n + 8 * i + 4 * kg];
                    const f32x4 l4 = *(const f32x4*)&scales[tile & 7][2][32 * n + 8 * i + 4 * kg];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float v = x[n][4 * i + r] * k4[r];
                        if constexpr (decltype(hide)::value) {
                            const bool sees = (n ? hi : lo) & 1u << (8 * i + r);
                            v = sees ? v : -__builtin_inff();
                            top = fmaxf(top, sees ? v + l4[r] : -__builtin_inff());
                        } else {
                            top = __builtin_elementwise_maximum(top, v + l4[r]);
                        }
                        x[n][4 * i + r] = v;
                    }
                }
            return top;
        };
        // int8: the weights' sum, and the weights with the values' scales (0 for what is hidden, whatever its scale)
        auto scale_weights = [&](int tile, f32x16 (&x)[2], auto hide) INLINE {
            const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
            float part[2] = {0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    const f32x4 v4 = *(const f32x4*)&scales[tile & 7][1][32 * n + 8 * i + 4 * kg];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        part[r & 1] += x[n][4 * i + r];
                        x[n][4 * i + r] *= !decltype(hide)::value || (n ? hi : lo) & 1u << (8 * i + r) ? v4[r] : 0.0f;
                    }
                }
            l += part[0] + part[1];
        };
        // What every step begins with: K of the next tile and V of this one are in LDS behind its barrier.
        auto begin = [&](int it) INLINE {
            if constexpr (Q8) {
                store_tile(it + 1, 0);
                store_tile(it, 1);
            } else {
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // this wave's part is in LDS
            }
        };
        auto behind_barrier = [&](int it) INLINE {
            if (Q8 && (it - tile0 & 3) == 2) put_scales(it + 2);
            if ((it - tile0 & 3) == 0) {
                put_info(it + 4, page);
                page = page_of(it + 8);
            }
        };

        // Looks at the tile whose scores x are there, `top` a lane's largest: hides what is not seen, moves the maximum.
        auto prepare = [&](int tile, uint64_t which, f32x16 (&x)[2], float top) INLINE {
            look(tile, which);
            if (no_rows) return;
            mine = ~0ull;
            if (__builtin_expect(edge, 0)) {
                // the tile's places that this row sees: up to its own, but for those between the sinks and its window
                auto below = [](int32_t n) INLINE { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };
                auto place_of = [&](int32_t j) INLINE { return (j < sinks ? j : j < sinks + gap ? sinks : j - gap) - tile * kKeys; };
                uint64_t seen = ok & below(place_of(p + 1));
                if (a.window && p >= a.window) seen &= ~below(place_of(p - a.window + 1)) | below(place_of(a.sinks));
                any |= seen != 0;
                mine = seen >> here(4 * kg);
                if constexpr (Q8) {
                    top = scale_scores(tile, x, std::true_type());
                } else {
                    const uint32_t lo = (uint32_t)mine, hi = (uint32_t)(mine >> 32);
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[n][e] = (n ? hi : lo) & 1u << (8 * (e >> 2) + (e & 3)) ? x[n][e] : -__builtin_inff();
                    top = largest(x);
                }
            } else {
                any = true;
                if constexpr (Q8) top = scale_scores(tile, x, std::false_type());
            }
            raise(top);
        };

        // One step: the tile's weights from its scores x, while the next tile's scores are made (into y), then its values.
        auto step = [&](int it, f32x16 (&x)[2], f32x16 (&y)[2]) INLINE {
            begin(it);
            if (!Q8 && __builtin_expect(edge, 0)) {
                char* const vb = lds + (2 * (it & 1) + 1) * TILE;
#pragma nounroll
                for (int i = 0; i < DMAS; ++i) {
                    const int slot = (wave * DMAS + i) * 64 + lane, r = slot / CHL;
                    const u32x4 v = *(const u32x4*)(vb + slot * 16);
                    if (not_finite<DT>(v)) {
                        *(u32x4*)(vb + slot * 16) = finite_only<DT>(v);
                        atomicOr((unsigned long long*)&bad[it % 3], 1ull << r);
                    }
                }
            }
            __syncthreads();
            if (!Q8 && tid == 0) bad[(it + 2) % 3] = 0;
            if (__builtin_expect(no_rows, 0)) {
                behind_barrier(it);
                load_tile(it + 2, 0);
                load_tile(it + 1, 1);
                look(it + 1, info_ok[it + 1 & 7]);
                return;
            }
            const uint32_t k_from = lds0 + 2 * (it + 1 & 1) * TILE + here(k_at);
            auto k_operand = [&](int i) INLINE { return lds_load(k_from ^ (i >> 1) << 5, 32 * (i & 1) * LS); };
            constexpr int AHEAD1 = Q8 ? 4 : 6;
            u32x4 k_ring[AHEAD1];
#pragma unroll
            for (int i = 0; i < AHEAD1; ++i) k_ring[i] = k_operand(i);
            behind_barrier(it);
            // What is sent for: K two tiles on, V one (past the last: rows of zeros, or ones that are not used).  The 16-bit
            // loads go out between the products, their addresses being read here.
            constexpr int SENDS = Q8 ? 1 : 2 * DMAS;
            Global from[SENDS];
            if constexpr (Q8) {
                load_tile(it + 2, 0);
                load_tile(it + 1, 1);
            } else {
#pragma unroll
                for (int i = 0; i < SENDS; ++i) from[i] = address(i < DMAS ? it + 2 : it + 1, i / DMAS, i % DMAS);
            }
            const uint64_t ok_next = info_ok[it + 1 & 7];  // asked for here, used at the step's end
            const uint32_t v_from = lds0 + (2 * (it & 1) + 1) * TILE + here(v_at);
            auto v_operand = [&](int i) INLINE {
                const uint32_t from = v_from ^ (i % NB) << 6;
                const u32x2 lo = lds_tr16(from, 16 * (i / NB) * LS), hi = lds_tr16(from, (16 * (i / NB) + 8) * LS);
                return (u32x4){lo[0], lo[1], hi[0], hi[1]};
            };
            constexpr int AHEAD2 = Q8 ? 2 : 4;
            u32x4 v_ring[AHEAD2];
            // the next tile's scores, with this one's weights between the products
            {
                constexpr int N = 2 * KS, FIRST = 6;
                auto weight = [&](int k) INLINE {
                    float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[k >> 4][k & 15], factor, -m));
                    asm volatile("" : "+v"(w));  // made here, not where it is used
                    x[k >> 4][k & 15] = w;
                };
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[n][e] = 0.0f;
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int k = 0; k < FIRST; ++k) weight(k);  // while the first operands come
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    y[i & 1] = mma32<DT>(k_ring[i % AHEAD1], q[i >> 1], y[i & 1]);
                    if (i + AHEAD1 < N) k_ring[i % AHEAD1] = k_operand(i + AHEAD1);
                    if constexpr (!Q8) {
#pragma unroll
                        for (int k = i * SENDS / N; k < (i + 1) * SENDS / N; ++k)
                            send(k < DMAS ? it + 2 : it + 1, k / DMAS, k % DMAS, from[k]);
                    }
                    if (i >= N - AHEAD2) v_ring[i - N + AHEAD2] = v_operand(i - N + AHEAD2);
#pragma unroll
                    for (int k = FIRST + i * (32 - FIRST) / N; k < FIRST + (i + 1) * (32 - FIRST) / N; ++k) weight(k);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (Q8) {
                if (__builtin_expect(edge, 0)) scale_weights(it, x, std::true_type());
                else scale_weights(it, x, std::false_type());
            } else if (__builtin_expect(edge, 0)) {
#pragma nounroll
                for (uint64_t left = uniform64(bad[it % 3]); left; left &= left - 1) {
                    const int key = __builtin_ctzll(left), own = key - here(4 * kg);
                    // this row's weight of the key, from whichever of the two lanes holds it, and whether it is seen
                    float w = 0.0f;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e) w = own == 32 * n + 8 * (e >> 2) + (e & 3) ? x[n][e] : w;
                    w = load_half_bits(pack2<DT>(pair_sum(w), 0.0f) & 0xffffu, DT);  // as the products round it
                    const bool sees = pair_max(own >= 0 && !(own & 4) && (mine >> (own & 63) & 1) ? 1.0f : 0.0f) != 0.0f;
                    const Global row = (Global)(uintptr_t)info[it & 7][key][1];
#pragma unroll
                    for (int i = 0; i < NB; ++i)
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const int d = 32 * i + 2 * e + 4 * kg;
                            const u32x2 bits = WHOLE || d < D ? load_global<u32x2>(row + d * 2) : (u32x2){0, 0};
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const uint32_t h = bits[r >> 1] >> (16 * (r & 1)) & 0xffffu;
                                if (sees && (h & exponent_of<DT>()) == exponent_of<DT>()) acc[i][e + r] += w * load_half_bits(h, DT);
                            }
                        }
                }
            }
            // acc += V^T P^T; between the products the weights' sum, their rounding to 16 bits, and the largest of the next scores
            float top = y[0][0];
            {
                constexpr int N = 4 * NB;
                auto weights = [&](int s, int i) INLINE {
                    return pack2<PV>(x[s >> 1][8 * (s & 1) + 2 * i], x[s >> 1][8 * (s & 1) + 2 * i + 1]);
                };
                u32x4 pw[2];
#pragma unroll
                for (int i = 0; i < 4; ++i) pw[0][i] = weights(0, i);
                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int s = i / NB;
                    acc[i % NB] = mma32<PV>(v_ring[i % AHEAD2], pw[s & 1], acc[i % NB]);
                    if (i + AHEAD2 < N) v_ring[i % AHEAD2] = v_operand(i + AHEAD2);
                    if (s < 3) {
#pragma unroll
                        for (int k = i % NB * 4 / NB; k < (i % NB + 1) * 4 / NB; ++k) pw[s + 1 & 1][k] = weights(s + 1, k);
                    }
                    if constexpr (!Q8) {
#pragma unroll
                        for (int k = i * 32 / N; k < (i + 1) * 32 / N; ++k) {
                            part[k & 3] += x[k >> 4][k & 15];
                            top = __builtin_elementwise_maximum(top, y[k >> 4][k & 15]);
                        }
                        asm volatile("" : "+v"(top), "+v"(part[0]), "+v"(part[1]), "+v"(part[2]), "+v"(part[3]));
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (!Q8) l += (part[0] + part[1]) + (part[2] + part[3]);
            }
            prepare(it + 1, ok_next, y, top);
        };

        f32x16 xa[2], xb[2];
        if (!no_rows) scores(tile0, xa);
        prepare(tile0, info_ok[tile0 & 7], xa, largest(xa));
        for (int it = tile0; it < tiles; it += 2) {
            step(it, xa, xb);
            if (it + 1 < tiles) step(it + 1, xb, xa);
        }
    }

    l = pair_sum(l);
    if (splits > 1) {
        const int64_t place = (blockIdx.x / (uint32_t)(c.kv_heads * g.splits)) * c.kv_heads + kvh;
        // in the order of the registers: whole lines, and the joining lane finds its own rows
        constexpr uint32_t SUMS = 4 * NB * 4 * 1024;
        auto part = [&](int s) INLINE { return make_rsrc((const char*)g.parts + (place * g.splits + s) * g.part_bytes, (uint32_t)g.part_bytes); };
        const __amdgpu_buffer_rsrc_t own = part(split);
        if (!no_rows) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    __builtin_amdgcn_raw_buffer_store_b128(
                        __builtin_bit_cast(u32x4, (f32x4){acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]}), own,
                        lane * 16, ((wave * NB + i) * 4 + e) * 1024, kCoherent);
            if (kg == 0)
                __builtin_amdgcn_raw_buffer_store_b64((u32x2){__float_as_uint(any ? m : -__builtin_inff()), __float_as_uint(l)}, own,
                                                      SUMS + (wave * 32 + col) * 8, 0, kCoherent);
        }
        if (!splitk_last(g.arrivals + place, (uint32_t)splits, g.tag)) return;
        m = -__builtin_inff();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
        if (!no_rows) {
            auto max_and_sum = [&](int s) INLINE {
                return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(part(s), SUMS + (wave * 32 + col) * 8, 0, kCoherent));
            };
            for (int s = 0; s < splits; s += 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k) m = fmaxf(m, __uint_as_float(max_and_sum(s + k < splits ? s + k : s)[0]));
            }
            // two parts in registers: one on its way while the other is added
            f32x4 v[2][NB][4];
            u32x2 ml[2];
            auto read = [&](int s, f32x4 (&to)[NB][4], u32x2& to_ml) INLINE {
                const __amdgpu_buffer_rsrc_t rs = part(s < splits ? s : splits - 1);
                to_ml = max_and_sum(s < splits ? s : splits - 1);
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        to[i][e] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, lane * 16, ((wave * NB + i) * 4 + e) * 1024, kCoherent));
            };
            auto add = [&](f32x4 (&from)[NB][4], u32x2 from_ml) INLINE {
                const float pm = __uint_as_float(from_ml[0]);
                const bool none = pm == -__builtin_inff();
                const float f = none ? 0.0f : __builtin_amdgcn_exp2f(pm - m);
                l += none ? 0.0f : __uint_as_float(from_ml[1]) * f;
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][e] += none ? 0.0f : from[i][e >> 2][e & 3] * f;
            };
            read(0, v[0], ml[0]);
            for (int s = 0; s < splits; s += 2) {
                read(s + 1, v[1], ml[1]);
                __builtin_amdgcn_sched_barrier(0);
                add(v[0], ml[0]);
                __builtin_amdgcn_sched_barrier(0);
                read(s + 2, v[0], ml[0]);
                __builtin_amdgcn_sched_barrier(0);
                if (s + 1 < splits) add(v[1], ml[1]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        any = m != -__builtin_inff();
    }
    if (wave * 32 + col >= rows) return;
    const float inv = 1.0f / l;
    const int64_t o = t * a.q_heads + h;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int d = 32 * i + 2 * e + 4 * kg;
            if (!WHOLE && d >= D) continue;
            f32x4 r;
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k] = any ? acc[i][e + k] * inv : 0.0f;
            *(u32x2*)((uint16_t*)a.out + o * D + d) = (u32x2){pack2<DT>(r[0], r[1]), pack2<DT>(r[2], r[3])};
        }
    if (kg == 0 && a.lse) a.lse[o] = any ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -__builtin_inff();
}

template <int DP, int DT, bool Q8>
void launch_width(const PromptArgs& g, int64_t grid, hipStream_t stream) {
    if (g.a.kv.c.head_dim == DP) attention_prompt<DP, DT, Q8, true><<<dim3((unsigned)grid), kThreads, 0, stream>>>(g);
    else attention_prompt<DP, DT, Q8, false><<<dim3((unsigned)grid), kThreads, 0, stream>>>(g);
}
template <int DT, bool Q8>
void launch_type(const PromptArgs& g, int64_t grid, hipStream_t stream) {
    const int64_t D = g.a.kv.c.head_dim;
    if (D <= 64) launch_width<64, DT, Q8>(g, grid, stream);
    else if (D <= 96 && !Q8) launch_width<96, DT, false>(g, grid, stream);
    else if (D <= 128) launch_width<128, DT, Q8>(g, grid, stream);
    else if (D <= 192) launch_width<192, DT, Q8>(g, grid, stream);
    else launch_width<256, DT, Q8>(g, grid, stream);
}

struct Plan {
    int64_t grid, arrivals_bytes, part_bytes;
    int splits;
};

Plan plan(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width, int64_t window, int64_t sinks) {
    Plan p = {};
    const int64_t group = q_heads / c.kv_heads;
    // at most: whole tiles, and a last one for every sequence and for the rows past them
    const int64_t some = batch < tokens ? batch : tokens;
    const int64_t tiles = (tokens * group / kRows + some + 1) * c.kv_heads;
    int64_t most = (table_width ? table_width : 1) * c.page_size;
    if (window && most > window && most - window > sinks + kRows) most = window + sinks + kRows;
    const int64_t steps = (most + kKeys - 1) / kKeys;
    int64_t splits = kResident / tiles;
    if (splits > steps / kSplitTiles) splits = steps / kSplitTiles;
    p.splits = splits < 1 ? 1 : (int)splits;
    p.grid = tiles * p.splits;
    if (p.splits > 1) {
        const int64_t D = c.head_dim, width = D <= 64 ? 64 : D <= 96 && c.dtype != QK_I8 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256;
        p.arrivals_bytes = (tiles * 8 + 255) / 256 * 256;
        p.part_bytes = kRows * (width + 2) * 4;
    }
    return p;
}

}  // namespace

size_t attention_prompt_workspace(int64_t tokens, int64_t batch, int64_t q_heads, const qk_kv_cache& c, int64_t table_width,
                                  int64_t window, int64_t sinks) {
    if (tokens == 0) return 0;
    const Plan p = plan(tokens, batch, q_heads, c, table_width, window, sinks);
    return (size_t)(p.arrivals_bytes + p.grid * p.part_bytes);
}

hipError_t launch_attention_prompt(const AttnArgs& a, void* workspace, hipStream_t stream) {
    const Plan p = plan(a.tokens, a.batch, a.q_heads, a.kv.c, a.kv.table_width, a.window, a.sinks);
    PromptArgs g = {};
    g.a = a;
    g.group_div = div31((uint32_t)(a.q_heads / a.kv.c.kv_heads));
    g.splits = p.splits;
    if (p.splits > 1) {
        g.tag = next_split_tag();
        g.arrivals = (uint64_t*)workspace;
        g.parts = (float*)((char*)workspace + p.arrivals_bytes);
        g.part_bytes = p.part_bytes;
    }
    const bool q8 = a.kv.c.dtype == QK_I8;
    if (a.dtype == QK_BF16) {
        if (q8) launch_type<QK_BF16, true>(g, p.grid, stream);
        else launch_type<QK_BF16, false>(g, p.grid, stream);
    } else {
        if (q8) launch_type<QK_F16, true>(g, p.grid, stream);
        else launch_type<QK_F16, false>(g, p.grid, stream);
    }
    return hipGetLastError();
}

}  // namespace qk
