// The end of a step of decoding with drafts: the way from a tree's root along the drafted tokens that were drawn, its rows of the cache
// moved right behind the context in every tensor, and the sequence cut to it.
//
// Bound by latency, and by HBM where many layers move many rows: each moved row is read and written once.  Measured on one MI355X:
// 16 rows of one sequence, 32 tensors, 5 us; 64 trees of up to 48 12 us, as long as the call's checks take on the host (fewer
// workgroups, each with the rows of several tensors, take longer: 512 of them 3 us more).  The drawn child of each
// row is found for all rows at once (the lowest wins by an atomic minimum in LDS), then the way is a chain of LDS reads;
// that is so little that every workgroup walks for itself instead of waiting for a launch that does.  A thread moves one
// column of all rows of the way: row j goes to a place at or before its own, and a child stands behind its parent, so the rows that a
// store could overwrite have been read by the same thread before, and nothing else orders the moves.
#include "attention.h"

namespace qk {
namespace {

constexpr int kThreads = 128;
constexpr int kTree = 1024;   // rows of a tree whose way is found in LDS; in larger ones a search in memory finds each step's child
constexpr int kTensors = 64;  // tensors per launch: 48 bytes of arguments each, of the 4 KB that a launch has
constexpr int kAhead = 8;     // rows of a column in flight

struct RowList {
    qk_rows t[kTensors];
};

struct AcceptArgs {
    PoolArgs p;
    const int32_t *seqs, *cu;
    int64_t n, total;
    const int32_t *tokens, *parents, *sampled;
    int32_t *path, *accepted, *next;
};

// A sequence's tree: rows first .. first + size of the call's, behind `past` tokens of context (size 0: passed over).
struct Tree {
    int32_t seq, first, end, size, past;
};
__device__ __forceinline__ int32_t length_of(const PoolArgs& p, int64_t seq) {
    const int64_t most = p.table_width * p.page_size, n = p.lens[seq];
    return (int32_t)(n < 0 ? 0 : n > most ? most : n);
}
__device__ __forceinline__ Tree tree_of(const AcceptArgs& a, int64_t i) {
    const int32_t T = (int32_t)a.total;
    Tree t = {a.seqs[i], a.cu[i], a.cu[i + 1], 0, 0};
    t.first = t.first < 0 ? 0 : t.first > T ? T : t.first;
    t.end = t.end < t.first ? t.first : t.end > T ? T : t.end;
    if (t.seq < 0 || t.seq >= a.p.max_seqs) return t;
    t.past = length_of(a.p, t.seq) - (t.end - t.first);
    if (t.past >= 0) t.size = t.end - t.first;
    return t;
}

// The slot (page * page_size + place) of a sequence's token, or -1.
__device__ __forceinline__ int64_t slot_of(const PoolArgs& p, int32_t seq, int64_t token) {
    const int64_t at = token / p.page_size;
    if (at >= p.table_width) return -1;
    const int32_t page = p.table[seq * p.table_stride + at];
    return page < 0 || page >= p.num_pages ? -1 : page * p.page_size + token % p.page_size;
}

// Units u of `T` of a token: where it lies in the token's bytes.
template <typename T>
__device__ __forceinline__ int64_t unit_at(const qk_rows& t, int64_t u) {
    const int64_t per_piece = t.piece_bytes / (int64_t)sizeof(T);
    return u / per_piece * t.piece_stride + u % per_piece * (int64_t)sizeof(T);
}
__device__ __forceinline__ int64_t token_at(const qk_rows& t, int64_t page_size, int64_t slot) {
    return slot / page_size * t.page_stride + slot % page_size * t.token_stride;
}

// Moves units u, u + step, ... of rows j0 .. n of the way; from(j), to(j): their slots.
template <typename T, typename F>
__device__ __forceinline__ void move_units(const qk_rows& t, int64_t page_size, int64_t u, int64_t step, int32_t j0, int32_t n, F slots) {
    const int64_t units = t.pieces * (t.piece_bytes / (int64_t)sizeof(T));
    for (; u < units; u += step) {
        char* const base = (char*)t.base + unit_at<T>(t, u);
        for (int32_t j = j0; j < n; j += kAhead) {
            T v[kAhead];
            int64_t to[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                to[k] = -1;
                if (j + k < n) {
                    int64_t from;
                    slots(j + k, from, to[k]);
                    if (from < 0) to[k] = -1;
                    if (to[k] >= 0) v[k] = *(const T*)(base + token_at(t, page_size, from));
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (to[k] >= 0) *(T*)(base + token_at(t, page_size, to[k])) = v[k];
        }
    }
}
template <typename F>
__device__ __forceinline__ void move_rows(const qk_rows& t, int64_t page_size, int64_t u, int64_t step, int32_t j0, int32_t n, F slots) {
    const uintptr_t any = (uintptr_t)t.base | (uintptr_t)t.page_stride | (uintptr_t)t.token_stride |
                          (t.pieces > 1 ? (uintptr_t)t.piece_stride : 0) | (uintptr_t)t.piece_bytes;
    if (any % 16 == 0) move_units<u32x4>(t, page_size, u, step, j0, n, slots);
    else if (any % 4 == 0) move_units<uint32_t>(t, page_size, u, step, j0, n, slots);
    else move_units<uint8_t>(t, page_size, u, step, j0, n, slots);
}

// The sequence's length, and the pages that it no longer needs.
__device__ __forceinline__ void finish(const AcceptArgs& a, const Tree& t, int32_t kept) {
    const int64_t S = a.p.page_size, len = (int64_t)t.past + kept, old = (int64_t)t.past + t.size;
    for (int64_t j = (len + S - 1) / S + threadIdx.x; j < (old + S - 1) / S; j += blockDim.x) {
        const int32_t page = atomicExch(a.p.table + t.seq * a.p.table_stride + j, -1);
        if (page >= 0 && page < a.p.num_pages && atomicSub(a.p.count + page, 1) <= 0) atomicAdd(a.p.count + page, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) a.p.lens[t.seq] = (int32_t)len;
}

// blockIdx.x: the sequence (n: the rows of none); blockIdx.y: the tensor (0, in the first launch: also writes the way).  arrivals: of the
// sequences' workgroups that have read its length and its table, the last of which may then change them (nullptr: a launch of
// its own does).
__global__ __launch_bounds__(kThreads) void accept_rows(RowList list, int tensors, AcceptArgs a, bool write, uint64_t* arrivals, uint64_t tag) {
    __shared__ int32_t child[kTree], way[kTree];
    __shared__ int64_t from[kTree], to[kTree];
    __shared__ int32_t found[2];
    write = write && blockIdx.y == 0;
    if (blockIdx.x == a.n) {
        if (!write) return;
        const int32_t begin = a.n ? a.cu[0] : 0, end = a.n ? a.cu[a.n] : 0;
        for (int64_t t = threadIdx.x; t < a.total; t += kThreads)
            if (t < begin || t >= end) a.path[t] = -1;
        return;
    }
    const Tree t = tree_of(a, blockIdx.x);
    if (t.size == 0) {
        if (!write) return;
        for (int32_t i = t.first + (int32_t)threadIdx.x; i < t.end; i += kThreads) a.path[i] = -1;
        if (threadIdx.x == 0) {
            a.accepted[blockIdx.x] = 0;
            a.next[blockIdx.x] = -1;
        }
        return;
    }
    const int32_t *tokens = a.tokens + t.first, *parents = a.parents + t.first, *sampled = a.sampled + t.first;
    if (t.size <= kTree) {
        for (int32_t i = threadIdx.x; i < t.size; i += kThreads) child[i] = t.size;
        __syncthreads();
        for (int32_t i = 1 + threadIdx.x; i < t.size; i += kThreads) {
            const int32_t up = parents[i], token = tokens[i];
            if (up >= 0 && up < i && token >= 0 && token == sampled[up]) atomicMin(&child[up], i);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int32_t n = 0, last = 0;
            for (int32_t at = 0; at < t.size; at = child[at]) way[n++] = last = at;
            found[0] = n;
            found[1] = last;
        }
        __syncthreads();
        const int32_t n = found[0];
        if (write) {
            for (int32_t i = threadIdx.x; i < t.size; i += kThreads) a.path[t.first + i] = i < n ? t.first + way[i] : -1;
            if (threadIdx.x == 0) {
                a.accepted[blockIdx.x] = n;
                a.next[blockIdx.x] = sampled[found[1]];
            }
        }
        if (tensors == 0) {
            if (arrivals) finish(a, t, n);
            return;
        }
        for (int32_t j = threadIdx.x; j < n; j += kThreads) {
            from[j] = way[j] == j ? -1 : slot_of(a.p, t.seq, (int64_t)t.past + way[j]);
            to[j] = way[j] == j ? -1 : slot_of(a.p, t.seq, (int64_t)t.past + j);
        }
        __syncthreads();
        if (arrivals && splitk_last(arrivals + blockIdx.x, gridDim.y, tag)) finish(a, t, n);
        // the first rows of the way lie where they belong
        int32_t j0 = 0;
        while (j0 < n && way[j0] == j0) ++j0;
        move_rows(list.t[blockIdx.y], a.p.page_size, threadIdx.x, kThreads, j0, n, [&](int32_t j, int64_t& f, int64_t& o) {
            f = from[j];
            o = to[j];
        });
        return;
    }
    // A tree past what LDS holds: one workgroup a tensor step by step, each step's child searched in memory, one row at a time.
    int32_t at = 0, n = 0, last = 0;
    while (at < t.size) {
        if (write && threadIdx.x == 0) a.path[t.first + n] = t.first + at;
        if ((int)blockIdx.y < tensors && at != n) {
            const int64_t f = slot_of(a.p, t.seq, (int64_t)t.past + at), o = slot_of(a.p, t.seq, (int64_t)t.past + n);
            move_rows(list.t[blockIdx.y], a.p.page_size, threadIdx.x, kThreads, 0, 1, [&](int32_t, int64_t& x, int64_t& y) {
                x = f;
                y = o;
            });
        }
        last = at;
        ++n;
        const int32_t drawn = sampled[at];
        __syncthreads();  // found has been read
        if (threadIdx.x == 0) found[0] = t.size;
        __syncthreads();
        if (drawn >= 0)
            for (int32_t i = at + 1 + (int32_t)threadIdx.x; i < t.size; i += kThreads)
                if (parents[i] == at && tokens[i] == drawn) {
                    atomicMin(&found[0], i);
                    break;
                }
        __syncthreads();
        at = found[0];
    }
    if (write) {
        for (int32_t i = n + (int32_t)threadIdx.x; i < t.size; i += kThreads) a.path[t.first + i] = -1;
        if (threadIdx.x == 0) {
            a.accepted[blockIdx.x] = n;
            a.next[blockIdx.x] = sampled[last];
        }
    }
    if (arrivals && splitk_last(arrivals + blockIdx.x, gridDim.y, tag)) finish(a, t, n);
}

__global__ __launch_bounds__(64) void accept_finish(AcceptArgs a) {
    const Tree t = tree_of(a, blockIdx.x);
    if (t.size > 0) finish(a, t, a.accepted[blockIdx.x]);
}

}  // namespace

size_t kv_accept_workspace(int64_t n) { return (size_t)n * 8; }

hipError_t launch_kv_accept(const qk_rows* rows, int64_t tensors, const PoolArgs& p, const int32_t* seqs, const int32_t* cu,
                            int64_t n, int64_t total, const int32_t* tokens, const int32_t* parents, const int32_t* sampled,
                            int32_t* path, int32_t* accepted, int32_t* next, void* ws, hipStream_t stream) {
    const AcceptArgs a = {p, seqs, cu, n, total, tokens, parents, sampled, path, accepted, next};
    // one launch ends the sequences too; more of them read what that changes
    const bool one = tensors <= kTensors;
    const uint64_t tag = next_split_tag();
    int64_t i = 0;
    do {
        RowList list = {};
        const int k = (int)(tensors - i < kTensors ? tensors - i : kTensors);
        for (int j = 0; j < k; ++j) list.t[j] = rows[i + j];
        accept_rows<<<dim3((unsigned)(n + 1), (unsigned)(k < 1 ? 1 : k)), kThreads, 0, stream>>>(list, k, a, i == 0,
                                                                                                      one ? (uint64_t*)ws : nullptr, tag);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        i += kTensors;
    } while (i < tensors);
    if (n > 0 && !one) accept_finish<<<dim3((unsigned)n), 64, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace qk
