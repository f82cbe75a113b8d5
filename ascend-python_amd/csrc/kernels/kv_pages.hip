// The pages of a key-value cache on gfx950: copy, fork, extend, free, compact.
//
// The pool's state is a page table, the sequences' lengths and a count per page; no free list is kept.  A page is free when
// its count is 0, and the k-th page that a call needs is the k-th lowest free id: a prefix sum over the counts, which one
// workgroup of 1024 threads makes, 4096 counts at a time, stopping when it has found enough (a pool of 1024 pages is one
// step, one of 131072, some 200 GB of a 32-layer cache, at most 32).  So the same calls give the same pages,
// whatever the order of workgroups, and freeing is a subtraction.
//
// What moves bytes is one kernel: items of (pair of pages, tensor, 16 KB piece) handed to workgroups in turn, four
// 16-byte loads in flight per lane before the stores.  Bound by HBM: each byte is read and written once
// (a pool of 1024 pages of 1 MB packed: 75 us, 4.5 TB/s; pieces of 32 KB, eight loads in flight: 97 us).
#include "attention.h"

namespace qk {
namespace {

constexpr int kPlan = 1024;   // threads of a planning workgroup
constexpr int kWaves = kPlan / 64;
constexpr int kCopy = 256;    // threads of a copying workgroup
constexpr int64_t kPiece = 16384;
constexpr int kTensors = 120; // tensors per launch: 2880 bytes of arguments

struct PageList {
    qk_pages t[kTensors];
};

// Sum of v over the threads before this one, and over all (LDS: two barriers).
template <typename T>
__device__ __forceinline__ T scan_before(T v, T& total, T* sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T in = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(in, d);
        if (lane >= d) in += o;
    }
    __syncthreads();  // the sums of the previous call have been read
    if (lane == 63) sums[wave] = in;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    total = all;
    return before + in - v;
}

// The counts of pages 4 * i .. 4 * i + 3 (past the end: in use)
__device__ __forceinline__ void four_counts(const int32_t* count, int64_t pages, int64_t first, int32_t (&c)[4]) {
    if (first + 3 < pages && ((uintptr_t)count & 15) == 0) {
        const i32x4 v = *(const i32x4*)(count + first);
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k] = v[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k] = first + k < pages ? count[first + k] : 1;
    }
}

// The lowest `need` free pages, ascending, into out; returns how many there are (at most need).
__device__ int32_t lowest_free(const int32_t* count, int64_t pages, int32_t need, int32_t* out, int32_t* sums) {
    int32_t found = 0;
    for (int64_t base = 0; base < pages && found < need; base += 4 * kPlan) {
        const int64_t first = base + 4 * threadIdx.x;
        int32_t c[4], all;
        four_counts(count, pages, first, c);
        int32_t r = found + scan_before((c[0] <= 0) + (c[1] <= 0) + (c[2] <= 0) + (c[3] <= 0), all, sums);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c[k] <= 0) {
                if (r < need) out[r] = (int32_t)(first + k);
                ++r;
            }
        found += all;
    }
    return found < need ? found : need;
}

// Length of a sequence as the table can hold it.
__device__ __forceinline__ int32_t length_of(const PoolArgs& p, int64_t seq) {
    const int64_t most = p.table_width * p.page_size, n = p.lens[seq];
    return (int32_t)(n < 0 ? 0 : n > most ? most : n);
}

// ---------------------------------------------------------------- copies

template <typename T>
__device__ __forceinline__ void copy_piece(const char* s, char* d, int64_t bytes) {
    constexpr int kDeep = 4;
    const int64_t n = bytes / (int64_t)sizeof(T);
    const T* from = (const T*)s;
    T* to = (T*)d;
    for (int64_t i = threadIdx.x; i < n; i += kDeep * kCopy) {
        T v[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
            if (i + k * kCopy < n) v[k] = from[i + k * kCopy];
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
            if (i + k * kCopy < n) to[i + k * kCopy] = v[k];
    }
}

// Items (pair, tensor, piece) from `first` on, every `step`-th; pieces: of the largest page.
__device__ void copy_items(const PageList& list, int tensors, int64_t num_pages, const int32_t* src, const int32_t* dst,
                           int64_t pairs, int64_t pieces, int64_t first, int64_t step) {
    const int64_t per_pair = tensors * pieces;
    for (int64_t it = first; it < pairs * per_pair; it += step) {
        const int64_t pair = it / per_pair, rest = it % per_pair;
        const qk_pages t = list.t[rest / pieces];
        const int64_t at = (rest % pieces) * kPiece;
        const int32_t a = src[pair], b = dst[pair];
        if (a < 0 || b < 0 || a >= num_pages || b >= num_pages || at >= t.page_bytes) continue;
        const int64_t bytes = t.page_bytes - at < kPiece ? t.page_bytes - at : kPiece;
        const char* s = (const char*)t.base + a * t.page_stride + at;
        char* d = (char*)t.base + b * t.page_stride + at;
        const uintptr_t any = (uintptr_t)t.base | (uintptr_t)t.page_stride | (uintptr_t)t.page_bytes;
        if (any % 16 == 0) copy_piece<u32x4>(s, d, bytes);
        else if (any % 4 == 0) copy_piece<uint32_t>(s, d, bytes);
        else copy_piece<uint8_t>(s, d, bytes);
    }
}

__global__ __launch_bounds__(kCopy) void copy_pages(PageList list, int tensors, int64_t num_pages, const int32_t* src,
                                                    const int32_t* dst, int64_t pairs, int64_t pieces) {
    copy_items(list, tensors, num_pages, src, dst, pairs, pieces, blockIdx.x, gridDim.x);
}

int64_t pieces_of(const qk_pages* pages, int64_t tensors) {
    int64_t most = 1;
    for (int64_t i = 0; i < tensors; ++i) {
        const int64_t n = (pages[i].page_bytes + kPiece - 1) / kPiece;
        if (n > most) most = n;
    }
    return most;
}

// Calls launch(list, tensors in it, pieces of its largest page) for every kTensors tensors; once with none if there are none.
template <typename F>
hipError_t for_lists(const qk_pages* pages, int64_t tensors, F launch) {
    int64_t i = 0;
    do {
        PageList list = {};
        const int n = (int)(tensors - i < kTensors ? tensors - i : kTensors);
        for (int k = 0; k < n; ++k) list.t[k] = pages[i + k];
        launch(list, n, pieces_of(pages + i, n), i == 0);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        i += kTensors;
    } while (i < tensors);
    return hipSuccess;
}

// Workgroups for a number of items that may be large: as many as are resident four times over take them in turn (2048: 2 % slower).
unsigned copy_grid(int64_t items) {
    const int64_t most = 8192;
    return (unsigned)(items < 1 ? 1 : items < most ? items : most);
}

// ---------------------------------------------------------------- fork

// ws: [n] source pages, [n] destination pages (-1: none), [1] whether there are enough
__global__ __launch_bounds__(kPlan) void fork_plan(PoolArgs p, const int32_t* parents, const int32_t* children, int64_t n,
                                                   int32_t* missing, int32_t* ws) {
    __shared__ int32_t sums[kWaves];
    int32_t *src = ws, *dst = ws + n;
    int32_t need = 0;
    for (int64_t base = 0; base < n; base += kPlan) {
        const int64_t i = base + threadIdx.x;
        int32_t page = -1;
        bool started = false;
        if (i < n) {
            const int32_t from = parents[i], to = children[i];
            if (from >= 0 && from < p.max_seqs && to >= 0 && to < p.max_seqs) {
                const int32_t len = length_of(p, from);
                started = len % p.page_size != 0;
                if (started) page = p.table[from * p.table_stride + len / p.page_size];
            }
        }
        int32_t all;
        const int32_t rank = need + scan_before((int32_t)started, all, sums);
        need += all;
        if (i < n) {
            src[i] = page;
            dst[i] = started ? rank : -1;  // its place among the new pages, for now
        }
    }
    // the free pages go where the pairs' ranks can find them: behind the flag
    int32_t* fresh = ws + 2 * n + 1;
    const int32_t found = lowest_free(p.count, p.num_pages, need, fresh, sums);
    if (threadIdx.x == 0) {
        missing[0] = need - found;
        ws[2 * n] = need == found;
    }
    __syncthreads();
    if (need != found) return;
    for (int64_t i = threadIdx.x; i < n; i += kPlan)
        if (dst[i] >= 0) dst[i] = fresh[dst[i]];
}

// The first `rows` workgroups write the children's rows, lengths and counts; the others copy the started pages.
__global__ __launch_bounds__(kCopy) void fork_do(PageList list, int tensors, int64_t pieces, PoolArgs p,
                                                 const int32_t* parents, const int32_t* children, int64_t n, int64_t rows,
                                                 const int32_t* ws) {
    if (!ws[2 * n]) return;
    const int32_t *src = ws, *dst = ws + n;
    if ((int64_t)blockIdx.x >= rows) {
        copy_items(list, tensors, p.num_pages, src, dst, n, pieces, blockIdx.x - rows, gridDim.x - rows);
        return;
    }
    const int64_t i = blockIdx.x;
    const int32_t from = parents[i], to = children[i];
    if (from < 0 || from >= p.max_seqs || to < 0 || to >= p.max_seqs) return;
    const int32_t len = length_of(p, from), whole = (int32_t)(len / p.page_size);
    for (int64_t j = threadIdx.x; j < p.table_width; j += kCopy) {
        int32_t page = p.table[from * p.table_stride + j];
        if (j < whole) {
            if (page >= 0 && page < p.num_pages) atomicAdd(p.count + page, 1);
        } else if (j == whole && dst[i] >= 0) {
            page = dst[i];
            p.count[page] = 1;
        }
        p.table[to * p.table_stride + j] = page;
    }
    if (threadIdx.x == 0) p.lens[to] = len;
}

// ---------------------------------------------------------------- free

__global__ __launch_bounds__(kCopy) void free_seqs(PoolArgs p, const int32_t* seqs) {
    const int32_t seq = seqs[blockIdx.x];
    if (seq < 0 || seq >= p.max_seqs) return;
    const int64_t held = (length_of(p, seq) + p.page_size - 1) / p.page_size;
    for (int64_t j = threadIdx.x; j < held; j += kCopy) {
        // the exchange hands each entry to one workgroup, should the sequence be named twice
        const int32_t page = atomicExch(p.table + seq * p.table_stride + j, -1);
        if (page >= 0 && page < p.num_pages && atomicSub(p.count + page, 1) <= 0) atomicAdd(p.count + page, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) p.lens[seq] = 0;
}

// ---------------------------------------------------------------- extend

__device__ __forceinline__ int64_t grown_by(const int32_t* cu, int64_t i) {
    const int64_t d = (int64_t)cu[i + 1] - cu[i];
    return d < 0 ? 0 : d;
}

// The last i < n with v[i] <= x (v not falling, v[0] <= x)
__device__ __forceinline__ int64_t last_at_most(const int32_t* v, int64_t n, int32_t x) {
    int64_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) / 2;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Slot and position of new token t, the sequences' lengths being the new ones.
__device__ __forceinline__ void place_token(const PoolArgs& p, const int32_t* seqs, const int32_t* cu, int64_t n, int64_t t,
                                            bool ok, int32_t* slots, int32_t* positions) {
    int32_t slot = -1, position = -1;
    if (ok && n > 0 && t >= cu[0] && t < cu[n]) {
        const int64_t i = last_at_most(cu, n, (int32_t)t);
        const int32_t seq = seqs[i];
        if (seq >= 0 && seq < p.max_seqs) {
            position = (int32_t)(p.lens[seq] - grown_by(cu, i) + (t - cu[i]));
            const int64_t at = position / p.page_size;
            if (position >= 0 && at < p.table_width)
                slot = (int32_t)(p.table[seq * p.table_stride + at] * p.page_size + position % p.page_size);
        }
    }
    slots[t] = slot;
    positions[t] = position;
}

// ws: [n] first new page of each sequence, [need] the pages.  Slots of up to kPlan tokens are written here too.  T: of the
// pages' sum, 64 bits where the sequences could ask for 2^31 and more between them (cu_tokens that fall, and rise again,
// ask for any number: 64 bits throughout take 7.4 us for 64 sequences, 32 bits 6.5).
template <typename T>
__global__ __launch_bounds__(kPlan) void extend_plan(PoolArgs p, const int32_t* seqs, const int32_t* cu, int64_t n,
                                                     int64_t total, int32_t* slots, int32_t* positions, int32_t* missing,
                                                     int32_t* ws) {
    __shared__ int32_t sums[kWaves];
    __shared__ T counts[kWaves];
    __shared__ int64_t wide[kWaves];
    int32_t *first = ws, *fresh = ws + n;
    T need = 0;
    int64_t over = 0;
    for (int64_t base = 0; base < n; base += kPlan) {
        const int64_t i = base + threadIdx.x;
        T pages = 0;
        int64_t excess = 0;
        if (i < n && seqs[i] >= 0 && seqs[i] < p.max_seqs) {
            const int64_t old = length_of(p, seqs[i]), len = old + grown_by(cu, i);
            const int64_t now = (len + p.page_size - 1) / p.page_size;
            if (now > p.table_width) excess = now - p.table_width;
            else pages = (T)(now - (old + p.page_size - 1) / p.page_size);
        }
        T all;
        const T rank = need + scan_before(pages, all, counts);
        need += all;
        if (i < n) first[i] = (int32_t)rank;  // read only where all ranks fit the pool
        if (__syncthreads_or(excess != 0)) {
            int64_t columns;
            scan_before(excess, columns, wide);
            over += columns;
        }
    }
    int64_t lack = over;
    if (!lack) {
        const int32_t most = (int32_t)(need < p.num_pages ? need : p.num_pages);
        lack = need - lowest_free(p.count, p.num_pages, most, fresh, sums);
    }
    if (threadIdx.x == 0) missing[0] = (int32_t)(lack < 0x7fffffff ? lack : 0x7fffffff);
    __syncthreads();
    if (!lack) {
        for (int32_t r = threadIdx.x; r < need; r += kPlan) {
            const int64_t i = last_at_most(first, n, r);
            const int64_t old = length_of(p, seqs[i]);
            p.table[seqs[i] * p.table_stride + (old + p.page_size - 1) / p.page_size + (r - first[i])] = fresh[r];
            p.count[fresh[r]] = 1;
        }
        __syncthreads();
        for (int64_t i = threadIdx.x; i < n; i += kPlan)
            if (seqs[i] >= 0 && seqs[i] < p.max_seqs) p.lens[seqs[i]] = (int32_t)(length_of(p, seqs[i]) + grown_by(cu, i));
        __syncthreads();
    }
    if (total <= kPlan && (int64_t)threadIdx.x < total)
        place_token(p, seqs, cu, n, threadIdx.x, lack == 0, slots, positions);
}

__global__ __launch_bounds__(kCopy) void extend_slots(PoolArgs p, const int32_t* seqs, const int32_t* cu, int64_t n,
                                                      int64_t total, int32_t* slots, int32_t* positions,
                                                      const int32_t* missing) {
    const int64_t t = (int64_t)blockIdx.x * kCopy + threadIdx.x;
    if (t < total) place_token(p, seqs, cu, n, t, missing[0] == 0, slots, positions);
}

// ---------------------------------------------------------------- compact

// ws: [1] pairs, then [num_pages] places, [num_pages / 2 + 1] sources, [num_pages / 2 + 1] destinations
struct CompactWs {
    int32_t *pairs, *place, *src, *dst;
};
__host__ __device__ inline CompactWs compact_ws(int32_t* ws, int64_t pages) {
    const int64_t half = pages / 2 + 1;
    return {ws, ws + 1, ws + 1 + pages, ws + 1 + pages + half};
}

__global__ __launch_bounds__(kPlan) void compact_plan(PoolArgs p, int32_t* new_count, int32_t* moved, int32_t* ws_) {
    __shared__ int32_t sums[kWaves];
    const CompactWs ws = compact_ws(ws_, p.num_pages);
    int32_t mine = 0, live;
    for (int64_t base = 0; base < p.num_pages; base += 4 * kPlan) {
        const int64_t first = base + 4 * threadIdx.x;
        int32_t c[4];
        four_counts(p.count, p.num_pages, first, c);
#pragma unroll
        for (int k = 0; k < 4; ++k) mine += first + k < p.num_pages && c[k] > 0;
    }
    scan_before(mine, live, sums);
    int32_t srcs = 0, dsts = 0;
    for (int64_t base = 0; base < p.num_pages; base += 4 * kPlan) {
        const int64_t first = base + 4 * threadIdx.x;
        int32_t c[4], n_src = 0, n_dst = 0, all;
        four_counts(p.count, p.num_pages, first, c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t id = first + k;
            n_src += id < p.num_pages && id >= live && c[k] > 0;
            n_dst += id < live && c[k] <= 0;
        }
        int32_t r_src = srcs + scan_before(n_src, all, sums);
        srcs += all;
        int32_t r_dst = dsts + scan_before(n_dst, all, sums);
        dsts += all;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t id = first + k;
            if (id >= p.num_pages) continue;
            ws.place[id] = (int32_t)id;
            new_count[id] = c[k] > 0 ? c[k] : 0;
            if (id >= live && c[k] > 0) ws.src[r_src++] = (int32_t)id;
            if (id < live && c[k] <= 0) ws.dst[r_dst++] = (int32_t)id;
        }
    }
    __syncthreads();
    for (int32_t k = threadIdx.x; k < srcs; k += kPlan) {
        const int32_t from = ws.src[k], to = ws.dst[k];
        ws.place[from] = to;
        new_count[to] = p.count[from];
        new_count[from] = 0;
    }
    if (threadIdx.x == 0) moved[0] = ws.pairs[0] = srcs;
}

// The first `rows` workgroups write the new table, the others copy the pages.
__global__ __launch_bounds__(kCopy) void compact_do(PageList list, int tensors, int64_t pieces, PoolArgs p,
                                                    int32_t* new_table, int64_t rows, int32_t* ws_) {
    const CompactWs ws = compact_ws(ws_, p.num_pages);
    if ((int64_t)blockIdx.x >= rows) {
        copy_items(list, tensors, p.num_pages, ws.src, ws.dst, ws.pairs[0], pieces, blockIdx.x - rows, gridDim.x - rows);
        return;
    }
    const int64_t n = p.max_seqs * p.table_width;
    for (int64_t i = (int64_t)blockIdx.x * kCopy + threadIdx.x; i < n; i += rows * kCopy) {
        const int32_t page = p.table[(i / p.table_width) * p.table_stride + i % p.table_width];
        new_table[i] = page >= 0 && page < p.num_pages ? ws.place[page] : page;
    }
}

}  // namespace

hipError_t launch_kv_copy_pages(const qk_pages* pages, int64_t tensors, int64_t num_pages, const int32_t* src,
                                const int32_t* dst, int64_t n, hipStream_t stream) {
    return for_lists(pages, tensors, [&](const PageList& list, int k, int64_t pieces, bool) {
        copy_pages<<<copy_grid(n * k * pieces), kCopy, 0, stream>>>(list, k, num_pages, src, dst, n, pieces);
    });
}

size_t kv_fork_workspace(int64_t n) { return (size_t)(3 * n + 1) * sizeof(int32_t); }

hipError_t launch_kv_fork(const qk_pages* pages, int64_t tensors, const PoolArgs& p, const int32_t* parents,
                          const int32_t* children, int64_t n, int32_t* missing, void* ws, hipStream_t stream) {
    fork_plan<<<1, kPlan, 0, stream>>>(p, parents, children, n, missing, (int32_t*)ws);
    if (const hipError_t e = hipGetLastError()) return e;
    if (n == 0) return hipSuccess;
    return for_lists(pages, tensors, [&](const PageList& list, int k, int64_t pieces, bool first) {
        const int64_t rows = first ? n : 0;
        const unsigned copies = k ? copy_grid(n * k * pieces) : 0;
        fork_do<<<dim3((unsigned)rows + copies), kCopy, 0, stream>>>(list, k, pieces, p, parents, children, n, rows,
                                                                    (const int32_t*)ws);
    });
}

hipError_t launch_kv_free(const PoolArgs& p, const int32_t* seqs, int64_t n, hipStream_t stream) {
    free_seqs<<<dim3((unsigned)n), kCopy, 0, stream>>>(p, seqs);
    return hipGetLastError();
}

size_t kv_extend_workspace(int64_t n, int64_t num_pages) { return (size_t)(n + num_pages) * sizeof(int32_t); }

hipError_t launch_kv_extend(const PoolArgs& p, const int32_t* seqs, const int32_t* cu, int64_t n, int64_t total,
                            int32_t* slots, int32_t* positions, int32_t* missing, void* ws, hipStream_t stream) {
    const bool wide = p.table_width > 0x7fffffff / (n < 1 ? 1 : n);  // no sequence takes more pages than the table has columns
    if (wide) extend_plan<int64_t><<<1, kPlan, 0, stream>>>(p, seqs, cu, n, total, slots, positions, missing, (int32_t*)ws);
    else extend_plan<int32_t><<<1, kPlan, 0, stream>>>(p, seqs, cu, n, total, slots, positions, missing, (int32_t*)ws);
    if (const hipError_t e = hipGetLastError()) return e;
    if (total <= kPlan) return hipSuccess;
    extend_slots<<<dim3((unsigned)((total + kCopy - 1) / kCopy)), kCopy, 0, stream>>>(p, seqs, cu, n, total, slots,
                                                                                     positions, missing);
    return hipGetLastError();
}

size_t kv_compact_workspace(int64_t num_pages) {
    return (size_t)(1 + num_pages + 2 * (num_pages / 2 + 1)) * sizeof(int32_t);
}

hipError_t launch_kv_compact(const qk_pages* pages, int64_t tensors, const PoolArgs& p, int32_t* new_table,
                             int32_t* new_count, int32_t* moved, void* ws, hipStream_t stream) {
    compact_plan<<<1, kPlan, 0, stream>>>(p, new_count, moved, (int32_t*)ws);
    if (const hipError_t e = hipGetLastError()) return e;
    const int64_t entries = p.max_seqs * p.table_width;
    return for_lists(pages, tensors, [&](const PageList& list, int k, int64_t pieces, bool first) {
        int64_t rows = first ? (entries + kCopy * 8 - 1) / (kCopy * 8) : 0;
        if (rows > 1024) rows = 1024;
        const unsigned copies = k ? copy_grid(p.num_pages / 2 * k * pieces) : 0;
        if (rows + copies == 0) return;
        compact_do<<<dim3((unsigned)rows + copies), kCopy, 0, stream>>>(list, k, pieces, p, new_table, rows, (int32_t*)ws);
    });
}

}  // namespace qk
