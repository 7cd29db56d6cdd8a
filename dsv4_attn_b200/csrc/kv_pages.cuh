// Pages of the cache: copying, forking, freeing, compacting; and moving single entries.
//
// A page holds 64 entries of 656 bytes; a pool has `layers` times `num_pages` of them, one block table per request serves all layers.
// refs[p] counts the block-table slots that hold page p; a page with a count of 0 is free.  The bytes that move bound the large
// calls (a copy reads and writes every byte once), launches and the chain lengths -> table -> page the small ones.  Every answer is a
// function of the arguments alone: free pages are taken in ascending order, and counts are integers, whose atomics commute.
//
// Measured: a pool of 4,600 pages in eight layers packed (751 MB moved) 126 us, 5.9 TB/s, of which the plan by one block is 9; 48 requests of 4,000 entries
// forked through 16 layers 12.8 us and four in one layer 8.6, two launches in a chain each; accepted rows of 64 requests in 16 layers 3.7, of which the comparison of the lists is 0.8;
// where lists overlap: five rows each of 64 requests in 16 layers 8.0, 64 windows of 128 rows that slide in 16 layers 160.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"
#include "decode_kernel.cuh"

namespace dsv4 {

constexpr int kPageEntries = 64;
constexpr int kEntryVecs = 41;                                   // 656 bytes as 16-byte vectors
constexpr int kPageVecs = kPageEntries * kEntryVecs;             // 2624
constexpr int kPagesThreads = 256;
constexpr int kPagesPlanThreads = 1024;
// A warp copies 256 vectors (4 KB) at a time, eight loads in flight per lane: 16 warps an SM then have more on the way than a DRAM
// access takes, and a single page still spreads over eleven warps.
constexpr int kCopyVecs = 256;
constexpr int kCopyBatches = (kPageVecs + kCopyVecs - 1) / kCopyVecs;
constexpr int kStatusNoPage = 10;                                // a fork found no free page
constexpr int kStatusOverlap = 11;                               // too long a list of copies or moves whose sources and destinations overlap
// Comparing the lists of a copy or a move.
constexpr int kMeetTable = 4096, kMeetFew = kMeetTable / 2;
constexpr int kMoveThreads = 512, kMoveBlocks = 2;                // an SM
constexpr int kMoveStage = 16384;                                // 32-bit words of a column
constexpr int kMoveGroup = kCopyVecs / kEntryVecs;               // entries of a warp at a time, at most

struct KvPagesArgs {
    uint4* pool;                 // [layers, num_pages, 64, 656 bytes]
    int64_t num_pages, layers;
    int B, max_pages;
    int n;                       // copy: pairs; fork: children; free: requests
    const int32_t* src;          // copy: pages; fork: parents; free: requests; move: entries
    const int32_t* dst;          // copy: pages; fork: children; move: entries
    int32_t* block_table;        // [B, max_pages]
    int32_t* kv_len;             // [B]
    int32_t* refs;               // [num_pages]
    // compact
    int32_t* new_table;          // may be block_table
    int32_t* new_refs;           // may be refs
    int32_t* count;              // live pages
    int32_t* from;               // scratch [num_pages]: pages that move, ascending
    int32_t* to;                 // scratch [num_pages]: where they go, ascending
    int32_t* moves;              // scratch [1]: how many move
    int64_t entries;             // move: entries per layer
    int width;                   // move: words of an entry in a column
    int group;                   // move: entries of a warp at a time
    int32_t* status;
};

// Vectors [at, at + 256) of `total`, from src to dst, by one warp.
__device__ __forceinline__ void copy_batch(uint4* dst, const uint4* src, int at, int total, int lane) {
    uint4 v[kCopyVecs / 32];
#pragma unroll
    for (int i = 0; i < kCopyVecs / 32; ++i)
        if (at + i * 32 + lane < total) v[i] = ptx::ldg_stream_v4(src + at + i * 32 + lane);
#pragma unroll
    for (int i = 0; i < kCopyVecs / 32; ++i)
        if (at + i * 32 + lane < total) dst[at + i * 32 + lane] = v[i];
}

__device__ __forceinline__ bool in_pool(const KvPagesArgs& a, int page) { return page >= 0 && page < a.num_pages; }

// Whether pair i, of items below `count`, is copied: a negative number leaves it out, and so does one out of range.
__device__ __forceinline__ bool item_pair(const KvPagesArgs& a, int64_t count, int i, int& s, int& d) {
    s = ptx::ld(a.src + i);
    d = ptx::ld(a.dst + i);
    return s >= 0 && d >= 0 && s < count && d < count;
}

// Whether any item is in both lists, found out by one block; every thread calls.  A bit per item of the pool, ROOM of them at a time: the sources set theirs, the
// destinations look.  Short lists in a pool of more than ROOM: a table of the sources, at most half full.
template <int THREADS, int ROOM>
struct Meet {
    static_assert(ROOM / 8 >= kMeetTable * 4, "room for the table");
    static __host__ __device__ bool by_table(int n, int64_t count) { return n <= kMeetFew && count > ROOM; }
    // (shared memory that it takes)
    static __host__ __device__ int bytes(int n, int64_t count) { return by_table(n, count) ? kMeetTable * 4 : int((count < ROOM ? count : ROOM) + 127) / 128 * 16; }
    // (needs no global memory: before the wait)
    static __device__ __forceinline__ void clear(const KvPagesArgs& a, int64_t count, int32_t* words) {
        const int vecs = bytes(a.n, count) / 16, fill = by_table(a.n, count) ? -1 : 0;
        for (int i = threadIdx.x; i < vecs; i += THREADS) reinterpret_cast<int4*>(words)[i] = make_int4(fill, fill, fill, fill);
        __syncthreads();
    }
    static __device__ __forceinline__ bool find(const KvPagesArgs& a, int64_t count, int32_t* words) {
        const uint32_t n = uint32_t(a.n), tid = threadIdx.x;      // (a counter that passes n may pass 2^31)
        if (by_table(a.n, count)) {
            auto place_of = [](int item) { return (uint32_t(item) * 2654435769u) >> 20; };       // 12 bits; then the first free place from there on
            constexpr uint32_t kLast = kMeetTable - 1;
            for (uint32_t i = tid; i < n; i += THREADS) {
                int s, d;
                if (!item_pair(a, count, int(i), s, d)) continue;
                for (uint32_t at = place_of(s);; at = (at + 1u) & kLast) {
                    const int there = atomicCAS(&words[at], -1, s);
                    if (there == -1 || there == s) break;
                }
            }
            __syncthreads();
            bool mine = false;
            for (uint32_t i = tid; i < n; i += THREADS) {
                int s, d;
                if (item_pair(a, count, int(i), s, d))
                    for (uint32_t at = place_of(d); words[at] != -1; at = (at + 1u) & kLast) mine |= words[at] == d;
            }
            return __syncthreads_or(mine);
        }
        uint32_t* const bits = reinterpret_cast<uint32_t*>(words);
        for (int64_t begin = 0;;) {
            const int64_t end = min(count, begin + ROOM);
#pragma unroll 4
            for (uint32_t i = tid; i < n; i += THREADS) {
                int s, d;
                if (item_pair(a, count, int(i), s, d) && s >= begin && s < end) atomicOr(&bits[(s - begin) >> 5], 1u << ((s - begin) & 31));
            }
            __syncthreads();
            bool mine = false;
#pragma unroll 4
            for (uint32_t i = tid; i < n; i += THREADS) {
                int s, d;
                if (item_pair(a, count, int(i), s, d) && d >= begin && d < end) mine |= (bits[(d - begin) >> 5] >> ((d - begin) & 31)) & 1u;
            }
            if (__syncthreads_or(mine)) return true;
            begin = end;
            if (begin >= count) return false;
            for (uint32_t i = tid; i < ROOM / 32; i += THREADS) bits[i] = 0u;
            __syncthreads();
        }
    }
};
using PagesMeet = Meet<kPagesThreads, 1 << 17>;
using EntriesMeet = Meet<kMoveThreads, kMoveStage * 32>;

// Page src[i] of every layer to page dst[i].  A negative number leaves the pair out; one beyond the pool is reported.  So are lists that overlap, by a block
// more (where there is a status): nobody waits for it, and what such pages hold is not known afterwards.
__global__ void __launch_bounds__(kPagesThreads) kv_copy_pages_kernel(const __grid_constant__ KvPagesArgs a) {
    extern __shared__ __align__(16) int32_t s_words[];
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int blocks = int(gridDim.x) - (a.status != nullptr), lane = threadIdx.x & 31;
    if (int(blockIdx.x) == blocks) {
        PagesMeet::clear(a, a.num_pages, s_words);
        if (PagesMeet::find(a, a.num_pages, s_words) && threadIdx.x == 0) report_status(a.status, kStatusOverlap, 6, a.n);
        return;
    }
    const int64_t units = int64_t(a.n) * a.layers * kCopyBatches;
    for (int64_t u = int64_t(blockIdx.x) * (kPagesThreads / 32) + (threadIdx.x >> 5); u < units; u += int64_t(blocks) * (kPagesThreads / 32)) {
        const int batch = int(u % kCopyBatches);
        const int64_t page = u / kCopyBatches, layer = page / a.n;
        int s, d;
        if (!item_pair(a, a.num_pages, int(page % a.n), s, d)) {
            if (lane == 0 && s >= 0 && d >= 0) report_status(a.status, kStatusBadIndex, 6, int(page % a.n));
            continue;
        }
        copy_batch(a.pool + (layer * a.num_pages + d) * kPageVecs, a.pool + (layer * a.num_pages + s) * kPageVecs, batch * kCopyVecs, kPageVecs, lane);
    }
}

// Moved entries of lists that overlap.  The same few words of every entry, a.width of T, are a column of a layer; no two columns touch the same bytes.  A block
// brings a column of all entries to shared memory, meets, and writes it.
template <typename T>
__device__ __forceinline__ void move_columns(const KvPagesArgs& a, T* s_stage) {
    constexpr int kWords = kEntryVecs * 16 / int(sizeof(T));
    const int tid = threadIdx.x;
    const int64_t columns = (kWords + a.width - 1) / a.width, units = columns * a.layers;
#pragma unroll 1
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int first = int(u % columns) * a.width, w = min(a.width, kWords - first), total = a.n * w;
        T* const base = reinterpret_cast<T*>(a.pool) + u / columns * a.entries * kWords + first;
#pragma unroll 4
        for (int at = tid; at < total; at += kMoveThreads) {
            const int i = at / w;
            int s, d;
            if (item_pair(a, a.entries, i, s, d)) s_stage[at] = ptx::ld(base + int64_t(s) * kWords + (at - i * w));
        }
        __syncthreads();
        // (a thread takes back what it put there: the next column needs no barrier before it)
#pragma unroll 4
        for (int at = tid; at < total; at += kMoveThreads) {
            const int i = at / w;
            int s, d;
            if (item_pair(a, a.entries, i, s, d)) base[int64_t(d) * kWords + (at - i * w)] = s_stage[at];
        }
    }
}

// Entry src[i] of every layer to entry dst[i] (numbers within a layer), as if all were read before any is written: accepted rows close up, a window slides.
// A warp takes up to six entries of a layer at a time.  The first ones are on their way while every block finds out whether the lists overlap; if they do not, as
// with rows that go to places of their own, the order does not matter; else the entries go by columns, as long as one of a single 32-bit word fits.
__global__ void __launch_bounds__(kMoveThreads, kMoveBlocks) kv_move_entries_kernel(const __grid_constant__ KvPagesArgs a) {
    extern __shared__ __align__(16) uint4 s_stage[];
    int32_t* const s_words = reinterpret_cast<int32_t*>(s_stage);
    ptx::pdl_trigger();
    EntriesMeet::clear(a, a.entries, s_words);
    ptx::pdl_wait();
    constexpr int kWarps = kMoveThreads / 32;
    const int lane = threadIdx.x & 31, vecs = a.group * kEntryVecs;
    const int64_t groups = (a.n + a.group - 1) / a.group, units = groups * a.layers;
    int64_t u = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    uint4 v[kCopyVecs / 32];
    int to = -1;                                       // of entry `lane` of the group
    uint4* base = a.pool;
    auto read = [&]() {
        const int64_t i = u % groups * a.group + lane;
        int s = -1;
        to = -1;
        if (u < units && lane < a.group && i < a.n && !item_pair(a, a.entries, int(i), s, to)) {
            if (s >= 0 && to >= 0) report_status(a.status, kStatusBadIndex, 6, int(i));
            to = -1;
        }
        base = a.pool + u / groups * a.entries * kEntryVecs;
#pragma unroll
        for (int j = 0; j < kCopyVecs / 32; ++j) {
            if (j * 32 >= vecs) break;
            const int at = j * 32 + lane, of = at / kEntryVecs, s_of = __shfl_sync(0xFFFFFFFFu, s, of), to_of = __shfl_sync(0xFFFFFFFFu, to, of);
            if (at < vecs && to_of >= 0) v[j] = ptx::ldg_stream_v4(base + int64_t(s_of) * kEntryVecs + (at - of * kEntryVecs));
        }
    };
    read();
    if (EntriesMeet::find(a, a.entries, s_words)) {
        if (blockIdx.x == 0)                           // (those that no warp has come to)
            for (uint32_t i = threadIdx.x; i < uint32_t(a.n); i += kMoveThreads) {
                int s, d;
                if (!item_pair(a, a.entries, int(i), s, d) && s >= 0 && d >= 0) report_status(a.status, kStatusBadIndex, 6, int(i));
            }
        if (a.n <= kMoveStage / 4) move_columns(a, s_stage);
        else if (a.n <= kMoveStage) move_columns(a, s_words);
        else if (blockIdx.x == 0 && threadIdx.x == 0) report_status(a.status, kStatusOverlap, 6, a.n);
        return;
    }
#pragma unroll 1
    for (;;) {
#pragma unroll
        for (int j = 0; j < kCopyVecs / 32; ++j) {
            if (j * 32 >= vecs) break;
            const int at = j * 32 + lane, of = at / kEntryVecs, to_of = __shfl_sync(0xFFFFFFFFu, to, of);
            if (at < vecs && to_of >= 0) base[int64_t(to_of) * kEntryVecs + (at - of * kEntryVecs)] = v[j];
        }
        u += int64_t(gridDim.x) * kWarps;
        if (u >= units) break;
        read();
    }
}

// The pages of request src[i] are given back: one reference less each, its row of the table -1, its length 0.  One block per request: all
// of its threads have read the length before the barrier behind which it is written.
__global__ void __launch_bounds__(kPagesThreads) kv_free_kernel(const __grid_constant__ KvPagesArgs a) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int r = ptx::ld(a.src + blockIdx.x);
    if (r < 0) return;
    if (r >= a.B) {
        if (threadIdx.x == 0) report_status(a.status, kStatusBadIndex, 6, int(blockIdx.x));
        return;
    }
    const int len = ptx::ld(a.kv_len + r), held = len > 0 ? (len - 1) / kPageEntries + 1 : 0;
    int32_t* row = a.block_table + int64_t(r) * a.max_pages;
    for (int i = threadIdx.x; i < a.max_pages; i += kPagesThreads) {
        const int page = row[i];
        if (i < held && in_pool(a, page)) atomicSub(a.refs + page, 1);
        row[i] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) a.kv_len[r] = 0;
}

// A parent's length as a fork sees it.
__device__ __forceinline__ int fork_length(const KvPagesArgs& a, int parent) {
    return int(min(int64_t(max(ptx::ld(a.kv_len + parent), 0)), int64_t(a.max_pages) * kPageEntries));
}
__device__ __forceinline__ bool fork_pair(const KvPagesArgs& a, int i, int& parent, int& child) {
    parent = ptx::ld(a.src + i);
    child = ptx::ld(a.dst + i);
    return parent >= 0 && parent < a.B && child >= 0 && child < a.B;
}

// Exclusive prefix sum of `v` over the block, and the block's total; every thread calls.
__device__ __forceinline__ int block_prefix(int v, int* s_warp, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                  // the sums of the call before have been read
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xFFFFFFFFu, w, 31);
    return x - v + (warp > 0 ? __shfl_sync(0xFFFFFFFFu, w, warp - 1) : 0);
}

// A planning block goes through the counts 16 neighbouring pages a thread at a time, with four loads in flight each (100,000 pages: four at a time took 66 us for
// a compaction's plan).
constexpr int kPlanPages = 16, kPlanChunk = kPagesPlanThreads * kPlanPages;
// Bit j: page p + j is one of the pool and held.
__device__ __forceinline__ uint32_t held_pages(const KvPagesArgs& a, int64_t p, int32_t (&refs)[kPlanPages]) {
    if (p + kPlanPages <= a.num_pages && (reinterpret_cast<uintptr_t>(a.refs) & 15u) == 0u) {
#pragma unroll
        for (int j = 0; j < kPlanPages / 4; ++j) {
            const int4 v = ptx::ld(reinterpret_cast<const int4*>(a.refs + p) + j);
            refs[4 * j] = v.x;  refs[4 * j + 1] = v.y;  refs[4 * j + 2] = v.z;  refs[4 * j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kPlanPages; ++j) refs[j] = p + j < a.num_pages ? ptx::ld(a.refs + p + j) : 0;
    }
    uint32_t held = 0u;
#pragma unroll
    for (int j = 0; j < kPlanPages; ++j) held |= uint32_t(refs[j] > 0) << j;
    return held;
}
// Bit j: page p + j is one of the pool.
__device__ __forceinline__ uint32_t pool_pages(const KvPagesArgs& a, int64_t p) {
    return p + kPlanPages <= a.num_pages ? (1u << kPlanPages) - 1u : (p < a.num_pages ? (1u << (a.num_pages - p)) - 1u : 0u);
}

// First half of a fork, one block: the children whose parent ends in a partly filled page get the lowest-numbered free pages, in the order
// of the children.  Writes those pages' table slots and counts, and the children's lengths:
// places that it does not read again, the lengths because no child is a parent, the counts because a later round looks at pages from `next` on.
__global__ void __launch_bounds__(kPagesPlanThreads) kv_fork_plan_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ int s_warp[32];
    __shared__ int s_free[kPagesPlanThreads];          // free pages for the children of this round
    __shared__ int s_last;
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int tid = threadIdx.x;
    int64_t page0 = 0, next = 0;                       // pages before `next` are taken; page0: where to look, a multiple of 16
    for (int base = 0; base < a.n; base += kPagesPlanThreads) {
        const int i = base + tid;
        int parent = 0, child = 0, len = 0;
        bool ok = false;
        if (i < a.n) {
            ok = fork_pair(a, i, parent, child);
            if (!ok && (parent >= 0 && child >= 0)) report_status(a.status, kStatusBadIndex, 6, i);
            if (ok) len = fork_length(a, parent);
        }
        const bool need = len % kPageEntries != 0;
        int wanted, found = 0;
        const int rank = block_prefix(need ? 1 : 0, s_warp, wanted);
        // pages in ascending order until there are enough
        while (found < wanted && page0 < a.num_pages) {
            const int64_t p = page0 + tid * kPlanPages;
            int32_t refs[kPlanPages];
            uint32_t free_bits = ~held_pages(a, p, refs) & pool_pages(a, p);
            if (p < next) free_bits &= next - p >= kPlanPages ? 0u : ~0u << (next - p);        // (taken in the round before)
            int in_chunk, at = found + block_prefix(__popc(free_bits), s_warp, in_chunk);
            for (uint32_t bits = free_bits; bits != 0u && at < wanted; bits &= bits - 1u, ++at) {
                const int page = int(p) + __ffs(bits) - 1;
                s_free[at] = page;
                if (at == wanted - 1) s_last = page;
            }
            __syncthreads();
            found += in_chunk;
            if (found >= wanted) {
                // (the next round begins behind the last page taken, in the same group of 16)
                next = int64_t(s_last) + 1;
                page0 = next / kPlanPages * kPlanPages;
            } else {
                page0 += kPlanChunk;
            }
        }
        if (ok) {
            const int full = len / kPageEntries;
            if (need) {
                const bool has = rank < found;
                const int page = has ? s_free[rank] : -1;
                a.block_table[int64_t(child) * a.max_pages + full] = page;
                if (has) a.refs[page] = 1;
                else report_status(a.status, kStatusNoPage, 6, i);
                if (!has) len = full * kPageEntries;
            }
            a.kv_len[child] = len;
        }
        __syncthreads();                               // s_free is read before the next round fills it
    }
}

// Second half: units of a child are its table row and 4 KB batches of its partly filled page in every layer.  (A row's unit leaves the slot of that page, which the
// batches read, as the plan wrote it; parents' rows are only read.)
__global__ void __launch_bounds__(kPagesThreads) kv_fork_apply_kernel(const __grid_constant__ KvPagesArgs a) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t per_child = 1 + a.layers * kCopyBatches, units = a.n * per_child;
    for (int64_t u = int64_t(blockIdx.x) * (kPagesThreads / 32) + (threadIdx.x >> 5); u < units; u += int64_t(gridDim.x) * (kPagesThreads / 32)) {
        // (rows first, batches afterwards: neighbouring warps then copy neighbouring bytes)
        const bool row = u < a.n;
        const int64_t v = u - a.n;
        const int i = row ? int(u) : int(v / (a.layers * kCopyBatches));
        int parent, child;
        if (!fork_pair(a, i, parent, child)) continue;
        const int len = fork_length(a, parent), full = len / kPageEntries, rest = len % kPageEntries;
        const int32_t* from = a.block_table + int64_t(parent) * a.max_pages;
        int32_t* to = a.block_table + int64_t(child) * a.max_pages;
        if (row) {
            for (int k = lane; k < a.max_pages; k += 32) {
                if (k < full) {
                    const int page = ptx::ld(from + k);
                    to[k] = page;
                    if (in_pool(a, page)) atomicAdd(a.refs + page, 1);
                } else if (k > full || rest == 0) {
                    to[k] = -1;
                }
            }
        } else if (rest != 0) {
            const int s = ptx::ld(from + full), d = ptx::ld(to + full);
            const int64_t w = v % (a.layers * kCopyBatches), layer = w / kCopyBatches;
            const int at = int(w % kCopyBatches) * kCopyVecs;
            if (d < 0 || at >= rest * kEntryVecs) continue;
            if (!in_pool(a, s)) {
                if (lane == 0) report_status(a.status, kStatusBadIndex, 6, s);
                continue;
            }
            copy_batch(a.pool + (layer * a.num_pages + d) * kPageVecs, a.pool + (layer * a.num_pages + s) * kPageVecs, at, rest * kEntryVecs, lane);
        }
    }
}

// First half of a compaction, one block: with `count` live pages, the k-th live page from `count` on goes to the k-th free page below it (which
// moves as few pages as possible, and none over another that has yet to move).  new_refs may be refs: all counts have been read before the barrier behind which they change.
__global__ void __launch_bounds__(kPagesPlanThreads) kv_compact_plan_kernel(const __grid_constant__ KvPagesArgs a) {
    __shared__ int s_warp[32];
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int tid = threadIdx.x;
    int mine = 0, live = 0;
    int32_t refs[kPlanPages];
    uint32_t last = 0u;                                // of the chunk looked at last, which is the only one of most pools
    for (int64_t p = int64_t(tid) * kPlanPages; p < a.num_pages; p += kPlanChunk) mine += __popc(last = held_pages(a, p, refs));
    block_prefix(mine, s_warp, live);
    int holes = 0, movers = 0;
    for (int64_t base = 0; base < a.num_pages; base += kPlanChunk) {
        const int64_t p = base + int64_t(tid) * kPlanPages;
        const uint32_t held = a.num_pages <= kPlanChunk ? last : held_pages(a, p, refs), all = pool_pages(a, p);
        const uint32_t low = p + kPlanPages <= live ? ~0u : (p < live ? (1u << (live - p)) - 1u : 0u);      // pages below `live`
        uint32_t hole_bits = ~held & all & low, mover_bits = held & ~low;
        // (both counts of a chunk fit 16 bits)
        int found;
        const int before = block_prefix((__popc(hole_bits) << 16) | __popc(mover_bits), s_warp, found);
        int h = holes + (before >> 16), m = movers + (before & 0xFFFF);
        for (; hole_bits != 0u; hole_bits &= hole_bits - 1u) a.to[h++] = int(p) + __ffs(hole_bits) - 1;
        for (; mover_bits != 0u; mover_bits &= mover_bits - 1u) a.from[m++] = int(p) + __ffs(mover_bits) - 1;
        holes += found >> 16;
        movers += found & 0xFFFF;
    }
    if (a.new_refs != a.refs) {
        constexpr int kDeep = 8;
        for (int64_t p0 = tid; p0 < a.num_pages; p0 += kDeep * kPagesPlanThreads) {
            int v[kDeep];
#pragma unroll
            for (int j = 0; j < kDeep; ++j) v[j] = p0 + j * kPagesPlanThreads < a.num_pages ? ptx::ld(a.refs + p0 + j * kPagesPlanThreads) : 0;
#pragma unroll
            for (int j = 0; j < kDeep; ++j)
                if (p0 + j * kPagesPlanThreads < a.num_pages) a.new_refs[p0 + j * kPagesPlanThreads] = v[j];
        }
    }
    __syncthreads();
    // (as many holes below `live` as live pages above it)
    for (int k = tid; k < movers; k += kPagesPlanThreads) {
        const int s = a.from[k], d = a.to[k];
        a.new_refs[d] = a.new_refs[s];
        a.new_refs[s] = 0;
    }
    if (tid == 0) {
        *a.moves = movers;
        *a.count = live;
    }
}

// Second half: the pages move, and the tables name their new places.
__global__ void __launch_bounds__(kPagesThreads) kv_compact_apply_kernel(const __grid_constant__ KvPagesArgs a) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t slots = int64_t(a.B) * a.max_pages, stride = int64_t(gridDim.x) * kPagesThreads;
    const int64_t moves = ptx::ld(a.moves);
    const int live = ptx::ld(a.count);
    for (int64_t i = int64_t(blockIdx.x) * kPagesThreads + threadIdx.x; i < slots; i += stride) {
        int page = a.block_table[i];
        if (page >= live && moves > 0) {
            int64_t lo = 0, hi = moves - 1;            // among the pages that move
            while (lo < hi) {
                const int64_t mid = (lo + hi) / 2;
                if (ptx::ld(a.from + mid) < page) lo = mid + 1;
                else hi = mid;
            }
            if (ptx::ld(a.from + lo) == page) page = ptx::ld(a.to + lo);
        }
        a.new_table[i] = page;
    }
    const int64_t units = moves * a.layers * kCopyBatches;
    for (int64_t u = int64_t(blockIdx.x) * (kPagesThreads / 32) + (threadIdx.x >> 5); u < units; u += int64_t(gridDim.x) * (kPagesThreads / 32)) {
        const int64_t page = u / kCopyBatches, layer = page / moves, k = page % moves;
        const int s = ptx::ld(a.from + k), d = ptx::ld(a.to + k);
        copy_batch(a.pool + (layer * a.num_pages + d) * kPageVecs, a.pool + (layer * a.num_pages + s) * kPageVecs, int(u % kCopyBatches) * kCopyVecs, kPageVecs, lane);
    }
}

}  // namespace dsv4
