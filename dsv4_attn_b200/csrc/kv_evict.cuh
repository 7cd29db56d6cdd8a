// Eviction: a request that holds more entries than it may keeps its first and its most recent ones and, of the others, those that got the most attention; they close
// up in their order, in every layer, and the pages behind them are given back.
//
//   evict_plan_kernel   a block per request: the threshold of the weights by a radix select (11, 11 and 10 bits of an order-preserving 32-bit key; equal weights: the
//                       lower place), then the list of what stays, in ascending order, with its weights, table row and length.
//   evict_move_kernel   moves the entries.  New place j takes old place s(j) >= j, ascending in j: a block has a column of an entry's bytes of one
//                       request, layer and pool and goes through the places in ascending steps; what a step writes lies at or before what it has read, and before
//                       everything that later steps read, so that one barrier between a step's loads and its stores is all it takes.
//
// Bound by the bytes that move, each read and written once; the order of entries is worth that to a cache whose masks go by places.  Columns are as wide as
// leaves four blocks for every SM, 32 bytes (a sector) at least; 16 where that leaves not even one block for each (a sector is then fetched by two blocks, and a request's places take one step of
// loads instead of two).  24 requests of 4,608 entries to 4,096, eight layers: 680-840 us, 4.8-5.9 TB/s; one of 2,176 to 2,048, two layers: 15 us, the
// plan's chain 8 of them.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace dsv4 {

constexpr int kEvictPools = 4;
constexpr int kEvictPlanThreads = 1024, kEvictMoveThreads = 256;
constexpr int kEvictBins = 2048;
constexpr int kEvictEach = 4;                                     // places of a thread in a step of the list
constexpr int kEvictLoads = 8;                                    // 16-byte loads in flight per thread
constexpr int kEvictStatusBadIndex = 7, kEvictStatusShared = 12;

struct KvEvictArgs {
    int B, max_pages, pools;
    int64_t num_pages, layers;
    int keep, first, recent;
    const int32_t* keep_each;         // [B], or null: `keep` for all
    const int32_t* block_table;       // [B, max_pages]
    const int32_t* kv_len;            // [B]
    const int32_t* refs;              // [num_pages]
    const float* weights;             // [B, weight_stride]
    int64_t weight_stride;
    int32_t* new_table;               // each of these may be the old one
    int32_t* new_len;
    int32_t* new_refs;
    float* new_weights;               // [B, weight_stride]
    int32_t* kept;                    // [B, max_pages * 64]
    int32_t* from;                    // scratch [B, max_pages * 64]: pool entries that move to the places from moves[b][0] on
    int32_t* moves;                   // scratch [B][4]: first place that changes, places (0: none do); first slot given back, slots
    uint4* pool[kEvictPools];
    int vecs[kEvictPools];            // 16-byte vectors of an entry
    int width[kEvictPools];           // of a column
    int columns[kEvictPools];
    int all_columns;                  // layers * the sum of columns
    int32_t* status;
};

// Larger weights have larger keys; NaN the lowest, -0 is 0.
__device__ __forceinline__ uint32_t evict_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sum over the threads before this one of a value per thread, and over all threads.
__device__ __forceinline__ uint32_t evict_prefix(uint32_t v, uint32_t& total, uint32_t* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();                                              // (the sums of the call before have been read)
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    uint32_t s = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, s, d);
        if (lane >= d) s += y;
    }
    total = __shfl_sync(0xFFFFFFFFu, s, 31);
    const uint32_t before = __shfl_sync(0xFFFFFFFFu, s, warp > 0 ? warp - 1 : 0);
    return (warp > 0 ? before : 0u) + x - v;
}

__device__ __noinline__ void evict_report(int32_t* status, int code, int b, int what) {
    if (status != nullptr && atomicCAS(status, 0, code) == 0) {
        status[1] = int(blockIdx.x);
        status[2] = b;
        status[3] = what;
    }
}

__global__ void __launch_bounds__(kEvictPlanThreads) evict_plan_kernel(const __grid_constant__ KvEvictArgs a) {
    __shared__ uint32_t bins[kEvictBins];
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t found[2];
    __shared__ int first_change, bad;
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int b = blockIdx.x, tid = threadIdx.x;
    const int64_t cap = int64_t(a.max_pages) * 64;
    // counts of the pages, before any is given back (by the kernel that moves)
    if (a.new_refs != a.refs)
        for (int64_t p = int64_t(b) * kEvictPlanThreads + tid; p < a.num_pages; p += int64_t(gridDim.x) * kEvictPlanThreads) a.new_refs[p] = ptx::ld(a.refs + p);

    const int given = max(ptx::ld(a.kv_len + b), 0), n = given < cap ? given : int(cap);
    const int keep = max(a.keep_each != nullptr ? ptx::ld(a.keep_each + b) : a.keep, 0);
    const int32_t* const table = a.block_table + int64_t(b) * a.max_pages;
    int32_t* const new_table = a.new_table + int64_t(b) * a.max_pages;
    const float* const weights = a.weights + int64_t(b) * a.weight_stride;
    float* const new_weights = a.new_weights + int64_t(b) * a.weight_stride;
    int32_t* const kept = a.kept + int64_t(b) * cap;
    int32_t* const from = a.from + int64_t(b) * cap;
    if (tid == 0) {
        first_change = keep;
        bad = 0;
        if (given > cap) evict_report(a.status, kEvictStatusBadIndex, b, given);
    }
    bool evict = n > keep && given <= cap;
    uint32_t threshold = 0, ties = 0;                             // of the others: keys above it stay, and the first `ties` that equal it
    const int lo = min(a.first, keep), hi = n - min(a.recent, keep - lo);
    if (evict) {
        uint32_t want = uint32_t(keep - lo - (n - hi)), prefix = 0;
        if (want == 0) {
            threshold = 0xFFFFFFFFu;                              // (no key is that large)
        } else {
            // (a request of up to 4096 others: their keys stay in registers)
            uint32_t keys[kEvictEach];
            const bool few = hi - lo <= kEvictPlanThreads * kEvictEach;
            if (few) {
#pragma unroll
                for (int i = 0; i < kEvictEach; ++i) {
                    const int j = lo + i * kEvictPlanThreads + tid;
                    keys[i] = j < hi ? evict_key(ptx::ld(weights + j)) : 0u;
                }
            }
            int shift = 32;
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const int bits = pass < 2 ? 11 : 10;
                const int above = shift;
                shift -= bits;
                for (int i = tid; i < kEvictBins; i += kEvictPlanThreads) bins[i] = 0;
                __syncthreads();
                if (few) {
#pragma unroll
                    for (int i = 0; i < kEvictEach; ++i)
                        if (lo + i * kEvictPlanThreads + tid < hi && (pass == 0 || (keys[i] >> above) == prefix)) atomicAdd(&bins[(keys[i] >> shift) & ((1u << bits) - 1u)], 1u);
                } else
#pragma unroll 4
                for (int j = lo + tid; j < hi; j += kEvictPlanThreads) {
                    const uint32_t key = evict_key(ptx::ld(weights + j));
                    if (pass == 0 || (key >> above) == prefix) atomicAdd(&bins[(key >> shift) & ((1u << bits) - 1u)], 1u);
                }
                __syncthreads();
                // from the largest bin down: the one in which the count reaches `want`
                const int at = kEvictBins - 1 - 2 * tid;
                const uint32_t c0 = bins[at], c1 = bins[at - 1];
                uint32_t all;
                const uint32_t before = evict_prefix(c0 + c1, all, warp_sums);
                if (before < want && before + c0 + c1 >= want) {
                    const bool second = before + c0 < want;
                    found[0] = uint32_t(second ? at - 1 : at);
                    found[1] = want - before - (second ? c0 : 0u);
                }
                __syncthreads();
                prefix = (prefix << bits) | found[0];
                want = found[1];
            }
            threshold = prefix;
            ties = want;
        }
    }
    __syncthreads();
    // The list, in steps of 4096 places: what stays and what equals the threshold are counted together, 16 bits each.
    uint32_t stayed = 0, tied = 0;
    for (int j0 = 0; j0 < n; j0 += kEvictPlanThreads * kEvictEach) {
        uint32_t sure = 0, equal = 0;                             // bits of the thread's places
        const int j = j0 + tid * kEvictEach;
#pragma unroll
        for (int i = 0; i < kEvictEach; ++i) {
            if (j + i < n) {
                const uint32_t key = evict_key(ptx::ld(weights + j + i));
                if (!evict || j + i < lo || j + i >= hi || key > threshold) sure |= 1u << i;
                else if (key == threshold) equal |= 1u << i;
            }
        }
        uint32_t total;
        const uint32_t before = evict_prefix(uint32_t(__popc(sure)) | uint32_t(__popc(equal)) << 16, total, warp_sums);
        uint32_t sures = before & 0xFFFFu, equals = before >> 16;
        // places of the thread's own: `stayed` has what earlier steps kept; of the equal ones before it here, those that stay
#pragma unroll
        for (int i = 0; i < kEvictEach; ++i) {
            const bool is_equal = (equal >> i) & 1u;
            const uint32_t rank = tied + equals;
            if (((sure >> i) & 1u) || (is_equal && rank < ties)) {
                const uint32_t equal_before = min(rank, ties) - min(tied, ties);
                const uint32_t to = stayed + sures + equal_before;
                kept[to] = j + i;
                if (int(to) != j + i) atomicMin(&first_change, int(to));
            }
            sures += (sure >> i) & 1u;
            equals += is_equal;
        }
        stayed += (total & 0xFFFFu) + min(tied + (total >> 16), ties) - min(tied, ties);
        tied += total >> 16;
    }
    __syncthreads();
    const int change = evict ? first_change : n, length = int(stayed), slots = (n + 63) / 64;
    // Pages that are written must be the request's own, and those that are read must be there.
    if (evict) {
        for (int s = change / 64 + tid; s < slots; s += kEvictPlanThreads) {
            const int page = ptx::ld(table + s);
            if (page < 0 || page >= a.num_pages) {
                atomicMax(&bad, 2);
                evict_report(a.status, kEvictStatusBadIndex, b, page);
            } else if (change < length && s <= (length - 1) / 64 && ptx::ld(a.refs + page) > 1) {
                atomicMax(&bad, 1);
                evict_report(a.status, kEvictStatusShared, b, page);
            }
        }
    }
    __syncthreads();
    const bool done = evict && bad == 0;
    if (evict && !done) {                                         // the request stays as it is
        for (int j = tid; j < n; j += kEvictPlanThreads) kept[j] = j;
    }
    const int new_len = done ? length : n, changed = done ? change : n, held = (new_len + 63) / 64;
    __syncthreads();
    // weights and sources, in steps: a step's reads lie at or behind its writes
    for (int64_t j0 = 0; j0 < a.weight_stride; j0 += kEvictPlanThreads * kEvictEach) {
        int old[kEvictEach], page[kEvictEach];
        float w[kEvictEach];
#pragma unroll
        for (int i = 0; i < kEvictEach; ++i) {
            const int64_t j = j0 + i * kEvictPlanThreads + tid;
            old[i] = j < new_len ? kept[j] : -1;
        }
#pragma unroll
        for (int i = 0; i < kEvictEach; ++i) {
            const int64_t j = j0 + i * kEvictPlanThreads + tid;
            w[i] = old[i] >= 0 ? ptx::ld(weights + old[i]) : 0.f;
            page[i] = old[i] >= 0 && j >= changed ? ptx::ld(table + (old[i] >> 6)) : 0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEvictEach; ++i) {
            const int64_t j = j0 + i * kEvictPlanThreads + tid;
            if (j < a.weight_stride) new_weights[j] = w[i];
            if (old[i] >= 0) {
                if (j >= changed) from[j] = page[i] * 64 + (old[i] & 63);
            } else if (j < cap) {
                kept[j] = -1;
            }
        }
    }
    // pages given back: their numbers are kept for the kernel that moves, behind the sources
    for (int s0 = 0; s0 < a.max_pages; s0 += kEvictPlanThreads) {
        const int s = s0 + tid;
        if (s >= a.max_pages) break;
        const int page = ptx::ld(table + s);
        const bool goes = s >= held && s < slots && done;
        if (goes) from[int64_t(s) * 64] = page;
        new_table[s] = goes ? -1 : page;
    }
    if (tid == 0) {
        a.new_len[b] = done ? new_len : given;
        *reinterpret_cast<int4*>(a.moves + 4 * b) = make_int4(changed, new_len - changed, held, done ? slots - held : 0);
    }
}

__global__ void __launch_bounds__(kEvictMoveThreads) evict_move_kernel(const __grid_constant__ KvEvictArgs a) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int b = blockIdx.y, tid = threadIdx.x;
    const int64_t cap = int64_t(a.max_pages) * 64;
    const int4 moves = ptx::ld(reinterpret_cast<const int4*>(a.moves + 4 * b));
    const int32_t* const from = a.from + int64_t(b) * cap;
    const int32_t* const table = a.new_table + int64_t(b) * a.max_pages;
    if (blockIdx.x == 0)
        for (int i = tid; i < moves.w; i += kEvictMoveThreads) {
            const int page = ptx::ld(from + int64_t(moves.z + i) * 64);
            if (page >= 0 && page < a.num_pages) atomicSub(&a.new_refs[page], 1);
        }
    if (moves.y == 0) return;
    for (int column = blockIdx.x; column < a.all_columns; column += gridDim.x) {
        // which layer, pool and bytes
        int c = column, pool = 0;
        for (; pool + 1 < a.pools && int64_t(c) >= a.layers * a.columns[pool]; ++pool) c -= int(a.layers) * a.columns[pool];
        const int layer = c / a.columns[pool], x0 = (c - layer * a.columns[pool]) * a.width[pool], width = min(a.width[pool], a.vecs[pool] - x0), vecs = a.vecs[pool];
        uint4* const base = a.pool[pool] + int64_t(layer) * a.num_pages * 64 * vecs + x0;
        const int lanes = a.width[pool], per = kEvictMoveThreads / lanes, r = tid / lanes, x = tid - r * lanes, step = per * kEvictLoads;
        for (int i0 = 0; i0 < moves.y; i0 += step) {
            uint4 v[kEvictLoads];
            int to[kEvictLoads];
#pragma unroll
            for (int u = 0; u < kEvictLoads; ++u) {
                const int i = i0 + u * per + r;
                to[u] = -1;
                if (r < per && x < width && i < moves.y) {
                    const int j = moves.x + i;
                    to[u] = ptx::ld(table + (j >> 6)) * 64 + (j & 63);
                    v[u] = ptx::ldg_stream_v4(base + int64_t(ptx::ld(from + j)) * vecs + x);
                }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < kEvictLoads; ++u)
                if (to[u] >= 0) base[int64_t(to[u]) * vecs + x] = v[u];
        }
    }
}

}  // namespace dsv4
