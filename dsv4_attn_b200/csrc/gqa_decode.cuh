// Attention of new tokens over pages of ordinary K and V heads (grouped queries): the cache's length is shared out evenly over resident blocks.
//
// For request b, KV head h and query head h * G + g, a token at place p of its request sees the entries j <= p that exist, with a window those with
// p - j < window or j < first only, and
//     out = sum_j exp(x_j - m) v_j / (sum_j exp(x_j - m) + exp(sink - m)),   x_j = sm_scale q . k_j,   lse = m + log sum_j exp(x_j - m)
//
// Layout of the work.  The rows of a KV head are its (token, query head) pairs, in groups of R = 16, 32 or 64; a unit is (request, KV head, row group), its tiles the
// pages of 64 entries that some row of the group sees.  All units' tiles lie behind one another on one axis, which is cut into equal shares, one per resident block: every
// block streams the same number of tiles whatever the lengths are.  Each block finds its place on the axis by a scan over the
// lengths (no planner, nothing read back).  A unit inside one share writes its output; one that a cut runs through leaves FP32 partials, which gqa_merge_kernel joins.  Of small calls a cluster
// has each unit to itself and joins its blocks' parts through distributed shared memory.
//
// What bounds it: the bytes of K and V, each read once.  A producer warp keeps a ring of K and V tiles filled by TMA (swizzled) across the
// block's units; four warps take 16 entries of a tile each, or 32 of two pages where pages are small (with more rows: fewer entries, more rows), S = Q K^T and O += P V by mma.sync m16n8k16 with
// FP32 accumulators, the running maximum and sum in registers.  A tile of 64 entries x 128 in 16 bits is 128 instructions of 16 rows, 2.2 cycles each: a fifth of the time
// that its 32 KB take from memory, so that tcgen05's M = 128 would multiply padding and its way through tensor memory would only lengthen
// the chain; more rows take gqa_rows_kernel and prompts gqa_prefill_kernel.
// 64 requests x 8,000 entries, 8 heads: of 128 in BF16 314-322 us (6.5 TB/s), in e4m3 232 (4.5: a page of 16 KB takes its warps 1,080 cycles); of 64 193 (5.4); of 256 611 (6.9, the copy
// that 6.4 is measured by writes too).  One request of 1,000 entries 8.3 us, of 16,000 24, of 130,000 92 (5.8 TB/s).
//
// Rounding: P is rounded to the type of V, off by half a step at most (BF16 2^-8, FP16 2^-11 of a weight); everything else is FP32.  Weights in FP16 are taken 2^7 larger, so that with scores that pass
// a row's reference by 2^8 they reach 2^15 of its 2^16, and have all their bits down to 2^-21 of the reference (with a reference at 1 they had them to 2^-14: 3,000 entries of 10.45 * 2^-24 beside one
// that outweighs them came out 4 % low); what is below 2^-32 of it vanishes.  An e4m3 cache is read as
// FP16, which holds its values exactly; BF16 queries then go through FP16 after each row has been brought near 1 by a power of two, which is exact but for elements
// below 2^-14 of the row's largest (off by 2^-25 of that).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gqa_span.h"
#include "ptx.cuh"

namespace dsv4 {

constexpr int kGqaBf16 = 0, kGqaF16 = 1, kGqaE4m3 = 2;            // types of K and V
constexpr int kGqaConsumers = 128, kGqaThreads = kGqaConsumers + 32;
constexpr int kGqaMergeThreads = 256, kGqaWeightThreads = 256;
constexpr float kGqaLazy = 8.f;                                   // log2 of how far scores may pass a row's reference
constexpr float kGqaUp = 7.f;                                     // log2 of how far weights in FP16 are raised
constexpr int kGqaStatusBadIndex = 7, kGqaStatusWait = 1;

struct GqaArgs {
    int B, T, Hkv, G, max_pages, window, first;
    int64_t rows;                    // tokens of all requests (rows of q)
    const int32_t* q_start;          // [B + 1], or null: T tokens each
    const int32_t* kv_len;           // [B]
    const int32_t* block_table;      // [B, max_pages]
    int64_t num_pages;
    const void* q;
    int64_t q_stride_b, q_stride_t, q_stride_h;    // elements (packed tokens: stride_b is not read)
    int q_bf16;                      // type of q and out
    const float* k_scale;            // [Hkv], e4m3
    const float* v_scale;
    const float* sink;               // [H]
    float scale_log2;                // sm_scale * log2(e)
    void* out;                       // [rows, H, D]
    float* lse;                      // [rows, H]
    float* part_o;                   // [2 * blocks][R][D]
    float* part_lse;                 // [2 * blocks][R], log2
    int blocks;                      // of the attention kernel
    int group_rows;                  // R
    int cluster;                     // blocks of a cluster that has a unit to itself, or 0: shares
    int one_group;                   // not packed, and a request's rows of a KV head fit a group
    int min_share;                   // tiles of a block, at least
    int merge_warps;                 // of gqa_merge_kernel for a row: 1, 2, 4 or 8
    int streams;                     // parts that a block leaves of a piece (gqa_rows_kernel; and a place more), or 0: one
    // weights of the entries
    float* logits;                   // [B][Hkv * T * G][logit_stride], log2 units; null: not wanted
    int64_t logit_stride;            // whole tiles
    int logit_end;                   // the same, or 0 without weights: scores of entries behind it are not kept
    int weight_len;                  // entries that can get weights
    float* total;                    // [B][Hkv * T * G]: log2 of the denominators
    float* weights;                  // [B][weight_stride], added to
    int64_t weight_stride;
    uint32_t wait_ns;
    int dbg_drop_tile;
    int32_t* status;
    alignas(64) CUtensorMap k_map, v_map;
};

// ── one request ──
struct GqaRequest {
    int tokens, place0, entries;     // new tokens; place of the first of them (negative where the cache is shorter); entries that can be looked up
    int64_t row0;                    // the first token's row in q
    bool bad;                        // lengths or offsets that point outside
};
__device__ __forceinline__ GqaRequest gqa_request(const GqaArgs& a, int b) {
    GqaRequest r;
    const int n = max(ptx::ld(a.kv_len + b), 0);
    r.bad = false;
    if (a.q_start != nullptr) {
        const int s = ptx::ld(a.q_start + b), e = ptx::ld(a.q_start + b + 1), last = int(a.rows);
        const int lo = min(max(s, 0), last), hi = min(max(e, lo), last);
        r.bad = lo != s || hi != e;
        r.row0 = lo;
        r.tokens = hi - lo;
    } else {
        r.row0 = int64_t(b) * a.T;
        r.tokens = a.T;
    }
    const int64_t room = int64_t(a.max_pages) * kGqaTile;
    r.entries = n < room ? n : int(room);
    r.bad |= n > room;
    r.place0 = n - r.tokens;
    return r;
}

// ── the tiles of a row group ──
// (Rows and tokens of a request are below 2^29: 32-bit divisions, which take a twentieth of the time of 64-bit ones.  With those, and one more for every group, a call for one
// request took 18.2 us instead of 12.8.)
__device__ __forceinline__ GqaSpan gqa_span(const GqaArgs& a, const GqaRequest& r, int rg) {
    if (a.one_group) return gqa_token_span(r.place0, r.entries, 0, r.tokens - 1, a.window, a.first);
    const uint32_t row = uint32_t(rg) * uint32_t(a.group_rows), rows = uint32_t(r.tokens) * uint32_t(a.G);
    return gqa_token_span(r.place0, r.entries, int(row / uint32_t(a.G)), int((min(row + uint32_t(a.group_rows), rows) - 1) / uint32_t(a.G)), a.window, a.first);
}
__device__ __forceinline__ int gqa_groups(const GqaArgs& a, const GqaRequest& r) {
    if (a.one_group) return 1;
    return int((uint32_t(r.tokens) * uint32_t(a.G) + uint32_t(a.group_rows) - 1) / uint32_t(a.group_rows));
}
// Tiles of one KV head of a request.
__device__ __forceinline__ int64_t gqa_head_tiles(const GqaArgs& a, const GqaRequest& r) {
    if (a.one_group) return gqa_span(a, r, 0).count;
    int64_t n = 0;
    for (int rg = 0, groups = gqa_groups(a, r); rg < groups; ++rg) n += gqa_span(a, r, rg).count;
    return n;
}
// a / b, neither negative: in 32 bits where they fit
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return uint32_t(a) / uint32_t(b);
    return a / b;
}

// Sum of one value per thread over the threads before this one, and over all.
template <int THREADS>
__device__ __forceinline__ int64_t block_prefix(int64_t v, int64_t& total, int64_t* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xFFFFFFFFu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    return before + x - v;
}

// The length of a share, which the attention kernel and the merge work out alike.
__device__ __forceinline__ int64_t gqa_share(const GqaArgs& a, int64_t total) { return max(quotient(total + a.blocks - 1, a.blocks), int64_t(a.min_share)); }

__device__ __forceinline__ void gqa_report(int32_t* status, int code, int role, int what) {
    if (status != nullptr && atomicCAS(status, 0, code) == 0) {
        status[1] = int(blockIdx.x);
        status[2] = role;
        status[3] = what;
    }
}

// ── mma.sync ──
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t saddr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t saddr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(saddr) : "memory");
}
// Eight BF16 of a row that LANES lanes hold, brought to FP16 near 1 by a power of two, which is returned inverted: 2^e <= the row's largest < 2^(e + 1); zeros, infinities and what 2^-e cannot
// bring there stay near enough.
template <int LANES>
__device__ __forceinline__ float gqa_near_one(uint4& v) {
    float f[8], top = 0.f;
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
        top = fmaxf(top, fmaxf(fabsf(f[2 * i]), fabsf(f[2 * i + 1])));
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const int e = min(max(int(__float_as_uint(top) >> 23) - 127, -100), 126);
    const float down = __uint_as_float(uint32_t(127 - e) << 23);
    v.x = ptx::pack_f16x2(f[0] * down, f[1] * down);
    v.y = ptx::pack_f16x2(f[2] * down, f[3] * down);
    v.z = ptx::pack_f16x2(f[4] * down, f[5] * down);
    v.w = ptx::pack_f16x2(f[6] * down, f[7] * down);
    return __uint_as_float(uint32_t(127 + e) << 23);
}
// For kernels that set what a row does not see to -inf before they scale its scores, which takes a factor above 0: a head's negative scale stands in its products' signs (the kernels turn Q or K
// round), and a factor of 0 (a scale of 0, or a product too small) is the smallest number, by which scores are 0 as well and -inf remains what it is.
__device__ __forceinline__ float gqa_positive(float scale) {
    const float s = fabsf(scale);
    return s == 0.f ? __uint_as_float(1u) : s;
}
__host__ __device__ constexpr int gqa_blocks_per_sm(int D) { return D > 128 ? 1 : 2; }

// D: head dimension; KVT: type of K and V; WM: warps side by side over the rows, 16 each
template <int D_, int KVT_, int WM_>
struct GqaCfg {
    static constexpr int D = D_, KVT = KVT_, WM = WM_, R = 16 * WM;
    static constexpr int ES = KVT == kGqaE4m3 ? 1 : 2;
    static constexpr int RowBytes = D * ES;
    static constexpr int Box = RowBytes < 128 ? RowBytes : 128;               // bytes of a row in one TMA box, and the width of the swizzle
    static constexpr int Boxes = RowBytes / Box;
    static constexpr int Slot = kGqaTile * RowBytes;
    // Some 130 KB of an SM are on the way: by two blocks with 64 KB each, or one with 128 KB for heads of 256.
    static constexpr int BlocksPerSm = gqa_blocks_per_sm(D);
    static constexpr int Ring = (BlocksPerSm == 1 ? 128 : 64) * 1024;
    static constexpr int Slots = Ring / Slot, Pages = Slots / 2;
    // Where rows are 16, the four warps share a page's entries, 16 each; where the ring holds four pages or more, two warps have every other page, 32 entries each: what a
    // visit costs besides its products (barriers, masks, maxima: 260 instructions of 400) then counts for twice as many.
    static constexpr int PG = WM == 1 && Pages % 4 == 0 ? 2 : 1;              // groups of warps that take turns with the pages
    static constexpr int WN = 4 / (WM * PG);                                  // warps over a page's entries
    static constexpr int Sub = WM == 1 && PG == 1 ? 1 : 2;                    // blocks of 16 entries that a warp takes at a time
    static constexpr int Parts = 4 / WM;                                      // warps that have a part of a row
    static constexpr int QPitch = D * 2 + 16;                                 // bytes
    static constexpr int MergePitch = D + 8;                                  // floats
    static constexpr int Q = R * QPitch, Merge = 4 * 16 * MergePitch * 4;
    static constexpr int Shared = Q > Merge ? Q : Merge;                      // Q is done with when the warps' parts are joined
    static constexpr int OffShared = Ring, OffStats = OffShared + (Shared + 127) / 128 * 128;
    static constexpr int OffBars = OffStats + (2 * 4 * 16 + R) * 4;
    static constexpr int OffValid = OffBars + 2 * Slots * 8, OffScan = OffValid + Slots * 4, Bytes = OffScan + 96 + 1024;
    static_assert((Slots & (Slots - 1)) == 0 && Pages % PG == 0, "a slot's turns belong to one group");
};

// The sequence of pieces (parts of units) of a block, walked by each warp for itself.
struct GqaWalk {
    int b, h, rg, k0, k1;            // tiles [k0, k1) of the unit
    GqaRequest req;
    GqaSpan span;
    int64_t left;                    // tiles of the share from this piece on
    int nth;
    __device__ __forceinline__ void piece() {
        k1 = int(min(int64_t(span.count), k0 + left));
    }
    __device__ __forceinline__ void begin(const GqaArgs& a, int b0, int64_t off, int64_t tiles) {
        b = b0;
        left = tiles;
        nth = 0;
        if (left <= 0) return;
        req = gqa_request(a, b);
        const int64_t per_head = gqa_head_tiles(a, req);
        h = int(quotient(off, per_head));
        off -= h * per_head;
        span = gqa_span(a, req, rg = 0);
        for (const int groups = gqa_groups(a, req); off >= span.count && rg + 1 < groups;) {
            off -= span.count;
            span = gqa_span(a, req, ++rg);
        }
        k0 = int(off);
        piece();
    }
    __device__ __forceinline__ void next(const GqaArgs& a) {
        left -= k1 - k0;
        ++nth;
        if (left <= 0) return;
        if (++rg >= gqa_groups(a, req)) {
            rg = 0;
            if (++h >= a.Hkv) {
                h = 0;
                do { req = gqa_request(a, ++b); } while (req.tokens == 0 && b + 1 < a.B);
            }
        }
        span = gqa_span(a, req, rg);
        k0 = 0;
        piece();
    }
};

__device__ __forceinline__ float4 gqa_cluster_v4(uint32_t caddr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(caddr) : "memory");
    return v;
}
// A sink's part of the denominator, in units of 2^ref, ref >= s: one that 32 bits hold as infinite leaves nothing to the entries.
__device__ __forceinline__ float gqa_sink(float s, float ref) { return s == ref ? 1.f : ptx::ex2(s - ref); }
// Four columns, from x on, of a complete row: v = sum of exp2(x_j - top) v_j, sum = sum of exp2(x_j - top).
template <int D>
__device__ __forceinline__ void gqa_write_row(const GqaArgs& a, int64_t token, int head, int64_t weight_row, int x, const float4& v, float top, float sum, float v_scale) {
    const int H = a.Hkv * a.G;
    const bool none = sum == 0.f;                                             // nothing seen (or nothing but -inf): 0, and an lse of -inf
    float all = sum, by = 1.f, ref = top;
    if (a.sink != nullptr && !none) {
        const float s = ptx::ld(a.sink + head) * 1.4426950408889634f;
        ref = fmaxf(top, s);
        by = ptx::ex2(top - ref);
        all = sum * by + gqa_sink(s, ref);
    }
    const float per = none ? 0.f : by * v_scale / all;
    const float o[4] = {v.x * per, v.y * per, v.z * per, v.w * per};
    uint2 w;
    if (a.q_bf16) w = make_uint2(ptx::pack_bf16x2(o[0], o[1]), ptx::pack_bf16x2(o[2], o[3]));
    else w = make_uint2(ptx::pack_f16x2(o[0], o[1]), ptx::pack_f16x2(o[2], o[3]));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + (token * H + head) * D + x) = w;
    if (x == 0) {
        if (a.lse != nullptr) a.lse[token * H + head] = none ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        if (a.total != nullptr) a.total[weight_row] = none ? INFINITY : ref + log2f(all);
    }
}

template <class C>
__global__ void __launch_bounds__(kGqaThreads, C::BlocksPerSm) gqa_decode_kernel(const __grid_constant__ GqaArgs a) {
    constexpr int D = C::D, WN = C::WN, R = C::R, Sub = C::Sub;
    constexpr bool kE4m3 = C::KVT == kGqaE4m3, kBf16 = C::KVT == kGqaBf16;
    constexpr bool kQInRegs = D <= 128;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const base = smem_raw + (smem - ptx::smem_u32(smem_raw));
    const uint32_t bar_full = smem + C::OffBars, bar_empty = bar_full + 8 * C::Slots;
    volatile uint32_t* const valid = reinterpret_cast<volatile uint32_t*>(base + C::OffValid);
    int64_t* const scan = reinterpret_cast<int64_t*>(base + C::OffScan);                    // 5 warp sums; request and offset of the share
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < C::Slots; ++i) {
            ptx::mbar_init(bar_full + 8 * i, 1);
            ptx::mbar_init(bar_empty + 8 * i, 4 / C::PG);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&a.k_map);
        ptx::prefetch_tensormap(&a.v_map);
    }
    ptx::pdl_wait();
    ptx::pdl_trigger();              // (behind the wait: the kernels that follow read lengths and offsets before theirs)

    GqaWalk w;
    uint32_t rank = 0;
    if (a.cluster > 0) {
        // Small calls: a cluster has a unit to itself, and its blocks' parts are joined through distributed shared memory: no scan over the lengths, and no second kernel.
        const uint32_t unit = blockIdx.x / uint32_t(a.cluster);
        rank = blockIdx.x - unit * uint32_t(a.cluster);
        w.b = int(unit / uint32_t(a.Hkv));
        w.h = int(unit) - w.b * a.Hkv;
        w.rg = w.nth = 0;
        w.req = gqa_request(a, w.b);
        w.span = gqa_span(a, w.req, 0);
        w.k0 = int(uint32_t(w.span.count) * rank / uint32_t(a.cluster));
        w.k1 = int(uint32_t(w.span.count) * (rank + 1) / uint32_t(a.cluster));
        w.left = w.k1 - w.k0;
        if (w.req.bad && tid == 0 && w.h == 0 && rank == 0) gqa_report(a.status, kGqaStatusBadIndex, 4, w.b);
        __syncthreads();                                                      // (the barriers have been initialised)
    } else {
    // where this block's share begins
    const int each = (a.B + kGqaThreads - 1) / kGqaThreads, b_from = tid * each, b_to = min(b_from + each, a.B);
    int64_t mine = 0, total;
    for (int b = b_from; b < b_to; ++b) {
        const GqaRequest r = gqa_request(a, b);
        if (r.bad && blockIdx.x == 0) gqa_report(a.status, kGqaStatusBadIndex, 4, b);
        mine += gqa_head_tiles(a, r) * a.Hkv;
    }
    const int64_t before = block_prefix<kGqaThreads>(mine, total, scan);
    const int64_t share = gqa_share(a, total), begin = int64_t(blockIdx.x) * share;
    const int64_t tiles = min(share, total - begin);
    if (tiles <= 0) return;
    if (begin >= before && begin < before + mine) {
        int64_t off = begin - before;
        for (int b = b_from; b < b_to; ++b) {
            const int64_t w = gqa_head_tiles(a, gqa_request(a, b)) * a.Hkv;
            if (off < w) {
                scan[5] = b;
                scan[6] = off;
                break;
            }
            off -= w;
        }
    }
    __syncthreads();
    w.begin(a, int(scan[5]), scan[6], tiles);
    }

    if (warp == 4) {
        // ── producer ──
        uint32_t seq = 0;
        bool ok = true;
        for (; w.left > 0 && ok; w.next(a)) {
            for (int k = w.k0; k < w.k1 && ok; k += 32) {
                // the pages of the next 32 tiles, one per lane
                int page = -1;
                if (k + lane < w.k1 && w.span.has(w.span.slot(k + lane))) {
                    page = ptx::ld(a.block_table + int64_t(w.b) * a.max_pages + w.span.slot(k + lane));
                    if (page < 0 || page >= a.num_pages) {
                        gqa_report(a.status, kGqaStatusBadIndex, 4, page);
                        page = -1;
                    }
                }
                const int n = min(32, w.k1 - k);
                for (int i = 0; i < n && ok; ++i) {
                    const int pg = __shfl_sync(0xFFFFFFFFu, page, i);
#pragma unroll
                    for (int kv = 0; kv < 2 && ok; ++kv, ++seq) {
                        const uint32_t st = seq % C::Slots, round = seq / C::Slots;
                        if (round > 0 && !ptx::mbar_wait_warp(bar_empty + 8 * st, (round - 1) & 1u, a.wait_ns)) {
                            if (lane == 0) gqa_report(a.status, kGqaStatusWait, 0, int(seq));
                            ok = false;
                            break;
                        }
                        if (a.dbg_drop_tile >= 0 && int(seq) == 2 * a.dbg_drop_tile) continue;       // a test's lost arrival
                        if (ptx::elect_one()) {
                            valid[st] = pg >= 0;
                            ptx::mbar_arrive_expect_tx(bar_full + 8 * st, C::Slot);
                            // (a page that is not there: rows behind the pool, which arrive as zeros)
                            const int row = pg >= 0 ? pg * kGqaTile : int(a.num_pages * kGqaTile);
#pragma unroll
                            for (int x = 0; x < C::Boxes; ++x)
                                ptx::tma_load_3d(smem + st * C::Slot + x * kGqaTile * C::Box, kv ? &a.v_map : &a.k_map, x * C::Box / C::ES, w.h, row, bar_full + 8 * st);
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (!ok) {
            // copies that are on their way land within microseconds
            const uint32_t t0 = ptx::globaltimer_lo();
            while (ptx::globaltimer_lo() - t0 < 1000000u) __nanosleep(1000);
        }
        if (a.cluster > 0) {
            ptx::cluster_sync();                                              // (the parts are there; they have been read)
            ptx::cluster_sync();
        }
        return;
    }

    // ── attention ──
    const int wm = warp % C::WM, wn = warp / C::WM % WN, turn = warp / (C::WM * WN), g = lane >> 2, c = lane & 3;
    const uint32_t q_sm = smem + C::OffShared;
    float* const merge = reinterpret_cast<float*>(base + C::OffShared);
    float* const stat_m = reinterpret_cast<float*>(base + C::OffStats);       // [4][16]
    float* const stat_l = stat_m + 4 * 16;
    float* const row_factor = stat_l + 4 * 16;                                // [R]
    // entry of column n of a block of eight (e4m3 rows of 128 bytes and more: the eight lanes that load together then meet all banks)
    constexpr bool kPermuted = kE4m3 && C::RowBytes >= 128;
    auto entry_of = [](int n) { return kPermuted ? (n >> 1) + 4 * (n & 1) : n; };
    uint32_t tiles_before = 0;
    bool failed = false;
    auto wait_full = [&](uint32_t s) {
        if (!failed && !ptx::mbar_wait_warp(bar_full + 8 * (s % C::Slots), (s / C::Slots) & 1u, a.wait_ns)) {
            if (lane == 0) gqa_report(a.status, kGqaStatusWait, 1, int(s));
            failed = true;                                                    // (the rest of the block's work is gone through without waiting)
        }
    };

    for (; w.left > 0; w.next(a)) {
        const int rows = w.req.tokens * a.G, row_first = w.rg * R;
        ptx::bar_sync(1, kGqaConsumers);
        // Q of the group: rows of zeros behind the last one
        ptx::bar_sync(1, kGqaConsumers);
        {
            const uint8_t* const q0 = static_cast<const uint8_t*>(a.q);
            constexpr int kLanes = D / 8;                                     // 16 bytes each
            const int l = tid % kLanes;
#pragma unroll 4
            for (int r = tid / kLanes; r < R; r += kGqaConsumers / kLanes) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row_first + r < rows) {
                    const int t = int(uint32_t(row_first + r) / uint32_t(a.G)), gg = row_first + r - t * a.G;
                    const int64_t at = (a.q_start != nullptr ? (w.req.row0 + t) * a.q_stride_t : int64_t(w.b) * a.q_stride_b + t * a.q_stride_t) +
                                       int64_t(w.h * a.G + gg) * a.q_stride_h + 8 * l;
                    v = *reinterpret_cast<const uint4*>(q0 + at * 2);
                }
                if (kE4m3) {
                    const float factor = a.q_bf16 ? gqa_near_one<kLanes>(v) : 1.f;
                    if (l == 0) row_factor[r] = factor;
                }
                ptx::sts_v4(q_sm + r * C::QPitch + 16 * l, v);
            }
        }
        ptx::bar_sync(1, kGqaConsumers);

        uint32_t qf[kQInRegs ? D / 16 : 1][4];
        // A fragment of 16 dimensions; e4m3: of the dimensions that the lanes' 16-byte pieces of K hold (64 j + 16 c + 4 s + 0..3)
        auto q_fragment = [&](uint32_t (&r)[4], int ks) {
            const uint32_t row = q_sm + uint32_t(wm * 16) * C::QPitch;
            if (kE4m3) {
                const uint32_t at = row + g * C::QPitch + (ks / 4) * 128 + c * 32 + (ks % 4) * 8;
                const uint2 lo = ptx::lds_v2(at), hi = ptx::lds_v2(at + 8 * C::QPitch);
                r[0] = lo.x;  r[1] = hi.x;  r[2] = lo.y;  r[3] = hi.y;
            } else {
                ldmatrix4(r, row + (lane & 15) * C::QPitch + ks * 32 + (lane >> 4) * 16);
            }
        };
        if (kQInRegs) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) q_fragment(qf[kQInRegs ? ks : 0], ks);
        }
        int place[2];                                                         // of the rows' tokens; -1: no row
        float scale[2];
        const float head_scale = a.scale_log2 * (a.k_scale != nullptr ? ptx::ld(a.k_scale + w.h) : 1.f);
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const int r = wm * 16 + g + 8 * hh;
            place[hh] = row_first + r < rows ? w.req.place0 + int(uint32_t(row_first + r) / uint32_t(a.G)) : -1;
            scale[hh] = kE4m3 ? head_scale * row_factor[r] : head_scale;
        }
        // m: reference of a row's weights, in log2 units: a maximum that the row's later ones have not passed by 2^8, for weights in FP16 less kGqaUp
        constexpr float kUp = kBf16 ? 0.f : kGqaUp, kLazy = kGqaLazy + kUp;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        const int place_first = w.req.place0 + w.span.t0, place_last = w.req.place0 + w.span.t1;

        // this group's pages
        for (int k = w.k0 + (C::PG > 1 ? int((uint32_t(turn) - tiles_before) % C::PG) : 0); k < w.k1; k += C::PG) {
            const uint32_t seq = 2 * (tiles_before + uint32_t(k - w.k0)), ks_ = seq % C::Slots, vs_ = (seq + 1) % C::Slots;
            wait_full(seq);
            const bool there = valid[ks_] != 0;
            const uint32_t k_sm = smem + ks_ * C::Slot, v_sm = smem + vs_ * C::Slot;
            const int e0 = w.span.slot(k) * kGqaTile;
            // a page that all rows see
            const bool page_whole = there && e0 + kGqaTile - 1 <= place_first && e0 + kGqaTile <= w.req.entries && (a.window == 0 || e0 > place_last - a.window || e0 + kGqaTile <= a.first);
            bool v_waited = false, k_given_back = false;
#pragma unroll 1
            for (int sl = wn * Sub; sl < 4; sl += WN * Sub) {
                const int p0 = e0 + 16 * sl;                                  // entries p0 .. p0 + 16 Sub - 1
                constexpr int kEntries = 16 * Sub;
                // seen by all rows, or by none, or by some
                bool whole = page_whole;
                if (!page_whole) {
                    whole = there && p0 + kEntries - 1 <= place_first && p0 + kEntries <= w.req.entries && (a.window == 0 || p0 > place_last - a.window || p0 + kEntries <= a.first);
                    if (!(p0 < w.span.hi && (p0 + kEntries > w.span.lo || p0 < w.span.first))) continue;
                }
                float s[2 * Sub][4];
#pragma unroll
                for (int i = 0; i < 2 * Sub; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
                if constexpr (!kE4m3) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        uint32_t qq[4];
                        if (!kQInRegs) q_fragment(qq, ks);
                        const uint32_t(&qa)[4] = kQInRegs ? qf[kQInRegs ? ks : 0] : qq;
#pragma unroll
                        for (int i = 0; i < Sub; ++i) {
                            const int e = 16 * (sl + i) + (lane & 7) + ((lane >> 4) << 3);
                            uint32_t kf[4];
                            ldmatrix4(kf, k_sm + e * 128 + (ks / 4) * (kGqaTile * 128) + ((((ks % 4) * 2 + ((lane >> 3) & 1)) ^ (e & 7)) << 4));
                            mma16816<kBf16>(s[2 * i], qa, kf[0], kf[1]);
                            mma16816<kBf16>(s[2 * i + 1], qa, kf[2], kf[3]);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        uint4 kb[2 * Sub];
#pragma unroll
                        for (int i = 0; i < 2 * Sub; ++i) {
                            const int e = 16 * sl + 8 * i + entry_of(g);
                            kb[i] = ptx::lds_v4(C::Box == 128 ? k_sm + (j / 2) * (kGqaTile * 128) + e * 128 + ((((j & 1) * 4 + c) ^ (e & 7)) << 4) : k_sm + e * 64 + ((c ^ ((e >> 1) & 3)) << 4));
                        }
#pragma unroll
                        for (int st = 0; st < 4; ++st) {
                            uint32_t qq[4];
                            if (!kQInRegs) q_fragment(qq, 4 * j + st);
                            const uint32_t(&qa)[4] = kQInRegs ? qf[kQInRegs ? 4 * j + st : 0] : qq;
#pragma unroll
                            for (int i = 0; i < 2 * Sub; ++i) {
                                uint32_t k0, k1;
                                ptx::e4m3x4_to_f16x4(st == 0 ? kb[i].x : st == 1 ? kb[i].y : st == 2 ? kb[i].z : kb[i].w, k0, k1);
                                mma16816<false>(s[i], qa, k0, k1);
                            }
                        }
                    }
                }
                // scores in log2 units; what a row does not see is -inf
#pragma unroll
                for (int i = 0; i < 2 * Sub; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s[i][q] *= scale[q >> 1];
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 2 * Sub; ++i)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int p = p0 + 8 * i + entry_of(2 * c + (q & 1)), at = place[q >> 1];
                            if (!(there && p <= at && p < w.req.entries && (a.window == 0 || p > at - a.window || p < a.first))) s[i][q] = -INFINITY;
                        }
                }
                if (p0 < a.logit_end) {
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        const int r = row_first + wm * 16 + g + 8 * hh;
                        if (r < rows) {
                            float* const to = a.logits + ((int64_t(w.b) * a.Hkv + w.h) * rows + r) * a.logit_stride + p0;
#pragma unroll
                            for (int i = 0; i < 2 * Sub; ++i) {
                                if (kPermuted) {
                                    to[8 * i + entry_of(2 * c)] = s[i][2 * hh];
                                    to[8 * i + entry_of(2 * c + 1)] = s[i][2 * hh + 1];
                                } else {
                                    *reinterpret_cast<float2*>(to + 8 * i + 2 * c) = make_float2(s[i][2 * hh], s[i][2 * hh + 1]);
                                }
                            }
                        }
                    }
                }
                // References move where a score has passed them by 2^8 (or at a row's first entry): looked at by each lane, and agreed upon by the four of a row only then.
                float top[2];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    top[hh] = fmaxf(s[0][2 * hh], s[0][2 * hh + 1]);
#pragma unroll
                    for (int i = 1; i < 2 * Sub; ++i) top[hh] = ptx::max3(top[hh], s[i][2 * hh], s[i][2 * hh + 1]);
                }
                if (__any_sync(0xFFFFFFFFu, (m[0] == -INFINITY ? top[0] > m[0] : top[0] - m[0] > kLazy) || (m[1] == -INFINITY ? top[1] > m[1] : top[1] - m[1] > kLazy))) {
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        float t = fmaxf(top[hh], m[hh]);
                        t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 1));
                        t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, 2));
                        // (a row goes by its own scores only)
                        const bool first = m[hh] == -INFINITY, moves = first ? t > m[hh] : t - m[hh] > kLazy;
                        const float to = t - kUp, by = moves && !first ? ptx::ex2(m[hh] - to) : 1.f;
                        if (moves) m[hh] = to;
                        l[hh] *= by;
#pragma unroll
                        for (int j = 0; j < D / 8; ++j) {
                            o[j][2 * hh] *= by;
                            o[j][2 * hh + 1] *= by;
                        }
                    }
                }
                uint32_t pf[Sub][4];
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    const float ref = m[hh] == -INFINITY ? 0.f : m[hh];
                    float sum = 0.f;                                          // (of the visit: one rounding of the row's sum for all of its entries)
#pragma unroll
                    for (int i = 0; i < 2 * Sub; ++i) {
                        const float e_lo = ptx::ex2(s[i][2 * hh] - ref), e_hi = ptx::ex2(s[i][2 * hh + 1] - ref);
                        sum += e_lo + e_hi;
                        pf[i / 2][2 * (i % 2) + hh] = kBf16 ? ptx::pack_bf16x2(e_lo, e_hi) : ptx::pack_f16x2(e_lo, e_hi);
                    }
                    l[hh] += sum;
                }
                if (sl + WN * Sub >= 4) {
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(bar_empty + 8 * ks_);
                    k_given_back = true;
                }
                if (!v_waited) {
                    wait_full(seq + 1);
                    v_waited = true;
                }
#pragma unroll
                for (int i = 0; i < Sub; ++i) {
                    // V of entries that no row of the group sees may be anything: it counts as zero (0 * inf is not 0)
                    uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
                    if (!whole) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            keep[x] = 0;
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const int p = p0 + 16 * i + 8 * x + entry_of(2 * c + q);
                                if (p < w.span.hi && (p >= w.span.lo || p < w.span.first)) keep[x] |= q ? 0xFFFF0000u : 0xFFFFu;
                            }
                        }
                    }
                    const int ve = 16 * (sl + i) + ((lane >> 3) & 1) * 8 + entry_of(lane & 7), vc = lane >> 4;
#pragma unroll
                    for (int j = 0; j < D * C::ES / 32; ++j) {                // 32 bytes of a row: 16 dimensions in 16 bits, 32 in 8
                        uint32_t vf[4];
                        const int ch = 2 * j + vc;
                        ldmatrix4_trans(vf, C::Box == 128 ? v_sm + (ch / 8) * (kGqaTile * 128) + ve * 128 + (((ch & 7) ^ (ve & 7)) << 4)
                                                          : v_sm + ve * 64 + ((ch ^ ((ve >> 1) & 3)) << 4));
                        if constexpr (!kE4m3) {
                            if (!whole) { vf[0] &= keep[0];  vf[1] &= keep[1];  vf[2] &= keep[0];  vf[3] &= keep[1]; }
                            mma16816<kBf16>(o[2 * j], pf[i], vf[0], vf[1]);
                            mma16816<kBf16>(o[2 * j + 1], pf[i], vf[2], vf[3]);
                        } else {
                            // a word: dimensions 2n, 2n + 1 of two entries -> two words of one dimension each; o[4 j' ..]: even and odd ones of 16
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const uint32_t w0 = __byte_perm(vf[2 * q], 0, 0x3120), w1 = __byte_perm(vf[2 * q + 1], 0, 0x3120);
                                uint32_t b[4];
                                ptx::e4m3x4_to_f16x4(w0, b[0], b[2]);
                                ptx::e4m3x4_to_f16x4(w1, b[1], b[3]);
                                if (!whole) { b[0] &= keep[0];  b[1] &= keep[1];  b[2] &= keep[0];  b[3] &= keep[1]; }
                                mma16816<false>(o[4 * j + 2 * q], pf[i], b[0], b[1]);
                                mma16816<false>(o[4 * j + 2 * q + 1], pf[i], b[2], b[3]);
                            }
                        }
                    }
                }
            }
            // (every warp of the group waits for both tiles of every page of its own: its arrivals then belong to the turn that they are counted in)
            if (!v_waited) wait_full(seq + 1);
            __syncwarp();
            if (lane == 0) {
                if (!k_given_back) ptx::mbar_arrive(bar_empty + 8 * ks_);
                ptx::mbar_arrive(bar_empty + 8 * vs_);
            }
        }
        tiles_before += uint32_t(w.k1 - w.k0);

        // ── the warps' parts of a row are joined ──
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            l[hh] += __shfl_xor_sync(0xFFFFFFFFu, l[hh], 1);
            l[hh] += __shfl_xor_sync(0xFFFFFFFFu, l[hh], 2);
            if (c == 0) {
                stat_m[warp * 16 + g + 8 * hh] = m[hh];
                stat_l[warp * 16 + g + 8 * hh] = l[hh];
            }
        }
        const bool complete = w.k0 == 0 && w.k1 == w.span.count;
        const int64_t part = 2 * int64_t(blockIdx.x) + (w.nth > 0);           // only the first and the last piece of a share can be parts
        const float v_scale = a.v_scale != nullptr ? ptx::ld(a.v_scale + w.h) : 1.f;
        ptx::bar_sync(1, kGqaConsumers);
        auto row_max = [&](int of_wm, int r) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < C::Parts; ++n) top = fmaxf(top, stat_m[(n * C::WM + of_wm) * 16 + r]);
            return top;
        };
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            const float top = row_max(wm, g + 8 * hh), by = m[hh] == -INFINITY ? 0.f : ptx::ex2(m[hh] - top);
            float* const to = merge + (warp * 16 + g + 8 * hh) * C::MergePitch;
            if constexpr (!kE4m3) {
#pragma unroll
                for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(to + 8 * j + 2 * c) = make_float2(o[j][2 * hh] * by, o[j][2 * hh + 1] * by);
            } else {
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    *reinterpret_cast<float4*>(to + 16 * j + 4 * c) = make_float4(o[2 * j][2 * hh] * by, o[2 * j + 1][2 * hh] * by, o[2 * j][2 * hh + 1] * by, o[2 * j + 1][2 * hh + 1] * by);
            }
        }
        ptx::bar_sync(1, kGqaConsumers);
        constexpr int kLanes = D / 4;
        const int x = 4 * (tid % kLanes);
        // a cluster's block leaves its joined part in the ring, which is idle: [R][D], then a maximum and a sum a row
        float* const joined = reinterpret_cast<float*>(base);
#pragma unroll 2
        for (int r = tid / kLanes; r < R; r += kGqaConsumers / kLanes) {
            const int of_wm = r >> 4, rl = r & 15, row = row_first + r;
            if (row >= rows) break;
            const int token = int(uint32_t(row) / uint32_t(a.G));
            const float top = row_max(of_wm, rl);
            float sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int n = 0; n < C::Parts; ++n) {
                const int at = (n * C::WM + of_wm) * 16 + rl;
                const float mm = stat_m[at], ll = stat_l[at];
                sum += mm == -INFINITY ? ll : ll * ptx::ex2(mm - top);         // (a NaN row has a maximum of -inf and a NaN sum)
                const float4 u = *reinterpret_cast<const float4*>(merge + at * C::MergePitch + x);
                v.x += u.x;  v.y += u.y;  v.z += u.z;  v.w += u.w;
            }
            if (a.cluster > 0) {
                *reinterpret_cast<float4*>(joined + r * D + x) = v;
                if (x == 0) *reinterpret_cast<float2*>(joined + R * D + 2 * r) = make_float2(top, sum);
                continue;
            }
            if (!complete) {
                const float per = sum == 0.f ? 0.f : 1.f / sum;
                *reinterpret_cast<float4*>(a.part_o + (part * R + r) * D + x) = make_float4(v.x * per, v.y * per, v.z * per, v.w * per);
                if (x == 0) a.part_lse[part * R + r] = top + log2f(sum);
                continue;
            }
            gqa_write_row<D>(a, w.req.row0 + token, w.h * a.G + row - token * a.G, (int64_t(w.b) * a.Hkv + w.h) * rows + row, x, v, top, sum, v_scale);
        }
        if (a.cluster > 0) break;
    }
    if (a.cluster == 0) return;
    // ── the cluster's blocks share out the rows ──
    ptx::cluster_sync();
    const int rows = w.req.tokens * a.G;
    constexpr int kLanes = D / 4;
    const uint32_t part = smem;                                               // the same place in every block
    const float v_scale = a.v_scale != nullptr ? ptx::ld(a.v_scale + w.h) : 1.f;
    for (uint32_t at = rank * kGqaConsumers + tid; at < uint32_t(rows) * kLanes; at += uint32_t(a.cluster) * kGqaConsumers) {
        const int row = int(at) / kLanes, x = 4 * (int(at) % kLanes), token = int(uint32_t(row) / uint32_t(a.G));
        float top = -INFINITY, sum = 0.f, by_of[8], sum_of[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            by_of[i] = -INFINITY;
            sum_of[i] = 0.f;
            // (a block without tiles has left nothing)
            if (i < a.cluster && int(uint32_t(w.span.count) * (i + 1) / uint32_t(a.cluster)) > int(uint32_t(w.span.count) * i / uint32_t(a.cluster))) {
                const uint32_t from = ptx::mapa(part + (R * D + 2 * row) * 4, i);
                by_of[i] = __uint_as_float(ptx::lds_cluster_u32(from));
                sum_of[i] = __uint_as_float(ptx::lds_cluster_u32(from + 4));
            }
            top = fmaxf(top, by_of[i]);
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= a.cluster || sum_of[i] == 0.f) continue;
            const float by = by_of[i] == -INFINITY ? 1.f : ptx::ex2(by_of[i] - top);       // (a NaN row has a maximum of -inf and a NaN sum)
            sum = fmaf(sum_of[i], by, sum);
            const float4 u = gqa_cluster_v4(ptx::mapa(part + (row * D + x) * 4, i));
            v.x = fmaf(u.x, by, v.x);  v.y = fmaf(u.y, by, v.y);  v.z = fmaf(u.z, by, v.z);  v.w = fmaf(u.w, by, v.w);
        }
        gqa_write_row<D>(a, w.req.row0 + token, w.h * a.G + row - token * a.G, (int64_t(w.b) * a.Hkv + w.h) * rows + row, x, v, top, sum, v_scale);
    }
    ptx::cluster_sync();
}

// ── parts of units that a cut ran through ──
// A warp takes a row, or with few rows some of a row's parts, and finds out, from the same scan as above, which blocks had a part of its unit.  Bound by latency: a warp has four parts on
// their way at once (one request of 16,000 entries in 296 parts: the call 27 us instead of 35 with one warp a row), and reads lengths before the attention kernel's end (24).
constexpr int kGqaMergeWarps = kGqaMergeThreads / 32;
template <int D>
__global__ void __launch_bounds__(kGqaMergeThreads) gqa_merge_kernel(const __grid_constant__ GqaArgs a) {
    constexpr int kWarps = kGqaMergeWarps;
    __shared__ int64_t sums[2][kWarps];
    __shared__ int request;
    __shared__ __align__(16) float slices[kWarps][D + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, H = a.Hkv * a.G, row_warps = a.merge_warps, slice = warp & (row_warps - 1);
    const int64_t row0 = int64_t(blockIdx.x) * (kWarps / row_warps), token0 = quotient(row0, H);
    // the request of the block's first row
    int first_b = a.B;
    if (a.q_start == nullptr) {
        first_b = int(quotient(token0, a.T));
    } else {
        if (tid == 0) request = a.B;
        __syncthreads();
        for (int b = tid; b < a.B; b += kGqaMergeThreads) {
            const GqaRequest r = gqa_request(a, b);
            if (token0 < r.row0 + r.tokens && r.tokens > 0) atomicMin(&request, b);     // (or the first behind it, where the row is no request's)
        }
        __syncthreads();
        first_b = request;
    }
    // tiles of all requests, and of those before it
    int64_t total = 0, ahead = 0;
    for (int b = tid; b < a.B; b += kGqaMergeThreads) {
        const int64_t n = gqa_head_tiles(a, gqa_request(a, b)) * a.Hkv;
        total += n;
        if (b < first_b) ahead += n;
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        total += __shfl_xor_sync(0xFFFFFFFFu, total, d);
        ahead += __shfl_xor_sync(0xFFFFFFFFu, ahead, d);
    }
    if (lane == 0) {
        sums[0][warp] = total;
        sums[1][warp] = ahead;
    }
    __syncthreads();
    total = ahead = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        total += sums[0][i];
        ahead += sums[1][i];
    }
    // this warp's row
    const int64_t row = row0 + warp / row_warps, token = token0 + int(uint32_t(row - token0 * H) / uint32_t(H));
    GqaRequest req{};
    int b = first_b;
    for (; b < a.B; ++b) {
        req = gqa_request(a, b);
        if (token < req.row0 + req.tokens && req.tokens > 0) break;
        ahead += gqa_head_tiles(a, req) * a.Hkv;
    }
    bool mine = b < a.B && token >= req.row0;
    int head = 0, h = 0, at = 0, r = 0, c0 = 0, parts = 0, later = 0;
    const int streams = max(a.streams, 1), places = 2 * streams + (a.streams > 0);
    if (mine) {
        head = int(row - token * H);
        h = int(uint32_t(head) / uint32_t(a.G));
        at = int(token - req.row0) * a.G + head - h * a.G;                     // row of the KV head
        const int rg = a.one_group ? 0 : int(uint32_t(at) / uint32_t(a.group_rows));
        r = at - rg * a.group_rows;
        int64_t unit = ahead + h * gqa_head_tiles(a, req);
        for (int i = 0; i < rg; ++i) unit += gqa_span(a, req, i).count;
        const int64_t share = gqa_share(a, total);
        c0 = int(quotient(unit, share));
        const int c1 = int(quotient(unit + gqa_span(a, req, rg).count - 1, share));
        later = unit != c0 * share;                                            // (every later block begins with its part)
        parts = (c1 - c0 + 1) * streams;
        mine = c0 != c1;
    }
    constexpr int kVecs = D > 128 ? D / 128 : 1, kAtOnce = 4;
    float4 v[kVecs];
#pragma unroll
    for (int x = 0; x < kVecs; ++x) v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, sum = 0.f;
    const bool in_row = 4 * lane < D;
    // (until here only what was there before the attention kernel's own wait had ended)
    ptx::pdl_wait();
    ptx::pdl_trigger();
    if (mine) {
        auto part = [&](int i) {
            const int block = streams == 2 ? i >> 1 : i;
            return (int64_t(c0 + block) * places + (block == 0 ? later * streams : 0) + (i - block * streams)) * a.group_rows + r;
        };
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, a.part_lse[part(i)]);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        const int each = (parts + row_warps - 1) / row_warps, end = min(parts, (slice + 1) * each);
        for (int i0 = slice * each; i0 < end; i0 += 32) {
            float weight = 0.f;
            if (i0 + lane < end) {
                const float p = a.part_lse[part(i0 + lane)];
                weight = p == -INFINITY ? 0.f : ptx::ex2(p - (top == -INFINITY ? 0.f : top));
            }
            for (int i = 0; i < min(32, end - i0); i += kAtOnce) {
                float4 u[kAtOnce][kVecs];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const float4* const from = reinterpret_cast<const float4*>(a.part_o + part(i0 + i + k) * D + 4 * lane);
#pragma unroll
                    for (int x = 0; x < kVecs; ++x) u[k][x] = in_row && i0 + i + k < end ? from[32 * x] : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const float by = __shfl_sync(0xFFFFFFFFu, weight, i + k);
                    sum += by;
#pragma unroll
                    for (int x = 0; x < kVecs; ++x) {
                        v[x].x = fmaf(by, u[k][x].x, v[x].x);  v[x].y = fmaf(by, u[k][x].y, v[x].y);
                        v[x].z = fmaf(by, u[k][x].z, v[x].z);  v[x].w = fmaf(by, u[k][x].w, v[x].w);
                    }
                }
            }
        }
    }
    if (row_warps > 1) {
        // the row's first warp adds up
        if (slice > 0) {
            if (in_row)
#pragma unroll
                for (int x = 0; x < kVecs; ++x) *reinterpret_cast<float4*>(&slices[warp][128 * x + 4 * lane]) = v[x];
            if (lane == 0) slices[warp][D] = sum;
        }
        __syncthreads();
        if (slice > 0) return;
        for (int i = 1; i < row_warps; ++i) {
            sum += slices[warp + i][D];
            if (in_row)
#pragma unroll
                for (int x = 0; x < kVecs; ++x) {
                    const float4 u = *reinterpret_cast<const float4*>(&slices[warp + i][128 * x + 4 * lane]);
                    v[x].x += u.x;  v[x].y += u.y;  v[x].z += u.z;  v[x].w += u.w;
                }
        }
    }
    if (!mine || !in_row) return;
    const float v_scale = a.v_scale != nullptr ? ptx::ld(a.v_scale + h) : 1.f;
#pragma unroll
    for (int x = 0; x < kVecs; ++x) gqa_write_row<D>(a, token, head, (int64_t(b) * a.Hkv + h) * (int64_t(req.tokens) * a.G) + at, 128 * x + 4 * lane, v[x], top, sum, v_scale);
}

// ── weights of the entries ──
// weights[b][j] += sum over the tokens that see j and over the heads of exp(x_j) / denominator, from the scores that the attention kernel has left.  A thread takes an
// entry and adds in a fixed order.  Bound by the scores, read once (32 requests of up to 8,192 entries, 32 heads: 33 MB).
__global__ void __launch_bounds__(kGqaWeightThreads) gqa_weights_kernel(const __grid_constant__ GqaArgs a) {
    ptx::pdl_trigger();
    const int b = blockIdx.y, p = blockIdx.x * kGqaWeightThreads + threadIdx.x;
    const GqaRequest req = gqa_request(a, b);
    ptx::pdl_wait();                 // (lengths were there before the kernels before this one triggered it)
    if (p >= min(req.entries, a.weight_len)) return;
    const int rows = req.tokens * a.G;
    const int64_t base = int64_t(b) * a.Hkv * rows;
    float sum = 0.f;
    bool any = false;
    for (int t = 0; t < req.tokens; ++t) {
        const int at = req.place0 + t;
        if (!(p <= at && (a.window == 0 || p > at - a.window || p < a.first))) continue;
        any = true;
        for (int h = 0; h < a.Hkv; ++h)
#pragma unroll 4
            for (int g = 0; g < a.G; ++g) {
                const int64_t r = base + int64_t(h) * rows + t * a.G + g;
                sum += ptx::ex2(a.logits[r * a.logit_stride + p] - a.total[r]);
            }
    }
    if (any) a.weights[int64_t(b) * a.weight_stride + p] += sum;
}

// ── new rows into the pages ──
struct GqaInsertArgs {
    int B, T, Hkv, D, max_pages;
    int block_tokens;                // of a block, at most kGqaInsertTokens
    int64_t rows;                    // tokens of all requests
    const int32_t* q_start;          // [B + 1], or null: T tokens each
    const int32_t* n_rows;           // [B], or null: all T
    const int32_t* insert_pos;       // [B]
    const int32_t* block_table;      // [B, max_pages]
    int64_t num_pages;
    const void* src[2];              // K, V: 16-bit
    int64_t stride_b[2], stride_t[2], stride_h[2];
    int src_bf16;
    const float* scale[2];           // [Hkv], e4m3
    void* pool[2];                   // [num_pages, 64, Hkv, D]
    int32_t* status;
};
constexpr int kGqaInsertThreads = 256;

__device__ __forceinline__ uint32_t quant_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
    return r;
}

// x / s from the correctly rounded 1 / s: Markstein's step, which gives the correctly rounded quotient.  Quotients beyond e4m3's range are left as they are (the step would make NaN of
// infinite ones).
__device__ __forceinline__ float by_scale(float x, float s, float inverse) {
    const float q = x * inverse, r = fmaf(fmaf(q, s, -x), -inverse, q);        // (with these signs a zero keeps its own)
    return fabsf(q) < 1024.f ? r : q;
}

// The quotient over any scale; over 0 zeros stay zeros (as which a head of zeros is read back, whose largest value, 0, made the scale).
__device__ __forceinline__ float over_scale(float x, float s) { return s == 0.f && x == 0.f ? x : __fdiv_rn(x, s); }

// A block takes some consecutive tokens: a thread each finds out where they go (offset, position, page: one chain of loads for the block), then all threads copy, 16 bytes a thread
// and load, four on the way.  Bound by that chain when small (64 tokens 3.3 us) and by memory when large (six prompts to 4,096 into e4m3 pages: 24-26 us, 4 TB/s).
constexpr int kGqaInsertTokens = 32;
template <bool E4M3>
__global__ void __launch_bounds__(kGqaInsertThreads, 4) gqa_insert_kernel(const __grid_constant__ GqaInsertArgs a) {
    __shared__ int64_t src_row[kGqaInsertTokens], src_row_v[kGqaInsertTokens];      // first element of the token's row of K and of V
    __shared__ int32_t entry[kGqaInsertTokens];                               // where it goes, -1: nowhere
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int tid = threadIdx.x, n = a.block_tokens;
    const int64_t first = int64_t(blockIdx.x) * n;
    if (tid < n) {
        const int64_t token = first + tid;
        int b = -1, t = 0, to = -1;
        if (token < a.rows) {
            if (a.q_start == nullptr) {
                b = int(quotient(token, a.T));
                t = int(token - int64_t(b) * a.T);
                if (a.n_rows != nullptr && t >= ptx::ld(a.n_rows + b)) b = -1;
            } else {
                // the last request whose rows begin at or before the token
                int lo = 0, hi = a.B;                                         // q_start[lo] <= token or lo = 0; q_start[hi] > token or hi = B
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (ptx::ld(a.q_start + mid) <= token) lo = mid;
                    else hi = mid;
                }
                const int from = ptx::ld(a.q_start + lo), end = ptx::ld(a.q_start + lo + 1);
                if (token >= from && token < end) {
                    b = lo;
                    t = int(token - from);
                }
            }
        }
        if (b >= 0) {
            const int64_t pos = int64_t(ptx::ld(a.insert_pos + b)) + t, slot = pos >> 6;
            int page = -1;
            if (pos >= 0 && slot < a.max_pages) page = ptx::ld(a.block_table + int64_t(b) * a.max_pages + slot);
            if (page >= 0 && page < a.num_pages) to = page * kGqaTile + int(pos & (kGqaTile - 1));
            else gqa_report(a.status, 16, b, int(pos));
            src_row[tid] = a.q_start == nullptr ? b * a.stride_b[0] + t * a.stride_t[0] : token * a.stride_t[0];
            src_row_v[tid] = a.q_start == nullptr ? b * a.stride_b[1] + t * a.stride_t[1] : token * a.stride_t[1];
        }
        entry[tid] = to;
    }
    __syncthreads();
    // A warp takes whole tokens, a lane four pieces of 16 bytes of K and of V at a time: where they lie in a row, and their heads' scales, are worked out once.
    const int lane = tid & 31, per_head = a.D / 8, pieces = a.Hkv * per_head;
    for (int x0 = lane; x0 < pieces; x0 += 128) {
        int32_t off[2][4];                                                    // (of a row: below 2^31)
        float scale[2][4];
        bool plain = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = min(x0 + 32 * i, pieces - 1), h = x / per_head;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                off[kv][i] = int32_t(h * a.stride_h[kv]) + 8 * (x - h * per_head);
                if (E4M3) {
                    scale[kv][i] = ptx::ld(a.scale[kv] + h);
                    plain &= scale[kv][i] > 1e-25f && scale[kv][i] < 1e25f;
                }
            }
        }
        for (int t = tid >> 5; t < n; t += kGqaInsertThreads / 32) {
            const int e = entry[t];
            if (e < 0) continue;
            uint4 v[2][4];
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const uint8_t* const src = static_cast<const uint8_t*>(a.src[kv]) + (kv ? src_row_v[t] : src_row[t]) * 2;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (x0 + 32 * i < pieces) v[kv][i] = ptx::ldg_stream_v4(src + int64_t(off[kv][i]) * 2);
            }
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                uint8_t* const dst = static_cast<uint8_t*>(a.pool[kv]) + (int64_t(e) * pieces + x0) * (E4M3 ? 8 : 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (x0 + 32 * i >= pieces) continue;
                    if constexpr (E4M3) {
                        const uint32_t u[4] = {v[kv][i].x, v[kv][i].y, v[kv][i].z, v[kv][i].w};
                        uint32_t o[4];
                        const float inverse = __frcp_rn(scale[kv][i]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float lo, hi;
                            if (a.src_bf16) {
                                lo = __uint_as_float(u[j] << 16);
                                hi = __uint_as_float(u[j] & 0xFFFF0000u);
                            } else {
                                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
                                lo = f.x;
                                hi = f.y;
                            }
                            o[j] = plain ? quant_pair(by_scale(lo, scale[kv][i], inverse), by_scale(hi, scale[kv][i], inverse))
                                         : quant_pair(over_scale(lo, scale[kv][i]), over_scale(hi, scale[kv][i]));
                        }
                        *reinterpret_cast<uint2*>(dst + 256 * i) = make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
                    } else {
                        *reinterpret_cast<uint4*>(dst + 512 * i) = v[kv][i];
                    }
                }
            }
        }
    }
}

}  // namespace dsv4
