// Attention of prompts over pages of K and V heads, on the tensor cores.
//
// A unit is (request, block of tokens, KV head): 128 rows a tile, row = (token, query head of the group), floor(128 / G) tokens each; two tiles a block (heads of 256: one).
// It goes through the pages that some row sees, 64 entries a step:
//     S = Q K^T               tcgen05.mma, M = 128, both operands in shared memory, S in tensor memory (two buffers a tile)
//     P = exp2(c (S - ref))   in the softmax warps, a thread a row; back to tensor memory over S, in the queries' 16-bit type (FP16: times 2^7)
//     O += P V                A = P from tensor memory, V as it lies in the cache (MN-major)
// The scores of a step are computed while the softmax warps have those of the step before, and the two tiles take turns.  The reference of a row moves only when its maximum has
// passed it by 2^8; then O is rescaled in tensor memory by the row's thread.  Units are listed by gqa_plan_kernel, those with most steps first, and dealt out to resident
// blocks, one an SM; the next unit's Q comes in, and its first scores are computed, while the last one's output is written.
//
// What bounds it, per step of two tiles with D = 128, in cycles of an SM: the tensor pipe 1280 (scores 48 an instruction, bound by their operands' way out of shared memory, outputs 64),
// the 16,384 exponentials 1024.  A step takes 1800, of which a softmax warp spends 1100 in exponentials, two warps a scheduler; and from some 20 ms on the power limit holds the clock:
// 4,096 tokens behind 12,288 in 0.91 ms for the first calls after a pause, 0.99-1.02 under load, 0.94-0.97 PFLOP/s (the library's products: 1.42).  Measured and taken back: steps of 128 entries with
// one score buffer a tile, where scores, softmax and outputs of a tile follow one another (1.06 ms; a window of 1,024: 320 us against 275); one warp for all products (1.12: a look at a
// barrier takes 130 to 210 cycles while products keep the shared memory busy); a quarter to a half of the exponentials as polynomials on the multiply-add pipe (0.995 to 1.03).
//
// K and V come by TMA in boxes of a page, 128-byte swizzle.  V of entries that no row sees must count as zero whatever the memory holds: pages at the ends of what is seen
// are fetched in boxes of eight rows and of one, zeros (rows behind the pool) in the place of those.
#pragma once

#include "gqa_decode.cuh"

namespace dsv4 {

constexpr int kPrefillPlanThreads = 1024, kPrefillBuckets = 1024;
constexpr float kPrefillLazy = 8.f;               // log2 of how far a row's maximum may pass its reference

struct GqaPrefillArgs {
    GqaArgs g;                       // group_rows: rows of a unit (tokens of a block x G); k_map, v_map: boxes of a page
    alignas(64) CUtensorMap q_map;   // (element, head, row of q): boxes of 64 elements x G heads x the tokens of a tile
    CUtensorMap v8_map, v1_map;      // boxes of eight entries and of one
    int32_t* plan;                   // [0] units of one KV head; from [4] on (request, block) pairs
    int plan_units;                  // room for them
    int tile_tokens;                 // floor(128 / G)
    int own_pages;                   // if not 0, the pools are the call's copies: slot s of request b is page b * own_pages + s, the first head h0
    int h0, heads;                   // KV heads of this launch
    int b0;                          // its first request, for reports
    int64_t pool_rows;               // entries of the pools: the first row behind them
};

template <int D_, bool BF16_>
struct PrefillCfg {
    static constexpr int D = D_;
    static constexpr bool BF16 = BF16_;
    static constexpr int NT = D <= 128 ? 2 : 1, NE = kGqaTile;
    static constexpr int Slot = NE * D * 2, QTile = 128 * D * 2;
    static constexpr int Slots = (225 * 1024 - NT * QTile) / Slot / 2 * 2;      // (even: a slot holds K always, or V, and the same warps see all of its turns)
    static constexpr int Flags = 16;              // steps whose page flags are kept: the producer is at most Slots / 2 + 2 ahead of the softmax warps
    static_assert(Slots / 2 + 2 < Flags, "");
    static constexpr int SoftmaxWarps = 4 * NT, Threads = (SoftmaxWarps + 2 + NT) * 32;
    static constexpr int OffRing = NT * QTile, OffBars = OffRing + Slots * Slot, OffThere = OffBars + 8 * (2 * Slots + 2 * NT + 6 * NT), OffMisc = OffThere + 4 * Flags;
    static constexpr int Bytes = (OffMisc + 16 + 127) / 128 * 128 + 1024;
    static constexpr int ColO = 256;
};

// Units in the order of their steps: a counting sort.
__global__ void __launch_bounds__(kPrefillPlanThreads) gqa_plan_kernel(const __grid_constant__ GqaPrefillArgs p) {
    __shared__ int count[kPrefillBuckets];
    __shared__ int64_t sums[kPrefillPlanThreads / 32];
    __shared__ int most;
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const GqaArgs& a = p.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int block_tokens = a.group_rows / a.G;
    for (int i = tid; i < kPrefillBuckets; i += kPrefillPlanThreads) count[i] = 0;
    if (tid == 0) most = 0;
    __syncthreads();
    auto each = [&](auto&& f) {
        for (int b = warp; b < a.B; b += kPrefillPlanThreads / 32) {
            const GqaRequest r = gqa_request(a, b);
            for (int i = lane; i * int64_t(block_tokens) < r.tokens; i += 32) f(b, i, gqa_token_span(r.place0, r.entries, i * block_tokens, min((i + 1) * block_tokens, r.tokens) - 1, a.window, a.first).count);
        }
    };
    for (int b = tid; b < a.B; b += kPrefillPlanThreads)
        if (gqa_request(a, b).bad) gqa_report(a.status, kGqaStatusBadIndex, 4, p.b0 + b);
    int top = 0;
    each([&](int, int, int steps) { top = max(top, steps); });
    atomicMax(&most, top);
    __syncthreads();
    const int shift = max(0, 32 - __clz(most) - 10);                          // steps >> shift < 1024
    each([&](int, int, int steps) { atomicAdd(&count[kPrefillBuckets - 1 - (steps >> shift)], 1); });
    __syncthreads();
    int64_t total;
    const int64_t before = block_prefix<kPrefillPlanThreads>(count[tid], total, sums);
    __syncthreads();
    count[tid] = int(before);
    __syncthreads();
    int2* const list = reinterpret_cast<int2*>(p.plan + 4);
    // (offsets that overlap, which are reported, can name more blocks than there are rows for)
    each([&](int b, int i, int steps) {
        const int at = atomicAdd(&count[kPrefillBuckets - 1 - (steps >> shift)], 1);
        if (at < p.plan_units) list[at] = make_int2(b, i);
    });
    if (tid == 0) p.plan[0] = int(min(total, int64_t(p.plan_units)));
}

// ── tcgen05, one block ──
// Descriptors as halves: from one instruction to the next only the low one changes, by a constant (computed anew for each they took longer than the products).
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}\n"
                 :: "r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}\n"
                 :: "r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                    "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const void* tensor_map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(smem_dst), "l"(reinterpret_cast<uint64_t>(tensor_map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}

// The units of a block, walked by each role for itself.
struct PrefillWalk {
    int u, total, h;
    GqaRequest req;
    GqaSpan span;
    int b;
    __device__ __forceinline__ void take(const GqaPrefillArgs& p) {
        if (u >= total) return;
        const GqaArgs& a = p.g;
        const int nth = u / p.heads;
        h = p.h0 + u - nth * p.heads;
        const int32_t* const at = p.plan + 4 + 2 * nth;
        b = ptx::ld(at);
        const int block = ptx::ld(at + 1), tokens = a.group_rows / a.G;
        req = gqa_request(a, b);
        span = gqa_token_span(req.place0, req.entries, block * tokens, min((block + 1) * tokens, req.tokens) - 1, a.window, a.first);
    }
    __device__ __forceinline__ void begin(const GqaPrefillArgs& p) {
        total = ptx::ld(p.plan) * p.heads;
        u = blockIdx.x;
        take(p);
    }
    __device__ __forceinline__ bool more() const { return u < total; }
    __device__ __forceinline__ void next(const GqaPrefillArgs& p) {
        u += gridDim.x;
        take(p);
    }
};

template <class C>
__global__ void __launch_bounds__(C::Threads, 1) gqa_prefill_kernel(const __grid_constant__ GqaPrefillArgs p) {
    constexpr int D = C::D, NT = C::NT, NE = C::NE;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const base = smem_raw + (smem - ptx::smem_u32(smem_raw));
    const uint32_t ring = smem + C::OffRing;
    const uint32_t kv_full = smem + C::OffBars, kv_empty = kv_full + 8 * C::Slots, q_full = kv_empty + 8 * C::Slots, q_empty = q_full + 8 * NT;
    const uint32_t s_full = q_empty + 8 * NT, p_full = s_full + 16 * NT, o_full = p_full + 16 * NT;     // of (tile, buffer)
    volatile uint32_t* const there = reinterpret_cast<volatile uint32_t*>(base + C::OffThere);      // of a step: its page is in the pool
    volatile uint32_t* const tmem_at = reinterpret_cast<volatile uint32_t*>(base + C::OffMisc);
    const GqaArgs& a = p.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < C::Slots; ++i) { ptx::mbar_init(kv_full + 8 * i, 1);  ptx::mbar_init(kv_empty + 8 * i, NT); }
        for (int i = 0; i < NT; ++i) { ptx::mbar_init(q_full + 8 * i, 1);  ptx::mbar_init(q_empty + 8 * i, 1); }
        for (int i = 0; i < 2 * NT; ++i) { ptx::mbar_init(s_full + 8 * i, 1);  ptx::mbar_init(p_full + 8 * i, 4);  ptx::mbar_init(o_full + 8 * i, 1); }
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&p.q_map);
        ptx::prefetch_tensormap(&a.k_map);
        ptx::prefetch_tensormap(&a.v_map);
    }
    if (warp == C::SoftmaxWarps) {
        ptx::tmem_alloc(smem + C::OffMisc, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = *tmem_at;
    ptx::pdl_trigger();
    ptx::pdl_wait();
    PrefillWalk w;
    w.begin(p);
    bool ok = true;
    // Two barriers at a time where a role waits for two: a look takes long while products keep the shared memory busy.
    auto wait = [&](uint32_t bar, uint32_t turn, int role, int what) {
        if (!ok) return;
        // (in line: a called function would take registers by the convention of calls, which the split of registers leaves no room for)
        if (__all_sync(0xFFFFFFFFu, ptx::mbar_try_wait(bar, turn & 1u))) return;
        const uint32_t t0 = ptx::globaltimer_lo();
        bool done;
        do { done = ptx::mbar_try_wait(bar, turn & 1u); } while (!done && ptx::globaltimer_lo() - t0 < a.wait_ns);
        if (!__all_sync(0xFFFFFFFFu, done)) {
            if (lane == 0) gqa_report(a.status, kGqaStatusWait, role, what);
            ok = false;
        }
    };

    auto wait2 = [&](uint32_t bar_a, uint32_t turn_a, uint32_t bar_b, uint32_t turn_b, int role, int what) {
        const bool a_done = ptx::mbar_try_wait(bar_a, turn_a & 1u), b_done = ptx::mbar_try_wait(bar_b, turn_b & 1u);
        if (__all_sync(0xFFFFFFFFu, a_done && b_done)) return;
        wait(bar_a, turn_a, role, what);
        wait(bar_b, turn_b, role, what);
    };

    if (warp == C::SoftmaxWarps) {
        // ── producer ──
        uint32_t seq = 0, unit = 0;
        for (; w.more() && ok; w.next(p), ++unit) {
            for (int t = 0; t < NT && ok; ++t) {
                if (unit > 0) wait(q_empty + 8 * t, unit - 1, 0, int(unit));
                if (ok && ptx::elect_one()) {
                    ptx::mbar_arrive_expect_tx(q_full + 8 * t, uint32_t(p.tile_tokens * a.G * D * 2));
#pragma unroll
                    for (int x = 0; x < D / 64; ++x)
                        ptx::tma_load_3d(smem + t * C::QTile + x * (128 * 128), &p.q_map, 64 * x, w.h * a.G, int(w.req.row0) + w.span.t0 + t * p.tile_tokens, q_full + 8 * t);
                }
                __syncwarp();
            }
            for (int k = 0; k < w.span.count && ok; k += 32) {
                // the pages of the next 32 steps, one per lane
                int page = -1;
                const int slot = w.span.slot(k + lane);
                if (k + lane < w.span.count && w.span.has(slot)) {
                    page = ptx::ld(a.block_table + int64_t(w.b) * a.max_pages + slot);
                    if (page < 0 || page >= a.num_pages || (p.own_pages > 0 && slot >= p.own_pages)) {
                        gqa_report(a.status, kGqaStatusBadIndex, 4, page);
                        page = -1;
                    } else if (p.own_pages > 0) {
                        page = w.b * p.own_pages + slot;
                    }
                }
                const int n = min(32, w.span.count - k);
                for (int i = 0; i < n && ok; ++i) {
                    const int pg = __shfl_sync(0xFFFFFFFFu, page, i), e0 = w.span.slot(k + i) * NE;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv, ++seq) {
                        const uint32_t st = seq % C::Slots, round = seq / C::Slots;
                        if (round > 0) wait(kv_empty + 8 * st, round - 1, 0, int(seq));
                        if (!ok) break;
                        if (a.dbg_drop_tile >= 0 && int(seq) == 2 * a.dbg_drop_tile) continue;       // a test's lost arrival
                        if (ptx::elect_one()) {
                            const uint32_t full = kv_full + 8 * st, at = ring + st * C::Slot;
                            if (kv == 0) there[(seq / 2) % C::Flags] = pg >= 0;
                            ptx::mbar_arrive_expect_tx(full, C::Slot);
                            const int row = pg >= 0 ? pg * kGqaTile : int(p.pool_rows);
                            if (kv == 0 || pg < 0 || (e0 + NE <= w.span.hi && (e0 >= w.span.lo || e0 + NE <= w.span.first))) {
#pragma unroll
                                for (int x = 0; x < D / 64; ++x) ptx::tma_load_3d(at + x * (NE * 128), kv ? &a.v_map : &a.k_map, 64 * x, w.h - p.h0, row, full);
                            } else {
                                auto seen = [&](int i) { return i < w.span.hi && (i >= w.span.lo || i < w.span.first); };
                                for (int r8 = 0; r8 < NE; r8 += 8) {
                                    uint32_t bits = 0;
                                    for (int r = 0; r < 8; ++r) bits |= uint32_t(seen(e0 + r8 + r)) << r;
                                    for (int x = 0; x < D / 64; ++x) {
                                        const uint32_t to = at + x * (NE * 128) + r8 * 128;
                                        if (bits == 0u || bits == 255u) {
                                            ptx::tma_load_3d(to, &p.v8_map, 64 * x, w.h - p.h0, bits ? row + r8 : int(p.pool_rows), full);
                                        } else {
                                            for (int r = 0; r < 8; ++r)
                                                ptx::tma_load_3d(to + r * 128, &p.v1_map, 64 * x, w.h - p.h0, (bits >> r) & 1u ? row + r8 + r : int(p.pool_rows), full);
                                        }
                                    }
                                }
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
    } else if (warp == C::SoftmaxWarps + 1) {
        // ── outputs ──
        // (this warp for these products, one for each tile's scores: while one looks at its barriers, 130 to 210 cycles a look, the tensor cores have the others' products)
        constexpr uint32_t kIdesc = C::BF16 ? ptx::make_idesc_bf16(128, D, false, true) : ptx::make_idesc_f16(128, D, false, true), kDescHi = ptx::smem_desc_hi(1024);
        const uint32_t ring_lo = ptx::smem_desc_lo(ring, NE * 128);
        uint32_t at = 0;                                                      // steps of all units so far
        for (; w.more() && ok; w.next(p)) {
            for (int j = 0; j < w.span.count && ok; ++j, ++at) {
                const uint32_t st = (2 * at + 1) % C::Slots, v_lo = ring_lo + st * (C::Slot >> 4);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint32_t bar = p_full + 8 * (2 * t + (at & 1));
                    if (t == 0) wait2(kv_full + 8 * st, (2 * at + 1) / C::Slots, bar, at >> 1, 1, int(at));
                    else wait(bar, at >> 1, 1, int(at));
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
                    const uint32_t p_at = tmem + (2 * t + (at & 1)) * NE;
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int k = 0; k < NE / 16; ++k) mma_ts(tmem + C::ColO + t * D, p_at + k * 8, v_lo + (k * 2048 >> 4), kDescHi, kIdesc, j > 0 || k ? 1u : 0u);
                        ptx::mma_commit(o_full + 8 * (2 * t + (at & 1)));
                        if (t == NT - 1)
                            for (int i = 0; i < NT; ++i) ptx::mma_commit(kv_empty + 8 * st);         // (as many arrivals as K's slots get)
                    }
                    __syncwarp();
                }
            }
        }
    } else if (warp >= C::SoftmaxWarps + 2) {
        // ── scores of a tile ──
        constexpr uint32_t kIdesc = C::BF16 ? ptx::make_idesc_bf16(128, NE, false, false) : ptx::make_idesc_f16(128, NE, false, false), kDescHi = ptx::smem_desc_hi(1024);
        const int t = warp - C::SoftmaxWarps - 2;
        const uint32_t q_lo = ptx::smem_desc_lo(smem + t * C::QTile, 16), ring_lo = ptx::smem_desc_lo(ring, 16);
        uint32_t at = 0, unit = 0;
        for (; w.more() && ok; w.next(p), ++unit) {
            wait(q_full + 8 * t, unit, 1, int(unit));
            for (int j = 0; j < w.span.count; ++j, ++at) {
                const uint32_t st = (2 * at) % C::Slots, buffer = 2 * t + (at & 1);
                // K is there, and the buffer's P, of two steps ago, has been multiplied
                if (at >= 2) wait2(kv_full + 8 * st, (2 * at) / C::Slots, o_full + 8 * buffer, (at - 2) >> 1, 1, int(at));
                else wait(kv_full + 8 * st, (2 * at) / C::Slots, 1, int(at));
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const uint32_t k_lo = ring_lo + st * (C::Slot >> 4), s_at = tmem + buffer * NE;
                const bool last = j + 1 == w.span.count;
                if (ptx::elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_ss(s_at, q_lo + (((k / 4) * (128 * 128) + (k % 4) * 32) >> 4), k_lo + (((k / 4) * (NE * 128) + (k % 4) * 32) >> 4), kDescHi, kIdesc, k ? 1u : 0u);
                    ptx::mma_commit(s_full + 8 * buffer);
                    if (last) ptx::mma_commit(q_empty + 8 * t);
                    ptx::mma_commit(kv_empty + 8 * st);
                }
                __syncwarp();
            }
        }
    } else {
        // ── softmax: a thread has a row ──
        const int t = warp >> 2;
        const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
        const int r = (warp & 3) * 32 + lane, tok = r / a.G, gg = r - tok * a.G;
        const int H = a.Hkv * a.G;
        const bool real = r < p.tile_tokens * a.G;                            // (rows behind hold what the memory held)
        const float neg = -INFINITY;
        constexpr float kUp = C::BF16 ? 0.f : kGqaUp;                         // (P in FP16, taken 2^7 larger)
        uint32_t step = 0, unit = 0;
        bool ahead = false;                                                   // the next step's scores are known to be there
        for (; w.more() && ok; w.next(p), ++unit) {
            const int token = w.span.t0 + t * p.tile_tokens + tok, place = w.req.place0 + token;
            const int first_place = w.req.place0 + w.span.t0 + t * p.tile_tokens, last_place = first_place + p.tile_tokens - 1;
            const float scale = a.k_scale != nullptr ? gqa_positive(a.scale_log2 * ptx::ld(a.k_scale + w.h)) : a.scale_log2;
            float ref = neg, l = 0.f;
            for (int j = 0; j < w.span.count; ++j, ++step) {
                const int i = 2 * t + int(step & 1);
                const uint32_t s_at = lane_base + i * NE;
                const int e0 = w.span.slot(j) * NE;
                // (the producer's flags: K has arrived when its scores have)
                if (!ahead) wait(s_full + 8 * i, step >> 1, 2, int(step));
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const bool page = there[step % C::Flags] != 0;
                const bool whole = page && e0 + NE - 1 <= first_place && e0 + NE <= w.req.entries &&
                                   (a.window == 0 || e0 > last_place - a.window || e0 + NE - 1 < a.first);
                // A row whose maximum has passed its reference by too much, or that sees its first entry, takes the maximum as its reference; O so far is rescaled.
                auto refer = [&](float top) {
                    const bool move = real && (ref == neg ? top > neg : (top - ref) * scale > kPrefillLazy);
                    if (!__any_sync(0xFFFFFFFFu, move)) return;
                    float by = 1.f;
                    if (move) {
                        if (ref != neg) by = ptx::ex2((ref - top) * scale);
                        ref = top;
                        l *= by;
                    }
                    if (j == 0) return;
                    wait(o_full + 8 * (2 * t + int((step - 1) & 1)), (step - 1) >> 1, 2, int(step));
                    ptx::tc_fence_after_sync();
                    const uint32_t o_at = lane_base + C::ColO + t * D;
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16(o_at + 16 * c, o);
                        ptx::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * by);
                        tmem_st16(o_at + 16 * c, o);
                    }
                    ptx::tmem_wait_st();
                };
                bool done = false;
                if (whole) {
                    // all of the row's scores in registers
                    uint32_t v[NE / 32][32];
#pragma unroll
                    for (int c = 0; c < NE / 32; ++c) ptx::tmem_ld32(s_at + 32 * c, v[c]);
                    ptx::tmem_wait_ld();
                    float top[4] = {neg, neg, neg, neg};
#pragma unroll
                    for (int c = 0; c < NE / 32; ++c)
#pragma unroll
                        for (int x = 0; x < 32; x += 8)
#pragma unroll
                            for (int q = 0; q < 4; ++q) top[q] = ptx::max3(top[q], __uint_as_float(v[c][x + 2 * q]), __uint_as_float(v[c][x + 2 * q + 1]));
                    refer(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                    const float sub = ref == neg ? kUp : fmaf(-ref, scale, kUp);
                    // (where scores are so large that the rounding of this product would tell, the other way)
                    done = !__any_sync(0xFFFFFFFFu, fabsf(sub) >= 16777216.f);
                    if (done) {
                        const uint64_t sub2 = ptx::pack_f32x2(sub, sub), scale2 = ptx::pack_f32x2(scale, scale);
                        // the step's own sum, which the row's joins last (0.997 ms; with `l += a0 + a1` instead, or the row's sum kept in two parts, 1.035)
                        uint64_t s0 = 0, s1 = 0;
#pragma unroll
                        for (int c = 0; c < NE / 32; ++c) {
                            uint32_t pk[16];
#pragma unroll
                            for (int x = 0; x < 32; x += 2) {
                                float x0, x1;
                                ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(__uint_as_float(v[c][x]), __uint_as_float(v[c][x + 1])), scale2, sub2), x0, x1);
                                x0 = ptx::ex2(x0);
                                x1 = ptx::ex2(x1);
                                const uint64_t both = ptx::pack_f32x2(x0, x1);
                                if (x & 2) s1 = c == 0 && x == 2 ? both : ptx::add_f32x2(s1, both);
                                else s0 = c == 0 && x == 0 ? both : ptx::add_f32x2(s0, both);
                                pk[x / 2] = C::BF16 ? ptx::pack_bf16x2(x0, x1) : ptx::pack_f16x2(x0, x1);
                            }
                            tmem_st16(s_at + 16 * c, pk);
                        }
                        float a0, a1;
                        ptx::unpack_f32x2(ptx::add_f32x2(ptx::add_f32x2(s0, ptx::pack_f32x2(l, 0.f)), s1), a0, a1);
                        l = a0 + a1;
                    }
                }
                if (!done) {
                    // 32 scores at a time; what the row does not see is -inf.  Differences are taken before they are scaled: at the maximum 0, however large it is.
                    auto load = [&](uint32_t (&v)[32], int c) {
                        ptx::tmem_ld32(s_at + 32 * c, v);
                        const int at = e0 + 32 * c;
                        auto below = [](int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; };
                        uint32_t see = below(min(place + 1, w.req.entries) - at);
                        if (a.window > 0) see &= ~below(place - a.window + 1 - at) | below(a.first - at);
                        if (!page) see = 0u;
                        ptx::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (!((see >> x) & 1u)) v[x] = __float_as_uint(neg);
                    };
                    float t0 = neg, t1 = neg;
#pragma unroll 1
                    for (int c = 0; c < NE / 32; ++c) {
                        uint32_t v[32];
                        load(v, c);
#pragma unroll
                        for (int x = 0; x < 32; x += 4) {
                            t0 = ptx::max3(t0, __uint_as_float(v[x]), __uint_as_float(v[x + 1]));
                            t1 = ptx::max3(t1, __uint_as_float(v[x + 2]), __uint_as_float(v[x + 3]));
                        }
                    }
                    refer(fmaxf(t0, t1));
                    const float sub = ref == neg ? 0.f : ref;
                    float sum = 0.f;
                    // (P of 32 entries takes the place of scores that have been read)
#pragma unroll 1
                    for (int c = 0; c < NE / 32; ++c) {
                        uint32_t v[32], pk[16];
                        load(v, c);
#pragma unroll
                        for (int x = 0; x < 32; x += 2) {
                            const float x0 = ptx::ex2(fmaf(__uint_as_float(v[x]) - sub, scale, kUp)), x1 = ptx::ex2(fmaf(__uint_as_float(v[x + 1]) - sub, scale, kUp));
                            sum += x0 + x1;
                            pk[x / 2] = C::BF16 ? ptx::pack_bf16x2(x0, x1) : ptx::pack_f16x2(x0, x1);
                        }
                        tmem_st16(s_at + 16 * c, pk);
                    }
                    l += sum;
                }
                // a look at the next step's scores, whose answer comes while P is on its way
                ahead = ptx::mbar_try_wait(s_full + 8 * (2 * t + int((step + 1) & 1)), ((step + 1) >> 1) & 1u);
                ptx::tmem_wait_st();
                ptx::tc_fence_before_sync();
                ahead = __all_sync(0xFFFFFFFFu, ahead);
                if (lane == 0) ptx::mbar_arrive(p_full + 8 * i);
            }
            if (!ok) break;
            // ── the row's output ──
            // (scores of the last step came after the outputs of two steps before, so that the wait cannot take an earlier turn of the barrier for this one)
            wait(o_full + 8 * (2 * t + int((step - 1) & 1)), (step - 1) >> 1, 3, int(unit));
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const bool mine = real && token <= w.span.t1;
            const int head = w.h * a.G + gg;
            const int64_t row = (w.req.row0 + token) * H + head;
            const bool none = l == 0.f;
            float all = l, by = 1.f;
            if (mine && a.sink != nullptr && !none) {
                const float s = ptx::ld(a.sink + head) * 1.4426950408889634f, top = fmaf(ref, scale, -kUp), m2 = fmaxf(top, s);
                by = ptx::ex2(top - m2);
                all = l * by + gqa_sink(s, m2);
            }
            const float per = none ? 0.f : by * (a.v_scale != nullptr ? ptx::ld(a.v_scale + w.h) : 1.f) / all;
            uint8_t* const to = static_cast<uint8_t*>(a.out) + row * (D * 2);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t v[32];
                ptx::tmem_ld32(lane_base + C::ColO + t * D + 32 * c, v);
                ptx::tmem_wait_ld();
                if (mine) {
                    uint32_t o[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const float o0 = none ? 0.f : __uint_as_float(v[2 * x]) * per, o1 = none ? 0.f : __uint_as_float(v[2 * x + 1]) * per;
                        o[x] = C::BF16 ? ptx::pack_bf16x2(o0, o1) : ptx::pack_f16x2(o0, o1);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) *reinterpret_cast<uint4*>(to + 64 * c + 16 * x) = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
                }
            }
            if (mine && a.lse != nullptr) a.lse[row] = none ? neg : (fmaf(ref, scale, -kUp) + log2f(l)) * 0.6931471805599453f;
            ptx::tc_fence_before_sync();
        }
    }
    // common exit: every role comes here, with or without a failure
    ptx::tc_fence_before_sync();
    const bool failed = __syncthreads_or(!ok);
    if (failed) {
        const uint32_t t0 = ptx::globaltimer_lo();                            // copies and products that are on their way end within microseconds
        while (ptx::globaltimer_lo() - t0 < 1000000u) __nanosleep(1000);
    }
    if (warp == C::SoftmaxWarps) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, 512);
    }
}

// ── an 8-bit cache's pages in 16 bits ──
// e4m3 values (exact in BF16 and FP16; the scales go into scores and outputs, but for the sign of K's, which is put in here) of every page that some token sees, to pages of the call's own:
// [requests * own_pages][64][heads][D].  A request has some blocks, which go through the pages that it holds.
constexpr int kGqaUnpackThreads = 256;
struct GqaUnpackArgs {
    GqaArgs g;                       // the launch's requests
    const uint8_t* pool[2];
    uint8_t* rows[2];
    int own_pages, blocks;           // pages and blocks of a request
    int h0, heads, D;
};
template <bool BF16>
__global__ void __launch_bounds__(kGqaUnpackThreads) gqa_unpack_kernel(const __grid_constant__ GqaUnpackArgs u) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const GqaArgs& a = u.g;
    const int b = int(blockIdx.x / uint32_t(u.blocks));
    const GqaRequest r = gqa_request(a, b);
    if (r.tokens == 0) return;
    // 16-byte pieces: 2^head_log2 of a head's row, `entry` of an entry's heads, of which a thread's next one is `entries` entries and `rest` pieces on
    const uint32_t head_log2 = 31 - __clz(uint32_t(u.D) / 16), entry = uint32_t(u.heads) << head_log2, vecs = entry * kGqaTile, entries = kGqaUnpackThreads / entry, rest = kGqaUnpackThreads - entries * entry;
    const uint32_t e0 = threadIdx.x / entry, at0 = threadIdx.x - e0 * entry;
    const int64_t pool_entry = int64_t(a.Hkv) << head_log2;
    const int lo = a.window > 0 ? max(r.place0 - a.window + 1, 0) : 0, pages = min((r.entries + kGqaTile - 1) / kGqaTile, u.own_pages);
    for (int slot = int(blockIdx.x) - b * u.blocks; slot < pages; slot += u.blocks) {
        const int from = slot * kGqaTile;
        if (from + kGqaTile <= lo && from >= a.first) continue;
        const int page = ptx::ld(a.block_table + int64_t(b) * a.max_pages + slot);
        if (page < 0 || page >= a.num_pages) continue;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
            const uint4* const src = reinterpret_cast<const uint4*>(u.pool[kv]) + int64_t(page) * kGqaTile * pool_entry + (u.h0 << head_log2);
            uint4* const dst = reinterpret_cast<uint4*>(u.rows[kv]) + (int64_t(b) * u.own_pages + slot) * vecs * 2;
            uint32_t e = e0, at = at0;
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < vecs; i += kGqaUnpackThreads) {
                const uint4 v = ptx::ldg_stream_v4(src + e * pool_entry + at);
                const uint32_t turn = kv == 0 && ptx::ld(a.k_scale + u.h0 + (at >> head_log2)) < 0.f ? 0x80008000u : 0u;
                e += entries;
                at += rest;
                if (at >= entry) {
                    at -= entry;
                    ++e;
                }
                const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ptx::e4m3x4_to_f16x4(x[j], o[2 * j], o[2 * j + 1]);
                    if (BF16)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[2 * j + q]));
                            o[2 * j + q] = ptx::pack_bf16x2(f.x, f.y);
                        }
                    o[2 * j] ^= turn;
                    o[2 * j + 1] ^= turn;
                }
                ptx::stg_v8(dst + 2 * i, make_uint4(o[0], o[1], o[2], o[3]), make_uint4(o[4], o[5], o[6], o[7]));
            }
        }
    }
}

}  // namespace dsv4
