// Attention of new tokens where a KV head has many rows (drafted tokens x query heads of a group): the decode kernel's shares of the cache on the tensor cores.
//
// The shares, units and parts are those of gqa_decode.cuh, with up to 128 rows in a group; the products are those of gqa_prefill.cuh.  A block's pages go in turns to two
// streams with scores, outputs and softmax warps of their own (heads of 256: one stream), so that one stream's products run beside the other's softmax.  Of a unit inside the
// share the first stream joins both parts and writes the output; of one that a cut runs through each stream leaves an FP32 part, and gqa_merge_kernel joins those of all blocks.
//
// An 8-bit cache's pages come into a ring of raw tiles; four warps bring them to FP16 (exact) in the operands' layout, zeros for V of entries that no row sees.  Q then is FP16
// too, each row brought near 1 by a power of two, and turned round where the head's scale is negative.
//
// Why not mma.sync with more rows: 64 rows x 64 entries x 128 are 512 instructions of m16n8k16, 1111 cycles at the measured 2.17 an instruction and SM, where an 8-bit page is there after
// 700; and every warp of 16 rows converts the page for itself.  64 requests x 8,000 entries, 64 query heads for each of 8 KV heads of 128: 385 us against 670, in 8 bits 401 against 999.
//
// What bounds it: the shared-memory port with 8-bit pages (12 x 5 tokens of 64 heads behind 32,768 entries 277-291 us, of which the bytes need 125: 1,024 of a page's 1,275 cycles go to the raw page in
// and out, the FP16 page in and out, and Q again for every page); DRAM with 16-bit ones.
#pragma once

#include "gqa_prefill.cuh"

namespace dsv4 {

struct GqaRowsArgs {
    GqaArgs g;                       // group_rows: tile_tokens * G; k_map, v_map: boxes of a page (e4m3: whole rows, not swizzled)
    alignas(64) CUtensorMap q_map;   // 16 bits: (element, head, token, request)
    CUtensorMap v8_map, v1_map;      // 16 bits: boxes of eight entries and of one
    int tile_tokens;                 // of a group: floor(128 / G), or floor(64 / G)
    int second;                      // 64: the second stream has its rows there (groups of up to 64 rows: the streams' softmax warps then sit on different schedulers), or 0
};

template <int D_, int KVT_>
struct RowsCfg {
    static constexpr int D = D_, KVT = KVT_;
    static constexpr bool E4M3 = KVT == kGqaE4m3, BF16 = KVT == kGqaBf16;
    static constexpr int NT = D <= 128 ? 2 : 1, NE = kGqaTile;                // streams; entries of a step
    static constexpr int Slot = NE * D * 2, QTile = 128 * D * 2, RawSlot = NE * D;
    // (a multiple of twice the streams: a slot then belongs to one stream's K or V, and the same warp sees all of its turns)
    static constexpr int Slots = E4M3 ? (D > 128 ? 2 : 8) : (D > 128 ? 4 : 8);
    static constexpr int RawSlots = E4M3 ? (D > 128 ? 4 : 8) : 1;
    static constexpr int SoftmaxWarps = 4 * NT, Convert = SoftmaxWarps + 2 + NT, Warps = Convert + (E4M3 ? 4 : 0), Threads = Warps * 32;
    static constexpr int OffRing = QTile, OffRaw = OffRing + Slots * Slot, OffBars = OffRaw + (E4M3 ? RawSlots * RawSlot : 0);
    static constexpr int Bars = 2 * Slots + 2 * RawSlots + 2 + 6 * NT + 2;
    static constexpr int Flags = 32;                                          // pages whose flags are kept
    static_assert(Slots / 2 + RawSlots / 2 + 2 * NT + 4 < Flags, "");
    static constexpr int OffThere = OffBars + 8 * Bars, OffFactor = OffThere + 4 * Flags, OffScan = OffFactor + 128 * 4, OffMisc = OffScan + 8 * 20;
    static constexpr int Bytes = (OffMisc + 16 + 127) / 128 * 128 + 1024;
    static constexpr int ColO = 256;
    static_assert(Slots % (2 * NT) == 0 && Threads <= 512 && Bytes <= 232448, "");
};

template <class C>
__global__ void __launch_bounds__(C::Threads, 1) gqa_rows_kernel(const __grid_constant__ GqaRowsArgs p) {
    constexpr int D = C::D, NT = C::NT, NE = C::NE;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const base = smem_raw + (smem - ptx::smem_u32(smem_raw));
    const uint32_t ring = smem + C::OffRing, raw = smem + C::OffRaw;
    const uint32_t kv_full = smem + C::OffBars, kv_empty = kv_full + 8 * C::Slots, raw_full = kv_empty + 8 * C::Slots, raw_empty = raw_full + 8 * C::RawSlots;
    const uint32_t q_full = raw_empty + 8 * C::RawSlots, q_empty = q_full + 8, s_full = q_empty + 8, p_full = s_full + 16 * NT, o_full = p_full + 16 * NT;      // the last three of (stream, buffer)
    const uint32_t join_full = o_full + 16 * NT, join_empty = join_full + 8;
    volatile uint32_t* const there = reinterpret_cast<volatile uint32_t*>(base + C::OffThere);      // of a tile: its page is in the pool
    float* const row_factor = reinterpret_cast<float*>(base + C::OffFactor);
    int64_t* const scan = reinterpret_cast<int64_t*>(base + C::OffScan);      // 16 warp sums; request and offset of the share
    volatile uint32_t* const tmem_at = reinterpret_cast<volatile uint32_t*>(base + C::OffMisc);
    const GqaArgs& a = p.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (tid == 0) {
        for (int i = 0; i < C::Slots; ++i) { ptx::mbar_init(kv_full + 8 * i, C::E4M3 ? 2 : 1);  ptx::mbar_init(kv_empty + 8 * i, 1); }
        for (int i = 0; i < C::RawSlots; ++i) { ptx::mbar_init(raw_full + 8 * i, 1);  ptx::mbar_init(raw_empty + 8 * i, 2); }
        ptx::mbar_init(q_full, C::E4M3 ? 4 : 1);
        ptx::mbar_init(q_empty, NT + C::SoftmaxWarps);
        ptx::mbar_init(join_full, 4);
        ptx::mbar_init(join_empty, 4);
        for (int i = 0; i < 2 * NT; ++i) { ptx::mbar_init(s_full + 8 * i, 1);  ptx::mbar_init(p_full + 8 * i, 4);  ptx::mbar_init(o_full + 8 * i, 1); }
        ptx::fence_mbar_init();
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
    ptx::pdl_wait();
    ptx::pdl_trigger();              // (behind the wait: the merge reads lengths before its own)

    // where this block's share begins
    const int each = (a.B + C::Threads - 1) / C::Threads, b_from = tid * each, b_to = min(b_from + each, a.B);
    int64_t mine = 0, total;
    for (int b = b_from; b < b_to; ++b) {
        const GqaRequest r = gqa_request(a, b);
        if (r.bad && blockIdx.x == 0) gqa_report(a.status, kGqaStatusBadIndex, 4, b);
        mine += gqa_head_tiles(a, r) * a.Hkv;
    }
    const int64_t before = block_prefix<C::Threads>(mine, total, scan);
    const int64_t share = gqa_share(a, total), begin = int64_t(blockIdx.x) * share, tiles = max(min(share, total - begin), int64_t(0));
    if (tiles > 0 && begin >= before && begin < before + mine) {
        int64_t off = begin - before;
        for (int b = b_from; b < b_to; ++b) {
            const int64_t n = gqa_head_tiles(a, gqa_request(a, b)) * a.Hkv;
            if (off < n) {
                scan[16] = b;
                scan[17] = off;
                break;
            }
            off -= n;
        }
    }
    __syncthreads();
    GqaWalk w;
    w.left = 0;
    if (tiles > 0) w.begin(a, int(scan[16]), scan[17], tiles);
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t turn, int role, int what) {
        if (!ok) return;
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
    // A tile of the block (`tile` counts them) belongs to stream tile % NT, whose step tile / NT it is.
    uint32_t tile = 0, piece = 0;

    if (warp == C::SoftmaxWarps) {
        // ── producer ──
        constexpr int kRing = C::E4M3 ? C::RawSlots : C::Slots, kBytes = C::E4M3 ? C::RawSlot : C::Slot;
        const uint32_t full = C::E4M3 ? raw_full : kv_full, empty = C::E4M3 ? raw_empty : kv_empty, at = C::E4M3 ? raw : ring;
        for (; w.left > 0 && ok; w.next(a), ++piece) {
            if (!C::E4M3) {
                if (piece > 0) wait(q_empty, piece - 1, 0, int(piece));
                if (ok && ptx::elect_one()) {
                    ptx::mbar_arrive_expect_tx(q_full, uint32_t(p.tile_tokens * a.G * D * 2) * (p.second ? 2u : 1u));
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        tma_load_4d(smem + x * (128 * 128), &p.q_map, 64 * x, w.h * a.G, w.span.t0, w.b, q_full);
                        if (p.second) tma_load_4d(smem + x * (128 * 128) + p.second * 128, &p.q_map, 64 * x, w.h * a.G, w.span.t0, w.b, q_full);
                    }
                }
                __syncwarp();
            }
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
                for (int i = 0; i < n && ok; ++i, ++tile) {
                    const int pg = __shfl_sync(0xFFFFFFFFu, page, i), e0 = w.span.slot(k + i) * NE;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const uint32_t seq = 2 * tile + kv, st = seq % kRing, round = seq / kRing;
                        if (round > 0) wait(empty + 8 * st, round - 1, 0, int(seq));
                        if (!ok) break;
                        if (a.dbg_drop_tile >= 0 && int(seq) == 2 * a.dbg_drop_tile) continue;       // a test's lost arrival
                        if (ptx::elect_one()) {
                            const uint32_t bar = full + 8 * st, to = at + st * kBytes;
                            if (kv == 0) there[tile % C::Flags] = pg >= 0;
                            ptx::mbar_arrive_expect_tx(bar, kBytes);
                            const int none = int(a.num_pages * kGqaTile), row = pg >= 0 ? pg * kGqaTile : none;
                            if (C::E4M3) {
                                ptx::tma_load_3d(to, kv ? &a.v_map : &a.k_map, 0, w.h, row, bar);
                            } else if (kv == 0 || pg < 0 || (e0 + NE <= w.span.hi && (e0 >= w.span.lo || e0 + NE <= w.span.first))) {
#pragma unroll
                                for (int x = 0; x < D / 64; ++x) ptx::tma_load_3d(to + x * (NE * 128), kv ? &a.v_map : &a.k_map, 64 * x, w.h, row, bar);
                            } else {
                                auto seen = [&](int i) { return i < w.span.hi && (i >= w.span.lo || i < w.span.first); };
                                for (int r8 = 0; r8 < NE; r8 += 8) {
                                    uint32_t bits = 0;
                                    for (int r = 0; r < 8; ++r) bits |= uint32_t(seen(e0 + r8 + r)) << r;
                                    for (int x = 0; x < D / 64; ++x) {
                                        const uint32_t to8 = to + x * (NE * 128) + r8 * 128;
                                        if (bits == 0u || bits == 255u) {
                                            ptx::tma_load_3d(to8, &p.v8_map, 64 * x, w.h, bits ? row + r8 : none, bar);
                                        } else {
                                            for (int r = 0; r < 8; ++r) ptx::tma_load_3d(to8 + r * 128, &p.v1_map, 64 * x, w.h, (bits >> r) & 1u ? row + r8 + r : none, bar);
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
        constexpr uint32_t kIdesc = C::BF16 ? ptx::make_idesc_bf16(128, D, false, true) : ptx::make_idesc_f16(128, D, false, true), kDescHi = ptx::smem_desc_hi(1024);
        const uint32_t ring_lo = ptx::smem_desc_lo(ring, NE * 128);
        for (; w.left > 0 && ok; w.next(a)) {
            for (int k = w.k0; k < w.k1 && ok; ++k, ++tile) {
                const uint32_t seq = 2 * tile + 1, st = seq % C::Slots, t = tile % NT, at = tile / NT, buffer = 2 * t + (at & 1);
                wait2(kv_full + 8 * st, seq / C::Slots, p_full + 8 * buffer, at >> 1, 1, int(tile));
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const uint32_t v_lo = ring_lo + st * (C::Slot >> 4), p_at = tmem + buffer * NE, o_at = tmem + C::ColO + t * D;
                const uint32_t add = k - w.k0 >= NT ? 1u : 0u;                // (the stream's first tile of the piece begins anew)
                if (ptx::elect_one()) {
#pragma unroll
                    for (int x = 0; x < NE / 16; ++x) mma_ts(o_at, p_at + x * 8, v_lo + (x * 2048 >> 4), kDescHi, kIdesc, x ? 1u : add);
                    ptx::mma_commit(o_full + 8 * buffer);
                    ptx::mma_commit(kv_empty + 8 * st);
                }
                __syncwarp();
            }
        }
    } else if (warp >= C::SoftmaxWarps + 2 && warp < C::Convert) {
        // ── scores of a stream ──
        constexpr uint32_t kIdesc = C::BF16 ? ptx::make_idesc_bf16(128, NE, false, false) : ptx::make_idesc_f16(128, NE, false, false), kDescHi = ptx::smem_desc_hi(1024);
        const uint32_t t = warp - C::SoftmaxWarps - 2;
        const uint32_t q_lo = ptx::smem_desc_lo(smem, 16), ring_lo = ptx::smem_desc_lo(ring, 16);
        for (; w.left > 0 && ok; w.next(a), ++piece) {
            wait(q_full, piece, 1, int(piece));
            for (int k = w.k0; k < w.k1 && ok; ++k, ++tile) {
                if (tile % NT != t) continue;
                const uint32_t seq = 2 * tile, st = seq % C::Slots, at = tile / NT, buffer = 2 * t + (at & 1);
                // K is there, and the buffer's P, of two steps ago, has been multiplied
                if (at >= 2) wait2(kv_full + 8 * st, seq / C::Slots, o_full + 8 * buffer, (at - 2) >> 1, 1, int(tile));
                else wait(kv_full + 8 * st, seq / C::Slots, 1, int(tile));
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const uint32_t k_lo = ring_lo + st * (C::Slot >> 4), s_at = tmem + buffer * NE;
                if (ptx::elect_one()) {
#pragma unroll
                    for (int x = 0; x < D / 16; ++x)
                        mma_ss(s_at, q_lo + (((x / 4) * (128 * 128) + (x % 4) * 32) >> 4), k_lo + (((x / 4) * (NE * 128) + (x % 4) * 32) >> 4), kDescHi, kIdesc, x ? 1u : 0u);
                    ptx::mma_commit(s_full + 8 * buffer);
                    ptx::mma_commit(kv_empty + 8 * st);
                }
                __syncwarp();
            }
            if (!ok) break;
            // this stream is done with Q when its products so far are
            if (ptx::elect_one()) ptx::mma_commit(q_empty);
            __syncwarp();
        }
    } else if (C::E4M3 && warp >= C::Convert) {
        // ── e4m3 -> FP16 ──
        const int cw = warp - C::Convert;
        for (; w.left > 0 && ok; w.next(a), ++piece) {
            if (piece > 0) wait(q_empty, piece - 1, 0, int(piece));
            if (!ok) break;
            {
                constexpr int kLanes = D / 8, kRows = 32 / kLanes;            // lanes of a row, 16 bytes each; rows of a load
                const uint32_t turn = ptx::ld(a.k_scale + w.h) < 0.f ? 0x80008000u : 0u;
                const int l = lane % kLanes, rows = w.req.tokens * a.G, first = w.rg * a.group_rows;
#pragma unroll 4
                for (int i = 0; i < 32 / kRows; ++i) {
                    const int r = 32 * cw + i * kRows + lane / kLanes, of = p.second > 0 && r >= p.second ? r - p.second : r;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (of < a.group_rows && first + of < rows) {
                        const int t = int(uint32_t(first + of) / uint32_t(a.G)), gg = first + of - t * a.G;
                        v = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.q) + 2 * (int64_t(w.b) * a.q_stride_b + t * a.q_stride_t + int64_t(w.h * a.G + gg) * a.q_stride_h + 8 * l));
                    }
                    const float factor = a.q_bf16 ? gqa_near_one<kLanes>(v) : 1.f;
                    if (l == 0) row_factor[r] = factor;
                    v.x ^= turn;  v.y ^= turn;  v.z ^= turn;  v.w ^= turn;
                    ptx::sts_v4(smem + (l / 8) * (128 * 128) + r * 128 + (((l % 8) ^ (r & 7)) << 4), v);
                }
            }
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(q_full);
            for (int k = w.k0; k < w.k1 && ok; ++k, ++tile) {
                const int e0 = w.span.slot(k) * NE;
                const bool all = e0 + NE <= w.span.hi && (e0 >= w.span.lo || e0 + NE <= w.span.first);
                // Two warps have K, two V, half a page each.  A lane takes 16 bytes: pairs of rows, of which one has the even and the other the odd 64 bytes, so that eight lanes meet all
                // banks both ways.
                constexpr int kHalves = D / 64;
                const int c = lane & 3, u = (lane >> 2) & 1, kv = cw >> 1, e_first = 32 * (cw & 1) + 2 * (lane >> 3) + u;
                const uint32_t seq = 2 * tile + kv, from = seq % C::RawSlots, st = seq % C::Slots, dst = ring + st * C::Slot;
                if (seq >= C::Slots) wait2(raw_full + 8 * from, seq / C::RawSlots, kv_empty + 8 * st, seq / C::Slots - 1, 0, int(seq));
                else wait(raw_full + 8 * from, seq / C::RawSlots, 0, int(seq));
                if (!ok) break;
                uint4 v[4][kHalves];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) v[i][h] = ptx::lds_v4(raw + from * C::RawSlot + (e_first + 8 * i) * D + 16 * (4 * (kHalves > 1 ? h ^ u : 0) + c));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = e_first + 8 * i, at = e0 + e;
                    const bool zero = kv == 1 && !all && !(at < w.span.hi && (at >= w.span.lo || at < w.span.first));
#pragma unroll
                    for (int h = 0; h < kHalves; ++h) {
                        const int ch = 4 * (kHalves > 1 ? h ^ u : 0) + c;
                        uint4 lo, hi;
                        ptx::e4m3x4_to_f16x4(v[i][h].x, lo.x, lo.y);
                        ptx::e4m3x4_to_f16x4(v[i][h].y, lo.z, lo.w);
                        ptx::e4m3x4_to_f16x4(v[i][h].z, hi.x, hi.y);
                        ptx::e4m3x4_to_f16x4(v[i][h].w, hi.z, hi.w);
                        if (zero) lo = hi = make_uint4(0, 0, 0, 0);
                        const uint32_t to = dst + (ch / 4) * (NE * 128) + e * 128;
                        ptx::sts_v4(to + (((2 * (ch % 4)) ^ (e & 7)) << 4), lo);
                        ptx::sts_v4(to + (((2 * (ch % 4) + 1) ^ (e & 7)) << 4), hi);
                    }
                }
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    ptx::mbar_arrive(kv_full + 8 * st);
                    ptx::mbar_arrive(raw_empty + 8 * from);
                }
            }
        }
    } else if (warp < C::SoftmaxWarps) {
        // ── softmax: a thread has a row of a stream ──
        const uint32_t t = warp >> 2;
        const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
        const int at_row = (warp & 3) * 32 + lane, r = at_row - (t == 1 ? p.second : 0);      // row of the tile, and of the group
        const float neg = -INFINITY;
        constexpr float kUp = C::BF16 ? 0.f : kGqaUp;
        uint32_t joined = 0;                                                  // units that both streams have joined
        for (; w.left > 0 && ok; w.next(a), ++piece) {
            const int rows = w.req.tokens * a.G, row = w.rg * a.group_rows + r;
            const bool real = r >= 0 && r < a.group_rows && row < rows;
            const int token = real ? int(uint32_t(row) / uint32_t(a.G)) : w.span.t1, place = w.req.place0 + token;
            const int first_place = w.req.place0 + w.span.t0, last_place = w.req.place0 + w.span.t1;
            const bool warp_real = __any_sync(0xFFFFFFFFu, real);
            float scale = a.scale_log2 * (a.k_scale != nullptr ? ptx::ld(a.k_scale + w.h) : 1.f);
            // (without the wait a stream that has no tile of a piece would arrive for the next one too early)
            wait(q_full, piece, 2, int(piece));
            if (!ok) break;
            if (C::E4M3) scale = gqa_positive(scale * row_factor[at_row]);
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(q_empty);                         // (its factors have been read)
            float* const logits = a.logits != nullptr && real ? a.logits + ((int64_t(w.b) * a.Hkv + w.h) * rows + row) * a.logit_stride : nullptr;
            float ref = neg, l = 0.f;
            uint32_t last = 0;
            bool any = false;                                                 // the stream has had a tile of the piece
            for (int k = w.k0; k < w.k1; ++k, ++tile) {
                if (tile % NT != t) continue;
                const uint32_t at = tile / NT, buffer = 2 * t + (at & 1), s_at = lane_base + buffer * NE;
                const int e0 = w.span.slot(k) * NE;
                wait(s_full + 8 * buffer, at >> 1, 2, int(tile));
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const bool page = there[tile % C::Flags] != 0;
                if (warp_real) {
                    const bool whole = page && e0 + NE - 1 <= first_place && e0 + NE <= w.req.entries && (a.window == 0 || e0 > last_place - a.window || e0 + NE <= a.first);
                    // the row's scores, not scaled; what it does not see is -inf
                    uint32_t v[2][32];
                    ptx::tmem_ld32(s_at, v[0]);
                    ptx::tmem_ld32(s_at + 32, v[1]);
                    ptx::tmem_wait_ld();
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int from = e0 + 32 * c;
                            auto below = [](int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; };
                            uint32_t see = below(min(place + 1, w.req.entries) - from);
                            if (a.window > 0) see &= ~below(place - a.window + 1 - from) | below(a.first - from);
                            if (!page) see = 0u;
#pragma unroll
                            for (int x = 0; x < 32; ++x)
                                if (!((see >> x) & 1u)) v[c][x] = __float_as_uint(neg);
                        }
                    }
                    float tops[4] = {neg, neg, neg, neg};
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int x = 0; x < 32; x += 8)
#pragma unroll
                            for (int q = 0; q < 4; ++q) tops[q] = ptx::max3(tops[q], __uint_as_float(v[c][x + 2 * q]), __uint_as_float(v[c][x + 2 * q + 1]));
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (logits != nullptr && e0 < a.logit_end) {
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int x = 0; x < 32; x += 4)
                                *reinterpret_cast<float4*>(logits + e0 + 32 * c + x) = make_float4(__uint_as_float(v[c][x]) * scale, __uint_as_float(v[c][x + 1]) * scale,
                                                                                                  __uint_as_float(v[c][x + 2]) * scale, __uint_as_float(v[c][x + 3]) * scale);
                    }
                    const bool move = real && (ref == neg ? top > neg : (top - ref) * scale > kPrefillLazy);
                    if (__any_sync(0xFFFFFFFFu, move)) {
                        float by = 1.f;
                        if (move) {
                            if (ref != neg) by = ptx::ex2((ref - top) * scale);
                            ref = top;
                            l *= by;
                        }
                        if (any) {
                            // (scores of this step came after the outputs of two steps before: the wait cannot take an earlier turn of the barrier for this one)
                            wait(o_full + 8 * (2 * t + ((at - 1) & 1)), (at - 1) >> 1, 2, int(tile));
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
                        }
                    }
                    // Differences are taken before they are scaled: at the maximum 0, however large it is.
                    const float sub = ref == neg ? 0.f : -ref;
                    const uint64_t sub2 = ptx::pack_f32x2(sub, sub), scale2 = ptx::pack_f32x2(scale, scale), up2 = ptx::pack_f32x2(kUp, kUp);
                    uint64_t s0 = ptx::pack_f32x2(0.f, 0.f), s1 = s0;                         // (the step's own sum: the row's is rounded once for its 64 entries)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t pk[16];
#pragma unroll
                        for (int x = 0; x < 32; x += 2) {
                            float x0, x1;
                            ptx::unpack_f32x2(ptx::fma_f32x2(ptx::add_f32x2(ptx::pack_f32x2(__uint_as_float(v[c][x]), __uint_as_float(v[c][x + 1])), sub2), scale2, up2), x0, x1);
                            x0 = ptx::ex2(x0);
                            x1 = ptx::ex2(x1);
                            if (x & 2) s1 = ptx::add_f32x2(s1, ptx::pack_f32x2(x0, x1));
                            else s0 = ptx::add_f32x2(s0, ptx::pack_f32x2(x0, x1));
                            pk[x / 2] = C::BF16 ? ptx::pack_bf16x2(x0, x1) : ptx::pack_f16x2(x0, x1);
                        }
                        tmem_st16(s_at + 16 * c, pk);
                    }
                    float a0, a1;
                    ptx::unpack_f32x2(ptx::add_f32x2(s0, s1), a0, a1);
                    l += a0 + a1;
                    ptx::tmem_wait_st();
                }
                // (a warp of rows that are none leaves whatever stands there: those rows of O are not read)
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(p_full + 8 * buffer);
                any = true;
                last = at;
            }
            if (!ok) break;
            // ── the stream's part of the row ──
            if (any) {
                wait(o_full + 8 * (2 * t + (last & 1)), last >> 1, 3, int(piece));
                if (!ok) break;
                ptx::tc_fence_after_sync();
            }
            ref = ref == neg ? neg : fmaf(ref, scale, -kUp);                  // (in log2 units from here on, as the weights were taken)
            const bool complete = w.k0 == 0 && w.k1 == w.span.count, mine = complete && t == 0;
            // the block's places: two pieces that a cut runs through, and the second stream's part of a unit that none does
            const int64_t part = int64_t(blockIdx.x) * (2 * NT + 1) + (complete ? 2 * NT : (w.nth > 0) * NT + t);
            float* const at_part = a.part_o + (part * a.group_rows + r) * D;
            float l2 = 0.f, ref2 = neg;
            if (complete && NT > 1) {
                if (t == 0) {
                    wait(join_full, joined, 3, int(piece));
                    if (!ok) break;
                    if (real) {
                        const float lse = a.part_lse[part * a.group_rows + r];
                        if (lse != neg) {
                            ref2 = lse;
                            l2 = 1.f;
                        }
                    }
                } else if (joined > 0) {
                    wait(join_empty, joined - 1, 3, int(piece));
                    if (!ok) break;
                }
            }
            if (mine && warp_real) {
                // both streams' parts: the second one's is normalised
                const float top = fmaxf(ref, ref2), by = ref == neg ? (l == l ? 0.f : l) : ptx::ex2(ref - top), by2 = ref2 == neg ? 0.f : l2 * ptx::ex2(ref2 - top);
                const float sum = l * by + by2, v_scale = a.v_scale != nullptr ? ptx::ld(a.v_scale + w.h) : 1.f;
#pragma unroll 1
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    if (any) {
                        tmem_ld16(lane_base + C::ColO + t * D + 16 * c, o);
                        ptx::tmem_wait_ld();
                    }
                    if (real) {
#pragma unroll
                        for (int x = 0; x < 16; x += 4) {
                            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (any) v = make_float4(__uint_as_float(o[x]) * by, __uint_as_float(o[x + 1]) * by, __uint_as_float(o[x + 2]) * by, __uint_as_float(o[x + 3]) * by);
                            if (l2 != 0.f) {
                                const float4 u = *reinterpret_cast<const float4*>(at_part + 16 * c + x);
                                v.x = fmaf(u.x, by2, v.x);  v.y = fmaf(u.y, by2, v.y);  v.z = fmaf(u.z, by2, v.z);  v.w = fmaf(u.w, by2, v.w);
                            }
                            gqa_write_row<D>(a, w.req.row0 + token, w.h * a.G + row - token * a.G, (int64_t(w.b) * a.Hkv + w.h) * rows + row, 16 * c + x, v, top, sum, v_scale);
                        }
                    }
                }
            } else if (warp_real) {
                const float per = l == 0.f ? 0.f : 1.f / l;
                if (any) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tmem_ld16(lane_base + C::ColO + t * D + 16 * c, o);
                        ptx::tmem_wait_ld();
                        if (real) {
#pragma unroll
                            for (int x = 0; x < 16; x += 4)
                                *reinterpret_cast<float4*>(at_part + 16 * c + x) = l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                    : make_float4(__uint_as_float(o[x]) * per, __uint_as_float(o[x + 1]) * per, __uint_as_float(o[x + 2]) * per, __uint_as_float(o[x + 3]) * per);
                        }
                    }
                } else if (real) {
                    for (int x = 0; x < D; x += 4) *reinterpret_cast<float4*>(at_part + x) = make_float4(0.f, 0.f, 0.f, 0.f);
                }
                if (real) a.part_lse[part * a.group_rows + r] = l == 0.f ? neg : ref + log2f(l);
            }
            if (complete && NT > 1) {
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(t == 0 ? join_empty : join_full);
                ++joined;
            }
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

}  // namespace dsv4
