// Tree decode for many (node, head) rows per request: every group of 128 rows reads the same entries, so these are dequantised once, into FP16 rows
// in a workspace, and the attention kernel gets its operands from there by TMA, in the layout the MMAs want.
//
//   tree_unpack_kernel   entries of a request (cache, then window) -> FP16 [B, cap, 576] and a bit per entry that takes part
//   tree_mma_kernel      the pair scheme of decode_kernel.cuh (cta_group::2, M = 128: 64 rows, half of the entries and half of the value columns a
//                        block; S and O in tensor memory) without its resolve, fetch and dequantise warps; two buffers for K and V.
//
// What that changes per tile of 64 entries and SM: 69 KB by TMA from L2 instead of 30 KB of raw records, but no raw reads, conversions and
// operand stores, which kept the shared-memory port busy for 1130 of its 2000 cycles.  Bounds, in SM cycles: tensor pipe 1244 (as there), shared-memory port 540
// in + 860 out, L2 at the measured 16.4 TB/s (58 bytes a cycle and SM) 1190.  The direct kernel takes 2570.  512 groups of 15 tiles take 2000 with their
// set-up and output, and the tensor pipe is at work for 68 % of the kernel's cycles; from some 500 groups on the power limit holds the clock at
// 1.5 GHz: 1,024 groups take 265 to 269 us for the first calls after a pause and 308 under load, 0.86 PFLOP/s (a library product: 1.39, at 1.32 GHz).
//
// Rounding: an entry is e4m3 x scale in FP16, in the same operations as in the direct kernel (the scale is rounded, then the product: up to 2^-10 of an element);
// results differ from it in nothing but the order of sums.  At its 128 registers the attention kernel spills 44 bytes, the unpacking 4 at 64.
#pragma once

#include "decode_kernel.cuh"

namespace dsv4 {

constexpr int kUnpackThreads = 512;
constexpr int kUnpackEach = 8;                 // entries of a warp

struct TreeUnpackArgs {
    int B, T, max_pages, win_cap, mask_words, cap;
    int64_t num_pages;
    const uint8_t* kv_pool;
    const uint8_t* win_pool;
    const int32_t* block_table;
    const int32_t* kv_len;
    const int32_t* win_len;
    const int32_t* tree_mask;
    uint8_t* rows;             // FP16 [B, cap, 576]
    uint32_t* valid;           // [B, cap / 32]
    int32_t* status;
};

// A warp takes eight entries at a time and has all of their bytes on the way at once; a lane has 16 latent bytes of each and their block's scale, and a piece
// of two of the RoPE tails.  Rows that take no part (out of range, or window rows that no node sees) are zero: whatever probability they get is zero too,
// and zero times what the memory held might not be.  Bound by the chain
// of its loads (lengths and page, record) and by memory, 656 bytes read and 1152 written an entry: 51,000 entries in 20 us, 23 with four entries a warp and
// blocks that met for the bits of a tile.
__global__ void __launch_bounds__(kUnpackThreads, 2) tree_unpack_kernel(const __grid_constant__ TreeUnpackArgs a) {
    constexpr int kEach = kUnpackEach, kParts = kTileN / kEach;
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int lane = threadIdx.x & 31, tiles = a.cap / kTileN, units = a.B * tiles * kParts;
    for (int u = (blockIdx.x * kUnpackThreads + threadIdx.x) >> 5; u < units; u += gridDim.x * (kUnpackThreads / 32)) {
        const int b = u / (tiles * kParts), v0 = (u - b * tiles * kParts) * kEach;
        // where the warp's entries live (lane i: entry i)
        const int v = v0 + (lane & (kEach - 1)), slot = v >> 6, page = slot < a.max_pages ? ptx::ld(a.block_table + int64_t(b) * a.max_pages + slot) : -1;
        const int kv_len = max(ptx::ld(a.kv_len + b), 0), win_len = max(ptx::ld(a.win_len + b), 0);
        const int64_t n_tok = int64_t(kv_len) + win_len;
        if (v0 == 0 && n_tok > a.cap && lane == 0) report_status(a.status, kStatusBadIndex, 4, kv_len);
        if (v0 / kTileN * kTileN >= n_tok) continue;
        const uint8_t* rec = nullptr;
        if (v < n_tok) {
            if (v < kv_len) {
                if (page >= 0 && page < a.num_pages) rec = a.kv_pool + (int64_t(page) * 64 + (v & 63)) * 656;
                else if (lane < kEach) report_status(a.status, kStatusBadIndex, 4, slot < a.max_pages ? page : v);
            } else if (v - kv_len < a.win_cap) {
                rec = a.win_pool + (int64_t(b) * a.win_cap + (v - kv_len)) * 656;
            } else if (lane < kEach) {
                report_status(a.status, kStatusBadIndex, 4, v);
            }
        }
        if (v0 + kEach > kv_len) {
            // (window rows among them) the rows that any node sees: their bits lie in two words at most
            const int w0 = max(v0 - kv_len, 0) >> 5;
            uint32_t any0 = 0u, any1 = 0u;
            for (int t = lane; t < a.T; t += 32) {
                const int32_t* words = a.tree_mask + (int64_t(b) * a.T + t) * a.mask_words;
                if (w0 < a.mask_words) any0 |= uint32_t(ptx::ld(words + w0));
                if (w0 + 1 < a.mask_words) any1 |= uint32_t(ptx::ld(words + w0 + 1));
            }
            any0 = __reduce_or_sync(0xFFFFFFFFu, any0);
            any1 = __reduce_or_sync(0xFFFFFFFFu, any1);
            const int w = v - kv_len;
            if (w >= 0 && !(((w >> 5) == w0 ? any0 : any1) >> (w & 31) & 1u)) rec = nullptr;
        }
        const uint32_t valid = __ballot_sync(0xFFFFFFFFu, rec != nullptr);
        const unsigned long long rec_bits = reinterpret_cast<unsigned long long>(rec);
        uint4 x[kEach], rope[kEach / 4];
        float scale[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint8_t* p = reinterpret_cast<const uint8_t*>(__shfl_sync(0xFFFFFFFFu, rec_bits, i));
            x[i] = make_uint4(0, 0, 0, 0);
            scale[i] = 0.f;
            if (p != nullptr) {
                x[i] = ptx::ldg_stream_v4(p + lane * 16);
                scale[i] = ptx::ld(reinterpret_cast<const float*>(p + 512) + (lane >> 3));
            }
        }
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
            const uint8_t* p = reinterpret_cast<const uint8_t*>(__shfl_sync(0xFFFFFFFFu, rec_bits, 4 * i + (lane >> 3)));
            rope[i] = make_uint4(0, 0, 0, 0);
            if (p != nullptr) rope[i] = ptx::ldg_stream_v4(p + 528 + (lane & 7) * 16);
        }
        uint8_t* const row = a.rows + (int64_t(b) * a.cap + v0) * 1152;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const __half2 scale2 = __float2half2_rn(fminf(scale[i], 146.f));
            uint4 lo, hi;
            dequant4_f16(x[i].x, scale2, lo.x, lo.y);
            dequant4_f16(x[i].y, scale2, lo.z, lo.w);
            dequant4_f16(x[i].z, scale2, hi.x, hi.y);
            dequant4_f16(x[i].w, scale2, hi.z, hi.w);
            ptx::stg_v8(row + i * 1152 + lane * 32, lo, hi);
        }
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) *reinterpret_cast<uint4*>(row + (4 * i + (lane >> 3)) * 1152 + 1024 + (lane & 7) * 16) = bf16x8_to_f16x8(rope[i]);
        if (lane == 0) reinterpret_cast<uint8_t*>(a.valid)[(int64_t(b) * a.cap + v0) / 8] = uint8_t(valid);
    }
}

// Warp roles of the attention kernel.
constexpr int kTreeQWarps = 8;                 // warps 4-11: Q into tensor memory, BF16 to FP16; and the output
constexpr int kTreeFirstQWarp = 4;
constexpr int kTreeSWarp = 12;                 // tensor-memory allocation; (even block) issue of the S MMAs
constexpr int kTreeOWarp = 13;                 // (even block) issue of the O MMAs
constexpr int kTreeKWarp = 14;                 // K tiles
constexpr int kTreeVWarp = 15;                 // V tiles, and Q (with K and V in one warp, K waited behind V: 1650 cycles a tile)
constexpr int kTreeThreads = 16 * 32;

struct TreeArgs {
    alignas(64) CUtensorMap q_map;             // BF16 [B * H, 576], box 64 x 64
    alignas(64) CUtensorMap k_map;             // FP16 [B * cap, 576], box 64 columns x 32 rows
    alignas(64) CUtensorMap v_map;             // the same, 64 columns x 64 rows
    alignas(64) CUtensorMap out_map;           // BF16 [B, H, 512], box 64 columns x 32 rows
    alignas(64) CUtensorMap part_map;          // FP16 partials: [slots, 128, 512] with a plan, else [num_splits * B, H, 512]
    int B, H, heads;                           // H: (node, head) rows of a request
    int cap;                                   // rows per request in the workspace, a multiple of 64
    int mask_words;
    int num_splits;
    float scale_log2;
    const uint32_t* valid;
    const int32_t* kv_len;
    const int32_t* win_len;
    const int32_t* tree_mask;
    const float* attn_sink;
    __nv_bfloat16* out;
    float* lse;
    float* partial_o;
    float* partial_lse;
    int32_t* status;
    const int32_t* sched_pair_begin;
    const int32_t* sched_items;
    uint32_t wait_ns;
    int dbg_drop_tile;
    bool dealt;                                // without a plan, resident pairs share out the row groups
};
constexpr int kTreeDealt = 256;                // requests at most of which that is done

struct TreeSmem {
    static constexpr int kQBytes = 3 * kQChunkBytes;            // chunks 6-8 stay here
    static constexpr int kStageBytes = 6 * kQChunkBytes;        // chunks 0-5 on their way to tensor memory, then 6-8
    static constexpr int kKBytes = 9 * kKChunkBytes;
    static constexpr int kVBytes = 4 * kVChunkBytes;
    static constexpr int kQOff = 0;
    static constexpr int kStageOff = kQOff + kQBytes;
    static constexpr int kKOff = kStageOff + kStageBytes;
    static constexpr int kVOff = kKOff + 2 * kKBytes;
    static constexpr int kPOff = kVOff + 2 * kVBytes;
    static constexpr int kMiscOff = kPOff + 2 * kQChunkBytes;
    static constexpr int kTotal = kMiscOff + 3072;
    static_assert(kTotal <= 232448, "shared memory of a block");
    static_assert(kKOff % 1024 == 0 && kVOff % 1024 == 0 && kPOff % 1024 == 0, "swizzled operands");
};

struct TreeMisc {
    float exch[2 * kHeadsPerBlock];
    float inv[2][kHeadsPerBlock];    // per item, in turn: what the rows' outputs are multiplied by
    uint64_t bar_tmem;
    uint64_t bar_q_full[2];          // per item: chunks 0-5 / 6-8 of Q landed in the staging area
    uint64_t bar_q_read;             // per item: chunks 0-5 have been read there by every Q warp
    uint64_t bar_q_placed;           // per item: 6-8 have been copied to their place by every Q warp
    uint64_t bar_stage_free;         // per item: 6-8 have been, and the output of the item before has left it
    uint64_t bar_inv[2];             // per item, in turn: inv written (the softmax warps may finish the next item before the last Q warp comes to this)
    // signalled in both blocks by the commits of the MMA warps
    uint64_t bar_q_free;             // per item: its S MMAs complete
    uint64_t bar_o_last;             // per item: its P.V complete
    uint64_t bar_s_full[2];          // S of a tile complete: S buffer full, K buffer free
    uint64_t bar_o_full[2];          // P.V of a tile complete: V and P buffer free, O up to date
    // in the even block only, signalled by the warps of both
    uint64_t bar_q_ready;
    uint64_t bar_o_read;             // per item: its O has been read
    uint64_t bar_k_full[2], bar_v_full[2];                // both blocks' halves of a tile landed (TMA transaction count, by the copies themselves)
    uint64_t bar_p_full[2];
    uint32_t tmem_base;
    uint8_t order[kTreeDealt];       // requests by length, the longest first
    int len[kTreeDealt];
};
static_assert(sizeof(TreeMisc) <= 3072 - 16, "the last word of the block's shared memory is failed_flag()");

// The window rows [o, o + 32) that a node sees; rows below 0 are entries of the cache, which every node sees.
__device__ __forceinline__ uint32_t window_bits(const int32_t* mask, int words, int o) {
    if (o <= -32) return ~0u;
    const int first = max(o, 0), w = first >> 5;
    const uint32_t lo = w < words ? uint32_t(ptx::ld(mask + w)) : 0u, hi = w + 1 < words ? uint32_t(ptx::ld(mask + w + 1)) : 0u;
    const uint32_t m = __funnelshift_r(lo, hi, first & 31);
    return o < 0 ? (m << -o) | ((1u << -o) - 1u) : m;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTreeThreads, 1) tree_mma_kernel(const __grid_constant__ TreeArgs a) {
    using L = TreeSmem;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t smem_base = ptx::smem_u32(smem_raw);
    if (smem_base & 1023u) {                      // the operand layout needs it; the same answer in every block
        report_status(a.status, kStatusWaitQ, 5, -1);
        return;
    }
    const uint32_t q_base = smem_base + L::kQOff, q_stage = smem_base + L::kStageOff, k_base = smem_base + L::kKOff, v_base = smem_base + L::kVOff,
                   p_base = smem_base + L::kPOff;
    TreeMisc* misc = reinterpret_cast<TreeMisc*>(smem_raw + L::kMiscOff);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = int(blockIdx.x & 1u);
    const bool sched = a.sched_pair_begin != nullptr;
    const uint32_t wait_ns = a.wait_ns;

    int item_begin = 0, n_items = 1;
    const int hgs = (a.H + kHeadsPerCta - 1) / kHeadsPerCta, pairs = int(gridDim.x >> 1), my_pair = int(blockIdx.x >> 1);
    auto get_item = [&](int k) -> Item {
        Item it;
        if (sched) {
            const int4* rec = reinterpret_cast<const int4*>(a.sched_items + int64_t(item_begin + k) * kItemWords);
            const int4 r0 = ptx::ld(rec), r1 = ptx::ld(rec + 1);
            it.n = r0.x;  it.hg = r0.y;  it.tile0 = r0.z;  it.ntiles = r0.w;
            it.slot = r1.x;  it.n_tok = r1.y;  it.kv_len_n = r1.z;
            // (lengths beyond the workspace have been reported: what lies there is left out)
            it.n_tok = min(it.n_tok, a.cap);
            it.ntiles = min(it.ntiles, max(a.cap / kTileN - it.tile0, 0));
        } else {
            it.n = blockIdx.y;  it.hg = my_pair;
            if (a.dealt) {
                const int at = k * pairs + ((k & 1) ? pairs - 1 - my_pair : my_pair);
                it.n = misc->order[at / hgs];  it.hg = at % hgs;
            }
            it.kv_len_n = max(ptx::ld(a.kv_len + it.n), 0);
            it.n_tok = int(min(int64_t(it.kv_len_n) + max(ptx::ld(a.win_len + it.n), 0), int64_t(a.cap)));
            const int split = blockIdx.z;
            const int tiles_total = (it.n_tok + kTileN - 1) / kTileN;
            const int tiles_per_split = (tiles_total + a.num_splits - 1) / a.num_splits;
            it.tile0 = min(split * tiles_per_split, tiles_total);
            it.ntiles = min(it.tile0 + tiles_per_split, tiles_total) - it.tile0;
            it.slot = a.num_splits > 1 ? split : -1;
        }
        return it;
    };

    const uint32_t bar_tmem = ptx::smem_u32(&misc->bar_tmem), bar_q_full = ptx::smem_u32(&misc->bar_q_full[0]), bar_q_read = ptx::smem_u32(&misc->bar_q_read), bar_stage_free = ptx::smem_u32(&misc->bar_stage_free), bar_q_placed = ptx::smem_u32(&misc->bar_q_placed),
                   bar_q_free = ptx::smem_u32(&misc->bar_q_free), bar_o_last = ptx::smem_u32(&misc->bar_o_last), bar_inv = ptx::smem_u32(&misc->bar_inv[0]),
                   bar_o_read = ptx::smem_u32(&misc->bar_o_read),
                   bar_s_full = ptx::smem_u32(&misc->bar_s_full[0]), bar_o_full = ptx::smem_u32(&misc->bar_o_full[0]), bar_q_ready = ptx::smem_u32(&misc->bar_q_ready),
                   bar_k_full = ptx::smem_u32(&misc->bar_k_full[0]), bar_v_full = ptx::smem_u32(&misc->bar_v_full[0]), bar_p_full = ptx::smem_u32(&misc->bar_p_full[0]);
    auto arrive_even = [&](uint32_t bar) {
        if (rank == 0) ptx::mbar_arrive(bar);
        else ptx::mbar_arrive_remote(ptx::mapa(bar, 0));
    };

    // ── set-up ──
    if (warp == kTreeVWarp && lane == 0) { ptx::prefetch_tensormap(&a.out_map);  ptx::prefetch_tensormap(&a.q_map);  ptx::prefetch_tensormap(&a.k_map);  ptx::prefetch_tensormap(&a.v_map); }
    if (tid == 0) {
        ptx::sts_u32(failed_flag(), 0u);
        ptx::mbar_init(bar_tmem, 1);
        ptx::mbar_init(bar_q_read, kTreeQWarps);
        ptx::mbar_init(bar_stage_free, kTreeQWarps);
        ptx::mbar_init(bar_q_placed, kTreeQWarps);
        ptx::mbar_init(bar_q_free, 1);
        ptx::mbar_init(bar_o_last, 1);
        ptx::mbar_init(bar_inv, kNumSoftmaxWarps);
        ptx::mbar_init(bar_inv + 8, kNumSoftmaxWarps);
        ptx::mbar_init(bar_o_read, 2 * kTreeQWarps);
        ptx::mbar_init(bar_q_ready, 2 * kTreeQWarps);
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(bar_q_full + 8 * i, 1);
            ptx::mbar_init(bar_s_full + 8 * i, 1);
            ptx::mbar_init(bar_o_full + 8 * i, 1);
            ptx::mbar_init(bar_k_full + 8 * i, 1);
            ptx::mbar_init(bar_v_full + 8 * i, 1);
            ptx::mbar_init(bar_p_full + 8 * i, 2 * kNumSoftmaxWarps);
        }
        ptx::fence_mbar_init();
    }
    __syncwarp();
    ptx::cluster_sync();
    ptx::pdl_wait();
    if (sched) {
        const int pair = blockIdx.x >> 1;
        item_begin = ptx::ld(a.sched_pair_begin + pair);
        n_items = ptx::ld(a.sched_pair_begin + pair + 1) - item_begin;
    } else if (a.dealt) {
        // The groups of the longest request come first, and every other round of them goes round backwards: nobody begins a long one last (92 ragged groups
        // in the order of the batch 83 us, so 71; 128 groups of 12,800 entries on average 440 and 390), and a pair's next Q and last output are under way during its tiles as they are with a plan.
        if (tid < a.B) misc->len[tid] = int(min(int64_t(max(ptx::ld(a.kv_len + tid), 0)) + max(ptx::ld(a.win_len + tid), 0), int64_t(a.cap)));
        __syncthreads();
        if (tid < a.B) {
            const int mine = misc->len[tid];
            int before = 0;
#pragma unroll 4
            for (int i = 0; i < a.B; ++i) before += misc->len[i] > mine || (misc->len[i] == mine && i < tid);
            misc->order[before] = uint8_t(tid);
        }
        __syncthreads();
        const int groups = a.B * hgs, rounds = groups / pairs, left = groups - rounds * pairs;      // (the last round may be a part of one)
        n_items = rounds + (((rounds & 1) ? pairs - 1 - my_pair : my_pair) < left ? 1 : 0);
    }
    constexpr uint32_t tmem = 0;                  // all 512 columns are allocated (checked)
    auto wait_tmem = [&]() -> bool {
        const bool w = ptx::mbar_wait_warp(bar_tmem, 0u, wait_ns);
        ptx::tc_fence_after_sync();
        return w;
    };
    auto wait_for = [&](uint32_t bar, uint32_t phase, int code, int role, int at) -> bool {
        const bool w = ptx::mbar_wait_warp(bar, phase & 1u, wait_ns);
        if (!w) wait_ran_out(a.status, code, role, at);
        return w;
    };

    // Running counters, as in decode_kernel.cuh: `g` the tiles over all items, `qn` the items that had tiles.  Tile g is the (g / 2)-th use of K, V, S and P
    // buffer g % 2.  Every waiter goes through a barrier's phases one by one.
    if (warp >= kTreeFirstQWarp && warp < kTreeSWarp) {
        // ───────────── Q warps: Q of the next item, then the output of this one ─────────────
        // Between two items the tensor pipe waits for Q (into tensor memory, and its last chunks) and for O to be read:
        // by eight warps that have nothing else to do then, while the softmax warps are at the next item's first tiles.  (With the output written by the softmax
        // warps, through shared memory, an item of 15 tiles cost five tiles more.)
        const int qw = warp - kTreeFirstQWarp;
        bool ok = wait_tmem();
        if (!ok) wait_ran_out(a.status, kStatusWaitQ, 2, -1);
        uint32_t qn = 0;
        Item last{};                                   // the item whose output is to be written
        auto write_out = [&]() -> bool {
            // 32 rows of this block, value columns [256 half + 128 (qw / 4), +128): 64 columns at a time through this warp's 4 KB of the staging area, and from there
            // by TMA, which leaves the rows past the last one out.  (Stored from registers, 32 bytes a row and lane, they kept the load/store unit busy
            // for 3,000 cycles, in which the MMAs did not get at their operands: 1,950 cycles a tile over items of 15, now 1,790.)
            const int row0 = rank * kHeadsPerBlock + (qw & 1) * 32, half = (qw >> 1) & 1, r = (qw & 1) * 32 + lane;
            const bool final_out = last.slot < 0;
            if (!wait_for(bar_inv + 8 * ((qn - 1u) & 1u), (qn - 1u) >> 1, kStatusWaitOFull, 2, 0) || !wait_for(bar_o_last, qn - 1u, kStatusWaitOFull, 2, 0)) return false;
            ptx::tc_fence_after_sync();
            const float inv = misc->inv[(qn - 1u) & 1u][r];
            const uint32_t from = tmem + (uint32_t((qw & 3) * 32) << 16) + kTmemO + 128u * uint32_t(qw >> 2);
            const uint32_t box = q_stage + uint32_t(qw) * 4096u, line = box + uint32_t(lane) * 128u, sw = uint32_t(lane & 7) << 4;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                ptx::tmem_ld32(from + 32u * uint32_t(c), o);
                ptx::tmem_wait_ld();
                if (c == 3) {
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) arrive_even(bar_o_read);
                }
                if (c == 2) {                          // the first half has left
                    if (lane == 0) ptx::tma_stores_read();
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x = __uint_as_float(o[8 * i + 2 * j]) * inv, y = __uint_as_float(o[8 * i + 2 * j + 1]) * inv;
                        w[j] = final_out ? ptx::pack_bf16x2(x, y) : ptx::pack_f16x2(x, y);
                    }
                    ptx::sts_v4(line + ((uint32_t(4 * (c & 1) + i) << 4) ^ sw), make_uint4(w[0], w[1], w[2], w[3]));
                }
                if (c & 1) {
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        const int x = 256 * half + 128 * (qw >> 2) + 32 * (c - 1);
                        if (final_out) ptx::tma_store_3d(&a.out_map, x, last.hg * kHeadsPerCta + row0, last.n, box);
                        else if (sched) ptx::tma_store_3d(&a.part_map, x, row0, last.slot, box);
                        else ptx::tma_store_3d(&a.part_map, x, last.hg * kHeadsPerCta + row0, last.slot * a.B + last.n, box);
                    }
                    __syncwarp();
                }
            }
            if (lane == 0) ptx::tma_stores_read();
            __syncwarp();
            return true;
        };
#pragma unroll 1
        for (int k = 0; k < n_items && ok; ++k) {
            const Item it = get_item(k);
            if (it.ntiles <= 0) continue;
            // Chunks 0-5 wait for their place in tensor memory in registers (96 a thread: half of a row's columns, as FP16), so that the others can come to
            // the staging area meanwhile.
            if (!wait_for(bar_q_full, qn, kStatusWaitQ, 2, k)) { ok = false;  break; }
            uint32_t x[2][48];
            const int half = qw >> 2;
            const uint32_t q_rows = q_stage + uint32_t((qw & 1) * 32 + lane) * 128u, sw = uint32_t(lane & 7) << 4;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 12; ++i) {
                    const uint32_t u = uint32_t(half * 12 + i);
                    const uint4 v = bf16x8_to_f16x8(ptx::lds_v4(q_rows + (3u * j + (u >> 3)) * kQChunkBytes + (((u & 7u) << 4) ^ sw)));
                    x[j][4 * i] = v.x;  x[j][4 * i + 1] = v.y;  x[j][4 * i + 2] = v.z;  x[j][4 * i + 3] = v.w;
                }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar_q_read);
            if (!wait_for(bar_q_full + 8, qn, kStatusWaitQ, 2, k) || (qn > 0u && !wait_for(bar_q_free, qn - 1u, kStatusWaitSFull, 2, k))) { ok = false;  break; }
            ptx::tc_fence_after_sync();
            const uint32_t q_tmem = tmem + (uint32_t((qw & 3) * 32) << 16) + kTmemQ + 48u * uint32_t(half);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                ptx::tmem_st32(q_tmem + 96u * j, reinterpret_cast<const uint32_t(&)[32]>(x[j][0]));
                ptx::tmem_st8(q_tmem + 96u * j + 32u, make_uint4(x[j][32], x[j][33], x[j][34], x[j][35]), make_uint4(x[j][36], x[j][37], x[j][38], x[j][39]));
                ptx::tmem_st8(q_tmem + 96u * j + 40u, make_uint4(x[j][40], x[j][41], x[j][42], x[j][43]), make_uint4(x[j][44], x[j][45], x[j][46], x[j][47]));
            }
            constexpr int kVecs = L::kQBytes / 16 / (kTreeQWarps * 32);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const uint32_t at = uint32_t((i * kTreeQWarps + qw) * 32 + lane) * 16u;
                ptx::sts_v4(q_base + at, bf16x8_to_f16x8(ptx::lds_v4(q_stage + at)));
            }
            ptx::tmem_wait_st();
            ptx::tc_fence_before_sync();
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                arrive_even(bar_q_ready);
                ptx::mbar_arrive(bar_q_placed);
            }
            // (the output goes through the staging area, which the other Q warps may still be reading)
            if (qn > 0u && (!wait_for(bar_q_placed, qn, kStatusWaitQ, 2, k) || !write_out())) { ok = false;  break; }
            if (lane == 0) ptx::mbar_arrive(bar_stage_free);
            last = it;
            ++qn;
        }
        if (ok && qn > 0u) write_out();
        if (lane == 0) ptx::tma_stores_done();
        __syncwarp();
    } else if (warp == kTreeKWarp) {
        // ───────────── K tiles: both blocks' copies report to the even one, which expects the bytes of both ─────────────
        const uint32_t k_full = ptx::mapa(bar_k_full, 0);
        bool ok = true;
        uint32_t g = 0;
#pragma unroll 1
        for (int k = 0; k < n_items && ok; ++k) {
            const Item it = get_item(k);
#pragma unroll 1
            for (int i = 0; i < it.ntiles; ++i, ++g) {
                const uint32_t buf = g & 1u;
                const int row = it.n * a.cap + (it.tile0 + i) * kTileN + rank * kRowsPerBlock;
                if (g >= 2u && !wait_for(bar_s_full + 8 * buf, (g - 2u) >> 1, kStatusWaitKvFree, 4, int(g))) { ok = false;  break; }
                if (ptx::elect_one()) {
                    if (rank == 0 && !(a.dbg_drop_tile >= 0 && g == uint32_t(a.dbg_drop_tile))) ptx::mbar_arrive_expect_tx(bar_k_full + 8 * buf, 2 * L::kKBytes);
#pragma unroll
                    for (int c = 0; c < 9; ++c) ptx::tma_load_2d_pair(k_base + buf * L::kKBytes + c * kKChunkBytes, &a.k_map, c * 64, row, k_full + 8 * buf);
                }
                __syncwarp();
            }
        }
        __syncwarp();
    } else if (warp == kTreeVWarp) {
        // ───────────── V tiles; Q of the next item while this one is at work ─────────────
        const uint32_t v_full = ptx::mapa(bar_v_full, 0);
        bool ok = true;
        uint32_t g = 0, qn = 0;
        auto q_row = [&](const Item& it) { return it.n * a.H + it.hg * kHeadsPerCta + rank * kHeadsPerBlock; };
        // chunks 0-5, and when these have been read the others, to the staging area
        auto send_q = [&](const Item& it, int part) {
            if (ptx::elect_one()) {
                ptx::mbar_arrive_expect_tx(bar_q_full + 8 * part, part ? L::kQBytes : L::kStageBytes);
#pragma unroll
                for (int c = 0; c < 6; ++c)
                    if (part == 0 || c < 3) ptx::tma_load_2d(q_stage + c * kQChunkBytes, &a.q_map, (6 * part + c) * 64, q_row(it), bar_q_full + 8 * part);
            }
            __syncwarp();
        };
        auto next_item = [&](int& k) -> Item {         // the next one with tiles
            Item it{};
            while (++k < n_items) {
                it = get_item(k);
                if (it.ntiles > 0) break;
            }
            return it;
        };
        int k = -1;
        Item it = next_item(k);
        if (k < n_items) {
            send_q(it, 0);
            if (wait_for(bar_q_read, 0u, kStatusWaitQ, 5, 0)) send_q(it, 1);
            else ok = false;
        }
#pragma unroll 1
        while (k < n_items && ok) {
            int k2 = k;
            const Item next = next_item(k2);
#pragma unroll 1
            for (int i = 0; i < it.ntiles; ++i, ++g) {
                const uint32_t buf = g & 1u;
                const int row = it.n * a.cap + (it.tile0 + i) * kTileN;
                if (g >= 2u && !wait_for(bar_o_full + 8 * buf, (g - 2u) >> 1, kStatusWaitKvFree, 4, int(g))) { ok = false;  break; }
                if (ptx::elect_one()) {
                    if (rank == 0) ptx::mbar_arrive_expect_tx(bar_v_full + 8 * buf, 2 * L::kVBytes);
#pragma unroll
                    for (int c = 0; c < 4; ++c) ptx::tma_load_2d_pair(v_base + buf * L::kVBytes + c * kVChunkBytes, &a.v_map, rank * 256 + c * 64, row, v_full + 8 * buf);
                }
                __syncwarp();
                // (by the fifth tile this item's Q is in place, and the output of the one before has left the staging area)
                if (i == min(it.ntiles - 1, 4) && k2 < n_items) {
                    if (!wait_for(bar_stage_free, qn, kStatusWaitQ, 5, k)) { ok = false;  break; }
                    send_q(next, 0);
                }
                if (i == min(it.ntiles - 1, 7) && k2 < n_items) {
                    if (!wait_for(bar_q_read, qn + 1u, kStatusWaitQ, 5, k)) { ok = false;  break; }
                    send_q(next, 1);
                }
            }
            k = k2;
            it = next;
            ++qn;
        }
        __syncwarp();
    } else if (warp == kTreeSWarp) {
        // ───────────── tensor-memory allocation, S = Q . K^T ─────────────
        ptx::tmem2_alloc(ptx::smem_u32(&misc->tmem_base), kTmemCols);
        ptx::tmem2_relinquish();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0 && *reinterpret_cast<volatile uint32_t*>(&misc->tmem_base) == tmem) ptx::mbar_arrive(bar_tmem);
        bool ok = wait_tmem();
        if (rank == 0) {
            constexpr uint32_t kDescHi = ptx::smem_desc_hi(1024), idesc = ptx::make_idesc_f16(128, kTileN, false, false);
            const uint32_t q_lo = ptx::smem_desc_lo(q_base, 16), k_lo0 = ptx::smem_desc_lo(k_base, 16);
            uint32_t g = 0, qn = 0;
#pragma unroll 1
            for (int k = 0; k < n_items && ok; ++k) {
                const int ntiles = get_item(k).ntiles;
                if (ntiles <= 0) continue;
                if (!wait_for(bar_q_ready, qn, kStatusWaitQ, 1, int(g))) break;
#pragma unroll 1
                for (int i = 0; i < ntiles; ++i, ++g) {
                    const uint32_t buf = g & 1u;
                    // the S buffer has been read by the softmax of the tile two before
                    if ((g >= 2u && !wait_for(bar_p_full + 8 * buf, (g - 2u) >> 1, kStatusWaitPFull, 1, int(g))) ||
                        !wait_for(bar_k_full + 8 * buf, g >> 1, kStatusWaitKvFull, 1, int(g))) { ok = false;  break; }
                    ptx::tc_fence_after_sync();
                    const uint32_t d = tmem + kTmemS + buf * 32u, k_lo = k_lo0 + buf * uint32_t(L::kKBytes >> 4);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int c = 0; c < 9; ++c)
#pragma unroll
                            for (int s = 0; s < 4; ++s) {
                                const uint32_t b_lo = k_lo + uint32_t((c * kKChunkBytes + s * 32) >> 4);
                                if (c < kQTmemChunks) ptx::mma2_ts(d, tmem + kTmemQ + c * 32 + s * 8, b_lo, kDescHi, idesc, (c | s) ? 1u : 0u);
                                else ptx::mma2_ss(d, q_lo + uint32_t(((c - kQTmemChunks) * kQChunkBytes + s * 32) >> 4), b_lo, kDescHi, idesc, 1u);
                            }
                        ptx::mma2_commit(bar_s_full + 8 * buf);
                        if (i + 1 == ntiles) ptx::mma2_commit(bar_q_free);
                    }
                    __syncwarp();
                }
                ++qn;
            }
        }
        __syncwarp();
    } else if (warp == kTreeOWarp) {
        // ───────────── O += P . V ─────────────
        if (rank == 0) {
            constexpr uint32_t kDescHi = ptx::smem_desc_hi(1024), idesc = ptx::make_idesc_f16(128, 256, false, true);
            bool ok = wait_tmem();
            const uint32_t p_lo0 = ptx::smem_desc_lo(p_base, 16), v_lo0 = ptx::smem_desc_lo(v_base, kVChunkBytes);
            uint32_t g = 0, qn = 0;
#pragma unroll 1
            for (int k = 0; k < n_items && ok; ++k) {
                const Item it = get_item(k);
                if (it.ntiles <= 0) continue;
                // O of the item before has been read
                if (qn > 0u && !wait_for(bar_o_read, qn - 1u, kStatusWaitOFull, 3, int(g))) break;
                ++qn;
#pragma unroll 1
                for (int i = 0; i < it.ntiles; ++i, ++g) {
                    const uint32_t buf = g & 1u;
                    const int ksteps = (it.tile_entries(i) + 15) >> 4;
                    if (!wait_for(bar_p_full + 8 * buf, g >> 1, kStatusWaitPFull, 3, int(g)) || !wait_for(bar_v_full + 8 * buf, g >> 1, kStatusWaitKvFull, 3, int(g))) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint32_t p_lo = p_lo0 + buf * uint32_t(kQChunkBytes >> 4), v_lo = v_lo0 + buf * uint32_t(L::kVBytes >> 4);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                            for (int s = 0; s < 4; ++s)
                                if (s < ksteps)
                                    ptx::mma2_ss(tmem + kTmemO + jj * 128, p_lo + uint32_t((s * 32) >> 4), v_lo + uint32_t((2 * jj * kVChunkBytes + s * 16 * 128) >> 4), kDescHi,
                                                 idesc, (i > 0 || s > 0) ? 1u : 0u);
                        ptx::mma2_commit(bar_o_full + 8 * buf);
                        if (i + 1 == it.ntiles) ptx::mma2_commit(bar_o_last);
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
    } else {
        // ───────────── softmax warps: as in decode_kernel.cuh, but for the output ─────────────
        // Thread tid owns row tid % 64 of this block and, of its S row, the entries 32 (tid / 64) .. +31 of the tile.
        const int r = tid & 63, colhalf = tid >> 6;
        const uint32_t lane_addr = uint32_t(warp * 32) << 16;
        const uint32_t pair_bar = 1u + uint32_t(warp & 1);
        bool ok = wait_tmem();
        if (!ok) wait_ran_out(a.status, kStatusWaitQ, 0, -1);
        ok = !ptx::bar_any(pair_bar, 64, !ok);
        const uint32_t p_row = p_base + uint32_t(r) * 128u;
        const uint32_t p_sw = (uint32_t(4 * colhalf) ^ uint32_t(r & 7)) << 4;
        uint32_t gt = 0, qn = 0;
        Item cur = get_item(0);
#pragma unroll 1
        for (int k = 0; k < n_items && ok; ++k) {
            const int nb = cur.ntiles;
            const int n = cur.n, h0 = cur.hg * kHeadsPerCta + rank * kHeadsPerBlock, slot = cur.slot;
            const bool final_out = slot < 0, write = h0 + r < a.H;
            const int64_t prow0 = final_out ? 0 : (sched ? int64_t(slot) * kHeadsPerCta + rank * kHeadsPerBlock : (int64_t(slot) * a.B + n) * a.H + h0);
            __nv_bfloat16* const out_rows = final_out ? a.out + (int64_t(n) * a.H + h0) * 512 : reinterpret_cast<__nv_bfloat16*>(a.partial_o) + prow0 * 512;
            if (nb <= 0) {
#pragma unroll 1
                for (int i = tid; i < kHeadsPerBlock * 64; i += kNumSoftmaxWarps * 32)
                    if (h0 + (i >> 6) < a.H) *reinterpret_cast<uint4*>(out_rows + int64_t(i >> 6) * 512 + (i & 63) * 8) = make_uint4(0, 0, 0, 0);
                if (colhalf == 0 && write) {
                    if (!final_out) a.partial_lse[prow0 + r] = -CUDART_INF_F;
                    else if (a.lse != nullptr) a.lse[int64_t(n) * a.H + h0 + r] = -CUDART_INF_F;
                }
                if (k + 1 < n_items) cur = get_item(k + 1);
                continue;
            }
            // (rows past the last node are computed but not written)
            const int32_t* const node_mask = a.tree_mask + (int64_t(n) * (a.H / a.heads) + min(h0 + r, a.H - 1) / a.heads) * a.mask_words;
            auto sees = [&](int i) -> uint32_t {
                const int v0 = (cur.tile0 + i) * kTileN + 32 * colhalf;
                return v0 >= cur.n_tok ? 0u : uint32_t(ptx::ld(reinterpret_cast<const int32_t*>(a.valid) + (int64_t(n) * a.cap + v0) / 32)) &
                       window_bits(node_mask, a.mask_words, v0 - cur.kv_len_n);
            };
            uint32_t next_seen = sees(0);
            float m_ref = -CUDART_INF_F, l_sum = 0.f;
            bool left = false;
#pragma unroll 1
            for (int it = 0; it < nb; ++it) {
                const uint32_t g = gt + uint32_t(it), vmask = next_seen;
                if (it + 1 < nb) next_seen = sees(it + 1);
                const uint32_t s_tmem = tmem + lane_addr + kTmemS + (g & 1u) * 32u;
                if (ok) ok = wait_for(bar_s_full + 8 * (g & 1u), g >> 1, kStatusWaitSFull, 0, int(g));
                ptx::tc_fence_after_sync();
                uint32_t s0[32];
                ptx::tmem_ld32(s_tmem, s0);
                ptx::tmem_wait_ld();
                if (vmask != ~0u) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!((vmask >> i) & 1u)) s0[i] = 0xFF800000u;
                }
                float t4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) t4[i] = fmaxf(__uint_as_float(s0[i]), __uint_as_float(s0[i + 4]));
#pragma unroll
                for (int i = 8; i < 32; i += 8)
#pragma unroll
                    for (int j = 0; j < 4; ++j) t4[j] = ptx::max3(t4[j], __uint_as_float(s0[i + 2 * j]), __uint_as_float(s0[i + 2 * j + 1]));
                const float tmax = ptx::max3(ptx::max3(t4[0], t4[1], t4[2]), t4[3], -CUDART_INF_F) * a.scale_log2;
                float alpha = 1.f;
                const bool moved = ptx::bar_any(pair_bar, 64, !ok || tmax > m_ref + kRescaleThreshold);
                if (moved) {
                    misc->exch[tid] = tmax;
                    if (ptx::bar_any(pair_bar + 2u, 64, !ok)) { ok = false;  left = true;  break; }
                    const float rmax = fmaxf(tmax, misc->exch[tid ^ 64]);
                    if (rmax > m_ref + kRescaleThreshold) {
                        alpha = (m_ref == -CUDART_INF_F) ? 0.f : ptx::ex2(m_ref - rmax);
                        m_ref = rmax;
                    }
                }
                const float neg_m = (m_ref == -CUDART_INF_F) ? 0.f : -m_ref;
                const uint64_t scale2 = ptx::pack_f32x2(a.scale_log2, a.scale_log2), neg2 = ptx::pack_f32x2(neg_m, neg_m);
                uint64_t ps2[2] = {0ull, 0ull};
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float e0, e1;
                    ptx::unpack_f32x2(ptx::fma_f32x2(ptx::pack_f32x2(__uint_as_float(s0[2 * i]), __uint_as_float(s0[2 * i + 1])), scale2, neg2), e0, e1);
                    const float p0 = ptx::ex2(e0), p1 = ptx::ex2(e1);
                    ps2[i & 1] = ptx::add_f32x2(ps2[i & 1], ptx::pack_f32x2(p0, p1));
                    s0[i] = ptx::pack_f16x2(p0, p1);
                }
                float ps_lo, ps_hi;
                ptx::unpack_f32x2(ptx::add_f32x2(ps2[0], ps2[1]), ps_lo, ps_hi);
                l_sum = l_sum * alpha + (ps_lo + ps_hi);
                // the P buffer has been read by the O MMAs of the tile two before
                if (g >= 2u && !(ok = wait_for(bar_o_full + 8 * (g & 1u), (g - 2u) >> 1, kStatusWaitOFull, 0, int(g)))) continue;      // leaves at the next barrier
                if (it > 0 && moved && __any_sync(0xFFFFFFFFu, alpha != 1.f)) {
                    if (!(ok = wait_for(bar_o_full + 8 * ((g - 1u) & 1u), (g - 1u) >> 1, kStatusWaitOFull, 0, int(g)))) continue;
                    ptx::tc_fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        uint32_t o[32];
                        ptx::tmem_ld32(tmem + lane_addr + kTmemO + c * 32, o);
                        ptx::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        ptx::tmem_st32(tmem + lane_addr + kTmemO + c * 32, o);
                    }
                    ptx::tmem_wait_st();
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    ptx::sts_v4(p_row + (g & 1u) * kQChunkBytes + (p_sw ^ (uint32_t(c) << 4)), make_uint4(s0[4 * c], s0[4 * c + 1], s0[4 * c + 2], s0[4 * c + 3]));
                ptx::fence_proxy_async_smem();
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) arrive_even(bar_p_full + 8 * (g & 1u));
            }
            if (left) break;
            // ── the row's sum, and what its output is multiplied by ──
            gt += uint32_t(nb);
            if (k + 1 < n_items) cur = get_item(k + 1);
            if (ptx::bar_any(pair_bar, 64, !ok)) { ok = false;  break; }
            misc->exch[tid] = l_sum;
            ptx::bar_sync(pair_bar + 2u, 64);
            l_sum += misc->exch[tid ^ 64];
            if (tid == 0 && k == n_items - 1 && (sched || a.num_splits > 1)) ptx::pdl_trigger();      // (a merge follows)
            float denom = l_sum;
            if (final_out && a.attn_sink != nullptr && write) {
                const float s2 = ptx::ld(a.attn_sink + (h0 + r) % a.heads) * 1.4426950408889634f;
                denom = (l_sum != 0.f) ? l_sum + ptx::ex2(s2 - m_ref) : 1.f;
            }
            if (colhalf == 0) misc->inv[qn & 1u][r] = (l_sum != 0.f) ? 1.f / denom : 0.f;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar_inv + 8 * (qn & 1u));
            ++qn;
            if (write && colhalf == 0) {
                const float lse2 = (l_sum != 0.f) ? m_ref + log2f(l_sum) : -CUDART_INF_F;
                if (!final_out) a.partial_lse[prow0 + r] = lse2;
                else if (a.lse != nullptr) a.lse[int64_t(n) * a.H + h0 + r] = (l_sum != 0.f) ? lse2 * 0.6931471805599453f : -CUDART_INF_F;
            }
        }
    }

    // ── common exit ──
    __syncwarp();
    ptx::tc_fence_before_sync();
    ptx::cluster_sync();
    if (warp == kTreeSWarp) {
        ptx::tc_fence_after_sync();
        if (ptx::lds_u32(failed_flag())) hold_block();
        ptx::tmem2_dealloc(misc->tmem_base, kTmemCols);
    }
}

}  // namespace dsv4
