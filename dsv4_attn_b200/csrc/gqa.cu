// Entry points of include/dsv4_gqa.h: argument validation, tensor maps, launches.  No allocation, no synchronisation, and nothing kept between calls but facts
// about the device.
#include "../../include/dsv4_gqa.h"

#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cmath>

#include "gqa_decode.cuh"
#include "gqa_prefill.cuh"
#include "gqa_rows.cuh"
#include "kv_evict.cuh"
#include "host_state.h"

namespace dsv4 {
namespace {

constexpr int kMaxDevices = 64;

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

template <typename Kernel>
cudaError_t ensure_smem(Kernel kernel, int bytes, std::atomic<bool>* done_per_device) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    if (!done_per_device[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return e;
        done_per_device[dev].store(true, std::memory_order_release);
    }
    return cudaSuccess;
}

// Every kernel is a programmatic dependent of whatever precedes it in the stream, as in api.cu.
template <class Args>
cudaError_t launch(void (*kernel)(Args), dim3 grid, int threads, size_t smem, cudaStream_t stream, const Args& args, int cluster = 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    unsigned used = 0;
    if (cluster > 0) {
        attr[used].id = cudaLaunchAttributeClusterDimension;
        attr[used].val.clusterDim.x = unsigned(cluster);
        attr[used].val.clusterDim.y = attr[used].val.clusterDim.z = 1;
        ++used;
    }
    if (!(host_state().flags & 64)) {
        attr[used].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[used].val.programmaticStreamSerializationAllowed = 1;
        ++used;
    }
    cfg.attrs = attr;
    cfg.numAttrs = used;
    return cudaLaunchKernelEx(&cfg, kernel, args);
}

// What L2 fetches around a request: no more than the head's row, whose neighbours are another head's (heads of 128 bytes, with 256: 64 x 8,000 entries 241 us instead of 193).
CUtensorMapL2promotion promotion(int row_bytes) {
    return row_bytes >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : row_bytes >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
}

// A pool of K or V heads by (element, head, entry): boxes of 128 bytes (or a shorter row) of one head in 64 entries.
cudaError_t make_pool_map(CUtensorMap* map, const void* pool, int64_t pages, int Hkv, int D, int kv_dtype, int box_rows = kGqaTile) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return cudaErrorNotSupported;
    const bool bytes = kv_dtype == DSV4_DTYPE_E4M3;
    const int es = bytes ? 1 : 2, box_bytes = D * es < 128 ? D * es : 128;
    const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(Hkv), cuuint64_t(pages) * kGqaTile};
    const cuuint64_t strides[2] = {cuuint64_t(D) * es, cuuint64_t(Hkv) * D * es};
    const cuuint32_t box[3] = {cuuint32_t(box_bytes / es), 1, cuuint32_t(box_rows)}, estr[3] = {1, 1, 1};
    const CUresult r = fn(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(pool), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          promotion(D * es),
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

int64_t up(int64_t n) { return (n + 127) / 128 * 128; }

// An 8-bit pool: boxes of a head's whole rows of a page, as they lie.
cudaError_t make_raw_map(CUtensorMap* map, const void* pool, int64_t pages, int Hkv, int D) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {cuuint64_t(D), cuuint64_t(Hkv), cuuint64_t(pages) * kGqaTile}, strides[2] = {cuuint64_t(D), cuuint64_t(Hkv) * D};
    const cuuint32_t box[3] = {cuuint32_t(D), 1, kGqaTile}, estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pool), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                          promotion(D), CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// ── which form of the kernel ──
// Rows of a KV head: 16, 32 or 64 in a group, the fewest that hold a request's (with 64: several groups).
int group_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
constexpr int kMinShare = 2;         // tiles (one request of 2,000 entries: 12.3 us, with 1 15, with 4 13.8)
// A cluster's parts are joined in one kernel, which is worth kClusterMore tiles that shares would have spread over more blocks (heads of 128, 16 bits): eight units, 4 tiles a block of a cluster against
// 0.7 of a share 9.3 against 9.7 us, 8 against 1.7 13.9 against 12.3; 32 units, 16 against 13.8 27.6 against 35; 128 units, 32 against 28 45 against 54.  Beyond kClusterTiles lengths that differ,
// which shares even out, cost more than that.  Of rows: 24 of one request's 1,000 entries 11 us in clusters against 13 in gqa_rows_kernel, 40 18 against 13.
constexpr int kClusterMore = 5, kClusterTiles = 32, kClusterRows = 32;

template <class C>
cudaError_t run_decode(GqaArgs& a, cudaStream_t stream) {
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = ensure_smem(gqa_decode_kernel<C>, C::Bytes, done);
    if (e != cudaSuccess) return e;
    return launch(gqa_decode_kernel<C>, dim3(unsigned(a.blocks)), kGqaThreads, C::Bytes, stream, a, a.cluster);
}
template <int D, int KVT>
cudaError_t run_decode(GqaArgs& a, cudaStream_t stream) {
    if (a.group_rows == 16) return run_decode<GqaCfg<D, KVT, 1>>(a, stream);
    if (a.group_rows == 32) return run_decode<GqaCfg<D, KVT, 2>>(a, stream);
    return run_decode<GqaCfg<D, KVT, 4>>(a, stream);
}
template <int D>
cudaError_t run_decode(GqaArgs& a, int kv_dtype, cudaStream_t stream) {
    if (kv_dtype == DSV4_DTYPE_BF16) return run_decode<D, kGqaBf16>(a, stream);
    if (kv_dtype == DSV4_DTYPE_F16) return run_decode<D, kGqaF16>(a, stream);
    return run_decode<D, kGqaE4m3>(a, stream);
}

// Sizes that a call's blocks and workspace follow from.
struct Sizes {
    int blocks, group_rows;
    int64_t parts;                   // partial rows
    int64_t logit_rows, logit_stride;
    bool prefill;                    // gqa_prefill_kernel
    int streams;                     // gqa_rows_kernel, if not 0
    int cluster;                     // blocks of a cluster that has a unit, or 0: shares
    int64_t plan_words;
    int own_pages;                   // of a request, 16-bit copies of an 8-bit cache's, or 0
    int round_b, round_h;            // requests and KV heads that a launch of gqa_prefill_kernel takes
    int64_t own_bytes() const { return int64_t(round_b) * own_pages * kGqaTile * round_h * D * 2; }      // of K's copies, and of V's
    int D;
};

// ── which kernel takes tokens that are not packed ──
// Rows of a KV head beyond which gqa_rows_kernel takes them: 64 requests x 8,000 entries, heads of 128, 16 rows 322 us in gqa_decode_kernel against 336, 20 rows 359 against 339; in 8 bits 248
// against 347 and 424 against 355.  Short 16-bit rows: 32 rows of 64 elements 246 against 265.
constexpr int kRowsMore = 16, kRowsMore64 = 32;

// ── which kernel takes a prompt ──
// A block of tokens is 256 rows (heads of 256: 128) in gqa_prefill_kernel and has an SM to itself, where a step of 64 entries takes 1 us; the decode kernel takes 64 rows at a time, 2 us for that, and shares
// the entries out over all SMs, for 10 us more.  Eight heads, one prompt behind a cache of 2,048 entries: 64 tokens 46 us in gqa_prefill_kernel and 33 in the other, 128 46 and 57; of 16,384:
// 128 tokens 254 and 192, 256 260 and 355.
constexpr int kPrefillMinUnits = 8, kPrefillStep = 10, kPrefillTile = 20, kPrefillMore = 100;      // 0.1 us
// An 8-bit cache's pages are brought to 16 bits in a workspace of that size at most, by the lengths that there can be: a call with room for more is gone through in rounds, some requests at a time, or
// some heads of one.
constexpr int64_t kPrefillOwnBytes = int64_t(4) << 30;
bool gqa_sizes(const Dsv4GqaParams* p, Sizes& s) {
    if (p == nullptr || p->B <= 0 || p->Hkv <= 0 || p->G <= 0 || p->max_pages <= 0 || p->T < 0 || p->rows < 0) return false;
    if (p->D != 64 && p->D != 128 && p->D != 256) return false;
    const int64_t tokens = p->q_start != nullptr ? p->rows : p->T;          // of a request, at most
    if (tokens <= 0 || int64_t(p->Hkv) * p->G > 65536 || tokens > (1 << 24) || tokens * p->G > 0x7FFFFFFF / 4 || int64_t(p->max_pages) * kGqaTile > 0x7FFFFFFF) return false;
    s.group_rows = group_rows(tokens * p->G);
    const int64_t entries = int64_t(p->max_pages) * kGqaTile;
    int64_t longest = p->max_len > 0 && p->max_len < entries ? p->max_len : entries;
    if (p->window > 0 && longest > int64_t(p->window) + p->first + tokens + 2 * kGqaTile) longest = int64_t(p->window) + p->first + tokens + 2 * kGqaTile;
    const int64_t groups = p->q_start != nullptr ? (p->rows * p->G + s.group_rows - 1) / s.group_rows + p->B : int64_t(p->B) * ((tokens * p->G + s.group_rows - 1) / s.group_rows);
    const int64_t tiles = groups * p->Hkv * ((longest + kGqaTile - 1) / kGqaTile + 1);
    const int64_t resident = int64_t(device_sms()) * gqa_blocks_per_sm(p->D), want = (tiles + kMinShare - 1) / kMinShare;
    s.blocks = int(want < resident ? want : resident);
    s.parts = 2 * int64_t(s.blocks) * s.group_rows;
    s.cluster = 0;
    if (p->q_start == nullptr && tokens * p->G <= kClusterRows) {
        // the widest cluster with which all units are resident at once
        const int64_t units = int64_t(p->B) * p->Hkv, most = (longest + kGqaTile - 1) / kGqaTile + 1;
        int c = 8;
        while (c > 1 && units * c > resident) c /= 2;
        // (with one block an SM clusters of eight do not come to lie side by side on all of them: 16 units of 256 elements 17 us, in shares 12; eight 9 against 11)
        if (c == 8 && p->D > 128 && units * 16 > resident) c = 4;
        const int64_t each = (most + c - 1) / c;
        if (c > 1 && each <= kClusterTiles && each - units * most / resident <= kClusterMore - (tokens * p->G > 16)) {
            s.cluster = c;
            s.blocks = int(units) * s.cluster;
            s.parts = 0;
        }
    }
    s.logit_rows = p->weights != nullptr ? int64_t(p->B) * p->Hkv * p->T * p->G : 0;
    s.logit_stride = p->max_len > 0 && p->max_len < entries ? (int64_t(p->max_len) + kGqaTile - 1) / kGqaTile * kGqaTile : entries;
    s.prefill = false;
    s.plan_words = 0;
    s.own_pages = s.round_b = s.round_h = 0;
    s.D = p->D;
    s.streams = 0;
    // (tensor maps have no axis that stays where it is)
    const bool spread = (p->Hkv * p->G == 1 || p->q_stride_h > 0) && (tokens == 1 || p->q_stride_t > 0) && (p->q_start != nullptr || p->B == 1 || p->q_stride_b > 0);
    if (p->q_start == nullptr && s.cluster == 0 && p->G <= 128 && (spread || p->kv_dtype == DSV4_DTYPE_E4M3) && tokens * p->G > (p->kv_dtype != DSV4_DTYPE_E4M3 && p->D == 64 ? kRowsMore64 : kRowsMore)) {
        s.streams = p->D > 128 ? 1 : 2;
        s.group_rows = (s.streams == 2 && tokens * p->G <= 64 ? 64 : 128) / p->G * p->G;
        const int64_t most = int64_t(p->B) * ((tokens * p->G + s.group_rows - 1) / s.group_rows) * p->Hkv * ((longest + kGqaTile - 1) / kGqaTile + 1);
        s.blocks = int(most < device_sms() ? most : device_sms());
        s.parts = int64_t(s.blocks) * (2 * s.streams + 1) * s.group_rows;
    }
    if (p->q_start != nullptr && p->G <= 128 && p->rows < 0x7FFFFFFF && spread) {
        const int tile_tokens = 128 / p->G, block_tokens = tile_tokens * (p->D > 128 ? 1 : 2);
        const int64_t blocks = p->rows / block_tokens + p->B, full = (p->rows + block_tokens - 1) / block_tokens;
        const bool e4m3 = p->kv_dtype == DSV4_DTYPE_E4M3;
        int64_t own_pages = 0, round_b = p->B, round_h = p->Hkv, rounds = 1;
        if (e4m3) {
            own_pages = p->max_len > 0 && p->max_len < entries ? (p->max_len + kGqaTile - 1) / kGqaTile : p->max_pages;
            const int64_t head_bytes = own_pages * kGqaTile * p->D * 4, most_b = kPrefillOwnBytes / (head_bytes * p->Hkv), most_h = kPrefillOwnBytes / head_bytes;
            if (most_b < p->B) {
                const int64_t n = most_b > 0 ? (p->B + most_b - 1) / most_b : p->B;
                round_b = (p->B + n - 1) / n;                                 // (rounds alike)
                rounds = (p->B + round_b - 1) / round_b;
            }
            if (most_b == 0 && most_h > 0) {
                const int64_t n = (p->Hkv + most_h - 1) / most_h;
                round_h = (p->Hkv + n - 1) / n;
                rounds *= (p->Hkv + round_h - 1) / round_h;
            }
            if (most_h == 0) rounds = 0;                                      // (a head of one request has more: 8 million entries of 128)
        }
        const int64_t steps = (longest + kGqaTile - 1) / kGqaTile, all = (full + p->B) * p->Hkv, least = rounds * device_sms(), units = all > least ? all : least;
        const int64_t groups = (p->rows * p->G + 63) / 64 * p->Hkv, tile = int64_t(kPrefillTile) * (p->D > 128 ? 2 : 1);
        const bool quicker = steps * (units * kPrefillStep - groups * tile) <= int64_t(kPrefillMore) * device_sms();
        s.prefill = quicker && full * p->Hkv >= kPrefillMinUnits && rounds > 0 && round_b * own_pages * kGqaTile < 0x7FFFFF00;
        if (s.prefill) {
            s.plan_words = 4 + 2 * blocks;
            s.own_pages = int(own_pages);
            s.round_b = int(round_b);
            s.round_h = int(round_h);
            const int64_t most = blocks * round_h;
            s.blocks = int(most < device_sms() ? most : device_sms());
            s.group_rows = block_tokens * p->G;
            s.parts = 0;
        }
    }
    return true;
}

template <int D, bool BF16>
cudaError_t run_prefill(const GqaPrefillArgs& a, cudaStream_t stream) {
    using C = PrefillCfg<D, BF16>;
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = ensure_smem(gqa_prefill_kernel<C>, C::Bytes, done);
    if (e != cudaSuccess) return e;
    return launch(gqa_prefill_kernel<C>, dim3(unsigned(a.g.blocks)), C::Threads, C::Bytes, stream, a);
}

template <int D, int KVT>
cudaError_t run_rows(const GqaRowsArgs& a, cudaStream_t stream) {
    using C = RowsCfg<D, KVT>;
    static std::atomic<bool> done[kMaxDevices];
    cudaError_t e = ensure_smem(gqa_rows_kernel<C>, C::Bytes, done);
    if (e != cudaSuccess) return e;
    return launch(gqa_rows_kernel<C>, dim3(unsigned(a.g.blocks)), C::Threads, C::Bytes, stream, a);
}
template <int D>
cudaError_t run_rows(const GqaRowsArgs& a, int kv_dtype, cudaStream_t stream) {
    if (kv_dtype == DSV4_DTYPE_BF16) return run_rows<D, kGqaBf16>(a, stream);
    if (kv_dtype == DSV4_DTYPE_F16) return run_rows<D, kGqaF16>(a, stream);
    return run_rows<D, kGqaE4m3>(a, stream);
}

// q by (element, head, token, request): boxes of 64 elements of a group's heads in a tile's tokens
cudaError_t make_tokens_map(CUtensorMap* map, const Dsv4GqaParams* p, int tile_tokens) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return cudaErrorNotSupported;
    const int H = p->Hkv * p->G;
    const int64_t row = int64_t(H) * p->D;
    const cuuint64_t dims[4] = {cuuint64_t(p->D), cuuint64_t(H), cuuint64_t(p->T), cuuint64_t(p->B)};
    // (axes of one element have any stride)
    const cuuint64_t strides[3] = {cuuint64_t(H > 1 ? p->q_stride_h : p->D) * 2, cuuint64_t(p->T > 1 ? p->q_stride_t : row) * 2, cuuint64_t(p->B > 1 ? p->q_stride_b : row * p->T) * 2};
    const cuuint32_t box[4] = {64, cuuint32_t(p->G), cuuint32_t(tile_tokens), 1}, estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(p->q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t decode_rows(const GqaArgs& g, const Dsv4GqaParams* p, cudaStream_t stream) {
    GqaRowsArgs a{};
    a.g = g;
    a.tile_tokens = g.group_rows / p->G;
    a.second = g.streams == 2 && g.group_rows <= 64 && int64_t(p->T) * p->G <= 64 ? 64 : 0;
    cudaError_t e = cudaSuccess;
    if (p->kv_dtype == DSV4_DTYPE_E4M3) {
        e = make_raw_map(&a.g.k_map, p->k_pool, p->num_pages, p->Hkv, p->D);
        if (e == cudaSuccess) e = make_raw_map(&a.g.v_map, p->v_pool, p->num_pages, p->Hkv, p->D);
    } else {
        e = make_pool_map(&a.g.k_map, p->k_pool, p->num_pages, p->Hkv, p->D, p->kv_dtype);
        if (e == cudaSuccess) e = make_pool_map(&a.g.v_map, p->v_pool, p->num_pages, p->Hkv, p->D, p->kv_dtype);
        if (e == cudaSuccess) e = make_pool_map(&a.v8_map, p->v_pool, p->num_pages, p->Hkv, p->D, p->kv_dtype, 8);
        if (e == cudaSuccess) e = make_pool_map(&a.v1_map, p->v_pool, p->num_pages, p->Hkv, p->D, p->kv_dtype, 1);
        if (e == cudaSuccess) e = make_tokens_map(&a.q_map, p, a.tile_tokens);
    }
    if (e != cudaSuccess) return e;
    return p->D == 64 ? run_rows<64>(a, p->kv_dtype, stream) : p->D == 128 ? run_rows<128>(a, p->kv_dtype, stream) : run_rows<256>(a, p->kv_dtype, stream);
}

// q by (element, head, row): boxes of 64 elements of a group's heads in a tile's tokens
cudaError_t make_rows_map(CUtensorMap* map, const Dsv4GqaParams* p, int tile_tokens) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return cudaErrorNotSupported;
    const int H = p->Hkv * p->G;
    const cuuint64_t dims[3] = {cuuint64_t(p->D), cuuint64_t(H), cuuint64_t(p->rows)};
    // (axes of one element have any stride)
    const cuuint64_t strides[2] = {cuuint64_t(H > 1 ? p->q_stride_h : p->D) * 2, cuuint64_t(p->rows > 1 ? p->q_stride_t : int64_t(H) * p->D) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(p->G), cuuint32_t(tile_tokens)}, estr[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(p->q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Requests b0 .. of a call, heads h0 .. of them
cudaError_t prefill_round(const GqaArgs& g, const Dsv4GqaParams* p, const Sizes& s, uint8_t* ws, int b0, int h0, cudaStream_t stream) {
    GqaPrefillArgs a{};
    a.g = g;
    a.g.B = p->B - b0 < s.round_b ? p->B - b0 : s.round_b;
    a.g.q_start += b0;
    a.g.kv_len += b0;
    a.g.block_table += int64_t(b0) * p->max_pages;
    a.b0 = b0;
    a.h0 = h0;
    a.heads = p->Hkv - h0 < s.round_h ? p->Hkv - h0 : s.round_h;
    a.plan = reinterpret_cast<int32_t*>(ws);
    a.plan_units = int((s.plan_words - 4) / 2);
    ws += up(s.plan_words * 4);
    const void *k = p->k_pool, *v = p->v_pool;
    int64_t pages = p->num_pages;
    a.tile_tokens = 128 / p->G;
    cudaError_t e = cudaSuccess;
    if (s.own_pages > 0) {
        GqaUnpackArgs u{};
        u.g = a.g;
        u.own_pages = a.own_pages = s.own_pages;
        u.h0 = h0;  u.heads = a.heads;  u.D = p->D;
        for (int i = 0; i < 2; ++i) {
            u.pool[i] = static_cast<const uint8_t*>(i ? v : k);
            u.rows[i] = ws;
            ws += up(s.own_bytes());
        }
        k = u.rows[0];
        v = u.rows[1];
        pages = int64_t(a.g.B) * s.own_pages;
        // eight blocks an SM over all requests
        const int64_t each = (int64_t(device_sms()) * 8 + a.g.B - 1) / a.g.B;
        u.blocks = int(each < s.own_pages ? each : s.own_pages);
        e = launch(g.q_bf16 ? gqa_unpack_kernel<true> : gqa_unpack_kernel<false>, dim3(unsigned(a.g.B) * unsigned(u.blocks)), kGqaUnpackThreads, 0, stream, u);
        if (e != cudaSuccess) return e;
    }
    a.pool_rows = pages * kGqaTile;
    const int pool_heads = s.own_pages > 0 ? a.heads : p->Hkv;
    e = make_pool_map(&a.g.k_map, k, pages, pool_heads, p->D, p->q_dtype);
    if (e == cudaSuccess) e = make_pool_map(&a.g.v_map, v, pages, pool_heads, p->D, p->q_dtype);
    if (e == cudaSuccess) e = make_pool_map(&a.v8_map, v, pages, pool_heads, p->D, p->q_dtype, 8);
    if (e == cudaSuccess) e = make_pool_map(&a.v1_map, v, pages, pool_heads, p->D, p->q_dtype, 1);
    if (e == cudaSuccess) e = make_rows_map(&a.q_map, p, a.tile_tokens);
    if (e == cudaSuccess) e = launch(gqa_plan_kernel, dim3(1), kPrefillPlanThreads, 0, stream, a);
    if (e != cudaSuccess) return e;
    if (p->D == 64) return g.q_bf16 ? run_prefill<64, true>(a, stream) : run_prefill<64, false>(a, stream);
    if (p->D == 128) return g.q_bf16 ? run_prefill<128, true>(a, stream) : run_prefill<128, false>(a, stream);
    return g.q_bf16 ? run_prefill<256, true>(a, stream) : run_prefill<256, false>(a, stream);
}

cudaError_t prefill(const GqaArgs& g, const Dsv4GqaParams* p, const Sizes& s, uint8_t* ws, cudaStream_t stream) {
    cudaError_t e = cudaSuccess;
    for (int64_t b = 0; b < p->B && e == cudaSuccess; b += s.round_b)
        for (int64_t h = 0; h < p->Hkv && e == cudaSuccess; h += s.round_h) e = prefill_round(g, p, s, ws, int(b), int(h), stream);
    return e;
}

}  // namespace
}  // namespace dsv4

using namespace dsv4;

extern "C" int64_t dsv4_gqa_workspace_bytes(const Dsv4GqaParams* p) {
    Sizes s;
    if (!gqa_sizes(p, s)) return -1;
    return 128 + up(s.parts * p->D * 4) + up(s.parts * 4) + up(s.logit_rows * s.logit_stride * 4) + up(s.logit_rows * 4) + up(s.plan_words * 4) + 2 * up(s.own_bytes());
}

static int gqa_fwd(const Dsv4GqaParams* p, void* stream_) {
    Sizes s;
    if (!gqa_sizes(p, s)) return int(cudaErrorInvalidValue);
    const bool e4m3 = p->kv_dtype == DSV4_DTYPE_E4M3;
    if ((p->q_dtype != DSV4_DTYPE_BF16 && p->q_dtype != DSV4_DTYPE_F16) || (!e4m3 && p->kv_dtype != p->q_dtype)) return int(cudaErrorInvalidValue);
    if (p->num_pages <= 0 || p->num_pages >= 0x7FFFFFFF / kGqaTile || p->window < 0 || p->first < 0 || !(p->sm_scale > 0.f) || !(p->sm_scale < INFINITY)) return int(cudaErrorInvalidValue);
    if (!p->q || !p->k_pool || !p->v_pool || !p->block_table || !p->kv_len || !p->out || (e4m3 && (!p->k_scale || !p->v_scale))) return int(cudaErrorInvalidValue);
    if (p->q_start == nullptr && p->rows != int64_t(p->B) * p->T) return int(cudaErrorInvalidValue);
    if (!aligned(p->q, 16) || !aligned(p->k_pool, 16) || !aligned(p->v_pool, 16) || !aligned(p->out, 16)) return int(cudaErrorInvalidValue);
    if (p->q_stride_b % 8 || p->q_stride_t % 8 || p->q_stride_h % 8) return int(cudaErrorInvalidValue);
    if (p->weights != nullptr && (p->q_start != nullptr || p->B > 65535 || p->weight_stride < int64_t(p->max_pages) * kGqaTile)) return int(cudaErrorInvalidValue);
    if (p->workspace == nullptr || !aligned(p->workspace, 128) || p->workspace_bytes < dsv4_gqa_workspace_bytes(p)) return int(cudaErrorInvalidValue);
    const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    const HostState state = host_state();

    GqaArgs a{};
    a.B = p->B;  a.T = p->T;  a.Hkv = p->Hkv;  a.G = p->G;  a.max_pages = p->max_pages;
    constexpr int kFar = 1 << 30;                                             // (sums of places stay within 32 bits; no entry is further back)
    a.window = p->window < kFar ? p->window : kFar;
    a.first = p->first;
    a.rows = p->rows;  a.q_start = p->q_start;  a.kv_len = p->kv_len;  a.block_table = p->block_table;  a.num_pages = p->num_pages;
    a.q = p->q;  a.q_stride_b = p->q_stride_b;  a.q_stride_t = p->q_stride_t;  a.q_stride_h = p->q_stride_h;  a.q_bf16 = p->q_dtype == DSV4_DTYPE_BF16;
    a.k_scale = e4m3 ? p->k_scale : nullptr;  a.v_scale = e4m3 ? p->v_scale : nullptr;  a.sink = p->attn_sink;
    a.scale_log2 = p->sm_scale * 1.4426950408889634f;
    a.out = p->out;  a.lse = p->lse;
    a.blocks = s.blocks;  a.group_rows = s.group_rows;  a.min_share = kMinShare;
    a.one_group = p->q_start == nullptr && int64_t(p->T) * p->G <= s.group_rows;
    uint8_t* ws = static_cast<uint8_t*>(p->workspace);
    a.part_o = reinterpret_cast<float*>(ws);  ws += up(s.parts * p->D * 4);
    a.part_lse = reinterpret_cast<float*>(ws);  ws += up(s.parts * 4);
    if (p->weights != nullptr) {
        a.logits = reinterpret_cast<float*>(ws);  ws += up(s.logit_rows * s.logit_stride * 4);
        a.total = reinterpret_cast<float*>(ws);
        a.logit_stride = s.logit_stride;
        a.logit_end = int(s.logit_stride);
        a.weight_len = p->max_len > 0 && p->max_len < s.logit_stride ? p->max_len : a.logit_end;
        a.weights = p->weights;  a.weight_stride = p->weight_stride;
    }
    a.wait_ns = uint32_t(state.wait_ns < 4000000000ull ? state.wait_ns : 4000000000ull);
    a.dbg_drop_tile = state.drop_tile;
    a.status = p->status;
    if (s.prefill) return int(prefill(a, p, s, ws, stream));
    a.streams = s.streams;
    a.cluster = s.cluster;
    cudaError_t e = cudaSuccess;
    if (s.streams > 0) {
        e = decode_rows(a, p, stream);
    } else {
        e = make_pool_map(&a.k_map, p->k_pool, p->num_pages, p->Hkv, p->D, p->kv_dtype);
        if (e == cudaSuccess) e = make_pool_map(&a.v_map, p->v_pool, p->num_pages, p->Hkv, p->D, p->kv_dtype);
        if (e != cudaSuccess) return int(e);
        e = p->D == 64 ? run_decode<64>(a, p->kv_dtype, stream) : p->D == 128 ? run_decode<128>(a, p->kv_dtype, stream) : run_decode<256>(a, p->kv_dtype, stream);
    }
    if (e != cudaSuccess) return int(e);
    // a row has as many warps as stay within 32 for every SM
    const int64_t merge_rows = p->rows * p->Hkv * p->G;
    a.merge_warps = kGqaMergeWarps;
    while (a.merge_warps > 1 && merge_rows * a.merge_warps > int64_t(device_sms()) * 32) a.merge_warps /= 2;
    const int64_t block_rows = kGqaMergeWarps / a.merge_warps, merge_blocks = (merge_rows + block_rows - 1) / block_rows;
    if (s.cluster == 0 && (s.blocks > 1 || s.streams > 0)) {
        const dim3 grid{unsigned(merge_blocks)};
        e = p->D == 64 ? launch(gqa_merge_kernel<64>, grid, kGqaMergeThreads, 0, stream, a)
                       : p->D == 128 ? launch(gqa_merge_kernel<128>, grid, kGqaMergeThreads, 0, stream, a) : launch(gqa_merge_kernel<256>, grid, kGqaMergeThreads, 0, stream, a);
        if (e != cudaSuccess) return int(e);
    }
    if (p->weights != nullptr) {
        e = launch(gqa_weights_kernel, dim3(unsigned((a.weight_len + kGqaWeightThreads - 1) / kGqaWeightThreads), unsigned(p->B)), kGqaWeightThreads, 0, stream, a);
    }
    return int(e);
}

extern "C" int dsv4_gqa_decode_fwd(const Dsv4GqaParams* p, void* stream) {
    if (p == nullptr || p->q_start != nullptr) return int(cudaErrorInvalidValue);
    return gqa_fwd(p, stream);
}

extern "C" int dsv4_gqa_prefill_fwd(const Dsv4GqaParams* p, void* stream) {
    if (p == nullptr || p->q_start == nullptr || p->weights != nullptr) return int(cudaErrorInvalidValue);
    return gqa_fwd(p, stream);
}

extern "C" int dsv4_gqa_insert(const Dsv4GqaInsertParams* p, void* stream) {
    if (p == nullptr || p->B <= 0 || p->T < 0 || p->rows < 0 || p->Hkv <= 0 || p->max_pages <= 0 || p->num_pages <= 0) return int(cudaErrorInvalidValue);
    if (p->D <= 0 || p->D % 8 != 0 || int64_t(p->Hkv) * p->D > (1 << 24) || p->num_pages > 0x7FFFFFFF / kGqaTile) return int(cudaErrorInvalidValue);
    const bool e4m3 = p->kv_dtype == DSV4_DTYPE_E4M3;
    if ((p->src_dtype != DSV4_DTYPE_BF16 && p->src_dtype != DSV4_DTYPE_F16) || (!e4m3 && p->kv_dtype != p->src_dtype)) return int(cudaErrorInvalidValue);
    if (!p->k || !p->v || !p->k_pool || !p->v_pool || !p->block_table || !p->insert_pos || (e4m3 && (!p->k_scale || !p->v_scale))) return int(cudaErrorInvalidValue);
    if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->k_pool, 16) || !aligned(p->v_pool, 16)) return int(cudaErrorInvalidValue);
    if (p->q_start == nullptr && (p->T == 0 ? p->rows != 0 : p->rows != int64_t(p->B) * p->T)) return int(cudaErrorInvalidValue);
    GqaInsertArgs a{};
    const int64_t strides[6] = {p->k_stride_b, p->k_stride_t, p->k_stride_h, p->v_stride_b, p->v_stride_t, p->v_stride_h};
    for (int i = 0; i < 6; ++i)
        if (strides[i] % 8 != 0) return int(cudaErrorInvalidValue);
    for (int i = 2; i < 6; i += 3)
        if (strides[i] < 0 || strides[i] > (int64_t(1) << 30) / p->Hkv) return int(cudaErrorInvalidValue);      // (places within a row stay within 32 bits)
    if (p->rows == 0) return 0;
    a.B = p->B;  a.T = p->T;  a.Hkv = p->Hkv;  a.D = p->D;  a.max_pages = p->max_pages;  a.rows = p->rows;
    a.q_start = p->q_start;  a.n_rows = p->n_rows;  a.insert_pos = p->insert_pos;  a.block_table = p->block_table;  a.num_pages = p->num_pages;
    a.src[0] = p->k;  a.src[1] = p->v;
    for (int i = 0; i < 2; ++i) { a.stride_b[i] = strides[3 * i];  a.stride_t[i] = strides[3 * i + 1];  a.stride_h[i] = strides[3 * i + 2]; }
    a.src_bf16 = p->src_dtype == DSV4_DTYPE_BF16;
    a.scale[0] = p->k_scale;  a.scale[1] = p->v_scale;
    a.pool[0] = p->k_pool;  a.pool[1] = p->v_pool;
    a.status = p->status;
    // as many tokens a block (2 to 32) as leave four blocks for every SM
    int block_tokens = kGqaInsertTokens;
    while (block_tokens > 2 && p->rows < int64_t(block_tokens) * device_sms() * 4) block_tokens /= 2;
    a.block_tokens = block_tokens;
    const int64_t blocks = (p->rows + block_tokens - 1) / block_tokens;
    if (blocks > 0x7FFFFFFF || int64_t(block_tokens) * p->Hkv * p->D > 0x7FFFFFFF) return int(cudaErrorInvalidValue);
    return int(launch(e4m3 ? gqa_insert_kernel<true> : gqa_insert_kernel<false>, dim3(unsigned(blocks)), kGqaInsertThreads, 0, static_cast<cudaStream_t>(stream), a));
}

extern "C" int dsv4_kv_evict(const Dsv4KvEvictParams* p, void* stream_) {
    if (p == nullptr || p->B <= 0 || p->B > 65535 || p->max_pages <= 0 || p->num_pages <= 0 || p->layers <= 0 || p->pools < 0 || p->pools > DSV4_EVICT_POOLS) return int(cudaErrorInvalidValue);
    const int64_t cap = int64_t(p->max_pages) * 64;
    if (p->num_pages > 0x7FFFFFFF / 64 || cap > 0x7FFFFFFF - kEvictPlanThreads * kEvictEach || p->first < 0 || p->recent < 0 || (p->keep_each == nullptr && p->keep < 0))
        return int(cudaErrorInvalidValue);
    if (!p->block_table || !p->kv_len || !p->refs || !p->weights || !p->new_table || !p->new_len || !p->new_refs || !p->new_weights || !p->kept || !p->scratch)
        return int(cudaErrorInvalidValue);
    if (p->weight_stride < cap || p->weight_stride > 0x7FFFFFFF - kEvictPlanThreads || !aligned(p->scratch, 16)) return int(cudaErrorInvalidValue);
    const cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    KvEvictArgs a{};
    a.B = p->B;  a.max_pages = p->max_pages;  a.pools = p->pools;  a.num_pages = p->num_pages;  a.layers = p->layers;
    a.keep = p->keep;  a.first = p->first;  a.recent = p->recent;  a.keep_each = p->keep_each;
    a.block_table = p->block_table;  a.kv_len = p->kv_len;  a.refs = p->refs;  a.weights = p->weights;  a.weight_stride = p->weight_stride;
    a.new_table = p->new_table;  a.new_len = p->new_len;  a.new_refs = p->new_refs;  a.new_weights = p->new_weights;  a.kept = p->kept;
    a.moves = p->scratch;  a.from = p->scratch + 4 * int64_t(p->B);
    a.status = p->status;
    int64_t vecs_of_all = 0;
    for (int i = 0; i < p->pools; ++i) {
        if (p->pool[i] == nullptr || !aligned(p->pool[i], 16) || p->entry_bytes[i] <= 0 || p->entry_bytes[i] % 16 != 0 || p->entry_bytes[i] > (1 << 20)) return int(cudaErrorInvalidValue);
        a.pool[i] = static_cast<uint4*>(p->pool[i]);
        a.vecs[i] = int(p->entry_bytes[i] / 16);
        vecs_of_all += p->layers * a.vecs[i];
        // (a pool that is given twice would be moved twice, by blocks that do not know of one another)
        const int64_t entries = p->layers * p->num_pages * 64;
        for (int j = 0; j < i; ++j) {
            const uint8_t *x = static_cast<const uint8_t*>(p->pool[i]), *y = static_cast<const uint8_t*>(p->pool[j]);
            if (x < y + entries * p->entry_bytes[j] && y < x + entries * p->entry_bytes[i]) return int(cudaErrorInvalidValue);
        }
    }
    // as wide columns as leave four blocks for every SM, from 512 bytes down to a sector; half of one where that leaves not even a block for each (one request, two layers: one step of loads
    // instead of two, 17.2 -> 14.7 us with the plan's)
    int width = 32;
    while (width > 2 && vecs_of_all * p->B / width < int64_t(device_sms()) * 4) width /= 2;
    if (vecs_of_all * p->B / width < device_sms()) width = 1;
    int64_t columns = 0;
    for (int i = 0; i < p->pools; ++i) {
        a.width[i] = width;
        a.columns[i] = (a.vecs[i] + width - 1) / width;
        columns += p->layers * a.columns[i];
    }
    if (columns > 0x7FFFFFFF) return int(cudaErrorInvalidValue);
    a.all_columns = int(columns);
    cudaError_t e = launch(evict_plan_kernel, dim3(unsigned(p->B)), kEvictPlanThreads, 0, stream, a);
    if (e == cudaSuccess) e = launch(evict_move_kernel, dim3(unsigned(columns < 1 ? 1 : columns), unsigned(p->B)), kEvictMoveThreads, 0, stream, a);
    return int(e);
}
