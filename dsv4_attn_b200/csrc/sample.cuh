// Sampling from logits with temperature, top-k, top-p and min-p, from given random numbers.
//
// Weights are integers, w_i = floor(2^40 exp((l_i - l_max) / t)): sums do not depend on their order, so the token is the same whatever the
// cluster size, the batch around the row or the way the sums are split (in FP32, sums in another order move the borders of the
// distribution by 1e-7, and one row in a few hundred with a flat distribution draws its neighbour).
//
// A cluster of up to eight blocks works on a row.  Each block reads its part of the row once, keeps it in shared memory as FP32
// and takes part in
//   maximum -> (top-k, top-p: the cut, by digits of the ordered bits of the logits, with histograms that the blocks add up) -> sums of the
//   kept weights per warp -> the warp in whose part the random number falls finds the token.
// A cut is a pair (key, ties): kept are the tokens whose key is above it, and the first `ties` of those that have it.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>

#include "ptx.cuh"

namespace dsv4 {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleMaxCluster = 8;
constexpr int kSampleStep = 256;                 // elements a warp looks at at a time, eight neighbouring ones a lane
constexpr int kSampleOneBits = 40;               // weights are multiples of 2^-40

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int N, V;
    int warp_span;           // elements a warp owns, a multiple of kSampleStep: neighbouring ones, in the order of the vocabulary
    const float* u;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* token;
    float* logprob;
};

struct SampleShared {
    float max[kSampleMaxCluster];                                // written by every block of the cluster
    unsigned long long sum[kSampleMaxCluster * kSampleWarps];    // kept weight above the cut, per warp of the cluster
    uint32_t ties[kSampleMaxCluster * kSampleWarps];             // tokens at the cut
    unsigned long long hist[2][256];                             // this block's histogram of one digit, read by the others
    unsigned long long all[256];                                 // the cluster's
    unsigned long long digit_above;
    uint32_t digit;
    float warp_max[kSampleWarps];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_blocks() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void sts_cluster_u64(uint32_t caddr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(caddr), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned long long lds_cluster_u64(uint32_t caddr) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(caddr) : "memory");
    return v;
}

// Bits whose unsigned order is the order of the values.
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// What a row's settings come to.
struct SampleRow {
    float top;               // largest logit
    float per;               // 1 / temperature
    float min_p;             // 0: off
    int k;                   // 0: off
    int p24;                 // top-p in multiples of 2^-24, -1: off
    bool greedy;

    // exp((l - top) / t), in the operations and the order in which it is defined (no contraction, CUDA's expf)
    __device__ __forceinline__ float exponent(float l) const { return l == top ? 0.f : __fmul_rn(__fsub_rn(l, top), per); }
    __device__ __forceinline__ float ratio(float l) const { return expf(exponent(l)); }
    // floor(2^40 e) from the bits of e <= 1 (a conversion of the product to 64 bits takes four times as long)
    static __device__ __forceinline__ unsigned long long fixed(float e) {
        const uint32_t b = __float_as_uint(e), shift = 127u - (b >> 23);
        return (uint64_t((b & 0x7FFFFFu) | 0x800000u) << (kSampleOneBits - 23)) >> min(shift, 63u);
    }
    __device__ __forceinline__ unsigned long long weight(float l) const {
        const float e = ratio(l);
        return e >= min_p ? fixed(e) : 0ull;
    }
    __device__ __forceinline__ unsigned long long weight_unfiltered(float l) const { return fixed(ratio(l)); }
};

// floor(total * m / 2^24)
__device__ __forceinline__ unsigned long long share_of(unsigned long long total, uint32_t m) {
    return (total >> 24) * m + (((total & 0xFFFFFFull) * m) >> 24);
}
__device__ __forceinline__ uint32_t in_24_bits(float x) {       // floor(2^24 x), 0 for what is not in [0, 1]
    return x > 0.f ? uint32_t(fminf(x, 1.f) * 16777216.f) : 0u;
}

__device__ __forceinline__ float logit_value(float x) { return x; }
__device__ __forceinline__ float logit_value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float logit_value(__half x) { return __half2float(x); }
// NaN counts as -inf, and -0 as 0
__device__ __forceinline__ float clean_logit(float x) { return x == x ? x + 0.f : -CUDART_INF_F; }

// The row as a warp sees it: the elements it owns, eight a lane and step.
template <typename T, bool RESIDENT>
struct RowPart {
    const T* base;           // 16-byte aligned: element 0 is `lead` elements before the row's first
    int lead, end;           // the row is [lead, end)
    int first;               // the warp's first element
    float* kept;             // resident: the warp's elements as FP32, step by step, the lanes' first four and then their last four
    int lane;

    __device__ __forceinline__ int at(int step) const { return first + step * kSampleStep + lane * 8; }
    __device__ __forceinline__ void load(int step, float (&v)[8]) const {
        const int e = at(step);
        if (e >= lead && e + 8 <= end) {
            alignas(16) T x[8];
#pragma unroll
            for (int i = 0; i < int(sizeof(x) / 16); ++i) reinterpret_cast<uint4*>(x)[i] = ptx::ldg_stream_v4(reinterpret_cast<const uint4*>(base + e) + i);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = clean_logit(logit_value(x[i]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = e + i >= lead && e + i < end ? clean_logit(logit_value(ptx::ld(base + e + i))) : -CUDART_INF_F;
        }
    }
    __device__ __forceinline__ void keep(int step, const float (&v)[8]) const {
        float4* p = reinterpret_cast<float4*>(kept + step * kSampleStep) + lane;
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[32] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __device__ __forceinline__ void get(int step, float (&v)[8]) const {
        if constexpr (RESIDENT) {
            const float4* p = reinterpret_cast<const float4*>(kept + step * kSampleStep) + lane;
            const float4 a = p[0], b = p[32];
            v[0] = a.x;  v[1] = a.y;  v[2] = a.z;  v[3] = a.w;
            v[4] = b.x;  v[5] = b.y;  v[6] = b.z;  v[7] = b.w;
        } else {
            load(step, v);
        }
    }
};

__device__ __forceinline__ unsigned long long warp_total(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_upto(unsigned long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += y;
    }
    return v;
}

// One digit of a cut.  The blocks' histograms of bits [shift, shift + 8) have been filled; in descending order of the digit, the first one up to which
// at least `wanted` lies goes to sh.digit, what lies above it to sh.digit_above.  Returns the sum over all digits.  Every thread of the
// cluster calls.
__device__ __forceinline__ unsigned long long find_digit(SampleShared& sh, int buffer, unsigned long long wanted, uint32_t blocks) {
    ptx::cluster_sync();                           // (releases and acquires: every block's histogram is complete)
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < 256) {
        const uint32_t at = ptx::smem_u32(&sh.hist[buffer][tid]);
        unsigned long long s = 0;
        for (uint32_t b = 0; b < blocks; ++b) s += lds_cluster_u64(ptx::mapa(at, b));
        sh.all[255 - tid] = s;
    }
    __syncthreads();
    // all warps alike: lane l has the digits 255 - 8 l down to 248 - 8 l
    unsigned long long v[8], mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { v[i] = sh.all[lane * 8 + i];  mine += v[i]; }
    const unsigned long long upto = warp_upto(mine, lane);
    unsigned long long above = upto - mine;
    if (tid < 32 && above < wanted && upto >= wanted) {
        int i = 0;
        while (i < 7 && above + v[i] < wanted) above += v[i++];
        sh.digit = uint32_t(255 - (lane * 8 + i));
        sh.digit_above = above;
    }
    __syncthreads();
    return __shfl_sync(0xFFFFFFFFu, upto, 31);
}

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) float s_row[];
    __shared__ SampleShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank(), blocks = cluster_blocks();
    const int n = int(blockIdx.x / blocks);
    ptx::pdl_trigger();
    ptx::pdl_wait();
    // (the other blocks' shared memory may be written once they are there; that is waited for below)
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");

    const T* row = static_cast<const T*>(a.logits) + int64_t(n) * a.stride;
    RowPart<T, RESIDENT> part;
    part.lead = int((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    part.base = row - part.lead;
    part.end = part.lead + a.V;
    part.first = (int(rank) * kSampleWarps + warp) * a.warp_span;
    part.kept = s_row + warp * a.warp_span;
    part.lane = lane;
    const int steps = a.warp_span / kSampleStep;

    // ── maximum ──
    SampleRow r;
    r.top = -CUDART_INF_F;
#pragma unroll 4
    for (int s = 0; s < steps; ++s) {
        float v[8];
        part.load(s, v);
        if constexpr (RESIDENT) part.keep(s, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.top = fmaxf(r.top, v[i]);
    }
    const float t = a.temperature != nullptr ? ptx::ld(a.temperature + n) : 1.f;
    r.greedy = !(t > 0.f);
    r.per = r.greedy ? 1.f : __frcp_rn(t);
    const int k = a.top_k != nullptr ? ptx::ld(a.top_k + n) : 0;
    r.k = k > 0 && k < a.V ? k : 0;
    const float p = a.top_p != nullptr ? ptx::ld(a.top_p + n) : 1.f;
    r.p24 = p < 1.f ? int(in_24_bits(p)) : -1;
    const float mp = a.min_p != nullptr ? ptx::ld(a.min_p + n) : 0.f;
    r.min_p = mp > 0.f ? fminf(mp, 1.f) : 0.f;
    const uint32_t u24 = min(in_24_bits(ptx::ld(a.u + n)), 0xFFFFFFu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.top = fmaxf(r.top, __shfl_xor_sync(0xFFFFFFFFu, r.top, o));
    if (lane == 0) sh.warp_max[warp] = r.top;
    for (int i = tid; i < 512; i += kSampleThreads) (&sh.hist[0][0])[i] = 0ull;
    __syncthreads();
    r.top = sh.warp_max[lane & (kSampleWarps - 1)];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) r.top = fmaxf(r.top, __shfl_xor_sync(0xFFFFFFFFu, r.top, o));
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < int(blocks)) ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.max[rank]), tid), __float_as_uint(r.top));
    ptx::cluster_sync();
    for (uint32_t b = 0; b < blocks; ++b) r.top = fmaxf(r.top, sh.max[b]);
    if (r.top == -CUDART_INF_F) {                  // the same in every block: nothing to draw from
        if (rank == 0 && tid == 0) {
            a.token[n] = -1;
            if (a.logprob != nullptr) a.logprob[n] = -CUDART_INF_F;
        }
        return;
    }

    // ── the cut ──
    uint32_t cut = 0;                              // every key is above 0
    unsigned long long cut_ties = 0;
    int buffer = 0;
    auto clear = [&](int b) {
        __syncthreads();
        for (int i = tid; i < 256; i += kSampleThreads) sh.hist[b][i] = 0ull;
        __syncthreads();
    };
    if (r.greedy) {
        cut = order_key(r.top);
        cut_ties = 1;
    } else {
        if (r.k > 0) {
            unsigned long long wanted = (unsigned long long)(r.k);
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int s = 0; s < steps; ++s) {
                    float v[8];
                    part.get(s, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t key = order_key(v[i]);
                        if (shift == 24 || (key >> (shift + 8)) == (cut >> (shift + 8))) atomicAdd(&sh.hist[buffer][(key >> shift) & 255u], 1ull);
                    }
                }
                find_digit(sh, buffer, wanted, blocks);
                cut |= sh.digit << shift;
                wanted -= sh.digit_above;
                buffer ^= 1;
                clear(buffer);                     // (two uses ago: every block has read it, since it has come to the barrier of the last one)
            }
            cut_ties = wanted;
        }
        if (r.p24 >= 0) {
            const uint32_t above = cut;            // top-p looks at the tokens above top-k's cut, and at those of its ties that are kept
            unsigned long long most = 0, ahead = 0;
            uint32_t found = 0;
            bool inside = true;
            for (int shift = 24; shift >= 0 && inside; shift -= 8) {
                for (int s = 0; s < steps; ++s) {
                    float v[8];
                    part.get(s, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t key = order_key(v[i]);
                        if (key > above && (shift == 24 || (key >> (shift + 8)) == (found >> (shift + 8)))) {
                            const unsigned long long w = r.weight_unfiltered(v[i]);
                            if (w != 0ull) atomicAdd(&sh.hist[buffer][(key >> shift) & 255u], w);
                        }
                    }
                }
                if (shift == 24) {
                    // (the sum comes with the first digit, so that its search follows with the share known)
                    const unsigned long long over = find_digit(sh, buffer, 1ull, blocks);
                    const unsigned long long tie = cut_ties != 0ull ? r.weight_unfiltered(key_value(above)) : 0ull;
                    most = max(share_of(over + cut_ties * tie, uint32_t(r.p24)), 1ull);
                    if (most > over) {             // all above the cut, and some of the ties
                        cut_ties = min(cut_ties, (most - over + tie - 1ull) / tie);
                        inside = false;
                    } else {
                        find_digit(sh, buffer, most, blocks);
                    }
                } else {
                    find_digit(sh, buffer, most - ahead, blocks);
                }
                if (inside) {
                    found |= sh.digit << shift;
                    ahead += sh.digit_above;
                }
                buffer ^= 1;
                clear(buffer);
            }
            if (inside) {
                cut = found;
                const unsigned long long tie = r.weight_unfiltered(key_value(cut));
                cut_ties = (most - ahead + tie - 1ull) / tie;
            }
        }
    }

    // ── sums of the kept weights, per warp ──
    {
        unsigned long long sum = 0;
        uint32_t ties = 0;
        for (int s = 0; s < steps; ++s) {
            float v[8];
            part.get(s, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t key = order_key(v[i]);
                if (key > cut) sum += r.weight(v[i]);
                ties += key == cut;
            }
        }
        sum = warp_total(sum);
        ties = __reduce_add_sync(0xFFFFFFFFu, ties);
        if (lane < int(blocks)) {
            sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.sum[rank * kSampleWarps + warp]), lane), sum);
            ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.ties[rank * kSampleWarps + warp]), lane), ties);
        }
        ptx::cluster_sync();
    }

    // ── the warp that has the token (every warp finds out for itself) ──
    const unsigned long long tie_weight = cut_ties != 0ull ? r.weight(key_value(cut)) : 0ull;
    const int parts = int(blocks) * kSampleWarps, me = int(rank) * kSampleWarps + warp;
    unsigned long long sums[4], mine = 0, tie_before = 0;
    uint32_t ties[4], my_ties = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ties[i] = lane * 4 + i < parts ? sh.ties[lane * 4 + i] : 0u;
        my_ties += ties[i];
    }
    tie_before = warp_upto(my_ties, lane) - my_ties;
    unsigned long long my_tie_before = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned long long left = cut_ties > tie_before ? cut_ties - tie_before : 0ull;
        if (lane * 4 + i == me) my_tie_before = tie_before;
        tie_before += ties[i];
        sums[i] = lane * 4 + i < parts ? sh.sum[lane * 4 + i] + min(left, (unsigned long long)(ties[i])) * tie_weight : 0ull;
        mine += sums[i];
    }
    const unsigned long long upto = warp_upto(mine, lane), total = __shfl_sync(0xFFFFFFFFu, upto, 31);
    const unsigned long long target = share_of(total, u24);
    unsigned long long before = upto - mine, my_before = 0, my_sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (lane * 4 + i == me) { my_before = before;  my_sum = sums[i]; }
        before += sums[i];
    }
    my_before = __shfl_sync(0xFFFFFFFFu, my_before, me >> 2);
    my_sum = __shfl_sync(0xFFFFFFFFu, my_sum, me >> 2);
    my_tie_before = __shfl_sync(0xFFFFFFFFu, my_tie_before, me >> 2);
    if (target < my_before || target >= my_before + my_sum) return;

    unsigned long long run = my_before, tie_run = my_tie_before;
    for (int s = 0; s < steps; ++s) {
        float v[8];
        part.get(s, v);
        uint32_t here = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) here += order_key(v[i]) == cut;
        unsigned long long tie_at = tie_run + warp_upto(here, lane) - here, w[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t key = order_key(v[i]);
            w[i] = key > cut ? r.weight(v[i]) : 0ull;
            if (key == cut && tie_at++ < cut_ties) w[i] = tie_weight;
            sum += w[i];
        }
        const unsigned long long lane_upto = run + warp_upto(sum, lane);
        unsigned long long at = lane_upto - sum;
        if (target >= at && target < lane_upto) {
            int i = 0;
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (i == j && target >= at + w[j]) { at += w[j];  i = j + 1; }
            float x = v[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) x = i == j ? v[j] : x;
            a.token[n] = part.at(s) + i - part.lead;
            if (a.logprob != nullptr) a.logprob[n] = r.exponent(x) - logf(__ull2float_rn(total) * 9.094947017729282e-13f);
        }
        run = __shfl_sync(0xFFFFFFFFu, lane_upto, 31);
        tie_run = tie_run + __reduce_add_sync(0xFFFFFFFFu, here);
        if (target < run) return;
    }
}

}  // namespace dsv4
