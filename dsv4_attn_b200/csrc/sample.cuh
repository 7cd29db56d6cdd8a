// Sampling from logits with temperature, top-k, top-p and min-p, from given random numbers.
//
// Weights are integers, w_i = floor(2^40 exp((l_i - l_max) / t)): sums do not depend on their order, so the token is the same whatever the
// cluster size, the batch around the row or the way the sums are split (in FP32, sums in another order move the borders of the
// distribution by 1e-7, and one row in a few hundred with a flat distribution draws its neighbour).
//
// A block, or a cluster of up to four where there are few and long rows, works on a row; every warp owns neighbouring logits.  The row is read from DRAM once, for
// its maximum; what is looked at again comes from L1 or L2 (kept in shared memory, rows of 131,072 left room for clusters of eight blocks of 16,384 only,
// whose barriers cost more than the second reading: 1,024 rows, as first built, 302 us against 245).  Then
//   maximum -> (top-k, top-p: the cut) -> sums of the kept weights per warp -> the part of the row in which the random number falls, again by
//   warps -> the token.
// A cut is a pair (logit, ties): kept are the tokens above it, and the first `ties` of those that are equal to it.
//
// Top-k of up to 1,024 a block is sought among candidates: every thread has the largest of each quarter of its logits at hand, and where ceil(k / blocks)
// of a block's are at least x, at least k logits are, so that all logits from x on (some 2 k of them) hold the cut.  Only the quarters that have one are
// looked at again, and the token is found among them.
// Any other cut: a histogram over (l_max - l) / t in bins of 1/128, a count per bin, says where it should be (and, where min-p keeps less than that,
// that there is no need of it); what lies above is then summed exactly, and the logits of two and a half bins there are the candidates, those of the bins
// next to them if the exact sums say so.  Equal logits of sixteen bits are counted, not listed; what else is too much for the lists is gone through
// by digits of ordered bits.
//
// Bounds, at 1,024 rows of 131,072 BF16 logits (268 MB, 41 us at the measured copy rate): greedy rows, read once, 54 us; by temperature alone 125, 18
// instructions a logit, 14 of them expf and the sum, and 1,760 a warp whatever its row's length; top-p alone 255 to 315, 36 and 3,800 (a histogram, then that sum with the
// candidates); both with some 60 % of the issue slots in use, at 64 registers a thread, of which 72 to 152 bytes are spilled; top-k 50 71, with the chain of its short
// steps; a mixture of all 134.  A cut among thousands of nearly equal logits, found digit by digit, takes ten to twenty times as long as others.  A single row of 32,000: 9 us, of which the
// barriers and reads of its chain are nearly all.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>
#include <stdint.h>
#include <type_traits>

#include "ptx.cuh"

namespace dsv4 {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleMaxCluster = 4;
constexpr int kSampleStep = 256;                 // logits a warp looks at at a time, eight neighbouring ones a lane
constexpr int kSampleOneBits = 40;               // weights are multiples of 2^-40
constexpr int kSampleList = 2048;                // candidates
constexpr int kSampleShort = 256;                // candidates that are compared all with all
constexpr int kSampleBins = 4096;                // of the histogram over (l_max - l) / t,
constexpr float kSampleBin = 128.f;              // 1/128 each
constexpr uint32_t kSampleSpare = 64;            // candidates next to the bin of a cut
constexpr int kSampleQuarters = 4;               // a thread knows the largest logit of each quarter of its own
constexpr uint32_t kSampleMany = 300;            // within three bins of it: a part of a bin will do
constexpr int kSampleValues = 128;               // different logits, of sixteen bits, that may be near a cut
constexpr int kSampleMostTerms = 4095;           // of a FixedSum

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int N, V;
    bool heavy_first;        // blocks take the rows that take longest first
    const float* u;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* token;
    float* logprob;
};

struct SampleShared {
    // written by every block of the cluster, for itself
    float max[kSampleMaxCluster];
    uint32_t bound[kSampleMaxCluster];                           // a key that enough of its threads reach
    // of row_totals, in turn: a block may be at the next call while another still reads the results of one
    uint32_t found[2][kSampleMaxCluster];                        // candidates
    unsigned long long x[2][kSampleMaxCluster], y[2][kSampleMaxCluster];
    unsigned long long sum[kSampleMaxCluster * kSampleWarps];    // per warp: kept weight above the cut
    uint32_t ties[kSampleMaxCluster * kSampleWarps];             // and tokens at the cut
    // read by the other blocks
    unsigned long long hist[2][256];                             // one digit
    uint32_t bins[kSampleBins];
    unsigned long long list[kSampleList];                        // candidates: key << 32 | ~index
    // the block's own
    unsigned long long sorted[kSampleList];
    unsigned long long all[256];
    unsigned long long digit_above;
    unsigned long long warp_x[kSampleWarps], warp_y[kSampleWarps];
    float warp_max[kSampleWarps];
    uint32_t digit, count;
    int bin;
    float place;                                                 // where in that bin the cut should be
    float by_min_p;                                              // what lies above the logit that min-p asks for, by the histogram
    // the cut, from the first block to all
    uint32_t cut, kept, reached;                                 // reached: all of what was wanted lies up to it
    unsigned long long cut_ties;
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
// A rendezvous of all of the row's blocks, after which each sees what the others wrote.
__device__ __forceinline__ void sync_row(uint32_t blocks) {
    if (blocks > 1u) ptx::cluster_sync();
    else __syncthreads();
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

// A sum of floor(2^40 e), e <= 1: next to 4096 a 64-bit number counts in steps of 2^-40, and a sum that is rounded towards zero takes in of each e
// the whole steps.  A conversion and an addition a term (1,024 rows by temperature alone: 126 us, with two sums of 20 bits each in 32-bit numbers 135, with the
// conversion by shifts 132).  At most 4,095 terms.
struct FixedSum {
    double sum = 4096.0;
    __device__ __forceinline__ void add(float e) { sum = __dadd_rz(sum, double(e)); }
    // Two terms; each also to another sum where `too` says so.
    __device__ __forceinline__ void add2(float e0, float e1, FixedSum* other = nullptr, bool too0 = false, bool too1 = false) {
        const double d0 = e0, d1 = e1;
        sum = __dadd_rz(__dadd_rz(sum, d0), d1);
        if (other != nullptr) {
            if (too0) other->sum = __dadd_rz(other->sum, d0);
            if (too1) other->sum = __dadd_rz(other->sum, d1);
        }
    }
    __device__ __forceinline__ unsigned long long total() const { return static_cast<unsigned long long>(__double_as_longlong(sum) - __double_as_longlong(4096.0)); }
};
__device__ __forceinline__ unsigned long long fixed(float e) {
    FixedSum s;
    s.add(e);
    return s.total();
}
__device__ __forceinline__ float max_of(const float (&v)[8]) {
    return fmaxf(ptx::max3(ptx::max3(v[0], v[1], v[2]), v[3], v[4]), ptx::max3(v[5], v[6], v[7]));
}

// What a row's settings come to.
struct SampleRow {
    float top;               // largest logit
    float per;               // 1 / temperature
    float min_p;             // 0: off
    int k;                   // 0: off
    int p24;                 // top-p in multiples of 2^-24, -1: off
    bool greedy;

    // Infinite logits, or a temperature whose reciprocal is infinite: all tokens with the largest logit weigh 1, the others nothing.
    bool odd;

    // The exponent (l - top) / t of a logit, in the operations and the order of the definition; from -200 down, where NaN ends up as well, it makes no
    // difference any more.  Not for odd rows.
    __device__ __forceinline__ float exponent(float l) const { return fmaxf(__fmul_rn(__fsub_rn(l, top), per), -200.f); }
    __device__ __forceinline__ float ratio(float l) const { return expf(exponent(l)); }
    // of two logits, in packed operations
    __device__ __forceinline__ void exponents(float l0, float l1, float& x0, float& x1) const {
        const uint64_t d = ptx::add_f32x2(ptx::pack_f32x2(l0, l1), ptx::pack_f32x2(-top, -top));
        ptx::unpack_f32x2(ptx::mul_f32x2(d, ptx::pack_f32x2(per, per)), x0, x1);
        x0 = fmaxf(x0, -200.f);
        x1 = fmaxf(x1, -200.f);
    }
    __device__ __forceinline__ unsigned long long weight(float l) const {
        const float e = ratio(l);
        return e >= min_p ? fixed(e) : 0ull;
    }
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
template <typename T> __device__ __forceinline__ T no_logit();
template <> __device__ __forceinline__ float no_logit<float>() { return -CUDART_INF_F; }
template <> __device__ __forceinline__ __nv_bfloat16 no_logit<__nv_bfloat16>() { return __ushort_as_bfloat16(0xFF80); }
template <> __device__ __forceinline__ __half no_logit<__half>() { return __ushort_as_half(0xFC00); }

// A row, whose elements are counted from the 16-byte boundary at or before its start: it is [lead, end).
template <typename T>
struct LogitRow {
    static constexpr int kVecs = int(sizeof(T)) / 2;
    const T* base;
    int lead, end, lane;

    // The largest logit of this thread's, for the warp's `steps` steps from element `first` on; NaN left out, -inf where there is none.  Sixteen-bit logits
    // are compared two at a time.
    __device__ __forceinline__ float largest(int first, int steps) const {
        constexpr int kDeep = 8 / kVecs;         // loads in flight: 8 of 16 bytes
        float top = -CUDART_INF_F;
        int s = 0;
        // (the warp's first step may begin before the row, its last one end behind it)
        while (s < steps && first + s * kSampleStep < lead) top = fmaxf(top, largest_of_edge(first + s++ * kSampleStep + lane * 8));
        const int whole = max(s, min(steps, (end - first) / kSampleStep));
        Pair best[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) best[i] = none();
#pragma unroll 1
        for (; s < whole; s += kDeep) {
            uint4 x[kDeep][kVecs];
            const uint4* p = reinterpret_cast<const uint4*>(base + first + s * kSampleStep + lane * 8);
#pragma unroll
            for (int j = 0; j < kDeep; ++j)
#pragma unroll
                for (int i = 0; i < kVecs; ++i) {
                    x[j][i] = make_uint4(none().bits, none().bits, none().bits, none().bits);
                    if (s + j < whole) x[j][i] = ptx::ld(p + j * 32 * kVecs + i);
                }
#pragma unroll
            for (int j = 0; j < kDeep; ++j)
#pragma unroll
                for (int i = 0; i < kVecs; ++i) keep(best, x[j][i]);
        }
        s = whole;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, value(best[i]));
        for (; s < steps; ++s) top = fmaxf(top, largest_of_edge(first + s * kSampleStep + lane * 8));
        return top;
    }
    __device__ __forceinline__ float largest_of_edge(int e) const {
        float top = -CUDART_INF_F;
        for (int i = max(e, lead); i < min(e + 8, end); ++i) top = fmaxf(top, logit_value(ptx::ld(base + i)));
        return top;
    }
    // two 16-bit logits, or one of 32 bits
    struct Pair { uint32_t bits; };
    static __device__ __forceinline__ Pair none() { return {sizeof(T) == 4 ? 0xFF800000u : (sizeof(T) == 2 && is_bf16() ? 0xFF80FF80u : 0xFC00FC00u)}; }
    // Sixteen-bit logits: the bits of their keys from this one on say all.
    static constexpr int kKeyShift = std::is_same<T, __nv_bfloat16>::value ? 16 : 13;
    static __host__ __device__ constexpr bool is_bf16() { return std::is_same<T, __nv_bfloat16>::value; }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        uint32_t r;
        if constexpr (sizeof(T) == 4) r = __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
        else if constexpr (is_bf16()) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ void keep(Pair (&best)[4], const uint4& x) {
        best[0].bits = larger(best[0].bits, x.x);
        best[1].bits = larger(best[1].bits, x.y);
        best[2].bits = larger(best[2].bits, x.z);
        best[3].bits = larger(best[3].bits, x.w);
    }
    static __device__ __forceinline__ float value(Pair p) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(p.bits);
        else if constexpr (is_bf16()) return fmaxf(__uint_as_float(p.bits << 16), __uint_as_float(p.bits & 0xFFFF0000u));
        else { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p.bits));  return fmaxf(f.x, f.y); }
    }

    // Eight logits from e on, -inf where that is not of the row.
    __device__ __forceinline__ void load(int e, T (&x)[8]) const {
        if (e >= lead && e + 8 <= end) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(x)[i] = ptx::ld(reinterpret_cast<const uint4*>(base + e) + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = e + i >= lead && e + i < end ? ptx::ld(base + e + i) : no_logit<T>();
        }
    }
    // visit(v, e): the eight logits from e on, for the warp's `steps` steps from element `first` on; -inf where that is not of the row.  A step at a time,
    // with the next one on its way: what is done with a step takes longer than a load from L2, and with four steps in a loop body the instructions did not
    // come fast enough.
    template <typename Visit>
    __device__ __forceinline__ void each(int first, int steps, Visit visit) const {
        if (steps <= 0) return;
        int e = first + lane * 8;
        alignas(16) T next[8];
        load(e, next);
#pragma unroll 1
        for (int s = 0; s < steps; ++s, e += kSampleStep) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = logit_value(next[i]);
            if (s + 1 < steps) load(e + kSampleStep, next);
            visit(v, e);
            __syncwarp();                          // (lanes that had more to do: the next loads go out together again)
        }
    }
};

__device__ __forceinline__ unsigned long long warp_total(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ uint32_t warp_upto32(uint32_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += y;
    }
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

// Two sums over the row, and the blocks' counts of candidates.  `turn` changes with every call.  Every thread of the cluster calls.
__device__ __forceinline__ void row_totals(SampleShared& sh, uint32_t blocks, uint32_t rank, int& turn, unsigned long long& x, unsigned long long& y) {
    turn ^= 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    x = warp_total(x);
    y = warp_total(y);
    if (lane == 0) { sh.warp_x[warp] = x;  sh.warp_y[warp] = y; }
    __syncthreads();
    if (warp == 0) {
        x = warp_total(lane < kSampleWarps ? sh.warp_x[lane] : 0ull);
        y = warp_total(lane < kSampleWarps ? sh.warp_y[lane] : 0ull);
        if (lane < int(blocks)) {
            ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.found[turn][rank]), lane), sh.count);
            sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.x[turn][rank]), lane), x);
            sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.y[turn][rank]), lane), y);
        }
    }
    sync_row(blocks);
    x = y = 0ull;
    for (uint32_t b = 0; b < blocks; ++b) { x += sh.x[turn][b];  y += sh.y[turn][b]; }
}

// One digit of a cut.  The blocks' histograms of one digit have been filled; in descending order of the digit, the first one up to which
// at least `wanted` lies goes to sh.digit, what lies above it to sh.digit_above.  Every thread of the cluster calls.
__device__ __forceinline__ void find_digit(SampleShared& sh, int buffer, unsigned long long wanted, uint32_t blocks) {
    sync_row(blocks);
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < 256) {
        const uint32_t at = ptx::smem_u32(&sh.hist[buffer][tid]);
        unsigned long long s = 0;
        for (uint32_t b = 0; b < blocks; ++b) s += lds_cluster_u64(ptx::mapa(at, b));
        sh.all[255 - tid] = s;
    }
    __syncthreads();
    if (tid < 32) {
        // lane l has the digits 255 - 8 l down to 248 - 8 l
        unsigned long long v[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i] = sh.all[lane * 8 + i];  mine += v[i]; }
        const unsigned long long upto = warp_upto(mine, lane);
        unsigned long long above = upto - mine;
        if (above < wanted && upto >= wanted) {
            int i = 0;
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (i == j && above + v[j] < wanted) { above += v[j];  i = j + 1; }
            sh.digit = uint32_t(255 - (lane * 8 + i));
            sh.digit_above = above;
        }
    }
    __syncthreads();
}

// sh.sorted[0, n) into descending order, by way of sh.list: 2,048 buckets over the range of the logits, and within a bucket by comparing all with all
// (there are two or three in one, unless many logits are equal).  A bitonic network took 4 us for 200 candidates and 26 for 1,400, this 2 to 3.
// Every thread of the block calls.
__device__ __forceinline__ void sort_list(SampleShared& sh, int n) {
    constexpr int kBuckets = 2048, kPer = kBuckets / kSampleThreads, kMine = kSampleList / kSampleThreads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (n <= kSampleShort) {
        // a few: all with all
        const unsigned long long c = tid < n ? sh.sorted[tid] : 0ull;
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += sh.sorted[j] > c;
        __syncthreads();
        if (tid < n) sh.sorted[rank] = c;
        __syncthreads();
        return;
    }
    uint32_t* const count = sh.bins;
    uint32_t* const start = sh.bins + kBuckets;
    for (int i = tid; i < kBuckets; i += kSampleThreads) count[i] = 0u;
    uint32_t top = 0u, bottom = 0xFFFFFFFFu;
    unsigned long long mine[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (tid + i * kSampleThreads < n) {
            mine[i] = sh.sorted[tid + i * kSampleThreads];
            top = max(top, uint32_t(mine[i] >> 32));
            bottom = min(bottom, uint32_t(mine[i] >> 32));
        }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    bottom = __reduce_min_sync(0xFFFFFFFFu, bottom);
    if (lane == 0) sh.warp_x[warp] = (static_cast<unsigned long long>(top) << 32) | bottom;
    __syncthreads();
    {
        const unsigned long long x = sh.warp_x[lane & (kSampleWarps - 1)];
        top = __reduce_max_sync(0xFFFFFFFFu, uint32_t(x >> 32));
        bottom = __reduce_min_sync(0xFFFFFFFFu, uint32_t(x));
    }
    // (never decreasing as the logit falls; evenly over the logits, not over their bits, which are denser towards 0)
    const float highest = key_value(top), scale = float(kBuckets - 1) / fmaxf(highest - key_value(bottom), 1e-30f);
    auto bucket_of = [&](unsigned long long c) { return min(uint32_t((highest - key_value(uint32_t(c >> 32))) * scale), uint32_t(kBuckets - 1)); };
    uint32_t place[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (tid + i * kSampleThreads < n) place[i] = atomicAdd(&count[bucket_of(mine[i])], 1u);
    __syncthreads();
    uint32_t c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { c[i] = count[tid * kPer + i];  sum += c[i]; }
    uint32_t at = warp_upto32(sum, lane);
    if (lane == 31) sh.warp_y[warp] = at;
    __syncthreads();
    at -= sum;
#pragma unroll
    for (int w = 0; w < kSampleWarps - 1; ++w) at += w < warp ? uint32_t(sh.warp_y[w]) : 0u;
#pragma unroll
    for (int i = 0; i < kPer; ++i) { start[tid * kPer + i] = at;  at += c[i]; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (tid + i * kSampleThreads < n) sh.list[start[bucket_of(mine[i])] + place[i]] = mine[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (tid + i * kSampleThreads < n) {
            const uint32_t bucket = bucket_of(mine[i]), from = start[bucket], m = count[bucket];
            uint32_t rank = 0;
            if (m > 1u)
                for (uint32_t j = 0; j < m; ++j) rank += sh.list[from + j] > mine[i];
            sh.sorted[from + rank] = mine[i];
        }
    __syncthreads();
}

// A logit goes to the block's list.  (+ 0: -0 is 0)
__device__ __forceinline__ void list_logit(SampleShared& sh, float l, int index) {
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < uint32_t(kSampleList)) sh.list[at] = (static_cast<unsigned long long>(order_key(l + 0.f)) << 32) | uint32_t(~index);
}

// take(v[i], i) for the bits of `here`, a lane's eight logits: there are one or two in a warp's 256, so a short loop takes less than eight tests in a row do.
template <typename Take>
__device__ __forceinline__ void each_of(uint32_t here, const float (&v)[8], Take take) {
#pragma unroll 1
    for (; here != 0u; here &= here - 1u) {
        const int i = __ffs(here) - 1;
        const float a = (i & 1) ? v[1] : v[0], b = (i & 1) ? v[3] : v[2], c = (i & 1) ? v[5] : v[4], d = (i & 1) ? v[7] : v[6];
        const float low = (i & 2) ? b : a, high = (i & 2) ? d : c;
        take((i & 4) ? high : low, i);
    }
}

// How many candidates the lists have (-1: too many), after row_totals.
__device__ __forceinline__ int listed(const SampleShared& sh, uint32_t blocks, int turn) {
    int n = 0;
    for (uint32_t b = 0; b < blocks; ++b) n += int(min(sh.found[turn][b], uint32_t(kSampleList) + 1u));
    return n <= kSampleList ? n : -1;
}

// The cut among the candidates of all blocks (n of them, in sh.sorted afterwards, in descending order): the first k, and of those the ones before which less
// than `most` lies (0: the share of the k that top-p says).  To sh.cut, sh.cut_ties and sh.kept.  Every thread of the first block calls.
__device__ __forceinline__ void cut_of_list(SampleShared& sh, const SampleRow& r, uint32_t blocks, int turn, int n, int k, unsigned long long most) {
    constexpr int kPer = kSampleList / kSampleThreads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) sh.reached = 0u;
    for (int i = tid; i < n; i += kSampleThreads) {
        uint32_t b = 0, at = uint32_t(i);
        while (at >= sh.found[turn][b]) at -= sh.found[turn][b++];
        sh.sorted[i] = blocks > 1u ? lds_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.list[at]), b)) : sh.list[at];
    }
    __syncthreads();
    sort_list(sh, n);
    unsigned long long w[kPer], mine = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = tid * kPer + i;
        w[i] = at < k ? fixed(r.ratio(key_value(uint32_t(sh.sorted[at] >> 32)))) : 0ull;
        mine += w[i];
    }
    unsigned long long ahead = warp_upto(mine, lane) - mine;
    if (lane == 31) sh.warp_x[warp] = ahead + mine;
    __syncthreads();
    const unsigned long long of_warp = lane < kSampleWarps ? sh.warp_x[lane] : 0ull, upto = warp_upto(of_warp, lane);
    if (most == 0ull) most = max(share_of(__shfl_sync(0xFFFFFFFFu, upto, 31), uint32_t(r.p24)), 1ull);
    ahead += __shfl_sync(0xFFFFFFFFu, upto - of_warp, warp);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = tid * kPer + i;
        const bool kept = at < k && ahead < most;
        ahead += w[i];
        if (kept && (at + 1 >= k || ahead >= most)) {              // the last one kept
            const uint32_t key = uint32_t(sh.sorted[at] >> 32);
            int lo = 0, hi = at;                                   // the first one with its key
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (uint32_t(sh.sorted[mid] >> 32) > key) lo = mid + 1;
                else hi = mid;
            }
            sh.cut = key;
            sh.cut_ties = static_cast<unsigned long long>(at - lo + 1);
            sh.kept = uint32_t(at + 1);
            sh.reached = most == ~0ull || ahead >= most;
        }
    }
    __syncthreads();
    if (tid > 0 && tid < int(blocks)) {
        ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.cut), tid), sh.cut);
        ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.kept), tid), sh.kept);
        ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.reached), tid), sh.reached);
        sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.cut_ties), tid), sh.cut_ties);
    }
}

// The token among the sh.kept candidates at the front of sh.sorted: the weights of 256 equal parts of the vocabulary say in which part it is, and those of its
// part are compared with one another.  Every thread of the first block calls.
__device__ __forceinline__ void token_of_list(SampleShared& sh, const SampleRow& r, const SampleArgs& a, int n, uint32_t u24) {
    constexpr int kMine = kSampleList / kSampleThreads;
    const int tid = threadIdx.x, lane = tid & 31, kept = int(sh.kept), shift = max(24 - __clz(a.V), 0);      // V >> shift < 256
    if (kept <= kSampleShort) {
        // a few: a thread each adds up what the others of lower index weigh
        float x = 0.f;
        unsigned long long w = 0;
        uint32_t index = 0;
        if (tid < kept) {
            const unsigned long long c = sh.sorted[tid];
            x = r.exponent(key_value(uint32_t(c >> 32)));
            const float e = expf(x);
            w = e >= r.min_p ? fixed(e) : 0ull;
            index = ~uint32_t(c);
            sh.all[tid] = w;
        }
        __syncthreads();
        if (tid >= kept) return;
        unsigned long long total = 0, before = 0;
#pragma unroll 4
        for (int j = 0; j < kept; ++j) {
            const unsigned long long wj = sh.all[j];
            total += wj;
            before += ~uint32_t(sh.sorted[j]) < index ? wj : 0ull;
        }
        const unsigned long long target = share_of(total, u24);
        if (target >= before && target < before + w) {
            a.token[n] = int(index);
            if (a.logprob != nullptr) a.logprob[n] = x - logf(__ull2float_rn(total) * 9.094947017729282e-13f);
        }
        return;
    }
    if (tid < 256) sh.all[tid] = 0ull;
    if (tid == 0) sh.count = 0u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (tid + i * kSampleThreads < kept) {
            const unsigned long long c = sh.sorted[tid + i * kSampleThreads];
            const float e = r.ratio(key_value(uint32_t(c >> 32)));
            if (e >= r.min_p) atomicAdd(&sh.all[~uint32_t(c) >> shift], fixed(e));
        }
    __syncthreads();
    unsigned long long v[8], sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { v[i] = sh.all[lane * 8 + i];  sum += v[i]; }
    const unsigned long long upto = warp_upto(sum, lane), total = __shfl_sync(0xFFFFFFFFu, upto, 31), target = share_of(total, u24);
    unsigned long long before = upto - sum;
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, target >= before && target < upto);
    int part = 0;
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (part == i && target >= before + v[i]) { before += v[i];  part = i + 1; }
    const int from = __ffs(hit) - 1;
    part = from * 8 + __shfl_sync(0xFFFFFFFFu, part, from);
    before = __shfl_sync(0xFFFFFFFFu, before, from);
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (tid + i * kSampleThreads < kept) {
            const unsigned long long c = sh.sorted[tid + i * kSampleThreads];
            if (int(~uint32_t(c) >> shift) == part) sh.list[atomicAdd(&sh.count, 1u)] = c;
        }
    __syncthreads();
    const int m = int(sh.count);
    for (int i = tid; i < m; i += kSampleThreads) {
        const uint32_t index = ~uint32_t(sh.list[i]);
        unsigned long long at = before, w = 0;
        float l = 0.f;
        for (int j = 0; j < m; ++j) {
            const unsigned long long c = sh.list[j];
            if (~uint32_t(c) > index) continue;
            const float lj = key_value(uint32_t(c >> 32)), e = r.ratio(lj);
            const unsigned long long wj = e >= r.min_p ? fixed(e) : 0ull;
            if (j == i) { w = wj;  l = lj; }
            else at += wj;
        }
        if (target >= at && target < at + w) {
            a.token[n] = int(index);
            if (a.logprob != nullptr) a.logprob[n] = r.exponent(l) - logf(__ull2float_rn(total) * 9.094947017729282e-13f);
        }
    }
}

// The token among up to kSampleShort candidates (n of them, in the lists of all blocks), of which the first k and top-p's share are kept: a thread has one, and
// adds up what comes before it, in their order for the cut and in the vocabulary's for the token.  Every thread of the first block calls; `read` is called when the
// lists have been read.
template <typename Read>
__device__ __forceinline__ void token_of_few(SampleShared& sh, const SampleRow& r, const SampleArgs& a, uint32_t blocks, int turn, int n, int k, int row, uint32_t u24, Read read) {
    const int tid = threadIdx.x;
    unsigned long long c = 0, w = 0;
    float x = 0.f, e = 0.f;
    if (tid < n) {
        uint32_t b = 0, at = uint32_t(tid);
        while (at >= sh.found[turn][b]) at -= sh.found[turn][b++];
        c = blocks > 1u ? lds_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.list[at]), b)) : sh.list[at];
        x = r.exponent(key_value(uint32_t(c >> 32)));
        e = expf(x);
        w = fixed(e);
        sh.sorted[tid] = c;
        sh.all[tid] = w;
    }
    __syncthreads();
    read();
    int rank = 0;
    unsigned long long before = 0;
    if (tid < n) {
#pragma unroll 4
        for (int j = 0; j < n; ++j) {
            const bool first = sh.sorted[j] > c;
            rank += first;
            before += first ? sh.all[j] : 0ull;
        }
        if (rank == k - 1) sh.digit_above = before + w;
    }
    __syncthreads();
    if (tid < n) {
        if (rank >= k || (r.p24 >= 0 && before >= max(share_of(sh.digit_above, uint32_t(r.p24)), 1ull)) || e < r.min_p) w = 0ull;
        sh.all[tid] = w;
    }
    __syncthreads();
    if (w == 0ull) return;
    const uint32_t index = ~uint32_t(c);
    unsigned long long total = 0;
    before = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
        const unsigned long long wj = sh.all[j];
        total += wj;
        before += ~uint32_t(sh.sorted[j]) < index ? wj : 0ull;
    }
    const unsigned long long target = share_of(total, u24);
    if (target >= before && target < before + w) {
        a.token[row] = int(index);
        if (a.logprob != nullptr) a.logprob[row] = x - logf(__ull2float_rn(total) * 9.094947017729282e-13f);
    }
}

// The row at place `at` where those that take longest, with a cut that no list of candidates gives (top-p alone, a large top-k), come first: they take three
// times as long, and one that is begun last is waited for by the whole call (1,024 rows, one in five of them, at a time when they took a sixth longer: 169 us, heavy ones first 157).  Every block looks at all rows' settings.
__device__ __forceinline__ int row_in_order(SampleShared& sh, const SampleArgs& a, int at) {
    uint32_t* const flags = sh.bins;
    const int lane = threadIdx.x & 31;
    // (two rows a thread at a time, their settings on the way together: one after the other, and only as far as needed, they took 2 us)
    for (int n0 = int(threadIdx.x) - lane; n0 < a.N; n0 += 2 * kSampleThreads) {
        float t[2], p[2];
        int k[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int n = min(n0 + i * kSampleThreads + lane, a.N - 1);
            t[i] = a.temperature != nullptr ? ptx::ld(a.temperature + n) : 1.f;
            k[i] = a.top_k != nullptr ? ptx::ld(a.top_k + n) : 0;
            p[i] = a.top_p != nullptr ? ptx::ld(a.top_p + n) : 1.f;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool heavy = t[i] > 0.f && (k[i] <= 0 || k[i] >= a.V ? p[i] < 1.f : k[i] > kSampleThreads * kSampleQuarters / 2);
            const uint32_t b = __ballot_sync(0xFFFFFFFFu, heavy && n0 + i * kSampleThreads + lane < a.N);
            if (lane == 0 && n0 + i * kSampleThreads < a.N) flags[(n0 + i * kSampleThreads) >> 5] = b;
        }
    }
    __syncthreads();
    // every warp for itself: the words in runs, one a lane
    const int words = (a.N + 31) / 32, run = (words + 31) / 32, from = lane * run, to = min(from + run, words);
    int heavy = 0;
    for (int w = from; w < to; ++w) heavy += __popc(flags[w]);
    int before = int(warp_upto32(uint32_t(heavy), lane)) - heavy;
    const int all = __shfl_sync(0xFFFFFFFFu, before + heavy, 31);
    const bool want = at < all;
    if (!want) at -= all;
    int rows_before = min(from * 32, a.N);
    if (!want) {                                   // the light ones
        before = rows_before - before;
        heavy = min(to * 32, a.N) - rows_before - heavy;
    }
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, to > from && at >= before && at < before + heavy);
    int row = 0;
    if (to > from && at >= before && at < before + heavy)
        for (int w = from; w < to; ++w) {
            uint32_t bits = want ? flags[w] : ~flags[w];
            if (w * 32 + 32 > a.N) bits &= (1u << (a.N & 31)) - 1u;
            const int c = __popc(bits);
            if (at < before + c) {
                row = w * 32 + int(__fns(bits, 0, at - before + 1));
                break;
            }
            before += c;
        }
    row = __shfl_sync(0xFFFFFFFFu, row, __ffs(hit) - 1);
    __syncthreads();                               // (the flags lie where the histogram will)
    return row;
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
    extern __shared__ __align__(16) uint8_t s_sample[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(s_sample);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_rank(), blocks = cluster_blocks();
    int n = int(blockIdx.x / blocks);
    ptx::pdl_trigger();
    ptx::pdl_wait();
    if (a.heavy_first) n = row_in_order(sh, a, n);
    // (the other blocks' shared memory may be written once they are there; that is waited for below)
    if (blocks > 1u) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");

    const T* start = static_cast<const T*>(a.logits) + int64_t(n) * a.stride;
    LogitRow<T> row;
    row.lead = int((reinterpret_cast<uintptr_t>(start) & 15u) / sizeof(T));
    row.base = start - row.lead;
    row.end = row.lead + a.V;
    row.lane = lane;
    // The row's steps are dealt out evenly: every warp of the cluster has neighbouring ones, in the order of the vocabulary.
    const int row_steps = (row.end + kSampleStep - 1) / kSampleStep, parts = int(blocks) * kSampleWarps, me = int(rank) * kSampleWarps + warp;
    auto first_step = [&](int part) { return row_steps * part / parts; };       // (at most 16,385 steps and 64 parts)
    const int first = first_step(me) * kSampleStep, steps = first_step(me + 1) - first_step(me);

    // ── maximum ──
    float quarter[kSampleQuarters], mine = -CUDART_INF_F;
    auto quarter_step = [&](int q) { return steps * q / kSampleQuarters; };
#pragma unroll
    for (int q = 0; q < kSampleQuarters; ++q) {
        quarter[q] = row.largest(first + quarter_step(q) * kSampleStep, quarter_step(q + 1) - quarter_step(q));
        mine = fmaxf(mine, quarter[q]);
    }
    SampleRow r;
    const float t = a.temperature != nullptr ? ptx::ld(a.temperature + n) : 1.f;
    r.greedy = !(t > 0.f);
    r.per = r.greedy ? 1.f : fmaxf(__frcp_rn(t), __uint_as_float(1u));      // (an infinite temperature: -inf has to stay below all)
    const int k = a.top_k != nullptr ? ptx::ld(a.top_k + n) : 0;
    r.k = k > 0 && k < a.V ? k : 0;
    const float p = a.top_p != nullptr ? ptx::ld(a.top_p + n) : 1.f;
    r.p24 = p < 1.f ? int(in_24_bits(p)) : -1;
    const float mp = a.min_p != nullptr ? ptx::ld(a.min_p + n) : 0.f;
    r.min_p = mp > 0.f ? fminf(mp, 1.f) : 0.f;
    const uint32_t u24 = min(in_24_bits(ptx::ld(a.u + n)), 0xFFFFFFu);
    r.top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.top = fmaxf(r.top, __shfl_xor_sync(0xFFFFFFFFu, r.top, o));
    if (lane == 0) sh.warp_max[warp] = r.top;
    if (tid == 0) { sh.count = sh.digit = 0u;  sh.kept = 0x7FFFFFFFu; }
    __syncthreads();
    // a key that enough threads' largest logits reach: from the top, a bit at a time
    const int groups = (r.k + int(blocks) - 1) / int(blocks);
    // (a quarter of the threads, or half of their quarters: more would bring the bound down to logits that most of them exceed several times, and the
    // lists would not hold the candidates)
    const bool by_list = !r.greedy && r.k > 0 && groups <= kSampleThreads * kSampleQuarters / 2;
    uint32_t bound = 0u;
    if (by_list) {
        const bool few = groups <= kSampleThreads / 4;
        const uint32_t key = order_key(mine);
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit >= 0x8000u; bit >>= 1) {
            int reach = __syncthreads_count((few ? key : order_key(quarter[0])) >= (bound | bit));
            if (!few)
#pragma unroll
                for (int q = 1; q < kSampleQuarters; ++q) reach += __syncthreads_count(order_key(quarter[q]) >= (bound | bit));
            if (reach >= groups) {
                bound |= bit;
                if (reach <= groups + groups / 8 + 4) break;                     // (near enough)
            }
        }
    }
    r.top = sh.warp_max[lane & (kSampleWarps - 1)];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) r.top = fmaxf(r.top, __shfl_xor_sync(0xFFFFFFFFu, r.top, o));
    if (blocks > 1u) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        if (tid < int(blocks)) {
            ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.max[rank]), tid), __float_as_uint(r.top));
            ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.bound[rank]), tid), bound);
        }
        ptx::cluster_sync();
        for (uint32_t b = 0; b < blocks; ++b) {
            r.top = fmaxf(r.top, sh.max[b]);
            bound = min(bound, sh.bound[b]);
        }
    }
    if (r.top == -CUDART_INF_F) {                  // the same in every block: nothing to draw from
        if (rank == 0 && tid == 0) {
            a.token[n] = -1;
            if (a.logprob != nullptr) a.logprob[n] = -CUDART_INF_F;
        }
        return;
    }
    r.odd = r.top == CUDART_INF_F || r.per == CUDART_INF_F;
    if (r.greedy) {
        // the lowest index of the largest logit
        constexpr int kDeep = 4;
#pragma unroll 1
        for (int q = 0; q < kSampleQuarters; ++q) {
            const int from = first + quarter_step(q) * kSampleStep + lane * 8, many = quarter_step(q + 1) - quarter_step(q);
            if (!(q == 0 ? quarter[0] == r.top : q == 1 ? quarter[1] == r.top : q == 2 ? quarter[2] == r.top : quarter[3] == r.top)) continue;
#pragma unroll 1
            for (int s = 0; s < many; s += kDeep) {
                alignas(16) T x[kDeep][8];
#pragma unroll
                for (int d = 0; d < kDeep; ++d)
                    if (s + d < many) row.load(from + (s + d) * kSampleStep, x[d]);
#pragma unroll
                for (int d = kDeep - 1; d >= 0; --d)
#pragma unroll
                    for (int i = 7; i >= 0; --i)
                        if (s + d < many && logit_value(x[d][i]) == r.top) atomicMin(&sh.kept, uint32_t(from + (s + d) * kSampleStep + i - row.lead));
            }
        }
        __syncthreads();
        uint32_t token = sh.kept;
        if (blocks > 1u) {
            if (tid == 0) ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.found[0][rank]), 0), token);
            ptx::cluster_sync();
            for (uint32_t b = 0; b < blocks; ++b) token = min(token, sh.found[0][b]);
        }
        if (rank == 0 && tid == 0) {
            a.token[n] = int(token);
            if (a.logprob != nullptr) a.logprob[n] = 0.f;
        }
        return;
    }

    // ── the cut ──
    uint32_t cut = 0;                              // a key; every key is above 0
    unsigned long long cut_ties = 0;
    int turn = 0;
    bool sums_known = false;                       // of the kept weights, per warp
    auto part_of = [&](int index) { return (((index + row.lead) / kSampleStep + 1) * parts - 1) / row_steps; };
    bool have_cut = r.k == 0 && r.p24 < 0;
    if (r.odd) {
        // the tokens with the largest logit, of equal weight, as far as the filters let them
        uint32_t mine_count = 0;
        row.each(first, steps, [&](const float (&v)[8], int) {
#pragma unroll
            for (int i = 0; i < 8; ++i) mine_count += v[i] == r.top;
        });
        unsigned long long x = mine_count, y = 0;
        row_totals(sh, blocks, rank, turn, x, y);
        cut = order_key(r.top + 0.f);
        cut_ties = r.k > 0 ? min(x, static_cast<unsigned long long>(r.k)) : x;
        if (r.p24 >= 0) cut_ties = min(cut_ties, (max(share_of(cut_ties << kSampleOneBits, uint32_t(r.p24)), 1ull) + (1ull << kSampleOneBits) - 1ull) >> kSampleOneBits);
        have_cut = true;
    } else if (by_list) {
        const float from = fmaxf(key_value(bound), -3.402823466e38f);       // (-inf is no candidate)
        // The quarters that have a candidate go to a list (first element and steps), and all threads share out their eights of logits: each waits for one or
        // two loads.
        uint2* const hits = reinterpret_cast<uint2*>(sh.sorted);
#pragma unroll
        for (int q = 0; q < kSampleQuarters; ++q)
            if (quarter[q] >= from)
                hits[atomicAdd(&sh.digit, 1u)] = make_uint2(uint32_t(first + quarter_step(q) * kSampleStep + lane * 8), uint32_t(quarter_step(q + 1) - quarter_step(q)));
        __syncthreads();
        const int most = (row_steps / parts + 1 + kSampleQuarters - 1) / kSampleQuarters, shift = 32 - __clz(most - 1);     // steps of a quarter at most, as a power of two
        // (with one in four of them on the list the row is swept instead: eights here and there are read at half a sector each, 1,100 quarters of a row of 131,072
        // in 31 us, the row in 21)
        const bool sweep = int(sh.digit) > kSampleThreads * kSampleQuarters / 4;
        const int eights = sweep ? 0 : int(sh.digit) << shift;
        if (sweep)
            row.each(first, steps, [&](const float (&v)[8], int e) {
                if (max_of(v) < from) return;
                uint32_t here = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) here |= uint32_t(v[j] >= from) << j;
                each_of(here, v, [&](float l, int j) { list_logit(sh, l, e + j - row.lead); });
            });
        constexpr int kDeep = 4;
#pragma unroll 1
        for (int i0 = tid; i0 - tid < eights; i0 += kDeep * kSampleThreads) {
            alignas(16) T x[kDeep][8];
            int e[kDeep];
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                const int i = i0 + d * kSampleThreads, step = i & ((1 << shift) - 1);
                e[d] = -1;
                if (i < eights) {
                    const uint2 hit = hits[i >> shift];
                    if (step < int(hit.y)) e[d] = int(hit.x) + step * kSampleStep;
                }
                if (e[d] >= 0) row.load(e[d], x[d]);
            }
#pragma unroll
            for (int d = 0; d < kDeep; ++d) {
                float v[8];
                uint32_t here = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = logit_value(x[d][j]);
                    here |= uint32_t(v[j] >= from) << j;
                }
                if (e[d] < 0) here = 0u;
                each_of(here, v, [&](float l, int j) { list_logit(sh, l, e[d] + j - row.lead); });
            }
        }
        if (blocks > 1u) {
            unsigned long long x = 0, y = 0;
            row_totals(sh, blocks, rank, turn, x, y);
        } else {
            __syncthreads();
            if (tid == 0) sh.found[turn][0] = sh.count;
            __syncthreads();
        }
        const int m = listed(sh, blocks, turn);
        if (m >= 0 && m <= kSampleShort) {
            // (the other blocks may leave when their lists have been read)
            if (rank == 0)
                token_of_few(sh, r, a, blocks, turn, m, min(r.k, m), n, u24, [&] {
                    if (blocks > 1u) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
                });
            else asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
            __syncwarp();
            if (blocks > 1u) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
            return;
        }
        if (m >= 0) {
            if (rank == 0) cut_of_list(sh, r, blocks, turn, m, min(r.k, m), r.p24 < 0 ? ~0ull : 0ull);
            sync_row(blocks);                      // (the lists have been read)
            if (rank == 0) token_of_list(sh, r, a, n, u24);
            return;
        }
    }
    if (!have_cut) {
        // min-p keeps all of what a cut keeps (with room for the rounding of expf)
        auto min_p_idle = [&](uint32_t key) { return r.min_p == 0.f || r.ratio(key_value(key)) >= r.min_p * 1.0001f; };
        // The cut up to which `wanted` lies, among the finite logits above `above` (a key): tokens, or weight, of which `wanted` is then the share that
        // top-p says of all of it and of `ties`, the weight of the tokens kept at `above`.  False: it lies beyond (in the ties; no cut at all).
        auto find_cut = [&](auto weights, auto limited, uint32_t above, unsigned long long wanted, unsigned long long ties, unsigned long long& over) -> bool {
            constexpr bool BY_WEIGHT = decltype(weights)::value, by_weight = BY_WEIGHT, LIMITED = decltype(limited)::value;
            constexpr bool all_in = BY_WEIGHT && !LIMITED;                         // (-inf weighs nothing)
            const float above_value = LIMITED ? key_value(above) : -CUDART_INF_F;
            for (int i = tid; i < kSampleBins; i += kSampleThreads) sh.bins[i] = 0u;
            __syncthreads();
            // Bin of a logit: 1, its distance in bins and `off`, rounded to a whole number by the addition of 2^23.  (Near enough: what is decided
            // by it is checked with the exact sums.)  The last bin is for what is further away, and left out below.
            const float slope = -kSampleBin * r.per, offset = fmaf(-slope, r.top, 8388609.f), off = fmaf(slope, r.top, offset - 8388609.f);
            row.each(first, steps, [&](const float (&v)[8], int) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t bin = __float_as_uint(fminf(fmaf(v[i], slope, offset), 8388608.f + kSampleBins - 1)) & (kSampleBins - 1);
                    if (!LIMITED || v[i] > above_value) atomicAdd(&sh.bins[bin], 1u);
                }
            });
            sync_row(blocks);
            uint32_t* const counts = reinterpret_cast<uint32_t*>(sh.sorted);       // of the row
            if (blocks > 1u) {
                // every block adds up a part of the bins, and tells the others
                const int share = kSampleBins / int(blocks);
                for (int i = tid; i < share; i += kSampleThreads) {
                    const int bin = int(rank) * share + i;
                    uint32_t c = 0;
                    for (uint32_t b = 0; b < blocks; ++b) c += ptx::lds_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.bins[bin]), b));
                    for (uint32_t b = 0; b < blocks; ++b) ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&counts[bin]), b), c);
                }
                ptx::cluster_sync();
            }
            // The first bin up to which the tokens, or the share of the weight, lie; and the counts up to every bin.  Eight neighbouring bins a thread.
            {
                constexpr int kPer = kSampleBins / kSampleThreads;
                const uint32_t* const from = blocks > 1u ? counts : sh.bins;
                uint32_t c[kPer], n_mine = 0;
                float mine_sum = 0.f;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const int bin = kPer * tid + i;
                    c[i] = bin < kSampleBins - 1 ? from[bin] : 0u;
                    n_mine += c[i];
                    mine_sum += by_weight ? float(c[i]) * __expf(float(1 - bin) / kSampleBin) : float(c[i]);
                }
                float upto = mine_sum;
                uint32_t n_upto = n_mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const float y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
                    const uint32_t z = __shfl_up_sync(0xFFFFFFFFu, n_upto, o);
                    if (lane >= o) { upto += y;  n_upto += z; }
                }
                if (tid == 0) { sh.bin = kSampleBins - 1;  sh.by_min_p = CUDART_INF_F;  sh.place = 0.5f; }
                if (lane == 31) { sh.warp_max[warp] = upto;  sh.warp_x[warp] = n_upto; }
                __syncthreads();
                float before = upto - mine_sum, total = 0.f;
                uint32_t n_before = n_upto - n_mine;
                for (int w = 0; w < kSampleWarps; ++w) {
                    if (w < warp) { before += sh.warp_max[w];  n_before += uint32_t(sh.warp_x[w]); }
                    total += sh.warp_max[w];
                }
                // (ties: in units of the largest weight)
                // (min-p: the bin of the smallest weight it keeps, and two for rounding)
                const int floor_bin = by_weight && !LIMITED && r.min_p > 0.f ? int(-kSampleBin * logf(r.min_p)) + 3 : kSampleBins;
                // (top-p 0: the first bin that has any)
                const float goal = by_weight ? fmaxf(float(r.p24) * 5.9604645e-8f * (total + __ull2float_rn(ties) * 9.094947e-13f), 1e-30f) : float(wanted);
                // The first bin up to which the goal lies: every thread has its first one, whether or not its bins begin below the goal.  (A sum up to a thread's first
                // bin is rounded otherwise than the sum up to the last one of the thread before it; where the goal lay between the two, a condition on both sides found no bin.)
                float place = 0.5f;
                int crossed = kSampleBins - 1;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    const int bin = kPer * tid + i;
                    const float v = by_weight ? float(c[i]) * __expf(float(1 - bin) / kSampleBin) : float(c[i]);
                    if (before + v >= goal && crossed == kSampleBins - 1) {
                        crossed = bin;
                        if (v > 0.f) place = __saturatef((goal - before) / v);
                    }
                    before += v;
                    if (bin == floor_bin) sh.by_min_p = before;
                    counts[bin] = n_before += c[i];
                }
                const int first_bin = __reduce_min_sync(0xFFFFFFFFu, crossed);
                if (lane == 0) atomicMin(&sh.bin, first_bin);
                __syncthreads();
                if (crossed == sh.bin) sh.place = place;
                // Where all that min-p keeps weighs clearly less than top-p's share, top-p leaves out none of it: no cut.  A bin's tokens are within one bin of
                // it (as long as 2^23 and their distance add up exactly), which is 0.8% of their weight.
                if (sh.by_min_p * 1.03f < goal && fabsf(slope * r.top) < 1e6f) { over = 0ull;  return true; }
            }
            // That bin, one and a quarter each way, and as far each way as there are not more than kSampleSpare tokens: where they are few, rounding
            // moves the cut from one to the next, bins away.
            int low = 0, high = kSampleBins - 1;
            float half_width = 0.f;
            {
                const int bin = sh.bin;
                const uint32_t left = bin > 0 ? counts[bin - 1] : 0u, right = counts[bin];
                for (int hi = bin; low < hi;) {                        // the first bin from which at most so many lie before `bin`
                    const int mid = (low + hi) / 2;
                    if (left - (mid > 0 ? counts[mid - 1] : 0u) <= kSampleSpare) hi = mid;
                    else low = mid + 1;
                }
                for (int lo = bin; lo < high;) {
                    const int mid = (lo + high + 1) / 2;
                    if (counts[mid] - right <= kSampleSpare) lo = mid;
                    else high = mid - 1;
                }
                low = min(low, bin);
                high = max(high, bin);
                // Where they are many, and spread evenly (32-bit logits), less will do, around the place in the bin: what an estimate from counts is off by there
                // is a small part of a bin.
                const uint32_t near = counts[min(bin + 1, kSampleBins - 1)] - (bin > 1 ? counts[bin - 2] : 0u);
                if (sizeof(T) == 4 && near > kSampleMany) half_width = fmaxf(float(kSampleMany) / float(near), 0.05f);
            }
            __syncthreads();                       // (the counts lie where the candidates will be sorted)
            // Exactly: what all weigh, what lies nearer than `from`, and the candidates from there to `to`.
            float from = fminf(float(low - 1) - off - 0.5f, float(sh.bin - 1) - off - 1.25f), to = fmaxf(float(high - 1) - off + 0.5f, float(sh.bin - 1) - off + 1.25f);
            if (half_width > 0.f) {
                from = float(sh.bin - 1) - off + sh.place - 0.5f - half_width;
                to = from + 2.f * half_width;
            }
            float next = half_width > 0.f ? 2.f * half_width : 2.5f;                // (where the cut is not there after all: the next part, twice as long each time)
            unsigned long long ahead;
            for (int moved = 0, tries = 0;; ++tries) {
                // (many steps: all the way; and what is not a number is everything)
                if (!(from >= 1.f) || (tries > 8 && moved < 0)) from = -1.f;
                if (!(to <= kSampleBins - 8) || (tries > 8 && moved > 0)) to = CUDART_INF_F;
                const bool open = to == CUDART_INF_F;
                __syncthreads();
                if (tid == 0) sh.count = 0u;
                __syncthreads();
                FixedSum sum_all, sum_ahead;
                uint32_t n_all = 0, n_ahead = 0;
                // (bins are powers of two: the same comparisons on the exponent itself)
                const float x_from = from * (-1.f / kSampleBin), x_to = open ? -CUDART_INF_F : to * (-1.f / kSampleBin);
                // (candidates are within `near` of `mid`, a little more than they need to be; where that is not a number, any may be one)
                const float mid = r.top + 0.5f * (x_from + x_to) / r.per, near_by = 0.5001f * (x_from - x_to) / r.per + 1e-6f * (fabsf(r.top) + fabsf(mid));
                const bool may_be = !(near_by < CUDART_INF_F) || !(fabsf(mid) < CUDART_INF_F);
                // Logits of sixteen bits: there are few different ones there, equal ones by the hundred, and instead of a list to be sorted every warp has a
                // table of how often it meets each.
                uint32_t* const table = reinterpret_cast<uint32_t*>(sh.list) + warp * kSampleValues;
                const uint32_t top_value = (order_key(mid + near_by) >> row.kKeyShift) + 1u;
                const bool by_value = sizeof(T) == 2 && !may_be && top_value - (order_key(mid - near_by) >> row.kKeyShift) < uint32_t(kSampleValues - 1);
                if (by_value)
                    for (int i = lane; i < kSampleValues; i += 32) table[i] = 0u;
                __syncwarp();
                row.each(first, steps, [&](const float (&v)[8], int e) {
                    float off = CUDART_INF_F;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        float x0, x1;
                        r.exponents(v[i], v[i + 1], x0, x1);
                        const bool in0 = all_in || v[i] > above_value, in1 = all_in || v[i + 1] > above_value, ahead0 = in0 && x0 > x_from, ahead1 = in1 && x1 > x_from;
                        if constexpr (BY_WEIGHT) {
                            sum_all.add2(in0 ? expf(x0) : 0.f, in1 ? expf(x1) : 0.f, &sum_ahead, ahead0, ahead1);
                        } else {
                            n_all += in0 + in1;
                            n_ahead += ahead0 + ahead1;
                        }
                        off = fminf(off, fminf(fabsf(v[i] - mid), fabsf(v[i + 1] - mid)));
                    }
                    if (off <= near_by || may_be) {
                        uint32_t here = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) here |= uint32_t(may_be || fabsf(v[i] - mid) <= near_by) << i;
                        each_of(here, v, [&](float l, int i) {
                            const float x = r.exponent(l);
                            if (!(l > above_value && !(x > x_from) && x > x_to)) return;
                            if (by_value) atomicAdd(&table[min(top_value - (order_key(l + 0.f) >> row.kKeyShift), uint32_t(kSampleValues - 1))], 1u);
                            else list_logit(sh, l, e + i - row.lead);
                        });
                    }
                });
                over = by_weight ? sum_all.total() : n_all;
                ahead = by_weight ? sum_ahead.total() : n_ahead;
                const unsigned long long of_warp = warp_total(ahead);
                // (per warp, for the token, where this turns out to be the cut)
                if (by_weight && lane < int(blocks)) sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.sum[me]), lane), of_warp);
                uint32_t* const values = sh.bins + (turn ^ 1) * kSampleValues;         // (in turn, as in row_totals)
                if (by_value) {
                    __syncthreads();
                    if (tid < kSampleValues) {
                        uint32_t c = 0;
                        for (int w = 0; w < kSampleWarps; ++w) c += reinterpret_cast<const uint32_t*>(sh.list)[w * kSampleValues + tid];
                        values[tid] = c;
                    }
                }
                row_totals(sh, blocks, rank, turn, over, ahead);
                if (by_weight) wanted = max(share_of(over + ties, uint32_t(r.p24)), 1ull);
                if (wanted > over) { over = wanted - over;  return false; }
                if (wanted <= ahead) { to = from;  from -= next;  next *= 2.f;  moved = -1;  continue; }
                if (by_value) {
                    // Every warp for itself: four neighbouring values a lane, the largest first.
                    constexpr int kPer = kSampleValues / 32;
                    uint32_t* const all = sh.bins + 2 * kSampleValues;
                    if (tid < kSampleValues) {
                        uint32_t c = 0;
                        for (uint32_t b = 0; b < blocks; ++b) c += ptx::lds_cluster_u32(ptx::mapa(ptx::smem_u32(values + tid), b));
                        all[tid] = c;
                    }
                    __syncthreads();
                    auto key_of = [&](int i) {
                        const uint32_t q = (top_value - uint32_t(i)) << row.kKeyShift;
                        return (q >> 31) ? q : q | ((1u << row.kKeyShift) - 1u);
                    };
                    unsigned long long each[kPer], mine_sum = 0;
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        each[i] = !by_weight ? 1ull : all[kPer * lane + i] != 0u ? fixed(r.ratio(key_value(key_of(kPer * lane + i)))) : 0ull;
                        mine_sum += all[kPer * lane + i] * each[i];
                    }
                    const unsigned long long upto = warp_upto(mine_sum, lane), want = wanted - ahead;
                    unsigned long long before = upto - mine_sum, ties_there = 0, my_sum = 0;
                    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, upto >= want);
                    if (hit != 0u) {
                        int at = 0;
                        bool done = false;
#pragma unroll
                        for (int i = 0; i < kPer; ++i) {
                            const unsigned long long v = all[kPer * lane + i] * each[i];
                            if (!done && before + v >= want) {
                                at = kPer * lane + i;
                                ties_there = (want - before + each[i] - 1ull) / max(each[i], 1ull);
                                done = true;
                            }
                            before += v;
                        }
                        const int from_lane = __ffs(hit) - 1;
                        at = __shfl_sync(0xFFFFFFFFu, at, from_lane);
                        cut = key_of(at);
                        cut_ties = __shfl_sync(0xFFFFFFFFu, ties_there, from_lane);
                        if (by_weight && min_p_idle(cut)) {
                            // what this warp has above the cut, and at it
#pragma unroll
                            for (int i = 0; i < kPer; ++i) my_sum += kPer * lane + i < at ? table[kPer * lane + i] * each[i] : 0ull;
                            my_sum = warp_total(my_sum) + of_warp;
                            if (lane < int(blocks)) {
                                sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.sum[me]), lane), my_sum);
                                ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.ties[me]), lane), table[at]);
                            }
                            sums_known = true;
                        }
                        if (!by_weight) sync_row(blocks);              // (the bins are cleared next)
                        return true;
                    }
                    from = to;                     // (a little further away)
                    to += next;  next *= 2.f;
                    moved = 1;
                    continue;
                }
                const int m = listed(sh, blocks, turn);
                if (m >= 0 && (by_weight || wanted - ahead <= static_cast<unsigned long long>(m))) {
                    if (rank == 0) {
                        cut_of_list(sh, r, blocks, turn, m, by_weight ? m : int(wanted - ahead), by_weight ? wanted - ahead : ~0ull);
                        if (by_weight && sh.reached && min_p_idle(sh.cut)) {
                            // what the candidates above the cut add to their warps' sums, and the ties; to all blocks
                            if (tid < parts) sh.ties[tid] = 0u;
                            __syncthreads();
                            for (int i = tid; i < m; i += kSampleThreads) {
                                const unsigned long long c = sh.sorted[i];
                                const uint32_t key = uint32_t(c >> 32);
                                const int of = part_of(int(~uint32_t(c)));
                                if (key > sh.cut) atomicAdd(&sh.sum[of], fixed(r.ratio(key_value(key))));
                                else if (key == sh.cut) atomicAdd(&sh.ties[of], 1u);
                            }
                            __syncthreads();
                            for (int i = tid; i < parts * (int(blocks) - 1); i += kSampleThreads) {
                                const int part = i % parts, to_block = 1 + i / parts;
                                sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.sum[part]), to_block), sh.sum[part]);
                                ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.ties[part]), to_block), sh.ties[part]);
                            }
                        }
                    }
                    sync_row(blocks);
                    if (sh.reached) {
                        cut = sh.cut;
                        cut_ties = sh.cut_ties;
                        sums_known = by_weight && min_p_idle(cut);
                        return true;
                    }
                }
                if (m < 0) {
                    // more candidates than the lists hold: do they reach the cut?
                    FixedSum sum_upto;
                    uint32_t n_upto = 0;
                    row.each(first, steps, [&](const float (&v)[8], int) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = r.exponent(v[i]);
                            const bool in = v[i] > above_value && x > x_to;
                            if (by_weight) sum_upto.add(in ? expf(x) : 0.f);
                            n_upto += in;
                        }
                    });
                    unsigned long long upto = by_weight ? sum_upto.total() : n_upto, unused = 0;
                    row_totals(sh, blocks, rank, turn, upto, unused);
                    if (wanted <= upto) break;
                }
                from = to;
                to += next;  next *= 2.f;
                moved = 1;
            }
            wanted -= ahead;
            // Digit by digit, then.
            const float x_from = from * (-1.f / kSampleBin), x_to = to == CUDART_INF_F ? -CUDART_INF_F : to * (-1.f / kSampleBin);
            uint32_t found = 0;
            int buffer = 0;
            for (int i = tid; i < 256; i += kSampleThreads) sh.hist[0][i] = 0ull;
#pragma unroll 1
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                row.each(first, steps, [&](const float (&v)[8], int) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t key = order_key(v[i] + 0.f);
                        const float x = r.exponent(v[i]);
                        const bool in = v[i] > above_value && !(x > x_from) && x > x_to && (shift == 24 || (key >> (shift + 8)) == (found >> (shift + 8)));
                        const uint32_t digit = (key >> shift) & 255u, who = __ballot_sync(0xFFFFFFFFu, in);
                        if (who != 0u) {
                            unsigned long long w = in ? (by_weight ? fixed(expf(x)) : 1ull) : 0ull;
                            // (equal logits, the usual case here, with one atomic a warp)
                            const uint32_t same = __shfl_sync(0xFFFFFFFFu, digit, __ffs(who) - 1);
                            if (__all_sync(0xFFFFFFFFu, !in || digit == same)) {
                                w = warp_total(w);
                                if (lane == 0) atomicAdd(&sh.hist[buffer][same], w);
                            } else if (in) {
                                atomicAdd(&sh.hist[buffer][digit], w);
                            }
                        }
                    }
                });
                find_digit(sh, buffer, wanted, blocks);
                found |= sh.digit << shift;
                wanted -= sh.digit_above;
                buffer ^= 1;
                for (int i = tid; i < 256; i += kSampleThreads) sh.hist[buffer][i] = 0ull;      // (two uses ago: read by every block before the last barrier)
            }
            cut = found;
            const unsigned long long each = by_weight ? fixed(r.ratio(key_value(cut))) : 1ull;
            cut_ties = (wanted + each - 1ull) / each;
            return true;
        };
        unsigned long long beyond;
        if (r.k > 0) find_cut(std::false_type{}, std::false_type{}, 0u, static_cast<unsigned long long>(r.k), 0ull, beyond);
        if (r.p24 >= 0) {
            // top-p looks at the tokens above top-k's cut, and at those of its ties that are kept
            const unsigned long long tie = cut_ties != 0ull ? fixed(r.ratio(key_value(cut))) : 0ull;
            if (r.k == 0 || cut_ties == 0ull) find_cut(std::true_type{}, std::false_type{}, 0u, 0ull, 0ull, beyond);
            else if (!find_cut(std::true_type{}, std::true_type{}, cut, 0ull, cut_ties * tie, beyond)) cut_ties = min(cut_ties, (beyond + tie - 1ull) / tie);
        }
    }

    // ── sums of the kept weights, per warp ──
    const float cut_value = cut != 0u ? key_value(cut) : -CUDART_INF_F;
    const unsigned long long tie_weight = cut_ties != 0ull ? (r.odd ? 1ull << kSampleOneBits : r.weight(cut_value)) : 0ull;
    // Below this no token is kept: the cut, or a little below where min-p is.  (Ties at a cut that min-p leaves out weigh nothing, counted or not.)
    float floor_value = cut_value;
    if (r.min_p > 0.f && !r.odd) floor_value = fmaxf(floor_value, r.top + (logf(r.min_p) - 1e-4f) / r.per - 1e-5f * fabsf(r.top));
    auto part_sums = [&](int from, int count, unsigned long long& sum, uint32_t& ties) {
        FixedSum kept;
        ties = 0;
        if (cut_ties == 0ull && r.min_p == 0.f) {
            row.each(from, count, [&](const float (&v)[8], int) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float x0, x1;
                    r.exponents(v[i], v[i + 1], x0, x1);
                    kept.add2(expf(x0), expf(x1));
                }
            });
        } else {
            row.each(from, count, [&](const float (&v)[8], int) {
                if (!__any_sync(0xFFFFFFFFu, max_of(v) >= floor_value)) return;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float e = r.ratio(v[i]);
                    kept.add(v[i] > cut_value && e >= r.min_p ? e : 0.f);
                    ties += v[i] == cut_value;
                }
            });
        }
        sum = warp_total(kept.total());
        ties = __reduce_add_sync(0xFFFFFFFFu, ties);
    };
    // Of `parts` neighbouring parts of the row with these sums and ties: the one in which more than `target` is reached, if that is in them.  before and
    // tie_before: what lies before the first, and afterwards before the part.
    auto find_part = [&](const unsigned long long* sums, const uint32_t* ties, int parts, unsigned long long target, unsigned long long& before,
                         unsigned long long& tie_before) -> int {
        unsigned long long v[4], all = 0;
        uint32_t c[4], all_ties = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = lane * 4 + i < parts ? ties[lane * 4 + i] : 0u;
            all_ties += c[i];
        }
        unsigned long long tie_at = tie_before + warp_upto(all_ties, lane) - all_ties;
        const unsigned long long lane_ties = tie_at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned long long left = cut_ties > tie_at ? cut_ties - tie_at : 0ull;
            v[i] = lane * 4 + i < parts ? sums[lane * 4 + i] + min(left, static_cast<unsigned long long>(c[i])) * tie_weight : 0ull;
            tie_at += c[i];
            all += v[i];
        }
        unsigned long long at = before + warp_upto(all, lane) - all;
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, target >= at && target < at + all);
        int part = 0;
        tie_at = lane_ties;
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (part == i && target >= at + v[i]) { at += v[i];  tie_at += c[i];  part = i + 1; }
        const int from = __ffs(hit) - 1;
        before = __shfl_sync(0xFFFFFFFFu, at, from & 31);
        tie_before = __shfl_sync(0xFFFFFFFFu, tie_at, from & 31);
        return from * 4 + __shfl_sync(0xFFFFFFFFu, part, from & 31);
    };
    auto total_of = [&](const unsigned long long* sums, const uint32_t* ties, int parts) -> unsigned long long {
        unsigned long long v = 0, c = 0;
        for (int i = lane; i < parts; i += 32) { v += sums[i];  c += ties[i]; }
        return warp_total(v) + min(cut_ties, warp_total(c)) * tie_weight;
    };
    if (!sums_known) {
        unsigned long long sum;
        uint32_t ties;
        part_sums(first, steps, sum, ties);
        if (lane < int(blocks)) {
            sts_cluster_u64(ptx::mapa(ptx::smem_u32(&sh.sum[rank * kSampleWarps + warp]), lane), sum);
            ptx::sts_cluster_u32(ptx::mapa(ptx::smem_u32(&sh.ties[rank * kSampleWarps + warp]), lane), ties);
        }
    }
    sync_row(blocks);
    // ── the warp's part that has the token, by all warps of its block in finer parts, and of those the one that has it ──
    const unsigned long long total = total_of(sh.sum, sh.ties, parts), target = share_of(total, u24);
    unsigned long long before = 0, tie_before = 0;
    const int owner = find_part(sh.sum, sh.ties, parts, target, before, tie_before);
    if (owner / kSampleWarps != int(rank)) return;
    const int owner_first = first_step(owner), owner_steps = first_step(owner + 1) - owner_first;
    const int fine_first = owner_steps * warp / kSampleWarps, mine_steps = owner_steps * (warp + 1) / kSampleWarps - fine_first;
    const int mine_first = (owner_first + fine_first) * kSampleStep;
    {
        unsigned long long sum;
        uint32_t ties;
        part_sums(mine_first, mine_steps, sum, ties);
        __syncthreads();
        if (lane == 0) { sh.sum[warp] = sum;  sh.ties[warp] = ties; }
        __syncthreads();
        if (find_part(sh.sum, sh.ties, kSampleWarps, target, before, tie_before) != warp) return;
    }
    bool searching = true;
    row.each(mine_first, mine_steps, [&](const float (&v)[8], int e) {
        if (!searching) return;
        uint32_t here = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) here += v[i] == cut_value;
        unsigned long long tie_at = tie_before + warp_upto(here, lane) - here, w[8], sum = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = v[i] > cut_value ? r.weight(v[i]) : 0ull;
            if (v[i] == cut_value && tie_at++ < cut_ties) w[i] = tie_weight;
            sum += w[i];
        }
        const unsigned long long lane_upto = before + warp_upto(sum, lane);
        unsigned long long at = lane_upto - sum;
        if (target >= at && target < lane_upto) {
            int i = 0;
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (i == j && target >= at + w[j]) { at += w[j];  i = j + 1; }
            float l = v[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) l = i == j ? v[j] : l;
            a.token[n] = e + i - row.lead;
            if (a.logprob != nullptr) a.logprob[n] = (l == r.top ? 0.f : r.exponent(l)) - logf(__ull2float_rn(total) * 9.094947017729282e-13f);
        }
        before = __shfl_sync(0xFFFFFFFFu, lane_upto, 31);
        tie_before += __reduce_add_sync(0xFFFFFFFFu, here);
        searching = target >= before;
    });
}

}  // namespace dsv4
