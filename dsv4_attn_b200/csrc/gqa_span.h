// The pages that new tokens of a request see: plain arithmetic, for kernels and host programs alike.
#pragma once

#if defined(__CUDACC__)
#define DSV4_GQA_HD __host__ __device__ __forceinline__
#else
#define DSV4_GQA_HD inline
#endif

namespace dsv4 {

constexpr int kGqaTile = 64;                                      // entries of a tile: a page

// ── the tiles of some tokens ──
struct GqaSpan {
    int t0, t1;                      // the tokens
    int lo, hi, first;               // entries that some token sees: [0, first) and [lo, hi)
    int head, skip, count;           // tiles: `head` from 0 on, the others `skip` pages further on; count >= 1 (tokens that see nothing have one tile, whose page is not looked up: hi is 0)
    DSV4_GQA_HD int slot(int k) const { return k < head ? k : k + skip; }
    // entries of slot s can be seen, so that the table has a page for it
    DSV4_GQA_HD bool has(int s) const { return s < (hi + kGqaTile - 1) / kGqaTile; }
};

// Tokens t0 .. t1 of a request whose first token stands at place0 and of which `entries` entries, at most what its table has room for, can be looked up.
DSV4_GQA_HD GqaSpan gqa_token_span(int place0, int entries, int t0, int t1, int window, int first) {
    GqaSpan s;
    s.t0 = t0;
    s.t1 = t1;
    const int end_place = place0 + t1 + 1;
    s.hi = end_place < entries ? (end_place > 0 ? end_place : 0) : entries;
    s.lo = 0;
    s.first = 0;
    if (window > 0) {
        const int from = place0 + t0 - window + 1;
        s.lo = from < s.hi ? (from > 0 ? from : 0) : s.hi;
        s.first = first < s.hi ? first : s.hi;
        // (a window that lies behind all entries: a length beyond the table)
        if (s.lo == s.hi && s.first == 0) s.lo = s.hi = 0;
    }
    const int end = (s.hi + kGqaTile - 1) / kGqaTile, heads = (s.first + kGqaTile - 1) / kGqaTile, from = s.lo / kGqaTile;
    s.head = heads < from ? heads : from;
    s.skip = from - s.head;
    s.count = end - s.skip > 1 ? end - s.skip : 1;
    return s;
}

}  // namespace dsv4
