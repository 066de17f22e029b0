// Paged caches: which cached rows the queries of a sequence see, how those rows are dealt out to the CTAs of a launch, and the launch
// parameters that the kernels of paged_attention.cu share.
//
// A cache is pages [pages, Hkv, page, D]; position j of sequence b lies in row j % page of page table[b, j / page].  lengths[b] counts the positions
// of the sequence with its new tokens, counts[b] the new tokens: query s of the sequence sits at position lengths[b] - counts[b] + s.
//
// Sequences of a batch have lengths of their own, so a fixed number of CTAs per sequence would leave most of the GPU waiting for the longest one.
// The visible rows are cut into tiles of 8, 16 or 32 positions (p.tile), and all tiles of all (sequence, kv head) pairs, one pair behind the other, are
// dealt out evenly: each CTA takes one run of `share` tiles, which may end one pair, hold a few whole ones and begin another.  A pair that
// lies in one CTA is finished there; the parts of the others go to a workspace and are joined by a second kernel.  A CTA has at most two parts:
// the pair its run begins inside of (slot 0) and the pair it ends inside of (slot 1); it records the one that begins in it and ends elsewhere.  The lengths are on
// the device, so every CTA works out the division itself.  Where the block table has room for a few tiles only, a pair is not worth cutting: each has a CTA.
#pragma once
#include <limits.h>

#include "common.cuh"

namespace mynn {

// Division of a number below 2^31 by a fixed one: (umulhi(n, mul) + n) >> shift with mul = floor(2^32 (2^shift - d) / d) + 1, 2^shift the next power of two.
struct FixedDivisor {
    unsigned d = 1, mul = 1, shift = 0;
    FixedDivisor() = default;
    explicit FixedDivisor(int divisor) : d((unsigned)divisor) {
        while (shift < 31 && (1u << shift) < d) shift++;
        mul = (unsigned)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const { return (int)((__umulhi((unsigned)n, mul) + (unsigned)n) >> shift); }
    __device__ __forceinline__ int mod(int n, int q) const { return n - q * (int)d; }
};

struct PagedAttention {
    void *out;
    const void *q, *k, *v;
    const int32_t *table, *lengths, *counts;  // counts null: S each
    float scale, softcap;
    int window, sinks;
    int B, S, Hq, G, group, D;
    int page, pages, width;  // rows of a page, pages of the cache, pages in a row of the table
    FixedDivisor by_page, by_S, by_pieces;  // by_pieces: copies of a row, of the kernel for any sizes
    int row_blocks, block_rows;  // the group * S query rows of a pair, row r = head * S + s, in blocks
    int tile, round, toll;             // shares are multiples of `round`, the tiles that the warps of a CTA take at a time; toll: see PagedRun
    int4 *records;               // per CTA the pair that begins in it and ends in another: {b, h, last CTA, slot}, or b == -1; null: no pair can end elsewhere
    float *ws;                   // [row block][CTA][2] parts of part_floats floats: block_rows rows of D, then maxima, then sums
    int part_floats;             // a multiple of 4
    int whole;                   // each pair is left to a CTA of its own
    int strips;                  // eight positions lie in one page, and rows are as long on the chip as in the cache
};

// What the new queries of a sequence see: the tiles of the first tokens, then those from the oldest query's window on.
struct PagedSpan {
    int len, count, rows;         // rows: positions that the block table has entries for
    int sink_tiles, skip, tiles;  // skip: tiles between the two parts
    __device__ __forceinline__ int at(int t) const { return t + (t < sink_tiles ? 0 : skip); }  // in tiles from the first position
};

__device__ __forceinline__ PagedSpan paged_span(const PagedAttention &p, int b) {
    PagedSpan s;
    s.len = max(p.lengths[b], 0);
    s.rows = min(s.len, p.width * p.page);
    s.count = p.counts ? min(max(p.counts[b], 0), p.S) : p.S;
    const int oldest = s.len - s.count;
    const int shift = p.tile == 8 ? 3 : p.tile == 16 ? 4 : 5, up = p.tile - 1;
    const int all = (s.rows + up) >> shift;
    const int lo = p.window > 0 ? min(max(0, max(oldest, 0) - p.window + 1) >> shift, all) : 0;  // the tile that the windows begin in (new tokens may lie before position 0)
    s.sink_tiles = min((min(p.sinks, s.rows) + up) >> shift, lo);
    s.skip = lo - s.sink_tiles;
    s.tiles = s.count > 0 ? all - s.skip : 0;
    return s;
}

// Does query s (position oldest + s) see position j?
__device__ __forceinline__ bool paged_sees(const PagedAttention &p, const PagedSpan &sp, int s, int j) {
    const int at = sp.len - sp.count + s;
    return s < sp.count && j <= at && (p.window <= 0 || at - j < p.window || j < p.sinks);
}

// The row of the cache that holds position j of sequence b for kv head h; -1 where no query sees it or the table names no page.
__device__ __forceinline__ int paged_row(const PagedAttention &p, const PagedSpan &sp, int b, int h, int j) {
    if (j >= sp.rows || (p.window > 0 && sp.len - sp.count - j >= p.window && j >= p.sinks)) return -1;
    const int i = p.by_page.div(j), pg = p.table[(size_t)b * p.width + i];
    return (unsigned)pg < (unsigned)p.pages ? (pg * p.G + h) * p.page + (j - i * p.page) : -1;
}
// All queries of the sequence see all of the tile (what a tile holds that only some see has to be kept from the others, not only weighted by zero: it may
// be infinite).
__device__ __forceinline__ bool paged_tile_full(const PagedAttention &p, const PagedSpan &sp, int base, int tile) {
    return base + tile - 1 <= sp.len - sp.count && (p.window <= 0 || sp.len - 1 - base < p.window || base + tile <= p.sinks);
}

struct PagedShare {
    long long total, share;
    int b, h, t;  // where this CTA's run begins (b == B: it has none)
};

// 64-bit divisions take some hundred instructions, which a CTA has to wait for before it can begin: the totals of real batches fit 32 bits.
__device__ __forceinline__ long long paged_divide(long long a, int d) { return a < INT_MAX ? (unsigned)a / (unsigned)d : a / d; }

__device__ __forceinline__ long long paged_share(long long total, int ctas, int round) { return max(paged_divide(paged_divide(total + ctas - 1, ctas) + round - 1, round), 1ll) * round; }

// What a CTA takes one after the other: tiles t0 .. t1 - 1 of pair (b, h).  To begin with a pair takes time as well, so a pair counts as `toll` tiles more: they lie in front
// of its tiles, v0 .. v1 - 1 counts both.
struct PagedRun {
    int b, h, t0, t1, v0, v1;
    long long share, left;
    int4 record;
    bool first;
    __device__ __forceinline__ void begin(const PagedShare &s) {
        b = s.b, h = s.h, v0 = s.t;
        share = left = s.share;
        record = make_int4(-1, 0, 0, 0);
        first = true;
    }
    // On to the next pair that has tiles; false: there is none.
    __device__ __forceinline__ bool more(const PagedAttention &p, PagedSpan &sp) {
        for (; b < p.B && left > 0; b++, h = v0 = 0) {
            sp = paged_span(p, b);
            if (sp.tiles == 0) continue;
            const int cost = sp.tiles + p.toll;
            v1 = (int)min((long long)cost, v0 + left);
            t0 = max(v0 - p.toll, 0);
            t1 = max(v1 - p.toll, 0);
            if (t1 <= t0) break;  // the run ends in the toll: the pair is the next CTA's
            if (t0 == 0 && v1 < cost) record = make_int4(b, h, blockIdx.x + (int)paged_divide(cost - v1 + share - 1, (int)share), first ? 0 : 1);  // (share < v1 <= 2^31)
            return true;
        }
        left = 0;
        return false;
    }
    __device__ __forceinline__ void advance(const PagedAttention &p) {
        left -= v1 - v0;
        v0 = 0;
        first = false;
        if (++h == p.G) h = 0, b++;
    }
};

__device__ __forceinline__ long long paged_cost(const PagedAttention &p, int b) {
    const int n = paged_span(p, b).tiles;
    return n > 0 ? n + p.toll : 0;
}

// Called by all threads of a CTA: the total cost and the place cta * share in it.  Each thread sums a run of sequences.
template <int THREADS>
__device__ __forceinline__ PagedShare paged_find(const PagedAttention &p, int cta, int ctas) {
    __shared__ long long warp_sums[THREADS / 32];
    __shared__ int warp_most[THREADS / 32];
    __shared__ PagedShare found;
    auto whole = [&]() -> PagedShare {  // pair `cta`, all of it
        const int b = cta / p.G;
        return b < p.B ? PagedShare{0, paged_cost(p, b), b, cta - b * p.G, 0} : PagedShare{0, 0, p.B, 0, 0};
    };
    if (p.whole) return whole();
    const int per = (p.B + THREADS - 1) / THREADS, b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    long long mine = 0;
    int most = 0;
    for (int b = b0; b < b1; b++) {
        const int n = (int)paged_cost(p, b);
        mine += (long long)n * p.G;
        most = max(most, n);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sums[warp] = incl, warp_most[warp] = most;
    __syncthreads();
    long long before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
        most = max(most, warp_most[w]);
    }
    const long long share = paged_share(total, ctas, p.round), begin = cta * share, end = before + incl;
    // Sequences of about one length, no more pairs than CTAs: cutting and joining takes longer than the longest pair on its own (32 sequences of 2048, 256 pairs for 296
    // CTAs: 44.4 us uncut, 50.6 cut).
    if ((long long)p.B * p.G <= ctas && most <= share + max(share / 4, (long long)p.toll)) return whole();
    long long at = end - mine;
    if (threadIdx.x == 0 && begin >= total) found = {total, share, p.B, 0, 0};
    if (begin >= at && begin < end) {
        for (int b = b0; b < b1; b++) {
            const long long n = paged_cost(p, b);
            if (begin < at + n * p.G) {
                const long long rest = begin - at;
                const int h = (int)paged_divide(rest, (int)n);
                found = {total, share, b, h, (int)(rest - h * n)};
                break;
            }
            at += n * p.G;
        }
    }
    __syncthreads();
    return found;
}

}  // namespace mynn
