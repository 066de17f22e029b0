// Attention of the new tokens of each sequence over a paged cache: o = softmax(cap(scale q k^T)) v over the positions a query sees, in one pass with a running reference
// m and sum l of the weights e^(x - m).  paged.cuh says how the work is dealt out; parts of pairs that lie in several CTAs are joined by a second kernel.
#include <algorithm>
#include <atomic>

#include "attention_internal.cuh"
#include "paged.cuh"

namespace mynn {

// One element of the output: the parts' sums over the parts' weights.  A row that sees nothing has weights of 0 and is zero; a part without keys has a maximum
// of -inf, and adds nothing.
__device__ __forceinline__ float paged_quotient(float O, float L) { return L == 0.f ? 0.f : O / L; }

constexpr int kPlainTile = 8;

// ---- any sizes ----------------------------------------------------------------------------------------------------------
// f32 caches, heads that are no multiple of 8 numbers, unaligned tensors.  Each warp takes tiles of 8 positions into shared memory as f32; in the first product
// a lane has one key and a quarter of the dimensions, in the second the dimensions lane, lane + 32, ...  Small tiles leave room for many warps, which hide each other's
// chains: with tiles of 16 and half the warps 64 sequences of 1000, 8 heads of 128, took 192 us, with every lane of a key going on with all rows 166, now 125 = 0.64 of the
// copy bandwidth with four rows, 92 = 0.87 with one.  Bound by chains: a tile is copies, product, exchange, exponentials and product one behind the other, in eight warps per SM at D = 128 (140 KB
// of shared memory: one CTA), sixteen up to D = 96, with a third of the issue slots used.  (Products of three bf16 parts per number on the tensor cores would keep 24 bits too; not built.)
// RB: query rows of a CTA (one head per kv head: with eight rows where one is needed 7 sequences of 1 to 1501, 12 heads of 80, took 46 us).
// VEC: elements of a copy to shared memory (cp.async, f32); 0: 16-bit elements, converted on the way.
template <int DL>
constexpr int kPlainWarps = DL > 4 ? 4 : 8;
template <int DL, int RB>
struct PlainShape {
    static constexpr int W = kPlainWarps<DL>, PITCH = DL * 32 + 4;
    static constexpr int RING = 2 * 2 * kPlainTile * PITCH;  // floats of a warp: two stages, keys and values
    static constexpr int WEIGHTS = kPlainTile * (RB < 4 ? 4 : RB), SUMS = RB * DL * 32;
    static constexpr size_t SMEM = sizeof(float) * (size_t)(RB * PITCH + W * (RING + WEIGHTS + SUMS));
    static constexpr int CTAS = SMEM <= 112 * 1024 ? 2 : 1;  // per SM
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void *smem, const void *gmem, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(smem)), "l"(gmem), "n"(BYTES), "r"(in ? BYTES : 0) : "memory");
}

template <typename T, int DL, int RB, int VEC>
__global__ void __launch_bounds__(kPlainWarps<DL> * 32, PlainShape<DL, RB>::CTAS) paged_attention_plain_kernel(const PagedAttention p) {
    using Shape = PlainShape<DL, RB>;
    constexpr int W = Shape::W, PITCH = Shape::PITCH, TILE = kPlainTile, WR = Shape::WEIGHTS / TILE;
    extern __shared__ __align__(16) float sm[];
    __shared__ float part_m[W][RB], part_l[W][RB];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, key = lane & 7, side = lane >> 3;
    const int cta = blockIdx.x, ctas = gridDim.x, r0 = blockIdx.y * RB, rows = min(p.group * p.S - r0, RB), D = p.D;
    float *sq = sm, *ring = sm + RB * PITCH + warp * Shape::RING, *weights = sm + RB * PITCH + W * Shape::RING + warp * Shape::WEIGHTS;
    float *sums = sm + RB * PITCH + W * (Shape::RING + Shape::WEIGHTS);
    for (int i = threadIdx.x; i < RB * PITCH; i += W * 32) sq[i] = 0.f;
    for (int i = lane; i < Shape::RING; i += 32) ring[i] = 0.f;  // what lies behind D is never written again
    __syncwarp();  // other lanes copy to these places, and of a table that is left whole no barrier comes before
    constexpr bool SPREAD = RB >= 4;
    constexpr int OWN = SPREAD ? RB / 4 : RB;
    const int own = SPREAD ? side * OWN : 0;  // the first row that this lane goes on with
    auto place = [&](int b, int h, int r, int d) {
        const int head = p.by_S.div(r);
        return (((size_t)b * p.S + p.by_S.mod(r, head)) * p.Hq + h * p.group + head) * D + d;
    };
    for (int b = cta; b < p.B; b += ctas)  // sequences that see nothing at all are in no CTA's run
        if (paged_span(p, b).tiles == 0)
            for (int h = 0; h < p.G; h++)
                for (int i = threadIdx.x; i < rows * D; i += W * 32) reinterpret_cast<T *>(p.out)[place(b, h, r0 + i / D, i % D)] = from_f32<T>(0.f);
    // this lane's 16-byte pieces of a tile's rows: row and first number, -1: none
    constexpr int COPIES = VEC == 4 ? TILE * DL * 8 / 32 : 1;
    int copies[COPIES];
#pragma unroll
    for (int u = 0; u < COPIES; u++) {
        const int i = lane + 32 * u, r = p.by_pieces.div(i);
        copies[u] = r < TILE ? r << 16 | 4 * (i - r * (D / 4)) : -1;
    }
    PagedRun run;
    run.begin(paged_find<W * 32>(p, cta, ctas));
    PagedSpan sp;
    for (; run.more(p, sp); run.advance(p)) {
        const int b = run.b, h = run.h, t0 = run.t0, t1 = run.t1;
        auto row_of = [&](int t) { return t < t1 ? paged_row(p, sp, b, h, sp.at(t) * TILE + key) : -1; };
        auto issue = [&](int row, int stage) {
            float *to = ring + stage * 2 * TILE * PITCH;
            if constexpr (VEC == 4) {
#pragma unroll
                for (int u = 0; u < COPIES; u++) {
                    const int r = copies[u] >> 16 & 7, d = copies[u] & 0xffff;
                    const int from = __shfl_sync(0xffffffffu, row, r);
                    if (copies[u] < 0) continue;
                    const size_t at = (size_t)(uint32_t)max(from, 0) * (uint32_t)(D * 4) + 4 * d;
                    float *dst = to + r * PITCH + d;
                    copy_async<16>(dst, reinterpret_cast<const char *>(p.k) + at, from >= 0);
                    copy_async<16>(dst + TILE * PITCH, reinterpret_cast<const char *>(p.v) + at, from >= 0);
                }
            } else {
                const int pieces = D;
#pragma unroll 2
                for (int i = lane; i < (TILE * pieces + 31) / 32 * 32; i += 32) {
                    const int r = p.by_pieces.div(i), d = i - r * pieces;
                    const int from = __shfl_sync(0xffffffffu, row, r & 7);
                    if (r >= TILE) continue;
                    const size_t at = (size_t)(uint32_t)max(from, 0) * (uint32_t)D + d;
                    float *dst = to + r * PITCH + d;
                    if constexpr (VEC == 1) {
                        copy_async<4>(dst, reinterpret_cast<const float *>(p.k) + at, from >= 0);
                        copy_async<4>(dst + TILE * PITCH, reinterpret_cast<const float *>(p.v) + at, from >= 0);
                    } else {
                        dst[0] = from >= 0 ? to_f32<T>(reinterpret_cast<const T *>(p.k)[at]) : 0.f;
                        dst[TILE * PITCH] = from >= 0 ? to_f32<T>(reinterpret_cast<const T *>(p.v)[at]) : 0.f;
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int row = row_of(t0 + warp), next = row_of(t0 + warp + W);
        if (t0 + warp < t1) issue(row, 0);
        __syncthreads();  // the queries and sums of the pair in front are done with
        for (int i = threadIdx.x; i < rows * D; i += W * 32) {
            const int r = r0 + i / D, head = p.by_S.div(r);
            sq[i / D * PITCH + i % D] = to_f32<T>(reinterpret_cast<const T *>(p.q)[(((size_t)b * p.Hq + h * p.group + head) * p.S + p.by_S.mod(r, head)) * D + i % D]);
        }
        __syncthreads();
        // The sums of four and more rows are dealt out to the four lanes of a key, each of which goes on with a quarter of the rows; of fewer every lane has all.
        float m[OWN], l[OWN], o[RB][DL];
#pragma unroll
        for (int r = 0; r < OWN; r++) m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int i = 0; i < DL; i++) o[r][i] = 0.f;
        for (int t = t0 + warp, stage = 0; t < t1; t += W, stage ^= 1) {
            const int after = row_of(t + 2 * W);
            if (t + W < t1) {
                issue(next, stage ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncwarp();
            const float *K = ring + stage * 2 * TILE * PITCH, *V = K + TILE * PITCH;
            float x[RB] = {};
            const int quarter = (D + 15) / 16 * 4;
#pragma unroll 4
            for (int d = side * quarter; d < (side + 1) * quarter; d += 4) {
                const float4 a = *reinterpret_cast<const float4 *>(K + key * PITCH + d);
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float4 c = *reinterpret_cast<const float4 *>(sq + r * PITCH + d);
                    x[r] += a.x * c.x + a.y * c.y + a.z * c.z + a.w * c.w;
                }
            }
            const int j = sp.at(t) * TILE + key;
            float z[OWN];
            if constexpr (SPREAD) {
                float y[RB / 2];
#pragma unroll
                for (int r = 0; r < RB / 2; r++) y[r] = (side & 2 ? x[r + RB / 2] : x[r]) + __shfl_xor_sync(0xffffffffu, side & 2 ? x[r] : x[r + RB / 2], 16);
#pragma unroll
                for (int r = 0; r < OWN; r++) z[r] = (side & 1 ? y[r + OWN] : y[r]) + __shfl_xor_sync(0xffffffffu, side & 1 ? y[r] : y[r + OWN], 8);
            } else {
#pragma unroll
                for (int r = 0; r < OWN; r++) {
                    z[r] = x[r] + __shfl_xor_sync(0xffffffffu, x[r], 8);
                    z[r] += __shfl_xor_sync(0xffffffffu, z[r], 16);
                }
            }
            bool moved = false;
#pragma unroll
            for (int r = 0; r < OWN; r++) {
                const int i = own + r;
                z[r] *= p.scale;
                if (p.softcap > 0.f) z[r] = p.softcap * tanhf(z[r] / p.softcap);
                if (i >= rows || row < 0 || (p.S > 1 && !paged_sees(p, sp, p.by_S.mod(r0 + i, p.by_S.div(r0 + i)), j))) z[r] = -INFINITY;  // (one query sees what there is)
                moved |= z[r] > m[r];
            }
            if (__any_sync(0xffffffffu, moved)) {  // most tiles raise no maximum
                float keep[OWN];
#pragma unroll
                for (int r = 0; r < OWN; r++) {
                    float top = z[r];
#pragma unroll
                    for (int s = 4; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                    const float now = fmaxf(m[r], top);
                    keep[r] = expf(m[r] - merge_reference(now));
                    m[r] = now;
                    l[r] *= keep[r];
                }
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float f = SPREAD ? __shfl_sync(0xffffffffu, keep[r % OWN], r / OWN * 8) : keep[r % OWN];
#pragma unroll
                    for (int i = 0; i < DL; i++) o[r][i] *= f;
                }
            }
#pragma unroll
            for (int r = 0; r < OWN; r++) {
                const float w = expf(z[r] - merge_reference(m[r]));
                if (SPREAD || side == 0) l[r] += w, weights[key * WR + own + r] = w;
            }
            __syncwarp();
            const bool full = p.S == 1 || paged_tile_full(p, sp, sp.at(t) * TILE, TILE);
            auto weigh = [&](auto guarded) {  // guarded: what a row does not see has to be kept from it, not only weighted by zero
#pragma unroll
                for (int k = 0; k < TILE; k++) {
                    float w[WR];
#pragma unroll
                    for (int r = 0; r < WR; r += 4) {
                        const float4 u = *reinterpret_cast<const float4 *>(weights + k * WR + r);
                        w[r] = u.x, w[r + 1] = u.y, w[r + 2] = u.z, w[r + 3] = u.w;
                    }
#pragma unroll
                    for (int i = 0; i < DL; i++) {
                        const float v = V[k * PITCH + lane + 32 * i];
#pragma unroll
                        for (int r = 0; r < RB; r++)
                            if (!decltype(guarded)::value || w[r] != 0.f) o[r][i] += w[r] * v;
                    }
                }
            };
            if (full) weigh(std::false_type());
            else weigh(std::true_type());
            __syncwarp();
            row = next;
            next = after;
        }
        // the warps' parts meet
#pragma unroll
        for (int r = 0; r < OWN; r++) {
#pragma unroll
            for (int s = 4; s > 0; s >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], s);
            if (key == 0 && (SPREAD || side == 0)) part_m[warp][own + r] = m[r], part_l[warp][own + r] = l[r];
        }
#pragma unroll
        for (int r = 0; r < RB; r++)
#pragma unroll
            for (int i = 0; i < DL; i++) sums[warp * Shape::SUMS + r * DL * 32 + lane + 32 * i] = o[r][i];
        __syncthreads();
        const bool whole = t0 == 0 && t1 == sp.tiles;
        float *part = p.ws + (((size_t)blockIdx.y * ctas + cta) * 2 + (run.first ? 0 : 1)) * p.part_floats;
        for (int i = threadIdx.x; i < rows * D; i += W * 32) {
            const int r = i / D, d = i - r * D;
            float top = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, part_m[w][r]);
            const float ref = merge_reference(top);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float f = expf(part_m[w][r] - ref);
                L += part_l[w][r] * f;
                O += sums[w * Shape::SUMS + r * DL * 32 + d] * f;
            }
            if (whole) {
                reinterpret_cast<T *>(p.out)[place(b, h, r0 + r, d)] = from_f32<T>(paged_quotient(O, L));
            } else {
                part[i] = O;
                if (d == 0) part[RB * D + r] = top, part[RB * D + RB + r] = L;
            }
        }
    }
    if (blockIdx.y == 0 && threadIdx.x == 0 && p.records) p.records[cta] = run.record;
}

// ---- 16-bit caches on the tensor cores --------------------------------------------------------------------------------
// Bound by the one pass over the cache.  A team of RW warps takes tiles of 16 or 32 positions: cp.async brings a tile's rows, wherever their pages lie, to a ring in
// shared memory whose entries are the keys or the values of a tile, each warp a share of the rows, and each warp then multiplies the whole tile with query rows of its
// own, eight or NT times eight, so that a row of the cache is read once for up to 64 query rows (all heads of a group, all drafts).  Both products are mma.m16n8k16 on
// fragments that are whole 8 x 8 blocks from ldmatrix, without a byte moved: S^T = K Q^T, eight query rows as columns, and O^T = V^T P^T, whose second operand is
// the first product's result behind a transposition of its 8 x 8 blocks.  Weights enter as a 16-bit part and its remainder (16 bits in all, kTop says how f16 keeps them); scores, maxima and
// sums are f32.  The reference of the weights is moved only when a score exceeds it by 2^kLag, so most tiles need no maximum across lanes and no rescaling.  D is padded
// to DP with zeros, on the chip only.
// The chain of one tile is long (two products, a softmax) and each warp walks it alone, so warps are what hides it: sixteen per SM with eight query rows each (with eight
// warps of sixteen rows 96 mixed sequences of heads of 64 took a fifth longer).  From 17 rows on sixteen rows of a warp share the blocks of keys and values and what goes on around the
// products (20 rows over 131072 positions: 110 us with eight rows per warp, 105 with sixteen), and the chain bounds it: eight warps per SM (255 registers), a quarter of the issue slots and of the
// tensor pipe, stalls that are fixed latencies and a loop that does not fit the instruction cache.  Rows are laid out for the batch's S, so places without a token are worked on as well.
// Measured per call, with the joining kernel behind it, 8 kv heads of 128, bf16: 32 sequences of 2048 47 us = 0.87 of the copy bandwidth, 16 of 1500 to 4500 with 5 queries of 4
// heads 56 us = 0.54, with 8 queries 61, with one query in 5 places 56, 48 with windows of 1000 over pages of 24 42 us = 0.72, one of 300 14 us (7 on the device); f16: one of 131071
// 94 us = 0.87, 4 kv heads of 64, 96 of 1 to 6000 57 us = 0.79.  What is left of one query is what a launch costs around its pass: to find its run, the first copies, the last sums and
// the join take some 8 us.
template <int DP, int RW, int NT>
struct MmaShape {
    static constexpr int W = 8, TEAMS = W / RW, ROWS = 8 * NT * RW;
    static constexpr int CTAS = DP > 128 || (DP == 128 && NT == 2) ? 1 : 2;  // per SM
    static constexpr int SPACE = (CTAS == 1 ? 192 : NT == 2 ? 80 : 96) * 1024 / TEAMS;
    // A tile is 32 positions where three entries of that size fit, else 16: what goes on around the products takes as long as they do.
    static constexpr int TILE = SPACE / (32 * DP * 2) >= 3 ? 32 : 16, ENTRY = TILE * DP * 2;
    // Large teams have room for the keys and values of a tile together, and meet once per tile instead of twice.
    static constexpr bool JOINT = RW > 1 && SPACE / ENTRY >= 5;
    static constexpr int FIT = JOINT ? SPACE / ENTRY / 2 - 1 : (SPACE / ENTRY - 1) / 2, AHEAD = FIT < 3 ? FIT : 3;  // tiles on their way while one is worked on
    static constexpr int STAGES = 2 * AHEAD + (JOINT ? 2 : 1), WAIT = JOINT ? 2 * AHEAD - 2 : STAGES - 2;             // groups of copies that may still be on their way
    static constexpr size_t RING = (size_t)TEAMS * STAGES * ENTRY;
    static constexpr size_t SMEM = RING + W * 8 * NT * 64 * sizeof(float);  // and 64 dimensions of all warps' sums
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Where a 16-byte piece c of a row lies among the eight of its 128 bytes: the same piece of eight rows is in different banks.
__device__ __forceinline__ int paged_swizzle(int row, int c) { return c ^ (row & 7); }
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void copy16_now(uint32_t smem, const void *gmem) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t special_mask(uint32_t x) {  // all ones over each of two 16-bit numbers that is infinite or NaN
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return ((x & e) == e ? 0xffffu : 0u) | ((x >> 16 & e) == e ? 0xffff0000u : 0u);
}

// Weights of the second product are 2^(x - m + kTop), m lagging behind the largest score by up to kLag, and two 16-bit parts hold them.  bf16 has the range of f32.  Both parts
// of an f16 number end at 2^-24: with the largest weight near the other end of its range, 2^15, 16 bits are left of one 2^22 times as small as that of m (2^-9).  Where a lane has
// none as large, the tile is multiplied with weights that are 2^up times as large, its own largest near 2^15, by sums that are brought there and back, powers of two that change no
// bit.  So behind a key that leads by any number of nats, and whose value may be zero, the others keep 16 bits; those that share its tile are right to 2^-38 of
// the largest.  Tiles that are all so small take longer: behind a first key that leads by 20 nats 131071 positions, 8 kv heads of 128, 119 us instead of 113 (32 sequences of 2048
// 75 instead of 67; cold caches).  The check itself costs nothing with eight rows of a warp and heads of up to 128, up to 5 % else (20 rows of 64 numbers over 60000 positions 59.5 us,
// 56 without).
template <typename T>
constexpr int kTop = std::is_same<T, __half>::value ? 13 : 0;
template <typename T>
constexpr int kLag = std::is_same<T, __half>::value ? 2 : 8;

template <typename T, int DP, int RW, int NT>
__global__ void __launch_bounds__(256, MmaShape<DP, RW, NT>::CTAS) paged_attention_mma_kernel(const PagedAttention p) {
    using Shape = MmaShape<DP, RW, NT>;
    constexpr bool JOINT = Shape::JOINT;
    constexpr int W = Shape::W, TEAMS = Shape::TEAMS, STAGES = Shape::STAGES, AHEAD = Shape::AHEAD, TILE = Shape::TILE, KT = TILE / 16, KS = DP / 16, CPR = DP / 8;
    constexpr bool NARROW = kTop<T> != 0;
    constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ float part_m[W][8 * NT], part_l[W][8 * NT];
    __shared__ __align__(8) float to_reference[W][8 * NT];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, team = warp / RW;
    const int cta = blockIdx.x, ctas = gridDim.x, D = p.D, R = p.group * p.S;
    // A warp's number says which of the SM's four schedulers it is on; the last members of a team may have fewer rows, and are spread over them.
    const int member = (warp + team + (RW == 2 ? team >> 1 : 0)) % RW, slot = team * RW + member, r0 = blockIdx.y * Shape::ROWS + member * 8 * NT;
    uint8_t *ring = raw + (size_t)team * STAGES * Shape::ENTRY;
    float *sums = reinterpret_cast<float *>(raw + Shape::RING);
    const uint32_t ring_at = smem_u32(ring);
    const bool busy = r0 < R, more_rows = NT > 1 && r0 + 8 < R;  // a warp without rows of its own only helps to copy
    // this lane's places: of its first copy in the cache and in an entry, of the first piece of a row of keys (row lane % 16) and, transposed, of values.  Entries
    // begin on 128 bytes, so that another piece or row is an exclusive or away.
    constexpr int COPIES = (TILE * CPR + 32 * RW - 1) / (32 * RW), STEP = 32 * RW / CPR;
    constexpr bool EVEN = 32 * RW % CPR == 0;
    constexpr int STRIPS = TILE / 8;
    constexpr uint32_t ALL = 0xffffffffu >> (32 - TILE);
    const char *k_rows = reinterpret_cast<const char *>(p.k) + (member * 32 + lane) * 16, *v_rows = reinterpret_cast<const char *>(p.v) + (member * 32 + lane) * 16;
    const int copy_row = (member * 32 + lane) / CPR, copy_piece = (member * 32 + lane) % CPR, k_row = lane & 15, v_row = (lane & 7) + (lane >> 4) * 8;
    const uint32_t copy_lane = copy_row * (DP * 2) + (copy_piece >> 3) * 128 + paged_swizzle(copy_row, copy_piece & 7) * 16;
    const uint32_t k_lane = ring_at + k_row * (DP * 2) + paged_swizzle(k_row, lane >> 4) * 16, v_lane = ring_at + v_row * (DP * 2) + paged_swizzle(v_row, lane >> 3 & 1) * 16;
    for (int b = cta; b < p.B; b += ctas)  // sequences that see nothing at all are in no CTA's run
        if (paged_span(p, b).tiles == 0)  // (a share for each block of rows)
            for (size_t n = (size_t)p.S * p.Hq * D / 8, i = blockIdx.y * (W * 32) + threadIdx.x; i < n; i += (size_t)gridDim.y * (W * 32)) reinterpret_cast<uint4 *>(p.out)[b * n + i] = make_uint4(0, 0, 0, 0);
    auto team_sync = [&]() {
        if constexpr (RW == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(RW * 32) : "memory");
    };
    // scores in units of ln 2, or of the cap
    const float unit = p.softcap > 0.f ? p.scale / p.softcap : p.scale * kLog2e;
    PagedRun run;
    run.begin(paged_find<W * 32>(p, cta, ctas));
    PagedSpan sp;
    // the pair that was worked on last, whose sums are still the warps' own
    int done_b = -1, done_h = 0;
    bool whole = false;
    float *part = nullptr;
    float o[NT][KS][4], m[NT][2], l[NT][2], ref[NT][2], limit[NT][2];  // ref, limit: what weights are relative to, and the score that moves it
    for (;;) {
        const bool more = run.more(p, sp);
        const int b = run.b, h = run.h, t0 = run.t0, t1 = run.t1;
        const int mine = more && t0 + team < t1 ? (t1 - t0 - team + TEAMS - 1) / TEAMS : 0;
        const int oldest = sp.len - sp.count;
        // last position that row r0 + i sees, -1: it is no query
        auto last_seen = [&](int i) {
            const int r = r0 + i, s = p.by_S.mod(r, p.by_S.div(r));
            return r < R && s < sp.count ? oldest + s : -1;
        };
        int at[NT][2];  // of this lane's rows 8 n + 2 t and + 1
#pragma unroll
        for (int n = 0; n < NT; n++) at[n][0] = last_seen(8 * n + 2 * t), at[n][1] = last_seen(8 * n + 2 * t + 1);
        auto sees = [&](int last, int j) { return j <= last && (p.window <= 0 || last - j < p.window || j < p.sinks); };
        auto base_of = [&](int j) { return (int)((unsigned)sp.at(t0 + team + TEAMS * j) * TILE); };  // (behind the last tile it may wrap, and is not used)
        // The first row of eight positions whose rows lie one behind the other and are all seen, for 32 such strips at once, one per lane; -1 for others.
        auto strips_of = [&](int i) {
            const int j = i / STRIPS, pos = base_of(j) + i % STRIPS * 8;
            if (j >= mine || !p.strips || pos + 8 > sp.rows || (p.window > 0 && oldest - pos >= p.window && pos + 8 > p.sinks)) return -1;
            return paged_row(p, sp, b, h, pos);
        };
        auto row_of = [&](int j) { return j < mine ? paged_row(p, sp, b, h, base_of(j) + (lane & (TILE - 1))) : -1; };
        // The keys or the values of a tile to an entry of the ring, from strips (uniform) where there are any, else row by row (row: of position lane % TILE).
        auto issue = [&](const char *rows, uint32_t entry, int j, bool fast, int strips, int row, uint32_t there) {
            if (j < mine) {
                const uint32_t to = ring_at + entry + copy_lane;
                if (fast) {
                    const char *src = rows;
#pragma unroll
                    for (int i = 0; i < COPIES; i++) {
                        if constexpr (EVEN && STEP <= 8) {  // the lane's row moves on by STEP rows, its piece stays
                            if (STEP * i % 8 == 0) src = rows + (size_t)(uint32_t)__shfl_sync(0xffffffffu, strips, (j * STRIPS + STEP * i / 8) & 31) * (DP * 2);
                            copy16_now((to ^ (STEP * i & 7) << 4) + STEP * i * DP * 2, src + STEP * i % 8 * (DP * 2));
                        } else {
                            const int idx = (i * RW + member) * 32 + lane, r = idx / CPR, c = idx % CPR;
                            if (TILE * CPR % (32 * RW) != 0 && idx >= TILE * CPR) break;  // (a whole warp)
                            const int from = __shfl_sync(0xffffffffu, strips, (j * STRIPS + (r >> 3)) & 31) + (r & 7);
                            copy16_now(ring_at + entry + r * (DP * 2) + (c >> 3) * 128 + paged_swizzle(r, c & 7) * 16, rows + (size_t)(uint32_t)from * (DP * 2) + c * 16 - (member * 32 + lane) * 16);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < COPIES; i++) {
                        const int idx = (i * RW + member) * 32 + lane, r = idx / CPR, c = idx % CPR;
                        if (TILE * CPR % (32 * RW) != 0 && idx >= TILE * CPR) break;  // (a whole warp)
                        const int from = __shfl_sync(0xffffffffu, row, r);
                        const bool in = (there >> r & 1) && 8 * c < D;
                        const char *src = rows - (member * 32 + lane) * 16 + (size_t)(uint32_t)from * (uint32_t)(2 * D) + (8 * c < D ? 16 * c : 0);
                        copy16_at(EVEN ? (to ^ (STEP * i & 7) << 4) + STEP * i * DP * 2 : ring_at + entry + r * (DP * 2) + (c >> 3) * 128 + paged_swizzle(r, c & 7) * 16, src, in);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        // What issue() needs for tile j, and which rows of it there are.
        int strips = -1, strips_next = -1, row = -1;
        uint32_t strips_there = 0;
        uint32_t there = 0;
        bool fast = false;
        auto look_up = [&](int j) {
            if ((j * STRIPS & 31) == 0) {
                strips = strips_next, strips_next = strips_of(j * STRIPS + 32 + lane);
                strips_there = __ballot_sync(0xffffffffu, strips >= 0);
            }
            fast = (strips_there >> (j * STRIPS & 31) & ((1u << STRIPS) - 1)) == (1u << STRIPS) - 1;
            there = ALL;
            if (!fast) {
                row = row_of(j);
                there = __ballot_sync(0xffffffffu, row >= 0) & ALL;
                row = max(row, 0);
            }
        };
        uint32_t exist[AHEAD + 1];  // which rows of the next tiles there are
        uint32_t qb[NT][KS][2];  // row 8 n + g, dimensions 16 i + 2 t and + 8
        if (more) {
            team_sync();  // the ring is free
            strips_next = strips_of(lane);
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                look_up(j);
                exist[j] = there;
                issue(k_rows, 2 * j * Shape::ENTRY, j, fast, strips, row, there);
                issue(v_rows, (2 * j + 1) * Shape::ENTRY, j, fast, strips, row, there);
            }
            look_up(AHEAD);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int r = min(r0 + 8 * n + g, R - 1), head = p.by_S.div(r), s = p.by_S.mod(r, head);
                const bool in = r0 + 8 * n + g < R && s < sp.count;
                const T *qr = reinterpret_cast<const T *>(p.q) + (((size_t)b * p.Hq + h * p.group + head) * p.S + s) * D;
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int d = 16 * i + 8 * e + 2 * t;
                        qb[n][i][e] = in && d < D ? *reinterpret_cast<const uint32_t *>(qr + d) : 0u;
                    }
            }
        }
        // ---- the teams meet, while the first tiles of the next pair are on their way: 64 dimensions of all warps' sums at a time ----
        if (done_b >= 0) {
            const int rows = min(R - (int)blockIdx.y * Shape::ROWS, Shape::ROWS);
            __syncthreads();  // nobody reads what the pair in front left any more
            if (g == 0) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) part_m[slot][8 * n + 2 * t + e] = m[n][e], part_l[slot][8 * n + 2 * t + e] = l[n][e];
            }
            __syncthreads();
            float f[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < TEAMS; w++) top = fmaxf(top, part_m[w * RW + member][8 * n + 2 * t + e]);
                    f[n][e] = exp2_approx(m[n][e] - merge_reference(top));
                }
#pragma unroll
            for (int s = 0; s < DP / 64; s++) {
                if (s > 0) __syncthreads();
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int k = 0; k < 4; k++)  // (dimensions 8 apart for neighbouring t: all banks)
                            sums[(slot * 8 * NT + 8 * n + 2 * t + (k & 1)) * 64 + ((16 * i + 8 * (k >> 1) + g) ^ (t * 8))] = o[n][4 * s + i][k] * f[n][k & 1];
                __syncthreads();
                for (int i = threadIdx.x; i < rows * 32; i += W * 32) {
                    const int r = i >> 5, d = 2 * (i & 31), w0 = r / (8 * NT), own = r % (8 * NT), at = r * 64 + (d ^ ((r >> 1 & 3) * 8));
                    float2 O = make_float2(0.f, 0.f);
                    float top = -INFINITY, L = 0.f;
#pragma unroll
                    for (int w = 0; w < TEAMS; w++) {
                        const float2 u = *reinterpret_cast<const float2 *>(sums + at + w * RW * 512 * NT);
                        O.x += u.x, O.y += u.y;
                        top = fmaxf(top, part_m[w * RW + w0][own]);
                    }
#pragma unroll
                    for (int w = 0; w < TEAMS; w++) L += part_l[w * RW + w0][own] * exp2_approx(part_m[w * RW + w0][own] - merge_reference(top));
                    if (64 * s + d >= D) continue;
                    if (whole) {
                        const int q = blockIdx.y * Shape::ROWS + r, head = p.by_S.div(q);
                        T *to = reinterpret_cast<T *>(p.out) + (((size_t)done_b * p.S + p.by_S.mod(q, head)) * p.Hq + done_h * p.group + head) * D + 64 * s + d;
                        const float inv = __frcp_rn(L);  // (a second rounding of 2^-24 in front of one of 2^-9 or 2^-11)
                        __align__(4) T y[2] = {from_f32<T>(L == 0.f ? 0.f : O.x * inv), from_f32<T>(L == 0.f ? 0.f : O.y * inv)};
                        *reinterpret_cast<uint32_t *>(to) = *reinterpret_cast<const uint32_t *>(y);
                    } else {
                        *reinterpret_cast<float2 *>(part + (size_t)r * D + 64 * s + d) = O;
                        if (s == 0 && d == 0) {
                            part[Shape::ROWS * D + r] = top * kLn2;
                            part[Shape::ROWS * D + Shape::ROWS + r] = L;
                        }
                    }
                }
            }
        }
        if (!more) break;
        // offsets: the entry that is read next, the one that is empty (JOINT: the first of two)
        uint32_t cur = 0, free_entry = (STAGES - (JOINT ? 2 : 1)) * Shape::ENTRY;
        auto step_on = [&]() {
            free_entry = JOINT ? cur - Shape::ENTRY : cur;  // (JOINT: called behind the values)
            cur = cur + Shape::ENTRY == STAGES * Shape::ENTRY ? 0 : cur + Shape::ENTRY;
        };
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int e = 0; e < 2; e++) m[n][e] = limit[n][e] = -INFINITY, ref[n][e] = -kTop<T>, l[n][e] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[n][i][e] = 0.f;
        }
#pragma unroll 1
        for (int j = 0; j < mine; j++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(Shape::WAIT) : "memory");
            team_sync();  // the keys of tile j are here (JOINT: its values too), and the values of tile j - 1 are done with
            const int ahead = j + AHEAD;
            exist[AHEAD] = there;
            issue(k_rows, free_entry, ahead, fast, strips, row, there);
            if constexpr (JOINT) {
                issue(v_rows, free_entry + Shape::ENTRY, ahead, fast, strips, row, there);
                look_up(ahead + 1);
            }
            const int base = base_of(j);
            const uint32_t K = k_lane + cur;
            if constexpr (JOINT) cur += Shape::ENTRY;
            else step_on();
            // ---- S^T = K Q^T: x[n][k][2 c + e] is position base + 16 k + g + 8 c, row 8 n + 2 t + e ----
            uint32_t hi[NT][KT][2], lo[NT][KT][2];
            unsigned small = 0;  // bit n: the tile is multiplied by itself for rows 8 n .. 8 n + 7, and then brought to the reference by to_reference
            const bool full = exist[0] == ALL && (p.S == 1 || paged_tile_full(p, sp, base, TILE));
            auto scores = [&](auto groups) {
                constexpr int N = decltype(groups)::value;
                float x[N][KT][4], y[N][KT][4];
#pragma unroll
                for (int n = 0; n < N; n++)
#pragma unroll
                    for (int k = 0; k < KT; k++)
#pragma unroll
                        for (int i = 0; i < 4; i++) x[n][k][i] = y[n][k][i] = 0.f;
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int k = 0; k < KT; k++) {
                        uint32_t a[4];
                        ldsm4_at(a, (K ^ (i & 3) << 5) + (i >> 2) * 128 + k * 16 * DP * 2);
#pragma unroll
                        for (int n = 0; n < N; n++) mma_kv<T>(KT == 1 && N == 1 && (i & 1) ? y[n][k] : x[n][k], a[0], a[1], a[2], a[3], qb[n][i][0], qb[n][i][1]);
                    }
#pragma unroll
                for (int n = 0; n < N; n++) {
                    float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < KT; k++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            if (KT == 1 && N == 1) x[n][k][i] += y[n][k][i];
                            x[n][k][i] *= unit;
                        }
                    if (p.softcap > 0.f) {  // (tanhf is right relative to itself: a cap far above the scores leaves them as they are; no slower than a form in e^x)
#pragma unroll
                        for (int k = 0; k < KT; k++)
#pragma unroll
                            for (int i = 0; i < 4; i++) x[n][k][i] = kLog2e * (p.softcap * tanhf(x[n][k][i]));
                    }
                    if (!full) {
#pragma unroll
                        for (int k = 0; k < KT; k++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const int bit = 16 * k + g + 8 * (i >> 1);
                                if (!((exist[0] >> bit & 1) && sees(at[n][i & 1], base + bit))) x[n][k][i] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int k = 0; k < KT; k++)
#pragma unroll
                        for (int i = 0; i < 4; i++) most[i & 1] = fmaxf(most[i & 1], x[n][k][i]);
                    auto below = [&](int e) { return NARROW && most[e] < ref[n][e] - 9.f && most[e] > -INFINITY && ref[n][e] < INFINITY; };
                    if (__any_sync(0xffffffffu, most[0] > limit[n][0] || most[1] > limit[n][1] || below(0) || below(1))) {
                        float tops[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            float top = most[e];
#pragma unroll
                            for (int s = 4; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                            // (only of rows that exceed it: what a row gives does not hang on the rows beside it)
                            const float now = top > limit[n][e] ? top : m[n][e], keep = exp2_approx(m[n][e] - merge_reference(now));
                            m[n][e] = now;
                            ref[n][e] = merge_reference(now) - kTop<T>;
                            limit[n][e] = now + kLag<T>;
                            tops[e] = top;
                            l[n][e] *= keep;
#pragma unroll
                            for (int i = 0; i < KS; i++) o[n][i][e] *= keep, o[n][i][2 + e] *= keep;
                        }
                        if (NARROW && __any_sync(0xffffffffu, below(0) || below(1))) {
                            small |= 1u << n;
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                // brings the tile's largest weight to 2^14 .. 2^15 (or 2^60 times nearer: the sums have to stay numbers)
                                const bool own = (__ballot_sync(0xffffffffu, below(e)) & 0x11111111u << t) != 0u;  // (the row's lanes)
                                const float up = own ? fminf(floorf(ref[n][e] + 15.f - tops[e]), 60.f) : 0.f;
#pragma unroll
                                for (int k = 0; k < KT; k++) x[n][k][e] += up, x[n][k][2 + e] += up;
                                const float there = __int_as_float((127 + (int)up) << 23);  // 2^up
                                l[n][e] *= there;
#pragma unroll
                                for (int i = 0; i < KS; i++) o[n][i][e] *= there, o[n][i][2 + e] *= there;
                                if (g == 0) to_reference[warp][8 * n + 2 * t + e] = __int_as_float((127 - (int)up) << 23);  // 2^-up
                            }
                            __syncwarp();
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KT; k++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) x[n][k][i] = exp2_approx(x[n][k][i] - ref[n][i & 1]);
                        l[n][0] += x[n][k][0] + x[n][k][2];  // of this lane's positions
                        l[n][1] += x[n][k][1] + x[n][k][3];
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            split_pack<T>(x[n][k][2 * c], x[n][k][2 * c + 1], hi[n][k][c], lo[n][k][c]);
                            hi[n][k][c] = transpose_8x8(hi[n][k][c]), lo[n][k][c] = transpose_8x8(lo[n][k][c]);  // positions 16 k + 8 c + 2 t, + 1 of row 8 n + g
                        }
                    }
                }
            };
            if (more_rows) scores(std::integral_constant<int, NT>());
            else if (busy) scores(std::integral_constant<int, 1>());
            if constexpr (!JOINT) {
                asm volatile("cp.async.wait_group %0;" ::"n"(Shape::WAIT) : "memory");
                team_sync();  // the values of tile j are here, and its keys are done with
                issue(v_rows, free_entry, ahead, fast, strips, row, there);
                look_up(ahead + 1);
            }
            const uint32_t V = v_lane + cur, v_entry = cur;
            step_on();
            // ---- O^T += V^T P^T: o[n][i] is dimensions 16 i + g (registers 0, 1) and + 8 (2, 3) of rows 8 n + 2 t and + 1 ----
            // Values that are no numbers, in a tile that not every row sees all of?
            bool odd = false;
            if (!full && p.S > 1) {
#pragma unroll 1
                for (int i = lane; i < TILE * CPR; i += 32) {
                    const uint4 u = *reinterpret_cast<const uint4 *>(ring + v_entry + i * 16);
                    odd |= (special_mask<T>(u.x) | special_mask<T>(u.y) | special_mask<T>(u.z) | special_mask<T>(u.w)) != 0u;
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            auto values = [&](auto groups, auto rare) {
                constexpr int N = decltype(groups)::value;
                const bool special = !NARROW || odd;
#pragma unroll
                for (int i = 0; i < KS; i++) {
#pragma unroll
                    for (int k = 0; k < KT; k++) {
                        uint32_t a[4], c[4];
                        ldsm4t_at(a, (V ^ (i & 3) << 5) + (i >> 2) * 128 + k * 16 * DP * 2);
                        if constexpr (decltype(rare)::value) {
#pragma unroll
                            for (int q = 0; q < 4; q++) {
                                if (special) c[q] = a[q] & special_mask<T>(a[q]), a[q] &= ~special_mask<T>(a[q]);
                                else c[q] = 0u;
                            }
                        }
#pragma unroll
                        for (int n = 0; n < N; n++) {
                            mma_kv<T>(o[n][i], a[0], a[1], a[2], a[3], hi[n][k][0], hi[n][k][1]);
                            mma_kv<T>(o[n][i], a[0], a[1], a[2], a[3], lo[n][k][0], lo[n][k][1]);
                        }
                        if constexpr (decltype(rare)::value) {
#pragma unroll 1
                            for (int q = special ? 0 : 16; q < 16; q++) {
                                const uint32_t one = (q & 7) >> 1 == t ? (q & 1 ? 0xffff0000u : 0xffffu) : 0u, first = q < 8 ? one : 0u, second = q < 8 ? 0u : one;
#pragma unroll
                                for (int n = 0; n < N; n++) {
                                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma_kv<T>(acc, c[0] & first, c[1] & first, c[2] & second, c[3] & second, hi[n][k][0], hi[n][k][1]);
#pragma unroll
                                    for (int e = 0; e < 2; e++)
                                        if ((exist[0] >> (16 * k + q) & 1) && sees(at[n][e], base + 16 * k + q)) o[n][i][e] += acc[e], o[n][i][2 + e] += acc[2 + e];
                                }
                            }
                        }
                    }
                }
                if constexpr (NARROW && decltype(rare)::value) {
#pragma unroll
                    for (int n = 0; n < N; n++)
                        if (small >> n & 1) {
                            const float2 back = *reinterpret_cast<const float2 *>(&to_reference[warp][8 * n + 2 * t]);
                            l[n][0] *= back.x, l[n][1] *= back.y;
#pragma unroll
                            for (int i = 0; i < KS; i++) o[n][i][0] *= back.x, o[n][i][1] *= back.y, o[n][i][2] *= back.x, o[n][i][3] *= back.y;
                        }
                }
            };
            // Values that are no numbers are taken out of the product and added position by position where they are seen, so that the other rows keep their bits.
            if (!odd && small == 0) {
                if (more_rows) values(std::integral_constant<int, NT>(), std::false_type());
                else if (busy) values(std::integral_constant<int, 1>(), std::false_type());
            } else {
                if (more_rows) values(std::integral_constant<int, NT>(), std::true_type());
                else if (busy) values(std::integral_constant<int, 1>(), std::true_type());
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) exist[i] = exist[i + 1];
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int s = 4; s < 32; s <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], s);
                if (at[n][e] < 0) m[n][e] = -INFINITY, l[n][e] = 0.f;  // a row that is no query, which tiles that all see are not masked for
            }
        done_b = b, done_h = h;
        whole = t0 == 0 && t1 == sp.tiles;
        part = p.ws + (((size_t)blockIdx.y * ctas + cta) * 2 + (run.first ? 0 : 1)) * p.part_floats;
        run.advance(p);
    }
    if (blockIdx.y == 0 && threadIdx.x == 0 && p.records) p.records[cta] = run.record;
}

// ---- parts of pairs that lie in several CTAs ------------------------------------------------------------------------------
// grid (CTAs of the kernel in front, row groups): a CTA takes `rows` rows (1, 2, 4 or 8) of the pair that the CTA of its number recorded, 8 / rows warps
// each; the parts of a row are dealt out to its warps, eight at a time and loads first.  V: floats of a load.
// Waits of L2 in a row: the record, the maxima, the rows.
constexpr int kJoinWarps = 8;
template <typename T, int V>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attention_join_kernel(const PagedAttention p, int ctas, int rows) {
    constexpr int ITEMS = 8 / V, U = 8;
    __shared__ float sums[kJoinWarps][256], weights[kJoinWarps];
    pdl_trigger();
    pdl_wait();
    const int4 rec = p.records[blockIdx.x];
    if (rec.x < 0) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = kJoinWarps / rows, sub = warp & (per - 1);
    const int c0 = blockIdx.x, n = rec.z - c0 + 1, R = p.block_rows, D = p.D;
    const int r = blockIdx.y * rows + warp / per, block = r / R, i0 = r - block * R;
    const bool in = r < p.group * p.S;
    const float *parts = p.ws + (size_t)block * ctas * 2 * p.part_floats;
    auto part = [&](int c) { return parts + ((size_t)(c0 + c) * 2 + (c == 0 ? rec.w : 0)) * p.part_floats; };
    float top = -INFINITY, L = 0.f, O[ITEMS][V] = {};
    if (in) {
        for (int c = lane; c < n; c += 32) top = fmaxf(top, part(c)[R * D + i0]);
        top = warp_max(top);
        const float ref = merge_reference(top);
        for (int c = sub; c < n; c += per * U) {
            const int mine = c + per * (lane & (U - 1));
            float f = 0.f;
            if (mine < n) {
                const float *from = part(mine) + R * D + i0;
                f = expf(from[0] - ref);
                L += lane < U ? f * from[R] : 0.f;
            }
            float v[U][ITEMS][V];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float *from = part(min(c + per * u, n - 1)) + (size_t)i0 * D;
#pragma unroll
                for (int k = 0; k < ITEMS; k++) {
                    const int d = V * (lane + 32 * k);
                    if constexpr (V == 4) {
                        const float4 x = d < D ? *reinterpret_cast<const float4 *>(from + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                        v[u][k][0] = x.x, v[u][k][1] = x.y, v[u][k][2] = x.z, v[u][k][3] = x.w;
                    } else {
                        v[u][k][0] = d < D ? from[d] : 0.f;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float fu = __shfl_sync(0xffffffffu, f, u);
                if (c + per * u < n)
#pragma unroll
                    for (int k = 0; k < ITEMS; k++)
#pragma unroll
                        for (int e = 0; e < V; e++) O[k][e] += fu * v[u][k][e];
            }
        }
        L = warp_sum(L);
    }
    if (per > 1) {
        if (lane == 0) weights[warp] = L;
#pragma unroll
        for (int k = 0; k < ITEMS; k++)
#pragma unroll
            for (int e = 0; e < V; e++)
                if (V * (lane + 32 * k) < D) sums[warp][V * (lane + 32 * k) + e] = O[k][e];
        __syncthreads();
        if (sub > 0) return;
        for (int w = 1; w < per; w++) {
            L += weights[warp + w];
#pragma unroll
            for (int k = 0; k < ITEMS; k++)
#pragma unroll
                for (int e = 0; e < V; e++)
                    if (V * (lane + 32 * k) < D) O[k][e] += sums[warp + w][V * (lane + 32 * k) + e];
        }
    }
    if (!in) return;
    const int head = p.by_S.div(r);
    T *out = reinterpret_cast<T *>(p.out) + (((size_t)rec.x * p.S + p.by_S.mod(r, head)) * p.Hq + rec.y * p.group + head) * D;
#pragma unroll
    for (int k = 0; k < ITEMS; k++)
#pragma unroll
        for (int e = 0; e < V; e++)
            if (V * (lane + 32 * k) < D) out[V * (lane + 32 * k) + e] = from_f32<T>(paged_quotient(O[k][e], L));
}

// How the launch is cut: kernel, query rows of a block, CTAs.
struct PagedPlan {
    bool mma;
    int tile;
    int dim, team, groups;  // padded head dimension, warps of a team, groups of eight rows of a warp
    int ctas, block_rows, row_blocks, round;
    bool whole;
    bool cut() const { return !whole && ctas > 1; }  // are there parts to join?
    size_t bytes(int D) const { return !cut() ? 0 : (size_t)ctas * sizeof(int4) + (size_t)ctas * row_blocks * 2 * part_floats(D) * sizeof(float); }
    int part_floats(int D) const { return (block_rows * (D + 2) + 3) / 4 * 4; }  // 16-byte pieces of them are read
};

// Tile and CTAs per SM of the kernel for these sizes.
template <int DP, int RW, int NT>
static void mma_shape(int *tile, int *ctas) { *tile = MmaShape<DP, RW, NT>::TILE, *ctas = MmaShape<DP, RW, NT>::CTAS; }
template <int DP>
static void mma_shape_rows(int team, int groups, int *tile, int *ctas) {
    if constexpr (DP <= 128) {
        if (groups == 2) return team == 2 ? mma_shape<DP, 2, 2>(tile, ctas) : mma_shape<DP, 4, 2>(tile, ctas);
        return team == 1 ? mma_shape<DP, 1, 1>(tile, ctas) : mma_shape<DP, 2, 1>(tile, ctas);
    } else {
        return team == 1 ? mma_shape<DP, 1, 1>(tile, ctas) : team == 2 ? mma_shape<DP, 2, 1>(tile, ctas) : team == 4 ? mma_shape<DP, 4, 1>(tile, ctas) : mma_shape<DP, 8, 1>(tile, ctas);
    }
}

static int paged_sms(int *sms) {
    static std::atomic<int> known[64];  // of a device, once asked for
    int dev = 0;
    MYNN_CUDA_OK(cudaGetDevice(&dev));
    *sms = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
    if (*sms == 0) {
        MYNN_CUDA_OK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
        if (dev < 64) known[dev].store(*sms, std::memory_order_relaxed);
    }
    return MYNN_OK;
}

static int plain_rows(int R, int dtype) { return dtype != MYNN_F32 ? (R == 1 ? 1 : 8) : R == 1 ? 1 : R == 2 ? 2 : R <= 4 ? 4 : 8; }
template <int DL>
static int plain_ctas(int rows) {
    return rows == 1 ? PlainShape<DL, 1>::CTAS : rows == 2 ? PlainShape<DL, 2>::CTAS : rows == 4 ? PlainShape<DL, 4>::CTAS : PlainShape<DL, 8>::CTAS;
}

static PagedPlan paged_plan(int B, int S, int Hq, int Hkv, int D, int page, int width, int sms, bool mma, int dtype) {
    PagedPlan n;
    const int R = Hq / Hkv * S;
    n.mma = mma;
    n.dim = D <= 64 ? 64 : D <= 128 ? 128 : D <= 192 ? 192 : 256;
    n.groups = R > 16 && n.dim <= 128 ? 2 : 1;  // (more would not fit the registers)
    n.team = (R <= 8 ? 1 : R <= 16 ? 2 : R <= 32 ? 4 : 8) / n.groups;
    n.block_rows = mma ? 8 * n.team * n.groups : plain_rows(R, dtype);
    n.row_blocks = (R + n.block_rows - 1) / n.block_rows;
    n.round = mma ? 8 / n.team : D <= 128 ? kPlainWarps<4> : kPlainWarps<8>;
    int per_sm = 0;
    if (mma) {
        if (n.dim == 64) mma_shape_rows<64>(n.team, n.groups, &n.tile, &per_sm);
        else if (n.dim == 128) mma_shape_rows<128>(n.team, n.groups, &n.tile, &per_sm);
        else if (n.dim == 192) mma_shape_rows<192>(n.team, n.groups, &n.tile, &per_sm);
        else mma_shape_rows<256>(n.team, n.groups, &n.tile, &per_sm);
    } else {
        n.tile = kPlainTile;
        per_sm = D <= 32 ? plain_ctas<1>(n.block_rows) : D <= 64 ? plain_ctas<2>(n.block_rows) : D <= 96 ? plain_ctas<3>(n.block_rows) : D <= 128 ? plain_ctas<4>(n.block_rows) : plain_ctas<8>(n.block_rows);
    }
    const long long tiles = ((long long)width * page + n.tile - 1) / n.tile, most = (long long)sms * per_sm;
    // Tables of so many positions: pairs are not cut, and no second kernel follows.  One sequence, 8 kv heads of 128, 16 bits: 500 positions 8.0 us whole, 10.6 cut, 1000
    // 11.1 and 11.8; in f32 100 positions 10 us whole, 12 cut, 300 19 and 12.
    n.whole = (long long)width * page <= (mma ? 1024 : 256);
    // Every block of rows has as many CTAs, all of them together some full waves: one, or as few up to four as leave the least of the GPU idle.  So the parts stay below eight per resident
    // CTA, 80 MB, whatever the number of rows (a wave per block: 480 MB
    // for 777 tokens of 4 heads of 128), and pairs are not cut finer than that takes: 6 prompts of 777 tokens 1438 us with a wave per block, 868 so; f32, 8 tokens of 8 heads of 64 over 3000 positions 108 and 68.
    long long per_block = 1;
    double busy = 0.0;
    for (int waves = 1; waves <= 4 && busy < 0.95; waves++) {
        const long long c = waves * most / n.row_blocks;
        const double share = (double)(c * n.row_blocks) / (double)(waves * most);
        if (c > 0 && share > busy + 0.02) per_block = c, busy = share;
    }
    n.ctas = n.whole ? B * Hkv : (int)std::min<long long>(per_block, std::max<long long>(1, (tiles * Hkv * B + n.round - 1) / n.round));
    return n;
}

template <typename T, int DP, int RW, int NT>
static int launch_mma(cudaStream_t st, const PagedAttention &p, int ctas) {
    using Shape = MmaShape<DP, RW, NT>;
    static SmemLimit limit;
    MYNN_CUDA_OK(limit.raise((const void *)paged_attention_mma_kernel<T, DP, RW, NT>, Shape::SMEM));
    MYNN_CUDA_OK(launch_dependent(paged_attention_mma_kernel<T, DP, RW, NT>, dim3(ctas, p.row_blocks), dim3(256), Shape::SMEM, st, p));
    MYNN_LAUNCH_OK("paged_attention_mma_kernel");
    return MYNN_OK;
}
template <typename T, int DP>
static int launch_mma_rows(cudaStream_t st, const PagedAttention &p, const PagedPlan &n) {
    if (n.team == 1) return launch_mma<T, DP, 1, 1>(st, p, n.ctas);
    if constexpr (DP <= 128) {
        if (n.groups == 2) return n.team == 2 ? launch_mma<T, DP, 2, 2>(st, p, n.ctas) : launch_mma<T, DP, 4, 2>(st, p, n.ctas);
        return launch_mma<T, DP, 2, 1>(st, p, n.ctas);
    } else {
        return n.team == 2 ? launch_mma<T, DP, 2, 1>(st, p, n.ctas) : n.team == 4 ? launch_mma<T, DP, 4, 1>(st, p, n.ctas) : launch_mma<T, DP, 8, 1>(st, p, n.ctas);
    }
}
template <typename T>
static int launch_mma_any(cudaStream_t st, const PagedAttention &p, const PagedPlan &n) {
    switch (n.dim) {
        case 64: return launch_mma_rows<T, 64>(st, p, n);
        case 128: return launch_mma_rows<T, 128>(st, p, n);
        case 192: return launch_mma_rows<T, 192>(st, p, n);
        default: return launch_mma_rows<T, 256>(st, p, n);
    }
}

template <typename T, int DL, int RB, int VEC>
static int launch_plain(cudaStream_t st, const PagedAttention &p, int ctas) {
    static SmemLimit limit;
    MYNN_CUDA_OK(limit.raise((const void *)paged_attention_plain_kernel<T, DL, RB, VEC>, PlainShape<DL, RB>::SMEM));
    MYNN_CUDA_OK(launch_dependent(paged_attention_plain_kernel<T, DL, RB, VEC>, dim3(ctas, p.row_blocks), dim3(kPlainWarps<DL> * 32), PlainShape<DL, RB>::SMEM, st, p));
    MYNN_LAUNCH_OK("paged_attention_plain_kernel");
    return MYNN_OK;
}
template <typename T, int DL>
static int launch_plain_rows(cudaStream_t st, const PagedAttention &p, int ctas, int vec) {
    if constexpr (!std::is_same<T, float>::value) {
        return p.block_rows == 1 ? launch_plain<T, DL, 1, 0>(st, p, ctas) : launch_plain<T, DL, 8, 0>(st, p, ctas);
    } else {
        if (vec == 1) return p.block_rows == 1 ? launch_plain<T, DL, 1, 1>(st, p, ctas) : p.block_rows == 2 ? launch_plain<T, DL, 2, 1>(st, p, ctas) : p.block_rows == 4 ? launch_plain<T, DL, 4, 1>(st, p, ctas) : launch_plain<T, DL, 8, 1>(st, p, ctas);
        return p.block_rows == 1 ? launch_plain<T, DL, 1, 4>(st, p, ctas) : p.block_rows == 2 ? launch_plain<T, DL, 2, 4>(st, p, ctas) : p.block_rows == 4 ? launch_plain<T, DL, 4, 4>(st, p, ctas) : launch_plain<T, DL, 8, 4>(st, p, ctas);
    }
}

}  // namespace mynn

using namespace mynn;

static int paged_check(int B, int S, int Hq, int Hkv, int D, int page, int width) {
    if (B < 0 || S < 1 || Hq < 1 || Hkv < 1 || D < 1 || page < 1 || width < 1) return fail(MYNN_E_ARG, "paged_attention: bad shape");
    if (Hq % Hkv) return fail(MYNN_E_ARG, "paged_attention: %d query heads are no multiple of %d kv heads", Hq, Hkv);
    if (D > 256) return fail(MYNN_E_UNSUPPORTED, "paged_attention: heads of %d (at most 256)", D);
    if ((long long)page * width > INT_MAX - 64) return fail(MYNN_E_UNSUPPORTED, "paged_attention: %lld positions per sequence", (long long)page * width);
    if ((long long)Hq / Hkv * S > 1 << 16) return fail(MYNN_E_UNSUPPORTED, "paged_attention: %d new tokens of %d heads per kv head", S, Hq / Hkv);
    if ((long long)B * Hkv > INT_MAX) return fail(MYNN_E_UNSUPPORTED, "paged_attention: %d sequences of %d kv heads", B, Hkv);
    return MYNN_OK;
}

extern "C" size_t mynn_b200_paged_attention_workspace_bytes(int B, int S, int Hq, int Hkv, int D, int page, int table_pages) {
    int sms = 0;
    if (paged_check(B, S, Hq, Hkv, D, page, table_pages) != MYNN_OK || B == 0 || paged_sms(&sms) != MYNN_OK) return 0;
    size_t most = 0;  // of the kernels that the tensors' type and alignment may ask for
    for (const int dtype : {(int)MYNN_F32, (int)MYNN_BF16})
        for (const bool mma : {false, true}) most = std::max(most, paged_plan(B, S, Hq, Hkv, D, page, table_pages, sms, mma, dtype).bytes(D));
    return most;
}

extern "C" int mynn_b200_paged_attention(void *stream, void *out, const void *q, const void *k_pages, const void *v_pages, const int32_t *block_table,
                                         const int32_t *lengths, const int32_t *counts, float scale, float softcap, int window, int sinks, int B, int S,
                                         int Hq, int Hkv, int D, int page, int pages, int table_pages, int dtype, void *workspace, size_t workspace_bytes) {
    if (const int e = paged_check(B, S, Hq, Hkv, D, page, table_pages)) return e;
    if (!dtype_ok(dtype)) return fail(MYNN_E_ARG, "paged_attention: bad dtype %d", dtype);
    if (pages < 0 || sinks < 0) return fail(MYNN_E_ARG, "paged_attention: %d pages, %d first positions", pages, sinks);
    if ((long long)pages * Hkv * page > INT_MAX) return fail(MYNN_E_UNSUPPORTED, "paged_attention: a cache of %lld rows", (long long)pages * Hkv * page);
    if (B == 0) return MYNN_OK;
    if (!out || !q || !block_table || !lengths || (pages && (!k_pages || !v_pages))) return fail(MYNN_E_ARG, "paged_attention: null pointer");
    if (pages == 0) {  // nobody sees anything, and there is no address to copy from
        MYNN_CUDA_OK(cudaMemsetAsync(out, 0, (size_t)B * S * Hq * D * dtype_size(dtype), (cudaStream_t)stream));
        return MYNN_OK;
    }
    int sms = 0;
    if (const int e = paged_sms(&sms)) return e;
    const bool mma = dtype != MYNN_F32 && D % 8 == 0 && ((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0;
    const PagedPlan n = paged_plan(B, S, Hq, Hkv, D, page, table_pages, sms, mma, dtype);
    const size_t need = n.bytes(D);
    if (need && (!workspace || workspace_bytes < need)) return fail(MYNN_E_ARG, "paged_attention: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    if ((uintptr_t)workspace % 16) return fail(MYNN_E_ARG, "paged_attention: the workspace is not aligned to 16 bytes");
    const int vec = D % 4 == 0 && ((uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0 ? 4 : 1;
    PagedAttention p;
    p.out = out, p.q = q;
    p.k = k_pages, p.v = v_pages;
    p.table = block_table, p.lengths = lengths, p.counts = counts;
    p.scale = scale, p.softcap = softcap, p.window = window, p.sinks = sinks;
    p.B = B, p.S = S, p.Hq = Hq, p.G = Hkv, p.group = Hq / Hkv, p.D = D;
    p.page = page, p.pages = pages, p.width = table_pages;
    p.by_page = FixedDivisor(page), p.by_S = FixedDivisor(S), p.by_pieces = FixedDivisor(dtype == MYNN_F32 ? D / vec : D);
    p.row_blocks = n.row_blocks, p.block_rows = n.block_rows, p.part_floats = n.part_floats(D), p.round = n.round;
    p.whole = n.whole;
    p.tile = n.tile;
    // 96 mixed sequences of 1 to 6000, 4 kv heads of 64: 74 us with no toll, 66 with 8 tiles of 16 positions, 59 with 16, 58 with 32 (16 with drafts 72, 72, 71, 70; one of
    // 131071 95, 95, 95, 97); f32, 7 of 1 to 1501: 120 with none, 65 with one round of the warps, 64 with two, 72 with four.
    p.toll = n.mma ? 256 / n.tile : 2 * n.round;
    p.strips = n.mma && page % 8 == 0 && D == n.dim;
    p.records = n.cut() ? reinterpret_cast<int4 *>(workspace) : nullptr;
    p.ws = n.cut() ? reinterpret_cast<float *>(p.records + n.ctas) : nullptr;
    const cudaStream_t st = (cudaStream_t)stream;
    MYNN_DISPATCH_DTYPE(dtype, T, {
        int e = MYNN_OK;
        if (n.mma) {
            if constexpr (!std::is_same<T, float>::value) e = launch_mma_any<T>(st, p, n);
        } else if (D <= 32) e = launch_plain_rows<T, 1>(st, p, n.ctas, vec);
        else if (D <= 64) e = launch_plain_rows<T, 2>(st, p, n.ctas, vec);
        else if (D <= 96) e = launch_plain_rows<T, 3>(st, p, n.ctas, vec);
        else if (D <= 128) e = launch_plain_rows<T, 4>(st, p, n.ctas, vec);
        else e = launch_plain_rows<T, 8>(st, p, n.ctas, vec);
        if (e != MYNN_OK) return e;
        if (!n.cut()) return MYNN_OK;
        const int R = p.group * S, rows = R == 1 ? 1 : R == 2 ? 2 : R <= 4 ? 4 : 8;
        const dim3 grid(n.ctas, (R + rows - 1) / rows), block(kJoinWarps * 32);
        if (D % 4 == 0) MYNN_CUDA_OK(launch_dependent(paged_attention_join_kernel<T, 4>, grid, block, 0, st, p, n.ctas, rows));
        else MYNN_CUDA_OK(launch_dependent(paged_attention_join_kernel<T, 1>, grid, block, 0, st, p, n.ctas, rows));
        MYNN_LAUNCH_OK("paged_attention_join_kernel");
    });
    return MYNN_OK;
}
