// Attention of the new tokens of each sequence over a paged cache (paged.cuh says how the work is dealt out).
#include <algorithm>

#include "attention_internal.cuh"
#include "paged.cuh"

namespace mynn {

// One element of the output: the parts' sums over the parts' weights.  A row that sees nothing has weights of 0 and is zero; a part without keys has a maximum
// of -inf, and adds nothing.
__device__ __forceinline__ float paged_quotient(float O, float L) { return L == 0.f ? 0.f : O / L; }

// ---- any sizes ----------------------------------------------------------------------------------------------------------
// f32 caches, heads that are no multiple of 8 numbers, unaligned tensors.  Each warp takes tiles of 16 positions into shared memory as f32; in the first product
// a lane has one key and half of the dimensions, in the second the dimensions lane, lane + 32, ...
// VEC: elements of a copy to shared memory (cp.async, f32); 0: 16-bit elements, converted on the way.
constexpr int kPlainRows = 8;
template <int DL>
constexpr int kPlainWarps = DL > 4 ? 2 : 4;
template <int DL>
constexpr size_t plain_smem() {
    constexpr int pitch = DL * 32 + 4, warps = kPlainWarps<DL>;
    return sizeof(float) * (size_t)(warps * (2 * 2 * kPagedTile * pitch + kPagedTile * kPlainRows) + kPlainRows * pitch);
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void *smem, const void *gmem, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(smem)), "l"(gmem), "n"(BYTES), "r"(in ? BYTES : 0) : "memory");
}

template <typename T, int DL, int VEC>
__global__ void __launch_bounds__(kPlainWarps<DL> * 32) paged_attention_plain_kernel(const PagedAttention p) {
    constexpr int RB = kPlainRows, W = kPlainWarps<DL>, PITCH = DL * 32 + 4, TILE = kPagedTile;
    extern __shared__ __align__(16) float sm[];
    __shared__ float part_m[W][RB], part_l[W][RB];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, key = lane & 15, side = lane >> 4;
    const int cta = blockIdx.x, ctas = gridDim.x, r0 = blockIdx.y * RB, rows = min(p.group * p.S - r0, RB), D = p.D;
    float *sq = sm, *ring = sm + RB * PITCH + warp * (2 * 2 * TILE * PITCH), *weights = sm + RB * PITCH + W * (2 * 2 * TILE * PITCH) + warp * TILE * RB;
    for (int i = threadIdx.x; i < RB * PITCH; i += W * 32) sq[i] = 0.f;
    for (int i = lane; i < 2 * 2 * TILE * PITCH; i += 32) ring[i] = 0.f;  // what lies behind D is never written again
    const PagedShare run = paged_find<W * 32>(p, cta, ctas);
    auto place = [&](int b, int h, int r, int d) { return (((size_t)b * p.S + r % p.S) * p.Hq + h * p.group + r / p.S) * D + d; };
    for (int b = cta; b < p.B; b += ctas)  // sequences that see nothing at all belong to no run
        if (paged_span(p, b).tiles == 0)
            for (int i = threadIdx.x; i < p.G * rows * D; i += W * 32)
                reinterpret_cast<T *>(p.out)[place(b, i / (rows * D), r0 + i / D % rows, i % D)] = from_f32<T>(0.f);
    int b = run.b, h = run.h, t0 = run.t;
    long long left = run.share;
    for (bool first = true; b < p.B && left > 0; first = false) {
        const PagedSpan sp = paged_span(p, b);
        if (sp.tiles == 0) {
            b++;
            h = t0 = 0;
            continue;
        }
        const int t1 = (int)min((long long)sp.tiles, t0 + left);
        __syncthreads();
        for (int i = threadIdx.x; i < rows * D; i += W * 32) {
            const int r = r0 + i / D;
            sq[i / D * PITCH + i % D] = to_f32<T>(reinterpret_cast<const T *>(p.q)[(((size_t)b * p.Hq + h * p.group + r / p.S) * p.S + r % p.S) * D + i % D]);
        }
        __syncthreads();
        float m[RB], l[RB], o[RB][DL];
#pragma unroll
        for (int r = 0; r < RB; r++) {
            m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
            for (int i = 0; i < DL; i++) o[r][i] = 0.f;
        }
        auto row_of = [&](int t) { return t < t1 ? paged_row(p, sp, b, h, sp.base(t) + key) : -1; };
        auto issue = [&](int row, int stage) {
            float *to = ring + stage * 2 * TILE * PITCH;
#pragma unroll 4
            for (int r = 0; r < TILE; r++) {
                const int from = __shfl_sync(0xffffffffu, row, r);
                const size_t at = (size_t)max(from, 0) * D;
                if constexpr (VEC > 0) {
                    for (int d = lane * VEC; d < D; d += 32 * VEC) {
                        copy_async<4 * VEC>(to + r * PITCH + d, reinterpret_cast<const float *>(p.k) + at + d, from >= 0);
                        copy_async<4 * VEC>(to + (TILE + r) * PITCH + d, reinterpret_cast<const float *>(p.v) + at + d, from >= 0);
                    }
                } else {
                    for (int d = lane; d < D; d += 32) {
                        to[r * PITCH + d] = from >= 0 ? to_f32<T>(reinterpret_cast<const T *>(p.k)[at + d]) : 0.f;
                        to[(TILE + r) * PITCH + d] = from >= 0 ? to_f32<T>(reinterpret_cast<const T *>(p.v)[at + d]) : 0.f;
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int row = row_of(t0 + warp), next = row_of(t0 + warp + W);
        if (t0 + warp < t1) issue(row, 0);
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
            const int half = (D + 7) / 8 * 4;
            for (int d = side * half; d < (side + 1) * half; d += 4) {
                const float4 a = *reinterpret_cast<const float4 *>(K + key * PITCH + d);
#pragma unroll
                for (int r = 0; r < RB; r++) {
                    const float4 c = *reinterpret_cast<const float4 *>(sq + r * PITCH + d);
                    x[r] += a.x * c.x + a.y * c.y + a.z * c.z + a.w * c.w;
                }
            }
            const int j = sp.base(t) + key;
#pragma unroll
            for (int r = 0; r < RB; r++) {
                x[r] += __shfl_xor_sync(0xffffffffu, x[r], 16);
                x[r] *= p.scale;
                if (p.softcap > 0.f) x[r] = p.softcap * tanhf(x[r] / p.softcap);
                if (r >= rows || row < 0 || !paged_sees(p, sp, (r0 + r) % p.S, j)) x[r] = -INFINITY;
                float top = x[r];
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                const float now = fmaxf(m[r], top), ref = merge_reference(now), keep = expf(m[r] - ref), w = expf(x[r] - ref);
                m[r] = now;
                l[r] = l[r] * keep + (side ? 0.f : w);
                if (!side) weights[key * RB + r] = w;
#pragma unroll
                for (int i = 0; i < DL; i++) o[r][i] *= keep;
            }
            __syncwarp();
            const bool full = p.S == 1 || paged_tile_full(p, sp, sp.base(t));
#pragma unroll 2
            for (int k = 0; k < TILE; k++) {
                float w[RB];
#pragma unroll
                for (int r = 0; r < RB; r += 4) *reinterpret_cast<float4 *>(w + r) = *reinterpret_cast<const float4 *>(weights + k * RB + r);
#pragma unroll
                for (int i = 0; i < DL; i++) {
                    const float v = V[k * PITCH + lane + 32 * i];
#pragma unroll
                    for (int r = 0; r < RB; r++)
                        if (full || w[r] != 0.f) o[r][i] += w[r] * v;
                }
            }
            __syncwarp();
            row = next;
            next = after;
        }
        // the warps' parts meet in their (idle) stages
        __syncwarp();
#pragma unroll
        for (int r = 0; r < RB; r++) {
            l[r] = warp_sum(l[r]);
            if (lane == 0) part_m[warp][r] = m[r], part_l[warp][r] = l[r];
#pragma unroll
            for (int i = 0; i < DL; i++)
                if (lane + 32 * i < D) ring[r * D + lane + 32 * i] = o[r][i];
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == sp.tiles;
        float *part = p.ws + (((size_t)blockIdx.y * ctas + cta) * 2 + (first ? 0 : 1)) * RB * (D + 2);
        for (int i = threadIdx.x; i < rows * D; i += W * 32) {
            const int r = i / D;
            float top = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, part_m[w][r]);
            const float ref = merge_reference(top);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float f = expf(part_m[w][r] - ref);
                L += part_l[w][r] * f;
                O += sm[RB * PITCH + w * (2 * 2 * TILE * PITCH) + i] * f;
            }
            if (whole) {
                reinterpret_cast<T *>(p.out)[place(b, h, r0 + r, i - r * D)] = from_f32<T>(paged_quotient(O, L));
            } else {
                part[i] = O;
                if (i == r * D) part[RB * D + r] = top, part[RB * D + RB + r] = L;
            }
        }
        __syncthreads();
        // the stages' columns behind D are zeros again
        for (int i = lane; i < 2 * 2 * TILE * PITCH; i += 32) ring[i] = 0.f;
        left -= t1 - t0;
        t0 = 0;
        if (++h == p.G) {
            h = 0;
            b++;
        }
    }
}

// ---- parts of pairs that lie in several CTAs ------------------------------------------------------------------------------
constexpr int kJoinThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const PagedAttention p, int ctas) {
    __shared__ long long sums[2][kJoinThreads / 32];
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x / p.G, h = blockIdx.x - b * p.G, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    long long total = 0, before = 0;
    for (int i = threadIdx.x; i < p.B; i += kJoinThreads) {
        const long long n = (long long)paged_span(p, i).tiles * p.G;
        total += n;
        if (i < b) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) sums[0][warp] = total, sums[1][warp] = before;
    __syncthreads();
    total = before = 0;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; w++) total += sums[0][w], before += sums[1][w];
    const int tiles = paged_span(p, b).tiles;
    const long long share = paged_share(total, ctas, p.round), begin = before + (long long)h * tiles;
    if (tiles == 0) return;
    const int c0 = (int)(begin / share), c1 = (int)((begin + tiles - 1) / share);
    if (c0 == c1) return;
    const int R = p.block_rows, r0 = blockIdx.y * R, rows = min(p.group * p.S - r0, R), D = p.D;
    const int slot = begin > c0 * share ? 1 : 0;
    const float *parts = p.ws + (size_t)blockIdx.y * ctas * 2 * R * (D + 2);
    auto part = [&](int c) { return parts + ((size_t)c * 2 + (c == c0 ? slot : 0)) * R * (D + 2); };
    for (int i = threadIdx.x; i < rows * D; i += kJoinThreads) {
        const int r = i / D;
        float top = -INFINITY, L = 0.f, O = 0.f;
        for (int c = c0; c <= c1; c += 8) {
            float ms[8], ls[8], os[8], now = top;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool in = c + j <= c1;
                const float *from = part(in ? c + j : c1);
                ms[j] = in ? from[R * D + r] : -INFINITY;
                ls[j] = in ? from[R * D + R + r] : 0.f;
                os[j] = in ? from[i] : 0.f;
                now = fmaxf(now, ms[j]);
            }
            const float ref = merge_reference(now), keep = expf(top - ref);
            L *= keep;
            O *= keep;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float f = expf(ms[j] - ref);
                L += ls[j] * f;
                O += os[j] * f;
            }
            top = now;
        }
        const int row = r0 + r;
        reinterpret_cast<T *>(p.out)[(((size_t)b * p.S + row % p.S) * p.Hq + h * p.group + row / p.S) * D + i - r * D] = from_f32<T>(paged_quotient(O, L));
    }
}

struct PagedPlan {
    int ctas, block_rows, row_blocks, round;
};

static int paged_sms(int *sms) {
    int dev = 0;
    MYNN_CUDA_OK(cudaGetDevice(&dev));
    MYNN_CUDA_OK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return MYNN_OK;
}

static PagedPlan paged_plan(int B, int S, int Hq, int Hkv, int D, int page, int width, int sms) {
    PagedPlan n;
    n.block_rows = kPlainRows;
    n.row_blocks = (int)(((long long)Hq / Hkv * S + n.block_rows - 1) / n.block_rows);
    n.round = D > 128 ? kPlainWarps<8> : kPlainWarps<4>;
    const long long tiles = ((long long)width * page + kPagedTile - 1) / kPagedTile * Hkv * B;
    n.ctas = (int)std::min<long long>(sms, std::max<long long>(1, (tiles + n.round - 1) / n.round));
    return n;
}

template <typename T, int DL>
static int launch_plain(cudaStream_t st, const PagedAttention &p, int ctas, int vec) {
    const dim3 grid(ctas, p.row_blocks), block(kPlainWarps<DL> * 32);
    auto go = [&](auto kern) -> int {
        MYNN_CUDA_OK(cudaFuncSetAttribute((const void *)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plain_smem<DL>()));
        MYNN_CUDA_OK(launch_dependent(kern, grid, block, plain_smem<DL>(), st, p));
        MYNN_LAUNCH_OK("paged_attention_plain_kernel");
        return MYNN_OK;
    };
    if constexpr (std::is_same<T, float>::value) return vec == 4 ? go(paged_attention_plain_kernel<T, DL, 4>) : go(paged_attention_plain_kernel<T, DL, 1>);
    else return go(paged_attention_plain_kernel<T, DL, 0>);
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
    const PagedPlan n = paged_plan(B, S, Hq, Hkv, D, page, table_pages, sms);
    return (size_t)n.ctas * n.row_blocks * 2 * n.block_rows * (D + 2) * sizeof(float);
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
    int sms = 0;
    if (const int e = paged_sms(&sms)) return e;
    const PagedPlan n = paged_plan(B, S, Hq, Hkv, D, page, table_pages, sms);
    const size_t need = (size_t)n.ctas * n.row_blocks * 2 * n.block_rows * (D + 2) * sizeof(float);
    if (!workspace || workspace_bytes < need) return fail(MYNN_E_ARG, "paged_attention: workspace of %zu bytes, %zu are needed", workspace_bytes, need);
    if ((uintptr_t)workspace % 16) return fail(MYNN_E_ARG, "paged_attention: the workspace is not aligned to 16 bytes");
    PagedAttention p;
    p.out = out, p.q = q, p.k = k_pages, p.v = v_pages;
    p.table = block_table, p.lengths = lengths, p.counts = counts;
    p.scale = scale, p.softcap = softcap, p.window = std::min(window, kPagedWindow), p.sinks = sinks;
    p.B = B, p.S = S, p.Hq = Hq, p.G = Hkv, p.group = Hq / Hkv, p.D = D;
    p.page = page, p.pages = pages, p.width = table_pages;
    p.row_blocks = n.row_blocks, p.block_rows = n.block_rows, p.round = n.round;
    p.ws = reinterpret_cast<float *>(workspace);
    const cudaStream_t st = (cudaStream_t)stream;
    const int vec = D % 4 == 0 && ((uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0 ? 4 : 1;
    MYNN_DISPATCH_DTYPE(dtype, T, {
        int e;
        if (D <= 32) e = launch_plain<T, 1>(st, p, n.ctas, vec);
        else if (D <= 64) e = launch_plain<T, 2>(st, p, n.ctas, vec);
        else if (D <= 96) e = launch_plain<T, 3>(st, p, n.ctas, vec);
        else if (D <= 128) e = launch_plain<T, 4>(st, p, n.ctas, vec);
        else e = launch_plain<T, 8>(st, p, n.ctas, vec);
        if (e != MYNN_OK) return e;
        MYNN_CUDA_OK(launch_dependent(paged_attention_join_kernel<T>, dim3(B * Hkv, n.row_blocks), dim3(kJoinThreads), 0, st, p, n.ctas));
        MYNN_LAUNCH_OK("paged_attention_join_kernel");
    });
    return MYNN_OK;
}
