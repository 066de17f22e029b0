// The step between the q/k/v projection and attention over a paged cache: rotation of the new tokens' q and k, their division by the root mean square
// per head, and the append to the pages, in one launch.  Every sequence has a length and a number of new tokens of its own.
//
// Rotation and norm are f32, the result is rounded once.  A CTA takes one token.  Where heads come in pieces of eight numbers, a thread holds two pieces: piece i of
// the rotated half and its partner half a rotated range away, or two neighbours; it does so for one head after the other, so a token's angles are read once per
// thread, and a head's norm is a sum over the few threads that share it.  Other sizes (paged_append_any_kernel): a warp per head, staged in shared memory.
// Bound by bytes for prompts and by the chain of lengths, table and store for a step: 32 tokens of 48 heads of 128 take 2.4 us (a warp per head: 6.7), 6 prompts of 777
// places that are mostly padding, whose zero queries are 38 MB, 10.6 us (read before it was known that they are padding: 24), 2048 tokens 8.9 us = 0.86 of the copy
// bandwidth.
#include <algorithm>

#include "common.cuh"
#include "paged.cuh"

namespace mynn {

struct PagedAppend {
    void *q_out, *k, *v;
    const void *proj;
    const float *cos_t, *sin_t;
    const int32_t *lengths, *counts, *table;
    int B, S, Hq, G, D;
    int rot_dims, halves, qk_norm;
    float eps;
    int page, pages, width, positions;
};

constexpr int kAppendWarps = 8;

struct AppendToken {
    int b, s, pos;
    bool real;
    size_t row;   // of the cache for kv head 0 (heads are `page` rows apart)
    bool stored;  // the table names a page
};

__device__ __forceinline__ AppendToken append_token(const PagedAppend &p, int b, int s) {
    AppendToken k = {b, s, 0, false, 0, false};
    const int len = max(p.lengths[b], 0), count = p.counts ? min(max(p.counts[b], 0), p.S) : p.S;
    k.pos = len - count + s;
    k.real = s < count && k.pos >= 0 && k.pos < p.width * p.page && (p.rot_dims == 0 || k.pos < p.positions);
    if (k.real) {
        const int i = k.pos / p.page, pg = p.table[(size_t)b * p.width + i];
        k.stored = (unsigned)pg < (unsigned)p.pages;
        k.row = k.stored ? (size_t)pg * p.G * p.page + (k.pos - i * p.page) : 0;
    }
    return k;
}

// Eight numbers as they come from or go to memory.
template <typename T>
struct Piece {
    static constexpr int N = 8 * sizeof(T) / 16;
    uint4 raw[N];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < N; i++) raw[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int i = 0; i < N; i++) reinterpret_cast<uint4 *>(p)[i] = raw[i];
    }
    __device__ __forceinline__ float at(int i) const { return to_f32<T>(reinterpret_cast<const T *>(raw)[i]); }
    __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T *>(raw)[i] = from_f32<T>(v); }
};

// grid (S, B); a group of `lanes` threads (a power of two) per head, thread i of it with pieces c0 and c1.  D a multiple of 16, rot_dims of 16 (halves) or 8.
template <typename T>
__global__ void __launch_bounds__(512, 2) paged_append_kernel(const PagedAppend p, int lanes) {
    pdl_trigger();
    pdl_wait();
    const int s = blockIdx.x, b = blockIdx.y, sub = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = blockDim.x / lanes;
    const int heads = p.Hq + 2 * p.G, half = p.rot_dims >> 1, pairs = p.D / 16;
    const bool in = sub < pairs;
    const unsigned sharers = (0xffffffffu >> (32 - lanes)) << (threadIdx.x & 31 & ~(lanes - 1));  // the threads of this head
    // with halves the first half / 8 threads have partners, the others two pieces behind the rotated range
    const bool split = p.halves && sub < half / 8;
    const int d0 = split ? 8 * sub : 16 * sub, d1 = split ? d0 + half : d0 + 8;
    const T *src = reinterpret_cast<const T *>(p.proj) + ((size_t)b * p.S + s) * heads * p.D;
    Piece<T> x0, x1;
    // A place without a token is not read, and only its queries are written.
    if (p.counts && s >= p.counts[b]) {
        const uint4 z = make_uint4(0, 0, 0, 0);
        T *dst = reinterpret_cast<T *>(p.q_out) + ((size_t)b * p.Hq * p.S + s) * p.D;
        for (int i = 0; i < Piece<T>::N; i++) x0.raw[i] = z;
        if (in)
            for (int head = group; head < p.Hq; head += groups) x0.store(dst + (size_t)head * p.S * p.D + d0), x0.store(dst + (size_t)head * p.S * p.D + d1);
        return;
    }
    if (in && group < heads) x0.load(src + (size_t)group * p.D + d0), x1.load(src + (size_t)group * p.D + d1);
    const AppendToken k = append_token(p, b, s);
    // angles of the pairs in the two pieces: halves (d0 + i, d1 + i), else (d0 + 2 i, d0 + 2 i + 1) and the same in the second piece
    float c[8], a[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = 1.f, a[i] = 0.f;
    if (in && k.real && p.rot_dims > 0) {
        const float *cs = p.cos_t + (size_t)k.pos * half, *sn = p.sin_t + (size_t)k.pos * half;
        const int first = split ? d0 : d0 / 2;
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (split || (!p.halves && first + i < half)) c[i] = cs[first + i], a[i] = sn[first + i];
    }
    for (int head = group; head < heads; head += groups) {
        Piece<T> y0, y1;
        const bool key = head < p.Hq + p.G;
        if (key && k.real) {
            float u[8], w[8], ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = in ? x0.at(i) : 0.f, w[i] = in ? x1.at(i) : 0.f;
            if (split) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float lo = rope_low(u[i], w[i], c[i], a[i]), hi = rope_high(u[i], w[i], c[i], a[i]);
                    u[i] = lo, w[i] = hi;
                }
            } else if (!p.halves && p.rot_dims > 0) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (d0 + 2 * i < p.rot_dims) {
                        const float lo = rope_low(u[2 * i], u[2 * i + 1], c[i], a[i]), hi = rope_high(u[2 * i], u[2 * i + 1], c[i], a[i]);
                        u[2 * i] = lo, u[2 * i + 1] = hi;
                    }
                    if (d1 + 2 * i < p.rot_dims) {
                        const float lo = rope_low(w[2 * i], w[2 * i + 1], c[4 + i], a[4 + i]), hi = rope_high(w[2 * i], w[2 * i + 1], c[4 + i], a[4 + i]);
                        w[2 * i] = lo, w[2 * i + 1] = hi;
                    }
                }
            }
            float inv = 1.f;
            if (p.qk_norm) {
#pragma unroll
                for (int i = 0; i < 8; i++) ss += u[i] * u[i] + w[i] * w[i];
                for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(sharers, ss, o);
                inv = 1.0f / sqrtf(ss / (float)p.D + p.eps);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) y0.set(i, u[i] * inv), y1.set(i, w[i] * inv);
        } else {
            y0 = x0, y1 = x1;
        }
        if (in) {
            T *dst = nullptr;
            if (head < p.Hq) {
                dst = reinterpret_cast<T *>(p.q_out) + (((size_t)b * p.Hq + head) * p.S + s) * p.D;
                if (!k.real)
#pragma unroll
                    for (int i = 0; i < 8; i++) y0.set(i, 0.f), y1.set(i, 0.f);
            } else if (k.stored) {
                const int kv = head - p.Hq - (key ? 0 : p.G);
                dst = reinterpret_cast<T *>(key ? p.k : p.v) + (k.row + (size_t)kv * p.page) * p.D;
            }
            if (dst) y0.store(dst + d0), y1.store(dst + d1);
            const int next = head + groups;
            if (next < heads) x0.load(src + (size_t)next * p.D + d0), x1.load(src + (size_t)next * p.D + d1);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_append_any_kernel(const PagedAppend p) {
    extern __shared__ float sm[];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = p.Hq + 2 * p.G;
    const long long job = (long long)blockIdx.x * kAppendWarps + warp, token = job / heads;
    if (token >= (long long)p.B * p.S) return;
    const int head = (int)(job - token * heads), b = (int)(token / p.S), s = (int)(token - (long long)b * p.S);
    const AppendToken k = append_token(p, b, s);
    const T *src = reinterpret_cast<const T *>(p.proj) + (size_t)job * p.D;
    T *dst;
    if (head < p.Hq) {
        dst = reinterpret_cast<T *>(p.q_out) + (((size_t)b * p.Hq + head) * p.S + s) * p.D;
        if (!k.real) {
            for (int d = lane; d < p.D; d += 32) dst[d] = from_f32<T>(0.f);
            return;
        }
    } else {
        if (!k.stored) return;
        const int kv = (head - p.Hq) % p.G;
        dst = reinterpret_cast<T *>(head < p.Hq + p.G ? p.k : p.v) + (k.row + (size_t)kv * p.page) * p.D;
        if (head >= p.Hq + p.G) {
            for (int d = lane; d < p.D; d += 32) dst[d] = src[d];
            return;
        }
    }
    float *x = sm + (size_t)warp * p.D;
    for (int d = lane; d < p.D; d += 32) x[d] = to_f32<T>(src[d]);
    __syncwarp();
    const int half = p.rot_dims >> 1;
    const float *cs = p.cos_t + (size_t)k.pos * half, *sn = p.sin_t + (size_t)k.pos * half;
    for (int i = lane; i < half; i += 32) {
        const int lo = p.halves ? i : 2 * i, hi = p.halves ? i + half : 2 * i + 1;
        const float a = x[lo], c = x[hi];
        x[lo] = rope_low(a, c, cs[i], sn[i]);
        x[hi] = rope_high(a, c, cs[i], sn[i]);
    }
    __syncwarp();
    float inv = 1.f;
    if (p.qk_norm) {
        float ss = 0.f;
        for (int d = lane; d < p.D; d += 32) ss += x[d] * x[d];
        inv = 1.0f / sqrtf(warp_sum(ss) / (float)p.D + p.eps);
    }
    for (int d = lane; d < p.D; d += 32) dst[d] = from_f32<T>(x[d] * inv);
}

}  // namespace mynn

using namespace mynn;

extern "C" int mynn_b200_paged_rotary_append(void *stream, void *q_out, void *k_pages, void *v_pages, const void *proj, const float *cos_table,
                                             const float *sin_table, const int32_t *lengths, const int32_t *counts, const int32_t *block_table, int B,
                                             int S, int Hq, int Hkv, int D, int rot_dims, int halves, int qk_norm, float eps, int page, int pages,
                                             int table_pages, int positions, int dtype) {
    if (B < 0 || S < 1 || Hq < 1 || Hkv < 1 || D < 1 || page < 1 || pages < 0 || table_pages < 1 || rot_dims < 0 || rot_dims > D || rot_dims % 2 || positions < 0)
        return fail(MYNN_E_ARG, "paged_rotary_append: bad shape");
    if (!dtype_ok(dtype)) return fail(MYNN_E_ARG, "paged_rotary_append: bad dtype %d", dtype);
    if (S > 1 << 24) return fail(MYNN_E_UNSUPPORTED, "paged_rotary_append: %d new tokens", S);
    if ((long long)page * table_pages > INT_MAX - 64) return fail(MYNN_E_UNSUPPORTED, "paged_rotary_append: %lld positions per sequence", (long long)page * table_pages);
    if (D > 1024) return fail(MYNN_E_UNSUPPORTED, "paged_rotary_append: heads of %d", D);
    const long long blocks = ((long long)B * S * ((long long)Hq + 2ll * Hkv) + kAppendWarps - 1) / kAppendWarps;
    if (blocks > INT_MAX) return fail(MYNN_E_UNSUPPORTED, "paged_rotary_append: %d x %d tokens", B, S);
    if (B == 0) return MYNN_OK;
    if (!q_out || !proj || !lengths || !block_table || (pages && (!k_pages || !v_pages)) || (rot_dims && (!cos_table || !sin_table)))
        return fail(MYNN_E_ARG, "paged_rotary_append: null pointer");
    PagedAppend p;
    p.q_out = q_out, p.k = k_pages, p.v = v_pages, p.proj = proj;
    p.cos_t = cos_table, p.sin_t = sin_table;
    p.lengths = lengths, p.counts = counts, p.table = block_table;
    p.B = B, p.S = S, p.Hq = Hq, p.G = Hkv, p.D = D;
    p.rot_dims = rot_dims, p.halves = halves, p.qk_norm = qk_norm, p.eps = eps;
    p.page = page, p.pages = pages, p.width = table_pages, p.positions = positions;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool pieces = D % 16 == 0 && D <= 512 && rot_dims % (halves ? 16 : 8) == 0 && B <= 65535 &&
                        ((uintptr_t)proj | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages) % 16 == 0;
    if (pieces) {
        int lanes = 1;
        while (lanes < D / 16) lanes *= 2;
        // A step wants each head to begin at once, prompts want many CTAs side by side, since each begins with a chain of loads.  48 heads of 128, bf16, with 64 / 128 / 192 / 512
        // threads: 32 tokens 4.2 / 3.0 / 2.6 / 2.5 us, 512 tokens 6.2 / 5.3 / 4.4 / 4.9, 2048 tokens 9.2 / 8.9 / 10.0 / 15.0, 4662 places that are mostly padding 16 / 12.0 / 10.6 / 14.0.
        // Places with counts are taken to be mostly padding, since the host does not know them: prompts of one length are better off without counts (8.9 instead of 10.0 us).
        const long long tokens = (long long)B * S;
        const int threads = (int)std::min<long long>(tokens < 300 ? 512 : tokens < 1024 || counts ? 192 : 128, ((long long)(Hq + 2 * Hkv) * lanes + 31) / 32 * 32);
        MYNN_DISPATCH_DTYPE(dtype, T, { MYNN_CUDA_OK(launch_dependent(paged_append_kernel<T>, dim3(S, B), dim3(threads), 0, st, p, lanes)); });
        MYNN_LAUNCH_OK("paged_append_kernel");
        return MYNN_OK;
    }
    MYNN_DISPATCH_DTYPE(dtype, T, {
        MYNN_CUDA_OK(launch_dependent(paged_append_any_kernel<T>, dim3((unsigned)blocks), dim3(kAppendWarps * 32), (size_t)kAppendWarps * D * sizeof(float), st, p));
    });
    MYNN_LAUNCH_OK("paged_append_any_kernel");
    return MYNN_OK;
}
