// The step between the q/k/v projection and attention over a paged cache: rotation of the new tokens' q and k, their division by the root mean square
// per head, and the append to the pages, in one launch.  Every sequence has a length and a number of new tokens of its own.
//
// One warp takes one head of one token: rotated dimension i and its partner are half a rotated range apart or next door, so a head is staged as f32 in shared memory;
// rotation and norm are f32, the result is rounded once.
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

template <typename T>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_append_kernel(const PagedAppend p) {
    extern __shared__ float sm[];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = p.Hq + 2 * p.G;
    const long long job = (long long)blockIdx.x * kAppendWarps + warp, token = job / heads;
    if (token >= (long long)p.B * p.S) return;
    const int head = (int)(job - token * heads), b = (int)(token / p.S), s = (int)(token - (long long)b * p.S);
    const int len = max(p.lengths[b], 0), count = p.counts ? min(max(p.counts[b], 0), p.S) : p.S;
    const int pos = len - count + s;
    const bool real = s < count && pos >= 0 && pos < p.width * p.page && (p.rot_dims == 0 || pos < p.positions);
    const T *src = reinterpret_cast<const T *>(p.proj) + (size_t)job * p.D;
    T *dst;
    if (head < p.Hq) {
        dst = reinterpret_cast<T *>(p.q_out) + (((size_t)b * p.Hq + head) * p.S + s) * p.D;
        if (!real) {
            for (int d = lane; d < p.D; d += 32) dst[d] = from_f32<T>(0.f);
            return;
        }
    } else {
        if (!real) return;
        const int i = pos / p.page, pg = p.table[(size_t)b * p.width + i], kv = (head - p.Hq) % p.G;
        if ((unsigned)pg >= (unsigned)p.pages) return;
        dst = reinterpret_cast<T *>(head < p.Hq + p.G ? p.k : p.v) + (((size_t)pg * p.G + kv) * p.page + pos - i * p.page) * p.D;
        if (head >= p.Hq + p.G) {
            for (int d = lane; d < p.D; d += 32) dst[d] = src[d];
            return;
        }
    }
    float *x = sm + (size_t)warp * p.D;
    for (int d = lane; d < p.D; d += 32) x[d] = to_f32<T>(src[d]);
    __syncwarp();
    const int half = p.rot_dims >> 1;
    const float *cs = p.cos_t + (size_t)pos * half, *sn = p.sin_t + (size_t)pos * half;
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
    MYNN_DISPATCH_DTYPE(dtype, T, {
        MYNN_CUDA_OK(launch_dependent(paged_append_kernel<T>, dim3((unsigned)blocks), dim3(kAppendWarps * 32), (size_t)kAppendWarps * D * sizeof(float),
                                      (cudaStream_t)stream, p));
    });
    MYNN_LAUNCH_OK("paged_append_kernel");
    return MYNN_OK;
}
