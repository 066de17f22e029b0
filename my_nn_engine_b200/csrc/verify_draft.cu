// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft token x_i stands while u_i q_i(x_i) < p_i(x_i); the first one that does not, n, is replaced by a draw from max(p_n - q_n, 0), and behind K standing tokens
// comes a draw from p_K: the first token whose running sum exceeds r times the whole sum.  So the tokens are distributed as the target's own.
//
// Of (2 K + 1) V probabilities only the one or two rows of the draw are read whole.  A cluster of up to eight CTAs takes a sequence, each CTA a range of the vocabulary and each
// warp a part of it: sums per warp, then which CTA's and which warp's part the running sum ends in, then that part again, from L2.  A difference of two
// f32 numbers and sums of 1e5 of them decide on whole numbers, so they are held in 64 bits: a sum in f32 is off by more than many a token's
// probability.  The order of the sums is fixed.
#include "common.cuh"
#include "tcgen05.cuh"

namespace mynn {

struct VerifyDraft {
    int32_t *tokens_out, *accepted_out;
    const void *target, *draft;  // draft null: the drafted tokens are certain
    const int32_t *tokens, *counts;
    const float *accept, *sample;
    int B, K, V;
};

constexpr int kVerifyWarps = 8;

__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The row that the token is drawn from: p - q, or p without one token; what is not positive has no weight.
template <typename T>
struct DrawRow {
    const T *p, *q;  // q may be null
    int without;
    __device__ __forceinline__ double weight(float a, float c, int i) const {
        const double w = (double)a - (double)c;
        return i != without && w > 0.0 ? w : 0.0;
    }
};

// Numbers at + VEC * lane + 32 VEC u (u < U) of the row's two parts, zeros from `end` on.
template <typename T, int VEC, int U>
struct DrawPieces {
    __align__(16) T a[U][VEC], c[U][VEC];
    __device__ __forceinline__ void load(const DrawRow<T> &row, int at, int end, int lane) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = at + VEC * (lane + 32 * u);
            if constexpr (VEC > 1) {
                *reinterpret_cast<uint4 *>(a[u]) = i < end ? __ldg(reinterpret_cast<const uint4 *>(row.p + i)) : make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4 *>(c[u]) = row.q && i < end ? __ldg(reinterpret_cast<const uint4 *>(row.q + i)) : make_uint4(0, 0, 0, 0);
            } else {
                a[u][0] = i < end ? row.p[i] : from_f32<T>(0.f);
                c[u][0] = row.q && i < end ? row.q[i] : from_f32<T>(0.f);
            }
        }
    }
    __device__ __forceinline__ double weight(const DrawRow<T> &row, int at, int lane, int u, int e) const {
        return row.weight(to_f32<T>(a[u][e]), to_f32<T>(c[u][e]), at + VEC * (lane + 32 * u) + e);
    }
};

// grid (cluster, B).  VEC: elements of a 16-byte piece where all rows begin on 16 bytes, else 1.
template <typename T, int VEC>
__global__ void __launch_bounds__(kVerifyWarps * 32, 4) verify_draft_kernel(const VerifyDraft p) {
    constexpr int U = VEC == 1 ? 8 : 2;  // pieces of a lane in flight per row: 8 x 1, 2 x 4 or 2 x 8 numbers
    constexpr int STEP = 32 * VEC * U, GROUPS = 4;
    __shared__ double sums[kVerifyWarps], whole[2];
    __shared__ int pick;
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.y, rank = blockIdx.x, ranks = gridDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = p.K, V = p.V;
    const int drafts = p.counts ? min(max(p.counts[b], 0), K) : K;
    const T *target = reinterpret_cast<const T *>(p.target) + (size_t)b * (K + 1) * V;
    const T *draft = p.draft ? reinterpret_cast<const T *>(p.draft) + (size_t)b * K * V : nullptr;
    const float sample = p.sample[b];
    int n = drafts;  // drafts that stand: every warp looks for itself
    for (int i0 = 0; i0 < drafts; i0 += 32) {
        const int i = i0 + lane;
        bool falls = false;
        if (i < drafts) {
            const int x = p.tokens[(size_t)b * K + i];
            const float u = p.accept[(size_t)b * K + i];
            falls = true;
            if ((unsigned)x < (unsigned)V) {
                const double q = draft ? (double)to_f32<T>(draft[(size_t)i * V + x]) : 1.0;
                falls = !((double)u * q < (double)to_f32<T>(target[(size_t)i * V + x]));  // (24 by 24 bits: exact)
            }
        }
        const unsigned any = __ballot_sync(0xffffffffu, falls);
        if (any) {
            n = i0 + __ffs(any) - 1;
            break;
        }
    }
    DrawRow<T> row = {target + (size_t)n * V, n < drafts && draft ? draft + (size_t)n * V : nullptr, n < drafts && !draft ? p.tokens[(size_t)b * K + n] : -1};
    // parts of whole steps: the cluster's ranks in order, in each its warps
    const int parts = ranks * kVerifyWarps, per = ((V + parts - 1) / parts + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
    const int lo = (int)min((long long)(rank * kVerifyWarps + warp) * per, (long long)V), hi = min(lo + per, V);
    const int stride = (per + GROUPS * STEP - 1) / (GROUPS * STEP) * STEP;  // a part is summed in up to four groups, so that little of it is read again
    double group[GROUPS];
    double total = 0.0, before = 0.0, mine = 0.0;
    bool chosen = false;
    for (int pass = 0;; pass++) {
#pragma unroll
        for (int k = 0; k < GROUPS; k++) {
            group[k] = 0.0;
            const int end = min(lo + (k + 1) * stride, hi);
#pragma unroll 1
            for (int at = lo + k * stride; at < end; at += STEP) {
                DrawPieces<T, VEC, U> x;
                x.load(row, at, end, lane);
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < VEC; e++) group[k] += x.weight(row, at, lane, u, e);
            }
        }
#pragma unroll
        for (int k = 0; k < GROUPS; k++) group[k] = warp_sum_f64(group[k]);
        if (lane == 0) sums[warp] = (group[0] + group[1]) + (group[2] + group[3]);
        __syncthreads();
        mine = 0.0;
#pragma unroll
        for (int i = 0; i < kVerifyWarps; i++) mine += sums[i];
        if (threadIdx.x == 0) whole[pass] = mine;
        cluster_sync_all();
        // where the running sum exceeds sample * total; if it never does (the product was rounded up to the total) the last part with any weight
        double part[8];
#pragma unroll
        for (int r = 0; r < 8; r++) part[r] = r < ranks ? ld_cluster_f64(map_rank(smem_u32(&whole[pass]), r)) : 0.0;
        total = 0.0;
#pragma unroll
        for (int r = 0; r < 8; r++) total += part[r];
        const double goal = (double)sample * total;
        double run = 0.0;
        int at = -1;
#pragma unroll
        for (int r = 0; r < 8; r++) {
            if (part[r] > 0.0 && (at < 0 || run <= goal)) {
                at = r;
                before = run;
                run += part[r];
            }
        }
        chosen = at == rank;
        if (total > 0.0 || pass == 1 || (!row.q && row.without < 0)) break;
        row.q = nullptr;  // nothing is left of the target where the draft is taken off: the draw is from the target itself
        row.without = -1;
        __syncthreads();  // the sums have been read
    }
    if (chosen || (rank == 0 && !(total > 0.0))) {
        const double goal = (double)sample * total;
        if (threadIdx.x == 0) pick = -1;
        __syncthreads();
        double run = before;
        int at = -1;
#pragma unroll
        for (int i = 0; i < kVerifyWarps; i++) {
            if (sums[i] > 0.0 && (at < 0 || run <= goal)) {
                at = i;
                before = run;
                run += sums[i];
            }
        }
        if (chosen && warp == at) {
            int found = -1, k0 = -1;
            run = before;
#pragma unroll
            for (int k = 0; k < GROUPS; k++) {
                if (group[k] > 0.0 && (k0 < 0 || run <= goal)) {
                    k0 = k;
                    before = run;
                    run += group[k];
                }
            }
            const int from = lo + k0 * stride, end = min(from + stride, hi);
#pragma unroll 1
            for (int base = from; base < end && found < 0; base += 32 * VEC * U) {
                DrawPieces<T, VEC, U> x;
                double own[U];
                x.load(row, base, end, lane);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    own[u] = 0.0;
#pragma unroll
                    for (int e = 0; e < VEC; e++) own[u] += x.weight(row, base, lane, u, e);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const double all = warp_sum_f64(own[u]);
                    if (found >= 0) continue;
                    if (!(before + all > goal)) {
                        before += all;
                        continue;
                    }
                    double incl = own[u];
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double up = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += up;
                    }
                    double sum = before + (incl - own[u]);
                    int over = -1;
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const double w = x.weight(row, base, lane, u, e);
                        sum += w;
                        if (over < 0 && w > 0.0 && sum > goal) over = e;
                    }
                    const unsigned overs = __ballot_sync(0xffffffffu, over >= 0);
                    if (overs) {
                        const int l = __ffs(overs) - 1;
                        found = base + VEC * (l + 32 * u) + __shfl_sync(0xffffffffu, over, l);
                    }
                    before += all;
                }
            }
            if (found < 0) {  // sums in another order, or a goal that was rounded up to the total: the last token with any weight
                int last = -1;
                for (int i = from + lane; i < end; i += 32)
                    if (row.weight(to_f32<T>(row.p[i]), row.q ? to_f32<T>(row.q[i]) : 0.f, i) > 0.0) last = i;
                found = __reduce_max_sync(0xffffffffu, last);
            }
            if (lane == 0) pick = found;
        }
        __syncthreads();
        for (int i = threadIdx.x; i <= K; i += kVerifyWarps * 32) p.tokens_out[(size_t)b * (K + 1) + i] = i < n ? p.tokens[(size_t)b * K + i] : i == n ? pick : -1;
        if (threadIdx.x == 0) p.accepted_out[b] = n;
    }
    cluster_sync_all();  // nobody leaves while its sums may still be read
}

}  // namespace mynn

using namespace mynn;

extern "C" int mynn_b200_verify_draft(void *stream, int32_t *tokens_out, int32_t *accepted_out, const void *target, const void *draft, const int32_t *tokens,
                                      const int32_t *counts, const float *accept, const float *sample, int B, int K, int V, int dtype) {
    if (B < 0 || K < 0 || V < 1) return fail(MYNN_E_ARG, "verify_draft: bad shape");
    if (!dtype_ok(dtype)) return fail(MYNN_E_ARG, "verify_draft: bad dtype %d", dtype);
    if (K > 1024 || V > 1 << 30 || B > 65535) return fail(MYNN_E_UNSUPPORTED, "verify_draft: %d sequences of %d drafted tokens of a vocabulary of %d", B, K, V);
    if (B == 0) return MYNN_OK;
    if (!tokens_out || !accepted_out || !target || !sample || (K && (!tokens || !accept))) return fail(MYNN_E_ARG, "verify_draft: null pointer");
    VerifyDraft p;
    p.tokens_out = tokens_out, p.accepted_out = accepted_out;
    p.target = target, p.draft = draft;
    p.tokens = tokens, p.counts = counts;
    p.accept = accept, p.sample = sample;
    p.B = B, p.K = K, p.V = V;
    // As many CTAs per sequence as keep a warp's part at a step or more.
    int ranks = 1;
    while (ranks < 8 && (long long)V >= 2ll * ranks * kVerifyWarps * 256) ranks *= 2;
    const dim3 grid(ranks, B), block(kVerifyWarps * 32);
    const cudaStream_t st = (cudaStream_t)stream;
    MYNN_DISPATCH_DTYPE(dtype, T, {
        constexpr int VEC = 16 / sizeof(T);
        const bool vec = V % VEC == 0 && ((uintptr_t)target | (uintptr_t)draft) % 16 == 0;
        if (vec) MYNN_CUDA_OK(launch_ex(true, ranks, verify_draft_kernel<T, VEC>, grid, block, 0, st, p));
        else MYNN_CUDA_OK(launch_ex(true, ranks, verify_draft_kernel<T, 1>, grid, block, 0, st, p));
    });
    MYNN_LAUNCH_OK("verify_draft_kernel");
    return MYNN_OK;
}
