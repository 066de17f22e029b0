// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft token x_i stands while u_i q_i(x_i) < p_i(x_i); the first one that does not, n, is replaced by a draw from max(p_n - q_n, 0), and behind K standing tokens
// comes a draw from p_K: the first token whose running sum exceeds r times the whole sum.  So the tokens are distributed as the target's own.
//
// Of (2 K + 1) V probabilities only the one or two rows of the draw are read whole.  A cluster of up to eight CTAs takes a sequence, each CTA a range of the vocabulary and each
// warp a part of it: sums per warp, then which CTA's and which warp's part the running sum ends in, then that part again, from L2.  A difference of two
// f32 numbers and sums of 1e5 of them decide on whole numbers, so they are held in 64 bits: a sum in f32 is off by more than many a token's
// probability.  The order of the sums is fixed.
// Bound by the chain tokens - probabilities - row - sums - row again for few sequences (one over 32000 tokens: 6.5 us) and by too little on its way for many: 64 over
// 128256 tokens in f32 21 us (66 MB: 0.48 of the copy bandwidth), 200 over 50257 in bf16 18 us = 0.17.  45 % of the issue slots are used; warps wait for loads, one step of which is ahead of the sums (in 16
// bits one 16-byte load per lane), and for the cluster.
#include <type_traits>

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
        return i != without && a > c ? (double)a - (double)c : 0.0;
    }
};

// The draw's row in pieces of VEC numbers that begin on 16 bytes in p (VEC 1: single numbers).  In q, whose rows of an odd vocabulary begin elsewhere, such a piece
// lies in two; `shift` bytes into the first.  The numbers in front of the first piece and behind the last are taken one by one; they are so many that no
// piece reaches out of the row.
template <typename T, int VEC>
struct DrawPieces {
    DrawRow<T> row;
    int begin, end, shift;
    __device__ __forceinline__ void find(int V) {
        if constexpr (VEC == 1) {
            begin = 0, end = V, shift = 0;
        } else {
            const uintptr_t a = (uintptr_t)row.p, c = (uintptr_t)row.q;
            begin = (int)((16 - a % 16) % 16 / sizeof(T));
            shift = row.q ? (int)((c - a) % 16) : 0;
            if (shift && begin < VEC) begin += VEC;
            end = begin + (V - begin - (shift ? VEC : 0)) / VEC * VEC;
        }
    }
    // Numbers i .. i + VEC - 1 of p and of q as they lie in memory (zeros unless `in`).
    struct Raw {
        uint32_t a[VEC == 1 ? 1 : 4], c[VEC == 1 ? 1 : 4];
    };
    static __device__ __forceinline__ uint32_t bits(const T *x) {
        if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t *>(x);
        else return *reinterpret_cast<const uint16_t *>(x);
    }
    __device__ __forceinline__ void load(Raw &r, int i, bool in) const {
        if constexpr (VEC == 1) {
            r.a[0] = in ? bits(row.p + i) : 0u;
            r.c[0] = in && row.q ? bits(row.q + i) : 0u;
        } else {
            const uint4 z = make_uint4(0, 0, 0, 0), u = in ? __ldg(reinterpret_cast<const uint4 *>(row.p + i)) : z;
            r.a[0] = u.x, r.a[1] = u.y, r.a[2] = u.z, r.a[3] = u.w;
            const char *at = reinterpret_cast<const char *>(row.q + i) - shift;
            const uint4 v = in && row.q ? __ldg(reinterpret_cast<const uint4 *>(at)) : z;
            r.c[0] = v.x, r.c[1] = v.y, r.c[2] = v.z, r.c[3] = v.w;
            if (shift) {  // (of the whole row)
                const uint4 w = in ? __ldg(reinterpret_cast<const uint4 *>(at + 16)) : z;
                const uint32_t all[8] = {v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
                const unsigned sh = 8 * (shift & 3);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t lo = all[k], hi = all[k + 1];
#pragma unroll
                    for (int n = 1; n < 4; n++)
                        if (shift >> 2 == n) lo = all[k + n], hi = k + n + 1 < 8 ? all[k + n + 1] : 0u;
                    r.c[k] = __funnelshift_r(lo, hi, sh);
                }
            }
        }
    }
    static __device__ __forceinline__ float number(const uint32_t *x, int e) {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(x[e]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            return __uint_as_float(e & 1 ? x[e >> 1] & 0xffff0000u : x[e >> 1] << 16);
        } else {
            const uint16_t h = (uint16_t)(x[e >> 1] >> 16 * (e & 1));
            return __half2float(reinterpret_cast<const __half &>(h));
        }
    }
    // The weights of tokens i .. i + VEC - 1.  What is compared as f32 is subtracted only where it leaves something.
    __device__ __forceinline__ void weights(const Raw &r, int i, double (&w)[VEC]) const {
        if (row.q) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float a = number(r.a, e), c = number(r.c, e);
                const bool left = a > c;
                w[e] = (double)(left ? a : 0.f) - (double)(left ? c : 0.f);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) w[e] = (double)fmaxf(number(r.a, e), 0.f);  // (NaN: 0)
        }
        if ((unsigned)(row.without - i) < (unsigned)VEC) {
#pragma unroll
            for (int e = 0; e < VEC; e++)
                if (i + e == row.without) w[e] = 0.0;
        }
    }
    __device__ __forceinline__ double single(int i) const { return row.weight(to_f32<T>(row.p[i]), row.q ? to_f32<T>(row.q[i]) : 0.f, i); }
};

// One warp: the first token that the running sum exceeds the goal at, of 32 tokens whose weights the lanes hold in order; `before` moves on.  -1: none.
__device__ __forceinline__ int first_over(double own, double goal, double &before, int lane) {
    double incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, own > 0.0 && before + incl > goal);
    before += __shfl_sync(0xffffffffu, incl, 31);
    return over ? __ffs(over) - 1 : -1;
}

// grid (cluster, B).  VEC: numbers of a 16-byte piece, or 1 for small vocabularies.
template <typename T, int VEC>
__global__ void __launch_bounds__(kVerifyWarps * 32, 4) verify_draft_kernel(const VerifyDraft p) {
    constexpr int U = VEC == 1 ? 4 : 8 / VEC;  // pieces of a step and lane
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
    DrawPieces<T, VEC> x;
    x.row = {target + (size_t)n * V, n < drafts && draft ? draft + (size_t)n * V : nullptr, n < drafts && !draft ? p.tokens[(size_t)b * K + n] : -1};
    double total = 0.0, before = 0.0, group[GROUPS];
    bool chosen = false;
    int lo = 0, hi = 0, stride = 0;
    // the first warp of all has the numbers in front of the pieces as well, the last one those behind them
    const bool heads = rank == 0 && warp == 0, tails = rank == ranks - 1 && warp == kVerifyWarps - 1;
    for (int pass = 0;; pass++) {
        x.find(V);
        // parts of whole steps, the cluster's ranks in order, in each its warps; a part is summed in up to four groups, so that little of it is read again
        const int parts = ranks * kVerifyWarps, per = ((x.end - x.begin + parts - 1) / parts + 32 * VEC - 1) / (32 * VEC) * (32 * VEC);
        lo = (int)min(x.begin + (long long)(rank * kVerifyWarps + warp) * per, (long long)x.end);
        hi = min(lo + per, x.end);
        stride = (per + GROUPS * STEP - 1) / (GROUPS * STEP) * STEP;
#pragma unroll
        for (int k = 0; k < GROUPS; k++) group[k] = 0.0;
        if (heads && lane < x.begin) group[0] = x.single(lane);
        if (tails && lane < V - x.end) group[GROUPS - 1] = x.single(x.end + lane);
        typename DrawPieces<T, VEC>::Raw now[U], next[U];
        auto fetch = [&](typename DrawPieces<T, VEC>::Raw(&r)[U], int at) {
#pragma unroll
            for (int u = 0; u < U; u++) x.load(r[u], at + VEC * (lane + 32 * u), at + VEC * (lane + 32 * u) < hi);
        };
        if (lo < hi) fetch(now, lo);
#pragma unroll 1
        for (int at = lo, k = 0, left = stride; at < hi; at += STEP) {
            if (at + STEP < hi) fetch(next, at + STEP);  // on its way while this step is summed
            double sum = 0.0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                double w[VEC];
                x.weights(now[u], at + VEC * (lane + 32 * u), w);
#pragma unroll
                for (int e = 0; e < VEC; e++) sum += w[e];
            }
#pragma unroll
            for (int g = 0; g < GROUPS; g++) group[g] += g == k ? sum : 0.0;
#pragma unroll
            for (int u = 0; u < U; u++) now[u] = next[u];
            left -= STEP;
            if (left == 0) k++, left = stride;
        }
#pragma unroll
        for (int k = 0; k < GROUPS; k++) group[k] = warp_sum_f64(group[k]);
        if (lane == 0) sums[warp] = (group[0] + group[1]) + (group[2] + group[3]);
        __syncthreads();
        double mine = 0.0;
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
        if (total > 0.0 || pass == 1 || (!x.row.q && x.row.without < 0)) break;
        x.row.q = nullptr;  // nothing is left of the target where the draft is taken off: the draw is from the target itself
        x.row.without = -1;
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
            const bool in_front = heads && k0 == 0, behind = tails && k0 == GROUPS - 1;
            if (in_front) found = first_over(lane < x.begin ? x.single(lane) : 0.0, goal, before, lane);
#pragma unroll 1
            for (int base = from; base < end && found < 0; base += STEP) {
                typename DrawPieces<T, VEC>::Raw r[U];
                double own[U];
#pragma unroll
                for (int u = 0; u < U; u++) x.load(r[u], base + VEC * (lane + 32 * u), base + VEC * (lane + 32 * u) < end);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    double w[VEC];
                    x.weights(r[u], base + VEC * (lane + 32 * u), w);
                    own[u] = 0.0;
#pragma unroll
                    for (int e = 0; e < VEC; e++) own[u] += w[e];
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (found >= 0) continue;
                    double start = before;
                    const int l = first_over(own[u], goal, before, lane);  // the lane it is in
                    if (l < 0) continue;
                    double incl = own[u];
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double up = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += up;
                    }
                    double sum = start + (incl - own[u]);
                    int over = -1, some = -1;
                    double w[VEC];
                    x.weights(r[u], base + VEC * (lane + 32 * u), w);
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        sum += w[e];
                        if (w[e] > 0.0) some = e;
                        if (over < 0 && w[e] > 0.0 && sum > goal) over = e;
                    }
                    found = base + VEC * (l + 32 * u) + __shfl_sync(0xffffffffu, over >= 0 ? over : some, l);
                }
            }
            if (found < 0 && behind) {
                found = first_over(lane < V - x.end ? x.single(x.end + lane) : 0.0, goal, before, lane);
                if (found >= 0) found += x.end;
            }
            if (found < 0) {  // sums in another order, or a goal that was rounded up to the total: the last token with any weight
                int last = -1;
                if (in_front && lane < x.begin && x.single(lane) > 0.0) last = lane;
                for (int i = from + lane; i < end; i += 32)
                    if (x.single(i) > 0.0) last = i;
                if (behind && lane < V - x.end && x.single(x.end + lane) > 0.0) last = x.end + lane;
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
    // As many CTAs per sequence as leave a warp a few steps, and as are on the GPU at once (four on each of 148 SMs).
    int ranks = 1;
    while (ranks < 8 && (long long)V >= 2ll * ranks * kVerifyWarps * 256 && (long long)B * ranks * 2 <= 4 * 148) ranks *= 2;
    const dim3 grid(ranks, B), block(kVerifyWarps * 32);
    const cudaStream_t st = (cudaStream_t)stream;
    MYNN_DISPATCH_DTYPE(dtype, T, {
        if (V >= 256) MYNN_CUDA_OK(launch_ex(true, ranks, verify_draft_kernel<T, 16 / sizeof(T)>, grid, block, 0, st, p));
        else MYNN_CUDA_OK(launch_ex(true, ranks, verify_draft_kernel<T, 1>, grid, block, 0, st, p));
    });
    MYNN_LAUNCH_OK("verify_draft_kernel");
    return MYNN_OK;
}
