// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Draft token x_i stands while u_i q_i(x_i) < p_i(x_i); the first one that does not, n, is replaced by a draw from max(p_n - q_n, 0), and behind K standing tokens
// comes a draw from p_K: the first token whose running sum exceeds r times the whole sum.  So the tokens are distributed as the target's own.
//
// Of (2 K + 1) V probabilities only the one or two rows of the draw are read whole.  A cluster of CTAs takes a sequence, each CTA a range of the vocabulary and each warp a
// part of it: sums per warp, then which part the running sum ends in, then that part again, 128 tokens at a time.  A difference of two f32
// numbers and sums of 1e5 of them decide on whole numbers, so they are held in 64 bits: a sum in f32 is off by more than many a token's probability.
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

constexpr int kVerifyWarps = 16;

template <typename T>
__device__ __forceinline__ double weight_of(const T *p, const T *q, int i, int without) {
    const double a = (double)to_f32<T>(p[i]), w = q ? a - (double)to_f32<T>(q[i]) : a;
    return i != without && w > 0.0 ? w : 0.0;
}

// One CTA per sequence.
template <typename T>
__global__ void __launch_bounds__(kVerifyWarps * 32) verify_draft_kernel(const VerifyDraft p) {
    __shared__ double sums[kVerifyWarps];
    __shared__ int sm_n, sm_pick;
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, K = p.K, V = p.V;
    const int drafts = p.counts ? min(max(p.counts[b], 0), K) : K;
    const T *target = reinterpret_cast<const T *>(p.target) + (size_t)b * (K + 1) * V;
    const T *draft = p.draft ? reinterpret_cast<const T *>(p.draft) + (size_t)b * K * V : nullptr;
    if (warp == 0) {
        int n = drafts;
        for (int i = lane; i < drafts; i += 32) {
            const int x = p.tokens[(size_t)b * K + i];
            bool stands = false;
            if ((unsigned)x < (unsigned)V) {
                const double q = draft ? (double)to_f32<T>(draft[(size_t)i * V + x]) : 1.0;
                stands = (double)p.accept[(size_t)b * K + i] * q < (double)to_f32<T>(target[(size_t)i * V + x]);
            }
            if (!stands) {
                n = i;
                break;
            }
        }
        n = __reduce_min_sync(0xffffffffu, n);
        if (lane == 0) sm_n = n;
    }
    __syncthreads();
    const int n = sm_n;
    const T *pr = target + (size_t)n * V, *qr = n < drafts && draft ? draft + (size_t)n * V : nullptr;
    int without = n < drafts && !draft ? p.tokens[(size_t)b * K + n] : -1;
    const int per = (V + kVerifyWarps - 1) / kVerifyWarps, lo = min(warp * per, V), hi = min(lo + per, V);
    double total = 0.0;
    for (int pass = 0; pass < 2; pass++) {
        double mine = 0.0;
        for (int i = lo + lane; i < hi; i += 32) mine += weight_of(pr, qr, i, without);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) sums[warp] = mine;
        __syncthreads();
        total = 0.0;
        for (int w = 0; w < kVerifyWarps; w++) total += sums[w];
        __syncthreads();
        if (total > 0.0 || (!qr && without < 0)) break;
        qr = nullptr;  // nothing is left of the target where the draft is taken off: the draw is from the target itself
        without = -1;
        if (lane == 0) sums[warp] = 0.0;
    }
    if (threadIdx.x == 0) sm_pick = -1;
    __syncthreads();
    const double goal = (double)p.sample[b] * total;
    // the warp whose part the running sum exceeds the goal in; without one (the goal rounded up to the whole sum) the last that has any weight
    double before = 0.0;
    int chosen = -1;
    {
        double run = 0.0;
        for (int w = 0; w < kVerifyWarps; w++) {
            if (!(sums[w] > 0.0)) continue;
            chosen = w;
            before = run;
            run += sums[w];
            if (run > goal) break;
        }
    }
    if (warp == chosen) {
        int pick = -1, last = -1;
        double run = before;
        for (int base = lo; base < hi && pick < 0; base += 32) {
            const int i = base + lane;
            const double w = i < hi ? weight_of(pr, qr, i, without) : 0.0;
            double incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += up;
            }
            const unsigned over = __ballot_sync(0xffffffffu, w > 0.0 && run + incl > goal), some = __ballot_sync(0xffffffffu, w > 0.0);
            if (over) pick = base + __ffs(over) - 1;
            if (some) last = base + 31 - __clz(some);
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) sm_pick = pick >= 0 ? pick : last;
    }
    __syncthreads();
    for (int i = threadIdx.x; i <= K; i += kVerifyWarps * 32) p.tokens_out[(size_t)b * (K + 1) + i] = i < n ? p.tokens[(size_t)b * K + i] : i == n ? sm_pick : -1;
    if (threadIdx.x == 0) p.accepted_out[b] = n;
}

}  // namespace mynn

using namespace mynn;

extern "C" int mynn_b200_verify_draft(void *stream, int32_t *tokens_out, int32_t *accepted_out, const void *target, const void *draft, const int32_t *tokens,
                                      const int32_t *counts, const float *accept, const float *sample, int B, int K, int V, int dtype) {
    if (B < 0 || K < 0 || V < 1) return fail(MYNN_E_ARG, "verify_draft: bad shape");
    if (!dtype_ok(dtype)) return fail(MYNN_E_ARG, "verify_draft: bad dtype %d", dtype);
    if (K > 1024 || V > 1 << 30) return fail(MYNN_E_UNSUPPORTED, "verify_draft: %d drafted tokens of a vocabulary of %d", K, V);
    if (B == 0) return MYNN_OK;
    if (!tokens_out || !accepted_out || !target || !sample || (K && (!tokens || !accept))) return fail(MYNN_E_ARG, "verify_draft: null pointer");
    VerifyDraft p;
    p.tokens_out = tokens_out, p.accepted_out = accepted_out;
    p.target = target, p.draft = draft;
    p.tokens = tokens, p.counts = counts;
    p.accept = accept, p.sample = sample;
    p.B = B, p.K = K, p.V = V;
    MYNN_DISPATCH_DTYPE(dtype, T, { MYNN_CUDA_OK(launch_dependent(verify_draft_kernel<T>, dim3(B), dim3(kVerifyWarps * 32), 0, (cudaStream_t)stream, p)); });
    MYNN_LAUNCH_OK("verify_draft_kernel");
    return MYNN_OK;
}
