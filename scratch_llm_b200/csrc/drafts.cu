// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Row r has k drafts x_0 .. x_{k-1}, the target's distributions p_0 .. p_k (p_i after the drafts before i), the
// drafts' q_i (or none: a draft that was looked up, with all of its mass on x_i) and the numbers u_0 .. u_k in
// [0, 1).  x_i is accepted while u_i q_i(x_i) < p_i(x_i), which happens with probability min(1, p_i / q_i); at the
// first i that is not, the row's last token comes from max(p_i - q_i, 0), after k accepted ones from p_k.  The
// tokens that come out are then distributed as the target's own (accepted mass min(p, q) and what is left of p).
// Drawing: w_j the weights in the vocabulary's order, S_j = w_0 + .. + w_j, the first j with S_j > u_k S_{V-1}.
// Where no weight is left (p nowhere above q) the row draws from p_i, and where that has none either the
// token is -1.  A NaN counts as no probability: it is never accepted and never drawn.
//
// All of it in 64 bits: products and differences of 32-bit numbers are exact there, and a sum of 128,256 of them
// in another order moves by 1e-16 of itself, where a token's share of it is 1e-5: in 32 bits a draw in a
// hundred would fall on another token.
//
// A row needs its drafts' own entries (one warp, a draft a lane) and then one pass over the distribution that decides: a
// cluster of eight CTAs per row, every warp with a run of the vocabulary of its own.  Sums of runs go through shared
// memory, sums of CTAs through distributed shared memory; the run that holds the goal is gone through once more by
// all warps of its CTA (a few KB that the SM has just read), and the share that holds it by one: 4 rows of 128,256 entries
// 9 us, 64 rows 18 (66 MB, 10 us at the copy rate).  One CTA per row, every pass by itself, took 155 us for 4 rows.
#include <cooperative_groups.h>

#include "common.cuh"

namespace sllm {

constexpr int VERIFY_RANKS = 8;
// Four CTAs an SM, each warp requesting three strips of 128 entries at a time.  CTAs of 512 threads with four strips took 8.7 us
// instead of 9.0 for 4 rows of 128,256 entries and four drafts, but 13.1 instead of 10.3 for 16 and 35 instead of 18 for 64.
constexpr int VERIFY_THREADS = 256, VERIFY_WARPS = VERIFY_THREADS / 32, VERIFY_BATCH = 3;

__device__ __forceinline__ double weight(float p, float q) {
    const double w = (double)p - (double)q;
    return w > 0.0 ? w : 0.0;           // (a NaN too)
}

// What a row draws from: max(p - q, 0), without the entry `hot`; q may be null.
struct Weights {
    const float* p; const float* q;
    int hot;
    bool vec;                           // whole 16-byte words
    // of the entries j .. j + 3 below `end`
    __device__ __forceinline__ void load(int j, int end, float4& a, float4& b) const {
        b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (vec && j + 4 <= end) {
            a = __ldg(reinterpret_cast<const float4*>(p + j));
            if (q) b = __ldg(reinterpret_cast<const float4*>(q + j));
        } else {
            a = b;
            float* x = reinterpret_cast<float*>(&a);
            float* y = reinterpret_cast<float*>(&b);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (j + i < end) {
                    x[i] = __ldg(p + j + i);
                    if (q) y[i] = __ldg(q + j + i);
                }
        }
    }
    __device__ __forceinline__ void of(int j, const float4& a, const float4& b, double (&w)[4]) const {
        w[0] = j == hot ? 0.0 : weight(a.x, b.x);
        w[1] = j + 1 == hot ? 0.0 : weight(a.y, b.y);
        w[2] = j + 2 == hot ? 0.0 : weight(a.z, b.z);
        w[3] = j + 3 == hot ? 0.0 : weight(a.w, b.w);
    }
};

// the weights from `begin` to `end`, by a warp
__device__ __forceinline__ double sum_of(const Weights& w, int begin, int end) {
    const int lane = threadIdx.x & 31;
    double sum = 0.0;
    for (int j0 = begin; j0 < end; j0 += 128 * VERIFY_BATCH) {
        float4 a[VERIFY_BATCH], b[VERIFY_BATCH];
#pragma unroll
        for (int t = 0; t < VERIFY_BATCH; ++t) w.load(j0 + 128 * t + 4 * lane, end, a[t], b[t]);
#pragma unroll
        for (int t = 0; t < VERIFY_BATCH; ++t) {
            double x[4];
            w.of(j0 + 128 * t + 4 * lane, a[t], b[t], x);
            sum += (x[0] + x[1]) + (x[2] + x[3]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
// Of sums of parts in order, of which the first starts at `at`: the first part whose end lies past the goal, or the last one
// with any weight (-1: none has any).  `at` becomes the start of that part.
template <int N> __device__ __forceinline__ int part_of(const double* sums, double goal, double& at) {
    int own = -1;
    double upto = at, start = at, after = at;
    for (int i = 0; i < N; ++i) {
        if ((own < 0 || after <= goal) && sums[i] > 0.0) { own = i; start = upto; after = upto + sums[i]; }
        upto += sums[i];
    }
    at = start;
    return own;
}

__global__ void __cluster_dims__(VERIFY_RANKS, 1, 1) __launch_bounds__(VERIFY_THREADS, 4)
verify_drafts_kernel(const float* __restrict__ probs, int64_t p_stride, const float* __restrict__ draft_probs,
                     int64_t q_stride, const int* __restrict__ drafts, const int* __restrict__ start,
                     const float* __restrict__ uniforms, int V, int* __restrict__ tokens, int* __restrict__ accepted) {
    __shared__ double warp_sum[VERIFY_WARPS], share_sum[VERIFY_WARPS], cta_sum[2];
    __shared__ int n_accepted;
    pdl_wait();
    pdl_trigger();
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int rank = (int)cluster.block_rank(), r = blockIdx.x / VERIFY_RANKS;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int d0 = start[r], k = start[r + 1] - d0;
    const int64_t p0 = (int64_t)d0 + r;
    const double u = (double)uniforms[p0 + k];
    if (warp == 0) {
        int n = 0;
        for (; n < k; n += 32) {
            const int i = n + lane;
            bool kept = i < k;
            if (kept) {
                const int x = drafts[d0 + i];
                kept = x >= 0 && x < V;
                if (kept) {
                    const double q = draft_probs ? (double)draft_probs[(int64_t)(d0 + i) * q_stride + x] : 1.0;
                    kept = (double)uniforms[p0 + i] * q < (double)probs[(p0 + i) * p_stride + x];
                }
            }
            const uint32_t refused = __ballot_sync(0xffffffffu, !kept);
            if (refused) { n += __ffs(refused) - 1; break; }
        }
        if (lane == 0) n_accepted = min(n, k);
    }
    __syncthreads();
    const int n = n_accepted;
    Weights w = {probs + (p0 + n) * p_stride, draft_probs && n < k ? draft_probs + (int64_t)(d0 + n) * q_stride : nullptr,
                 !draft_probs && n < k ? drafts[d0 + n] : -1, false};
    // this warp's run: a share of the vocabulary, in whole fours
    const int run = ((V + VERIFY_RANKS * VERIFY_WARPS - 1) / (VERIFY_RANKS * VERIFY_WARPS) + 3) / 4 * 4;
    const int64_t run0 = (int64_t)(rank * VERIFY_WARPS + warp) * run;
    const int begin = (int)min((int64_t)V, run0), end = (int)min((int64_t)V, run0 + run);
    bool found = false;
    for (int turn = 0; turn < 2 && !found; ++turn) {          // the weights, or p itself (the same turn in all CTAs)
        if (turn) { w.q = nullptr; w.hot = -1; }
        w.vec = (((uintptr_t)w.p | (uintptr_t)w.q) & 15) == 0;
        const double mine = sum_of(w, begin, end);
        if (lane == 0) warp_sum[warp] = mine;
        __syncthreads();
        if (tid == 0) {
            double sum = 0.0;
            for (int i = 0; i < VERIFY_WARPS; ++i) sum += warp_sum[i];
            cta_sum[turn] = sum;
        }
        cluster.sync();
        double total = 0.0, sums[VERIFY_RANKS];
#pragma unroll
        for (int i = 0; i < VERIFY_RANKS; ++i) sums[i] = cluster.map_shared_rank(cta_sum, i)[turn];
        cluster.sync();                   // (all have read all sums: who has nothing to look for may leave)
#pragma unroll
        for (int i = 0; i < VERIFY_RANKS; ++i) total += sums[i];
        found = total > 0.0;
        if (!found) continue;
        // whose CTA, whose warp's run, and, the run shared out in strips of 128, which warp's share of it holds the goal
        const double goal = u * total;
        double past = 0.0;
        if (part_of<VERIFY_RANKS>(sums, goal, past) != rank) continue;
        const int own_warp = part_of<VERIFY_WARPS>(warp_sum, goal, past);
        const int64_t own0 = (int64_t)(rank * VERIFY_WARPS + own_warp) * run;
        const int own_end = (int)min((int64_t)V, own0 + run), strips = (own_end - (int)own0 + 127) / 128;
        const int share = (strips + VERIFY_WARPS - 1) / VERIFY_WARPS * 128;
        const int from = min(own_end, (int)own0 + warp * share), to = min(own_end, from + share);
        const double shared = sum_of(w, from, to);
        if (lane == 0) share_sum[warp] = shared;
        __syncthreads();
        if (part_of<VERIFY_WARPS>(share_sum, goal, past) != warp) continue;
        // and its entry
        int token = -1;
        bool there = false;
        for (int j0 = from; j0 < to && !there; j0 += 128 * VERIFY_BATCH) {
            float4 a[VERIFY_BATCH], b[VERIFY_BATCH];
#pragma unroll
            for (int t = 0; t < VERIFY_BATCH; ++t) w.load(j0 + 128 * t + 4 * lane, to, a[t], b[t]);
#pragma unroll
            for (int t = 0; t < VERIFY_BATCH; ++t) {
                if (there) break;
                const int j = j0 + 128 * t + 4 * lane;
                double x[4];
                w.of(j, a[t], b[t], x);
                double scan = (x[0] + x[1]) + (x[2] + x[3]);
                const double own = scan;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double up = __shfl_up_sync(0xffffffffu, scan, o);
                    if (lane >= o) scan += up;
                }
                // the lane whose entries pass the goal, and which of them; the last one of any weight stands in
                double at = past + (scan - own);
                int pick = -1, last = -1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    at += x[i];
                    if (x[i] > 0.0) last = j + i;
                    if (x[i] > 0.0 && pick < 0 && at > goal) pick = j + i;
                }
                const uint32_t hits = __ballot_sync(0xffffffffu, pick >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
                there = hits != 0u;
                if (there) token = __shfl_sync(0xffffffffu, pick, __ffs(hits) - 1);
                else if (any) token = __shfl_sync(0xffffffffu, last, 31 - __clz(any));
                past += __shfl_sync(0xffffffffu, scan, 31);
            }
        }
        if (lane == 0) tokens[p0 + n] = token;
    }
    if (rank == 0) {
        for (int i = tid; i <= k; i += VERIFY_THREADS)
            if (i != n || !found) tokens[p0 + i] = i < n ? drafts[d0 + i] : -1;
        if (tid == 0) accepted[r] = n;
    }
}

}  // namespace sllm

using namespace sllm;

SLLM_EXPORT int sllm_verify_drafts(const float* probs, int64_t p_stride, const float* draft_probs, int64_t q_stride,
                                   const int* drafts, const int* start, const float* uniforms, int n_rows, int V,
                                   int* tokens, int* accepted, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (V <= 0 || V > 1 << 30 || n_rows > 0x7fffffff / VERIFY_RANKS) return (int)cudaErrorInvalidValue;
    return (int)sllm_launch_pdl(verify_drafts_kernel, dim3(n_rows * VERIFY_RANKS), dim3(VERIFY_THREADS), 0, stream, probs, p_stride,
                                draft_probs, q_stride, drafts, start, uniforms, V, tokens, accepted);
}
