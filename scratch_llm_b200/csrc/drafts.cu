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
#include "common.cuh"

namespace sllm {

constexpr int VERIFY_THREADS = 1024;

__device__ __forceinline__ double weight(float p, float q) {
    const double w = (double)p - (double)q;
    return w > 0.0 ? w : 0.0;           // (a NaN too)
}

__global__ void __launch_bounds__(VERIFY_THREADS)
verify_drafts_kernel(const float* __restrict__ probs, int64_t p_stride, const float* __restrict__ draft_probs,
                     int64_t q_stride, const int* __restrict__ drafts, const int* __restrict__ start,
                     const float* __restrict__ uniforms, int V, int* __restrict__ tokens, int* __restrict__ accepted) {
    __shared__ double part[VERIFY_THREADS];
    __shared__ int found;
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x, tid = threadIdx.x;
    const int d0 = start[r], k = start[r + 1] - d0, p0 = d0 + r;
    int n = 0;
    for (; n < k; ++n) {
        const int x = drafts[d0 + n];
        if (x < 0 || x >= V) break;
        const double q = draft_probs ? (double)draft_probs[(d0 + n) * q_stride + x] : 1.0;
        if (!((double)uniforms[p0 + n] * q < (double)probs[(p0 + n) * p_stride + x])) break;
    }
    const float* p = probs + (p0 + n) * p_stride;
    const float* q = draft_probs && n < k ? draft_probs + (d0 + n) * q_stride : nullptr;
    const int hot = !draft_probs && n < k ? drafts[d0 + n] : -1;
    const int per = (V + VERIFY_THREADS - 1) / VERIFY_THREADS, begin = min(V, tid * per), end = min(V, begin + per);
    int token = -1;
    for (int turn = 0; turn < 2 && token < 0; ++turn) {       // the weights, or p itself
        auto w = [&](int j) { return j == hot && !turn ? 0.0 : weight(p[j], q && !turn ? q[j] : 0.f); };
        double mine = 0.0;
        int last = -1;
        for (int j = begin; j < end; ++j) {
            const double x = w(j);
            mine += x;
            if (x > 0.0) last = j;
        }
        __syncthreads();
        part[tid] = mine;
        if (tid == 0) found = -1;
        __syncthreads();
        double before = 0.0, total = 0.0;
        for (int t = 0; t < VERIFY_THREADS; ++t) {
            if (t == tid) before = total;
            total += part[t];
        }
        const double goal = (double)uniforms[p0 + k] * total;
        if (last >= 0 && before <= goal) {                      // (the last such thread has it, or one after it none)
            double run = before;
            int pick = last;
            for (int j = begin; j < end; ++j) {
                run += w(j);
                if (run > goal) { pick = j; break; }
            }
            atomicMax(&found, pick);
        }
        __syncthreads();
        token = found;
    }
    for (int i = tid; i <= k; i += VERIFY_THREADS)
        tokens[p0 + i] = i < n ? drafts[d0 + i] : i == n ? token : -1;
    if (tid == 0) accepted[r] = n;
}

}  // namespace sllm

using namespace sllm;

SLLM_EXPORT int sllm_verify_drafts(const float* probs, int64_t p_stride, const float* draft_probs, int64_t q_stride,
                                   const int* drafts, const int* start, const float* uniforms, int n_rows, int V,
                                   int* tokens, int* accepted, cudaStream_t stream) {
    if (n_rows <= 0) return 0;
    if (V <= 0) return (int)cudaErrorInvalidValue;
    return (int)sllm_launch_pdl(verify_drafts_kernel, dim3(n_rows), dim3(VERIFY_THREADS), 0, stream, probs, p_stride,
                                draft_probs, q_stride, drafts, start, uniforms, V, tokens, accepted);
}
