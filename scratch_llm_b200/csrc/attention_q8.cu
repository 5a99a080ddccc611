// Causal attention of a packed batch over a paged cache held in 8 bits (q8.cuh): the token at absolute position p of
// row r attends to the keys 0 .. p of row r, or to the last `window` of them, and query head h reads kv head
// h / (H / G).  Scores, softmax and sums are 32-bit arithmetic.
//   s_j = scale * q . k_j,   out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// Compiled once per head size: -DSLLM_HEAD_DIM=<multiple of 16, at most 256>.
#include "q8.cuh"

#ifndef SLLM_HEAD_DIM
#error "compile with -DSLLM_HEAD_DIM=<head size>"
#endif

namespace sllm {

constexpr int HD = SLLM_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size: a multiple of 16 up to 256");
constexpr int DPL = (HD + 31) / 32;     // entries of a head a lane

struct Q8Args {
    int64_t q_stride, out_stride;
    const uint8_t* pages; const uint8_t* scales; const int* table;
    const int* row_start; const int* row_pos0; const int* row_list;
    int table_stride, page_size, block, H, G, window;
    float scale;
};

// A warp per token and head, key after key: grid (tokens of a row, rows, heads / 4).
template <typename T>
__global__ void __launch_bounds__(128) attn_q8_kernel(const T* __restrict__ q, T* __restrict__ out, const Q8Args a) {
    pdl_wait();
    pdl_trigger();
    const int r = a.row_list ? a.row_list[blockIdx.y] : blockIdx.y, lane = threadIdx.x & 31;
    const int h = blockIdx.z * 4 + threadIdx.x / 32, g = h / (a.H / a.G);
    const int t0 = a.row_start[r], n_new = a.row_start[r + 1] - t0;
    if ((int)blockIdx.x >= n_new || h >= a.H) return;
    const int64_t token = t0 + blockIdx.x;
    const int pos = a.row_pos0[r] + blockIdx.x;
    float x[DPL], o[DPL], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int c = 0; c < DPL; ++c) {
        const int d = lane + 32 * c;
        x[c] = d < HD ? to_float(q[token * a.q_stride + (int64_t)h * HD + d]) * a.scale : 0.f;
        o[c] = 0.f;
    }
    const int blocks = a.page_size / a.block;
    for (int j = a.window > 0 ? max(0, pos - a.window + 1) : 0; j <= pos; ++j) {
        const int page = a.table[(int64_t)r * a.table_stride + j / a.page_size], off = j % a.page_size;
        if (page < 0) continue;
        const int64_t k_plane = (int64_t)page * 2 * a.G + g, v_plane = k_plane + a.G;
        const uint8_t* k = a.pages + (k_plane * a.page_size + off) * HD;
        const uint8_t* v = a.pages + (v_plane * a.page_size + off) * HD;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < DPL; ++c)
            if (lane + 32 * c < HD) s = fmaf(x[c], q8_float2(k[lane + 32 * c]).x, s);
        s = warp_sum(s) * q8_power(a.scales[k_plane * blocks + off / a.block]);
        const float top = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - top);
        const float p = expf(s - top), pv = p * q8_power(a.scales[v_plane * blocks + off / a.block]);
        m = top;
        l = l * keep + p;
#pragma unroll
        for (int c = 0; c < DPL; ++c)
            if (lane + 32 * c < HD) o[c] = o[c] * keep + pv * q8_float2(v[lane + 32 * c]).x;
    }
#pragma unroll
    for (int c = 0; c < DPL; ++c)
        if (lane + 32 * c < HD)
            out[token * a.out_stride + (int64_t)h * HD + lane + 32 * c] = from_float<T>(l != 0.f ? o[c] / l : 0.f);
}

}  // namespace sllm

using namespace sllm;

SLLM_EXPORT int sllm_attn_q8(const void* q, int64_t q_stride, const void* pages, const void* scales, const int* table,
                             int table_stride, int page_size, int block, const int* row_start, const int* row_pos0,
                             const int* row_list, int n_list, int max_new, void* out, int64_t out_stride, int H, int G,
                             float scale, int window, int dtype, cudaStream_t stream) {
    if (n_list <= 0 || max_new <= 0) return 0;
    if (H <= 0 || G <= 0 || H % G || page_size <= 0 || block <= 0 || page_size % block || window < 0 || n_list > 65535 ||
        (dtype != 0 && dtype != 1))
        return (int)cudaErrorInvalidValue;
    const Q8Args a = {q_stride, out_stride, (const uint8_t*)pages, (const uint8_t*)scales, table, row_start, row_pos0, row_list,
                      table_stride, page_size, block, H, G, window, scale};
    const dim3 grid(max_new, n_list, (H + 3) / 4);
    if (dtype == 0)
        return (int)sllm_launch_pdl(attn_q8_kernel<float>, grid, dim3(128), 0, stream, (const float*)q, (float*)out, a);
    return (int)sllm_launch_pdl(attn_q8_kernel<__nv_bfloat16>, grid, dim3(128), 0, stream, (const __nv_bfloat16*)q,
                                (__nv_bfloat16*)out, a);
}
