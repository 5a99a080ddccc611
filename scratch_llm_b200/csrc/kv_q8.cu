// Keys and values into a cache of 8-bit numbers, and back (q8.cuh says what such a cache holds).
//
// Write: rotary position encoding of q and k (32-bit angles and arithmetic, each product and each difference
// rounded on its own), the turned queries into a buffer of their own, keys and values quantised as they are
// stored.  The 8-bit form of rope_cache.cu, with its conventions: qkv [n_tokens, (H + 2G) * hd], q heads,
// then k heads, then v heads; `bias` (may be null) added first; only the first `rot` entries of a head
// turn, in pairs (2j, 2j + 1) or (j, j + rot / 2).  Row r brings the tokens row_start[r] .. row_start[r + 1] - 1, at
// the positions from row_pos0[r] on; tokens before the first row and behind the last are left alone.
//   pages  [n_pages, 2, G, page_size, hd]             e4m3
//   scales [n_pages, 2, G, page_size / block]         e8m0
// A block's scale comes from the values that this step stores in it and, where the row has stored earlier
// tokens in it (positions before row_pos0[r]), from the scale that it has: it only grows, and then the
// earlier tokens' numbers are rounded again at the new one.  What a block that starts with this step held
// before is never looked at.
#include "q8.cuh"

namespace sllm {

struct WriteArgs {
    const int* row_start; const int* row_pos0;
    const float* cos_t; const float* sin_t; const float* bias;
    uint8_t* pages; uint8_t* scales; const int* table;
    int table_stride, page_size, block, n_rows, n_tokens, H, G, hd, rot, interleaved, single;
    int lanes;              // threads of a block of the cache: a power of two up to 32, or whole warps
    int kv_ctas, q_groups, q_per_group, q_at_once, lane_tokens, page_blocks;
    Divisor by_lanes, by_upt, by_planes, by_g, by_block, by_page, by_q_groups;     // (a division costs twenty instructions)
    int n_tasks;
    int64_t n_q_items;
};

constexpr int WRITE_THREADS = 256;

// Unit u of a head: 2 W entries, W at e0 and W at e1; turned pairs are (e0 + i, e1 + i), or, where neighbours
// pair, the pairs within 2 W neighbouring entries.  Entries that do not turn come 2 W neighbours at a time.
template <int W> struct Unit {
    int e0, e1, pair0;      // pair0: its first pair's column of the tables; -1 where it does not turn
    __device__ __forceinline__ Unit(int u, int rot, int interleaved) {
        const int n_turn = rot / (2 * W);
        pair0 = u < n_turn ? W * u : -1;
        if (u < n_turn && !interleaved) { e0 = W * u; e1 = rot / 2 + W * u; }
        else { e0 = 2 * W * u; e1 = e0 + W; }
    }
};

template <typename T, int W> __device__ __forceinline__ void load_w(const T* p, float* v) {
    if constexpr (W == 1) v[0] = to_float(p[0]);
    else {
#pragma unroll
        for (int i = 0; i < W; i += Vec<T>::N) Vec<T>::load(p + i, v + i);
    }
}
template <typename T, int W> __device__ __forceinline__ void store_w(T* p, const float* v) {
    if constexpr (W == 1) p[0] = from_float<T>(v[0]);
    else if constexpr (W < Vec<T>::N) {
        uint32_t w[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < W; i += Vec<T>::N) Vec<T>::store(p + i, v + i);
    }
}

template <int W>
__device__ __forceinline__ void load_angles(const WriteArgs& a, const Unit<W>& u, int pos, float* c, float* s) {
    if (u.pair0 < 0) return;
    load_w<float, W>(a.cos_t + (int64_t)pos * (a.rot / 2) + u.pair0, c);
    load_w<float, W>(a.sin_t + (int64_t)pos * (a.rot / 2) + u.pair0, s);
}

// One unit of a head as it lies in memory: of a thread's units all are requested before the first is worked on.
template <typename T, int W> struct Raw {
    static constexpr int WORDS = (2 * W * (int)sizeof(T) + 3) / 4, HALF = W * (int)sizeof(T);
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T* head, const Unit<W>& u) {
        if constexpr (HALF == 16) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(head + u.e0)), y = __ldg(reinterpret_cast<const uint4*>(head + u.e1));
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
        } else if constexpr (HALF == 8) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(head + u.e0)), y = __ldg(reinterpret_cast<const uint2*>(head + u.e1));
            w[0] = x.x; w[1] = x.y; w[2] = y.x; w[3] = y.y;
        } else if constexpr (HALF == 4) {
            w[0] = __float_as_uint(to_float(__ldg(head + u.e0)));
            w[1] = __float_as_uint(to_float(__ldg(head + u.e1)));
        } else {
            w[0] = (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(head) + u.e0) |
                   (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(head) + u.e1) << 16;
        }
    }
    // v[0 .. W): the entries at e0, v[W .. 2 W): those at e1
    __device__ __forceinline__ void values(float* v) const {
#pragma unroll
        for (int i = 0; i < 2 * W; ++i)
            v[i] = sizeof(T) == 4 ? __uint_as_float(w[i]) : __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};

// A unit's values with the bias, turned.
template <typename T, int W, bool BIAS>
__device__ __forceinline__ void unit_values(const WriteArgs& a, const Raw<T, W>& raw, const float* bias, const Unit<W>& u,
                                            const float* c, const float* s, float* v) {
    raw.values(v);
    if constexpr (BIAS) {
        float b[2 * W];
        load_w<float, W>(bias + u.e0, b);
        load_w<float, W>(bias + u.e1, b + W);
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) v[i] = __fadd_rn(v[i], b[i]);
    }
    if (u.pair0 >= 0) {
        auto turn = [&](float& x0, float& x1, int i) {
            const float y0 = __fsub_rn(__fmul_rn(x0, c[i]), __fmul_rn(x1, s[i]));
            x1 = __fadd_rn(__fmul_rn(x0, s[i]), __fmul_rn(x1, c[i]));
            x0 = y0;
        };
        if (a.interleaved) {      // (places in registers are known to the compiler either way)
#pragma unroll
            for (int i = 0; i < W; ++i) turn(v[2 * i], v[2 * i + 1], i);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) turn(v[i], v[i + W], i);
        }
    }
}

// The last row r with row_start[r] < bound - step * r (the left side grows with r, the right one does not): 16 rows a
// look, whose loads do not wait for one another.
__device__ __forceinline__ int last_row(const WriteArgs& a, int64_t bound, int step) {
    int lo = 0, n = a.n_rows;
    while (n > 1) {
        const int stride = (n + 15) / 16;
        int past = 0;
#pragma unroll
        for (int j = 1; j < 16; ++j)
            if (j * stride < n) past += (int64_t)a.row_start[lo + j * stride] < bound - (int64_t)step * (lo + j * stride);
        lo += past * stride;
        n = min(stride, n - past * stride);
    }
    return lo;
}
// the row of token n: the last one that starts at or before it
__device__ __forceinline__ int row_of(const WriteArgs& a, int n) { return last_row(a, (int64_t)n + 1, 0); }

// CTAs 0 .. kv_ctas - 1: a group of a.lanes threads takes one block of the cache (what a row stores in it), for one
// plane and kv head, twice: for its largest value, then, from L1, to store it: blocks of any size, and room for the warps
// that its chain of look-ups and two reads wants.  8,192 tokens of 32 + 8 + 8 heads of 128, blocks of 16, with the
// queries: 42 us (29 at the copy rate; 46 where every unit asks for a bias); 1,581 tokens of 3 x 40 heads, blocks of 64,
// in 32 bits with biases: 38 (22); eight rows of one token 2.5.  With the block in registers 49, 60 and 3.0; with a CTA a
// block and a thread's unit in several heads 45, 36 and 2.9, but up to 60 % more where rows fill parts of blocks.  The
// queries stream (24.5 us alone); the blocks' CTAs are bound by instruction issue, so that the two parts' times add up in
// whichever order their CTAs start.
// Row r has the slots from row_start[r] / block + 2 r on, at least as many as it touches blocks: n new tokens touch at
// most n / block + 2.  The other CTAs turn the queries.
template <typename T, int W, bool BIAS>
__global__ void __launch_bounds__(WRITE_THREADS, 4)
rope_kv_write_q8_kernel(const T* __restrict__ qkv, T* __restrict__ q_out, const WriteArgs a) {
    __shared__ float warp_top[2][WRITE_THREADS / 32];
    pdl_wait();
    pdl_trigger();
    const int heads = a.H + 2 * a.G, upt = a.hd / (2 * W);
    if ((int)blockIdx.x >= a.kv_ctas) {
        // ---- queries: a thread takes a unit of a token and walks a share of the token's heads with it (an item: a token's
        // share of heads)
        const int per_group = a.q_per_group, at_once = a.q_at_once;
        const int mine = a.by_upt.quotient(threadIdx.x), u_ = threadIdx.x - mine * upt;
        if (mine >= at_once) return;
        for (int64_t i = (int64_t)(blockIdx.x - a.kv_ctas) * at_once + mine; i < a.n_q_items;
             i += (int64_t)(gridDim.x - a.kv_ctas) * at_once) {
            const int n = a.by_q_groups.quotient((int)i), group = (int)i - n * a.q_groups;
            if (n < a.row_start[0] || n >= a.row_start[a.n_rows]) continue;      // (of no row)
            const int r = row_of(a, n), pos = a.row_pos0[r] + n - a.row_start[r];
            const Unit<W> u(u_, a.rot, a.interleaved);
            float c[W], s[W];
            load_angles<W>(a, u, pos, c, s);
            const int end = min(a.H, (group + 1) * per_group);
            constexpr int HEADS = sizeof(T) == 2 ? 4 : 2;      // requested at a time
            for (int h0 = group * per_group; h0 < end; h0 += HEADS) {
                Raw<T, W> raw[HEADS];
#pragma unroll
                for (int j = 0; j < HEADS; ++j) raw[j].load(qkv + ((int64_t)n * heads + min(h0 + j, end - 1)) * a.hd, u);
#pragma unroll
                for (int j = 0; j < HEADS; ++j) {
                    const int h = h0 + j;
                    if (h >= end) break;
                    float v[2 * W];
                    unit_values<T, W, BIAS>(a, raw[j], BIAS ? a.bias + (int64_t)h * a.hd : nullptr, u, c, s, v);
                    T* to = q_out + ((int64_t)n * a.H + h) * a.hd;
                    store_w<T, W>(to + u.e0, v);
                    store_w<T, W>(to + u.e1, v + W);
                }
            }
        }
        return;
    }
    // ---- keys and values
    const int lanes = a.lanes, in_cta = a.by_lanes.quotient(blockDim.x), group = a.by_lanes.quotient(threadIdx.x);
    const int64_t at_task = (int64_t)blockIdx.x * in_cta + group;
    bool live = at_task < a.n_tasks;
    const int task = live ? (int)at_task : 0, lane = threadIdx.x - group * lanes;
    const int slot = a.by_planes.quotient(task), pg = task - slot * 2 * a.G, plane = a.by_g.quotient(pg), g = pg - plane * a.G;
    int r = slot, at = 0;
    if (live && !a.single) {
        // row_start[r] / block + 2 r <= slot
        r = last_row(a, ((int64_t)slot + 1) * a.block, 2 * a.block);
        at = slot - (a.by_block.quotient(a.row_start[r]) + 2 * r);
    }
    int t0 = 0, pos0 = 0, n_old = 0, first = 0, count = 0;
    if (live) {
        t0 = a.row_start[r];
        const int n_new = a.row_start[r + 1] - t0;
        pos0 = a.row_pos0[r];
        const int begin = (a.by_block.quotient(pos0) + at) * a.block;       // the block's first position
        first = max(pos0, begin);
        count = min(pos0 + n_new, begin + a.block) - first;
        n_old = first - begin;
        live = count > 0;
    }
    // (the page is looked up while the values are on their way)
    const int begin = first - n_old, at_page = a.by_page.quotient(begin), cell = begin - at_page * a.page_size;
    const int page = live ? a.table[(int64_t)r * a.table_stride + at_page] : -1;
    const float* bias = BIAS ? a.bias + (int64_t)(a.H + pg) * a.hd : nullptr;
    const T* src = qkv + ((int64_t)(t0 + first - pos0) * heads + a.H + pg) * a.hd;
    // every unit of the block's new tokens, `lanes` at a time, AT_ONCE of them requested before the first is worked on:
    // use(token, unit, values)
    constexpr int AT_ONCE = 2;
    const int rot = plane == 0 ? a.rot : 0;
    const int units = live ? count * upt : 0, d_tok = a.lane_tokens, d_u = lanes - d_tok * upt;
    auto walk = [&](auto use) {
        int tok = a.by_upt.quotient(lane), u_ = lane - tok * upt;
        for (int i = lane; i < units; i += AT_ONCE * lanes) {
            Raw<T, W> raw[AT_ONCE];
            int toks[AT_ONCE], us[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                toks[k] = tok;
                us[k] = u_;
                if (i + k * lanes < units) raw[k].load(src + (int64_t)tok * heads * a.hd, Unit<W>(u_, rot, a.interleaved));
                tok += d_tok;
                u_ += d_u;
                if (u_ >= upt) { u_ -= upt; ++tok; }
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                if (i + k * lanes >= units) break;
                const Unit<W> u(us[k], rot, a.interleaved);
                float c[W], s[W], v[2 * W];
                load_angles<W>(a, u, first + toks[k], c, s);
                unit_values<T, W, BIAS>(a, raw[k], bias, u, c, s, v);
                use(toks[k], u, v);
            }
        }
    };
    int turn = 0;                                                 // of the two places where warps meet
    auto over_group = [&](float x) {
        for (int o = min(lanes, 32) / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        if (lanes > 32) {                                         // (the CTA is one group)
            if ((threadIdx.x & 31) == 0) warp_top[turn][threadIdx.x >> 5] = x;
            __syncthreads();
            for (int w = 0; w < lanes / 32; ++w) x = fmaxf(x, warp_top[turn][w]);
            turn ^= 1;
        }
        return x;
    };
    float top = 0.f;
    walk([&](int, const Unit<W>&, const float* v) {
#pragma unroll
        for (int j = 0; j < 2 * W; ++j) top = fmaxf(top, fabsf(v[j]));                // (a NaN leaves it as it is)
    });
    const int64_t plane_of = ((int64_t)page * 2 + plane) * a.G + g;
    uint8_t* scale = a.scales + (page >= 0 ? plane_of * a.page_blocks + a.by_block.quotient(cell) : 0);
    const int had = page >= 0 && n_old > 0 ? *scale : 0;          // (read by all before the group meets, written by one after)
    top = over_group(top);
    const bool odd = !q8_finite(top);                             // an infinity: it leaves the scale to the others
    if (__any_sync(0xffffffffu, odd)) {
        top = 0.f;
        walk([&](int, const Unit<W>&, const float* v) {
#pragma unroll
            for (int j = 0; j < 2 * W; ++j) top = fmaxf(top, q8_finite(v[j]) ? fabsf(v[j]) : 0.f);
        });
        top = over_group(top);
    }
    if (!live || page < 0) return;                                // (no page, nothing to store)
    const int byte = max(q8_scale_byte(top), had);
    const float inv = q8_inverse(byte);
    uint8_t* cells = a.pages + (plane_of * a.page_size + cell) * a.hd;
    if (n_old > 0 && byte > had) {
        // the earlier tokens at the scale of now (hd is a multiple of 16, the tokens of a block are neighbours)
        const float shift = q8_power(max(had, 1)) * inv;
        for (int i = lane; i < n_old * a.hd / 16; i += lanes) {
            uint4 x = *reinterpret_cast<uint4*>(cells + 16 * i);
            uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 lo = q8_float2(w[k] & 0xffffu), hi = q8_float2(w[k] >> 16);
                w[k] = q8_pack4(lo.x * shift, lo.y * shift, hi.x * shift, hi.y * shift);
            }
            *reinterpret_cast<uint4*>(cells + 16 * i) = x;
        }
    }
    walk([&](int tok, const Unit<W>& u, const float* v) {
        uint8_t* to = cells + (int64_t)(n_old + tok) * a.hd;
        float x[2 * W];
#pragma unroll
        for (int j = 0; j < 2 * W; ++j) x[j] = v[j] * inv;
        if (odd)
#pragma unroll
            for (int j = 0; j < 2 * W; ++j) x[j] = q8_finite(x[j]) ? x[j] : __int_as_float(0x7fffffff);
        if constexpr (W == 4) {
            *reinterpret_cast<uint32_t*>(to + u.e0) = q8_pack4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<uint32_t*>(to + u.e1) = q8_pack4(x[4], x[5], x[6], x[7]);
        } else {
            const uint32_t two = q8_pack2(x[0], x[1]);
            to[u.e0] = (uint8_t)two;
            to[u.e1] = (uint8_t)(two >> 8);
        }
    });
    if (lane == 0) *scale = (uint8_t)byte;
}

// 32 bytes of T in one store: a whole sector
__device__ __forceinline__ void store_32_bytes(float* to, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
__device__ __forceinline__ void store_32_bytes(__nv_bfloat16* to, const float* v) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// Reading back: the values of positions from .. to - 1 of a row, into pages of T through a table of their own.  A page is
// one run of bytes; a thread takes READ_PIECES pieces of it, each of which becomes 32 bytes and leaves in one store:
// 131,072 tokens of 8 heads of 128 to bfloat16 123 us (the bytes at the copy rate: 125), nine rows of up to 1,777 tokens of
// heads of 64 to 32 bits 8.2.  Two stores of 16 bytes, so that a warp's store fills halves of sectors, took 148 and 13.6,
// pieces that become 16 bytes 143 and 10.3.  grid (pieces of a page, pages of a row, rows).
constexpr int READ_THREADS = 256, READ_PIECES = 4;
constexpr float BF16_MAX = 3.38953139e38f;
template <typename T> constexpr int READ_BYTES = 32 / (int)sizeof(T);

struct ReadArgs {
    const uint8_t* pages; const uint8_t* scales; const int* table; int table_stride;
    int page_size, block, G, hd, first_row;
    // positions [row_from[r], row_to[r]) of row r through out_table, or, where row_start is given: everything that the
    // queries of the listed rows see, page p of the i-th of them to page i * listed_pages + p, which the kernel writes
    // into out_table[r] itself (-1 where a page is not needed); a NaN becomes zero there, what would be infinite the largest
    // finite number, and odd[i * listed_pages + p, blockIdx.x] is set to whether the CTA met a NaN
    const int* row_from; const int* row_to;
    const int* row_start; const int* row_pos0; const int* row_list; int window, listed_pages;
    int* out_table; int out_stride; uint8_t* odd;
    Divisor by_hd, by_page, by_block; int page_blocks;
};

template <typename T, bool LISTED>
__global__ void __launch_bounds__(READ_THREADS) kv_read_q8_kernel(T* __restrict__ out, const ReadArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int BYTES = READ_BYTES<T>, WORDS = BYTES / 4;
    const int i = a.first_row + blockIdx.z, r = a.row_list ? a.row_list[i] : i;
    const int page_size = a.page_size, pieces = 2 * a.G * page_size * a.hd / BYTES;
    constexpr bool listed = LISTED;
    int from, to;
    if (listed) {
        const int n_new = a.row_start[r + 1] - a.row_start[r], pos0 = a.row_pos0[r];
        to = n_new > 0 ? pos0 + n_new : 0;
        // (whole pages: what the first one holds in front of the window meets a probability of zero)
        from = a.window > 0 ? a.by_page.quotient(max(0, pos0 - a.window + 1)) * page_size : 0;
    } else {
        from = max(a.row_from[r], 0);
        to = a.row_to[r];
    }
    const int first_page = a.by_page.quotient(from);
    const int64_t p_end = listed ? a.listed_pages : to > 0 ? a.by_page.quotient(to - 1) + 1 : 0;
    for (int64_t p = (listed ? 0 : first_page) + (int64_t)blockIdx.y; p < p_end; p += gridDim.y) {
        const bool needed = p >= first_page && p * page_size < to;
        const int page = needed ? a.table[(int64_t)r * a.table_stride + p] : -1;
        int out_page;
        if (listed) {
            out_page = page >= 0 ? (int)(i * (int64_t)a.listed_pages + p) : -1;
            if (blockIdx.x == 0 && threadIdx.x == 0) a.out_table[(int64_t)r * a.out_stride + p] = out_page;
        } else {
            out_page = needed ? a.out_table[(int64_t)r * a.out_stride + p] : -1;
        }
        if (!listed && (page < 0 || out_page < 0)) continue;
        const uint8_t* src = a.pages + (int64_t)page * pieces * BYTES;
        const uint8_t* sc = a.scales + (int64_t)page * (2 * a.G * a.page_blocks);
        T* dst = out + (int64_t)out_page * pieces * BYTES;
        const int c0 = blockIdx.x * READ_THREADS * READ_PIECES + threadIdx.x;
        uint32_t x[READ_PIECES][WORDS];
        int b[READ_PIECES];
        bool odd = false;
#pragma unroll
        for (int k = 0; k < READ_PIECES; ++k) {
            const int c = c0 + k * READ_THREADS, row = a.by_hd.quotient(c * BYTES);    // of the page's 2 G page_size rows
            const int64_t pos = p * page_size + row - a.by_page.quotient(row) * page_size;
            b[k] = -1;
            if (out_page >= 0 && c < pieces && pos >= from && pos < to) {
                if constexpr (WORDS == 4) {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(src) + c);
                    x[k][0] = w.x; x[k][1] = w.y; x[k][2] = w.z; x[k][3] = w.w;
                } else {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(src) + c);
                    x[k][0] = w.x; x[k][1] = w.y;
                }
                b[k] = sc[a.by_block.quotient(row)];
            }
        }
#pragma unroll
        for (int k = 0; k < READ_PIECES; ++k) {
            if (b[k] < 0) continue;
            const float power = q8_power(b[k]);
            float v[BYTES];
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                uint32_t w = x[k][j];
                if (listed) {
                    const uint32_t nan = (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u;      // (the top bits of such bytes)
                    odd |= nan != 0u;
                    if (nan) w &= ~((nan >> 7) * 255u);
                }
                const float2 lo = q8_float2(w & 0xffffu), hi = q8_float2(w >> 16);
                v[4 * j] = lo.x * power;
                v[4 * j + 1] = lo.y * power;
                v[4 * j + 2] = hi.x * power;
                v[4 * j + 3] = hi.y * power;
            }
            // (numbers from 2^128 on, which an infinity would stand for, would reach what does not see them as a NaN does)
            if (listed && b[k] >= 247 && b[k] < 255)
#pragma unroll
                for (int j = 0; j < BYTES; ++j) v[j] = fminf(fmaxf(v[j], -BF16_MAX), BF16_MAX);
            store_32_bytes(dst + (int64_t)(c0 + k * READ_THREADS) * BYTES, v);
        }
        if (listed) {
            const int any = __syncthreads_or(odd);
            if (threadIdx.x == 0) a.odd[(i * (int64_t)a.listed_pages + p) * gridDim.x + blockIdx.x] = any != 0;
        }
    }
}

}  // namespace sllm

using namespace sllm;

template <typename T, int W>
static int launch_write(const void* qkv, void* q_out, const WriteArgs& a, int64_t ctas, int threads, cudaStream_t stream) {
    return (int)sllm_launch_pdl(a.bias ? rope_kv_write_q8_kernel<T, W, true> : rope_kv_write_q8_kernel<T, W, false>,
                                dim3((unsigned)ctas), dim3(threads), 0, stream, (const T*)qkv, (T*)q_out, a);
}

// write = 0: only the queries.  dtype 0: float32, 1: bfloat16.  block divides page_size.
SLLM_EXPORT int sllm_rope_kv_write_q8(const void* qkv, void* q_out, const int* row_start, const int* row_pos0, int n_rows,
                                      int n_tokens, int max_new, const float* cos_t, const float* sin_t, int rot,
                                      int interleaved, const float* bias, void* pages, void* scales, const int* table,
                                      int table_stride, int page_size, int block, int H, int G, int hd, int write, int dtype,
                                      cudaStream_t stream) {
    if (n_rows <= 0 || n_tokens <= 0 || max_new <= 0) return 0;
    if (H <= 0 || G <= 0 || hd <= 0 || hd > 256 || hd % 16 || rot < 0 || rot > hd || rot % 2 || page_size <= 0 || block <= 0 ||
        page_size % block || (dtype != 0 && dtype != 1))
        return (int)cudaErrorInvalidValue;
    if (((uintptr_t)pages | (uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)bias | (uintptr_t)cos_t | (uintptr_t)sin_t) & 15)
        return (int)cudaErrorInvalidValue;
    const bool wide = rot % 8 == 0;      // (the tables' rows are then whole 16-byte words too)
    const int W = wide ? 4 : 1;
    WriteArgs a = {row_start, row_pos0, cos_t, sin_t, bias, (uint8_t*)pages, (uint8_t*)scales, table, table_stride, page_size,
                   block, n_rows, n_tokens, H, G, hd, rot, interleaved, max_new == 1};
    const int upt = hd / (2 * W);
    // a block's group: a thread for sixteen units of what a row stores in a block (for four: 53 and 52 us in the two cases
    // above, before divisions went), one for each where a warp holds them
    const int64_t units = (int64_t)(max_new < block ? max_new : block) * upt;
    a.lanes = 1;
    while (a.lanes < WRITE_THREADS && (a.lanes < 32 ? a.lanes < units : 16 * (int64_t)a.lanes < units)) a.lanes *= 2;
    while (a.lanes > 32 && a.lanes < upt) a.lanes *= 2;      // (upt <= 128: a CTA holds a head)
    const int threads = a.lanes > 32 ? a.lanes : WRITE_THREADS;
    const int64_t slots = a.single ? n_rows : (int64_t)n_tokens / block + 2 * (int64_t)n_rows;
    const int in_cta = threads / a.lanes;
    if (slots * 2 * G > 0x7fffffff) return (int)cudaErrorInvalidValue;
    a.n_tasks = write ? (int)(slots * 2 * G) : 0;
    const int64_t kv_ctas = ((int64_t)a.n_tasks + in_cta - 1) / in_cta;
    // (few tokens share a token's heads out further: a thread's heads come one after the other)
    a.q_groups = H < 4 ? H : 4;
    while (a.q_groups < H && (int64_t)n_tokens * a.q_groups * upt < 148 * 256) a.q_groups = a.q_groups * 2 < H ? a.q_groups * 2 : H;
    a.n_q_items = (int64_t)n_tokens * a.q_groups;
    if (a.n_q_items > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const int at_once = threads / upt;
    int64_t q_ctas = (a.n_q_items + at_once - 1) / at_once;
    const int64_t most = 148 * 16 * 256 / threads;
    if (q_ctas > most) q_ctas = most;
    if (kv_ctas + q_ctas > 0x7fffffff) return (int)cudaErrorInvalidValue;
    a.kv_ctas = (int)kv_ctas;
    a.q_per_group = (H + a.q_groups - 1) / a.q_groups;
    a.q_at_once = at_once;
    a.lane_tokens = a.lanes / upt;
    a.page_blocks = page_size / block;
    a.by_lanes = divisor(a.lanes);
    a.by_upt = divisor(upt);
    a.by_planes = divisor(2 * G);
    a.by_g = divisor(G);
    a.by_block = divisor(block);
    a.by_page = divisor(page_size);
    a.by_q_groups = divisor(a.q_groups);
    const int64_t ctas = kv_ctas + q_ctas;
    if (dtype == 0) return wide ? launch_write<float, 4>(qkv, q_out, a, ctas, threads, stream)
                                : launch_write<float, 1>(qkv, q_out, a, ctas, threads, stream);
    return wide ? launch_write<__nv_bfloat16, 4>(qkv, q_out, a, ctas, threads, stream)
                : launch_write<__nv_bfloat16, 1>(qkv, q_out, a, ctas, threads, stream);
}

static int launch_read(void* out, ReadArgs a, int n_rows, int64_t most, int dtype, cudaStream_t stream) {
    if (a.G <= 0 || a.hd <= 0 || a.hd % 16 || a.page_size <= 0 || a.block <= 0 || a.page_size % a.block ||
        (int64_t)a.G * a.page_size * a.hd > (1 << 27) || ((uintptr_t)a.pages & 15) || ((uintptr_t)out & 31) ||
        (dtype != 0 && dtype != 1))
        return (int)cudaErrorInvalidValue;
    const int pieces = 2 * a.G * a.page_size * a.hd / (dtype == 0 ? READ_BYTES<float> : READ_BYTES<__nv_bfloat16>),
              per = READ_THREADS * READ_PIECES;
    if (most > 65535) most = 65535;
    a.by_hd = divisor(a.hd);
    a.by_page = divisor(a.page_size);
    a.by_block = divisor(a.block);
    a.page_blocks = a.page_size / a.block;
    for (int r = 0; r < n_rows; r += 65535) {
        a.first_row = r;
        const dim3 grid((pieces + per - 1) / per, (unsigned)most, n_rows - r < 65535 ? n_rows - r : 65535);
        const cudaError_t e =
            a.row_start && dtype == 1 ? sllm_launch_pdl(kv_read_q8_kernel<__nv_bfloat16, true>, grid, dim3(READ_THREADS), 0,
                                                        stream, (__nv_bfloat16*)out, a)
            : a.row_start ? cudaErrorInvalidValue
            : dtype == 0 ? sllm_launch_pdl(kv_read_q8_kernel<float, false>, grid, dim3(READ_THREADS), 0, stream, (float*)out, a)
                         : sllm_launch_pdl(kv_read_q8_kernel<__nv_bfloat16, false>, grid, dim3(READ_THREADS), 0, stream,
                                           (__nv_bfloat16*)out, a);
        if (e != cudaSuccess) return (int)e;
    }
    return 0;
}

SLLM_EXPORT int sllm_kv_read_q8(const void* pages, const void* scales, const int* table, int table_stride,
                                const int* row_from, const int* row_to, void* out, int* out_table, int out_stride,
                                int n_rows, int max_tokens, int page_size, int block, int G, int hd, int dtype,
                                cudaStream_t stream) {
    if (n_rows <= 0 || max_tokens <= 0) return 0;
    if (page_size <= 0) return (int)cudaErrorInvalidValue;
    const ReadArgs a = {(const uint8_t*)pages, (const uint8_t*)scales, table, table_stride, page_size, block, G, hd, 0,
                        row_from, row_to, nullptr, nullptr, nullptr, 0, 0, out_table, out_stride, nullptr};
    // (max_tokens positions that start anywhere touch this many pages)
    return launch_read(out, a, n_rows, (int64_t)(max_tokens - 1) / page_size + 2, dtype, stream);
}

SLLM_EXPORT int sllm_kv_read_q8_shares(int page_size, int G, int hd) {
    return (int)(((int64_t)2 * G * page_size * hd / READ_BYTES<__nv_bfloat16> + READ_THREADS * READ_PIECES - 1) / (READ_THREADS * READ_PIECES));
}

// What the queries of the listed rows see (row_list null: rows 0 .. n_list - 1), at most listed_pages pages a row, into
// out [n_list * listed_pages, 2, G, page_size, hd]; row r's part of out_table names the pages.  odd: a byte for each page and
// sllm_kv_read_q8_shares() of it, not 0 where a NaN was met, for which zero is read.  bfloat16 only.
SLLM_EXPORT int sllm_kv_read_q8_listed(const void* pages, const void* scales, const int* table, int table_stride,
                                       const int* row_start, const int* row_pos0, const int* row_list, int n_list,
                                       int window, int listed_pages, void* out, int* out_table, int out_stride, uint8_t* odd,
                                       int page_size, int block, int G, int hd, cudaStream_t stream) {
    if (n_list <= 0 || listed_pages <= 0) return 0;
    if ((int64_t)n_list * listed_pages > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const ReadArgs a = {(const uint8_t*)pages, (const uint8_t*)scales, table, table_stride, page_size, block, G, hd, 0,
                        nullptr, nullptr, row_start, row_pos0, row_list, window, listed_pages, out_table, out_stride, odd};
    return launch_read(out, a, n_list, listed_pages, 1, stream);
}
