// Causal attention of a packed batch over a paged cache held in 8 bits (q8.cuh): the token at absolute position p of
// row r attends to the keys 0 .. p of row r, or to the last `window` of them, and query head h reads kv head
// h / (H / G).  Scores, softmax and sums are 32-bit arithmetic.
//   s_j = scale * q . k_j,   out = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s)
// Compiled once per head size: -DSLLM_HEAD_DIM=<multiple of 16, at most 256>.
//
// Numbers.  An e4m3 number is a half exactly, and one instruction turns two of them, so the products run on the tensor
// cores' f16 form with the cache's numbers as they are (by bit operations, seven for four numbers, 64 rows of 4,096
// keys took 141 us instead of 124).  The blocks' powers of two join the scores (2^ek) and the probabilities (2^ev) in 32
// bits.  A query is brought into f16's range by a power of two of its own (largest entry
// in [2^14, 2^15)): bfloat16 entries keep all their bits down to 2^-31 of the largest (a half's steps end at 2^-24), 32-bit
// ones are split into two halves (22 bits down to 2^-16 of the largest, then steps of 2^-38 of it).  A probability is
// multiplied by its key's 2^ev before it becomes a half, against a running maximum of its own, M = max(s + ev) rounded up: what
// counts towards the output keeps 11 bits down to 2^-19 of the largest, whatever the blocks' scales.  In the 32-bit form
// the rest beside the half becomes one too, 2^11 times as large, and is brought back in 32 bits: 22 bits down to 2^-18, 20 at
// 2^-20 (unscaled it ran into the halves' steps: next to a key with most of the probability and values of zero 4.1e-5 off
// sum p |v|, now below 1.1e-5).
//
// Layout.  The products are taken transposed, keys and then the values' entries as the 16 rows of mma.m16n8k16, queries as
// its 8 columns: a decoded token's group of up to 8 query heads fills the instruction, and an output is spread over
// half as many registers.  Which entry of a head stands in which k step is free as long as queries and keys agree:
// a lane takes a quarter of each key's bytes as they lie, and of the values an eighth of four keys; P becomes an operand
// by movmatrix.  Every warp fetches tiles of its own into shared memory by TMA (one request per plane and tile where a
// page holds whole tiles, else one per run of keys), so that no warp waits for another before the end.  One tile a warp
// is on its way or worked on, four warps a scheduler cover the wait: 64 rows of 4,096 keys, 32 heads of 128 on 8 kv heads,
// take 97 us (5.5 TB/s); two tiles in turn for three warps a scheduler took 121 us, the keys of the next tile requested as
// soon as this one's are read 111, loads straight into registers 210: what counts is instructions and the warps that are
// there to issue them.  128-byte (heads of 64: 64-byte) swizzle: no two lanes of a read meet in a bank.  Other
// heads, and pages of no whole eights of tokens, come by untiled bulk copies, as they lie.
#include <cooperative_groups.h>

#include "q8.cuh"
#include "tc_common.cuh"

#ifndef SLLM_HEAD_DIM
#error "compile with -DSLLM_HEAD_DIM=<head size>"
#endif

namespace sllm {

constexpr int HD = SLLM_HEAD_DIM;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size: a multiple of 16 up to 256");
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int KSTEPS = HD / 16;                          // k steps of q k; also 16-row tiles of the values' entries
constexpr bool V_WORDS = HD % 32 == 0;                   // a lane's entries of a value are whole words (else 2 bytes a tile)
constexpr int VREGS = V_WORDS ? HD / 32 : HD / 16;
constexpr int DPL = (HD + 31) / 32;                      // entries of a head a lane (scalar form)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LOWEST = -1e30f;                         // below every score; finite, so that differences are numbers
constexpr float STALE = 8.f;                             // how far a maximum may lag behind the scores (base 2)
constexpr int MAX_CLUSTER = 8;                           // CTAs of a cluster, on every device of the kind
constexpr float P_SHIFT = 6.f;                           // probabilities become halves times 2^6: 2^14 at most
constexpr float REST = 2048.f;                           // what is left of a probability beside its half, times this

struct Q8Args {
    int64_t q_stride, out_stride;
    const uint8_t* pages; const uint8_t* scales; const int* table;
    const int* row_start; const int* row_pos0; const int* row_list;
    // [part_tokens, H, n_splits, HD + 2]: sums, maximum, denominator; listed row i's tokens from i * part_new on, or, where that
    // is 0, every token of the step at its own place
    float* part; int64_t part_tokens; int part_new;
    int table_stride, table_width, page_size, block, H, G, window, n_splits, per_split, one_length, q_vec, run, tiled, cluster;
    float scale_log2;
    Divisor page_div, block_div;
};

constexpr int KT = HD <= 128 ? 32 : 16;                  // keys of a tile
constexpr bool WIDE = HD % 128 == 0;                     // a tile is columns of 128 bytes, each [KT][128]
constexpr bool CAN_TILE = WIDE || HD == 64;
constexpr int WIDTH = WIDE ? 128 : HD;
// where byte b of a key (or value) lies in a tile of KT rows
__device__ __forceinline__ int place(int row, int b, bool swizzled) {
    if constexpr (WIDE) return (b / 128) * KT * 128 + row * 128 + ((b % 128 / 16 ^ (swizzled ? row & 7 : 0)) << 4) + b % 16;
    else if constexpr (HD == 64) return row * 64 + ((b / 16 ^ (swizzled ? row >> 1 & 3 : 0)) << 4) + b % 16;
    else return row * HD + b;
}

template <typename T, int NT> struct Form {
    static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;           // halves that an operand of T is split into
    static constexpr int Q_REGS = NT * PARTS * KSTEPS * 2;
    static constexpr bool Q_SHARED = Q_REGS > 32;
    static constexpr int LD = HD + 4;
    static constexpr int TILE = 2 * KT * HD;                      // bytes of a tile: keys, then values
    static constexpr int TILES = WARPS * TILE;
    static constexpr int MERGE = (int)sizeof(float) * WARPS * 8 * NT * LD;
    static constexpr int Q_BYTES = Q_SHARED ? (int)sizeof(uint32_t) * 32 * Q_REGS : 0;
    // the tiles (at the end the meeting of the warps takes their place), then the queries
    static constexpr int Q_AT = ((TILES > MERGE ? TILES : MERGE) + 1023) / 1024 * 1024;
    static constexpr size_t smem() { return 1024 + Q_AT + Q_BYTES; }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// d (16 x 8, f32) += a (16 x 16, f16) * b (16 x 8, f16)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {       // an 8 x 8 tile of halves
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t halves(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// what is left of (a, b) beside their halves
__device__ __forceinline__ uint32_t halves_rest(float a, float b, uint32_t h, float times = 1.f) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return halves((a - f.x) * times, (b - f.y) * times);
}

// bytes 0 and 1 of a word, and bytes 2 and 3, as pairs of halves
__device__ __forceinline__ void halves_of(uint32_t w, uint32_t& low, uint32_t& high) {
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
        : "=r"(low), "=r"(high) : "r"(w));
}

// BYTES of shared memory into words; where they lie in pieces of 16 bytes, piece i at p[i]
template <int BYTES, int N> __device__ __forceinline__ void take(const uint8_t* const (&p)[(BYTES + 15) / 16], int off, uint32_t (&w)[N]) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(p[i] + off);
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) {
            const uint2 x = *reinterpret_cast<const uint2*>(p[0] + off + 8 * i);
            w[2 * i] = x.x; w[2 * i + 1] = x.y;
        }
    } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p[0] + off + 4 * i);
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 2; ++i) w[i] = *reinterpret_cast<const uint16_t*>(p[0] + off + 2 * i);
    }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

// One query over the keys lo .. hi that it sees, key after key, by a warp: sums relative to m (base 2) in o (entry
// lane + 32 c), and (m, l).  For tiles in which a NaN came out: a product on the tensor cores multiplies also what a query
// does not see, by zero, and zero times a NaN is one.
template <typename T>
__device__ __noinline__ void attend_scalar(const T* __restrict__ q, const Q8Args& a, const int* __restrict__ table, int g,
                                           int lo, int hi, float* o, float& m, float& l) {
    const int lane = threadIdx.x & 31, blocks = a.page_size / a.block;
    float x[DPL];
    m = LOWEST;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < DPL; ++c) {
        x[c] = lane + 32 * c < HD ? to_float(q[lane + 32 * c]) * a.scale_log2 : 0.f;
        o[c] = 0.f;
    }
    for (int j = lo; j <= hi; ++j) {
        const int page = table[j / a.page_size], off = j % a.page_size;
        if (page < 0) continue;
        const int64_t k_plane = (int64_t)page * 2 * a.G + g, v_plane = k_plane + a.G;
        const uint8_t* k = a.pages + (k_plane * a.page_size + off) * HD;
        const uint8_t* v = a.pages + (v_plane * a.page_size + off) * HD;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < DPL; ++c)
            if (lane + 32 * c < HD) s = fmaf(x[c], q8_float2(k[lane + 32 * c]).x, s);
        s = warp_sum(s) * q8_power(a.scales[k_plane * blocks + off / a.block]);
        const float top = fmaxf(m, s), keep = exp2f(m - top);
        const float p = exp2f(s - top), pv = p * q8_power(a.scales[v_plane * blocks + off / a.block]);
        m = top;
        l = l * keep + p;
#pragma unroll
        for (int c = 0; c < DPL; ++c)
            if (lane + 32 * c < HD) o[c] = o[c] * keep + pv * q8_float2(v[lane + 32 * c]).x;
    }
}

// The place in a.part of the first token of the i-th listed row, token t0 of the step, and how many of the row's have one.
struct PartPlace {
    int64_t first; int tokens;
    __device__ __forceinline__ PartPlace(const Q8Args& a, int i, int t0) {
        first = a.part_new ? (int64_t)i * a.part_new : t0;
        tokens = a.part_new ? a.part_new : (int)(a.part_tokens - t0);
    }
};

// The queries of a row and kv head are packed: p = token * GS + j is the row's token `token` and query head g GS + j.  A
// CTA takes 8 NT packed queries over a share of the keys; its warps take turns at the tiles.  (Warps that share the
// queries between them, up to four times as many a CTA, fetch and turn every key as often, and were slower nearly
// everywhere: 32 rows of up to six drafted tokens 72 us with two groups of 16, 58 so, 51 with eight queries a CTA; 24
// queries a CTA are a few per cent better for uniform rows with just as many, and 15 to 20 worse for ragged ones.)  Up to
// eight splits can be a cluster, whose CTAs merge their sums through distributed shared memory (one row of 1,000 keys: 10.3
// us against 12.4 with a merge kernel); in launches that fill the device clusters find less room than CTAs by themselves (24
// rows of 4,096 keys of 64, three splits: 47 against 37), and the splits' sums meet in attn_q8_merge_kernel.  Where the
// CTAs do not all fit, a share is as long for all rows as the longest row needs, so that short rows have fewer: 16 rows of up
// to 16,000 keys and 24 packed queries 260 us unsplit, 129 in shares of a sixth; else each row is cut evenly.
// grid (kv heads, splits x tiles of queries, rows), the tiles with the most keys first.
template <typename T, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 4 : 3)
attn_q8_kernel(const T* __restrict__ q, T* __restrict__ out, const __grid_constant__ CUtensorMap map, const Q8Args a) {
    using F = Form<T, NT>;
    constexpr int PARTS = F::PARTS, KG = KT / 16, LD = F::LD;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    float* smem = reinterpret_cast<float*>(tiles);
    __shared__ uint64_t full[WARPS];
    __shared__ float sm_m[WARPS][8 * NT], sm_l[WARPS][8 * NT];
    __shared__ float all_top[8 * NT], all_total[8 * NT];      // of the CTA, for the cluster

    if (threadIdx.x == 0 && a.tiled) asm volatile("prefetch.tensormap [%0];\n" ::"l"(&map) : "memory");
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n8 = lane >> 2, c4 = lane & 3;
    const int r = a.row_list ? a.row_list[blockIdx.z] : blockIdx.z, g = blockIdx.x, GS = a.H / a.G;
    const int split = blockIdx.y % a.n_splits;
    const int q0 = ((int)(gridDim.y / a.n_splits) - 1 - (int)blockIdx.y / a.n_splits) * 8 * NT;
    const int* table = a.table + (int64_t)r * a.table_stride;
    // (asked for at once: the row, and the page of this lane's first key if the row is as long as the call says)
    const int t0 = __ldg(a.row_start + r), t1 = __ldg(a.row_start + r + 1), pos0 = __ldg(a.row_pos0 + r);
    const int guess_at = min(a.page_div.quotient((split * a.per_split + warp) * KT + lane % KT), a.table_width - 1);
    const int guess = __ldg(table + guess_at);
    const int n_packed = (t1 - t0) * GS;
    if (q0 >= n_packed) return;
    const int nq = min(n_packed - q0, 8 * NT);
    const int first_pos = pos0 + q0 / GS, last_pos = pos0 + (q0 + nq - 1) / GS;
    const int k_lo = a.window > 0 ? max(0, first_pos - a.window + 1) / KT * KT : 0;
    const int n_tiles = (last_pos - k_lo) / KT + 1;
    const int per_split = max(a.one_length ? a.per_split : 1, (n_tiles + a.n_splits - 1) / a.n_splits);
    const int tile_begin = min(n_tiles, split * per_split), tile_end = min(n_tiles, tile_begin + per_split);

    if (tile_begin >= tile_end && a.n_splits > 1 && !a.cluster) {      // no share: nothing is read or merged
        const PartPlace place(a, blockIdx.z, t0);
        for (int i = tid; i < nq; i += THREADS) {
            const int p = q0 + i, tok = p / GS, h = g * GS + p - tok * GS;
            if (tok < place.tokens) a.part[(((place.first + tok) * a.H + h) * a.n_splits + split) * (HD + 2) + HD + 1] = 0.f;
        }
        return;
    }

    // ---- tiles: lane i looks up key i (its page, then its two scales); where a page holds whole tiles lane 0 requests
    // them, else lane i the i-th run of `run` keys
    const int blocks = a.page_size / a.block;
    uint8_t* mine_at = tiles + warp * F::TILE;
    if (lane == 0) {
        mbar_init(&full[warp], 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    __syncwarp();
    auto page_of = [&](int tile) {
        const int kpos = k_lo + tile * KT + lane % KT;
        return tile < tile_end && kpos <= last_pos ? __ldg(table + a.page_div.quotient(kpos)) : -1;
    };
    // requests a tile and returns the bytes of this lane's key's two scales; -1: no such key
    auto request = [&](int tile, int page) {
        const int kpos = k_lo + tile * KT + lane % KT, off = kpos - a.page_div.quotient(kpos) * a.page_size;
        const uint32_t bar = smem_u32(&full[warp]), dst = smem_u32(mine_at);
        if (CAN_TILE && a.run == KT) {                         // (one page: lane 0's key is the tile's first)
            if (lane == 0) {
                mbar_expect_tx(&full[warp], page >= 0 ? F::TILE : 0);
                if (page >= 0)
#pragma unroll
                    for (int x = 0; x < HD; x += WIDTH) {
                        tma_load_3d(dst + x * KT, &map, bar, x, off, page * 2 * a.G + g);
                        tma_load_3d(dst + x * KT + KT * HD, &map, bar, x, off, (page * 2 + 1) * a.G + g);
                    }
            }
        } else {
            const int from = lane * a.run % KT;                // the first key of this lane's run
            const int run_page = __shfl_sync(0xffffffffu, page, from), run_off = __shfl_sync(0xffffffffu, off, from);
            const bool mine = lane * a.run < KT && run_page >= 0;
            const uint32_t asked = __ballot_sync(0xffffffffu, mine);
            if (lane == 0) mbar_expect_tx(&full[warp], (uint32_t)__popc(asked) * 2u * a.run * HD);
            __syncwarp();
            if (mine) {
                const uint32_t to = dst + lane * a.run * WIDTH;
                const int plane = run_page * 2 * a.G + g;
                if (CAN_TILE && a.tiled) {
#pragma unroll
                    for (int x = 0; x < HD; x += WIDTH) {
                        tma_load_3d(to + x * KT, &map, bar, x, run_off, plane);
                        tma_load_3d(to + x * KT + KT * HD, &map, bar, x, run_off, plane + a.G);
                    }
                } else {
                    const uint8_t* src = a.pages + ((int64_t)plane * a.page_size + run_off) * HD;
                    const int64_t v_off = (int64_t)a.G * a.page_size * HD;
                    const int rows = HD == WIDTH ? 1 : a.run, bytes = HD == WIDTH ? a.run * HD : WIDTH;
                    for (int i = 0; i < rows; ++i)
#pragma unroll
                        for (int x = 0; x < HD; x += WIDTH) {
                            bulk_load(to + x * KT + i * WIDTH, src + i * HD + x, bytes, bar);
                            bulk_load(to + x * KT + i * WIDTH + KT * HD, src + v_off + i * HD + x, bytes, bar);
                        }
                }
            }
        }
        if (page < 0) return -1;
        const uint8_t* s = a.scales + ((int64_t)page * 2 * a.G + g) * blocks + a.block_div.quotient(off);
        return (int)__ldg(s) | (int)__ldg(s + (int64_t)a.G * blocks) << 8;
    };
    // where this lane's pieces of a key (rows n8 + 8 i) and of a value (rows 2 c4, 2 c4 + 1, and 8 i on) lie in a tile
    const uint8_t* k_at[(HD / 4 + 15) / 16];
    const uint8_t* v_at[2][(HD / 8 + 15) / 16];
#pragma unroll
    for (int i = 0; i < (HD / 4 + 15) / 16; ++i) k_at[i] = mine_at + place(n8, c4 * (HD / 4) + 16 * i, a.tiled);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < (HD / 8 + 15) / 16; ++i)
            v_at[k][i] = mine_at + KT * HD + place(2 * c4 + k, n8 * (HD / 8) + 16 * i, a.tiled);
    constexpr int EIGHT = 8 * WIDTH;         // eight rows

    int tile = tile_begin + warp, page = guess, sc = -1, parity = 0;
    const int first_key = k_lo + tile * KT + lane % KT;
    if (tile >= tile_end || first_key > last_pos || a.page_div.quotient(first_key) != guess_at) page = page_of(tile);
    bool ok = true;
    if (tile < tile_end) sc = request(tile, page);
    page = page_of(tile + WARPS);

    // ---- its queries, while the first tile is on its way
    uint32_t qf[F::Q_SHARED ? 1 : PARTS][F::Q_SHARED ? 1 : NT][F::Q_SHARED ? 1 : KSTEPS][2];
    uint2* q_sh = reinterpret_cast<uint2*>(tiles + F::Q_AT) + lane;   // [part][nt][ks][lane]
    float fq[NT][2];                      // scale * log2 e / the query's power of two, of queries 2 c4 and 2 c4 + 1
    int qpos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int i = nt * 8 + n8, p = q0 + i;
        const bool there = i < nq;
        const int tok = there ? p / GS : 0, j = there ? p - tok * GS : 0;
        const T* src = q + (int64_t)(t0 + tok) * a.q_stride + (int64_t)(g * GS + j) * HD + c4 * (HD / 4);
        float x[HD / 4], top = 0.f;
        if (a.q_vec) {
#pragma unroll
            for (int d = 0; d < HD / 4; d += 4) {
                if constexpr (sizeof(T) == 4) {
                    Vec<float>::load(reinterpret_cast<const float*>(src) + d, x + d);
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(src + d);
                    x[d] = __uint_as_float(w.x << 16); x[d + 1] = __uint_as_float(w.x & 0xffff0000u);
                    x[d + 2] = __uint_as_float(w.y << 16); x[d + 3] = __uint_as_float(w.y & 0xffff0000u);
                }
            }
        } else {
#pragma unroll
            for (int d = 0; d < HD / 4; ++d) x[d] = to_float(src[d]);
        }
#pragma unroll
        for (int d = 0; d < HD / 4; ++d) {
            if (!there) x[d] = 0.f;
            top = fmaxf(top, q8_finite(x[d]) ? fabsf(x[d]) : 0.f);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^k with top * 2^k in [2^14, 2^15); at most 2^100, so that its inverse times the scale is a normal number
        const int k = top > 0.f ? min(100, 14 + 127 - (__float_as_int(top) >> 23)) : 0;
        const float up = __int_as_float((k + 127) << 23);
        const float own = a.scale_log2 * __int_as_float((127 - k) << 23);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            fq[nt][e] = __shfl_sync(0xffffffffu, own, (2 * c4 + e) * 4);
            const int pe = nt * 8 + 2 * c4 + e;
            qpos[nt][e] = pe < nq ? pos0 + (q0 + pe) / GS : -1;
        }
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            const float y0 = x[4 * ks] * up, y1 = x[4 * ks + 1] * up, y2 = x[4 * ks + 2] * up, y3 = x[4 * ks + 3] * up;
            const uint32_t h0 = halves(y0, y1), h1 = halves(y2, y3);
            uint32_t r0 = 0, r1 = 0;
            if constexpr (PARTS == 2) {
                r0 = halves_rest(y0, y1, h0);
                r1 = halves_rest(y2, y3, h1);
            }
            if constexpr (F::Q_SHARED) {
                if (nt % WARPS == warp) {
                    q_sh[(nt * KSTEPS + ks) * 32] = make_uint2(h0, h1);
                    if constexpr (PARTS == 2) q_sh[((NT + nt) * KSTEPS + ks) * 32] = make_uint2(r0, r1);
                }
            } else {
                qf[0][nt][ks][0] = h0; qf[0][nt][ks][1] = h1;
                if constexpr (PARTS == 2) { qf[1][nt][ks][0] = r0; qf[1][nt][ks][1] = r1; }
            }
        }
    }

    if constexpr (F::Q_SHARED) __syncthreads();

    float o[KSTEPS][NT][4], m[NT][2], M[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < KSTEPS; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][nt][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) { m[nt][e] = M[nt][e] = LOWEST; l[nt][e] = 0.f; }
    }

    for (; tile < tile_end; tile += WARPS) {
        const int kt = k_lo + tile * KT;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[warp], parity, 1));      // (a warp goes on or gives up as a whole)
        if (!ok) {                        // (given up on: once more as long for the copies under way)
            mbar_wait(&full[warp], parity, 1);
            break;
        }
        // ---- scores, transposed: rows are keys, columns queries
        float s[KG][NT][4];
#pragma unroll
        for (int i = 0; i < KG; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][nt][e] = 0.f;
        uint32_t kr[2 * KG][KSTEPS];
#pragma unroll
        for (int i = 0; i < 2 * KG; ++i) take<HD / 4>(k_at, i * EIGHT, kr[i]);
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) {
            uint32_t b[PARTS][NT][2];
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (F::Q_SHARED) {
                        const uint2 w = q_sh[((part * NT + nt) * KSTEPS + ks) * 32];
                        b[part][nt][0] = w.x; b[part][nt][1] = w.y;
                    } else {
                        b[part][nt][0] = qf[part][nt][ks][0]; b[part][nt][1] = qf[part][nt][ks][1];
                    }
                }
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                uint32_t f[4];
                halves_of(kr[2 * i][ks], f[0], f[2]);
                halves_of(kr[2 * i + 1][ks], f[1], f[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; --part) mma_f16(s[i][nt], f, b[part][nt][0], b[part][nt][1]);
            }
        }
        const bool there = sc >= 0;
        const bool whole = __all_sync(0xffffffffu, there) && kt + KT - 1 <= first_pos && (a.window <= 0 || kt > last_pos - a.window);
        uint32_t seen_rows = 0;
        // (in front of the first query's window lies nothing that any query here sees)
        if (!whole) seen_rows = __ballot_sync(0xffffffffu, there && (a.window <= 0 || kt + lane % KT > first_pos - a.window));

        // ---- scaled scores, their maxima
        const float own_k = __int_as_float((sc & 0xff) << 23), own_v = (float)(sc >> 8 & 0xff) - 127.f;
        float ev[KG][2];                  // the values' exponents of this lane's keys
#pragma unroll
        for (int i = 0; i < KG; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int key = 16 * i + 8 * k + n8;
                const float fk = __shfl_sync(0xffffffffu, own_k, key);
                ev[i][k] = __shfl_sync(0xffffffffu, own_v, key);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = s[i][nt][2 * k + e] * fq[nt][e] * fk;
                        if (!whole) {
                            const int kpos = kt + key;
                            const bool ok = (seen_rows >> key & 1u) && kpos <= qpos[nt][e] &&
                                            (a.window <= 0 || kpos > qpos[nt][e] - a.window);
                            x = ok ? x : -INFINITY;
                        }
                        s[i][nt][2 * k + e] = x;
                    }
            }
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < KG; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float x = s[i][nt][2 * k + e];
                        moved |= x > m[nt][e] + STALE || x + ev[i][k] > M[nt][e] + STALE;
                    }
        if (__any_sync(0xffffffffu, moved)) {
            // (seldom after a row's first tiles: a maximum may lag by 2^8, which halves and sums hold)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = m[nt][e], Top = M[nt][e];
#pragma unroll
                    for (int i = 0; i < KG; ++i)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            top = fmaxf(top, s[i][nt][2 * k + e]);
                            Top = fmaxf(Top, s[i][nt][2 * k + e] + ev[i][k]);
                        }
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) {
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        Top = fmaxf(Top, __shfl_xor_sync(0xffffffffu, Top, x));
                    }
                    // (whole numbers: their differences are exact, and so are the powers of two that bring sums together)
                    top = ceilf(top);
                    Top = ceilf(Top);
                    l[nt][e] *= ex2(m[nt][e] - top);
                    const float keep = ex2(M[nt][e] - Top);
                    m[nt][e] = top;
                    M[nt][e] = Top;
#pragma unroll
                    for (int j = 0; j < KSTEPS; ++j) {
                        o[j][nt][e] *= keep;
                        o[j][nt][2 + e] *= keep;
                    }
                }
        }
        // ---- probabilities, as the second operand
        uint32_t p[PARTS][KG][NT][2];
#pragma unroll
        for (int i = 0; i < KG; ++i)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float y[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = s[i][nt][2 * k + e];
                        l[nt][e] += ex2(x - m[nt][e]);
                        y[e] = ex2(x + (ev[i][k] + P_SHIFT - M[nt][e]));
                    }
                    const uint32_t h = halves(y[0], y[1]);
                    p[0][i][nt][k] = transposed(h);
                    if constexpr (PARTS == 2) p[1][i][nt][k] = transposed(halves_rest(y[0], y[1], h, REST));
                }
        // ---- sums over the keys, transposed: rows are entries of a head.  The instruction cuts its sums off towards zero, which adds
        // up over a row's keys: in the 32-bit form a tile's products start from nothing, both parts by themselves, and are added
        // with a rounding.  300 tokens after 3,000, heads of 64: 0.7e-6 off the exact result instead of 2.1e-6 (32-bit arithmetic as
        // written: 1.3e-6).  (Product after product, each with its second part brought back, took 174 us for heads of 128; this 169.)
        auto take_values = [&](int i, uint32_t (&vr)[4][VREGS]) {             // of keys 16 i .. 16 i + 15
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                take<HD / 8>(v_at[k & 1], (2 * i + (k >> 1)) * EIGHT, vr[k]);
                if (!whole && !(seen_rows >> (16 * i + 2 * c4 + (k & 1) + 8 * (k >> 1)) & 1u))
#pragma unroll
                    for (int w = 0; w < VREGS; ++w) vr[k][w] = 0u;         // (a place without a key that is seen may hold a NaN)
            }
        };
        auto entries = [&](int j, const uint32_t (&vr)[4][VREGS], uint32_t (&f)[4]) {
            // (bytes 0 and 1: entry 2 j of two keys, bytes 2 and 3: entry 2 j + 1)
            constexpr uint32_t LOW = 0x5140, HIGH = 0x7362;
            const int w = V_WORDS ? j / 2 : j;
            const uint32_t pick = V_WORDS && (j & 1) ? HIGH : LOW;
            const uint32_t x = __byte_perm(vr[0][w], vr[1][w], pick);
            const uint32_t y = __byte_perm(vr[2][w], vr[3][w], pick);
            halves_of(x, f[0], f[1]);
            halves_of(y, f[2], f[3]);
        };
        if constexpr (PARTS == 1) {
#pragma unroll
            for (int i = 0; i < KG; ++i) {
                uint32_t vr[4][VREGS], f[4];
                take_values(i, vr);
#pragma unroll
                for (int j = 0; j < KSTEPS; ++j) {
                    entries(j, vr, f);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16(o[j][nt], f, p[0][i][nt][0], p[0][i][nt][1]);
                }
            }
        } else {
            uint32_t vr[KG][4][VREGS], f[KG][4];
#pragma unroll
            for (int i = 0; i < KG; ++i) take_values(i, vr[i]);
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j) {
#pragma unroll
                for (int i = 0; i < KG; ++i) entries(j, vr[i], f[i]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float x[PARTS][4] = {};
#pragma unroll
                    for (int i = 0; i < KG; ++i)
#pragma unroll
                        for (int part = 0; part < PARTS; ++part) mma_f16(x[part], f[i], p[part][i][nt][0], p[part][i][nt][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][nt][e] += fmaf(x[PARTS - 1][e], 1.f / REST, x[0][e]);
                }
            }
        }
        __syncwarp();                     // (the tile is read)
        if (tile + WARPS < tile_end) sc = request(tile + WARPS, page);
        page = page_of(tile + 2 * WARPS);
        parity ^= 1;
    }

    // ---- the groups of keys meet
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x *= 2) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
            if (n8 == 0) {
                sm_m[warp][nt * 8 + 2 * c4 + e] = m[nt][e];
                sm_l[warp][nt * 8 + 2 * c4 + e] = l[nt][e];
            }
        }
    __syncthreads();                      // (all tiles are done with)
    float* sums = smem;                   // [WARPS][8 NT][LD]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = nt * 8 + 2 * c4 + e;
            float top = LOWEST;
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_m[w][i]);
            const float f = ex2(M[nt][e] - P_SHIFT - top);
            float* to = sums + (warp * 8 * NT + i) * LD + n8 * (HD / 8);
#pragma unroll
            for (int j = 0; j < KSTEPS; ++j)
                *reinterpret_cast<float2*>(to + 2 * j) = make_float2(o[j][nt][e] * f, o[j][nt][2 + e] * f);
        }
    __syncthreads();
    auto to_out = [&](int i, int d, float sum, float total) {                 // query i's entry d
        const int p = q0 + i, tok = p / GS, h = g * GS + p - tok * GS;
        out[(int64_t)(t0 + tok) * a.out_stride + (int64_t)h * HD + d] = from_float<T>(total == 0.f ? 0.f : sum / total);
    };
    const PartPlace place(a, blockIdx.z, t0);
    auto leave = [&](int i, int d, float sum, float top, float total) {
        const int p = q0 + i, tok = p / GS, h = g * GS + p - tok * GS;
        if (a.n_splits == 1) {
            to_out(i, d, sum, total);
        } else if (a.cluster) {
            sums[i * LD + d] = sum;                      // (query i's place of the first warp)
            if (d == 0) { all_top[i] = top; all_total[i] = total; }
        } else if (tok < place.tokens) {
            float* part = a.part + (((place.first + tok) * a.H + h) * a.n_splits + split) * (HD + 2);
            part[d] = sum;
            if (d == 0) { part[HD] = top; part[HD + 1] = total; }
        }
    };
    bool odd = false;
    for (int idx = tid; idx < nq * HD; idx += THREADS) {
        const int i = idx / HD, d = idx - i * HD;
        float top = LOWEST, total = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, sm_m[w][i]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            total += sm_l[w][i] * ex2(sm_m[w][i] - top);
            sum += sums[(w * 8 * NT + i) * LD + d];
        }
        odd |= isnan(sum) || isnan(total);
        leave(i, d, sum, top, total);
    }
    // a NaN, and not all queries see the same keys (queries of one token do, and what they do not see is zeros above): each of
    // them by itself, but for those whose denominator is one: they see a key with a NaN
    if (__syncthreads_or(odd) && first_pos != last_pos) {
        for (int i = warp; i < nq; i += WARPS) {
            bool sees = false;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) sees |= isnan(sm_l[w][i]);
            if (sees) continue;
            const int p = q0 + i, tok = p / GS, pos = pos0 + tok;
            const int lo = max(k_lo + tile_begin * KT, a.window > 0 ? pos - a.window + 1 : 0);
            const int hi = min(k_lo + tile_end * KT - 1, pos);
            float sum[DPL], top, total;
            attend_scalar<T>(q + (int64_t)(t0 + tok) * a.q_stride + (int64_t)(g * GS + p - tok * GS) * HD, a, table, g, lo, hi,
                             sum, top, total);
#pragma unroll
            for (int c = 0; c < DPL; ++c)
                if (lane + 32 * c < HD) leave(i, lane + 32 * c, sum[c], top, total);
        }
    }
    if (a.n_splits > 1 && a.cluster) {
        // every CTA merges a share of the entries, in the splits' order
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        for (int idx = split * THREADS + tid; idx < nq * HD; idx += a.n_splits * THREADS) {
            const int i = idx / HD, d = idx - i * HD;
            float tops[MAX_CLUSTER], top = LOWEST, total = 0.f, sum = 0.f;
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; ++k) {
                tops[k] = k < a.n_splits ? cluster.map_shared_rank(all_top, k)[i] : LOWEST;
                top = fmaxf(top, tops[k]);
            }
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; ++k) {
                if (k >= a.n_splits) continue;
                const float f = ex2(tops[k] - top);
                total += cluster.map_shared_rank(all_total, k)[i] * f;
                sum += cluster.map_shared_rank(sums, k)[i * LD + d] * f;
            }
            to_out(i, d, sum, total);
        }
        cluster.sync();                   // (nobody leaves while others read)
    }
}

// Joins the splits: a CTA per token and head, whose warps share the splits.  grid (tokens of a row x heads, rows).
template <typename T>
__global__ void __launch_bounds__(THREADS) attn_q8_merge_kernel(T* __restrict__ out, const Q8Args a) {
    __shared__ float sums[WARPS][HD], totals[WARPS];
    pdl_wait();
    pdl_trigger();
    const int r = a.row_list ? a.row_list[blockIdx.y] : blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tok = blockIdx.x / a.H, h = blockIdx.x - tok * a.H, t0 = a.row_start[r];
    const PartPlace place(a, blockIdx.y, t0);
    if (tok >= a.row_start[r + 1] - t0 || tok >= place.tokens) return;
    const int64_t ld = HD + 2;
    const float* part = a.part + ((place.first + tok) * a.H + h) * a.n_splits * ld;
    float top = LOWEST, total = 0.f, sum[DPL];
    // (a total of zero: a share without a key)
    for (int k = lane; k < a.n_splits; k += 32)
        if (part[k * ld + HD + 1] != 0.f) top = fmaxf(top, part[k * ld + HD]);
    top = warp_max(top);
#pragma unroll
    for (int c = 0; c < DPL; ++c) sum[c] = 0.f;
#pragma unroll 4
    for (int k = warp; k < a.n_splits; k += WARPS) {
        const float mine = part[k * ld + HD + 1];
        if (mine == 0.f) continue;
        const float f = ex2(part[k * ld + HD] - top);
        total += mine * f;
#pragma unroll
        for (int c = 0; c < DPL; ++c)
            if (lane + 32 * c < HD) sum[c] += part[k * ld + lane + 32 * c] * f;
    }
#pragma unroll
    for (int c = 0; c < DPL; ++c)
        if (lane + 32 * c < HD) sums[warp][lane + 32 * c] = sum[c];
    if (lane == 0) totals[warp] = total;
    __syncthreads();
    total = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += totals[w];
    for (int d = threadIdx.x; d < HD; d += THREADS) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) x += sums[w][d];
        out[(int64_t)(t0 + tok) * a.out_stride + (int64_t)h * HD + d] = from_float<T>(total == 0.f ? 0.f : x / total);
    }
}

// After portions were attended to in 16 bits, where a NaN was read back as zero (a product on the tensor cores multiplies also
// what a query does not see, by zero, and zero times a NaN is one): the queries that see one get it, all entries where it is
// in a key, its entries where in a value.  A warp per token and kv head of the rows that hold any (bytes of the row's
// part of `odd`), which looks through the pages so marked up to the first such key.  All other outputs stay as they are.
// 2,048 tokens after 6,144, 32 heads of 128 on 8 kv heads: 3 us where there is none, 27 us for a token of NaN at place 10 and
// 290 at place 7,000 (attending to the queries one by one, key after key, took 1.4 s).
constexpr int ODD_THREADS = 512, ODD_WARPS = ODD_THREADS / 32;
__device__ __forceinline__ bool any_nan(const uint4& x) {
    auto of = [](uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u; };
    return (of(x.x) | of(x.y) | of(x.z) | of(x.w)) != 0u;
}
// whether a warp meets a NaN among `bytes` bytes, a multiple of 16
__device__ __forceinline__ bool warp_any_nan(const uint8_t* p, int bytes) {
    bool any = false;
#pragma unroll 4
    for (int i = (threadIdx.x & 31) * 16; i < bytes; i += 512) any |= any_nan(__ldg(reinterpret_cast<const uint4*>(p + i)));
    return __any_sync(0xffffffffu, any);
}
template <typename T>
__global__ void __launch_bounds__(ODD_THREADS) attn_q8_odd_kernel(T* __restrict__ out, const uint8_t* __restrict__ odd,
                                                                  int listed_pages, int shares, int n_list, const Q8Args a) {
    pdl_wait();
    pdl_trigger();
    const int64_t per_row = (int64_t)listed_pages * shares, n_odd = per_row * n_list;
    bool any = false;
    const int64_t head = min(n_odd, (int64_t)((16 - ((uintptr_t)odd & 15)) & 15)), words = (n_odd - head) / 16;
    for (int64_t i = threadIdx.x; i < words; i += ODD_THREADS) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(odd + head) + i);
        any |= (x.x | x.y | x.z | x.w) != 0u;
    }
    for (int64_t i = threadIdx.x; i < head; i += ODD_THREADS) any |= odd[i] != 0;
    for (int64_t i = head + words * 16 + threadIdx.x; i < n_odd; i += ODD_THREADS) any |= odd[i] != 0;
    if (!__syncthreads_or(any)) return;
    const int lane = threadIdx.x & 31, GS = a.H / a.G;
    const T nan = from_float<T>(__int_as_float(0x7fffffff));
    for (int k = 0; k < n_list; ++k) {
        const uint8_t* flags = odd + per_row * k;
        any = false;
        for (int64_t i = threadIdx.x; i < per_row; i += ODD_THREADS) any |= flags[i] != 0;
        if (!__syncthreads_or(any)) continue;
        const int r = a.row_list ? a.row_list[k] : k, t0 = a.row_start[r], n_new = a.row_start[r + 1] - t0;
        const int* table = a.table + (int64_t)r * a.table_stride;
        for (int64_t i = (int64_t)blockIdx.x * ODD_WARPS + threadIdx.x / 32; i < (int64_t)n_new * a.G; i += (int64_t)gridDim.x * ODD_WARPS) {
            const int tok = (int)(i / a.G), g = (int)(i - (int64_t)tok * a.G), pos = a.row_pos0[r] + tok;
            const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
            bool key = false, value[DPL];
#pragma unroll
            for (int c = 0; c < DPL; ++c) value[c] = false;
            for (int p = lo / a.page_size; p <= min(pos / a.page_size, listed_pages - 1) && !key; ++p) {
                bool marked = false;
                for (int s = lane; s < shares; s += 32) marked |= flags[(int64_t)p * shares + s] != 0;
                if (!__any_sync(0xffffffffu, marked)) continue;
                // (a page that is marked is one)
                const int from = max(0, lo - p * a.page_size), n = min(a.page_size, pos - p * a.page_size + 1) - from;
                const uint8_t* k_at = a.pages + (((int64_t)table[p] * 2 * a.G + g) * a.page_size + from) * HD;
                const uint8_t* v_at = k_at + (int64_t)a.G * a.page_size * HD;
                key = warp_any_nan(k_at, n * HD);
                if (key || !warp_any_nan(v_at, n * HD)) continue;
                for (int j = 0; j < n; ++j)
#pragma unroll
                    for (int c = 0; c < DPL; ++c)
                        if (lane + 32 * c < HD) value[c] |= (v_at[j * HD + lane + 32 * c] & 0x7f) == 0x7f;
            }
            T* to = out + (int64_t)(t0 + tok) * a.out_stride + (int64_t)g * GS * HD;
#pragma unroll
            for (int c = 0; c < DPL; ++c)
                if (lane + 32 * c < HD && (key || value[c]))
                    for (int h = 0; h < GS; ++h) to[h * HD + lane + 32 * c] = nan;
        }
    }
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
    static EncodeFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) == cudaSuccess &&
            found == cudaDriverEntryPointSuccess)
            fn = (EncodeFn)p;
    }
    return fn;
}

template <typename T, int NT>
static int launch(const T* q, T* out, Q8Args a, int64_t n_pages, int n_list, int max_new, int q_tiles, cudaStream_t stream) {
    const size_t smem = Form<T, NT>::smem();
    // runs of keys that lie in a page and start a tile's share of it
    a.run = KT;
    while (a.page_size % a.run) a.run /= 2;
    // tiles by TMA: boxes that start on a whole pattern of the swizzle (eight rows), of the cache as (byte of a head, place
    // in a page, page and plane and head)
    a.tiled = CAN_TILE && a.run >= 8;
    CUtensorMap map = {};
    if (a.tiled) {
        const EncodeFn encode = encode_fn();
        if (!encode) return (int)cudaErrorNotSupported;
        const cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)a.page_size, (cuuint64_t)n_pages * 2 * a.G};
        const cuuint64_t strides[2] = {(cuuint64_t)HD, (cuuint64_t)HD * a.page_size};
        const cuuint32_t box[3] = {(cuuint32_t)WIDTH, (cuuint32_t)a.run, 1u}, one[3] = {1u, 1u, 1u};
        if (encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(a.pages), dims, strides, box, one,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, WIDE ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return (int)cudaErrorInvalidValue;
    }
    cudaError_t e = cudaFuncSetAttribute(attn_q8_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.G, a.n_splits * q_tiles, n_list);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {1u, (unsigned)a.n_splits, 1u};
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, attn_q8_kernel<T, NT>, q, out, map, (const Q8Args)a);
    if (e != cudaSuccess || a.n_splits == 1 || a.cluster) return (int)e;
    return (int)sllm_launch_pdl(attn_q8_merge_kernel<T>, dim3((unsigned)(max_new * a.H), n_list), dim3(THREADS), 0, stream,
                                out, a);
}

template <typename T, int NT> static int slots() {
    int device = 0, sms = 0, per = 0;
    if (cudaGetDevice(&device) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaFuncSetAttribute(attn_q8_kernel<T, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)Form<T, NT>::smem()) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, attn_q8_kernel<T, NT>, THREADS, Form<T, NT>::smem()) !=
            cudaSuccess)
        return 0;
    return sms * per;
}

}  // namespace sllm

using namespace sllm;

// CTAs that the device holds at once, of the form for 8 (nt = 1) or 16 (nt = 2) queries; 0: not known.
SLLM_EXPORT int sllm_attn_q8_slots(int dtype, int nt) {
    if (dtype == 0) return nt == 1 ? slots<float, 1>() : slots<float, 2>();
    return nt == 1 ? slots<__nv_bfloat16, 1>() : slots<__nv_bfloat16, 2>();
}
// keys of a warp's tile
SLLM_EXPORT int sllm_attn_q8_tile() { return KT; }

// The code of a wait that was given up since the last call, 0 if none was (synchronises the device).
SLLM_EXPORT int sllm_attn_q8_error() {
    int code = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&code, g_tc_error, sizeof(int)) != cudaSuccess) return -1;
    if (code) cudaMemcpyToSymbol(g_tc_error, &zero, sizeof(int));
    return code;
}

// nt: queries of a CTA / 8, 1 or 2.  merge 1: up to 8 splits are a cluster; else part, float [part_tokens, H,
// n_splits, HD + 2], takes the splits' sums, of shares of one length (0) or of rows cut evenly (2): part_tokens is n_list *
// max_new, or the tokens of the step where these are fewer.
SLLM_EXPORT int sllm_attn_q8(const void* q, int64_t q_stride, const void* pages, int64_t n_pages, const void* scales,
                             const int* table, int table_stride, int table_width, int page_size, int block,
                             const int* row_start, const int* row_pos0, const int* row_list, int n_list, int max_new,
                             int max_context, void* out, int64_t out_stride, int H, int G,
                             float scale, int window, int dtype, int nt, int n_splits, float* part,
                             int64_t part_tokens, int merge, cudaStream_t stream) {
    if (n_list <= 0 || max_new <= 0) return 0;
    if (H <= 0 || G <= 0 || H % G || page_size <= 0 || block <= 0 || page_size % block || window < 0 || n_list > 65535 ||
        table_width <= 0 || (dtype != 0 && dtype != 1) || (nt != 1 && nt != 2) || n_splits < 1 ||
        (merge == 1 ? n_splits > MAX_CLUSTER : n_splits > 1 && part == nullptr) || ((uintptr_t)pages & 15))
        return (int)cudaErrorInvalidValue;
    const int64_t q_tiles = ((int64_t)max_new * (H / G) + 8 * nt - 1) / (8 * nt);
    if (q_tiles * n_splits > 65535 || (int64_t)max_new * H > (1u << 30)) return (int)cudaErrorInvalidValue;
    const int es = dtype == 0 ? 4 : 2;
    const int64_t keys = window > 0 && (int64_t)window + max_new < max_context ? (int64_t)window + max_new : max_context;
    const int64_t share = ((keys + KT - 1) / KT + n_splits - 1) / n_splits;          // a row's at most
    const int q_vec = (uintptr_t)q % (4 * es) == 0 && q_stride % 4 == 0;
    const Q8Args a = {q_stride, out_stride, (const uint8_t*)pages, (const uint8_t*)scales, table, row_start, row_pos0, row_list,
                      part, part_tokens, part_tokens == (int64_t)n_list * max_new ? max_new : 0, table_stride, table_width, page_size,
                      block, H, G, window, n_splits,
                      (int)(share < 1 ? 1 : share), merge == 0, q_vec, 0, 0, merge == 1 && n_splits > 1, scale * LOG2E,
                      divisor(page_size), divisor(block)};
    typedef __nv_bfloat16 bf16;
    if (dtype == 0)
        return nt == 1 ? launch<float, 1>((const float*)q, (float*)out, a, n_pages, n_list, max_new, (int)q_tiles, stream)
                       : launch<float, 2>((const float*)q, (float*)out, a, n_pages, n_list, max_new, (int)q_tiles, stream);
    return nt == 1 ? launch<bf16, 1>((const bf16*)q, (bf16*)out, a, n_pages, n_list, max_new, (int)q_tiles, stream)
                   : launch<bf16, 2>((const bf16*)q, (bf16*)out, a, n_pages, n_list, max_new, (int)q_tiles, stream);
}

// See attn_q8_odd_kernel; odd: a byte for each of `shares` shares of each of the listed rows' listed_pages pages.
SLLM_EXPORT int sllm_attn_q8_odd(const void* pages, const int* table, int table_stride, int page_size, const int* row_start,
                                 const int* row_pos0, const int* row_list, int n_list, void* out, int64_t out_stride, int H, int G,
                                 int window, const uint8_t* odd, int listed_pages, int shares, cudaStream_t stream) {
    if (n_list <= 0 || listed_pages <= 0 || shares <= 0) return 0;
    if (H <= 0 || G <= 0 || H % G || page_size <= 0 || ((uintptr_t)pages & 15)) return (int)cudaErrorInvalidValue;
    Q8Args a = {};
    a.pages = (const uint8_t*)pages;
    a.table = table;
    a.table_stride = table_stride;
    a.page_size = page_size;
    a.row_start = row_start;
    a.row_pos0 = row_pos0;
    a.row_list = row_list;
    a.out_stride = out_stride;
    a.H = H;
    a.G = G;
    a.window = window;
    return (int)sllm_launch_pdl(attn_q8_odd_kernel<__nv_bfloat16>, dim3(148), dim3(ODD_THREADS), 0, stream, (__nv_bfloat16*)out,
                                odd, listed_pages, shares, n_list, a);
}
