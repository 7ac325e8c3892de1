// paged_chunk_tc.cu -- attention of a chunk over a paged cache of 16-bit data on the tensor cores: heads of up to 128
// (a multiple of 8), up to 128 query heads per KV head.
//
// s = q k^T, w = 2^(s scale' - m), o = w v / sum w (scale' = scale log2 e).  A CTA per SM walks its share of the items (paged_schedule.h).  An
// item's rows are (token, query head) pairs that share a KV head, two tiles of up to 128 rows; keys come in tiles of 64.
//   warp 9      goes through the items and tells the others what they are, and copies the queries
//   warps 9 and 13, 11 and 15   copy K and V, every other tile each (an issuing thread has about 16 boxes a tile with pages of 16: one warp
//               for both took 401 us where four take 268).  K of a tile and V of the one two tiles earlier are a stage of a ring;
//               TMA boxes have as many rows as divide a page (at most a tile).  Rows of V past the sequence's last key, up to the next 16,
//               repeat that key, so that no weight of zero meets what the cache holds there; rows of K there only make scores that are masked
//   warps 8, 10 issue the products of the first and of the second tile of rows: scores (128 x 64, f32, in tensor memory), and, once
//               its weights are there, the weighted sum (weights from tensor memory, over their own scores) onto the tile's output
//   warps 0..3, 4..7   the softmax of the first and the second tile of rows, a thread per row: no exchange.  The output's
//               reference m is raised only when a score passes it by 2^8, by the same thread, in tensor memory
// Each tile of rows has two places for scores, so that the next ones are there when the softmax of a tile is done: scores of tile t + 2 are
// issued behind the weighted sum of tile t.  (With one place, for 128 keys, a tile of rows waited for its products half of the time.)
// With 128 rows or fewer (a decode step, drafts) both groups work on the same rows: even key tiles and odd ones, each with an output
// of its own, joined at the end of the item.
// One thread issues all products of a tile of rows, so they run in order: when the scores of tile t + 1 are there, the weighted sum of
// tile t - 1 is complete, and so are the reads of the weights that scores overwrite.
//
// What must not be seen.  A masked score becomes -infinity, its weight zero: but zero times a value that is no number is none.  A row whose
// output comes out as NaN is therefore done again by its warp, over the keys that it sees (rows_again).
//
// Rounding.  Weights are rounded to the data's type (their sum is of the unrounded ones, in f32); for f16 they are taken times 2^7, so that
// weights down to 2^-31 of the largest one keep their place (subnormal f16 begin at 2^-14); 2^8 2^7 is in range.
//
// What bounds it (times of calls that follow one another, with the merge; in brackets replayed in a graph).  Single tokens: HBM, 32 over up to 8192
// keys (8 KV heads of 128, f16, 568 MB) 130 us, 4.4 TB/s (111 us, 5.1 TB/s).  Prompts: the chain of a softmax thread per tile of keys, 2048
// tokens over 8192 keys (32 heads of 128, bf16, 241 GFLOP) 288 us, 0.84 PFLOP/s (260 us, 0.93); tensor pipe 47 % active.
#include "paged_chunk.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace luxcuda {

namespace {
namespace ctc {

using namespace tcptx;

constexpr int BM = 128, BN = 64;           // rows and keys per tile
constexpr int THREADS = 512;
constexpr int REGS = 128, REGS_S = 184, REGS_C = 72;       // at launch, of the two softmax groups, of the other two
static_assert(2 * REGS_S + 2 * REGS_C <= 4 * REGS, "what the launch has");
constexpr float RAISE = 8.0f;
constexpr int EMULATED = 2;               // of eight pairs of weights, those whose powers are taken on the FMA pipe (2048 new tokens over 8192: 0 273 us, 2 268)
// the polynomial of ex2_pair
constexpr float EX2_C0 = 1.0f, EX2_C1 = 0.6931471824645996f, EX2_C2 = 0.2402234971523285f, EX2_C3 = 0.055503811687231064f, EX2_C4 = 0.00966636836528778f,
                EX2_C5 = 0.0013381302123889327f;
constexpr uint32_t T_S = 0, T_O = 256;     // tensor memory columns: scores (and weights) 2 x 128, outputs 2 x DP

template <int DP> struct Layout {
    static constexpr int TILE = BN * DP * 2, QTILE = BM * DP * 2;          // a tile of K or V, of queries
    static constexpr int STAGES = DP == 128 ? 4 : 8;       // of the ring: K of a tile and V of an earlier one
    // queries, ring, 4 KB per softmax warp on the outputs' way out, maxima and sums of the second group, barriers, flags
    static constexpr int Q = 0, RING = 2 * QTILE, OUT = RING + 2 * STAGES * TILE, STAT = OUT + 8 * 4096, BAR = STAT + 128 * 8, FLAG = BAR + 176 + 16 * STAGES,
                         ITEMS = FLAG + 64, SMEM = ITEMS + 128 + 1024;
};

static_assert(Layout<128>::SMEM <= 232448 && Layout<64>::SMEM <= 232448, "shared memory");

struct Maps {
    CUtensorMap q, q_one, k, v, v_one;
};

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A bounded wait: false when it gave up or another thread has.  The limit, some seconds, allows for rows that are done again (at most 4 us a key
// of an item).
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
#pragma unroll 1
    for (uint32_t it = 0; it < (1u << 20); ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((it & 31u) == 31u && *abort_flag) return false;
    }
    *abort_flag = 1u;
    return false;
}
// By all lanes of a warp.  (One polling lane and a shuffle took 300 cycles more: decode of 32 sequences 149 against 134 us.)
__device__ __forceinline__ bool warp_wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
    const bool ok = __all_sync(0xffffffffu, wait_bar(bar, parity, abort_flag));
    __syncwarp();
    return ok;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// MN-major, 128-byte swizzle: rows of 128 bytes are keys, eight of them an atom (SBO 1024), the next 64 columns one half tile on (LBO)
__device__ __forceinline__ uint64_t make_v_desc(uint32_t smem_addr) {
    const uint32_t lo = ((smem_addr & 0x3FFFFu) >> 4) | ((uint32_t)((BN * 128) >> 4) << 16);
    const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32f(uint32_t taddr, const float (&f)[32]) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; i++) r[i] = __float_as_uint(f[i]);
    tmem_st32(taddr, r);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
          "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// NaN if one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float v;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
    return v;
}
// 2^x for two numbers below 2^7 on the FMA pipe: x = j + f, j whole and |f| <= 1/2; 2^f = 1 + f r(f), r the polynomial of degree 4 that
// interpolates (2^f - 1) / f at the Chebyshev nodes of [-1/2, 1/2] (relative error 2.6e-07 in f32, ex2.approx has 2.4e-7), j added to its
// exponent.  At -127 and below (-infinity too) that gives 0, since 2^0 comes out as 1 exactly; a NaN is not kept (the row's maximum tells).
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
    float a, b;
    unpair(x, a, b);
    x = pair(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
    const uint64_t magic = pair(12582912.0f, 12582912.0f), minus = pair(-12582912.0f, -12582912.0f), neg = pair(-1.0f, -1.0f);
    const uint64_t j = add2(x, magic);
    const uint64_t f = fma2(add2(j, minus), neg, x);
    uint64_t v = pair(EX2_C5, EX2_C5);
    v = fma2(v, f, pair(EX2_C4, EX2_C4));
    v = fma2(v, f, pair(EX2_C3, EX2_C3));
    v = fma2(v, f, pair(EX2_C2, EX2_C2));
    v = fma2(v, f, pair(EX2_C1, EX2_C1));
    v = fma2(v, f, pair(EX2_C0, EX2_C0));
    float lo, hi, jl, jh;
    unpair(v, lo, hi);
    unpair(j, jl, jh);
    return pair(__uint_as_float(__float_as_uint(lo) + (__float_as_uint(jl) << 23)), __uint_as_float(__float_as_uint(hi) + (__float_as_uint(jh) << 23)));
}

// A piece of an item, as warp 9 hands it to the others.
struct Item {
    uint32_t more;                         // 0: there is none, the CTA is done
    uint32_t seq, keys;                    // the sequence, and its keys
    uint32_t k0, n;                        // first key tile; key tiles
    uint32_t whole;                        // all of the item's
    uint32_t kv_head, row0, tokens;        // first token's row of q, tokens
    int32_t sight;                         // token i sees sight + i keys (causal)
    uint32_t solo;                         // both groups on one tile of rows
    uint32_t own[2];                       // key tiles that each group works on: every one, or every other
    // group w's first tile, and from one of its tiles to the next
    __device__ __forceinline__ uint32_t first(uint32_t w) const { return solo ? w : 0u; }
    __device__ __forceinline__ uint32_t step() const { return solo ? 2u : 1u; }
};
__device__ __forceinline__ void fill_item(Item& r, const ChunkParams& p, const ChunkWalk& walk) {
    const ChunkItem item = chunk_item(p, walk.at, walk.seq);
    const uint32_t half = p.shape.tile_tokens / 2;
    r.seq = walk.at.seq;
    r.keys = walk.seq.keys;
    r.k0 = walk.k0;
    r.n = walk.k1 - walk.k0;
    r.whole = walk.whole();
    r.kv_head = item.kv_head;
    r.row0 = walk.seq.first + item.token0;
    r.tokens = item.tokens;
    r.sight = (int32_t)walk.seq.keys - (int32_t)walk.seq.tokens + (int32_t)item.token0 + 1;
    r.solo = item.tokens <= half;
    // of this piece's tiles, those up to the last key that a tile's last token sees
    auto tiles = [&](uint32_t token) {
        const uint32_t sees = token_sees(p, walk.seq, item.token0 + token), n = (sees + BN - 1) / BN;
        return n > walk.k0 ? min(n - walk.k0, r.n) : 0u;
    };
    const uint32_t all = tiles(item.tokens - 1);
    r.own[0] = r.solo ? (all + 1) / 2 : tiles(half - 1);
    r.own[1] = r.solo ? all / 2 : all;
}

// Rows of a warp over the keys [key0, their key1): sum of 2^(s scale' - ref) v times f, straight from the cache, as data to `out` or, given
// a row of the parts, as f32 there.  For rows that met a value that is no number behind a weight of zero: nothing that the row does not see is touched.  `again`: the
// lanes whose rows they are.  The whole warp takes N rows at a time over 32 keys at a time: a lane per key for the scores (queries as f32 in
// `stage`, N DP of them), a lane per DP / 32 columns for the sums.  256 tokens over 8192 keys, 32 heads of 128, all rows done again because of a NaN
// that all see: 7 ms; eight rows at a time 4.4, but with registers spilled that calls without such values miss (a prompt 0.6 %); one row
// at a time 20, a thread per row 43.
template <bool BF16, int DP>
__device__ __noinline__ void rows_again(const ChunkParams& p, uint32_t seq, uint32_t kv_head, uint32_t again, uint32_t my_row, uint32_t my_part, uint32_t key0,
                                         uint32_t my_key1, float my_ref, float my_f, float* stage) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int C = DP / 32, N = 4;
    static_assert(N * DP * 4 <= 4096, "the stage");
    constexpr uint32_t ALL = 0xffffffffu;
    const uint32_t lane = threadIdx.x & 31, col = C * lane;            // (a head is whole vectors of 8 elements, so of C as well)
    const int32_t* const table = p.tables + (size_t)seq * p.width;
#pragma unroll 1
    while (again) {
        uint32_t key1[N], least = ALL, most = 0;
        float ref[N], o[N][C];
        const uint32_t these = again;
        __syncwarp();                                      // the queries before have been read
#pragma unroll
        for (int r = 0; r < N; r++) {
            const int from = again ? __ffs(again) - 1 : 0;
            const uint32_t end = __shfl_sync(ALL, my_key1, from);
            key1[r] = again ? end : 0u;
            ref[r] = __shfl_sync(ALL, my_ref, from);
            most = max(most, key1[r]);
            if (again) least = min(least, end);
            const T* const q = reinterpret_cast<const T*>(p.q) + (size_t)__shfl_sync(ALL, my_row, from) * p.dim;
            for (uint32_t d = lane; again && d < p.dim; d += 32) stage[r * DP + d] = to_f32(q[d]);
            again &= again - 1;
#pragma unroll
            for (int c = 0; c < C; c++) o[r][c] = 0.0f;
        }
        __syncwarp();
#pragma unroll 1
        for (uint32_t first = key0; first < most; first += 32) {
            const uint32_t key = first + lane;
            int64_t at = -1;
            if (key < most) {
                const uint32_t b = key / p.block_size, block = (uint32_t)load_i32(table + b);
                if (block < p.num_blocks) at = (int64_t)((((size_t)block * p.kv_heads + kv_head) * p.block_size + (key - b * p.block_size)) * p.dim);
            }
            float w[N];
#pragma unroll
            for (int r = 0; r < N; r++) w[r] = 0.0f;
            if (at >= 0) {
                const uint4* const k = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.k) + at);
#pragma unroll 2
                for (uint32_t d = 0; d < p.dim / 8; d++) {
                    alignas(16) T x[8];
                    *reinterpret_cast<uint4*>(x) = k[d];
                    float e[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) e[j] = to_f32(x[j]);
#pragma unroll
                    for (int r = 0; r < N; r++) {
                        const float4 a = *reinterpret_cast<const float4*>(stage + r * DP + 8 * d), b = *reinterpret_cast<const float4*>(stage + r * DP + 8 * d + 4);
                        w[r] = fmaf(a.w, e[3], fmaf(a.z, e[2], fmaf(a.y, e[1], fmaf(a.x, e[0], w[r]))));
                        w[r] = fmaf(b.w, e[7], fmaf(b.z, e[6], fmaf(b.y, e[5], fmaf(b.x, e[4], w[r]))));
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < N; r++) w[r] = chunk_ex2(fmaf(w[r], p.qscale, -ref[r]));
            const bool all_see = first + 32 <= least;
#pragma unroll 4
            for (int j = 0; j < 32; j++) {
                const int64_t v_at = __shfl_sync(ALL, at, j);
                if (v_at < 0) continue;                    // (the same in all lanes)
                alignas(16) T y[C];
                if (col < p.dim) {
                    const T* const v = reinterpret_cast<const T*>(p.v) + v_at + col;
                    if constexpr (C == 4) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(v);
                    else *reinterpret_cast<uint32_t*>(y) = *reinterpret_cast<const uint32_t*>(v);
                } else {
#pragma unroll
                    for (int c = 0; c < C; c++) y[c] = from_f32<T>(0.0f);
                }
#pragma unroll
                for (int r = 0; r < N; r++) {
                    const float weight = __shfl_sync(ALL, w[r], j);
                    if (all_see || first + j < key1[r]) {
#pragma unroll
                        for (int c = 0; c < C; c++) o[r][c] = fmaf(weight, to_f32(y[c]), o[r][c]);
                    }
                }
            }
        }
        uint32_t rest = these;
#pragma unroll
        for (int r = 0; r < N; r++) {
            const int from = rest ? __ffs(rest) - 1 : 0;
            const size_t row = __shfl_sync(ALL, my_row, from);
            const float f = __shfl_sync(ALL, my_f, from);
            const uint32_t part = __shfl_sync(ALL, my_part, from);
            if (rest && col < p.dim) {
#pragma unroll
                for (int c = 0; c < C; c++) {
                    if (part != ALL) p.parts[(size_t)part * p.part_pitch + col + c] = o[r][c];
                    else reinterpret_cast<T*>(p.out)[row * p.dim + col + c] = from_f32<T>(o[r][c] * f);
                }
            }
            rest &= rest - 1;
        }
    }
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(THREADS, 1) lux_paged_chunk_tc(const __grid_constant__ Maps maps, const __grid_constant__ ChunkParams p, const uint32_t box_rows) {
    using L = Layout<DP>;
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int COLS = DP / 64;          // 64 columns of a head are a row of 128 bytes
    constexpr float BIAS = BF16 ? 0.0f : 7.0f;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    uint32_t* flag = reinterpret_cast<uint32_t*>(smem + L::FLAG);
    volatile uint32_t* abort_flag = flag;
    uint32_t* tmem_slot = flag + 1;
    ChunkPlace* found = reinterpret_cast<ChunkPlace*>(smem + L::FLAG + 16);
    Item* items = reinterpret_cast<Item*>(smem + L::ITEMS);
    float2* stat = reinterpret_cast<float2*>(smem + L::STAT);
    const uint32_t q_full = sb + L::BAR, q_empty = q_full + 8, st_full = q_full + 16, st_free = q_full + 24;
    auto s_full = [&](uint32_t w, uint32_t h) { return sb + L::BAR + 32 + 16 * w + 8 * h; };
    auto p_ready = [&](uint32_t w, uint32_t h) { return sb + L::BAR + 64 + 16 * w + 8 * h; };
    auto o_almost = [&](uint32_t w) { return sb + L::BAR + 96 + 8 * w; };      // behind an item's last weighted sum but one,
    auto o_full = [&](uint32_t w) { return sb + L::BAR + 112 + 8 * w; };       // and its last one
    auto o_free = [&](uint32_t w) { return sb + L::BAR + 128 + 8 * w; };
    auto item_full = [&](uint32_t i) { return sb + L::BAR + 144 + 8 * (i & 1); };
    auto item_empty = [&](uint32_t i) { return sb + L::BAR + 160 + 8 * (i & 1); };
    // use i of the ring is in stage i % STAGES; K (v 0) and V (v 1) of a stage
    auto kv_full = [&](uint32_t i) { return sb + L::BAR + 176 + 8 * (i % L::STAGES); };
    auto kv_empty = [&](uint32_t i) { return sb + L::BAR + 176 + 8 * (L::STAGES + i % L::STAGES); };
    auto stage_at = [&](uint32_t v, uint32_t i) { return sb + L::RING + (2 * (i % L::STAGES) + v) * L::TILE; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_launch_dependents();
    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 2);
        mbar_init(st_full, 4);
        mbar_init(st_free, 4);
        for (uint32_t w = 0; w < 2; w++) {
            for (uint32_t h = 0; h < 2; h++) {
                mbar_init(s_full(w, h), 1);
                mbar_init(p_ready(w, h), 4);
            }
            mbar_init(o_almost(w), 1);
            mbar_init(o_full(w), 1);
            mbar_init(o_free(w), 4);
            mbar_init(item_full(w), 1);
            mbar_init(item_empty(w), 13);  // the softmax warps, the copying ones but the first, two issuing threads
        }
        for (uint32_t i = 0; i < L::STAGES; i++) {
            mbar_init(kv_full(i), 2);      // both copying warps
            mbar_init(kv_empty(i), 2);     // both issuing threads
        }
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    if (warp == 9 && elect_one()) {
#pragma unroll
        for (const CUtensorMap* m : {&maps.q, &maps.q_one, &maps.k, &maps.v, &maps.v_one})
            asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    pdl_wait();
    chunk_share<THREADS>(p, reinterpret_cast<uint64_t*>(smem + L::RING), found, blockIdx.x);
    if (tid == 0) {
        p.places[blockIdx.x] = found[0];
        if (blockIdx.x + 1 == p.grid) p.places[p.grid] = ChunkPlace{p.seqs, 0, 0, 0};
    }
    fence_proxy_async_smem();              // the ring has held the sums of the shares
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot, quad = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t half = p.shape.tile_tokens / 2;         // tokens of a tile of rows
    uint32_t it = 0;                                       // items so far

    if (warp >= 8) {
        regs_dec<REGS_C>();
        if (warp & 1) {
            // ---- copies: warp 9 goes through the items and tells the others; 9 and 13 copy K (9 the queries too), 11 and 15 V, every other stage each --------
            const bool is_v = warp & 2, leads = warp == 9;
            const uint32_t parity = warp >= 12 ? 1u : 0u;
            const CUtensorMap *const map = is_v ? &maps.v : &maps.k, *const one = &maps.v_one;
            // a lane's box of a tile lies this much further in the next one but one: in blocks and places
            const uint32_t blocks_on = 2 * BN / p.block_size, places_on = 2 * BN % p.block_size;
            const uint32_t box_shift = 31 - __clz(box_rows);
            const bool boxed = box_rows * 32 >= BN;        // a tile has at most 32 boxes; else each is looked up when it is copied
            uint32_t base = 0, queries = 0;                // uses of the ring before this item, and tiles of queries so far
            bool ok = true;
            ChunkWalk walk;
            if (leads) walk.begin(found[0], found[1]);
#pragma unroll 1
            for (; ok; it++) {
                Item& shared = items[it & 1];
                if (!leads) {
                    if (!warp_wait_bar(item_full(it), (it >> 1) & 1, abort_flag)) break;
                } else {
                    if (it >= 2 && !warp_wait_bar(item_empty(it), ((it >> 1) - 1) & 1, abort_flag)) break;
                    const bool more = walk.settle(p);      // (the same in all lanes)
                    if (lane == 0) {
                        shared.more = more;
                        if (more) fill_item(shared, p, walk);
                        mbar_arrive(item_full(it));
                    }
                    walk.next();
                    __syncwarp();
                }
                const Item item = shared;
                __syncwarp();
                if (!leads && lane == 0) mbar_arrive(item_empty(it));
                if (!item.more) break;
                const uint32_t n = item.n, last = item.keys - 1;
                if (!n) continue;
                const int32_t* const table = p.tables + (size_t)item.seq * p.width;
                auto checked = [&](uint32_t block) {
                    if (block < p.num_blocks) return block;
                    report_status(p.status, STATUS_CACHE_BLOCK);
                    return 0u;
                };
                // stage i of the item: K of tile i and V of the tile whose weighted sum comes right before its scores
                const uint32_t late = is_v ? 2 * item.step() : 0u, end = n + 2 * item.step();
                uint32_t i = (base & 1) == parity ? 0u : 1u;
                const uint32_t key = (item.k0 + i) * BN + lane * box_rows;     // this warp's first tile (late is even)
                uint32_t at = key / p.block_size, place = key - at * p.block_size;     // of this lane's box: entry of the table, place in the block
                uint32_t ahead = at, ahead_place = place, ahead_key = key;
                // the entries of the tiles to come are read three tiles of this warp's ahead
                auto fetch = [&]() -> uint32_t {
                    const uint32_t block = boxed && lane * box_rows < BN && ahead_key <= last ? (uint32_t)load_i32(table + ahead) : 0u;
                    ahead_key += 2 * BN;
                    ahead += blocks_on;
                    ahead_place += places_on;
                    if (ahead_place >= p.block_size) ahead_place -= p.block_size, ahead++;
                    return block;
                };
                uint32_t b0 = fetch(), b1 = fetch(), b2 = fetch();
                bool asked = false;
#pragma unroll 1
                for (; i < end; i += 2) {
                    const uint32_t t = i - late, use = base + i;
                    if (leads && !asked && (i >= 2 || i + 1 >= n)) {           // the queries, once the scores of the item before are done
                        asked = true;
                        if (queries && !warp_wait_bar(q_empty, (queries - 1) & 1, abort_flag)) ok = false;
                        if (!ok) break;
                        queries++;
                        const uint32_t tiles = item.solo ? 1u : 2u;
                        uint32_t bytes = 0;
                        for (uint32_t w = 0; w < tiles; w++) {
                            const uint32_t tokens = min(half, item.tokens - w * half);
                            bytes += (2 * tokens > half ? half : tokens) * p.group * 128 * COLS;
                        }
                        if (lane == 0) mbar_expect_tx(q_full, bytes);
                        __syncwarp();
#pragma unroll 1
                        for (uint32_t w = 0; w < tiles; w++) {
                            const uint32_t tokens = min(half, item.tokens - w * half), dst = sb + L::Q + w * L::QTILE;
                            const int token = (int)(item.row0 + w * half), head0 = (int)(item.kv_head * p.group);
                            // a tile that is more than half full in one box, tokens behind the last one included
                            const bool full = 2 * tokens > half;
#pragma unroll 1
                            for (uint32_t j = lane; j < (full ? 1u : tokens) * COLS; j += 32) {
                                const uint32_t c = j % COLS, k = j / COLS;
                                tma_load_3d(dst + c * (BM * 128) + k * p.group * 128, full ? &maps.q : &maps.q_one, (int)c * 128, head0, token + (int)k, q_full);
                            }
                        }
                    }
                    const uint32_t bar = kv_full(use), dst = stage_at(is_v, use);
                    if (use >= L::STAGES && !warp_wait_bar(kv_empty(use), (use / L::STAGES - 1) & 1, abort_flag)) ok = false;
                    if (!ok) break;
                    if (t >= n) {                          // (V: in front of the first tile; K: behind the last one)
                        if (lane == 0) mbar_arrive(bar);
                        continue;
                    }
                    const uint32_t key0 = (item.k0 + t) * BN, keys = min((uint32_t)BN, item.keys - key0);
                    // whole boxes; of V, the last one goes row by row if it reaches behind the last key, and so does what then lacks to the
                    // next 16 rows, which the products read: always, since the ring holds an earlier tile there (or what another kernel left)
                    uint32_t boxes = BN >> box_shift, rows = BN, whole = BN;
                    if (keys < BN) {
                        boxes = (keys + box_rows - 1) >> box_shift;
                        rows = whole = boxes << box_shift;
                        if (is_v) {
                            if (whole > keys) boxes--, whole -= box_rows;
                            rows = (keys + 15) / 16 * 16;
                        }
                    }
                    if (lane == 0) mbar_expect_tx(bar, rows * 128 * COLS);
                    __syncwarp();
                    if (boxed && (uint32_t)lane < boxes) {
                        const int row = (int)((checked(b0) * p.kv_heads + item.kv_head) * p.block_size + place);
#pragma unroll
                        for (int c = 0; c < COLS; c++) tma_load_2d(dst + c * (BN * 128) + lane * box_rows * 128, map, c * 128, row, bar);
                    }
                    if (!boxed || whole < rows) {
#pragma unroll 1
                        for (uint32_t j = boxed ? whole + lane : lane; j < rows; j += 32) {
                            const uint32_t k = min(key0 + j, last), b = k / p.block_size;
                            const int row = (int)((checked((uint32_t)load_i32(table + b)) * p.kv_heads + item.kv_head) * p.block_size + (k - b * p.block_size));
#pragma unroll
                            for (int c = 0; c < COLS; c++) tma_load_2d(dst + c * (BN * 128) + j * 128, is_v ? one : map, c * 128, row, bar);
                        }
                    }
                    b0 = b1;
                    b1 = b2;
                    b2 = fetch();
                    place += places_on;
                    if (place >= p.block_size) place -= p.block_size;
                }
                base += end;
            }
            // no arrival may come after the CTA's end: the last uses of the stages and of the queries have been given back
            if (!is_v) {
                for (uint32_t i = base > L::STAGES ? base - L::STAGES : 0u; ok && i < base; i++)
                    if ((i & 1) == parity) ok = warp_wait_bar(kv_empty(i), (i / L::STAGES) & 1, abort_flag);
                if (ok && queries) warp_wait_bar(q_empty, (queries - 1) & 1, abort_flag);
            }
        } else if (warp < 12) {
            // ---- products of one tile of rows ------------------------------------------------------------
            if (elect_one()) {
                constexpr uint32_t id_s = make_idesc(BF16, BN), id_o = make_idesc(BF16, DP) | (1u << 16);
                const uint32_t w = warp == 8 ? 0u : 1u, s_tmem = tmem + T_S + w * 128, o_tmem = tmem + T_O + w * DP;
                uint32_t base = 0, queries = 0, used = 0, ready = 0;       // uses of the rings before this item; tiles of queries, outputs, phases of p_ready
                bool ok = true;
                auto wait_stage = [&](uint32_t e) { return wait_bar(kv_full(e), (e / L::STAGES) & 1, abort_flag); };
#pragma unroll 1
                for (; ok; it++) {
                    if (!wait_bar(item_full(it), (it >> 1) & 1, abort_flag)) break;
                    const Item& from = items[it & 1];
                    const bool more = from.more, solo = from.solo;
                    const uint32_t n = from.n, k0 = from.k0, all_keys = from.keys, own = from.own[w], first = from.first(w), step = from.step();
                    mbar_arrive(item_empty(it));
                    if (!more) break;
                    if (!n) continue;
                    const uint32_t end = n + 2 * step;     // stages of the item
                    const uint64_t qd = make_kmajor_sw128_desc(sb + L::Q + (solo ? 0u : w) * L::QTILE);
                    ok = wait_bar(q_full, queries & 1, abort_flag);
                    queries++;
                    if (ok && first >= n) umma_commit(q_empty);
                    // the scores of this thread's tile i, behind the weighted sum of tile i - 2
#pragma unroll 1
                    for (uint32_t i = 0, t = 0; ok && t < end; t++) {
                        // Both threads wait for every stage and give it back, the other's too: a wait tells one bit of the lap that a stage is on, so that a
                        // stage of which a thread missed a lap could be taken for filled one lap early (copies land in any order), or never.
                        const uint32_t use = base + t, h = i & 1;
                        ok = wait_stage(use);
                        if (!ok) break;
                        if (solo && (t & 1) != w) {
                            mbar_arrive(kv_empty(use));
                            continue;
                        }
                        if (i >= 2 && i - 2 < own) {
                            // the weights are there, and the output of the item before has been read
                            ok = wait_bar(p_ready(w, h), (ready >> h) & 1, abort_flag) && (i > 2 || !used || wait_bar(o_free(w), (used - 1) & 1, abort_flag));
                            if (!ok) break;
                            ready ^= 1u << h;
                            tc_fence_after();
                            // steps of 16 keys: those behind the sequence's last key are left out
                            const uint64_t vd = make_v_desc(stage_at(1, use));
                            const uint32_t keys = all_keys - (k0 + t - 2 * step) * BN;
#pragma unroll
                            for (int s = 0; s < 4; s++)
                                if (s * 16 < keys) mma_ts(o_tmem, s_tmem + h * 64 + s * 8, vd + (uint64_t)(s * (16 * 128 / 16)), id_o, i > 2 || s != 0);
                            if (i == own) umma_commit(o_almost(w));
                            if (i == own + 1) umma_commit(o_full(w));
                        }
                        if (i < own) {
                            tc_fence_after();
                            const uint64_t kd = make_kmajor_sw128_desc(stage_at(0, use));
#pragma unroll
                            for (int c = 0; c < COLS; c++)
#pragma unroll
                                for (int s = 0; s < 4; s++)
                                    mma_ss(s_tmem + h * 64, qd + (uint64_t)(c * (BM * 128 / 16) + 2 * s), kd + (uint64_t)(c * (BN * 128 / 16) + 2 * s), id_s,
                                            (c | s) != 0);
                            umma_commit(s_full(w, h));
                        }
                        umma_commit(kv_empty(use));
                        if (t < n && t + step >= n) umma_commit(q_empty);
                        i++;
                    }
                    if (own) used++;
                    base += end;
                }
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: a thread per row -------------------------------------------------------------------
        regs_inc<REGS_S>();
        const uint32_t w = (uint32_t)warp >> 2, r = (uint32_t)(tid & 127), s_tmem = quad + T_S + w * 128, o_tmem = quad + T_O + w * DP;
        unsigned char* const out_s = smem + L::OUT + warp * 4096;
        uint32_t scored = 0, outs = 0, almost = 0, joined = 0;             // phases of s_full(w, h), o_full(w), o_almost(w), st_full or st_free
        bool ok = true;
#pragma unroll 1
        for (; ok; it++) {
            if (!warp_wait_bar(item_full(it), (it >> 1) & 1, abort_flag)) break;
            const Item item = items[it & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(item_empty(it));
            if (!item.more) break;
            const uint32_t own = w ? item.own[1] : item.own[0], other = w ? item.own[0] : item.own[1];
            const uint32_t token = (item.solo ? 0u : w * half) + r / p.group, head = r % p.group;   // of the tile, of the KV head
            const bool mine = r < half * p.group && token < item.tokens;
            const uint32_t sees = !mine ? 0u : p.shape.causal ? (uint32_t)max(item.sight + (int32_t)token, 0) : item.keys;
            const uint32_t least = __reduce_min_sync(0xffffffffu, mine ? sees : 0xffffffffu);
            const bool rows = __any_sync(0xffffffffu, mine);       // of this warp
            float top = -INFINITY, ref = 0.0f, l = 0.0f;
#pragma unroll 1
            for (uint32_t v = 0; v < own; v++) {
                const uint32_t h = v & 1;
                ok = warp_wait_bar(s_full(w, h), (scored >> h) & 1, abort_flag);
                if (!ok) break;
                scored ^= 1u << h;
                tc_fence_after();
                if (!rows) {                               // whatever its weights are, nobody wants their sums
                    if (lane == 0) mbar_arrive(p_ready(w, h));
                    continue;
                }
                float x[64];
#pragma unroll
                for (int c = 0; c < 2; c++) tmem_ld32(s_tmem + h * 64 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[32 * c]));
                tmem_ld_wait();
                const uint32_t key0 = (item.k0 + item.first(w) + item.step() * v) * BN, left = sees > key0 ? sees - key0 : 0u;
                if (key0 + BN > least) {                   // some row of the warp does not see all of the tile
#pragma unroll
                    for (int j = 0; j < BN; j++)
                        if ((uint32_t)j >= left) x[j] = -INFINITY;
                }
                float mx[4];
#pragma unroll
                for (int j = 0; j < 4; j++) mx[j] = max3(x[j], x[j + 4], x[j + 8]);
#pragma unroll
                for (int j = 12; j < 60; j += 8)
#pragma unroll
                    for (int i = 0; i < 4; i++) mx[i] = max3(mx[i], x[j + i], x[j + 4 + i]);
                const float most = max3(max3(mx[0], mx[1], x[60]), max3(mx[2], mx[3], x[61]), max3(x[62], x[63], x[63])) * p.qscale;
                // the reference is raised: a score passes it by too much, is the row's first, or is no number
                const bool raise = mine && (!(most <= top + RAISE) || (top == -INFINITY && most > top));
                if (__any_sync(0xffffffffu, raise)) {
                    float alpha = 1.0f;
                    if (raise) {
                        if (!(most < INFINITY)) l = NAN;   // a score that is no number, or an infinite one: so is the row
                        alpha = chunk_ex2(top - most);
                        l *= alpha;
                        top = most;
                        ref = most - BIAS;
                    }
                    if (v) {
                        // the weighted sum before this one is complete when the scores behind it are there
                        ok = v + 1 < own ? warp_wait_bar(s_full(w, 1 - h), (scored >> (1 - h)) & 1, abort_flag)
                                         : warp_wait_bar(o_almost(w), almost & 1, abort_flag);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DP / 32; c++) {
                            float o[32];
                            tmem_ld32(o_tmem + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(o));
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; j++) o[j] *= alpha;
                            tmem_st32f(o_tmem + 32 * c, o);
                        }
                    }
                }
                const uint64_t scale2 = pair(p.qscale, p.qscale), ref2 = pair(-ref, -ref);
                uint64_t sum[2] = {0ull, 0ull};
                uint32_t pw[16];
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    uint64_t e = fma2(pair(x[2 * j], x[2 * j + 1]), scale2, ref2);
                    float a, b;
                    if (j % 8 < EMULATED) {
                        e = ex2_pair(e);
                        unpair(e, a, b);
                    } else {
                        unpair(e, a, b);
                        a = chunk_ex2(a);
                        b = chunk_ex2(b);
                        e = pair(a, b);
                    }
                    sum[j & 1] = add2(sum[j & 1], e);
                    pw[j & 15] = pack2<BF16>(a, b);
                    if ((j & 15) == 15) tmem_st16(s_tmem + h * 64 + (j & 16), pw);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(w, h));
                float a, b;
                unpair(add2(sum[0], sum[1]), a, b);
                l += a + b;
            }
            if (!ok) break;
            const bool any = own != 0;
            if (own > 1) ok = warp_wait_bar(o_almost(w), almost++ & 1, abort_flag);
            if (any) ok = warp_wait_bar(o_full(w), outs++ & 1, abort_flag) && ok;
            if (!ok) break;
            float other_f = 0.0f, own_f = 1.0f;
            bool both = false;
            if (item.solo) {
                if (w == 1) {                              // the second group's rows go to the first
                    stat[r] = make_float2(top == -INFINITY ? -INFINITY : ref, l);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(st_full);
                    ok = warp_wait_bar(st_free, joined++ & 1, abort_flag);
                    continue;
                }
                ok = warp_wait_bar(st_full, joined++ & 1, abort_flag);
                if (!ok) break;
                const float2 o = stat[r];
                both = other != 0;
                const float here = top == -INFINITY ? -INFINITY : ref, join = fmaxf(here, o.x);
                if (join != -INFINITY) {
                    own_f = here == join ? 1.0f : chunk_ex2(here - join);
                    other_f = o.x == join ? 1.0f : chunk_ex2(o.x - join);
                    l = (l == 0.0f ? 0.0f : l * own_f) + (o.y == 0.0f ? 0.0f : o.y * other_f);
                    ref = join;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(st_free);
            }
            tc_fence_after();
            // The rows leave by 32 columns at a time through shared memory, so that a store covers whole lines of few rows.
            const bool whole = item.whole;
            const float f = l == 0.0f ? 0.0f : 1.0f / l, scale = whole ? f : 1.0f;
            const uint32_t out_row = (item.row0 + token) * p.heads + item.kv_head * p.group + head;
            const uint32_t part_row = (2 * blockIdx.x + (item.k0 ? 0 : 1)) * p.part_rows + token * p.group + head;
            const uint32_t row = !mine ? 0xffffffffu : whole ? out_row : part_row;
            float odd = 0.0f;                              // NaN where an output is one
#pragma unroll 1
            for (int c = 0; c < DP / 32; c++) {
                float o[32];
                if (any) tmem_ld32(o_tmem + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(o));
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    o[j] = any ? o[j] * own_f : 0.0f;
                    odd = fmaf(o[j], 0.0f, odd);
                }
                if (both) {
                    float b[32];
                    tmem_ld32(quad + T_O + DP + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(b));
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        o[j] = fmaf(b[j], other_f, o[j]);
                        odd = fmaf(b[j], 0.0f, odd);
                    }
                }
                __syncwarp();                              // the chunk before has been read
                if (whole) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        *reinterpret_cast<uint4*>(out_s + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                            make_uint4(pack2<BF16>(o[8 * j] * scale, o[8 * j + 1] * scale), pack2<BF16>(o[8 * j + 2] * scale, o[8 * j + 3] * scale),
                                        pack2<BF16>(o[8 * j + 4] * scale, o[8 * j + 5] * scale), pack2<BF16>(o[8 * j + 6] * scale, o[8 * j + 7] * scale));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        *reinterpret_cast<float4*>(out_s + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                }
                __syncwarp();
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t rr = i * 8 + (lane >> 2), j = lane & 3, at = __shfl_sync(0xffffffffu, row, rr), d = 32 * c + 8 * j;
                        const uint4 x = *reinterpret_cast<const uint4*>(out_s + rr * 64 + ((j ^ ((rr >> 1) & 3)) << 4));
                        if (at != 0xffffffffu && d < p.dim) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (size_t)at * p.dim + d) = x;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint32_t rr = i * 4 + (lane >> 3), j = lane & 7, at = __shfl_sync(0xffffffffu, row, rr), d = 32 * c + 4 * j;
                        const float4 x = *reinterpret_cast<const float4*>(out_s + rr * 128 + ((j ^ (rr & 7)) << 4));
                        if (at != 0xffffffffu && d < p.dim) *reinterpret_cast<float4*>(p.parts + (size_t)at * p.part_pitch + d) = x;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (any) mbar_arrive(o_free(w));
                if (both) mbar_arrive(o_free(1));
            }
            const uint32_t again = __ballot_sync(0xffffffffu, mine && odd != odd && l == l);
            if (again)
                rows_again<BF16, DP>(p, item.seq, item.kv_head, again, out_row, whole ? 0xffffffffu : part_row, item.k0 * BN, min((item.k0 + item.n) * BN, sees),
                                     ref, f, reinterpret_cast<float*>(out_s));
            if (mine) {
                if (!whole) p.stats[part_row] = make_float2(l == 0.0f ? -INFINITY : ref, l);
                else if (p.lse) p.lse[out_row] = l == 0.0f ? CHUNK_NO_KEYS : fmaf(ref, CHUNK_LN2, logf(l));
            }
            __syncwarp();
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a bounded wait gave up: report it, and give copies in flight time to land
        if (tid == 0) report_status(p.status, STATUS_ATTENTION_WAIT);
        for (int i = 0; i < 64; i++) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <bool BF16, int DP> LuxBackendError launch(Context* ctx, const ChunkParams& p, const Maps& maps, uint32_t box_rows) {
    auto kfn = lux_paged_chunk_tc<BF16, DP>;
    static std::atomic<bool> configured[64];
    std::atomic<bool>& done = configured[ctx->device & 63];
    if (!done.load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute((const void*)kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<DP>::SMEM);
        if (e != cudaSuccess) return map_cuda(e, "paged_chunk_attention");
        done.store(true, std::memory_order_relaxed);
    }
    const cudaError_t e = launch_pdl(g_tune.pdl != 2, kfn, dim3(p.grid), dim3(THREADS), (size_t)Layout<DP>::SMEM, ctx->stream, 1, maps, p, box_rows);
    if (e != cudaSuccess) return map_cuda(e, "paged_chunk_attention");
    count_launch("lux_paged_chunk_tc");
    return LUX_BACKEND_OK;
}

}  // namespace ctc
}  // namespace

// What the kernel takes: 16-bit data, rows of whole 16 bytes, a scale that keeps the order of the scores (and -infinity).
bool chunk_tc_takes(const ChunkParams& p, uint32_t dtype) {
    return dtype != LUX_QDTYPE_F32 && p.dim <= 128 && p.dim % 8 == 0 && p.group <= 128 && p.qscale > 0.0f && p.qscale < INFINITY &&
            (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.out) & 15u) == 0 &&
            (uint64_t)p.num_blocks * p.kv_heads * p.block_size <= 0x7fffffffu;
}
uint32_t chunk_tc_rows(uint32_t group) { return group <= 128 ? 2 * (128 / group) * group : 0; }

// Fills in the shape and the grid, and launches.
LuxBackendError launch_chunk_tc(Context* ctx, ChunkParams& p, uint32_t dtype) {
    using namespace ctc;
    Maps maps;
    const uint64_t row = (uint64_t)p.dim * 2, rows = (uint64_t)p.num_blocks * p.kv_heads * p.block_size;
    uint32_t box_rows = std::min(p.block_size & (0u - p.block_size), (uint32_t)BN);
    const uint64_t q_dims[3] = {row, p.heads, p.tokens}, q_strides[2] = {row, row * p.heads}, c_dims[2] = {row, rows}, c_strides[1] = {row};
    const uint32_t tokens = 128 / p.group;
    const uint32_t q_box[3] = {128, p.group, tokens}, q_one[3] = {128, p.group, 1}, c_box[2] = {128, box_rows}, c_one[2] = {128, 1};
    if (!make_tensor_map_u8(&maps.q, 3, p.q, q_dims, q_strides, q_box, true) || !make_tensor_map_u8(&maps.q_one, 3, p.q, q_dims, q_strides, q_one, true) ||
        !make_tensor_map_u8(&maps.k, 2, p.k, c_dims, c_strides, c_box, true) || !make_tensor_map_u8(&maps.v, 2, p.v, c_dims, c_strides, c_box, true) ||
        !make_tensor_map_u8(&maps.v_one, 2, p.v, c_dims, c_strides, c_one, true))
        return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    const bool bf16 = dtype == LUX_QDTYPE_BF16;
    if (p.dim <= 64) return bf16 ? ctc::launch<true, 64>(ctx, p, maps, box_rows) : ctc::launch<false, 64>(ctx, p, maps, box_rows);
    return bf16 ? ctc::launch<true, 128>(ctx, p, maps, box_rows) : ctc::launch<false, 128>(ctx, p, maps, box_rows);
}

const void* kernel_addr_paged_chunk_tc() { return (const void*)ctc::lux_paged_chunk_tc<true, 128>; }

}  // namespace luxcuda
