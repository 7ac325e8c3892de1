// paged_chunk_tc.cu -- attention of a chunk over a paged cache of 16-bit data on the tensor cores: heads of up to 128
// (a multiple of 8), up to 128 query heads per KV head.
//
// s = q k^T, w = 2^(s scale' - m), o = w v / sum w (scale' = scale log2 e).  A CTA per SM walks its share of the items (paged_schedule.h).  An
// item's rows are (token, query head) pairs that share a KV head, two tiles of up to 128 rows; keys come in tiles of 128.
//   warp 9      copies: the item's queries, K and V of every tile into a ring of 32 KB stages, by TMA boxes of as many rows as
//               divide a page (at most a tile).  Rows of V past the sequence's last key, up to the next 16, repeat that key, so
//               that no weight of zero meets what the cache holds there; rows of K there only make scores that are masked
//   warp 8      issues the products: scores of a tile (128 x 128, f32, in tensor memory), then, once its weights are
//               there, the weighted sum (weights from tensor memory, over their own scores) onto the tile's output
//   warps 0..3, 4..7   the softmax of the first and the second tile of rows, a thread per row: no exchange.  The output's
//               reference m is raised only when a score passes it by 2^8, by the same thread, in tensor memory
// With 128 rows or fewer (a decode step, drafts) both groups work on the same rows: even key tiles and odd ones, each with an output
// of its own, joined at the end of the item.
// One thread issues all products, so they run in order: when a tile's scores are there, the weighted sum that the same
// group waited for before is complete, and so are the reads of the weights that the scores overwrite.
//
// What must not be seen.  A masked score becomes -infinity, its weight zero: but zero times a value that is no number is none.  A row whose
// output comes out as NaN is therefore done again by its thread, key by key, over the keys that it sees (row_again).
//
// Rounding.  Weights are rounded to the data's type (their sum is of the unrounded ones, in f32); for f16 they are taken times 2^7, so that
// weights down to 2^-31 of the largest one keep their place (subnormal f16 begin at 2^-14); 2^8 2^7 is in range.
#include "paged_chunk.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <atomic>

namespace luxcuda {

namespace {
namespace ctc {

using namespace tcptx;

constexpr int BN = 128;                    // keys per tile
constexpr int THREADS = 384;
constexpr int REGS = 168, REGS_S = 216, REGS_C = 72;       // at launch, of the softmax groups, of the others
static_assert(2 * REGS_S + REGS_C <= 3 * REGS, "what the launch has");
constexpr float RAISE = 8.0f;
constexpr uint32_t T_S = 0, T_O = 256;     // tensor memory columns: scores (and weights) 2 x 128, outputs 2 x DP

template <int DP> struct Layout {
    static constexpr int TILE = BN * DP * 2;               // a tile of K or V, and of queries
    static constexpr int STAGES = DP == 128 ? 5 : 10;
    static constexpr int Q = 0, RING = 2 * TILE, STAT = RING + STAGES * TILE, BAR = STAT + 128 * 8, FLAG = BAR + 256, SMEM = FLAG + 64 + 1024;
};

struct Maps {
    CUtensorMap q, q_one, k, v, v_one;
};

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// A bounded wait: false when it gave up or another thread has.  The limit allows for rows that are done again.
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag) {
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
__device__ __forceinline__ bool warp_wait_bar(uint32_t bar, uint32_t parity, volatile uint32_t* abort_flag, int lane) {
    bool ok = true;
    if (lane == 0) ok = wait_bar(bar, parity, abort_flag);
    __syncwarp();
    return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
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
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

// A piece of an item as the roles see it; all of them walk the same places.
struct Piece {
    bool solo;                             // both groups on one tile of rows
    uint32_t k0, n[2];                     // first key tile; tiles of each group (solo: of both together in n[0] and n[1] alike)
};
__device__ __forceinline__ Piece piece_of(const ChunkParams& p, const ChunkWalk& w, const ChunkItem& item) {
    Piece r;
    const uint32_t half = p.shape.tile_tokens / 2;
    r.solo = item.tokens <= half;
    r.k0 = w.k0;
    r.n[0] = r.n[1] = w.k1 - w.k0;
    if (!r.solo) {
        // the first tile of rows may see fewer keys
        const uint32_t sees = token_sees(p, w.seq, item.token0 + half - 1), tiles = (sees + BN - 1) / BN;
        r.n[0] = tiles > w.k0 ? min(tiles, w.k1) - w.k0 : 0u;
    }
    return r;
}

// One row over the keys [key0, key1): sum of 2^(s scale' - ref) v times f, straight from the cache, as data to `out` or as f32 to
// `part`.  For rows that met a value that is no number behind a weight of zero: nothing that the row does not see is touched.
template <bool BF16, int DP>
__device__ __noinline__ void row_again(const ChunkParams& p, uint32_t seq, uint32_t kv_head, size_t row, uint32_t key0, uint32_t key1, float ref, float f,
                                       float* part) {
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    float o[DP];
    for (int d = 0; d < DP; d++) o[d] = 0.0f;
    const T* q = reinterpret_cast<const T*>(p.q) + row * p.dim;
    for (uint32_t key = key0; key < key1; key++) {
        const uint32_t b = key / p.block_size;
        const int32_t block = load_i32(p.tables + (size_t)seq * p.width + b);
        if ((uint32_t)block >= p.num_blocks) continue;
        const size_t at = (((size_t)block * p.kv_heads + kv_head) * p.block_size + (key - b * p.block_size)) * p.dim;
        const T *k = reinterpret_cast<const T*>(p.k) + at, *v = reinterpret_cast<const T*>(p.v) + at;
        float s = 0.0f;
        for (uint32_t d = 0; d < p.dim; d++) s = fmaf(to_f32(q[d]), to_f32(k[d]), s);
        const float w = chunk_ex2(fmaf(s, p.qscale, -ref));
        for (uint32_t d = 0; d < p.dim; d++) o[d] = fmaf(w, to_f32(v[d]), o[d]);
    }
    for (uint32_t d = 0; d < p.dim; d++) {
        if (part) part[d] = o[d];
        else reinterpret_cast<T*>(p.out)[row * p.dim + d] = from_f32<T>(o[d] * f);
    }
}

template <bool BF16, int DP>
__global__ void __launch_bounds__(THREADS, 1) lux_paged_chunk_tc(const __grid_constant__ Maps maps, const ChunkParams p, const uint32_t box_rows) {
    using L = Layout<DP>;
    using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
    constexpr int HALVES = DP / 64;        // 64 columns of a head are a row of 128 bytes
    constexpr float BIAS = BF16 ? 0.0f : 7.0f;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t sb = smem_u32(smem);
    uint32_t* flag = reinterpret_cast<uint32_t*>(smem + L::FLAG);
    volatile uint32_t* abort_flag = flag;
    uint32_t* tmem_slot = flag + 1;
    ChunkPlace* found = reinterpret_cast<ChunkPlace*>(smem + L::FLAG + 16);
    float2* stat = reinterpret_cast<float2*>(smem + L::STAT);
    const uint32_t q_full = sb + L::BAR, q_empty = q_full + 8, st_full = q_full + 16, st_free = q_full + 24;
    auto s_full = [&](uint32_t w) { return sb + L::BAR + 32 + 8 * w; };
    auto p_ready = [&](uint32_t w) { return sb + L::BAR + 48 + 8 * w; };
    auto o_full = [&](uint32_t w) { return sb + L::BAR + 64 + 8 * w; };
    auto o_free = [&](uint32_t w) { return sb + L::BAR + 80 + 8 * w; };
    auto kv_full = [&](uint32_t i) { return sb + L::BAR + 96 + 8 * i; };
    auto kv_empty = [&](uint32_t i) { return sb + L::BAR + 96 + 8 * L::STAGES + 8 * i; };
    static_assert(96 + 16 * L::STAGES <= 256, "layout of the barriers");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_launch_dependents();
    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(st_full, 4);
        mbar_init(st_free, 4);
        for (uint32_t w = 0; w < 2; w++) {
            mbar_init(s_full(w), 1);
            mbar_init(p_ready(w), 4);
            mbar_init(o_full(w), 1);
            mbar_init(o_free(w), 4);
        }
        for (uint32_t i = 0; i < L::STAGES; i++) {
            mbar_init(kv_full(i), 1);
            mbar_init(kv_empty(i), 1);
        }
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    if (warp == 9 && elect_one()) {
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
    const ChunkPlace from = found[0], to = found[1];
    ChunkWalk walk;
    const uint32_t half = p.shape.tile_tokens / 2;         // tokens of a tile of rows

    if (warp >= 8) {
        regs_dec<REGS_C>();
        if (warp == 9) {
            // ---- copies ------------------------------------------------------------------------------
            uint32_t entry = 0, items = 0;                 // ring entries and items so far
            bool ok = true;
            for (bool more = walk.begin(p, from, to); more && ok; more = walk.next(p)) {
                const ChunkItem item = chunk_item(p, walk.at, walk.seq);
                const Piece pc = piece_of(p, walk, item);
                const uint32_t n = pc.n[1];
                if (!n) continue;
                const int32_t* table = p.tables + (size_t)walk.at.seq * p.width;
                const uint32_t last = walk.seq.keys - 1;
                auto row_of = [&](uint32_t key) -> int {   // of the cache as rows of a head
                    const uint32_t b = key / p.block_size;
                    uint32_t block = (uint32_t)load_i32(table + b);
                    if (block >= p.num_blocks) {
                        atomicOr(p.status, PAGED_STATUS_TABLE);
                        block = 0;
                    }
                    return (int)((block * p.kv_heads + item.kv_head) * p.block_size + (key - b * p.block_size));
                };
                auto load = [&](uint32_t t, bool is_v) {
                    const uint32_t stage = entry % L::STAGES, use = entry / L::STAGES, bar = kv_full(stage), dst = sb + L::RING + stage * L::TILE;
                    entry++;
                    if (use && !warp_wait_bar(kv_empty(stage), (use - 1) & 1, abort_flag, lane)) return false;
                    const uint32_t key0 = t * BN, keys = min((uint32_t)BN, walk.seq.keys - key0);
                    // whole boxes; of V, those that reach behind the last key go row by row
                    const uint32_t boxes = is_v ? keys / box_rows : (keys + box_rows - 1) / box_rows;
                    const uint32_t tail = is_v ? (keys + 15) / 16 * 16 : 0u;
                    const uint32_t single = is_v && tail > boxes * box_rows ? tail - boxes * box_rows : 0u;
                    if (lane == 0) mbar_expect_tx(bar, (boxes * box_rows + single) * 128 * HALVES);
                    __syncwarp();
                    for (uint32_t i = lane; i < boxes; i += 32) {
                        const int row = row_of(key0 + i * box_rows);
#pragma unroll
                        for (int h = 0; h < HALVES; h++) tma_load_2d(dst + h * (BN * 128) + i * box_rows * 128, is_v ? &maps.v : &maps.k, h * 128, row, bar);
                    }
                    for (uint32_t i = boxes * box_rows + lane; i < boxes * box_rows + single; i += 32) {
                        const int row = row_of(min(key0 + i, last));
#pragma unroll
                        for (int h = 0; h < HALVES; h++) tma_load_2d(dst + h * (BN * 128) + i * 128, &maps.v_one, h * 128, row, bar);
                    }
                    return true;
                };
                const uint32_t lead = pc.solo ? 2u : 1u;
                for (uint32_t t = 0; ok && t < min(lead, n); t++) ok = load(pc.k0 + t, false);
                if (!ok) break;
                // the queries, once the scores of the item before are done
                if (items && !warp_wait_bar(q_empty, (items - 1) & 1, abort_flag, lane)) break;
                items++;
                const uint32_t tiles = pc.solo ? 1u : 2u, heads = item.heads;
                uint32_t bytes = 0;
                for (uint32_t w = 0; w < tiles; w++) {
                    const uint32_t tokens = min(half, item.tokens - w * half);
                    bytes += (2 * tokens > half ? half : tokens) * heads * 128 * HALVES;
                }
                if (lane == 0) mbar_expect_tx(q_full, bytes);
                __syncwarp();
                for (uint32_t w = 0; w < tiles; w++) {
                    const uint32_t tokens = min(half, item.tokens - w * half), dst = sb + L::Q + w * L::TILE;
                    const int token = (int)(walk.seq.first + item.token0 + w * half);
                    if (2 * tokens > half) {               // in one box, tokens behind the last one included
                        if (lane < HALVES) tma_load_3d(dst + lane * (BN * 128), &maps.q, lane * 128, (int)item.head0, token, q_full);
                    } else {
                        for (uint32_t i = lane; i < tokens * HALVES; i += 32) {
                            const uint32_t h = i / tokens, k = i - h * tokens;
                            tma_load_3d(dst + h * (BN * 128) + k * heads * 128, &maps.q_one, (int)h * 128, (int)item.head0, token + (int)k, q_full);
                        }
                    }
                }
                for (uint32_t t = 0; ok && t < n; t++) {
                    ok = load(pc.k0 + t, true);
                    if (ok && t + lead < n) ok = load(pc.k0 + t + lead, false);
                }
            }
        } else if (warp == 8) {
            // ---- products ----------------------------------------------------------------------------
            if (elect_one()) {
                constexpr uint32_t id_s = make_idesc(BF16, BN), id_o = make_idesc(BF16, DP) | (1u << 16);
                uint32_t entry = 0, items = 0, ready[2] = {0, 0}, used[2] = {0, 0};
                bool ok = true;
                auto wait_stage = [&](uint32_t e) { return wait_bar(kv_full(e % L::STAGES), (e / L::STAGES) & 1, abort_flag); };
                auto stage_at = [&](uint32_t e) { return sb + L::RING + (e % L::STAGES) * L::TILE; };
                auto scores = [&](uint32_t q_tile, uint32_t w, uint32_t e) {
                    const uint64_t qd = make_kmajor_sw128_desc(sb + L::Q + q_tile * L::TILE), kd = make_kmajor_sw128_desc(stage_at(e));
#pragma unroll
                    for (int h = 0; h < HALVES; h++)
#pragma unroll
                        for (int s = 0; s < 4; s++)
                            mma_ss(tmem + T_S + w * 128, qd + (uint64_t)(h * (BN * 128 / 16) + 2 * s), kd + (uint64_t)(h * (BN * 128 / 16) + 2 * s), id_s,
                                   (h | s) != 0);
                    umma_commit(s_full(w));
                };
                // steps of 16 keys: those behind the sequence's last key are left out
                auto weighted = [&](uint32_t w, uint32_t e, uint32_t steps, bool first) {
                    const uint64_t vd = make_v_desc(stage_at(e));
                    for (uint32_t s = 0; s < steps; s++)
                        mma_ts(tmem + T_O + w * DP, tmem + T_S + w * 128 + s * 8, vd + (uint64_t)(s * (16 * 128 / 16)), id_o, !first || s != 0);
                };
                for (bool more = walk.begin(p, from, to); more && ok; more = walk.next(p)) {
                    const ChunkItem item = chunk_item(p, walk.at, walk.seq);
                    const Piece pc = piece_of(p, walk, item);
                    const uint32_t n = pc.n[1], lead = pc.solo ? 2u : 1u;
                    if (!n) continue;
                    ok = wait_bar(q_full, items & 1, abort_flag);
                    items++;
                    for (uint32_t t = 0; ok && t < min(lead, n); t++, entry++) {
                        ok = wait_stage(entry);
                        if (!ok) break;
                        tc_fence_after();
                        if (pc.solo) {
                            scores(0, t, entry);
                        } else {
                            if (pc.n[0]) scores(0, 0, entry);
                            scores(1, 1, entry);
                        }
                        umma_commit(kv_empty(entry % L::STAGES));
                    }
                    if (ok && n <= lead) umma_commit(q_empty);
                    for (uint32_t t = 0; ok && t < n; t++) {
                        const uint32_t ve = entry, ke = entry + 1;
                        const bool next = t + lead < n;
                        const uint32_t steps = (min((uint32_t)BN, walk.seq.keys - (pc.k0 + t) * BN) + 15) / 16;
                        ok = wait_stage(ve);
                        for (uint32_t w = pc.solo ? t & 1 : 0; ok && w < (pc.solo ? (t & 1) + 1 : 2u); w++) {
                            if (!pc.solo && t >= pc.n[w]) continue;
                            ok = wait_bar(p_ready(w), ready[w]++ & 1, abort_flag);
                            const bool first = t < lead;
                            // the output of the item before has been read
                            if (ok && first && used[w]) ok = wait_bar(o_free(w), (used[w] - 1) & 1, abort_flag);
                            if (!ok) break;
                            tc_fence_after();
                            weighted(w, ve, steps, first);
                            const bool last = pc.solo ? t + 2 >= n : t + 1 == pc.n[w];
                            if (last) {
                                umma_commit(o_full(w));
                                used[w]++;
                            }
                            if (next && (pc.solo || t + 1 < pc.n[w])) {
                                ok = wait_stage(ke);
                                if (!ok) break;
                                tc_fence_after();
                                scores(pc.solo ? 0 : w, w, ke);
                            }
                        }
                        if (!ok) break;
                        umma_commit(kv_empty(ve % L::STAGES));
                        entry++;
                        if (next) {
                            umma_commit(kv_empty(ke % L::STAGES));
                            entry++;
                            if (t + lead + 1 == n) umma_commit(q_empty);
                        }
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: a thread per row -------------------------------------------------------------------
        regs_inc<REGS_S>();
        const uint32_t w = (uint32_t)warp >> 2, r = (uint32_t)(tid & 127);
        uint32_t tiles_done = 0, outs = 0, joined = 0;     // phases of s_full(w), of o_full(w), of st_full or st_free
        bool ok = true;
        for (bool more = walk.begin(p, from, to); more && ok; more = walk.next(p)) {
            const ChunkItem item = chunk_item(p, walk.at, walk.seq);
            const Piece pc = piece_of(p, walk, item);
            const uint32_t token = item.token0 + (pc.solo ? 0u : w * half) + r / item.heads, head = item.head0 + r % item.heads;
            const bool mine = r < half * item.heads && token < item.token0 + item.tokens;
            const uint32_t sees = mine ? token_sees(p, walk.seq, token) : 0u;
            const uint32_t step = pc.solo ? 2u : 1u, n = pc.n[w];
            float top = -INFINITY, ref = 0.0f, l = 0.0f;
            bool first = true;
            for (uint32_t t = pc.solo ? w : 0u; t < n; t += step) {
                ok = warp_wait_bar(s_full(w), tiles_done++ & 1, abort_flag, lane);
                if (!ok) break;
                tc_fence_after();
                float s[BN];
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld32(quad + T_S + w * 128 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
                tmem_ld_wait();
                const uint32_t key0 = (pc.k0 + t) * BN, left = sees > key0 ? sees - key0 : 0u;
                if (__any_sync(0xffffffffu, left < BN)) {
#pragma unroll
                    for (int j = 0; j < BN; j++)
                        if ((uint32_t)j >= left) s[j] = -INFINITY;
                }
                float mx[4];
#pragma unroll
                for (int j = 0; j < 4; j++) mx[j] = fmaxf(s[j], s[j + 4]);
#pragma unroll
                for (int j = 8; j < BN; j++) mx[j & 3] = fmaxf(mx[j & 3], s[j]);
                const float most = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.qscale;
                float alpha = 1.0f;
                if (most > top + RAISE || (top == -INFINITY && most > top)) {
                    alpha = chunk_ex2(top - most);
                    l *= alpha;
                    top = most;
                    ref = most - BIAS;
                }
                if (!first && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
                    for (int c = 0; c < DP / 32; c++) {
                        float o[32];
                        tmem_ld32(quad + T_O + w * DP + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(o));
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j++) o[j] *= alpha;
                        tmem_st32f(quad + T_O + w * DP + 32 * c, o);
                    }
                }
                first = false;
                const uint64_t scale2 = pair(p.qscale, p.qscale), ref2 = pair(-ref, -ref);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    uint32_t pw[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        float x, y;
                        unpair(fma2(pair(s[64 * c + 2 * j], s[64 * c + 2 * j + 1]), scale2, ref2), x, y);
                        x = chunk_ex2(x);
                        y = chunk_ex2(y);
                        sum[j & 1] = add2(sum[j & 1], pair(x, y));
                        pw[j] = pack2<BF16>(x, y);
                    }
                    tmem_st32(quad + T_S + w * 128 + 32 * c, pw);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(w));
                float x, y;
                unpair(add2(sum[0], sum[1]), x, y);
                l += x + y;
            }
            if (!ok) break;
            const bool whole = walk.whole(), any = pc.solo ? n > w : n > 0;
            // this group's output is complete
            if (any) {
                ok = warp_wait_bar(o_full(w), outs++ & 1, abort_flag, lane);
                if (!ok) break;
            }
            float other_f = 0.0f, own_f = 1.0f;
            bool both = false;
            if (pc.solo) {
                if (w == 1) {                              // the second group's rows go to the first
                    stat[r] = make_float2(top == -INFINITY ? -INFINITY : ref, l);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(st_full);
                    ok = warp_wait_bar(st_free, joined++ & 1, abort_flag, lane);
                    if (!ok) break;
                    continue;
                }
                ok = warp_wait_bar(st_full, joined++ & 1, abort_flag, lane);
                if (!ok) break;
                const float2 o = stat[r];
                both = n > 1;
                const float own = top == -INFINITY ? -INFINITY : ref, join = fmaxf(own, o.x);
                if (join != -INFINITY) {
                    own_f = own == join ? 1.0f : chunk_ex2(own - join);
                    other_f = o.x == join ? 1.0f : chunk_ex2(o.x - join);
                    l = (l == 0.0f ? 0.0f : l * own_f) + (o.y == 0.0f ? 0.0f : o.y * other_f);
                    ref = join;
                    top = join;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(st_free);
            }
            tc_fence_after();
            float o[DP];
#pragma unroll
            for (int c = 0; c < DP / 32; c++) {
                if (any) tmem_ld32(quad + T_O + w * DP + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&o[32 * c]));
            }
            tmem_ld_wait();
            float odd = 0.0f;                              // NaN where an output is one
#pragma unroll
            for (int j = 0; j < DP; j++) {
                if (!any) o[j] = 0.0f;
                o[j] *= own_f;
                odd = fmaf(o[j], 0.0f, odd);
            }
            if (both) {
#pragma unroll
                for (int c = 0; c < DP / 32; c++) {
                    float b[32];
                    tmem_ld32(quad + T_O + DP + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(b));
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        o[32 * c + j] = fmaf(b[j], other_f, o[32 * c + j]);
                        odd = fmaf(b[j], 0.0f, odd);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (any) mbar_arrive(o_free(w));
                if (both) mbar_arrive(o_free(1));
            }
            if (!mine) continue;
            const size_t row = (size_t)(walk.seq.first + token) * p.heads + head;
            const size_t slot = (2 * (size_t)blockIdx.x + (walk.k0 ? 0 : 1)) * p.part_rows + (token - item.token0) * item.heads + (head - item.head0);
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
            if (odd != odd) {
                row_again<BF16, DP>(p, walk.at.seq, item.kv_head, row, pc.k0 * BN, min(walk.k1 * BN, sees), ref, f,
                                    whole ? nullptr : p.parts + slot * p.part_pitch);
            } else if (whole) {
                T* dst = reinterpret_cast<T*>(p.out) + row * p.dim;
#pragma unroll
                for (int j = 0; j < DP; j += 8) {
                    if (j < (int)p.dim) {
                        uint4 v;
                        v.x = pack2<BF16>(o[j] * f, o[j + 1] * f);
                        v.y = pack2<BF16>(o[j + 2] * f, o[j + 3] * f);
                        v.z = pack2<BF16>(o[j + 4] * f, o[j + 5] * f);
                        v.w = pack2<BF16>(o[j + 6] * f, o[j + 7] * f);
                        *reinterpret_cast<uint4*>(dst + j) = v;
                    }
                }
            } else {
                float* dst = p.parts + slot * p.part_pitch;
#pragma unroll
                for (int j = 0; j < DP; j += 4)
                    if (j < (int)p.dim) *reinterpret_cast<float4*>(dst + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            }
            if (!whole) p.stats[slot] = make_float2(l == 0.0f ? -INFINITY : ref, l);
            else if (p.lse) p.lse[row] = l == 0.0f ? CHUNK_NO_KEYS : fmaf(ref, CHUNK_LN2, logf(l));
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        // a bounded wait gave up: report it, and give copies in flight time to land
        if (tid == 0) atomicOr(p.status, PAGED_STATUS_WAIT);
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
