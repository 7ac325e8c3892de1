// What the kernels of attention of a chunk over a paged cache share: parameters, the share of a CTA, the walk over its
// items, where partial results go.
#pragma once

#include "paged.cuh"
#include "paged_schedule.h"

namespace luxcuda {

struct ChunkParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;                    // may be null
    const int32_t* tables;
    const int32_t* q_starts;
    const int32_t* context;
    uint32_t* status;
    // workspace: the CTAs' first places (grid + 1), then maxima and sums and the unnormalised outputs of the items that are cut,
    // part_rows rows a part, two parts a CTA: 2 c for a piece that does not begin its item, 2 c + 1 for one that does
    ChunkPlace* places;
    float2* stats;
    float* parts;
    ChunkShape shape;
    uint32_t seqs, tokens, heads, kv_heads, group, dim, block_size, width, num_blocks;
    uint32_t item_heads, splits;   // query heads of an item (the last part of a group may have fewer), parts of a group
    uint32_t part_rows, part_pitch, grid;
    uint32_t weight, weight_rows;  // a key of an item of n rows weighs weight + n / weight_rows
    uint32_t narrow;               // the costs of a call of these sizes fit 32 bits
    float qscale;                  // scale * log2(e)
};

constexpr float CHUNK_NO_KEYS = -3.402823e+38f, CHUNK_LN2 = 0.6931471805599453f, CHUNK_LOG2E = 1.4426950408889634f;

// paged_chunk_tc.cu: the tensor-core kernel for 16-bit data
bool chunk_tc_takes(const ChunkParams& p, uint32_t dtype);
uint32_t chunk_tc_rows(uint32_t group);
LuxBackendError launch_chunk_tc(Context* ctx, ChunkParams& p, uint32_t dtype);

#ifdef __CUDACC__

struct ChunkSeq {
    uint32_t first, tokens, keys;
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, uint32_t s) {
    const int32_t total = (int32_t)p.tokens, limit = (int32_t)(p.width * p.block_size);
    const int32_t a = load_i32(p.q_starts + s), b = load_i32(p.q_starts + s + 1), n = load_i32(p.context + s);
    ChunkSeq r;
    r.first = (uint32_t)min(max(a, 0), total);
    r.tokens = (uint32_t)min(max(b, (int32_t)r.first), total) - r.first;
    r.keys = (uint32_t)min(max(n, 0), limit);
    return r;
}

// What the costs of a sequence weigh on the line that is dealt out: by the rows of its first tile.
__device__ __forceinline__ uint32_t chunk_weight(const ChunkParams& p, uint32_t tokens) {
    return p.weight + min(tokens, p.shape.tile_tokens) * p.item_heads / p.weight_rows;
}
// The places where this CTA begins and where the next one does, by all NT threads.  `scratch`: 2 * NT / 32 numbers,
// `found`: two places in shared memory.
template <int NT, typename U> __device__ __forceinline__ void chunk_share_of(const ChunkParams& p, U* scratch, ChunkPlace* found, uint32_t cta) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr uint32_t WARPS = NT / 32;
    U total = 0, first_cost = 0;
    ChunkSeq first_seq{};
#pragma unroll 1
    for (uint32_t s = tid; s < p.seqs; s += NT) {
        const ChunkSeq q = chunk_seq(p, s);
        const U c = chunk_weight(p, q.tokens) * sequence_cost<U>(p.shape, q.tokens, q.keys);
        if (s == tid) first_cost = c, first_seq = q;
        total += c;
    }
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (lane == 0) scratch[warp] = total;
    if (tid < 2) found[tid] = ChunkPlace{p.seqs, 0, 0, 0};
    __syncthreads();
    total = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < WARPS; i++) total += scratch[i];
    const U each = total / p.grid;
    const uint32_t rest = (uint32_t)(total - each * p.grid);
    U base = 0;
#pragma unroll 1
    for (uint32_t s0 = 0; s0 < p.seqs; s0 += NT) {
        const uint32_t s = s0 + tid;
        ChunkSeq q = first_seq;
        U c = first_cost;
        if (s0) {
            c = 0;
            if (s < p.seqs) {
                q = chunk_seq(p, s);
                c = chunk_weight(p, q.tokens) * sequence_cost<U>(p.shape, q.tokens, q.keys);
            }
        }
        U sum = c;
        for (int d = 1; d < 32; d <<= 1) {
            const U v = __shfl_up_sync(0xffffffffu, sum, d);
            if ((int)lane >= d) sum += v;
        }
        __syncthreads();
        if (lane == 31) scratch[WARPS + warp] = sum;
        __syncthreads();
        U before = base, all = base;
#pragma unroll 1
        for (uint32_t i = 0; i < WARPS; i++) {
            if (i < warp) before += scratch[WARPS + i];
            all += scratch[WARPS + i];
        }
        const U from = before + sum - c;
#pragma unroll 1
        for (uint32_t i = 0; i < 2; i++) {
            const U at = each * (cta + i) + rest * (cta + i) / p.grid;          // (rest and cta are below the grid)
            if (at >= from && at - from < c) found[i] = place_in<U>(p.shape, s, q.tokens, q.keys, (at - from) / chunk_weight(p, q.tokens));
        }
        base = all;
    }
    __syncthreads();
}

template <int NT> __device__ __forceinline__ void chunk_share(const ChunkParams& p, uint64_t* scratch, ChunkPlace* found, uint32_t cta) {
    if (p.narrow) chunk_share_of<NT, uint32_t>(p, reinterpret_cast<uint32_t*>(scratch), found, cta);
    else chunk_share_of<NT, uint64_t>(p, scratch, found, cta);
}

// The items of a CTA one after the other.
struct ChunkWalk {
    ChunkPlace at, end;
    ChunkSeq seq;
    uint32_t tiles;                // of the sequence
    bool fresh;                    // the sequence's lengths are still to be read
    uint32_t k0, k1, key_tiles;    // key tiles of the piece, and of the item
    // goes on to the next item with rows; false: there is none before the end.  (Used as for (walk.begin(..); walk.settle(p); walk.next()).)
    __device__ __forceinline__ bool settle(const ChunkParams& p) {
#pragma unroll 1
        while (true) {
            // beyond the end?
            if (at.seq > end.seq || at.seq >= p.seqs) return false;
            if (at.seq == end.seq) {
                if (at.head > end.head) return false;
                if (at.head == end.head && (at.tile > end.tile || (at.tile == end.tile && at.key_tile >= end.key_tile))) return false;
            }
            if (fresh) {
                fresh = false;
                seq = chunk_seq(p, at.seq);
                tiles = tiles_of(p.shape, seq.tokens);
            }
            if (at.tile < tiles) break;
            at.tile = at.key_tile = 0;
            if (tiles == 0 || ++at.head == p.shape.heads) {
                at.head = 0;
                at.seq++;
                fresh = true;
            }
        }
        const uint32_t sees = tile_sees(p.shape, seq.tokens, seq.keys, at.tile);
        key_tiles = sees / p.shape.tile_keys + (sees % p.shape.tile_keys != 0);
        k0 = at.key_tile;
        k1 = same_item(at, end) ? end.key_tile : key_tiles;
        return true;
    }
    __device__ __forceinline__ void begin(const ChunkPlace& from, const ChunkPlace& to) {
        at = from;
        end = to;
        fresh = true;
    }
    __device__ __forceinline__ void next() {
        at.tile++;
        at.key_tile = 0;
    }
    __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == key_tiles; }
};

// What an item is, from its place: the first query head, how many, the tokens of its tile.
struct ChunkItem {
    uint32_t kv_head, head0, heads, token0, tokens;        // token0: within the sequence
};
__device__ __forceinline__ ChunkItem chunk_item(const ChunkParams& p, const ChunkPlace& at, const ChunkSeq& seq) {
    ChunkItem r;
    r.kv_head = p.splits == 1 ? at.head : at.head / p.splits;
    const uint32_t part = at.head - r.kv_head * p.splits;
    r.head0 = r.kv_head * p.group + part * p.item_heads;
    r.heads = min(p.item_heads, p.group - part * p.item_heads);
    r.token0 = at.tile * p.shape.tile_tokens;
    r.tokens = min(p.shape.tile_tokens, seq.tokens - r.token0);
    return r;
}
// Keys that a token of the sequence's new ones sees.
__device__ __forceinline__ uint32_t token_sees(const ChunkParams& p, const ChunkSeq& seq, uint32_t token) {
    if (!p.shape.causal) return seq.keys;
    const int64_t n = (int64_t)seq.keys - seq.tokens + token + 1;
    return n > 0 ? (uint32_t)n : 0u;
}

__device__ __forceinline__ float chunk_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two f32 numbers in one register pair: one instruction for both
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


// An item that several CTAs share is put together by this kernel, a warp per row: a lane per part finds where the part is and
// its maximum and sum, then the warp adds the parts, scaled to the largest maximum, in the order of the keys (32 at a time, with
// the running-maximum rule in between).  blockIdx.x: the boundary between CTA x and x + 1; it acts where it is the first inside its item.
template <typename T> __global__ void __launch_bounds__(128) lux_paged_chunk_merge(const ChunkParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t c = blockIdx.x + 1, lane = threadIdx.x & 31;
    auto place = [&](uint32_t i) {
        const uint4 v = load_u32x4(p.places + i);
        return ChunkPlace{v.x, v.y, v.z, v.w};
    };
    const ChunkPlace prev = place(c - 1), at = place(c);
    if (at.key_tile == 0) return;
    if (same_item(prev, at) && prev.key_tile) return;
    const ChunkSeq seq = chunk_seq(p, at.seq);
    const ChunkItem item = chunk_item(p, at, seq);
    const uint32_t rows = item.heads * item.tokens;
    for (uint32_t r = blockIdx.y * 4 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 4) {
        float top = -INFINITY, sum = 0.0f, acc[8];
#pragma unroll
        for (int j = 0; j < 8; j++) acc[j] = 0.0f;
        // the parts: CTA c - 1's, which begins the item, and those of CTAs c, c + 1, .. that begin inside it and are not empty
#pragma unroll 1
        for (uint32_t i0 = c - 1; i0 < p.grid; i0 += 32) {
            const uint32_t i = i0 + lane;
            bool inside = false, part = false;
            if (i < p.grid) {
                const ChunkPlace here = place(i), next = place(i + 1);
                inside = i == c - 1 || same_item(here, at);
                part = i == c - 1 || (inside && !(same_item(here, next) && here.key_tile == next.key_tile));
            }
            const uint32_t slot = 2 * i + (i == c - 1 ? 1u : 0u);
            float2 st = make_float2(-INFINITY, 0.0f);
            if (part) st = load_f32x2(p.stats + (size_t)slot * p.part_rows + r);
            float most = fmaxf(top, st.x);
            for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            // (a part without keys has no maximum, and nothing was written for it)
            const float f = st.y == 0.0f ? 0.0f : st.x == most ? 1.0f : chunk_ex2(st.x - most), before = top == most ? 1.0f : chunk_ex2(top - most);
            float share = st.y == 0.0f ? 0.0f : st.y * f;
            for (int d = 16; d; d >>= 1) share += __shfl_xor_sync(0xffffffffu, share, d);
            sum = (sum == 0.0f ? 0.0f : sum * before) + share;
#pragma unroll
            for (int j = 0; j < 8; j++) acc[j] *= i0 == c - 1 ? 0.0f : before;
            top = most;
            uint32_t with = __ballot_sync(0xffffffffu, part && st.y != 0.0f);
#pragma unroll 1
            while (with) {
                // four parts at a time, so that their loads are under way together
                float x[4][8], g[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int from = with ? __ffs(with) - 1 : 0;
                    const bool some = with != 0;
                    with &= with - 1;
                    g[k] = __shfl_sync(0xffffffffu, f, from);
                    const float* src = p.parts + ((size_t)__shfl_sync(0xffffffffu, slot, from) * p.part_rows + r) * p.part_pitch;
                    if (!some) g[k] = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; j++) x[k][j] = some && 32 * j + lane < p.dim ? load_f32(src + 32 * j + lane) : 0.0f;
                }
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int j = 0; j < 8; j++) acc[j] = fmaf(x[k][j], g[k], acc[j]);
            }
            if (!__all_sync(0xffffffffu, inside)) break;
        }
        const uint32_t token = seq.first + item.token0 + r / item.heads, head = item.head0 + r % item.heads;
        T* dst = reinterpret_cast<T*>(p.out) + ((size_t)token * p.heads + head) * p.dim;
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (32 * j + lane < p.dim) dst[32 * j + lane] = from_f32<T>(sum == 0.0f ? 0.0f : acc[j] / sum);
        if (p.lse && lane == 0) p.lse[(size_t)token * p.heads + head] = sum == 0.0f ? CHUNK_NO_KEYS : fmaf(top, CHUNK_LN2, logf(sum));
    }
}

#endif  // __CUDACC__

}  // namespace luxcuda
