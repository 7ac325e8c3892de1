// paged_chunk.cu -- attention of a chunk of new tokens over a paged KV cache (lux/gpu/paged_ext.h): the entry point, and the
// kernel on the f32 FMA pipe, which takes every call that the tensor-core kernel (paged_chunk_tc.cu) does not: f32 data, heads
// wider than 128 or not a multiple of 8, unaligned views.
//
// Rows are (token, query head) pairs that share a KV head.  A CTA keeps RT rows and walks the keys that they see in tiles of 32, K
// and V of a tile in shared memory as f32, the next tile on its way: scores, the running maximum and sum of each row, and the weighted sum, whose
// outputs stay in registers.  Bound by the latency of a tile's chain (shared memory, maximum, powers): 8 sequences of a token over
// 4096 keys, 8 KV heads of 128, f32 (268 MB) 76 us, 3.5 TB/s; a prompt of 1024 over 2048 keys 730 us, 35 TFLOP/s of the FMA pipe's 72.  Sixteen
// threads share a row (in the scores each has 2 of the 32 keys, in the weighted sum 4 of every 64 columns), RT / 16 rows each, so that the softmax needs shuffles of half a warp only.  Work is dealt out evenly over one wave (paged_schedule.h); an item
// that several CTAs share leaves parts in the workspace, which lux_paged_chunk_merge puts together.
#include "paged_chunk.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace luxcuda {

namespace {

constexpr int CK = 32, CT = 256;           // keys per tile, threads

template <int RT, int DP> constexpr size_t chunk_smem() { return (size_t)(RT + 4 * CK) * (DP + 4) * 4 + (size_t)RT * (CK + 4) * 4; }

// CTAs per SM: what the launch bound asks the compiler for and the grid is made of.  (A third for heads of up to 64 would need 85 registers a
// thread where these forms take 119 to 128; a grid of three with room for two is a wave and a half of even shares.  Heads of 64, f32, 8 KV heads:
// 8 single tokens over 4096 keys 53.5 us, with a grid of three 69.3; 8 times five over 2000 47.3, 64.4; 1024 over 2048 418, 444.)
constexpr uint32_t chunk_ctas(uint32_t dp) { return dp > 128 ? 1 : 2; }
template <int RT, int DP> constexpr bool chunk_fits() {    // beside about 1 KB of its own, and 1 KB of the system's, per CTA
    return chunk_ctas(DP) * (chunk_smem<RT, DP>() + 2048) <= 228 * 1024;
}

template <typename T, int RT, int DP, bool VEC>
__global__ void __launch_bounds__(CT, chunk_ctas(DP)) lux_paged_chunk_f32(const ChunkParams p) {
    constexpr int R = RT / 16, P = DP + 4, C = DP / 64, J = CK / 16;
    extern __shared__ __align__(16) float smem[];
    float* const qs = smem;                // [RT][P]
    float* const ring = qs + RT * P;       // two tiles of K [CK][P] and V [CK][P]
    float* const ps = ring + 4 * CK * P;   // [RT][CK + 4]
    __shared__ int64_t rows_at[2][CK];     // where the tile's keys lie, in elements; -1: nowhere
    __shared__ uint64_t scratch[2 * CT / 32];
    __shared__ ChunkPlace found[2];
    const uint32_t tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    pdl_launch_dependents();
    pdl_wait();
    chunk_share<CT>(p, scratch, found, blockIdx.x);
    if (tid == 0) {
        p.places[blockIdx.x] = found[0];
        if (blockIdx.x + 1 == p.grid) p.places[p.grid] = ChunkPlace{p.seqs, 0, 0, 0};
    }
    const T* const q = reinterpret_cast<const T*>(p.q);
    const T* const k = reinterpret_cast<const T*>(p.k);
    const T* const v = reinterpret_cast<const T*>(p.v);
    constexpr uint32_t VE = VEC ? 16 / sizeof(T) : 1;
    const uint32_t per_row = p.dim / VE;   // (VEC: rows are whole vectors)

    // columns past the head's are zero throughout
    for (uint32_t i = tid; i < (RT + 4 * CK) * P; i += CT) smem[i] = 0.0f;
    auto fill = [&](float* dst, const T* src, uint32_t d) {
        if constexpr (VEC) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + d);
            alignas(16) T t[VE];
            *reinterpret_cast<uint4*>(t) = w;
#pragma unroll
            for (uint32_t i = 0; i < VE; i += 4)
                *reinterpret_cast<float4*>(dst + d + i) = make_float4(to_f32(t[i]), to_f32(t[i + 1]), to_f32(t[i + 2]), to_f32(t[i + 3]));
        } else {
            dst[d] = to_f32(src[d]);
        }
    };

    ChunkWalk walk;
    walk.begin(found[0], found[1]);
#pragma unroll 1
    for (; walk.settle(p); walk.next()) {
        const ChunkItem item = chunk_item(p, walk.at, walk.seq);
        const uint32_t rows = item.heads * item.tokens;
        uint32_t sees[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t r = ty * R + i;
            sees[i] = r < rows ? token_sees(p, walk.seq, item.token0 + r / item.heads) : 0u;
        }
        const bool busy = (ty & ~1u) * R < rows;       // this warp has rows
        const uint32_t all_see = token_sees(p, walk.seq, item.token0);       // what every row sees
        // a thread per key looks up where it lies: the table's entry is read a tile before its place is worked out
        int32_t entry = 0;
        auto read_entry = [&](uint32_t t) {
            const uint32_t key = t * CK + tid;
            if (tid < CK && key < walk.seq.keys) entry = load_i32(p.tables + (size_t)walk.at.seq * p.width + key / p.block_size);
        };
        auto look_up = [&](uint32_t t) {
            if (tid < CK) {
                const uint32_t key = t * CK + tid;
                int64_t at = -1;
                if (key < walk.seq.keys) {
                    if ((uint32_t)entry < p.num_blocks) at = (((int64_t)entry * p.kv_heads + item.kv_head) * p.block_size + key % p.block_size) * p.dim;
                    else report_status(p.status, STATUS_CACHE_BLOCK);
                }
                rows_at[t & 1][tid] = at;
            }
            read_entry(t + 1);
        };
        read_entry(walk.k0);
        __syncthreads();                   // the item before has been read
        for (uint32_t i = tid; i < RT * per_row; i += CT) {
            const uint32_t r = i / per_row, d = (i - r * per_row) * VE;
            if (r < rows) {
                const uint32_t token = walk.seq.first + item.token0 + r / item.heads, head = item.head0 + r % item.heads;
                fill(qs + r * P, q + ((size_t)token * p.heads + head) * p.dim, d);
            }
        }
        if (walk.k0 < walk.k1) look_up(walk.k0);
        if (walk.k0 + 1 < walk.k1) look_up(walk.k0 + 1);
        // a tile's K and V into their half of the ring: f32 by asynchronous copies, one tile ahead of its use; else widened on the way
        auto bring = [&](uint32_t t) {
            float* const kv = ring + (t & 1) * (2 * CK * P);
            constexpr uint32_t PER = DP / VE;      // vectors of a padded row
#pragma unroll 4
            for (uint32_t i = tid; i < CK * PER; i += CT) {
                const uint32_t key = i / PER, d = (i % PER) * VE;
                const int64_t at = d < p.dim ? rows_at[t & 1][key] : -1;
                if (at < 0) continue;
                if constexpr (VEC && sizeof(T) == 4) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(kv + key * P + d)), "l"(k + at + d) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(kv + (CK + key) * P + d)), "l"(v + at + d) : "memory");
                } else {
                    fill(kv + key * P, k + at, d);
                    fill(kv + (CK + key) * P, v + at, d);
                }
            }
        };
        __syncthreads();
        if (walk.k0 < walk.k1) bring(walk.k0);
        uint64_t o[R][2 * C];              // pairs of columns
        float top[R], sum[R];
#pragma unroll
        for (int i = 0; i < R; i++) {
            top[i] = -INFINITY;
            sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * C; j++) o[i][j] = 0ull;
        }
        for (uint32_t t = walk.k0; t < walk.k1; t++) {
            if constexpr (VEC && sizeof(T) == 4) asm volatile("cp.async.wait_all;" ::: "memory");
            __syncthreads();               // the tile is there, and the one before has been read
            if (t + 1 < walk.k1) bring(t + 1);
            if (t + 2 < walk.k1) look_up(t + 2);
            if (!busy) continue;
            const float* const ks = ring + (t & 1) * (2 * CK * P);
            const float* const vs = ks + CK * P;
            float s[R][J];
            {
                uint64_t s2[R][J];             // sums over even and odd columns
#pragma unroll
                for (int i = 0; i < R; i++)
#pragma unroll
                    for (int j = 0; j < J; j++) s2[i][j] = 0ull;
#pragma unroll 8
                for (int d = 0; d < DP; d += 4) {
                    ulonglong2 a[R], b[J];
#pragma unroll
                    for (int i = 0; i < R; i++) a[i] = *reinterpret_cast<const ulonglong2*>(qs + (ty * R + i) * P + d);
#pragma unroll
                    for (int j = 0; j < J; j++) b[j] = *reinterpret_cast<const ulonglong2*>(ks + (tx + 16 * j) * P + d);
#pragma unroll
                    for (int i = 0; i < R; i++)
#pragma unroll
                        for (int j = 0; j < J; j++) s2[i][j] = fma2(a[i].x, b[j].x, fma2(a[i].y, b[j].y, s2[i][j]));
                }
#pragma unroll
                for (int i = 0; i < R; i++)
#pragma unroll
                    for (int j = 0; j < J; j++) {
                        float even, odd;
                        unpair(s2[i][j], even, odd);
                        s[i][j] = even + odd;
                    }
            }
            const bool masked = all_see < (t + 1) * CK;
#pragma unroll
            for (int i = 0; i < R; i++) {
                float m = -INFINITY;
#pragma unroll
                for (int j = 0; j < J; j++) {
                    s[i][j] *= p.qscale;
                    if (masked && t * CK + tx + 16 * j >= sees[i]) s[i][j] = -INFINITY;
                    m = fmaxf(m, s[i][j]);
                }
#pragma unroll
                for (int d = 8; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
                m = fmaxf(m, top[i]);
                // (a row that has seen no key yet: nothing to scale, and no difference of infinities)
                const float f = m == -INFINITY ? 1.0f : chunk_ex2(top[i] - m), ref = m == -INFINITY ? 0.0f : m;
                top[i] = m;
                float part = 0.0f;
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const float w = chunk_ex2(s[i][j] - ref);
                    ps[(ty * R + i) * (CK + 4) + tx + 16 * j] = w;
                    part += w;
                }
                sum[i] = fmaf(sum[i], f, part);
#pragma unroll
                for (int j = 0; j < 2 * C; j++) o[i][j] = fma2(o[i][j], pair(f, f), 0ull);
            }
            __syncwarp();                  // a row's weights are written and read by the same half warp
            if (!masked) {
#pragma unroll 4
                for (int key = 0; key < CK; key += 4) {
                    float4 w[R];
#pragma unroll
                    for (int i = 0; i < R; i++) w[i] = *reinterpret_cast<const float4*>(ps + (ty * R + i) * (CK + 4) + key);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++)
#pragma unroll
                        for (int c = 0; c < C; c++) {
                            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(vs + (key + kk) * P + 64 * c + 4 * tx);
#pragma unroll
                            for (int i = 0; i < R; i++) {
                                const float f = kk == 0 ? w[i].x : kk == 1 ? w[i].y : kk == 2 ? w[i].z : w[i].w;
                                o[i][2 * c] = fma2(pair(f, f), x.x, o[i][2 * c]);
                                o[i][2 * c + 1] = fma2(pair(f, f), x.y, o[i][2 * c + 1]);
                            }
                        }
                }
            } else {
                // keys that a row does not see are left out, not weighted with zero: they may hold anything
                const uint32_t keys = min((uint32_t)CK, walk.seq.keys - t * CK);
                for (uint32_t key = 0; key < keys; key++) {
#pragma unroll
                    for (int i = 0; i < R; i++) {
                        if (t * CK + key >= sees[i]) continue;
                        const float f = ps[(ty * R + i) * (CK + 4) + key];
#pragma unroll
                        for (int c = 0; c < C; c++) {
                            const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(vs + key * P + 64 * c + 4 * tx);
                            o[i][2 * c] = fma2(pair(f, f), x.x, o[i][2 * c]);
                            o[i][2 * c + 1] = fma2(pair(f, f), x.y, o[i][2 * c + 1]);
                        }
                    }
                }
            }
        }
        const bool whole = walk.whole();
        const size_t slot = 2 * (size_t)blockIdx.x + (walk.k0 ? 0 : 1);
#pragma unroll
        for (int i = 0; i < R; i++) {
            const uint32_t r = ty * R + i;
#pragma unroll
            for (int d = 8; d; d >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
            if (r >= rows) continue;
            if (whole) {
                const size_t row = (size_t)(walk.seq.first + item.token0 + r / item.heads) * p.heads + item.head0 + r % item.heads;
                T* dst = reinterpret_cast<T*>(p.out) + row * p.dim;
#pragma unroll
                for (int j = 0; j < 2 * C; j++) {
                    const uint32_t d = 64 * (j / 2) + 4 * tx + 2 * (j & 1);
                    float x, y;
                    unpair(o[i][j], x, y);
                    if (d < p.dim) dst[d] = from_f32<T>(sum[i] == 0.0f ? 0.0f : x / sum[i]);
                    if (d + 1 < p.dim) dst[d + 1] = from_f32<T>(sum[i] == 0.0f ? 0.0f : y / sum[i]);
                }
                if (p.lse && tx == 0) p.lse[row] = sum[i] == 0.0f ? CHUNK_NO_KEYS : fmaf(top[i], CHUNK_LN2, logf(sum[i]));
            } else {
                float* dst = p.parts + (slot * p.part_rows + r) * p.part_pitch;
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const uint32_t d = 64 * c + 4 * tx;
                    if (d < p.part_pitch) *reinterpret_cast<ulonglong2*>(dst + d) = make_ulonglong2(o[i][2 * c], o[i][2 * c + 1]);
                }
                if (tx == 0) p.stats[slot * p.part_rows + r] = make_float2(top[i], sum[i]);
            }
        }
    }
}

// The grid of the FMA kernel's largest form, and its rows, which bound the workspace.
constexpr uint32_t MAX_CTAS_PER_SM = 2, MAX_ROWS = 64;

struct Sizes {
    size_t stats_at, parts_at, total;
    uint32_t part_rows, part_pitch;
};
// parts of at most `rows` rows for `ctas` CTAs; no item has more rows than the call's tokens have heads of a group
Sizes workspace_sizes(uint32_t ctas, uint32_t rows, uint64_t tokens, uint32_t group, uint32_t dim) {
    Sizes s{};
    s.part_rows = (uint32_t)std::min<uint64_t>(rows, std::max<uint64_t>(tokens * group, 1));
    s.part_pitch = (dim + 3) / 4 * 4;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    s.stats_at = up((size_t)(ctas + 1) * sizeof(ChunkPlace));
    s.parts_at = s.stats_at + up((size_t)2 * ctas * s.part_rows * sizeof(float2));
    s.total = s.parts_at + (size_t)2 * ctas * s.part_rows * s.part_pitch * 4;
    return s;
}

template <typename T, int RT, int DP> LuxBackendError launch_f32_form(Context* ctx, ChunkParams& p, bool vec) {
    static_assert(chunk_fits<RT, DP>(), "shared memory of the CTAs of an SM");
    auto kfn = vec ? lux_paged_chunk_f32<T, RT, DP, true> : lux_paged_chunk_f32<T, RT, DP, false>;
    static std::atomic<bool> configured[2][64];
    std::atomic<bool>& done = configured[vec][ctx->device & 63];
    if (!done.load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute((const void*)kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)chunk_smem<RT, DP>());
        if (e != cudaSuccess) return map_cuda(e, "paged_chunk_attention");
        done.store(true, std::memory_order_relaxed);
    }
    p.grid = (uint32_t)ctx->sm_count * chunk_ctas(DP);         // one wave
    const cudaError_t e = launch_pdl(g_tune.pdl != 2, kfn, dim3(p.grid), dim3(CT), chunk_smem<RT, DP>(), ctx->stream, 1, p);
    if (e != cudaSuccess) return map_cuda(e, "paged_chunk_attention");
    count_launch("lux_paged_chunk_f32");
    return LUX_BACKEND_OK;
}
template <typename T, int RT> LuxBackendError launch_f32_dim(Context* ctx, ChunkParams& p, bool vec) {
    if (p.dim <= 64) return launch_f32_form<T, RT, 64>(ctx, p, vec);
    if (p.dim <= 128) return launch_f32_form<T, RT, 128>(ctx, p, vec);
    return launch_f32_form<T, RT, 256>(ctx, p, vec);
}
template <typename T> LuxBackendError launch_f32(Context* ctx, ChunkParams& p, bool vec, uint32_t rt) {
    return rt == 16 ? launch_f32_dim<T, 16>(ctx, p, vec) : rt == 32 ? launch_f32_dim<T, 32>(ctx, p, vec) : launch_f32_dim<T, 64>(ctx, p, vec);
}

}  // namespace

const void* kernel_addr_paged_chunk_f32() { return (const void*)lux_paged_chunk_f32<float, 64, 128, true>; }
const void* kernel_addr_paged_chunk_merge() { return (const void*)lux_paged_chunk_merge<float>; }

}  // namespace luxcuda

using namespace luxcuda;

extern "C" size_t lux_cuda_paged_chunk_workspace(LuxBackendContext* context, uint32_t num_seqs, uint32_t num_tokens, uint32_t num_heads,
                                                 uint32_t num_kv_heads, uint32_t head_dim, uint32_t dtype) {
    const Context* ctx = as_ctx(context);
    (void)num_seqs;
    if (!ctx || !dtype_bytes(dtype) || num_kv_heads == 0 || num_heads == 0 || num_heads % num_kv_heads || head_dim == 0 || head_dim > 256) return 0;
    const uint32_t group = num_heads / num_kv_heads;
    size_t most = workspace_sizes((uint32_t)ctx->sm_count * MAX_CTAS_PER_SM, MAX_ROWS, num_tokens, group, head_dim).total;
    if (dtype != LUX_QDTYPE_F32) most = std::max(most, workspace_sizes((uint32_t)ctx->sm_count, chunk_tc_rows(group), num_tokens, group, head_dim).total);
    return most;
}

extern "C" LuxBackendError lux_cuda_paged_chunk_attention(LuxBackendContext* context, LuxBackendBuffer* q, LuxBackendBuffer* k_cache,
                                                          LuxBackendBuffer* v_cache, LuxBackendBuffer* block_tables,
                                                          LuxBackendBuffer* q_starts, LuxBackendBuffer* context_lens, LuxBackendBuffer* out,
                                                          LuxBackendBuffer* lse, LuxBackendBuffer* workspace, uint32_t num_seqs,
                                                          uint32_t num_tokens, uint32_t num_heads, uint32_t num_kv_heads, uint32_t head_dim,
                                                          uint32_t block_size, uint32_t max_blocks_per_seq, float scale, uint32_t dtype,
                                                          uint32_t flags) {
    Context* ctx = as_ctx(context);
    Buffer *bq = as_buf(q), *bk = as_buf(k_cache), *bv = as_buf(v_cache), *bt = as_buf(block_tables), *bs = as_buf(q_starts),
           *bc = as_buf(context_lens), *bo = as_buf(out), *bl = as_buf(lse), *bw = as_buf(workspace);
    const size_t e = dtype_bytes(dtype);
    if (!ctx || !e || head_dim == 0 || num_heads == 0 || num_kv_heads == 0 || num_heads % num_kv_heads || block_size == 0 || max_blocks_per_seq == 0 ||
        num_seqs > 0x7fffffffu || num_tokens > 0x7fffffffu)
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (head_dim > 256) return LUX_BACKEND_ERROR_NOT_SUPPORTED;
    const size_t qn = mul({num_tokens, num_heads, head_dim}), block_elems = mul({num_kv_heads, block_size, head_dim});
    if (!holds(bq, qn, e) || !holds(bo, qn, e) || !holds(bk, block_elems, e) || !holds(bv, block_elems, e) ||
        !holds(bt, mul({num_seqs, max_blocks_per_seq})) || !holds(bs, (size_t)num_seqs + 1) || !holds(bc, num_seqs) ||
        (bl && !holds(bl, mul({num_tokens, num_heads}))))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if ((uint64_t)max_blocks_per_seq * block_size > 0x7fffffffu || mul({num_tokens, num_heads}) > 0x7fffffffu) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!bw || !bw->ptr || ((uintptr_t)bw->ptr & 15u) ||
        bw->size < lux_cuda_paged_chunk_workspace(context, num_seqs, num_tokens, num_heads, num_kv_heads, head_dim, dtype))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (num_seqs == 0 || num_tokens == 0) return LUX_BACKEND_OK;
    ChunkParams p{};
    p.q = bq->ptr;
    p.k = bk->ptr;
    p.v = bv->ptr;
    p.out = bo->ptr;
    p.lse = bl ? (float*)bl->ptr : nullptr;
    p.tables = (const int32_t*)bt->ptr;
    p.q_starts = (const int32_t*)bs->ptr;
    p.context = (const int32_t*)bc->ptr;
    p.status = ctx->d_status;
    p.seqs = num_seqs;
    p.tokens = num_tokens;
    p.heads = num_heads;
    p.kv_heads = num_kv_heads;
    p.group = num_heads / num_kv_heads;
    p.dim = head_dim;
    p.block_size = block_size;
    p.width = max_blocks_per_seq;
    p.num_blocks = (uint32_t)std::min<size_t>(std::min(bk->size, bv->size) / e / block_elems, 0x7fffffffu);
    p.qscale = scale * CHUNK_LOG2E;
    p.shape.causal = (flags & LUX_ATTN_FLAG_CAUSAL) ? 1u : 0u;
    cudaSetDevice(ctx->device);

    auto place_parts = [&](const Sizes& w) {
        // at most tokens / tile_tokens + sequences tiles, each with all keys of a table's row
        const uint64_t tiles = num_tokens / p.shape.tile_tokens + (uint64_t)num_seqs, keys = (uint64_t)max_blocks_per_seq * block_size + p.shape.fixed;
        const uint64_t heaviest = p.weight + (uint64_t)p.shape.tile_tokens * p.item_heads / p.weight_rows;
        p.narrow = mul({p.shape.heads, tiles, keys, heaviest}) < (1ull << 31);
        p.part_rows = w.part_rows;
        p.part_pitch = w.part_pitch;
        p.places = (ChunkPlace*)bw->ptr;
        p.stats = (float2*)((unsigned char*)bw->ptr + w.stats_at);
        p.parts = (float*)((unsigned char*)bw->ptr + w.parts_at);
    };
    LuxBackendError le = LUX_BACKEND_ERROR_NOT_SUPPORTED;
    if (chunk_tc_takes(p, dtype)) {
        p.item_heads = p.group;
        p.splits = 1;
        p.shape.heads = num_kv_heads;
        p.shape.tile_tokens = 2 * (128 / p.group);
        p.shape.tile_keys = 64;
        p.shape.fixed = 256;
        // Two tiles of rows take longer over a tile of keys than one, which both softmax groups share (and which HBM bounds): 3 to 2.  A prompt
        // of 1000 among 31 single tokens over up to 4096 keys: 126 us, 1 to 1 140, 2 to 1 140; of 4000 tokens 241, 258, 287.
        p.weight = 2;
        p.weight_rows = 129;
        p.shape.snap = 3;
        p.grid = (uint32_t)ctx->sm_count;
        place_parts(workspace_sizes(p.grid, chunk_tc_rows(p.group), num_tokens, p.group, head_dim));
        le = launch_chunk_tc(ctx, p, dtype);
    }
    if (le == LUX_BACKEND_ERROR_NOT_SUPPORTED) {
        // Tiles of few rows where sequences have few on average; a tile that is too small costs more (all keys once more) than one that is too
        // large (idle warps).  8 sequences over 2000 keys, 8 KV heads of 128, f32, by rows: 4 rows 45 us in tiles of 16, 46 of 32, 62 of 64;
        // 8 rows 59, 54, 62; 16 rows 90, 65, 81; 20 rows 166, 75, 83; 32 rows 166, 104, 88.
        const uint64_t mean_rows = ((uint64_t)num_tokens * p.group + num_seqs - 1) / num_seqs;
        const uint32_t rt = mean_rows <= 6 ? 16 : mean_rows <= 24 ? 32 : 64;
        p.item_heads = std::min(p.group, rt);
        p.splits = (p.group + p.item_heads - 1) / p.item_heads;
        p.shape.heads = num_kv_heads * p.splits;
        p.shape.tile_tokens = rt / p.item_heads;
        p.shape.tile_keys = CK;
        p.shape.fixed = 2 * CK;
        // rows that are there cost time, the rest of the tile does too: 32 sequences of 1 to 5 tokens over up to 2000 keys 116 us, by keys alone
        // 131, with a third of the tile's rows 130
        p.weight = rt;
        p.weight_rows = 1;
        p.shape.snap = 1;
        const uint32_t dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
        place_parts(workspace_sizes((uint32_t)ctx->sm_count * chunk_ctas(dp), rt, num_tokens, p.group, head_dim));
        const bool vec = head_dim * e % 16 == 0 && (((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) & 15u) == 0;
        le = dtype == LUX_QDTYPE_F32 ? launch_f32<float>(ctx, p, vec, rt)
           : dtype == LUX_QDTYPE_F16 ? launch_f32<__half>(ctx, p, vec, rt) : launch_f32<__nv_bfloat16>(ctx, p, vec, rt);
    }
    if (le != LUX_BACKEND_OK) return le;
    if (p.grid > 1) {
        auto merge = dtype == LUX_QDTYPE_F32 ? lux_paged_chunk_merge<float> : dtype == LUX_QDTYPE_F16 ? lux_paged_chunk_merge<__half> : lux_paged_chunk_merge<__nv_bfloat16>;
        const cudaError_t err = launch_pdl(g_tune.pdl != 2, merge, dim3(p.grid - 1, std::max(1u, std::min((p.part_rows + 3) / 4, 16u))), dim3(128), 0, ctx->stream, 1, p);
        if (err != cudaSuccess) return map_cuda(err, "paged_chunk_attention");
        count_launch("lux_paged_chunk_merge");
    }
    return finish_op(ctx, (flags & LUX_QMATMUL_FLAG_NO_SYNC) != 0, "paged_chunk_attention");
}
