// paged_ops.cu -- what a serving step does around attention over a paged KV cache: blocks and slots for new tokens,
// the blocks given back, and the norm / rotation / append of queries, keys and values (lux/gpu/paged_ext.h).
#include "paged.cuh"
#include "tc_ptx.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

namespace cg = cooperative_groups;

namespace luxcuda {

namespace {

constexpr int PLAN_THREADS = 1024, PLAN_CLUSTER = 8;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;

// ---- blocks and slots --------------------------------------------------------------------------------
//
// Both kernels are one cluster: what they compute is a handful of sums over the sequences, so a call is bound by latency
// (launch, three or four trips to L2, two cluster barriers), and one launch without a second kernel or a grid-wide
// barrier is the shortest form.  Reserving takes the table entries that the new tokens reach as one list, sequence after sequence; how long it is
// follows from the lengths alone, so every CTA sums the lengths by itself, counts the empty entries of its share of
// the list, learns the other CTAs' counts through distributed shared memory and then knows which entry gets which free
// block.  No atomics: the outcome follows from the input alone.  64 sequences of a token each: 12.9 us for both calls, 300 sequences of
// 400 tokens 19.9 us.

struct ReserveParams {
    const int32_t* cached;
    const int32_t* fresh;
    int32_t* table;
    const int32_t* free_blocks;
    int32_t* free_count;
    int32_t* q_starts;
    int32_t* context;
    int32_t* positions;
    int32_t* slots;
    uint32_t* status;
    uint32_t seqs, width, block_size, max_tokens;
    uint64_t capacity;
};

// exclusive sum over the CTA's threads of two numbers at once, and the totals; `scratch` has 2 * (PLAN_WARPS + 1) places
__device__ __forceinline__ void block_sums(uint64_t& a, uint64_t& b, uint64_t& total_a, uint64_t& total_b, uint64_t* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint64_t x = a, y = b;
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
        if (lane >= d) x += u, y += v;
    }
    __syncthreads();                                       // the scratch of an earlier call has been read
    if (lane == 31) scratch[2 * warp] = x, scratch[2 * warp + 1] = y;
    __syncthreads();
    if (warp == 0) {
        uint64_t u = lane < warps ? scratch[2 * lane] : 0, v = lane < warps ? scratch[2 * lane + 1] : 0;
        for (int d = 1; d < 32; d <<= 1) {
            const uint64_t s = __shfl_up_sync(0xffffffffu, u, d), t = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) u += s, v += t;
        }
        if (lane < warps) scratch[2 * lane] = u, scratch[2 * lane + 1] = v;
    }
    __syncthreads();
    const uint64_t before_a = warp ? scratch[2 * warp - 2] : 0, before_b = warp ? scratch[2 * warp - 1] : 0;
    total_a = scratch[2 * warps - 2];
    total_b = scratch[2 * warps - 1];
    a = before_a + x - a;
    b = before_b + y - b;
}

// the last i of 0 .. n - 1 with v[i] <= x (v rises, v[0] = 0)
__device__ __forceinline__ uint32_t last_at_most(const uint32_t* v, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) lux_paged_reserve(const ReserveParams p) {
    extern __shared__ uint32_t plan_smem[];
    __shared__ uint64_t scratch[2 * (PLAN_WARPS + 1)];
    __shared__ uint32_t counts[PLAN_CLUSTER];              // empty entries in each CTA's share of the list
    uint32_t* starts = plan_smem;                          // [seqs]: first new token
    uint32_t* lists = starts + p.seqs;                     // [seqs]: first entry in the list
    int32_t* cached = reinterpret_cast<int32_t*>(lists + p.seqs);
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks(), tid = threadIdx.x;
    pdl_launch_dependents();
    auto started = cluster.barrier_arrive();
    pdl_wait();

    const int32_t count = load_i32(p.free_count);
    bool bad = count < 0 || (uint64_t)count > p.capacity;
    // the sums over the lengths, in runs of one sequence per thread
    uint64_t tokens = 0, entries = 0;
    for (uint32_t s0 = 0; s0 < p.seqs; s0 += PLAN_THREADS) {
        const uint32_t s = s0 + tid;
        int64_t c = 0, t = 0;
        if (s < p.seqs) c = load_i32(p.cached + s), t = load_i32(p.fresh + s);
        const bool wrong = c < 0 || t < 0 || (uint64_t)(c + t) > (uint64_t)p.width * p.block_size;
        bad |= wrong;
        uint64_t a = wrong ? 0 : (uint64_t)t, sum_a;
        uint64_t b = wrong || t == 0 ? 0 : (uint64_t)((uint32_t)(c + t - 1) / p.block_size - (uint32_t)c / p.block_size + 1), sum_b;
        block_sums(a, b, sum_a, sum_b, scratch);
        if (s < p.seqs) {                                  // (cut to 32 bits only where the call is refused below)
            starts[s] = (uint32_t)(tokens + a);
            lists[s] = (uint32_t)(entries + b);
            cached[s] = (int32_t)c;
        }
        tokens += sum_a;
        entries += sum_b;
    }
    bad = __syncthreads_or(bad) || tokens > p.max_tokens || entries > 0xffffffffu;

    // this CTA's share of the list, in order; an entry is one thread's
    const uint32_t lo = bad ? 0 : (uint32_t)(entries * rank / ctas), hi = bad ? 0 : (uint32_t)(entries * (rank + 1) / ctas);
    auto place = [&](uint32_t e) {
        const uint32_t s = last_at_most(lists, p.seqs, e);
        return p.table + (size_t)s * p.width + (uint32_t)cached[s] / p.block_size + (e - lists[s]);
    };
    uint32_t empty = 0;
    for (uint32_t e0 = lo; e0 < hi; e0 += PLAN_THREADS) empty += __syncthreads_count(e0 + tid < hi && load_i32(place(e0 + tid)) < 0);
    cluster.barrier_wait(std::move(started));              // the others run, so their shared memory may be written
    if (tid < ctas) *cluster.map_shared_rank(&counts[rank], tid) = empty;
    cluster.sync();
    uint32_t before = 0;
    uint64_t all = 0;
    for (uint32_t r = 0; r < ctas; r++) {
        if (r < rank) before += counts[r];
        all += counts[r];
    }
    bad |= all > (uint64_t)count;
    if (bad) {
        // nothing is handed out; the lengths and starts say so
        for (uint64_t i = rank * PLAN_THREADS + tid; i < p.max_tokens; i += ctas * PLAN_THREADS) p.positions[i] = 0, p.slots[i] = -1;
        if (rank == 0) {
            for (uint32_t s = tid; s <= p.seqs; s += PLAN_THREADS) p.q_starts[s] = 0;
            for (uint32_t s = tid; s < p.seqs; s += PLAN_THREADS) p.context[s] = cached[s];
            if (tid == 0) report_status(p.status, STATUS_FREE_BLOCKS);
        }
        cluster.sync();                                    // no CTA leaves while its counts may still be written or read
        return;
    }
    uint64_t taken = before;
    for (uint32_t e0 = lo; e0 < hi; e0 += PLAN_THREADS) {
        const uint32_t e = e0 + tid;
        int32_t* const at = e < hi ? place(e) : nullptr;
        uint64_t mine = at && load_i32(at) < 0, none = 0, sum, zero;
        const bool take = mine;
        block_sums(mine, none, sum, zero, scratch);
        if (take) store_i32(at, load_i32(p.free_blocks + (count - 1 - (int64_t)(taken + mine))));
        taken += sum;
    }
    if (rank == 0) {
        for (uint32_t s = tid; s < p.seqs; s += PLAN_THREADS) {
            p.q_starts[s] = (int32_t)starts[s];
            p.context[s] = (int32_t)((s + 1 < p.seqs ? starts[s + 1] : (uint32_t)tokens) - starts[s]) + cached[s];
        }
        if (tid == 0) {
            p.q_starts[p.seqs] = (int32_t)tokens;
            if (all) *p.free_count = count - (int32_t)all;
        }
    }
    __threadfence();
    cluster.sync();                                        // the tables are complete
    for (uint64_t i = rank * PLAN_THREADS + tid; i < p.max_tokens; i += ctas * PLAN_THREADS) {
        int32_t pos = 0, slot = -1;
        if (i < tokens) {
            const uint32_t s = last_at_most(starts, p.seqs, (uint32_t)i);
            pos = cached[s] + (int32_t)((uint32_t)i - starts[s]);
            const uint32_t b = (uint32_t)pos / p.block_size;
            // (a block number that no cache of 31-bit slots has must not come out as a slot of another one)
            const uint64_t at = (uint64_t)(uint32_t)load_i32(p.table + (size_t)s * p.width + b) * p.block_size + ((uint32_t)pos - b * p.block_size);
            if (at <= 0x7fffffffu) slot = (int32_t)at;
            else report_status(p.status, STATUS_CACHE_BLOCK);
        }
        p.positions[i] = pos;
        p.slots[i] = slot;
    }
}

struct ReleaseParams {
    const int32_t* keep;
    int32_t* table;
    int32_t* free_blocks;
    int32_t* free_count;
    uint32_t* status;
    uint32_t seqs, width, block_size;
    uint64_t capacity;
};

// A warp per sequence counts its entries from the first released one to the first empty one, 128 at a time; the counts are
// summed within the CTA, which owns a contiguous range of the sequences, and over the cluster.
__global__ void __launch_bounds__(PLAN_THREADS) lux_paged_release(const ReleaseParams p) {
    extern __shared__ uint32_t plan_smem[];                // [sequences of this CTA]: how many go
    __shared__ uint64_t scratch[2 * (PLAN_WARPS + 1)];
    __shared__ uint64_t counts[PLAN_CLUSTER];
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    auto started = cluster.barrier_arrive();
    pdl_wait();
    const int32_t count = load_i32(p.free_count);
    const uint32_t lo = (uint32_t)((uint64_t)p.seqs * rank / ctas), n = (uint32_t)((uint64_t)p.seqs * (rank + 1) / ctas) - lo;
    auto first_of = [&](uint32_t s) -> uint32_t {                      // the first entry that goes
        const int32_t keep = load_i32(p.keep + s);
        if (keep < 0) return p.width;
        const uint32_t held = ((uint32_t)keep + p.block_size - 1) / p.block_size;     // (both are below 2^31)
        return held < p.width ? held : p.width;
    };
    for (uint32_t i = warp; i < n; i += PLAN_WARPS) {
        const int32_t* row = p.table + (size_t)(lo + i) * p.width;
        const uint32_t first = first_of(lo + i);
        uint32_t held = 0;
        for (uint32_t b = first; b < p.width; b += 128) {
            uint32_t run = 0;
            bool open = true;                              // no empty entry so far
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t at = b + 32 * j + lane;
                const uint32_t full = __ballot_sync(0xffffffffu, at < p.width && load_i32(row + at) >= 0);
                if (open) run += full == 0xffffffffu ? 32 : __ffs(~full) - 1;
                open = open && full == 0xffffffffu;
            }
            held += run;
            if (!open) break;
        }
        if (lane == 0) plan_smem[i] = held;
    }
    __syncthreads();
    // where each sequence's blocks begin among those of this CTA
    uint64_t sum = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += PLAN_THREADS) {
        const uint32_t i = i0 + tid;
        uint64_t a = i < n ? plan_smem[i] : 0, none = 0, total, zero;
        block_sums(a, none, total, zero, scratch);
        if (i < n) plan_smem[i] = (uint32_t)(sum + a);
        sum += total;
    }
    cluster.barrier_wait(std::move(started));              // the others run, so their shared memory may be written
    if (tid < ctas) *cluster.map_shared_rank(&counts[rank], tid) = sum;
    cluster.sync();
    uint64_t before = 0, all = 0;
    for (uint32_t r = 0; r < ctas; r++) {
        if (r < rank) before += counts[r];
        all += counts[r];
    }
    const bool bad = count < 0 || (uint64_t)count > p.capacity || all > p.capacity - (uint64_t)count || all > 0x7fffffffu - (uint64_t)count;
    if (bad) {
        if (rank == 0 && tid == 0) report_status(p.status, STATUS_FREE_BLOCKS);
    } else {
        for (uint32_t i = warp; i < n; i += PLAN_WARPS) {
            const uint64_t at = before + plan_smem[i];
            const uint32_t held = (uint32_t)((i + 1 < n ? plan_smem[i + 1] : sum) - plan_smem[i]);
            int32_t* row = p.table + (size_t)(lo + i) * p.width + first_of(lo + i);
            for (uint32_t j = lane; j < held; j += 32) {
                p.free_blocks[(uint64_t)count + all - 1 - (at + j)] = load_i32(row + j);
                row[j] = -1;
            }
        }
        if (rank == 0 && tid == 0 && all) *p.free_count = count + (int32_t)all;
    }
    cluster.sync();                                        // no CTA leaves while its counts may still be written
}

// ---- norm, rotation and append -----------------------------------------------------------------------

struct QkvParams {
    const void* qkv;
    const float* wq;
    const float* wk;
    const float* cos_cache;
    const float* sin_cache;
    const int32_t* positions;
    const int32_t* slots;
    void* q_out;
    void* k_cache;
    void* v_cache;
    uint32_t* status;
    uint64_t stride, num_slots, table_rows;
    uint32_t tokens, heads, kv_heads, dim, half, block_size;   // half: pairs per head
    uint32_t units, lanes;                                     // units of 2 V elements per head; threads per head
    uint32_t row_bytes, slots_ahead;                           // STAGED: of a token, rounded up to 128 in shared memory; tokens in the ring
    float eps, per_dim;                                        // 1 / dim
};

template <int BYTES> struct Bits;
template <> struct Bits<16> { using type = uint4; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<4> { using type = uint32_t; };
template <> struct Bits<2> { using type = uint16_t; };

template <typename T, int V> __device__ __forceinline__ void widen(const typename Bits<(int)sizeof(T) * V>::type& w, float (&x)[V]) {
    alignas(16) T t[V];
    *reinterpret_cast<typename Bits<(int)sizeof(T) * V>::type*>(t) = w;
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = to_f32(t[i]);
}
template <typename T, int V> __device__ __forceinline__ void load_vec(const T* src, float (&x)[V]) {
    widen<T, V>(*reinterpret_cast<const typename Bits<(int)sizeof(T) * V>::type*>(src), x);
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* dst, const float (&x)[V]) {
    using W = typename Bits<(int)sizeof(T) * V>::type;
    alignas(16) T t[V];
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = from_f32<T>(x[i]);
    *reinterpret_cast<W*>(dst) = *reinterpret_cast<const W*>(t);
}

template <int V> __device__ __forceinline__ void load_floats(const float* src, float (&x)[V]) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(x + i) = *reinterpret_cast<const float4*>(src + i);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = src[i];
    }
}

// A CTA takes one token after the other.  A head is cut into units of two vectors of V elements, which hold both elements of V pairs
// (HALVES: the vectors lie half a rotation apart; else they are neighbours), and `lanes` threads share a head, one unit each,
// a thread's unit being the same in every head that it takes: its cos and sin are read once a token, its weights are in shared memory.
// f32 is bound by HBM (8192 tokens x 48 heads of 128, 402 MB: 73 us, 5.5 TB/s).  STAGED: 16-bit rows come by bulk copies into a ring of tokens, so that
// the next tokens are under way while one is worked on (the same in bf16, 206 MB: 60 to 65 us without, R heads requested at once and 20 warps per
// SM, against 49 us, 4.2 TB/s).  That is bound by neither HBM nor issue slots (47 % of them): 20 warps of 96 registers per SM, a few of these spilled,
// wait for cos and sin (L2), the row (shared memory) and each other once a token.
constexpr int QKV_THREADS = 128, QKV_MAX_AHEAD = 4, QKV_SHARED = 32 * 2 * 8;   // 32 units of two vectors of at most eight
constexpr uint32_t QKV_MAX_PITCH = 50u << 10, QKV_OPEN = 40u << 10;            // the largest row of a ring; what dynamic shared memory may have as it is

template <typename T, int V, bool HALVES, int R, bool STAGED>
__global__ void __launch_bounds__(QKV_THREADS, 5) lux_paged_qkv(const QkvParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t lane = threadIdx.x & (p.lanes - 1), first_head = threadIdx.x / p.lanes, step = QKV_THREADS / p.lanes;
    // the two vectors of unit u; unturned: behind the rotated part
    auto place = [&](uint32_t u, uint32_t& a, uint32_t& b, bool& turned) {
        turned = u * V < p.half;
        a = HALVES && turned ? u * V : 2 * u * V;
        b = a + (HALVES && turned ? p.half : V);
    };
    const bool has = lane < p.units;       // (one unit per thread)
    uint32_t ua = 0, ub = 0;
    bool uturned = false;
    if (has) place(lane, ua, ub, uturned);
    __shared__ alignas(16) float weights[2][QKV_SHARED];   // of queries and keys, as far as heads of one unit per thread reach
    if (p.wq && p.units <= p.lanes) {
        for (uint32_t i = threadIdx.x; i < p.dim; i += QKV_THREADS) weights[0][i] = p.wq[i], weights[1][i] = p.wk[i];
        __syncthreads();
    }
    extern __shared__ __align__(128) unsigned char qkv_ring[];     // STAGED: slots_ahead rows
    __shared__ alignas(8) uint64_t qkv_full[QKV_MAX_AHEAD];
    const uint32_t pitch = (p.row_bytes + 127) / 128 * 128;
    uint32_t use = 0;                                      // tokens of this CTA so far
    auto request = [&](uint32_t t, uint32_t i) {           // by one thread
        const uint32_t bar = tcptx::smem_u32(&qkv_full[i]);
        tcptx::mbar_expect_tx(bar, p.row_bytes);
        tcptx::bulk_g2s(tcptx::smem_u32(qkv_ring) + i * pitch, reinterpret_cast<const T*>(p.qkv) + t * p.stride, p.row_bytes, bar);
    };
    if (STAGED) {
        if (threadIdx.x == 0) {
            for (uint32_t i = 0; i < p.slots_ahead; i++) tcptx::mbar_init(tcptx::smem_u32(&qkv_full[i]), 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            for (uint32_t i = 0; i < p.slots_ahead; i++)
                if (blockIdx.x + (uint64_t)i * gridDim.x < p.tokens) request(blockIdx.x + i * gridDim.x, i);
        }
        __syncthreads();
    }
    int32_t next_slot = blockIdx.x < p.tokens ? p.slots[blockIdx.x] : 0, next_pos = p.half && blockIdx.x < p.tokens ? p.positions[blockIdx.x] : 0;
    for (uint32_t t = blockIdx.x; t < p.tokens; t += gridDim.x, use++) {
        const uint32_t ring = STAGED ? use % p.slots_ahead : 0u;
        if (STAGED) {
            if (use) {                                     // the slot of the token before is free: all have read it
                __syncthreads();
                const uint64_t later = t + (uint64_t)(p.slots_ahead - 1) * gridDim.x;
                if (threadIdx.x == 0 && later < p.tokens) {
                    tcptx::fence_proxy_async_smem();
                    request((uint32_t)later, (use - 1) % p.slots_ahead);
                }
            }
            const uint32_t bar = tcptx::smem_u32(&qkv_full[ring]);
            bool there = false;
            for (uint32_t i = 0; !there && i < (1u << 20); i++) {
                uint32_t ok;
                asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                             : "=r"(ok) : "r"(bar), "r"((use / p.slots_ahead) & 1u) : "memory");
                there = ok;
            }
            if (__syncthreads_or(!there)) {                // a bounded wait gave up
                if (threadIdx.x == 0) report_status(p.status, STATUS_ATTENTION_WAIT);
                for (int i = 0; i < 64; i++) __nanosleep(1000);
                return;
            }
        }
        const int64_t slot = next_slot, pos = next_pos;
        if (t + gridDim.x < p.tokens) {
            next_slot = p.slots[t + gridDim.x];
            if (p.half) next_pos = p.positions[t + gridDim.x];
        }
        if (slot < 0) continue;                            // padding
        if ((uint64_t)slot >= p.num_slots) {
            if (threadIdx.x == 0) report_status(p.status, STATUS_CACHE_BLOCK);
            continue;
        }
        if (p.half && (pos < 0 || (uint64_t)pos >= p.table_rows)) {
            if (threadIdx.x == 0) report_status(p.status, STATUS_POSITION);
            continue;
        }
        const T* src = STAGED ? reinterpret_cast<const T*>(qkv_ring + ring * pitch) : reinterpret_cast<const T*>(p.qkv) + t * p.stride;
        const uint32_t block = (uint32_t)slot / p.block_size, place_in = (uint32_t)slot - block * p.block_size;
        const uint32_t normed = p.heads + p.kv_heads, all = normed + p.kv_heads;
        T* const q_row = reinterpret_cast<T*>(p.q_out) + (size_t)t * p.heads * p.dim;
        const size_t slot_at = ((size_t)block * p.kv_heads * p.block_size + place_in) * p.dim, head_on = (size_t)p.block_size * p.dim;
        auto target = [&](uint32_t h) -> T* {
            if (h < p.heads) return q_row + (size_t)h * p.dim;
            return h < normed ? reinterpret_cast<T*>(p.k_cache) + slot_at + (h - p.heads) * head_on : reinterpret_cast<T*>(p.v_cache) + slot_at + (h - normed) * head_on;
        };
        // 1 / sqrt(sum / dim + eps): the estimate and a Newton step
        auto factor = [&](float sum) {
            const float x = fmaf(sum, p.per_dim, p.eps), y = rsqrtf(x), e = fmaf(-x * y, y, 1.0f);
            return x > 0.0f && x < INFINITY ? fmaf(0.5f * y, e, y) : y;
        };
        auto turn = [&](bool turned, const float (&c)[V], const float (&s)[V], float (&x)[V], float (&y)[V]) {
            if (!turned) return;
            if (HALVES) {
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float a = x[i], b = y[i];
                    x[i] = a * c[i] - b * s[i];
                    y[i] = a * s[i] + b * c[i];
                }
            } else {
                // pairs (2i, 2i + 1) of the 2 V neighbours x, y; angle i of the unit
                float z[2 * V];
#pragma unroll
                for (int i = 0; i < V; i++) z[i] = x[i], z[V + i] = y[i];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float a = z[2 * i], b = z[2 * i + 1];
                    z[2 * i] = a * c[i] - b * s[i];
                    z[2 * i + 1] = a * s[i] + b * c[i];
                }
#pragma unroll
                for (int i = 0; i < V; i++) x[i] = z[i], y[i] = z[V + i];
            }
        };
        auto angles = [&](uint32_t u, bool turned, float (&c)[V], float (&s)[V]) {
            if (!turned) return;
            load_floats<V>(p.cos_cache + (size_t)pos * p.half + u * V, c);
            load_floats<V>(p.sin_cache + (size_t)pos * p.half + u * V, s);
        };
        auto sum_over_head = [&](float x) {
            for (uint32_t d = p.lanes >> 1; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            return x;
        };
        if (p.units <= p.lanes) {
            const uint32_t a = ua, b = ub;
            alignas(16) float c[V], s[V];
            if (has) angles(lane, uturned, c, s);
            for (uint32_t h0 = first_head; h0 - first_head < all; h0 += R * step) {
                using W = typename Bits<(int)sizeof(T) * V>::type;
                W wx[R], wy[R];
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const uint32_t h = h0 + r * step;
                    if (has && h < all) {
                        wx[r] = *reinterpret_cast<const W*>(src + (size_t)h * p.dim + a);
                        wy[r] = *reinterpret_cast<const W*>(src + (size_t)h * p.dim + b);
                    }
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const uint32_t h = h0 + r * step;
                    if (has && h >= normed && h < all) {   // values go as they are
                        T* dst = target(h);
                        *reinterpret_cast<W*>(dst + a) = wx[r];
                        *reinterpret_cast<W*>(dst + b) = wy[r];
                    }
                    const bool work = has && h < normed;
                    alignas(16) float x[V], y[V];
                    if (work) {
                        widen<T, V>(wx[r], x);
                        widen<T, V>(wy[r], y);
                    }
                    float sum = 0.0f;
                    if (p.wq && work) {
                        float part[2] = {0.0f, 0.0f};
                        const float* weight = weights[h < p.heads ? 0 : 1];
                        alignas(16) float u[V], v[V];
                        load_floats<V>(weight + a, u);
                        load_floats<V>(weight + b, v);
#pragma unroll
                        for (int i = 0; i < V; i++) {
                            part[0] = fmaf(x[i], x[i], part[0]);
                            part[1] = fmaf(y[i], y[i], part[1]);
                            x[i] *= u[i];
                            y[i] *= v[i];
                        }
                        sum = part[0] + part[1];
                    }
                    if (work) turn(uturned, c, s, x, y);   // (before the factor, which all elements share)
                    if (p.wq) {
                        const float f = factor(sum_over_head(sum));
                        if (work) {
#pragma unroll
                            for (int i = 0; i < V; i++) x[i] *= f, y[i] *= f;
                        }
                    }
                    if (work) {
                        T* dst = target(h);
                        store_vec<T, V>(dst + a, x);
                        store_vec<T, V>(dst + b, y);
                    }
                }
            }
        } else {
            // a head of more units than a warp has lanes: twice over the input, the second time from L1
            for (uint32_t h0 = first_head; h0 - first_head < all; h0 += step) {
                const bool valid = h0 < all, norm = p.wq && h0 < normed;
                const T* head = src + (size_t)h0 * p.dim;
                float f = 1.0f;
                if (p.wq) {
                    float sum = 0.0f;
                    for (uint32_t u = lane; valid && norm && u < p.units; u += p.lanes) {
                        uint32_t a, b;
                        bool turned;
                        place(u, a, b, turned);
                        float x[V], y[V];
                        load_vec<T, V>(head + a, x);
                        load_vec<T, V>(head + b, y);
#pragma unroll
                        for (int i = 0; i < V; i++) sum = fmaf(x[i], x[i], fmaf(y[i], y[i], sum));
                    }
                    sum = sum_over_head(sum);
                    f = factor(sum);
                }
                for (uint32_t u = lane; valid && u < p.units; u += p.lanes) {
                    uint32_t a, b;
                    bool turned;
                    place(u, a, b, turned);
                    alignas(16) float x[V], y[V], c[V], s[V];
                    load_vec<T, V>(head + a, x);
                    load_vec<T, V>(head + b, y);
                    if (norm) {
                        const float* w = h0 < p.heads ? p.wq : p.wk;
#pragma unroll
                        for (int i = 0; i < V; i++) x[i] *= f * w[a + i], y[i] *= f * w[b + i];
                    }
                    if (h0 < normed) {
                        angles(u, turned, c, s);
                        turn(turned, c, s, x, y);
                    }
                    T* dst = target(h0);
                    store_vec<T, V>(dst + a, x);
                    store_vec<T, V>(dst + b, y);
                }
            }
        }
    }
}

template <typename T, int V> auto pick_qkv(bool halves, bool few, bool staged) {
    if constexpr (sizeof(T) == 2) {
        if (staged) return halves ? lux_paged_qkv<T, V, true, 1, true> : lux_paged_qkv<T, V, false, 1, true>;
    }
    return halves ? (few ? lux_paged_qkv<T, V, true, 1, false> : lux_paged_qkv<T, V, true, 3, false>)
                  : (few ? lux_paged_qkv<T, V, false, 1, false> : lux_paged_qkv<T, V, false, 3, false>);
}

LuxBackendError plan_args(Context* ctx, Buffer* table, Buffer* free_blocks, Buffer* free_count, uint32_t seqs, uint32_t width, uint32_t block_size) {
    if (!ctx || seqs > LUX_PAGED_MAX_SEQS || width == 0 || block_size == 0) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    // positions and slots are 32-bit numbers
    if ((uint64_t)width * block_size > 0x7fffffffu) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!holds(table, mul({seqs, width})) || !holds(free_blocks, 0) || !holds(free_count, 1)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    return LUX_BACKEND_OK;
}

cudaError_t allow_plan_smem(const void* kfn, int which, int device) {
    static std::atomic<bool> configured[2][64];
    std::atomic<bool>& done = configured[which][device & 63];
    if (done.load(std::memory_order_relaxed)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, LUX_PAGED_MAX_SEQS * 12);
    if (e == cudaSuccess) done.store(true, std::memory_order_relaxed);
    return e;
}

}  // namespace

const void* kernel_addr_paged_reserve() { return (const void*)lux_paged_reserve; }
const void* kernel_addr_paged_release() { return (const void*)lux_paged_release; }
const void* kernel_addr_paged_qkv() { return (const void*)lux_paged_qkv<__nv_bfloat16, 8, true, 1, true>; }

}  // namespace luxcuda

using namespace luxcuda;

extern "C" LuxBackendError lux_cuda_paged_reserve(LuxBackendContext* context, LuxBackendBuffer* cached_lens, LuxBackendBuffer* new_lens,
                                                  LuxBackendBuffer* block_tables, LuxBackendBuffer* free_blocks, LuxBackendBuffer* free_count,
                                                  LuxBackendBuffer* q_starts, LuxBackendBuffer* context_lens, LuxBackendBuffer* positions,
                                                  LuxBackendBuffer* slots, uint32_t num_seqs, uint32_t max_blocks_per_seq, uint32_t block_size,
                                                  uint32_t max_tokens, uint32_t flags) {
    Context* ctx = as_ctx(context);
    Buffer *bc = as_buf(cached_lens), *bn = as_buf(new_lens), *bt = as_buf(block_tables), *bf = as_buf(free_blocks), *bk = as_buf(free_count),
           *bq = as_buf(q_starts), *bl = as_buf(context_lens), *bp = as_buf(positions), *bs = as_buf(slots);
    const LuxBackendError bad = plan_args(ctx, bt, bf, bk, num_seqs, max_blocks_per_seq, block_size);
    if (bad != LUX_BACKEND_OK) return bad;
    if (!holds(bc, num_seqs) || !holds(bn, num_seqs) || !holds(bq, (size_t)num_seqs + 1) || !holds(bl, num_seqs) || !holds(bp, max_tokens) ||
        !holds(bs, max_tokens) || max_tokens > 0x7fffffffu)
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    ReserveParams p{};
    p.cached = (const int32_t*)bc->ptr;
    p.fresh = (const int32_t*)bn->ptr;
    p.table = (int32_t*)bt->ptr;
    p.free_blocks = (const int32_t*)bf->ptr;
    p.free_count = (int32_t*)bk->ptr;
    p.q_starts = (int32_t*)bq->ptr;
    p.context = (int32_t*)bl->ptr;
    p.positions = (int32_t*)bp->ptr;
    p.slots = (int32_t*)bs->ptr;
    p.status = ctx->d_status;
    p.seqs = num_seqs;
    p.width = max_blocks_per_seq;
    p.block_size = block_size;
    p.max_tokens = max_tokens;
    p.capacity = bf->size / 4;
    cudaSetDevice(ctx->device);
    cudaError_t e = allow_plan_smem((const void*)lux_paged_reserve, 0, ctx->device);
    // one CTA where it has no more than two tokens per thread, else a cluster (with release, 64 sequences of 1 token: 13.3 us with one CTA,
    // 13.7 with eight; of 32 14.4, 14.3; of 100 19.1, 14.2)
    const unsigned ctas = max_tokens <= 2 * PLAN_THREADS ? 1 : PLAN_CLUSTER;
    if (e == cudaSuccess)
        e = launch_pdl(g_tune.pdl != 2, lux_paged_reserve, dim3(1, 1, ctas), dim3(PLAN_THREADS), (size_t)num_seqs * 12, ctx->stream, ctas, p);
    if (e != cudaSuccess) return map_cuda(e, "paged_reserve");
    count_launch("lux_paged_reserve");
    return finish_op(ctx, (flags & LUX_QMATMUL_FLAG_NO_SYNC) != 0, "paged_reserve");
}

extern "C" LuxBackendError lux_cuda_paged_release(LuxBackendContext* context, LuxBackendBuffer* keep_lens, LuxBackendBuffer* block_tables,
                                                  LuxBackendBuffer* free_blocks, LuxBackendBuffer* free_count, uint32_t num_seqs,
                                                  uint32_t max_blocks_per_seq, uint32_t block_size, uint32_t flags) {
    Context* ctx = as_ctx(context);
    Buffer *bl = as_buf(keep_lens), *bt = as_buf(block_tables), *bf = as_buf(free_blocks), *bk = as_buf(free_count);
    const LuxBackendError bad = plan_args(ctx, bt, bf, bk, num_seqs, max_blocks_per_seq, block_size);
    if (bad != LUX_BACKEND_OK) return bad;
    if (!holds(bl, num_seqs)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (num_seqs == 0) return LUX_BACKEND_OK;
    ReleaseParams p{};
    p.keep = (const int32_t*)bl->ptr;
    p.table = (int32_t*)bt->ptr;
    p.free_blocks = (int32_t*)bf->ptr;
    p.free_count = (int32_t*)bk->ptr;
    p.status = ctx->d_status;
    p.seqs = num_seqs;
    p.width = max_blocks_per_seq;
    p.block_size = block_size;
    p.capacity = bf->size / 4;
    cudaSetDevice(ctx->device);
    // one CTA where each of its warps has one sequence (with reserve, 64 sequences: 14.0 us with one CTA, 13.3 with eight; 256: 22.9, 14.1)
    const unsigned ctas = num_seqs <= PLAN_WARPS ? 1 : PLAN_CLUSTER;
    cudaError_t e = launch_pdl(g_tune.pdl != 2, lux_paged_release, dim3(1, 1, ctas), dim3(PLAN_THREADS), ((size_t)num_seqs / ctas + 1) * 4, ctx->stream, ctas, p);
    if (e != cudaSuccess) return map_cuda(e, "paged_release");
    count_launch("lux_paged_release");
    return finish_op(ctx, (flags & LUX_QMATMUL_FLAG_NO_SYNC) != 0, "paged_release");
}

extern "C" LuxBackendError lux_cuda_paged_qkv(LuxBackendContext* context, LuxBackendBuffer* qkv, LuxBackendBuffer* q_weight,
                                              LuxBackendBuffer* k_weight, LuxBackendBuffer* cos_cache, LuxBackendBuffer* sin_cache,
                                              LuxBackendBuffer* positions, LuxBackendBuffer* slots, LuxBackendBuffer* q_out,
                                              LuxBackendBuffer* k_cache, LuxBackendBuffer* v_cache, uint32_t num_tokens, uint32_t qkv_stride,
                                              uint32_t num_heads, uint32_t num_kv_heads, uint32_t head_dim, uint32_t rotary_dim,
                                              uint32_t block_size, float eps, uint32_t dtype, uint32_t flags) {
    Context* ctx = as_ctx(context);
    Buffer *bx = as_buf(qkv), *bwq = as_buf(q_weight), *bwk = as_buf(k_weight), *bc = as_buf(cos_cache), *bs = as_buf(sin_cache),
           *bp = as_buf(positions), *bl = as_buf(slots), *bq = as_buf(q_out), *bk = as_buf(k_cache), *bv = as_buf(v_cache);
    const size_t e = dtype_bytes(dtype);
    if (!ctx || !e || head_dim == 0 || head_dim > 1024 || rotary_dim > head_dim || rotary_dim % 2 || head_dim % 2 || block_size == 0 ||
        (num_heads == 0 && num_kv_heads == 0) || num_tokens > 0x7fffffffu)
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    const uint64_t row = mul({(uint64_t)num_heads + 2ull * num_kv_heads, head_dim}), stride = qkv_stride ? qkv_stride : row;
    if (row > 0x7fffffffu || stride < row) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!holds(bx, num_tokens ? mul({num_tokens - 1u, stride}) + row : 0, e) || !holds(bq, mul({num_tokens, num_heads, head_dim}), e) ||
        !holds(bl, num_tokens))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if ((bwq != nullptr) != (bwk != nullptr) || (bwq && (!holds(bwq, head_dim) || !holds(bwk, head_dim)))) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    QkvParams p{};
    if (rotary_dim) {
        if (!holds(bc, rotary_dim / 2) || !holds(bs, rotary_dim / 2) || !holds(bp, num_tokens)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
        p.cos_cache = (const float*)bc->ptr;
        p.sin_cache = (const float*)bs->ptr;
        p.positions = (const int32_t*)bp->ptr;
        p.table_rows = std::min(bc->size, bs->size) / 4 / (rotary_dim / 2);
    }
    const size_t block_elems = mul({std::max(num_kv_heads, 1u), block_size, head_dim});
    if (!holds(bk, block_elems, e) || !holds(bv, block_elems, e)) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    p.num_slots = (uint64_t)(std::min(bk->size, bv->size) / e / block_elems) * block_size;
    if (num_tokens == 0) return LUX_BACKEND_OK;
    p.qkv = bx->ptr;
    p.wq = bwq ? (const float*)bwq->ptr : nullptr;
    p.wk = bwk ? (const float*)bwk->ptr : nullptr;
    p.slots = (const int32_t*)bl->ptr;
    p.q_out = bq->ptr;
    p.k_cache = bk->ptr;
    p.v_cache = bv->ptr;
    p.status = ctx->d_status;
    p.stride = stride;
    p.tokens = num_tokens;
    p.heads = num_heads;
    p.kv_heads = num_kv_heads;
    p.dim = head_dim;
    p.half = rotary_dim / 2;
    p.block_size = block_size;
    p.eps = eps;
    p.per_dim = 1.0f / (float)head_dim;
    const bool halves = (flags & LUX_ROPE_FLAG_HALVES) != 0;
    // the widest vector that pairs, heads, rows and views allow, 16 bytes at most
    const uintptr_t views = (uintptr_t)bx->ptr | (uintptr_t)bq->ptr | (uintptr_t)bk->ptr | (uintptr_t)bv->ptr;
    if (views % e) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    uint32_t v = (uint32_t)(16 / e);
    const uintptr_t tables = (uintptr_t)p.cos_cache | (uintptr_t)p.sin_cache | (uintptr_t)p.wq | (uintptr_t)p.wk;
    while (v > 1 && ((v % 4 == 0 && tables % 16) || p.half % v || (head_dim - rotary_dim) % (2 * v) || head_dim % v || stride % v || views % (v * e))) v /= 2;
    p.units = head_dim / (2 * v);
    p.lanes = 1;
    while (p.lanes < p.units && p.lanes < 32) p.lanes *= 2;
    // a few heads per thread are requested at once where there are as many
    const bool few = num_heads + 2 * num_kv_heads <= QKV_THREADS / p.lanes;
    cudaSetDevice(ctx->device);
    // 16-bit rows with more heads than a CTA takes at once come through a ring of up to 24 KB (two of them at least, of up to 50 KB) where
    // they are whole 16 bytes.  By tokens and heads, bf16, with the ring against without: 8192 x 48 of 128 49 us, 61; 16384 x 24 66, 92;
    // 2048 x 48 13.0, 14.6; 592 x 24 4.6, 5.0; 1 x 48 3.9, 4.1; but 16384 x 12, one round, 47, 42, and f32, with twice the bytes to a thread's
    // loads, 8192 x 48 75, 73, 2048 x 24 11.4, 9.4.
    p.row_bytes = (uint32_t)std::min<uint64_t>(row * e, 0x7fffffffu);
    const uint32_t pitch = (p.row_bytes + 127) / 128 * 128;
    p.slots_ahead = std::clamp((24u << 10) / std::max(pitch, 1u), 2u, (uint32_t)QKV_MAX_AHEAD);
    const bool staged = e == 2 && !few && pitch <= QKV_MAX_PITCH && p.row_bytes % 16 == 0 && stride * e % 16 == 0 &&
                        ((uintptr_t)p.qkv & 15u) == 0;
    using Kernel = void (*)(const QkvParams);
    auto pick = [&](auto tag) -> Kernel {
        using T = decltype(tag);
        if constexpr (sizeof(T) == 2) {
            if (v == 8) return pick_qkv<T, 8>(halves, few, staged);
        }
        return v == 4 ? pick_qkv<T, 4>(halves, few, staged) : v == 2 ? pick_qkv<T, 2>(halves, few, staged) : pick_qkv<T, 1>(halves, few, staged);
    };
    const Kernel kfn = dtype == LUX_QDTYPE_F32 ? pick(float{}) : dtype == LUX_QDTYPE_F16 ? pick(__half{}) : pick(__nv_bfloat16{});
    const size_t smem = staged ? (size_t)p.slots_ahead * pitch : 0;
    if (smem > QKV_OPEN) {
        // The largest ring's, whatever this call's is: the allowance belongs to the kernel, which calls of other threads and captured ones
        // share, so that no call may lower it.  (A call that sets it again is cheap.)
        const cudaError_t a = cudaFuncSetAttribute((const void*)kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * QKV_MAX_PITCH);
        if (a != cudaSuccess) return map_cuda(a, "paged_qkv");
    }
    // one wave of the CTAs that registers and shared memory allow goes through the tokens
    const unsigned per_sm = staged ? (unsigned)std::clamp<size_t>((222u << 10) / (smem + (6u << 10)), 1, 5) : 5u;
    const unsigned grid = std::min<unsigned>(num_tokens, (unsigned)ctx->sm_count * per_sm);
    cudaError_t err = launch_pdl(g_tune.pdl != 2, kfn, dim3(grid), dim3(QKV_THREADS), smem, ctx->stream, 1, p);
    if (err != cudaSuccess) return map_cuda(err, "paged_qkv");
    count_launch("lux_paged_qkv");
    return finish_op(ctx, (flags & LUX_QMATMUL_FLAG_NO_SYNC) != 0, "paged_qkv");
}
