// verify_drafts.cu -- which drafted tokens stand against the target's probabilities, and the token drawn behind them
// (lux/gpu/paged_ext.h).
//
// Of a sequence's rows the tests read one number per draft; only ONE row of the target's (and the draft's) distribution is
// read as a whole, the one a token is drawn from: 4 or 8 bytes per entry of the vocabulary and sequence, bound by HBM for
// a batch and by latency for one sequence.  A cluster of eight CTAs takes a sequence (one SM alone would need 10 us for the 1 MB of a
// 128k vocabulary; 64 sequences of 128256 entries, 66 MB: 15.8 us, 4.2 TB/s; one of 32000: 5.4 us): every CTA makes the tests by itself, sums its eighth of the row, tells the others through distributed
// shared memory, and the CTA in whose part the drawn sum is passed looks for the token, with all threads, in the one warp's
// segment that it falls into.
//
// Sums are in 64 bits, each in a fixed order: a token is drawn by comparing sums of up to 10^5 terms, and in 32 bits
// their order would decide which token it is.
#include "paged.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <utility>

namespace cg = cooperative_groups;

namespace luxcuda {

namespace {

constexpr int VD_THREADS = 256, VD_CLUSTER = 8, VD_WARPS = VD_THREADS / 32;

struct VerifyParams {
    const float* target;
    const float* draft;                                    // null: drafts are certain
    const int32_t* tokens;
    const float* uniforms;
    const int32_t* q_starts;
    const int32_t* context;
    int32_t* out;
    int32_t* accepted;
    int32_t* kept;
    uint32_t rows, vocab;
};

// What the row is drawn from.  x: the refused draft (-1: the target alone).
struct Weights {
    const float* p;
    const float* q;                                        // null: a certain draft of x, or none
    int32_t x;
    __device__ __forceinline__ double of(float a, float b, uint32_t i) const {
        // (the comparison is exact in 32 bits, and false for NaN, which counts as no weight)
        if (q) return a > b ? (double)a - (double)b : 0.0;
        const double w = (int32_t)i == x ? (double)a - 1.0 : (double)a;
        return w > 0.0 ? w : 0.0;
    }
    __device__ __forceinline__ double at(uint32_t i) const { return of(p[i], q ? q[i] : 0.0f, i); }
    // one, or a vector of four
    template <bool VEC> __device__ __forceinline__ void some(uint32_t i, double* x) const {
        if constexpr (VEC) {
            const float4 a = *reinterpret_cast<const float4*>(p + i);
            const float4 b = q ? *reinterpret_cast<const float4*>(q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[0] = of(a.x, b.x, i);
            x[1] = of(a.y, b.y, i + 1);
            x[2] = of(a.z, b.z, i + 2);
            x[3] = of(a.w, b.w, i + 3);
        } else {
            x[0] = at(i);
        }
    }
};

__device__ __forceinline__ double warp_sum(double v) {
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// The sum of weights [lo, hi) by a warp; four at a time where the rows are aligned for it.
template <bool VEC> __device__ __forceinline__ double segment_sum(const Weights& w, uint32_t lo, uint32_t hi, uint32_t lane) {
    double sum = 0.0;
    if (VEC) {
        constexpr int R = 4;
        for (uint32_t i0 = lo + 4 * lane; i0 - 4 * lane < hi; i0 += 128 * R) {
            float4 a[R], b[R];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const uint32_t i = i0 + 128 * r;
                a[r] = b[r] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < hi) {
                    a[r] = *reinterpret_cast<const float4*>(w.p + i);
                    if (w.q) b[r] = *reinterpret_cast<const float4*>(w.q + i);
                }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                const uint32_t i = i0 + 128 * r;
                if (i < hi) sum += (w.of(a[r].x, b[r].x, i) + w.of(a[r].y, b[r].y, i + 1)) + (w.of(a[r].z, b[r].z, i + 2) + w.of(a[r].w, b[r].w, i + 3));
            }
        }
    } else {
        for (uint32_t i = lo + lane; i < hi; i += 32) sum += w.at(i);
    }
    return warp_sum(sum);
}

template <bool VEC> __global__ void __launch_bounds__(VD_THREADS, 4) lux_verify_drafts(const VerifyParams p) {
    __shared__ double warp_sums[VD_WARPS], cta_sums[VD_CLUSTER], piece_sums[VD_WARPS];
    __shared__ uint32_t shared_taken;
    __shared__ int first_over, last_some;                  // of the threads that look for the token
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x / VD_CLUSTER;
    pdl_launch_dependents();
    pdl_wait();
    const uint32_t first = (uint32_t)min(max(load_i32(p.q_starts + s), 0), (int32_t)p.rows);
    const uint32_t end = (uint32_t)min(max(load_i32(p.q_starts + s + 1), (int32_t)first), (int32_t)p.rows);
    if (first == end) {                                    // no chunk (the same in all CTAs of the cluster)
        if (rank == 0 && tid == 0) {
            p.accepted[s] = 0;
            if (p.kept) p.kept[s] = load_i32(p.context + s);
        }
        return;
    }
    auto started = cluster.barrier_arrive();
    const uint32_t drafts = end - first - 1;
    const double uniform = p.uniforms[end - 1];            // (here, so that it is there when the sums are)
    if (warp == 0) {
        uint32_t taken = 0;
        for (uint32_t i0 = 0; i0 < drafts; i0 += 32) {
            bool stands = false;
            if (i0 + lane < drafts) {
                const uint32_t row = first + i0 + lane;
                const int32_t x = load_i32(p.tokens + row + 1);
                if (x >= 0 && (uint32_t)x < p.vocab) {
                    const size_t at = (size_t)row * p.vocab + (uint32_t)x;
                    // both factors are f32, so the product is exact
                    stands = (double)p.uniforms[row] * (p.draft ? (double)p.draft[at] : 1.0) < (double)p.target[at];
                }
            }
            const uint32_t all = __ballot_sync(0xffffffffu, stands);
            const uint32_t run = all == 0xffffffffu ? 32 : __ffs(~all) - 1;
            taken += run;
            if (run < 32) break;
        }
        if (lane == 0) {
            shared_taken = taken;
            first_over = VD_THREADS;
            last_some = -1;
        }
    }
    __syncthreads();
    const uint32_t taken = shared_taken, row = first + taken;
    Weights w{p.target + (size_t)row * p.vocab, nullptr, -1};
    const bool refused = taken < drafts;
    if (refused) {
        w.q = p.draft ? p.draft + (size_t)row * p.vocab : nullptr;
        w.x = p.draft ? -1 : load_i32(p.tokens + row + 1);
    }
    // parts and segments in whole vectors
    constexpr uint32_t unit = VEC ? 4 : 1;
    const uint32_t units = (p.vocab + unit - 1) / unit;
    auto cut = [&](uint32_t n, uint32_t i, uint32_t of) { return (uint32_t)((uint64_t)n * i / of); };
    const uint32_t part_lo = cut(units, rank, VD_CLUSTER), part = cut(units, rank + 1, VD_CLUSTER) - part_lo;
    const uint32_t lo = (part_lo + cut(part, warp, VD_WARPS)) * unit, hi = min((part_lo + cut(part, warp + 1, VD_WARPS)) * unit, p.vocab);
    cluster.barrier_wait(std::move(started));              // the others run, so their shared memory may be written
    double total = 0.0;
    for (int attempt = 0; attempt < 2; attempt++) {
        const double sum = segment_sum<VEC>(w, lo, hi, lane);
        if (lane == 0) warp_sums[warp] = sum;
        __syncthreads();
        if (tid < VD_CLUSTER) {
            double mine = 0.0;
            for (int i = 0; i < VD_WARPS; i++) mine += warp_sums[i];
            *cluster.map_shared_rank(&cta_sums[rank], tid) = mine;
        }
        cluster.sync();
        total = 0.0;
        for (int r = 0; r < VD_CLUSTER; r++) total += cta_sums[r];
        if (total > 0.0 || !refused || attempt) break;
        w.q = nullptr;                                     // the draft is the target: the target alone
        w.x = -1;
        cluster.sync();                                    // all have read the sums
    }
    const double goal = uniform * total;
    // the CTA and the warp in whose range the sum passes the goal, the last one with a weight if none does
    int cta = -1;
    double before = 0.0, base = 0.0;
    for (int r = 0; r < VD_CLUSTER; r++) {
        const double up_to = before + cta_sums[r];
        if (cta_sums[r] > 0.0) {
            cta = r;
            base = before;
            if (up_to > goal) break;
        }
        before = up_to;
    }
    if (cta == (int)rank) {
        int pick = -1;
        double from = base, start = base;
        for (int i = 0; i < VD_WARPS; i++) {
            const double up_to = from + warp_sums[i];
            if (warp_sums[i] > 0.0) {
                pick = i;
                start = from;
                if (up_to > goal) break;
            }
            from = up_to;
        }
        // the segment by all threads, a contiguous piece of whole vectors each
        const uint32_t seg_lo = part_lo + cut(part, pick, VD_WARPS), seg = part_lo + cut(part, pick + 1, VD_WARPS) - seg_lo;
        const uint32_t a = (seg_lo + cut(seg, tid, VD_THREADS)) * unit, b = min((seg_lo + cut(seg, tid + 1, VD_THREADS)) * unit, p.vocab);
        double mine = 0.0;
        for (uint32_t i = a; i < b; i += unit) {
            double x[unit];
            w.some<VEC>(i, x);
            if constexpr (VEC) mine += (x[0] + x[1]) + (x[2] + x[3]);
            else mine += x[0];
        }
        double sums = mine;
        for (int d = 1; d < 32; d <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, sums, d);
            if ((int)lane >= d) sums += v;
        }
        if (lane == 31) piece_sums[warp] = sums;
        __syncthreads();
        for (uint32_t i = 0; i < warp; i++) start += piece_sums[i];
        double at = __shfl_up_sync(0xffffffffu, sums, 1);
        at = start + (lane ? at : 0.0);
        if (mine > 0.0) {
            if (start + sums > goal) atomicMin(&first_over, (int)tid);
            atomicMax(&last_some, (int)tid);
        }
        __syncthreads();
        if ((int)tid == (first_over < VD_THREADS ? first_over : last_some)) {
            int32_t token = -1;
            for (uint32_t i = a; i < b; i++) {
                const double v = w.at(i);
                if (!(v > 0.0)) continue;
                token = (int32_t)i;
                at += v;
                if (at > goal) break;
            }
            p.out[row] = token;
        }
    }
    if (rank == 0) {
        for (uint32_t i = tid; i < end - first; i += VD_THREADS) {
            if (i < taken) p.out[first + i] = load_i32(p.tokens + first + i + 1);
            else if (i > taken || cta < 0) p.out[first + i] = -1;
        }
        if (tid == 0) {
            p.accepted[s] = (int32_t)taken;
            if (p.kept) p.kept[s] = load_i32(p.context + s) - (int32_t)(drafts - taken);
        }
    }
    cluster.sync();                                        // no CTA leaves while its sums may still be written
}

}  // namespace

const void* kernel_addr_verify_drafts() { return (const void*)lux_verify_drafts<true>; }

}  // namespace luxcuda

using namespace luxcuda;

extern "C" LuxBackendError lux_cuda_verify_drafts(LuxBackendContext* context, LuxBackendBuffer* target_probs, LuxBackendBuffer* draft_probs,
                                                  LuxBackendBuffer* tokens, LuxBackendBuffer* uniforms, LuxBackendBuffer* q_starts,
                                                  LuxBackendBuffer* out_tokens, LuxBackendBuffer* accepted, LuxBackendBuffer* context_lens,
                                                  LuxBackendBuffer* kept_lens, uint32_t num_seqs, uint32_t num_rows, uint32_t vocab,
                                                  uint32_t flags) {
    Context* ctx = as_ctx(context);
    Buffer *bt = as_buf(target_probs), *bd = as_buf(draft_probs), *bx = as_buf(tokens), *bu = as_buf(uniforms), *bq = as_buf(q_starts),
           *bo = as_buf(out_tokens), *ba = as_buf(accepted), *bc = as_buf(context_lens), *bk = as_buf(kept_lens);
    const size_t n = mul({num_rows, vocab});
    if (!ctx || vocab == 0 || vocab > 0x7ffffff0u || num_rows > 0x7fffffffu || num_seqs > 0x7fffffffu / VD_CLUSTER) return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (!holds(bt, n) || (bd && !holds(bd, n)) || !holds(bx, num_rows) || !holds(bu, num_rows) || !holds(bq, (size_t)num_seqs + 1) ||
        !holds(bo, num_rows) || !holds(ba, num_seqs) || (bc != nullptr) != (bk != nullptr) || (bc && (!holds(bc, num_seqs) || !holds(bk, num_seqs))))
        return LUX_BACKEND_ERROR_INVALID_ARGUMENT;
    if (num_seqs == 0) return LUX_BACKEND_OK;
    VerifyParams p{};
    p.target = (const float*)bt->ptr;
    p.draft = bd ? (const float*)bd->ptr : nullptr;
    p.tokens = (const int32_t*)bx->ptr;
    p.uniforms = (const float*)bu->ptr;
    p.q_starts = (const int32_t*)bq->ptr;
    p.context = bc ? (const int32_t*)bc->ptr : nullptr;
    p.out = (int32_t*)bo->ptr;
    p.accepted = (int32_t*)ba->ptr;
    p.kept = bk ? (int32_t*)bk->ptr : nullptr;
    p.rows = num_rows;
    p.vocab = vocab;
    cudaSetDevice(ctx->device);
    const bool vec = vocab % 4 == 0 && (((uintptr_t)p.target | (uintptr_t)p.draft) & 15u) == 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(num_seqs * VD_CLUSTER);
    cfg.blockDim = dim3(VD_THREADS);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = VD_CLUSTER;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_tune.pdl != 2 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, vec ? lux_verify_drafts<true> : lux_verify_drafts<false>, p);
    if (e != cudaSuccess) return map_cuda(e, "verify_drafts");
    count_launch("lux_verify_drafts");
    return finish_op(ctx, (flags & LUX_QMATMUL_FLAG_NO_SYNC) != 0, "verify_drafts");
}
