/*
 * lux/gpu/paged_ext.h -- serving over a paged KV cache, exported by libluxgpu_backend_cuda.so BESIDE the backend
 * vtable.  One step of a serving host, all lengths on the device, so that it can be captured once and replayed:
 *   lux_cuda_paged_reserve           blocks, slots and positions for the step's new tokens
 *   lux_cuda_paged_qkv               per layer: norms and rotates queries and keys, keys and values into the cache
 *   lux_cuda_paged_chunk_attention   per layer: the new tokens' attention over the cache
 *   lux_cuda_verify_drafts           after the last layer: which drafted tokens stand, and the token behind them
 *   lux_cuda_paged_release           the blocks behind what is kept go back
 * The cache has the layout that lux_cuda_paged_attention_f32 reads, [num_blocks, num_kv_heads, block_size, head_dim],
 * in f32, f16 or bf16 (LUX_QDTYPE_*); block tables are i32 [num_seqs, max_blocks_per_seq], an entry below 0 being no
 * block.  A token's slot is block * block_size + its place in the block.
 *
 * No counterpart in luxcpp/webgpu: its paged attention (kernels/wgsl/steel/attention/paged.wgsl) reads a cache that
 * nothing there fills.  Conventions of attention_ext.h: LuxBackendBuffer operands, arguments validated before anything
 * is launched, a LuxBackendError comes back, nothing throws; `flags` takes LUX_QMATMUL_FLAG_NO_SYNC.  Operands must
 * not overlap unless it says so.  What only the device can see (a block number outside the cache, a position outside
 * the cos/sin tables, too few free blocks) is reported as lux_cuda_paged_attention_f32 reports it: the next waiting
 * call answers DEVICE_LOST, lux_cuda_last_device_status says which, and the context stays usable.
 */
#ifndef LUX_GPU_PAGED_EXT_H
#define LUX_GPU_PAGED_EXT_H

#include "lux/gpu/attention_ext.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    /* lux_cuda_paged_qkv: pairs are the elements (i, i + rotary_dim / 2) instead of the adjacent ones (2i, 2i + 1). */
    LUX_ROPE_FLAG_HALVES = 1u << 6
};

enum { LUX_PAGED_MAX_SEQS = 8192 };      /* of lux_cuda_paged_reserve and lux_cuda_paged_release */

/*
 * Blocks and places for new tokens.  Sequence s holds cached_lens[s] tokens, in the blocks of its table row, and gets
 * new_lens[s] more (0: nothing happens to it).  Entries of its row that the new tokens reach and that are below 0 get blocks from the
 * END of the free list (the entry at *free_count - 1 first), sequences in order and blocks in order; entries that
 * hold a block already (kept by an earlier release) are used as they are.  A block belongs to one sequence.
 *   cached_lens, new_lens  i32 [num_seqs]
 *   block_tables           i32 [num_seqs, max_blocks_per_seq], updated
 *   free_blocks, free_count  the free list, i32 [capacity] (the buffer's size says how many) and i32 [1], updated;
 *                          entries behind the count are left as they are
 *   q_starts               i32 [num_seqs + 1] out: where each sequence's new tokens begin among all of them
 *   context_lens           i32 [num_seqs] out: cached_lens + new_lens (may be the buffer of cached_lens)
 *   positions, slots       i32 [max_tokens] out, one per new token; behind the last one 0 and -1
 * If a length is negative, a sequence outgrows its row, the new tokens are more than max_tokens or the free list
 * (or its count is no count of it) does not give enough, nothing is handed out: tables, list and count stay,
 * q_starts is all 0, context_lens is cached_lens, every slot is -1, and the device status is 0x7C05000B.
 * The number of blocks of the caches is not known here, so block numbers are taken as they are; where one (of the table or the
 * free list) is below 0 or has no 31-bit slots, its tokens' slots are -1 and the device status is 0x7C050009.
 */
LUX_GPU_PLUGIN_EXPORT LuxBackendError lux_cuda_paged_reserve(
    LuxBackendContext* ctx, LuxBackendBuffer* cached_lens, LuxBackendBuffer* new_lens, LuxBackendBuffer* block_tables,
    LuxBackendBuffer* free_blocks, LuxBackendBuffer* free_count, LuxBackendBuffer* q_starts, LuxBackendBuffer* context_lens,
    LuxBackendBuffer* positions, LuxBackendBuffer* slots,
    uint32_t num_seqs, uint32_t max_blocks_per_seq, uint32_t block_size, uint32_t max_tokens, uint32_t flags);

/*
 * The blocks behind the first keep_lens[s] tokens of each sequence go back to the free list and their entries become -1
 * (0: the sequence is finished, all go; below 0: it is left alone).  A row's blocks are its entries up to the first one
 * below 0.  They are put back so that reserving the same tokens again gives the same blocks.  If the list has no room
 * for them all nothing changes and the device status is 0x7C05000B.
 */
LUX_GPU_PLUGIN_EXPORT LuxBackendError lux_cuda_paged_release(
    LuxBackendContext* ctx, LuxBackendBuffer* keep_lens, LuxBackendBuffer* block_tables, LuxBackendBuffer* free_blocks,
    LuxBackendBuffer* free_count, uint32_t num_seqs, uint32_t max_blocks_per_seq, uint32_t block_size, uint32_t flags);

/*
 * What lies between the qkv projection and attention, in one pass.  Each query and key head x of a token is normalised,
 * y = x / sqrt(mean(x^2) + eps) * weight, and the first rotary_dim elements of y are rotated by the token's position,
 * (a, b) -> (a cos - b sin, a sin + b cos), in f32, rounded once; values are copied.  Queries go to q_out, keys and
 * values into the token's slot of the caches.
 *   qkv                    [num_tokens, qkv_stride]: num_heads query heads, then num_kv_heads key heads, then as many value
 *                          heads, head_dim each; qkv_stride 0 stands for (num_heads + 2 num_kv_heads) head_dim
 *   q_weight, k_weight     f32 [head_dim], both or neither (NULL: no norm)
 *   cos_cache, sin_cache   f32 [positions, rotary_dim / 2], as lux_cuda_rope_precompute_cache_f32 writes them for a head
 *                          of rotary_dim (NULL, both, with rotary_dim 0: no rotation, positions may be NULL too)
 *   positions, slots       i32 [num_tokens].  A token whose slot is below 0 is padding: nothing is written for it.  A slot
 *                          outside the caches or a position outside the tables is treated so too, and sets the device status
 *                          (0x7C050009, 0x7C05000A)
 *   q_out                  [num_tokens, num_heads, head_dim]
 *   dtype                  LUX_QDTYPE_* of qkv, q_out and the caches
 * head_dim and rotary_dim are even, rotary_dim at most head_dim, head_dim at most 1024.  Where two tokens have the same
 * slot, each element of its rows is one of theirs.
 */
LUX_GPU_PLUGIN_EXPORT LuxBackendError lux_cuda_paged_qkv(
    LuxBackendContext* ctx, LuxBackendBuffer* qkv, LuxBackendBuffer* q_weight, LuxBackendBuffer* k_weight,
    LuxBackendBuffer* cos_cache, LuxBackendBuffer* sin_cache, LuxBackendBuffer* positions, LuxBackendBuffer* slots,
    LuxBackendBuffer* q_out, LuxBackendBuffer* k_cache, LuxBackendBuffer* v_cache,
    uint32_t num_tokens, uint32_t qkv_stride, uint32_t num_heads, uint32_t num_kv_heads, uint32_t head_dim, uint32_t rotary_dim,
    uint32_t block_size, float eps, uint32_t dtype, uint32_t flags);

/*
 * Attention of each sequence's new tokens over its paged cache, which holds their own keys and values too.
 *   q, out         [num_tokens, num_heads, head_dim]; the new tokens of sequence s are rows q_starts[s] .. q_starts[s + 1] - 1
 *   k/v_cache      [num_blocks, num_kv_heads, block_size, head_dim]; query head h reads KV head h / (num_heads / num_kv_heads)
 *   block_tables   i32 [num_seqs, max_blocks_per_seq]
 *   q_starts       i32 [num_seqs + 1], rising; values outside 0 .. num_tokens are cut there
 *   context_lens   i32 [num_seqs]: keys of the sequence, its new tokens included; cut at max_blocks_per_seq * block_size
 *   lse            NULL or f32 [num_tokens, num_heads]: max + log(sum), -3.402823e38 for a row that sees no key
 *   workspace      lux_cuda_paged_chunk_workspace bytes at least, 16-byte aligned, owned by this call until it has run: calls that
 *                  may run at the same time, replays of captured ones too, need one each; nothing is kept in it
 *   dtype          LUX_QDTYPE_* of q, out and the caches
 * The new tokens are the last of the sequence: with LUX_ATTN_FLAG_CAUSAL new token i of n sees keys
 * 0 .. context_len - n + i, without it all of them.  A row that sees no key is zero (a context shorter than the chunk
 * leaves its first rows so).  Rows in front of q_starts[0] and behind q_starts[num_seqs] are left as they are.  What a row
 * must not see takes no part in it, whatever it holds (NaN and infinities included; beside values that are no numbers a row of 16-bit
 * data is summed another way, equal to rounding).  A block-table entry outside the
 * cache that a key lies in is not followed: the device status becomes 0x7C050009 and that sequence's rows are undefined.
 * Scores, softmax and sums are f32; with 16-bit data the weights are rounded to it before they meet the values.
 * The result depends on all lengths of the call (work is dealt out evenly, and where a long context is cut into parts
 * follows from them), to rounding; the same call gives the same bits.  head_dim up to 256.
 */
LUX_GPU_PLUGIN_EXPORT LuxBackendError lux_cuda_paged_chunk_attention(
    LuxBackendContext* ctx, LuxBackendBuffer* q, LuxBackendBuffer* k_cache, LuxBackendBuffer* v_cache,
    LuxBackendBuffer* block_tables, LuxBackendBuffer* q_starts, LuxBackendBuffer* context_lens, LuxBackendBuffer* out,
    LuxBackendBuffer* lse, LuxBackendBuffer* workspace,
    uint32_t num_seqs, uint32_t num_tokens, uint32_t num_heads, uint32_t num_kv_heads, uint32_t head_dim,
    uint32_t block_size, uint32_t max_blocks_per_seq, float scale, uint32_t dtype, uint32_t flags);

/* Bytes of workspace that lux_cuda_paged_chunk_attention needs for these sizes; a larger one serves as well.  0 for arguments that the call refuses. */
LUX_GPU_PLUGIN_EXPORT size_t lux_cuda_paged_chunk_workspace(
    LuxBackendContext* ctx, uint32_t num_seqs, uint32_t num_tokens, uint32_t num_heads, uint32_t num_kv_heads, uint32_t head_dim,
    uint32_t dtype);

/*
 * Which drafted tokens stand.  A sequence's chunk is its last known token followed by the drafted ones, in rows
 * q_starts[s] .. q_starts[s + 1] - 1 of `tokens`; row r of target_probs is the target's distribution of the token behind
 * it, row r of draft_probs the one that the draft in row r + 1 was drawn from.  Drafts are taken in order while
 * uniforms[r] * draft_probs[r][x] < target_probs[r][x], x = tokens[r + 1] (an x outside the vocabulary is refused).  At the first refused one, in the
 * row in front of it, a token is drawn from max(target - draft, 0), or from the target where that is zero everywhere;
 * behind the last accepted draft from the target.  It is the lowest token at which the sum of the weights up to it
 * exceeds uniforms[q_starts[s + 1] - 1] times their sum (the last one with a weight, if rounding or a uniform of 1 leaves none; -1 if
 * there is no weight at all).  Weights that are negative or NaN count as 0.  Comparisons and sums are in 64 bits.
 *   target_probs   f32 [num_rows, vocab]; draft_probs the same, or NULL: drafts are certain (1 at the token)
 *   tokens, out_tokens  i32 [num_rows]; out: the accepted drafts from q_starts[s] on, the drawn token, then -1
 *   uniforms       f32 [num_rows], in [0, 1)
 *   q_starts       i32 [num_seqs + 1], as for lux_cuda_paged_chunk_attention; rows outside are left as they are
 *   accepted       i32 [num_seqs] out: number of accepted drafts
 *   context_lens, kept_lens  i32 [num_seqs], both or neither: kept = context_len - refused drafts, which is what
 *                  lux_cuda_paged_release wants (may be the same buffer)
 */
LUX_GPU_PLUGIN_EXPORT LuxBackendError lux_cuda_verify_drafts(
    LuxBackendContext* ctx, LuxBackendBuffer* target_probs, LuxBackendBuffer* draft_probs, LuxBackendBuffer* tokens,
    LuxBackendBuffer* uniforms, LuxBackendBuffer* q_starts, LuxBackendBuffer* out_tokens, LuxBackendBuffer* accepted,
    LuxBackendBuffer* context_lens, LuxBackendBuffer* kept_lens,
    uint32_t num_seqs, uint32_t num_rows, uint32_t vocab, uint32_t flags);

#ifdef __cplusplus
}
#endif
#endif /* LUX_GPU_PAGED_EXT_H */
