/* native-hip: operators over a paged key-value cache in device memory - storing the rows of new tokens, attention
 * that reads the cache, eviction by accumulated attention weight.
 *
 * The products of native_hip.h leave q, k and v of a step in HBM; these calls are what stands between them and the
 * output projection for a caller that keeps its own cache: the reference's attention over paged K/V
 * (langtax/src/decode.rs:11126-11197, 12059-12100; langtax/src/kv_page.rs:47-53, 410-438) runs on the host and has
 * neither an f16 cache, nor the window with first tokens, nor the eviction.
 *
 * Conventions are those of native_hip.h: plain pointers and sizes, LNH_OK or an lnh_status, lnh_last_error(exec),
 * validation before anything is launched, no host synchronisation, `stream` a hipStream_t of the executor's GPU
 * (NULL = the executor's own stream).  All buffers are device memory of that GPU and belong to the caller; f32 and
 * f16 buffers start on 16 bytes and their row strides are multiples of four elements (LNH_ERR_INVALID otherwise),
 * u32 arrays on 4 bytes.  Outputs must not overlap inputs.
 *
 * What a call reads from device arrays (block tables, lengths, row starts) it cannot refuse, so it is held in bounds
 * by the kernels instead: a block number that is not below n_blocks is never followed (its positions are as if they
 * were not there: not seen, not written), a length counts up to max_len, rows up to n_tokens.
 */
#ifndef NATIVE_HIP_ATTENTION_H
#define NATIVE_HIP_ATTENTION_H

#include "native_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The cache: K and V as [n_blocks][n_layer][n_head_kv][kv_block][head_dim] of LNH_TYPE_F32 or LNH_TYPE_F16
 * (LNH_ERR_UNSUPPORTED otherwise), head_dim a multiple of 8, at most 256 (LNH_ERR_UNSUPPORTED otherwise), at most 2^31
 * rows of head_dim in all.  device_w, where weights are kept: [n_blocks][n_layer][n_head_kv][kv_block] f32, else NULL. */
typedef struct lnh_kv_cache {
    uint32_t ggml_type;
    uint32_t n_layer, n_head_kv, head_dim, kv_block, n_blocks;
    void *device_k, *device_v;
    float *device_w;
} lnh_kv_cache;

/* The sequences of a call.  Position t of sequence b lies in block device_tables[b * table_stride + t / kv_block] at
 * place t % kv_block.  device_lens[b] counts the sequence's positions, the call's new tokens among them: with n new
 * tokens, new token i stands at position device_lens[b] - n + i (one that would stand below 0 is as if not there: not
 * stored, its output 0).  The rows of token-major arrays (q, k, v, out) belong to the sequences in order:
 * device_starts[b] .. device_starts[b + 1] - 1 to sequence b (n_seqs + 1 ascending numbers, the last at most n_tokens),
 * or, with device_starts NULL, row b to sequence b (n_tokens = n_seqs).  Rows that belong to no sequence are left as
 * they are.  max_new and max_len bound the new tokens and the length of any one sequence (new tokens beyond max_new of
 * a sequence are left out): they size the launch, so a captured call may be replayed with any tables, lengths and
 * starts within them.  max_len must not exceed table_stride * kv_block. */
typedef struct lnh_kv_seqs {
    size_t n_seqs, n_tokens, max_new, max_len;
    const uint32_t *device_tables;
    size_t table_stride;
    const uint32_t *device_lens;
    const uint32_t *device_starts;
} lnh_kv_seqs;

/* K and V of the new tokens into `layer` of the cache: row r of device_k is n_head_kv * head_dim floats at
 * device_k + r * k_stride (strides in floats).  An f16 cache takes the nearest f16, ties to even, values beyond 65504 become
 * infinite.  Two new tokens that share a place (one block in two tables) race. */
int lnh_kv_store_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t layer,
                        const float *device_k, size_t k_stride, const float *device_v, size_t v_stride, void *stream);

/* out = softmax(scale q K^T) V for every new token and each of n_head query heads (a multiple of n_head_kv; query
 * head h reads key-value head h * n_head_kv / n_head; 0 < scale <= 2^127), over `layer` of the cache: the new tokens' own rows have to be
 * stored before.  The token at position p sees position t where t <= p and, with window > 0, p - t < window or
 * t < sinks (sinks without a window: LNH_ERR_INVALID).  Rows of q and out are n_head * head_dim floats, strides in
 * floats.  A token that sees nothing gets zeros; so does one whose every score is -infinity.  What lies in positions
 * that a token does not see, infinities and NaN among it, does not reach its row.
 * Scores, the softmax and the sums are f32; over an f16 cache q and the probabilities enter the matrix cores as two
 * f16 parts each (22 bits).  A row that comes out not finite so, or of scores beyond 2^21 / log2(e), is computed again
 * from the definition, its scores summed in 64 bits, at about a hundred times the time.
 * weights != 0 (needs device_w): for every position t below the length of a sequence with new tokens, per key-value head,
 * device_w = decay * device_w + the sum over the sequence's new tokens and the head's query heads of the softmax
 * probability they give t.  decay 1 sums over all calls, 0 keeps this call's alone, whatever the memory held before.
 * The caller sets the weight of a new position to zero before it is first counted (or passes decay 0).  Sequences
 * that share a block then race on its weights.
 * Uses the executor's workspace like lnh_gemm_device: calls of one executor on one stream at a time, and one call of
 * the largest shape before capturing.  Weights take workspace by max_len, for scores or sums of each of its positions: up to 16 rows (new tokens
 * times query heads of a key-value head) n_head * max_new * max_len floats a sequence, above that a float a position, key-value head and
 * block of 64 to 256 rows.  Sequences go in parts where theirs together pass 1 GiB. */
int lnh_attn_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t layer, size_t n_head,
                    const float *device_q, size_t q_stride, float *device_out, size_t out_stride, float scale,
                    size_t window, size_t sinks, int weights, float decay, void *stream);

/* Every sequence of more than `keep` positions is cut to `keep` of them, per layer (n_layers from first_layer on) and
 * key-value head: the first `first`, the last `recent` (first + recent <= keep) and of those between them the ones of
 * the largest device_w (NaN counts as largest, ties go to the lower position).  What stays moves together in its order
 * to positions 0 .. keep - 1 of the blocks of device_dst_tables (dst_stride entries a sequence), K, V and weights
 * alike, and device_new_lens[b] (may be device_lens itself) becomes min(length, keep).  device_dst_tables NULL or
 * device_tables itself: in place.  Otherwise sequences that need no cut are copied as they are, and the destination's
 * blocks must be none that any of the call's sequences reads.  In place, sequences must not share blocks.  Rows behind
 * the new lengths are left as they are, and so is the new place of a position that stays though its block is not there: it is one of the
 * sequence's positions from then on.  device_starts is not looked at.  Uses the executor's workspace: a word a layer, key-value head and
 * position that may stay, sequences in parts as above. */
int lnh_kv_evict_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t first_layer,
                        size_t n_layers, size_t keep, size_t first, size_t recent, const uint32_t *device_dst_tables,
                        size_t dst_stride, uint32_t *device_new_lens, void *stream);

#ifdef __cplusplus
}
#endif
#endif
