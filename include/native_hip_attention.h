/* native-hip: operators over a paged key-value cache in device memory - storing the rows of new tokens, with the rotation by
 * their positions on the way if wanted, attention that reads the cache, eviction by accumulated attention weight.
 *
 * The products of native_hip.h leave q, k and v of a step in HBM; these calls are what stands between them and the
 * output projection for a caller that keeps its own cache: the reference's attention over paged K/V
 * (langtax/src/decode.rs:11126-11197, 12059-12100; langtax/src/kv_page.rs:47-53, 410-438) runs on the host and has
 * neither an f16 or a 4-bit cache, nor the window with first tokens, nor the eviction.
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
 * or, in 4 bits, LNH_TYPE_Q4_0 (LNH_ERR_UNSUPPORTED otherwise), head_dim a multiple of 8 (LNH_TYPE_Q4_0: of 32), at most 256
 * (LNH_ERR_UNSUPPORTED otherwise), at most 2^31 rows of head_dim in all.  device_w, where weights are kept:
 * [n_blocks][n_layer][n_head_kv][kv_block] f32, else NULL.
 *
 * LNH_TYPE_Q4_0: 32 elements of a row share an f16 scale d and have a code of 4 bits each; an element is (code - 8) d.  K and V
 * are each [n_blocks][n_layer][n_head_kv][kv_block][head_dim / 2] bytes of codes - eight to a little-endian word, element 2 i of
 * the eight at bit 4 i, element 2 i + 1 at bit 16 + 4 i - and behind them [n_blocks][n_layer][n_head_kv][head_dim / 32][kv_block]
 * scales, 18 bytes for 32 elements in all.  Stored rows have d = -1/8 of the element of the largest size (the first of those),
 * rounded to eight significant bits and to an f16, at most 8160, and the nearest codes, ties to even: every element is then an
 * f16, and what the operators make of such a cache is what they make of an f16 cache of these values.  Larger numbers than 65280
 * are held to it; 32 of which one is infinite or NaN are all NaN.  Scales that a caller writes itself should keep to eight bits:
 * elements are rounded to f16. */
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

/* How queries and keys are turned by their position: pair i of a head's first n_rot elements (even, at most head_dim; 0: none is turned),
 * (x, y) -> (x c - y s, x s + y c) with (c, s) the pair at device_angles + 2 * (position * angle_stride + i) (floats, 8-byte
 * aligned; angle_stride in pairs).  Pairs are elements 2 i and 2 i + 1, or, with halves != 0, i and i + n_rot / 2.  A token's
 * position is its place in its sequence or, where device_positions is not NULL, device_positions[row]; a position that is not
 * below n_positions takes the last one's angles. */
typedef struct lnh_rope {
    const float *device_angles;
    size_t angle_stride, n_positions;
    uint32_t n_rot;
    int halves;
    const uint32_t *device_positions;
} lnh_rope;

/* The angles' cosines and sines of positions 0 .. n_positions - 1: pair i of n_rot / 2 turns by position * scale * base^(-2 i / n_rot),
 * divided by device_divisors[i] where those are not NULL; formed in 64 bits, rounded to f32.  base and scale positive. */
int lnh_rope_table_device(lnh_exec *exec, uint32_t n_rot, double base, double scale, const float *device_divisors, size_t n_positions,
                          float *device_angles, size_t angle_stride, void *stream);

/* lnh_kv_store_device with the rotation on the way: rows of device_q (n_head heads; n_head 0: none, device_q and device_q_out are not
 * looked at) are turned into device_q_out (may be device_q itself, of the same stride), rows of device_k into K; V as it is.  rope
 * NULL: nothing is turned.  Numbers are turned in 64 bits and rounded to f32, then to the cache's type.  Where the cache keeps
 * weights, those of the new positions become zero.  A new token below position 0 keeps its row of device_q_out as it was. */
int lnh_kv_append_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t layer, const lnh_rope *rope, size_t n_head,
                         const float *device_q, size_t q_stride, float *device_q_out, size_t q_out_stride, const float *device_k,
                         size_t k_stride, const float *device_v, size_t v_stride, void *stream);

/* What `layer` of the cache has for the new tokens, as f32 rows: lnh_kv_store_device's way back, for a prefix that goes to another cache or
 * program.  A new token that stands nowhere (below position 0, or in a block that is not there) gets zeros. */
int lnh_kv_load_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t layer, float *device_k, size_t k_stride,
                       float *device_v, size_t v_stride, void *stream);

/* out = softmax(scale q K^T) V for every new token and each of n_head query heads (a multiple of n_head_kv; query
 * head h reads key-value head h * n_head_kv / n_head; 0 < scale <= 2^127), over `layer` of the cache: the new tokens' own rows have to be
 * stored before.  The token at position p sees position t where t <= p and, with window > 0, p - t < window or
 * t < sinks (sinks without a window: LNH_ERR_INVALID).  Rows of q and out are n_head * head_dim floats, strides in
 * floats.  A token that sees nothing gets zeros; so does one whose every score is -infinity.  What lies in positions
 * that a token does not see, infinities and NaN among it, does not reach its row.
 * Scores, the softmax and the sums are f32; over an f16 or a 4-bit cache q and the probabilities enter the matrix cores as two
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

/* What the keys of a block of the cache lie between: the least and the largest value of each key element over the positions that the
 * sequence has in the block, as device_bounds [n_blocks][n_layer][n_head_kv][2][head_dim] (16-byte aligned), f32 for an f32 cache, else f16:
 * exactly numbers of the cache.  Formed anew, in `layer`, for every block that holds new tokens of the call, whose rows have to be
 * stored before; a NaN among the values makes both bounds NaN.  Blocks that are not there are left out.  Bounds hold as long as the rows of
 * their block do: lnh_kv_evict_device moves rows to other blocks, and lnh_kv_bounds_device forms the bounds of the whole sequences again where
 * every position counts as new - device_starts the running sum of the lengths, max_new = max_len, n_tokens at least the last start. */
int lnh_kv_bounds_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t layer, void *device_bounds, void *stream);

/* lnh_attn_device over n_select blocks of the cache for each new token and key-value head, those that device_bounds (lnh_kv_bounds_device, of all
 * blocks that the token sees whole) promise most of.  A block's score is the largest, over the query heads that share the key-value
 * head, of the sum over the head's elements of q hi where q > 0 and q lo elsewhere - at least every product q k of the block -, formed
 * in 64 bits and rounded to f32 (NaN counts as largest, a block that is not there as least).  A token at position p reads
 * the positions up to p of the first `first` of its p / kv_block + 1 blocks, of the last `recent` (at least one, its own;
 * first + recent <= n_select) and of those between them the ones of the largest score, ties to the lower; of all where they are
 * no more than n_select.  device_chosen (may be NULL): which, [n_tokens][n_head_kv][n_select] in ascending order, 0xffffffff behind
 * the last; rows that belong to no sequence are left as they are.  Otherwise as lnh_attn_device without window and weights, also in what it
 * does with the executor's workspace: a word for every block of max_len, new token and key-value head, tokens in parts where that
 * would pass 1 GiB or a launch's workgroups.  A prompt of thousands of tokens may take longer so than by lnh_attn_device, whose tokens share what they read. */
int lnh_attn_select_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t layer, size_t n_head, const void *device_bounds,
                           size_t n_select, size_t first, size_t recent, const float *device_q, size_t q_stride, float *device_out,
                           size_t out_stride, float scale, uint32_t *device_chosen, void *stream);

/* Every sequence of more than `keep` positions is cut to `keep` of them, per layer (n_layers from first_layer on) and
 * key-value head: the first `first`, the last `recent` (first + recent <= keep) and of those between them the ones of
 * the largest device_w (NaN counts as largest, ties go to the lower position).  What stays moves together in its order
 * to positions 0 .. keep - 1 of the blocks of device_dst_tables (dst_stride entries a sequence), K, V and weights
 * alike, and device_new_lens[b] (may be device_lens itself) becomes min(length, keep).  device_dst_tables NULL or
 * device_tables itself: in place.  Otherwise sequences that need no cut are copied as they are, and the destination's
 * blocks must be none that any of the call's sequences reads.  In place, sequences must not share blocks.  Rows behind
 * the new lengths are left as they are, and so is the new place of a position that stays though its block is not there: it is one of the
 * sequence's positions from then on.  device_starts is not looked at.  Bounds (lnh_kv_bounds_device) of the blocks that it writes to hold no longer.  Uses
 * the executor's workspace: a word a layer, key-value head and position that may stay, sequences in parts as above. */
int lnh_kv_evict_device(lnh_exec *exec, const lnh_kv_cache *cache, const lnh_kv_seqs *seqs, size_t first_layer,
                        size_t n_layers, size_t keep, size_t first, size_t recent, const uint32_t *device_dst_tables,
                        size_t dst_stride, uint32_t *device_new_lens, void *stream);

#ifdef __cplusplus
}
#endif
#endif
