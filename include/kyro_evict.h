/*
 * kyro_evict.h — caches that keep the tokens attention uses.
 *
 *   kyro_attn_weights  adds up, for every cached token and kv head, the softmax weight that a step's
 *                      query rows give it
 *   kyro_kv_evict      cuts caches longer than a budget down to it: each kv head keeps its first and its
 *                      newest tokens and those of the most weight, moved together into the front slots
 *
 * No counterpart in the reference, whose caches only grow (src/model/kv_cache.rs:49-75); both work on the
 * block-table cache of kyro_paged_attention_mq. Attention does not depend on the order of cached tokens,
 * so the moved ones need no particular slot: a slot whose token goes takes a token from behind the
 * budget, and every other one stays where it is.
 *
 * State, kept by the caller beside each layer's cache and handed from call to call:
 *   weights   [num_state_rows, Hkv, max_tokens] f32    accumulated weight of the token in each slot
 *   positions [num_state_rows, Hkv, max_tokens] int32  its position in the sequence
 * Slot t of kv head h of sequence b is entry [r][h][t] with r = state_rows[b] (NULL: r = b). Two sequences
 * of a call may not name the same row. After an eviction a token's slot differs between kv heads and is
 * no longer its position: rows appended from then on are rotated by positions of their own
 * (kyro_qkv_append's positions). Entries behind a sequence's tokens are not read or written.
 *
 * Both calls take scratch from the context's arena, as attention does: captured into HIP graphs, the calls of one
 * context run in order, one replay after the other.
 */
#ifndef KYRO_EVICT_H
#define KYRO_EVICT_H

#include <stddef.h>
#include <stdint.h>

#include "kyro_verify.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kyro_attn_weights_params {
    int32_t block_size;          /* tokens per KV block */
    int32_t num_heads;           /* query heads H */
    int32_t head_dim;            /* D: a multiple of 8, at most 256 */
    int32_t num_kv_heads;        /* Hkv; H % Hkv == 0; query head h reads kv head h / (H/Hkv) */
    int32_t batch_size;          /* B */
    int32_t total_q;             /* rows of query: B when q_start_loc is NULL */
    int32_t max_blocks_per_seq;  /* width of block_table */
    int32_t num_blocks;          /* leading dim of the cache */
    int32_t dtype;               /* kyro_dtype of query and key_cache */
    int32_t causal;              /* as for kyro_paged_attention_mq */
    float scale;                 /* >= 0; 0 => 1/sqrt(head_dim) */
    int32_t max_q_len;           /* upper bound on query rows per sequence; 0 => 1 without q_start_loc,
                                    total_q with it */
    int32_t num_state_rows;      /* leading dim of weights and positions */
    int32_t max_tokens;          /* their last dim; a context longer than it latches KYRO_EINVAL */
} kyro_attn_weights_params;

/*
 * For every sequence b, kv head h and cached token t < context_lens[b]:
 *   out_weights[r][h][t] = (t is new ? 0 : weights[r][h][t])
 *                          + sum over the sequence's rows j and the query heads g of kv head h of
 *                            softmax_t(scale * query[j][g] . key[t]) over the tokens row j sees
 * The new tokens are the sequence's last q_len, which the step has appended: their entries start at 0
 * whatever they held (a rejected draft's), and positions[r][h][t] becomes row_positions[row] (NULL: t). A
 * row that sees no token (of a context shorter than its rows, or empty as in a padded batch), or scores each it
 * sees -infinity, adds nothing. A sequence without rows keeps its weights and positions: out_weights gets its
 * weights as they are. Every row of the call weighs: after a verify step that may reject drafts, call it once
 * acceptance is known, with the query rows that stay (and their q_start_loc) and the context lengths that stay,
 * or older tokens keep the weight that rejected rows gave them. Sums and softmax are held in 32 bits; results do
 * not depend on the order of execution. out_weights may be weights itself; otherwise they do not overlap.
 *   query [total_q, H, D] dtype, q_start_loc, key_cache, block_table, context_lens: as for
 *     kyro_paged_attention_mq, after kyro_paged_kv_append or kyro_qkv_append has written the rows
 *   row_positions [total_q] int64 or NULL, state_rows [B] int32 or NULL (then B <= num_state_rows)
 * query and key_cache are on 16-byte boundaries. A bad block id, context length, q_start_loc or state row
 * latches KYRO_EINVAL for the next kyro_sync; a sequence with a bad context length, q_start_loc or state row
 * is left out, a bad block's tokens count as not seen.
 */
int kyro_attn_weights(kyro_ctx ctx, const kyro_attn_weights_params* params, const void* query,
                      const int32_t* q_start_loc, const int64_t* row_positions, const void* key_cache,
                      const int64_t* block_table, const int64_t* context_lens, const int32_t* state_rows,
                      const float* weights, float* out_weights, int32_t* positions);

/* Scratch bytes such a call takes from the context's arena (kyro_ctx_reserve). Host only; ctx may be
 * NULL, which sizes for a 256-CU device. */
int kyro_attn_weights_workspace(kyro_ctx ctx, const kyro_attn_weights_params* params, int has_q_start_loc,
                                size_t* bytes);

typedef struct kyro_kv_evict_params {
    int32_t block_size;
    int32_t num_kv_heads;
    int32_t head_dim;            /* D: a multiple of 8, at most 256 */
    int32_t batch_size;
    int32_t max_blocks_per_seq;  /* width of block_table */
    int32_t num_blocks;          /* leading dim of the caches */
    int32_t dtype;               /* kyro_dtype of the caches */
    int32_t budget;              /* tokens each kv head keeps, > 0 */
    int32_t sink;                /* tokens at positions < sink are kept, */
    int32_t recent;              /* and those at positions > newest - recent; sink + recent <= budget */
    int32_t num_state_rows;
    int32_t max_tokens;
} kyro_kv_evict_params;

/*
 * For every sequence b of n = context_lens[b] > budget tokens and every kv head on its own: ranks the
 * tokens by (position < sink or position > newest - recent, where newest is the head's largest position;
 * then weight; then the lower slot), keeps the first `budget` of them, and moves those in slots >= budget,
 * in ascending order, into the slots < budget whose token goes, in ascending order. K, V, weight and
 * position move together; a NaN weight ranks as -infinity. out_context_lens[b] = min(n, budget); shorter
 * sequences stay as they are.
 *   key_cache, value_cache [num_blocks, Hkv, block_size, D] dtype, written in place
 *   out_weights, out_positions: the kept entries [r][h][0, min(n, budget)); each may be its input itself
 *     and overlaps no input otherwise. The inputs' own entries then stay, so that a call can be repeated:
 *     the caches' slots >= budget are not written
 *   context_lens, out_context_lens [B] int64, not overlapping
 * A block that holds any of a sequence's first `budget` slots must be in no other table and twice in none
 * (kyro_bm_make_private_front of the budget sees to it). Afterwards the blocks behind the budget may be released
 * (kyro_bm_truncate). Caches are on 16-byte boundaries. A bad block id, context length or state row latches
 * KYRO_EINVAL for the next kyro_sync, and that sequence is left as it is.
 */
int kyro_kv_evict(kyro_ctx ctx, const kyro_kv_evict_params* params, void* key_cache, void* value_cache,
                  const int64_t* block_table, const int64_t* context_lens, const int32_t* state_rows,
                  const float* weights, const int32_t* positions, float* out_weights, int32_t* out_positions,
                  int64_t* out_context_lens);

/* Scratch bytes such a call takes from the context's arena (kyro_ctx_reserve). Host only. */
int kyro_kv_evict_workspace(const kyro_kv_evict_params* params, size_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* KYRO_EVICT_H */
