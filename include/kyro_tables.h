/*
 * kyro_tables.h — block tables, row ranges and cache slots of a step, built on the GPU from what each request
 * holds, with a pool of free blocks that lives there too.
 *
 *   kyro_tables_extend   room for each request's new rows: blocks from the pool, and everything that
 *                        kyro_qkv_append, kyro_paged_kv_append and kyro_paged_attention_mq read of the step
 *   kyro_tables_keep     after acceptance: the rows that stay count, the blocks behind them go back to the pool
 *   kyro_tables_release  requests that end give their blocks back
 *
 * kyro_bm_append_slots, kyro_bm_truncate and kyro_bm_write_tables do the same from the host, which then has to
 * wait for the accepted lengths that kyro_spec_verify leaves on the device in every step. Here nothing of a step
 * passes through the host, so steps can follow each other without a synchronisation, or as a captured graph.
 * The host hands a block manager's blocks to a pool in bulk (kyro_bm_allocate) and admits and ends requests.
 *
 * State, kept by the caller (device memory) and handed from call to call:
 *   requests   [num_state_rows, 4] int32        {tokens, blocks held, blocks at the front that are not the
 *                                               pool's (a shared prefix), unused}; on a 16-byte boundary
 *   blocks     [num_state_rows, max_state_blocks] int64   ids of the blocks a request holds, in order
 *   pool       [pool_capacity] int64            ids of free blocks, a stack:
 *   pool_count [1] int32                        its first *pool_count entries
 * Entry b of a batch is request r = state_rows[b] (NULL: r = b). A negative r is padding: no request, of context
 * length 0. Two entries may not name one request. With batch_size 0 no call reads or writes anything.
 * Sums over the batch follow its order, so that results do not depend on the order of execution.
 */
#ifndef KYRO_TABLES_H
#define KYRO_TABLES_H

#include <stddef.h>
#include <stdint.h>

#include "kyro_verify.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kyro_tables_params {
    int32_t block_size;          /* tokens per block */
    int32_t batch_size;          /* B, below 2^24 */
    int32_t max_blocks_per_seq;  /* width of block_table (extend), at most 2^31 - 2048 */
    int32_t num_state_rows;      /* requests the state holds, at most 131072 */
    int32_t max_state_blocks;    /* blocks a request may hold: at most 2^31 - 2048, and below 2^31 tokens */
    int32_t num_blocks;          /* leading dim of the caches; ids outside [0, num_blocks) latch KYRO_EINVAL */
    int32_t pool_capacity;
    int32_t max_rows;            /* entries of positions and slots (extend): rows of the step */
    int32_t kept_plus;           /* added to each entry of kept (keep) */
} kyro_tables_params;

/*
 * For every entry b with request r of n = requests[r].tokens tokens and its m = new_rows[b] new ones:
 *   blocks: as many as ceil((n + m) / block_size) needs beyond those held come off the top of the pool, in the
 *     order of the batch, and are added to blocks[r]. requests[r].tokens stays: that is kyro_tables_keep's, and a
 *     call that is repeated takes no more blocks;
 *   block_table[b][0, max_blocks_per_seq): the blocks held, 0 behind them;
 *   context_lens[b] = n + m;
 *   q_start_loc [B + 1]: the sums of new_rows, from 0;
 *   positions[i], slots[i] of row i = q_start_loc[b] + j: its position n + j in the request, and its place
 *     block * block_size + offset in the caches; -1 behind the last row. Either may be NULL.
 * An entry that the pool has no blocks left for (in the order of the batch: the sum of what it and those before it
 * need exceeds *pool_count, and it needs some) gets none: context length 0, a zero row of block_table, positions and
 * slots of -1, while q_start_loc keeps its rows. It latches KYRO_ENOSPACE for the next kyro_sync, also if that comes
 * behind the rest of the step, whose appends skip its rows. So do, as
 * KYRO_EINVAL, a state row that is out of range or named twice, a request whose record is not one, a length past
 * max_state_blocks or max_blocks_per_seq, new_rows < 0 (counted as 0) and rows past max_rows.
 */
int kyro_tables_extend(kyro_ctx ctx, const kyro_tables_params* params, const int32_t* state_rows,
                       const int32_t* new_rows, int32_t* requests, int64_t* blocks, const int64_t* pool,
                       int32_t* pool_count, int64_t* block_table, int64_t* context_lens, int32_t* q_start_loc,
                       int64_t* positions, int64_t* slots);

/*
 * For every entry b of a step that kyro_tables_extend made room for (its context_lens and q_start_loc, m rows):
 *   k = kept[b] + kept_plus of its rows stay, the first ones (after kyro_spec_verify: out_accepted and 1);
 *   requests[r].tokens = context_lens[b] - m + k; blocks behind ceil(tokens / block_size) and behind the
 *   request's shared ones go back to the pool, in the order of the batch and then of the request;
 *   out_context_lens[b] = requests[r].tokens.
 * An entry without rows keeps its length, whatever kept holds. One of context length 0 (kyro_tables_extend left it
 * out, it is padding, or an empty request without rows) is left alone and gets 0. k outside [0, m], and what extend
 * refuses of state rows and records, latch KYRO_EINVAL, and the entry is left alone; so does a pool that would pass
 * its capacity, and then no block moves and no record changes. out_context_lens may be context_lens.
 */
int kyro_tables_keep(kyro_ctx ctx, const kyro_tables_params* params, const int32_t* state_rows,
                     const int64_t* context_lens, const int32_t* q_start_loc, const int32_t* kept,
                     int32_t* requests, const int64_t* blocks, int64_t* pool, int32_t* pool_count,
                     int64_t* out_context_lens);

/* Ends the batch's requests: their blocks behind the shared ones go back to the pool, as above, and their records
 * become 0. The shared ones stay whose they are. */
int kyro_tables_release(kyro_ctx ctx, const kyro_tables_params* params, const int32_t* state_rows,
                        int32_t* requests, const int64_t* blocks, int64_t* pool, int32_t* pool_count);

/* Scratch bytes that any of these calls takes from the context's arena (kyro_ctx_reserve). Host only. */
int kyro_tables_workspace(const kyro_tables_params* params, size_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* KYRO_TABLES_H */
