/*
 * mimo_moe_paged.h — C ABI of serving many requests over a paged KV cache (same library, libmimo_moe.so; error
 * codes and conventions of mimo_moe.h): the decoder layer's cache operators of mimo_moe_layer.h for a batch of
 * requests of different lengths, with every length on the device.
 *
 * A step brings new_lens[r] >= 0 new tokens of each of R requests that hold lens[r] tokens already.  The step's token
 * rows are the requests' new tokens, one request after another; rows behind the last request's are padding, which
 * no entry point reads or writes (a CUDA graph keeps its row count while the lengths change).
 *
 * Paged KV cache of a layer: k_pages bf16 [num_pages][n_kv_heads][page_size][head_dim], v_pages bf16
 * [num_pages][n_kv_heads][page_size][v_head_dim]; page_size 16, 32, 64 or 128 tokens.  block_table int32
 * [R][table_width]: entry j of row r is the page of the positions j * page_size .. of request r, or -1.  A token's
 * cache slot is page * page_size + position % page_size.  All layers share one table: a page number names the same
 * positions in every layer's pool.
 *
 * A step has at most 2^30 token rows, and an attention call 2^30 work units (below).  Every pointer is a device pointer,
 * 16-byte aligned where it holds bf16 values.  Errors that the kernels find in device data (MIMO_ERANGE: no free page left, a length outside the table, a page outside the pool) go to the
 * optional status word; no device value makes a kernel read or write outside the arrays it is given.
 */
#ifndef MIMO_MOE_PAGED_H
#define MIMO_MOE_PAGED_H

#include "mimo_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Plan of one step, from the lengths on the device (R <= 4096 requests):
 *   cu_q [R + 1]       row offsets: request r has the rows cu_q[r] .. cu_q[r + 1] - 1
 *   seq_lens [R]       lens + new_lens
 *   positions [tokens] absolute position of each row's token, -1 for padding rows
 *   slots [tokens]     its cache slot, -1 for padding rows
 *   block_table        entries ceil(lens / page_size) .. ceil(seq_lens / page_size) - 1 of each row are set to pages
 *                      taken from the end of the free list (in row order, the first new page is
 *                      free_pages[n_free - 1], the next free_pages[n_free - 2], ...); other entries stay
 *   n_free_out         pages left
 * All or nothing: when the pages do not suffice, a length is negative or longer than the table row, or the rows are
 * more than `tokens`, status becomes MIMO_ERANGE and the outputs are those of a step without new tokens.  The inputs
 * lens and n_free stay as they are (seq_lens and n_free_out must not alias them), so a plan may be made again. */
int mimo_moe_page_plan(const int32_t* lens, const int32_t* new_lens, int32_t R, int32_t* block_table,
                       int32_t table_width, const int32_t* free_pages, const int32_t* n_free, int32_t num_pages,
                       int32_t page_size, int32_t tokens, int32_t* cu_q, int32_t* seq_lens, int32_t* n_free_out,
                       int32_t* positions, int32_t* slots, int32_t* status, void* stream);

/* Returns the pages of the requests with done[r] != 0 to the free list (in row order, behind its last entry), empties
 * their table rows (-1 in the entries they used) and sets their lens to 0.  All or nothing, as above (MIMO_ERANGE:
 * a length outside the table, a page outside the pool, more pages than the pool has).  The pages of different rows
 * must be distinct. */
int mimo_moe_page_release(const uint8_t* done, int32_t R, int32_t* lens, int32_t* block_table, int32_t table_width,
                          int32_t* free_pages, int32_t* n_free, int32_t num_pages, int32_t page_size,
                          int32_t* status, void* stream);

/* mimo_moe_layer_rope_store with a position and a cache slot per token row: RoPE of row t's q and k heads at
 * positions[t], v * v_scale (when > 0), q to q[t], k and v to slot slots[t] of every kv head.  Rows with a negative
 * slot are left out (their q rows stay as they were); the others have a slot each (two rows of one slot: either's k
 * and v, or parts of both); a slot outside the pool sets MIMO_ERANGE and the row's k and v
 * are not stored.  rotary_dim <= 256. */
int mimo_moe_paged_rope_store(const uint16_t* qkv, int32_t tokens, int32_t n_heads, int32_t n_kv_heads,
                              int32_t head_dim, int32_t v_head_dim, int32_t rotary_dim, float rope_theta,
                              float v_scale, const int32_t* positions, const int32_t* slots, int32_t num_pages,
                              int32_t page_size, uint16_t* q, uint16_t* k_pages, uint16_t* v_pages, int32_t* status,
                              void* stream);
/* The same, and the rows of `clear` (bf16 [tokens][clear_width], clear_width a multiple of 8) whose slot is negative
 * become zero: for the `out` of the attention that follows, which leaves padding rows as they are, when all of its rows
 * go on into the layer.  clear may be null. */
int mimo_moe_paged_rope_store_clear(const uint16_t* qkv, int32_t tokens, int32_t n_heads, int32_t n_kv_heads,
                                    int32_t head_dim, int32_t v_head_dim, int32_t rotary_dim, float rope_theta,
                                    float v_scale, const int32_t* positions, const int32_t* slots, int32_t num_pages,
                                    int32_t page_size, uint16_t* q, uint16_t* k_pages, uint16_t* v_pages,
                                    uint16_t* clear, int32_t clear_width, int32_t* status, void* stream);

/* Attention of the step's new tokens over the paged cache (k and v of the new tokens already stored): row
 * cu_q[r] + i of request r is the query at position p = seq_lens[r] - (cu_q[r + 1] - cu_q[r]) + i and sees the key
 * positions j <= p; with window > 0 only those with j > p - window or j < keep_first (the first keep_first tokens of
 * every request stay visible).  Softmax over scale * q.k_j, plus the logit sinks[h] without a value row when sinks is
 * not null.  q bf16 [tokens][n_heads][head_dim], out bf16 [tokens][n_heads][v_head_dim]; (head_dim, v_head_dim) in
 * {(192,128), (128,128), (64,64)}; n_heads / n_kv_heads <= 128.  Cache slots that no query of the call sees may hold
 * anything, NaN included, and table entries of such pages are not read; what one query of a request sees must be finite
 * in v, also for the queries before it, and below 2^40 in magnitude (a row's exponentials, before they are divided by
 * their sum, may be as large as 2^60).
 *
 * It takes two calls.  The plan deals the step's work (units of one kv head of some consecutive tokens of a request) to
 * the SMs from its lengths; it holds for all layers with the
 * same heads, window and keep_first (a caller-owned buffer, 16-byte aligned, of ..._plan_bytes).  A request whose
 * lengths do not fit (more rows than positions, more positions than its table row, rows outside `tokens`) sets
 * MIMO_ERANGE and gets no output.  The attention must be given the arguments that its plan was made with (otherwise
 * status becomes MIMO_ERANGE and nothing is computed) on the same GPU; a page outside the pool sets MIMO_ERANGE and
 * reads as zeros.  workspace: ..._workspace_bytes, for one call at a time; out and workspace are
 * 32-byte aligned. */
size_t mimo_moe_paged_attention_plan_bytes(int32_t tokens, int32_t R, int32_t n_heads, int32_t n_kv_heads);
int mimo_moe_paged_attention_plan(const int32_t* cu_q, const int32_t* seq_lens, int32_t R, int32_t tokens,
                                  int32_t n_heads, int32_t n_kv_heads, int32_t window, int32_t keep_first,
                                  int32_t table_width, int32_t page_size, void* plan, size_t plan_bytes,
                                  int32_t* status, void* stream);
size_t mimo_moe_paged_attention_workspace_bytes(int32_t tokens, int32_t R, int32_t n_heads, int32_t n_kv_heads,
                                                int32_t v_head_dim);
int mimo_moe_paged_attention(const uint16_t* q, const uint16_t* k_pages, const uint16_t* v_pages, const float* sinks,
                             const int32_t* block_table, int32_t table_width, int32_t R, int32_t tokens,
                             int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t v_head_dim, float scale,
                             int32_t window, int32_t keep_first, int32_t num_pages, int32_t page_size,
                             const void* plan, size_t plan_bytes, uint16_t* out, void* workspace,
                             size_t workspace_bytes, int32_t* status, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MIMO_MOE_PAGED_H */
