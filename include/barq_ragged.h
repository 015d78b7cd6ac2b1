/*
 * barq_ragged.h -- C ABI of libbarq_kv.so for ragged batches and drafted trees over the page pool of
 * barq_kv.h: block tables and slot maps built on the device from the requests' lengths, stores through a
 * slot map, and attention of a tree of drafted tokens over a row's pages.
 *
 * The conventions of barq_kv.h hold: device pointers, sizes and a HIP stream (NULL = the null stream); every
 * call enqueues its work, allocates no device memory, never synchronises with the host and returns a
 * BARQ_KV_* status; calls that name one pool are ordered on one stream.  No counterpart in the reference,
 * which appends equal numbers of tokens to every row and attends over a gathered cache.
 */
#ifndef BARQ_RAGGED_H
#define BARQ_RAGGED_H

#include <stdint.h>

#include "barq_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Request i, for i in [0, num_rows), appends lengths[i] >= 0 tokens to row rows[i] (rows NULL: row i) of
 * each of num_pools pools (a model's layers; distinct pools of one max_batch, max_blocks and page_size).
 * rows and lengths are HOST arrays, the rows distinct and in [0, max_batch); everything else is read on the
 * device when the launch runs.  The tokens are packed: token j of request i is number offsets[i] + j, where
 * offsets counts the tokens of the requests before.  It takes position seq_lens[row] + j of its row and
 * slot page * page_size + position % page_size of the pool, where page is the row's block position /
 * page_size: mapped already, or a page from the free stack, which the new blocks take in (request, block)
 * order.  Afterwards seq_lens[row] += lengths[i] and high_water[row] = max(high_water[row],
 * seq_lens[row]), as barq_kv_append leaves them: the caller stores the tokens (barq_write_slots, or a
 * kernel of its own) before it reads them.
 *   slots     : device int64, pool l's at slots + l * slot_stride, total = sum of lengths each; -1 for a
 *               token that found no page (BARQ_KV_ERRBIT_POOL_EXHAUSTED) or passes the row's blocks
 *               (BARQ_KV_ERRBIT_CAPACITY)
 *   positions : device int32 [total], the tokens' positions in the first pool's rows, or NULL
 *   requests  : device int32 [total], the tokens' requests, or NULL
 *   offsets   : device int32 [num_rows + 1], or NULL
 * total < 2^30.  One launch for each 256 requests of 32 pools.
 */
int barq_map_slots(const barq_kv_pool* pools, int64_t num_pools, const int32_t* rows, const int32_t* lengths,
                   int64_t num_rows, int64_t* slots, int64_t slot_stride, int32_t* positions, int32_t* requests,
                   int32_t* offsets, void* stream);

/*
 * Store token index[j] (index NULL: token j) of key / value in slot slots[j] of the pool, for j in
 * [0, count).  key / value: [num_tokens, kv_heads, head_dim] elements of elem_bytes, element strides
 * (stride_n, stride_h), contiguous last dimension.  slots and index are device int64; a negative slot is
 * passed over, a slot past the pool or an index outside [0, num_tokens) too, and flagged
 * (BARQ_KV_ERRBIT_BAD_INDEX).  Two tokens of one slot: either is stored.
 */
int barq_write_slots(const barq_kv_pool* pool, const int64_t* slots, const int64_t* index, int64_t count,
                     const void* key, const void* value, int64_t num_tokens, int64_t stride_n, int64_t stride_h,
                     void* stream);

/* Most nodes of a tree. */
#define BARQ_TREE_MAX_NODES 256

/*
 * Attention of T drafted tokens a row, the nodes of a tree, over the row's cached positions and over the
 * tree's own nodes, whose keys and values are arguments and not in the pool:
 *   out[b, h, i, :] = sum_x softmax_x(scale * q[b, h, i, :] . K_x) V_x
 * over the cached positions p < seq_lens[b] and the nodes j that mask[b, i, j] is not 0 for; h reads KV head
 * h / G, G = q_heads / kv_heads.  A node that sees nothing gets zeros, and what a node does not see takes no
 * part, whatever it holds.
 *   pool       : 2-byte elements (bf16, or fp16 with BARQ_KV_ATTN_FP16), head_dim D of 64, 128 or 256
 *   cold       : NULL, or the pool's cold store (D 64 or 128, page_size a multiple of 16, its element type
 *                the flags'; codes and key scales at multiples of 16 bytes): quantised blocks are read as their
 *                codes, as barq_kv_gather_cold gives them (a scale byte of 255 is a NaN)
 *   query      : [batch, q_heads, T, D], element strides q_stride_*
 *   node_key, node_value : [batch, kv_heads, T, D], element strides node_stride_* of both
 *   mask       : bytes [batch, T, T], strides mask_stride_* (0 for what is shared), or NULL: node i sees
 *                nodes 0 .. i (a chain)
 *   out        : [batch, q_heads, T, D] of the pool's type, or float32 with BARQ_KV_ATTN_OUT_F32; element
 *                strides out_stride_*
 * Addresses and strides of query and nodes are multiples of 16 bytes, of out multiples of 4 elements.
 * 1 <= T <= BARQ_TREE_MAX_NODES.  max_seq bounds every row's length (0: the pool's capacity; a longer row
 * is read up to it and flagged, BARQ_KV_ERRBIT_ATTN_SHORT); mean_seq, if not 0, is the rows' mean length as
 * far as the caller knows it and only guides the split of long rows.  workspace: device memory of
 * barq_tree_attention_workspace_bytes(the same arguments) bytes, 16-byte aligned, no initialisation
 * needed; launches that share it must not overlap.  A block naming no page reads page 0 and is flagged
 * (BARQ_KV_ERRBIT_BAD_INDEX).
 */
int barq_tree_attention(const barq_kv_pool* pool, const barq_kv_cold* cold, const void* query, int64_t batch,
                        int64_t q_heads, int64_t nodes, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                        const void* node_key, const void* node_value, int64_t node_stride_b, int64_t node_stride_h,
                        int64_t node_stride_t, const uint8_t* mask, int64_t mask_stride_b, int64_t mask_stride_i,
                        int64_t mask_stride_j, void* out, int64_t out_stride_b, int64_t out_stride_h,
                        int64_t out_stride_t, float scale, int64_t max_seq, int64_t mean_seq, int64_t flags,
                        void* workspace, int64_t workspace_bytes, void* stream);

/* Bytes of workspace barq_tree_attention needs (0: none; cold: whether it is given one), or -1 for arguments it rejects. */
int64_t barq_tree_attention_workspace_bytes(const barq_kv_pool* pool, int64_t cold, int64_t batch, int64_t q_heads,
                                            int64_t nodes, int64_t max_seq, int64_t mean_seq);

#ifdef __cplusplus
}
#endif

#endif /* BARQ_RAGGED_H */
