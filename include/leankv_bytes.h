/*
 * leankv_bytes — C ABI of the paged cache that holds keys and values in 8 bits, and of the attention over it
 * (libleankv_bytes.so, sm_100a). The reference project has no cache of this kind: its paged cache keeps fp16 pages
 * (leankv/turboquant/paged_cache.py) and its quantized one 3-bit codes (leankv/turboquant/cache.py). Conventions (device
 * pointers, ownership, streams, status codes, page table) are those of leankv_b200.h.
 *
 * Format. A block is the 16 tokens of a page, of one kv head, keys or values. It has one scale 2^e, e the smallest whole number >= -126
 * with |x| <= 127 * 2^e for all numbers x of the block, and codes rint(x * 2^-e), half to even. A token that joins a
 * block may raise e; the codes that are there become rint(code * 2^(e_old - e)). A block that is opened anew (its first token is
 * written) starts without a scale. Powers of two make x * 2^-e exact, so that the codes are the same in every precision and order
 * of work. An infinity, a NaN or a magnitude of 2^126 or more makes the block's scale NaN and with it the answer of every query
 * that sees the block.
 */
#ifndef LEANKV_BYTES_H
#define LEANKV_BYTES_H

#include "leankv_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LEANKV_BYTES_F16 0
#define LEANKV_BYTES_BF16 1
#define LEANKV_BYTES_F32 2
#define LEANKV_BYTES_MAX_BATCH 1024
#define LEANKV_BYTES_MAX_GROUP 16

/* One layer's pages. `dim` is 64 or 128. Both arrays 16-byte aligned; a zero-filled pool is a valid empty one.
 *   chunks  [n_pages][kv_heads][leankv_byte_chunk_bytes(dim)]   keys, values (16 * dim codes each, stored as code + 128), the two
 *           scales (fp32), 8 bytes of padding
 *   bounds  [n_pages][kv_heads][leankv_byte_bounds_bytes(dim)]  the largest and the smallest key code of each channel among the block's
 *           tokens (int8), the keys' scale, 12 bytes of padding */
typedef struct {
    int dim, kv_heads, n_pages;
    void* chunks;
    void* bounds;
} leankv_byte_pool_t;

/* Vectors of `dim` numbers, one of them contiguous and 16-byte aligned; elements from a sequence, a head, a token to the next
 * (multiples of 16 bytes). A stride of an extent of one is not used. */
typedef struct {
    void* data;
    long long seq, head, token;
} leankv_vectors_t;

size_t leankv_byte_chunk_bytes(int dim);
size_t leankv_byte_bounds_bytes(int dim);

/* `tokens` new tokens of `batch` sequences (k, v of `dtype`) become the last ones of each: the page table has been advanced already
 * (leankv_paged_table_step). Sequence b owns the pages kv_page_indices[kv_indptr[b]] .. ; a page id outside 0 .. n_pages - 1 is
 * not written, nor is a sequence of fewer tokens. batch <= LEANKV_BYTES_MAX_BATCH. */
typedef struct {
    leankv_byte_pool_t pool;
    int dtype, batch, tokens;
    leankv_vectors_t k, v;
    const int32_t* kv_indptr;
    const int32_t* kv_page_indices;
    const int32_t* kv_last_page_len;
} leankv_byte_append_t;
int leankv_byte_append(const leankv_byte_append_t* a /* host */, void* stream);

/* The stored numbers of the first T positions of B sequences, as `dtype`: k_out, v_out [B][kv_heads][T][dim], zeros behind a sequence's
 * last token; 16-byte aligned, fp32 32-byte. A number beyond the type's range becomes its largest one. */
int leankv_byte_unpack(const leankv_byte_pool_t* pool /* host */, int dtype, void* k_out, void* v_out, int B, int T,
                       const int32_t* kv_indptr, const int32_t* kv_page_indices, const int32_t* kv_last_page_len, void* stream);

/* Attention of the last `tokens` tokens of each of `batch` sequences over the cache, causal among themselves: q_heads / kv_heads (up to
 * LEANKV_BYTES_MAX_GROUP) query heads share a kv head; q and out of `dtype`. Softmax statistics and sums are fp32. A sequence
 * without tokens (kv_indptr[b + 1] <= kv_indptr[b]), and a query before the first token, gets zeros. A weight is rounded by 2^-35 of the
 * row's largest weight, or by 2^-21 of itself where that is more.
 * max_pages_seq, total_pages: upper bounds of any sequence's pages and of all sequences' together, for the launch's shape.
 * block_pages = NULL: every page. Else (tokens = 1) the pages of sequence b and kv head h are block_pages[(b * kv_heads + h) * n_blocks ..], as
 * many as there are blocks or n_blocks, the last of them the sequence's last page (leankv_byte_select writes such lists).
 * The workspace is zero-filled once; its first word is a status (0 = clean; leankv_byte_status): bit 0 a bounded wait ran out, bit 1 a page
 * id outside the pool, bit 2 more pages than total_pages (nothing was written). The launches of two streams need a workspace each. */
typedef struct {
    leankv_byte_pool_t pool;
    int dtype, batch, q_heads, tokens;
    leankv_vectors_t q, out;
    float scale;
    const int32_t* kv_indptr;
    const int32_t* kv_page_indices;
    const int32_t* kv_last_page_len;
    int max_pages_seq;
    long long total_pages;
    const int32_t* block_pages;
    int n_blocks;
    void* workspace;
    size_t workspace_bytes;
} leankv_byte_attn_t;
size_t leankv_byte_attn_workspace_bytes(void);       /* the same for all shapes */
int leankv_byte_attn(const leankv_byte_attn_t* a /* host */, void* stream);
/* The same for longer chunks of prompts, on tcgen05 (256 (token, head) rows against 128 keys at a time); q and out fp16 or bf16 (fp32:
 * LEANKV_EUNSUPPORTED), scale > 0, block_pages NULL. Each term of a row's output (weight times value) is rounded by 2^-11 of itself at most, where
 * leankv_byte_attn keeps 21 bits, or by 2^-24 of its largest weight times the largest number of that token's block where that is more; blocks that a
 * row does not see have no part in it. */
int leankv_byte_prompt_attn(const leankv_byte_attn_t* a /* host */, void* stream);

/* The blocks that one query token of each sequence reads, for each kv head: all of them where there are no more than n_blocks; else the
 * first `sinks`, the last `recent` (>= 1; sinks + recent <= n_blocks) and those with the largest score, ties to the lower block.
 *   i[g][d] = rint(q[g][d] * 2^-f), f the smallest whole number >= -126 with |q| <= 2047 * 2^f over the group's heads g
 *   u = sum over d of  max[d] * sum_g max(i, 0) + min[d] * sum_g min(i, 0)       (whole numbers below 2^31)
 *   score = fp32(u) * 2^e
 * an upper bound of the heads' summed scores over the block's tokens, up to the rounding of q. The score of a block whose scale is
 * NaN is larger than all others. Block numbers ascending, then -1: blocks [batch][kv_heads][n_blocks]; the page of each in block_pages
 * (0 behind the last). scores: scratch of batch * kv_heads * max_pages_seq fp32 words. */
typedef struct {
    leankv_byte_pool_t pool;
    int dtype, batch, q_heads;
    leankv_vectors_t q;
    const int32_t* kv_indptr;
    const int32_t* kv_page_indices;
    int max_pages_seq, n_blocks, sinks, recent;
    int32_t* blocks;
    int32_t* block_pages;
    float* scores;
} leankv_byte_select_t;
int leankv_byte_select(const leankv_byte_select_t* a /* host */, void* stream);

/* Host copy of a workspace's status word (synchronises). */
int leankv_byte_status(const void* workspace, int* status /* host */);

#ifdef __cplusplus
}
#endif
#endif
