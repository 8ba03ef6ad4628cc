/*
 * kriya_paged.h — a key/value cache in pages that sequences share, the
 * attention that reads it (from one token per sequence to whole prompts, and
 * trees of drafted tokens), and what a server that drafts needs around it: the
 * plan of a tree and the commit of its accepted path.  It stands beside the
 * contiguous caches of kriya_glue.h (bf16, one new token per sequence) and
 * kriya_kv8.h (8 bits).  Conventions as in kriya_q4.h: device pointers unless a
 * comment says otherwise, stream-ordered, no allocation, 0 or a negative KR_E*
 * code with the message in kr_last_error(); a call that fails a check enqueues
 * nothing.  Every call can be captured into a HIP graph.
 */
#ifndef KRIYA_PAGED_H
#define KRIYA_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "kriya_kv8.h"
#include "kriya_q4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the pages ----
 * One pool of pages for all sequences (the reference's pages are of 16 tokens, bsr_paged.rs:325): `page` slots of all
 * kv heads of one layer each, bf16,
 *   k, v [layers, pages, kv_heads, page / 16, 16 * head_dim], 16-byte aligned.
 * The 16 slots of a unit stand in the order of the matrix instructions' operands (kr_paged_read reads them back):
 *   k [head_dim / 8, 16 slots, 8 dims]
 *   v [head_dim / 32, 2 (h), 32 dims, 2 (a), 4 (j)], slot 8 a + 4 h + j
 * page: 16, 32, 64, .. 4096 (a power of two); head_dim 64, 96, 128, 192 or 256; pages * kv_heads * page / 16 below 2^32.  No initial contents are needed: what lies in
 * slots without a token is never seen, whatever its bits. */
typedef struct kr_paged_cache {
    uint16_t *k, *v;
    uint32_t layers, pages, page, kv_heads, head_dim;
} kr_paged_cache;

/* A step: the sequences, their pages and their new tokens.  Page i of sequence b, its slots i page .. , is table[b, i] (u32
 * [batch, max_pages]); a value >= pages is no page: nothing is written to its slots, and no row sees them.  Sequences may share pages
 * as long as no call writes to a shared one.  max_pages * page <= 2^30.
 * lengths (u32 [batch]): tokens of each sequence, this step's included; the new tokens of sequence b are rows starts[b] ..
 * starts[b + 1] - 1 of k, v and q (u32 [batch + 1], not decreasing; a sequence may have none) and take its last slots.  starts ==
 * NULL: tokens == batch, one each.  Values beyond `tokens`, slots beyond max_pages * page and lengths below the number of new
 * tokens are cut off, never followed.  Rows before the first sequence's and behind the last's are nobody's: nothing of them is
 * appended, and their results are left as they were.  All of it stays on the device and serves every layer of a step. */
typedef struct kr_paged_step {
    const uint32_t *table;
    uint32_t max_pages, batch;
    const uint32_t *starts, *lengths;
} kr_paged_step;

/* RMS norm of each head before its rotation: x rsqrt(mean(x^2) + eps) w, the squares summed in f32, w bf16 [head_dim], at any element
 * of a tensor.  A weight may be NULL: not normalised.  (fused_qknorm_rope_and_kv_append, paged_gqa_and_deltanet.metal:115-222) */
typedef struct kr_head_norm {
    const uint16_t *q_weight, *k_weight;
    float eps;
} kr_head_norm;

/* Appends k, v (bf16 [tokens, kv_heads, head_dim], tokens kv_stride elements apart) to the pages of `layer`.  norm, rope (host
 * pointers, may be NULL): k is normalised, then rotated by the table row of its token's position (kr_rope as in kriya_kv8.h), in f32,
 * and rounded once; so is q (bf16 [tokens, q_heads, head_dim], q_stride elements apart; NULL: none) into q_out (the same stride;
 * may equal q).  q_out and the layer's pages lie apart from each other and from all else that is read; rows may lie in one another's
 * gaps (k, v and q of a fused projection).  One launch.  k, v, q, q_out 16-byte aligned, strides multiples of 8; q needs norm or rope; rope->inverse
 * must be 0. */
int kr_paged_append(const kr_paged_cache *cache, uint32_t layer, const kr_paged_step *step, const kr_head_norm *norm,
                    const kr_rope *rope, const uint16_t *k, const uint16_t *v, size_t kv_stride, const uint16_t *q,
                    uint16_t *q_out, size_t q_stride, uint32_t q_heads, uint32_t tokens, void *stream);

/* Reads slots first[b] .. first[b] + count - 1 of each sequence (first: u32 [batch], NULL for 0) into k_out, v_out [batch, count,
 * kv_heads, head_dim] of dtype (either may be NULL); slots at or beyond lengths[b], and those of no page, give zeros.  Both
 * lie apart from each other and from what is read. */
int kr_paged_read(const kr_paged_cache *cache, uint32_t layer, const kr_paged_step *step, const uint32_t *first,
                  uint32_t count, void *k_out, void *v_out, int dtype, void *stream);

/* ---- attention over the pages ----
 * For token i of the m new tokens of a sequence of n tokens, and query head g of the group of a kv head:
 *   out = sum_p softmax_p(scale q . K_p) V_p,   lse = ln sum_p e^(scale q . K_p)
 * over slots p <= n - m + i (mask == NULL), or over the slots p < n - m and those p = n - m + j, j < m, whose bit j is set in the
 * token's row of `mask` (u32 [tokens, words], bit j % 32 of word j / 32; nodes from 32 words on are not seen): a tree of drafted
 * tokens (kr_tree_plan makes its masks), a chain, or any other rule.
 *   q: bf16 [tokens, q_heads, head_dim], tokens q_stride elements apart (a multiple of 8); out: bf16, contiguous; both 16-byte
 *   aligned; out, lse and the workspace lie apart from one another and from what is read; lse f32 [tokens, q_heads] or NULL; q_heads a multiple of kv_heads; |scale| < 2^100 (may
 *   be negative or 0).
 * Products are bf16 with sums in f32; the probabilities enter the second product as bf16 (half a step is 2^-8 of each), where rows are
 * few as two of them (2^-16); maxima, sums and joins are f32, for which |scale| sum |q| |K_p| must stay below 2^125 and finite values
 * below 2^89.  A row that sees no slot gives zeros and lse = -infinity.
 * Infinities and NaN count in the rows that see them alone: such a row gives what the formula gives, an infinity or NaN.
 * workspace: kr_paged_attention_workspace_bytes(cache, step, q_heads, tokens) bytes (of step only batch and max_pages are
 * read; 0 for sizes that the call refuses), 16-byte aligned, no initial contents; calls sharing it must not overlap in time.  Results are the same bits from run
 * to run. */
size_t kr_paged_attention_workspace_bytes(const kr_paged_cache *cache, const kr_paged_step *step, uint32_t q_heads,
                                          uint32_t tokens);
int kr_paged_attention(const kr_paged_cache *cache, uint32_t layer, const kr_paged_step *step, const uint16_t *q,
                       size_t q_stride, uint32_t q_heads, uint32_t tokens, const uint32_t *mask, uint32_t words,
                       float scale, uint16_t *out, float *lse, void *workspace, size_t workspace_bytes, void *stream);

/* ---- trees of drafted tokens ----
 * The new tokens of a sequence are the nodes of its tree in an order in which parents come first: parents[t] (i32 [tokens]) is the
 * place of a node's parent among its sequence's nodes; a value that is not 0 .. its own place - 1 means that the node follows the
 * tokens before the step (node 0 does).
 *
 * The plan: mask (u32 [tokens, words]) gets the bits of a node's ancestors and its own, positions (u32 [tokens]) n - m plus the
 * number of its ancestors: the mask of kr_paged_attention and the positions of kr_rope, for every layer of the step.  starts,
 * lengths as in kr_paged_step.  words 1 .. 128; a sequence's nodes from 32 words on get no bits and position n - m.  mask and positions lie
 * apart from each other and from what is read. */
int kr_tree_plan(const int32_t *parents, uint32_t tokens, const uint32_t *starts, const uint32_t *lengths, uint32_t batch,
                 uint32_t words, uint32_t *mask, uint32_t *positions, void *stream);

/* The commit, greedy: from node 0 of each sequence (which is the token that the last step chose) on, the path goes to the first child
 * whose token (drafted, i32 [tokens]) is the model's choice after the node (targets, i32 [tokens]; the argmax of its logits), until
 * there is none or the path has max_path nodes.  In every layer, the keys and values of the path's i-th node move to slot n - m + i.
 *   path        u32 [batch, max_path]: the path's nodes, then zeros
 *   counts      u32 [batch]: its length, 0 for a sequence without new tokens
 *   next        i32 [batch]: the model's choice after its last node: the next step's node 0 (a sequence without new tokens: left)
 *   new_lengths u32 [batch]: n - m + counts
 * All four lie apart from one another and from what is read (new_lengths is not lengths).  A node without a slot or a page has no keys
 * to move: a server gives a step's slots their pages before it.
 * Rows beyond new_lengths keep their bits (nothing sees them).  drafted, parents, targets as far as 4096 nodes a sequence; max_path
 * 1 .. 4096.  One launch for all layers. */
int kr_paged_commit(const kr_paged_cache *cache, const kr_paged_step *step, const int32_t *drafted, const int32_t *parents,
                    const int32_t *targets, uint32_t tokens, uint32_t max_path, uint32_t *path, uint32_t *counts,
                    int32_t *next, uint32_t *new_lengths, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* KRIYA_PAGED_H */
