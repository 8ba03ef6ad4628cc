/*
 * kriya_kv8.h — rotary positions in general form, a key/value cache held in
 * 8 bits, the attention that reads it, and the eviction of tokens from it, as
 * a C ABI beside kriya_glue.h (whose cache is bf16 and whose attention takes
 * one new token per sequence).  Conventions as in kriya_q4.h: device pointers
 * unless a comment says otherwise, stream-ordered, no allocation, 0 or a
 * negative KR_E* code with the message in kr_last_error(); a call that fails
 * a check enqueues nothing.  Every call can be captured into a HIP graph.
 */
#ifndef KRIYA_KV8_H
#define KRIYA_KV8_H

#include <stddef.h>
#include <stdint.h>

#include "kriya_q4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions ----
 * A table holds (cos, sin) of position x frequency, f32 [rows, rotary_dim / 2, 2] (the layout of
 * kr_rope_kv_append's cos_sin).  The first rotary_dim dims of a head are turned in pairs,
 *   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c),
 * the dims from rotary_dim on are passed through. */
#define KR_ROPE_HALF 0        /* pairs (i, i + rotary_dim / 2) */
#define KR_ROPE_INTERLEAVED 1 /* pairs (2 i, 2 i + 1)          */

/* Frequencies f_i = theta^(-2 i / rotary_dim), stretched for contexts longer than the trained one: */
#define KR_ROPE_SCALE_NONE 0
#define KR_ROPE_SCALE_LINEAR 1 /* f_i / factor (position interpolation)                          */
#define KR_ROPE_SCALE_NTK 2    /* theta replaced by theta * factor^(rotary_dim / (rotary_dim - 2)) */
#define KR_ROPE_SCALE_PARTS 3  /* by parts: with r = original_ctx f_i / (2 pi) turns over the trained
                                * context and g = clamp((r - slow) / (fast - slow), 0, 1):
                                * f_i (g + (1 - g) / factor): the YaRN paper's interpolation by
                                * parts, a ramp over turns.  Checkpoints stretched by its authors'
                                * program ramp over i between whole numbers instead (theta 1e6,
                                * 128 dims, 32768, factor 4: frequencies up to 71 % apart): make
                                * their table by their formula, the rotations take any table.     */
typedef struct kr_rope_scaling {
    int kind;             /* KR_ROPE_SCALE_*                                                  */
    double factor;        /* > 0; how much longer than trained                                */
    double original_ctx;  /* PARTS: > 0, the trained context                                  */
    double slow, fast;    /* PARTS: turns, slow < fast                                        */
    double gain;          /* multiplies cos and sin (1; YaRN's attention factor 0.1 ln s + 1) */
} kr_rope_scaling;

/* cos_sin[r] = the table row of position first + r, r < count.  Angles, sines and cosines
 * are computed in 64 bits and rounded once, so far positions are as exact as near ones.  scaling: host pointer, NULL for none.  rotary_dim even, 2 .. 256;
 * theta > 0.  cos_sin 8-byte aligned. */
int kr_rope_table(float *cos_sin, uint32_t first, uint32_t count, uint32_t rotary_dim, double theta,
                  const kr_rope_scaling *scaling, void *stream);

typedef struct kr_rope {
    const float *cos_sin;      /* f32 [rows, rotary_dim / 2, 2], 8-byte aligned */
    const uint32_t *positions; /* device u32 [tokens]                           */
    uint32_t rows;             /* a token whose position >= rows is not rotated */
    uint32_t rotary_dim;       /* even, 2 .. head_dim                           */
    int layout;                /* KR_ROPE_HALF or KR_ROPE_INTERLEAVED           */
    int inverse;               /* 1: by the negative angle (undoes it; also the gradient of the rotation) */
} kr_rope;

/* y[t, h] = x[t, h] turned by the table row of positions[t], computed in f32 and rounded once.
 * x, y: [tokens, heads, head_dim] of dtype, tokens x_stride / y_stride elements apart (>= heads * head_dim), so
 * q and k inside the rows of a fused projection can be turned where they are.  y may equal x with the same
 * stride; otherwise they must not overlap.  Any strides and element-aligned pointers; rows that keep 16-byte
 * alignment with rotary_dim % 16 == 0 (8 elements a load) are faster.  head_dim 2 .. 1024. */
int kr_rope_apply(const kr_rope *rope, const void *x, size_t x_stride, void *y, size_t y_stride, int dtype,
                  uint32_t tokens, uint32_t heads, uint32_t head_dim, void *stream);

/* ---- the 8-bit cache ----
 * Slots 0 .. max_ctx - 1 of each sequence and kv head in blocks of 32; a block has one f32 scale for its keys and
 * one for its values: an element stands for code * scale, with
 *   scale = max |x| over the block's tokens and dims / M,   code = x / scale rounded to nearest even
 * (M = 127 and a whole number for KR_KV8_INT8; M = 448 and a float8 e4m3 for KR_KV8_E4M3; both divisions in f32).
 * A block that is given an infinite value or NaN stands for NaN; nothing outside that block is touched by it.
 * The raw bf16 rows of the last block of each sequence are kept beside it (k_open, v_open): a block that is
 * filled token by token is coded again from them, so the codes do not depend on how the tokens arrived.
 *
 * Memory, nb = ceil(max_ctx / 32) (bytes in the order of the matrix instructions' operands; kr_kv8_dequant reads them back):
 *   k [batch, kv_heads, nb, head_dim / 16, 32 slots, 16 dims]                   bytes, 16-byte aligned
 *   v [batch, kv_heads, nb, head_dim / 32, 2 (h), 32 dims, 2 (a), 2 (s), 4 (j)] bytes, slot 16 s + 8 a + 4 h + j
 *   k_scale, v_scale f32 [batch, kv_heads, nb]
 *   k_open, v_open bf16 [batch, kv_heads, 32, head_dim], 16-byte aligned
 * No initial contents are needed.  head_dim 64, 96, 128, 192 or 256; max_ctx 1 .. 2^30.
 *
 * Batches: `lengths` (device u32 [batch]) is the number of tokens of each sequence, those new in this step
 * included; the same array serves the append and the attention of every layer of a step.  The new tokens of sequence
 * b are rows starts[b] .. starts[b + 1] - 1 of k, v, q (starts: device u32 [batch + 1], not decreasing; a
 * sequence may have none) and take its last slots.  starts == NULL: tokens == batch, one each.
 * Values beyond `tokens`, slots beyond max_ctx and lengths below the number of new tokens are cut off, never followed.
 * Rows before the first sequence's and behind the last's are nobody's: nothing of them is appended, and their results (q_out
 * among them) are left as they were.
 * A length may be lowered to take tokens back as long as one token of the sequence's last block stays: the raw rows are that
 * block's. */
#define KR_KV8_INT8 0
#define KR_KV8_E4M3 1
#define KR_KV8_BLOCK 32

typedef struct kr_kv8_cache {
    void *k, *v;
    float *k_scale, *v_scale;
    uint16_t *k_open, *v_open;
    uint32_t batch, kv_heads, head_dim, max_ctx;
    int format;
} kr_kv8_cache;

/* Appends k, v (bf16 [tokens, kv_heads, head_dim], tokens kv_stride elements apart) to the cache.  rope (host
 * pointer, may be NULL): k is rotated first, rounded to bf16 as kr_rope_apply does; and q (bf16 [tokens, q_heads, head_dim],
 * tokens q_stride elements apart; NULL: none) is rotated into q_out (the same stride; may equal q).  One launch.
 * k, v, q, q_out 16-byte aligned, strides multiples of 8.  Without rope q must be NULL; rope->inverse must be 0. */
int kr_kv8_append(const kr_kv8_cache *cache, const kr_rope *rope, const uint16_t *k, const uint16_t *v,
                  size_t kv_stride, const uint16_t *q, uint16_t *q_out, size_t q_stride, uint32_t q_heads,
                  uint32_t tokens, const uint32_t *starts, const uint32_t *lengths, void *stream);

/* Reads the cache back: k_out, v_out [batch, count, kv_heads, head_dim] of dtype (either may be NULL) are slots
 * first[b] .. first[b] + count - 1 of each sequence (first: device u32 [batch], NULL for 0); slots at or beyond
 * lengths[b] give zeros.  (bf16 with first = NULL and count = max_ctx is the cache layout of kriya_glue.h.) */
int kr_kv8_dequant(const kr_kv8_cache *cache, const uint32_t *lengths, const uint32_t *first, uint32_t count,
                   void *k_out, void *v_out, int dtype, void *stream);

/* ---- attention over the 8-bit cache ----
 * For token i of the m new tokens of a sequence of n tokens, and query head g * kv head:
 *   out = sum_p softmax_p(scale q . K_p) V_p   over slots p <= n - m + i,   lse = ln sum_p e^(scale q . K_p)
 * with K_p, V_p the values that the cache's codes stand for.  The codes enter the matrix cores as fp16 (exact), q as
 * fp16 times a power of two of its row (exact down to 2^-29 of the row's largest), the probabilities times
 * their block's scale of values as fp16 (half a step, and at most 2^-32 of the largest such product of the row);
 * sums, maxima and the softmax are f32, for which |scale| sum |q| |K_p| must stay below 2^126; values may be of any size.  A row that
 * sees no slot gives zeros and lse = -infinity.  A row whose q is infinite or NaN, or that sees a block that stands for NaN, gives NaN.
 *   q, out: bf16 [tokens, q_heads, head_dim], q tokens q_stride elements apart (a multiple of 8), out contiguous; both 16-byte
 *   aligned and apart from each other; lse f32 [tokens, q_heads] or NULL; q_heads a multiple of kv_heads; |scale| < 2^100 (may
 *   be negative or 0).
 * From one token per sequence to whole prompts; the launch is chosen from the cache's sizes, tokens and heads, the shares on the device.
 * workspace: kr_kv8_attention_workspace_bytes(cache, q_heads, tokens) bytes, 16-byte aligned, no initial contents; calls
 * sharing it must not overlap in time.  Results are the same bits from run to run. */
size_t kr_kv8_attention_workspace_bytes(const kr_kv8_cache *cache, uint32_t q_heads, uint32_t tokens);
int kr_kv8_attention(const kr_kv8_cache *cache, const uint16_t *q, size_t q_stride, uint32_t q_heads, uint32_t tokens,
                     const uint32_t *starts, const uint32_t *lengths, float scale, uint16_t *out, float *lse,
                     void *workspace, size_t workspace_bytes, void *stream);

/* ---- eviction by accumulated attention weight ----
 * weight f32 [batch, kv_heads, max_ctx]: for every slot p < lengths[b] of every kv head
 *   weight[p] = decay * (p < n - m ? weight[p] : 0) + sum over the m new tokens and the heads of the group of e^(scale q . K_p - lse)
 * with the lse that kr_kv8_attention gave for the same q (slots of the new tokens start at zero: no initial contents are
 * needed; slots from lengths[b] on are left as they were).  Sums in f32, in a fixed order.  tokens == 0 does nothing.  lse is f32, so a
 * weight is off by half a step of its row's score: little up to scores of 2^12, all of it from 2^24 on.
 * The codes enter the matrix cores as bf16 (exact), as q does; the scores are f32.
 * workspace: kr_kv8_weight_workspace_bytes(cache, q_heads, tokens) bytes (none for few rows, else about the size of weight), 16-byte
 * aligned, no initial contents; calls sharing it must not overlap in time. */
size_t kr_kv8_weight_workspace_bytes(const kr_kv8_cache *cache, uint32_t q_heads, uint32_t tokens);
int kr_kv8_accumulate_weight(const kr_kv8_cache *cache, const uint16_t *q, size_t q_stride, uint32_t q_heads,
                             uint32_t tokens, const uint32_t *starts, const uint32_t *lengths, float scale,
                             const float *lse, float decay, float *weight, void *workspace, size_t workspace_bytes,
                             void *stream);

/* Copies each sequence into `to`, cut to `budget` tokens where it is longer: every kv head keeps its first `sink` and
 * last `recent` tokens and, of those between, the budget - sink - recent of largest weight (ties to the lowest slot;
 * NaN counts below every number), in their order.  Keys are stored rotated, so what remains attends as before.
 * Blocks whose 32 tokens all keep their places are copied as they are; the others are coded again from the values that
 * their codes stand for, or from the raw rows for tokens of the last block; the new last block is coded from those
 * values rounded to bf16, which become its raw rows.
 *   kept      u32 [batch, kv_heads, budget]: the old slot of new slot i, i < min(lengths[b], budget)
 *   to_weight f32 [batch, kv_heads, to->max_ctx]: the weights, moved along; from the new length on left as they were
 *   to_lengths u32 [batch]: min(lengths[b], budget); NULL: not written
 * `to`: another cache of the same batch, kv_heads, head_dim and format, max_ctx >= budget; it shares no memory with
 * `cache`, nor to_weight with weight or to_lengths with lengths.  sink + recent <= budget, budget >= 1. */
int kr_kv8_evict(const kr_kv8_cache *cache, const uint32_t *lengths, const float *weight, uint32_t budget,
                 uint32_t sink, uint32_t recent, const kr_kv8_cache *to, float *to_weight, uint32_t *kept,
                 uint32_t *to_lengths, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* KRIYA_KV8_H */
