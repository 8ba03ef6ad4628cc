// paged_api.hip — the C ABI of include/kriya_paged.h: argument checks and dispatch.
#include <math.h>

#include "api_checks.hpp"
#include "kriya_paged.h"

namespace kr {
namespace {

int check_sizes(const kr_paged_cache *c) {
    if (!c) return fail(KR_E_INVALID, "cache: descriptor is NULL");
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 192 && c->head_dim != 256)
        return fail(KR_E_UNSUPPORTED, "cache: head_dim=%u is not 64, 96, 128, 192 or 256", c->head_dim);
    if (c->page < kPagedUnit || c->page > 4096 || (c->page & (c->page - 1)))
        return fail(KR_E_UNSUPPORTED, "cache: page=%u is not 16, 32, 64, .. 4096", c->page);
    if (c->kv_heads == 0 || c->kv_heads > 65535) return fail(KR_E_SHAPE, "cache: kv_heads=%u is not 1 .. 65535", c->kv_heads);
    if (c->pages == 0 || c->pages > 0x7FFFFFFFu) return fail(KR_E_SHAPE, "cache: pages=%u is not 1 .. 2^31 - 1", c->pages);
    if (c->layers == 0 || c->layers > 65535) return fail(KR_E_SHAPE, "cache: layers=%u is not 1 .. 65535", c->layers);
    if ((uint64_t)c->pages * c->kv_heads > 0xFFFFFFFFull / (c->page / kPagedUnit))
        return fail(KR_E_SHAPE, "cache: pages=%u of %u heads and %u slots are more than 2^32 units of 16 slots", c->pages, c->kv_heads, c->page);
    return KR_OK;
}
int check_cache(const kr_paged_cache *c, uint32_t layer) {
    if (int rc = check_sizes(c)) return rc;
    if (layer >= c->layers) return fail(KR_E_SHAPE, "layer=%u of %u", layer, c->layers);
    if (!c->k || !c->v) return fail(KR_E_INVALID, "cache: NULL pointer");
    if (!on(c->k, 16) || !on(c->v, 16)) return fail(KR_E_ALIGN, "cache: k and v must be 16-byte aligned");
    return KR_OK;
}

// Sizes only; the pointers are looked at where there is something to do.
int check_step(const kr_paged_cache *c, const kr_paged_step *s) {
    if (!s) return fail(KR_E_INVALID, "step: descriptor is NULL");
    if (s->batch > 65535) return fail(KR_E_SHAPE, "step: batch=%u exceeds 65535", s->batch);
    if (s->max_pages == 0 || (uint64_t)s->max_pages * c->page > (1u << 30))
        return fail(KR_E_SHAPE, "step: max_pages=%u pages of %u slots are not 1 .. 2^30 slots", s->max_pages, c->page);
    return KR_OK;
}
int check_sequences(const uint32_t *starts, const uint32_t *lengths, uint32_t batch, uint32_t tokens) {
    if (!lengths) return fail(KR_E_INVALID, "lengths is NULL");
    if (!starts && tokens != batch)
        return fail(KR_E_SHAPE, "tokens=%u and batch=%u: without starts every sequence has one new token", tokens, batch);
    if (!on(lengths, 4) || !on(starts, 4)) return fail(KR_E_ALIGN, "lengths and starts must be 4-byte aligned");
    return KR_OK;
}
int check_pointers(const kr_paged_step *s, uint32_t tokens) {
    if (!s->table) return fail(KR_E_INVALID, "step: table is NULL");
    if (!on(s->table, 4)) return fail(KR_E_ALIGN, "step: table must be 4-byte aligned");
    return check_sequences(s->starts, s->lengths, s->batch, tokens);
}

// Keys or values of `layers` layers from one on.
Range pool_of(const char *name, const uint16_t *at, const kr_paged_cache *c, uint32_t layer, uint32_t layers) {
    const size_t each = (size_t)c->pages * c->kv_heads * c->page * c->head_dim;
    return Range{name, at + layer * each, layers * each * 2};
}
// Rows of heads.
Range rows_of(const char *name, const uint16_t *at, uint32_t rows, uint32_t heads, uint32_t head_dim, size_t stride) {
    return Range{name, at, (size_t)heads * head_dim * 2, rows, stride * 2};
}
Range lengths_of(const kr_paged_step *s) { return Range{"lengths", s->lengths, (size_t)s->batch * 4}; }
Range starts_of(const kr_paged_step *s) { return Range{"starts", s->starts, ((size_t)s->batch + 1) * 4}; }
Range table_of(const kr_paged_step *s) { return Range{"table", s->table, (size_t)s->batch * s->max_pages * 4}; }

Paged to_paged(const kr_paged_cache *c, uint32_t layer, const kr_paged_step *s) {
    const size_t at = (size_t)layer * c->pages * c->kv_heads * c->page * c->head_dim;
    uint32_t shift = 0;
    while ((kPagedUnit << shift) < c->page) ++shift;
    return Paged{c->k + at, c->v + at, s->table, c->pages, s->max_pages, shift, s->batch, c->kv_heads, c->head_dim, s->max_pages * c->page};
}
RaggedStep to_step(const kr_paged_step *s, uint32_t tokens) { return RaggedStep{s->starts, s->lengths, s->batch, tokens}; }

int check_heads(const char *name, uint32_t heads) {
    return heads == 0 || heads > 65535 ? fail(KR_E_SHAPE, "%s: %u heads are not 1 .. 65535", name, heads) : KR_OK;
}
int check_rows(const char *name, const uint16_t *x, size_t stride, uint32_t heads, uint32_t head_dim) {
    if (int rc = check_heads(name, heads)) return rc;
    if (stride < (size_t)heads * head_dim || stride % 8)
        return fail(KR_E_SHAPE, "%s: a stride of %zu is not a multiple of 8, at least heads * head_dim", name, stride);
    if (!on(x, 16)) return fail(KR_E_ALIGN, "%s must be 16-byte aligned", name);
    return KR_OK;
}

// The sizes of an attention call on a cache and step whose own are right.
int check_attention(const kr_paged_cache *c, const kr_paged_step *s, uint32_t q_heads, uint32_t tokens) {
    if (q_heads == 0 || q_heads % c->kv_heads)
        return fail(KR_E_SHAPE, "q_heads=%u is not a positive multiple of kv_heads=%u", q_heads, c->kv_heads);
    if ((uint64_t)tokens * q_heads > 0x7FFFFFFFull) return fail(KR_E_SHAPE, "tokens * q_heads exceeds 2^31 - 1");
    if (tokens == 0 || s->batch == 0) return KR_OK;
    if (int rc = check_heads("q", q_heads)) return rc;
    if (paged_attention_groups(s->batch, c->kv_heads, q_heads / c->kv_heads, c->head_dim, tokens, s->max_pages * c->page) > kMostGroups)
        return fail(KR_E_SHAPE, "tokens=%u of %u sequences and %u heads are too many for one launch", tokens, s->batch, q_heads);
    return KR_OK;
}

}  // namespace
}  // namespace kr

using namespace kr;

extern "C" {

int kr_paged_append(const kr_paged_cache *cache, uint32_t layer, const kr_paged_step *step, const kr_head_norm *norm,
                    const kr_rope *rope, const uint16_t *k, const uint16_t *v, size_t kv_stride, const uint16_t *q,
                    uint16_t *q_out, size_t q_stride, uint32_t q_heads, uint32_t tokens, void *stream) {
    if (int rc = check_cache(cache, layer)) return rc;
    if (int rc = check_step(cache, step)) return rc;
    if (tokens == 0 || step->batch == 0) return ok();
    if (int rc = check_pointers(step, tokens)) return rc;
    if (norm) {
        if (!(norm->eps >= 0.0f && norm->eps < INFINITY)) return fail(KR_E_INVALID, "norm: eps must be finite, 0 or more");
        if (!on(norm->q_weight, 2) || !on(norm->k_weight, 2)) return fail(KR_E_ALIGN, "norm: weights must be 2-byte aligned");
    }
    if (rope) {
        if (int rc = check_rope(rope, cache->head_dim)) return rc;
        if (rope->inverse) return fail(KR_E_INVALID, "rope: the append rotates forward, inverse must be 0");
    }
    if (!k || !v) return fail(KR_E_INVALID, "k and v must not be NULL");
    if (int rc = check_rows("k", k, kv_stride, cache->kv_heads, cache->head_dim)) return rc;
    if (int rc = check_rows("v", v, kv_stride, cache->kv_heads, cache->head_dim)) return rc;
    if (q) {
        if (!rope && !norm) return fail(KR_E_INVALID, "q is given without norm and rope");
        if (!q_out) return fail(KR_E_INVALID, "q_out is NULL");
        if (int rc = check_rows("q", q, q_stride, q_heads, cache->head_dim)) return rc;
        if (int rc = check_rows("q_out", q_out, q_stride, q_heads, cache->head_dim)) return rc;
    }
    PagedAppendArgs a{};
    a.c = to_paged(cache, layer, step);
    a.step = to_step(step, tokens);
    if (rope) a.rope = to_rope(rope);
    if (norm) {
        a.q_norm = norm->q_weight;
        a.k_norm = norm->k_weight;
        a.eps = norm->eps;
    }
    a.k = k;
    a.v = v;
    a.q = q;
    a.q_out = q_out;
    a.kv_stride = kv_stride;
    a.q_stride = q_stride;
    a.q_heads = q_heads;
    if (paged_append_groups(a) > kMostGroups) return fail(KR_E_SHAPE, "tokens=%u are too many for one launch", tokens);
    // (a workgroup's rows are written while others read theirs)
    const uint32_t D = cache->head_dim;
    if (int rc = check_apart({rows_of("q_out", q ? q_out : nullptr, tokens, q_heads, D, q_stride),
                              pool_of("cache k", cache->k, cache, layer, 1), pool_of("cache v", cache->v, cache, layer, 1)},
                             {rows_of("q", q == q_out ? nullptr : q, tokens, q_heads, D, q_stride),
                              rows_of("k", k, tokens, cache->kv_heads, D, kv_stride), rows_of("v", v, tokens, cache->kv_heads, D, kv_stride),
                              {"q_weight", a.q_norm, D * 2ul}, {"k_weight", a.k_norm, D * 2ul},
                              {"positions", a.rope.positions, tokens * 4ul}, {"cos_sin", a.rope.cos_sin, (size_t)a.rope.rows * a.rope.rotary_dim * 4},
                              table_of(step), lengths_of(step), starts_of(step)}))
        return rc;
    return hip_status(launch_paged_append(a, (hipStream_t)stream), "kr_paged_append");
}

int kr_paged_read(const kr_paged_cache *cache, uint32_t layer, const kr_paged_step *step, const uint32_t *first,
                  uint32_t count, void *k_out, void *v_out, int dtype, void *stream) {
    if (int rc = check_cache(cache, layer)) return rc;
    if (int rc = check_step(cache, step)) return rc;
    if (dtype != KR_DTYPE_BF16 && dtype != KR_DTYPE_F32) return fail(KR_E_INVALID, "dtype %d invalid", dtype);
    if (count > (1u << 30)) return fail(KR_E_SHAPE, "count=%u exceeds 2^30", count);
    if (count == 0 || step->batch == 0 || (!k_out && !v_out)) return ok();
    if (int rc = check_pointers(step, step->batch)) return rc;
    if (!on(k_out, 16) || !on(v_out, 16)) return fail(KR_E_ALIGN, "k_out and v_out must be 16-byte aligned");
    if (!on(first, 4)) return fail(KR_E_ALIGN, "first must be 4-byte aligned");
    if ((uint64_t)count * cache->kv_heads * (cache->head_dim / 8) > kMostGroups * 256)
        return fail(KR_E_SHAPE, "count=%u is too large for one launch", count);
    const size_t bytes = (size_t)step->batch * count * cache->kv_heads * cache->head_dim * (dtype == KR_DTYPE_F32 ? 4 : 2);
    if (int rc = check_apart({{"k_out", k_out, bytes}, {"v_out", v_out, bytes}},
                             {pool_of("cache k", cache->k, cache, layer, 1), pool_of("cache v", cache->v, cache, layer, 1), table_of(step),
                              lengths_of(step), {"first", first, step->batch * 4ul}}))
        return rc;
    return hip_status(launch_paged_read(to_paged(cache, layer, step), to_step(step, 0), first, count, k_out, v_out,
                                        dtype == KR_DTYPE_F32, (hipStream_t)stream),
                      "kr_paged_read");
}

size_t kr_paged_attention_workspace_bytes(const kr_paged_cache *cache, const kr_paged_step *step, uint32_t q_heads,
                                          uint32_t tokens) {
    if (check_sizes(cache) || check_step(cache, step) || check_attention(cache, step, q_heads, tokens) || tokens == 0 || step->batch == 0) return 0;
    const size_t n = paged_attention_workspace_bytes(step->batch, cache->kv_heads, q_heads / cache->kv_heads, cache->head_dim,
                                                     tokens, step->max_pages * cache->page);
    return (n + 255) / 256 * 256;
}

int kr_paged_attention(const kr_paged_cache *cache, uint32_t layer, const kr_paged_step *step, const uint16_t *q,
                       size_t q_stride, uint32_t q_heads, uint32_t tokens, const uint32_t *mask, uint32_t words,
                       float scale, uint16_t *out, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_cache(cache, layer)) return rc;
    if (int rc = check_step(cache, step)) return rc;
    if (int rc = check_attention(cache, step, q_heads, tokens)) return rc;
    if (!(fabsf(scale) < kMaxScale)) return fail(KR_E_INVALID, "scale must be below 2^100 in size");
    if (mask && (words == 0 || words > (1u << 20))) return fail(KR_E_SHAPE, "mask: words=%u is not 1 .. 2^20", words);
    if (!on(mask, 4)) return fail(KR_E_ALIGN, "mask must be 4-byte aligned");
    if (tokens == 0 || step->batch == 0) return ok();
    if (int rc = check_pointers(step, tokens)) return rc;
    if (!q || !out) return fail(KR_E_INVALID, "q and out must not be NULL");
    if (int rc = check_rows("q", q, q_stride, q_heads, cache->head_dim)) return rc;
    if (!on(out, 16) || !on(lse, 4)) return fail(KR_E_ALIGN, "out must be 16-byte aligned, lse 4-byte");
    const Paged c = to_paged(cache, layer, step);
    const size_t need = kr_paged_attention_workspace_bytes(cache, step, q_heads, tokens);
    if (need && (!workspace || workspace_bytes < need))
        return fail(KR_E_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
    if (!on(workspace, 16)) return fail(KR_E_ALIGN, "workspace must be 16-byte aligned");
    const size_t rows = (size_t)tokens * q_heads;
    if (int rc = check_apart({{"out", out, rows * cache->head_dim * 2}, {"lse", lse, rows * 4}, {"workspace", workspace, need}},
                             {rows_of("q", q, tokens, q_heads, cache->head_dim, q_stride), {"mask", mask, (size_t)tokens * words * 4},
                              pool_of("cache k", cache->k, cache, layer, 1), pool_of("cache v", cache->v, cache, layer, 1), table_of(step),
                              lengths_of(step), starts_of(step)}))
        return rc;
    PagedAttnArgs a{};
    a.c = c;
    a.step = to_step(step, tokens);
    a.q = q;
    a.q_stride = q_stride;
    a.q_heads = q_heads;
    a.group = Divisor(q_heads / c.heads);
    a.mask = mask;
    a.words = words;
    a.scale_log2 = scale * 1.44269504f;
    a.out = out;
    a.lse = lse;
    a.part = (float *)workspace;
    return hip_status(launch_paged_attention(a, (hipStream_t)stream), "kr_paged_attention");
}

int kr_tree_plan(const int32_t *parents, uint32_t tokens, const uint32_t *starts, const uint32_t *lengths, uint32_t batch,
                 uint32_t words, uint32_t *mask, uint32_t *positions, void *stream) {
    if (words == 0 || words > kTreeNodes / 32) return fail(KR_E_SHAPE, "words=%u is not 1 .. %u", words, kTreeNodes / 32);
    if (batch > 65535) return fail(KR_E_SHAPE, "batch=%u exceeds 65535", batch);
    if (tokens == 0 || batch == 0) return ok();
    if (int rc = check_sequences(starts, lengths, batch, tokens)) return rc;
    if (!parents || !mask || !positions) return fail(KR_E_INVALID, "parents, mask and positions must not be NULL");
    if (!on(parents, 4) || !on(mask, 4) || !on(positions, 4)) return fail(KR_E_ALIGN, "parents, mask and positions must be 4-byte aligned");
    if (int rc = check_apart({{"mask", mask, (size_t)tokens * words * 4}, {"positions", positions, (size_t)tokens * 4}},
                             {{"parents", parents, (size_t)tokens * 4}, {"starts", starts, ((size_t)batch + 1) * 4}, {"lengths", lengths, (size_t)batch * 4}}))
        return rc;
    return hip_status(launch_tree_plan(parents, RaggedStep{starts, lengths, batch, tokens}, words, mask, positions, (hipStream_t)stream),
                      "kr_tree_plan");
}

int kr_paged_commit(const kr_paged_cache *cache, const kr_paged_step *step, const int32_t *drafted, const int32_t *parents,
                    const int32_t *targets, uint32_t tokens, uint32_t max_path, uint32_t *path, uint32_t *counts,
                    int32_t *next, uint32_t *new_lengths, void *stream) {
    if (int rc = check_cache(cache, 0)) return rc;
    if (int rc = check_step(cache, step)) return rc;
    if (max_path == 0 || max_path > kTreeNodes) return fail(KR_E_SHAPE, "max_path=%u is not 1 .. %u", max_path, kTreeNodes);
    if (step->batch == 0) return ok();
    if (int rc = check_pointers(step, tokens)) return rc;
    if ((tokens && (!drafted || !parents || !targets)) || !path || !counts || !next || !new_lengths)
        return fail(KR_E_INVALID, "NULL pointer");
    if (!on(drafted, 4) || !on(parents, 4) || !on(targets, 4) || !on(path, 4) || !on(counts, 4) || !on(next, 4) || !on(new_lengths, 4))
        return fail(KR_E_ALIGN, "tokens, path, counts, next and new_lengths must be 4-byte aligned");
    // (every layer's workgroups read what the first one's write)
    const size_t all = (size_t)tokens * 4, each = (size_t)step->batch * 4;
    if (int rc = check_apart({{"path", path, each * max_path}, {"counts", counts, each}, {"next", next, each}, {"new_lengths", new_lengths, each}},
                             {{"tokens", drafted, all}, {"parents", parents, all}, {"targets", targets, all}, lengths_of(step), starts_of(step),
                              table_of(step), pool_of("cache k", cache->k, cache, 0, cache->layers), pool_of("cache v", cache->v, cache, 0, cache->layers)}))
        return rc;
    PagedCommitArgs a{};
    a.c = to_paged(cache, 0, step);
    a.layers = cache->layers;
    a.step = to_step(step, tokens);
    a.drafted = drafted;
    a.parents = parents;
    a.targets = targets;
    a.max_path = max_path;
    a.path = path;
    a.counts = counts;
    a.next = next;
    a.new_lengths = new_lengths;
    return hip_status(launch_paged_commit(a, (hipStream_t)stream), "kr_paged_commit");
}

}  // extern "C"
