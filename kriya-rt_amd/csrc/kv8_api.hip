// kv8_api.hip — the C ABI of include/kriya_kv8.h: argument checks and dispatch.
#include <math.h>

#include "api_checks.hpp"

namespace kr {
namespace {

int check_cache(const kr_kv8_cache *c, const char *name) {
    if (!c) return fail(KR_E_INVALID, "%s: descriptor is NULL", name);
    if (c->format != KR_KV8_INT8 && c->format != KR_KV8_E4M3) return fail(KR_E_INVALID, "%s: format %d", name, c->format);
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128 && c->head_dim != 192 && c->head_dim != 256)
        return fail(KR_E_UNSUPPORTED, "%s: head_dim=%u is not 64, 96, 128, 192 or 256", name, c->head_dim);
    if (c->kv_heads == 0 || c->kv_heads > 65535) return fail(KR_E_SHAPE, "%s: kv_heads=%u is not 1 .. 65535", name, c->kv_heads);
    if (c->batch > 65535) return fail(KR_E_SHAPE, "%s: batch=%u exceeds 65535", name, c->batch);
    if (c->max_ctx == 0 || c->max_ctx > (1u << 30)) return fail(KR_E_SHAPE, "%s: max_ctx=%u is not 1 .. 2^30", name, c->max_ctx);
    if (c->batch == 0) return KR_OK;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_open || !c->v_open)
        return fail(KR_E_INVALID, "%s: NULL pointer", name);
    if (!on(c->k, 16) || !on(c->v, 16) || !on(c->k_open, 16) || !on(c->v_open, 16) || !on(c->k_scale, 4) || !on(c->v_scale, 4))
        return fail(KR_E_ALIGN, "%s: k, v, k_open and v_open must be 16-byte aligned, the scales 4-byte", name);
    return KR_OK;
}

Kv8 to_kv8(const kr_kv8_cache *c) {
    return Kv8{(uint8_t *)c->k, (uint8_t *)c->v, c->k_scale, c->v_scale, c->k_open, c->v_open, c->batch, c->kv_heads,
               c->head_dim, c->max_ctx, (c->max_ctx + kKv8Block - 1) / kKv8Block, c->format == KR_KV8_E4M3};
}

int check_step(const kr_kv8_cache *c, uint32_t tokens, const uint32_t *starts, const uint32_t *lengths) {
    if (!lengths) return fail(KR_E_INVALID, "lengths is NULL");
    if (!starts && tokens != c->batch)
        return fail(KR_E_SHAPE, "tokens=%u and batch=%u: without starts every sequence has one new token", tokens, c->batch);
    if (!on(lengths, 4) || !on(starts, 4)) return fail(KR_E_ALIGN, "lengths and starts must be 4-byte aligned");
    return KR_OK;
}

int check_queries(const kr_kv8_cache *c, const uint16_t *q, size_t q_stride, uint32_t q_heads, uint32_t tokens) {
    if (q_heads == 0 || q_heads % c->kv_heads)
        return fail(KR_E_SHAPE, "q_heads=%u is not a positive multiple of kv_heads=%u", q_heads, c->kv_heads);
    if ((uint64_t)tokens * q_heads > 0x7FFFFFFFull) return fail(KR_E_SHAPE, "tokens * q_heads exceeds 2^31 - 1");
    if (tokens == 0 || c->batch == 0) return KR_OK;
    if (!q) return fail(KR_E_INVALID, "q is NULL");
    if (q_stride < (size_t)q_heads * c->head_dim || q_stride % 8)
        return fail(KR_E_SHAPE, "q_stride=%zu is not a multiple of 8, at least q_heads * head_dim", q_stride);
    if (!on(q, 16)) return fail(KR_E_ALIGN, "q must be 16-byte aligned");
    return KR_OK;
}

bool finite_positive(double v) { return v > 0.0 && v < INFINITY; }

}  // namespace
}  // namespace kr

using namespace kr;

extern "C" {

int kr_rope_table(float *cos_sin, uint32_t first, uint32_t count, uint32_t rotary_dim, double theta,
                  const kr_rope_scaling *scaling, void *stream) {
    if (rotary_dim == 0 || rotary_dim % 2 || rotary_dim > kRopeMaxDim)
        return fail(KR_E_SHAPE, "rotary_dim=%u is not even, 2 .. %u", rotary_dim, kRopeMaxDim);
    if (!finite_positive(theta)) return fail(KR_E_INVALID, "theta must be positive and finite");
    const kr_rope_scaling none = {KR_ROPE_SCALE_NONE, 1.0, 1.0, 0.0, 1.0, 1.0};
    const kr_rope_scaling z = scaling ? *scaling : none;
    if (z.kind < KR_ROPE_SCALE_NONE || z.kind > KR_ROPE_SCALE_PARTS) return fail(KR_E_INVALID, "scaling kind %d", z.kind);
    if (z.kind != KR_ROPE_SCALE_NONE && !finite_positive(z.factor))
        return fail(KR_E_INVALID, "scaling factor must be positive and finite");
    if (z.kind == KR_ROPE_SCALE_NTK && rotary_dim == 2)
        return fail(KR_E_SHAPE, "NTK scaling needs rotary_dim > 2");
    if (z.kind == KR_ROPE_SCALE_PARTS && (!finite_positive(z.original_ctx) || !(z.slow < z.fast)))
        return fail(KR_E_INVALID, "scaling by parts needs original_ctx > 0 and slow < fast");
    if (!(fabsf((float)z.gain) < INFINITY)) return fail(KR_E_INVALID, "scaling gain must be finite in 32 bits");
    if ((uint64_t)first + count > (1ull << 32)) return fail(KR_E_SHAPE, "first + count exceeds 2^32");
    if (count == 0) return ok();
    if (!cos_sin) return fail(KR_E_INVALID, "cos_sin is NULL");
    if (!on(cos_sin, 8)) return fail(KR_E_ALIGN, "cos_sin must be 8-byte aligned");
    if ((uint64_t)count * (rotary_dim / 2) > kMostGroups * 256) return fail(KR_E_SHAPE, "count=%u is too large for one launch", count);
    RopeTurns f{};
    const double pi2 = 6.283185307179586476925, half = rotary_dim / 2;
    if (z.kind == KR_ROPE_SCALE_NTK) theta *= pow(z.factor, half / (half - 1.0));
    for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
        double w = pow(theta, -(double)i / half);
        if (z.kind == KR_ROPE_SCALE_LINEAR) w /= z.factor;
        if (z.kind == KR_ROPE_SCALE_PARTS) {
            const double r = z.original_ctx * w / pi2;
            const double g = fmin(fmax((r - z.slow) / (z.fast - z.slow), 0.0), 1.0);
            w *= g + (1.0 - g) / z.factor;
        }
        f.turns[i] = w / pi2;
    }
    return hip_status(launch_rope_table(f, rotary_dim / 2, first, count, z.gain, cos_sin, (hipStream_t)stream),
                      "kr_rope_table");
}

int kr_rope_apply(const kr_rope *rope, const void *x, size_t x_stride, void *y, size_t y_stride, int dtype,
                  uint32_t tokens, uint32_t heads, uint32_t head_dim, void *stream) {
    if (!rope) return fail(KR_E_INVALID, "rope is NULL");
    if (dtype != KR_DTYPE_BF16 && dtype != KR_DTYPE_F32) return fail(KR_E_INVALID, "dtype %d invalid", dtype);
    if (head_dim < 2 || head_dim > kRopeMaxHeadDim) return fail(KR_E_SHAPE, "head_dim=%u is not 2 .. %u", head_dim, kRopeMaxHeadDim);
    if (heads == 0 || heads > 65535) return fail(KR_E_SHAPE, "heads=%u is not 1 .. 65535", heads);
    if (tokens == 0) return ok();
    if (int rc = check_rope(rope, head_dim)) return rc;
    if (!x || !y) return fail(KR_E_INVALID, "NULL pointer");
    if (x_stride < (size_t)heads * head_dim || y_stride < (size_t)heads * head_dim)
        return fail(KR_E_SHAPE, "strides below heads * head_dim");
    if (x == y && x_stride != y_stride) return fail(KR_E_SHAPE, "in place with different strides");
    if (tokens > kMostGroups) return fail(KR_E_SHAPE, "tokens=%u is too many for one launch", tokens);
    const size_t es = dtype == KR_DTYPE_F32 ? 4 : 2;
    if (!on(x, es) || !on(y, es)) return fail(KR_E_ALIGN, "x and y must be aligned to their elements");
    return hip_status(launch_rope_apply(to_rope(rope), x, x_stride, y, y_stride, dtype == KR_DTYPE_F32, tokens, heads,
                                        head_dim, (hipStream_t)stream),
                      "kr_rope_apply");
}

int kr_kv8_append(const kr_kv8_cache *cache, const kr_rope *rope, const uint16_t *k, const uint16_t *v,
                  size_t kv_stride, const uint16_t *q, uint16_t *q_out, size_t q_stride, uint32_t q_heads,
                  uint32_t tokens, const uint32_t *starts, const uint32_t *lengths, void *stream) {
    if (int rc = check_cache(cache, "cache")) return rc;
    if (tokens == 0 || cache->batch == 0) return ok();
    if (int rc = check_step(cache, tokens, starts, lengths)) return rc;
    if (rope) {
        if (int rc = check_rope(rope, cache->head_dim)) return rc;
        if (rope->inverse) return fail(KR_E_INVALID, "rope: the append rotates forward, inverse must be 0");
    }
    if (!k || !v) return fail(KR_E_INVALID, "k and v must not be NULL");
    if (!on(k, 16) || !on(v, 16)) return fail(KR_E_ALIGN, "k and v must be 16-byte aligned");
    if (kv_stride < (size_t)cache->kv_heads * cache->head_dim || kv_stride % 8)
        return fail(KR_E_SHAPE, "kv_stride=%zu is not a multiple of 8, at least kv_heads * head_dim", kv_stride);
    if (q) {
        if (!rope) return fail(KR_E_INVALID, "q is given without rope");
        if (!q_out) return fail(KR_E_INVALID, "q_out is NULL");
        if (q_heads == 0 || q_heads > 65535) return fail(KR_E_SHAPE, "q_heads=%u is not 1 .. 65535", q_heads);
        if (q_stride < (size_t)q_heads * cache->head_dim || q_stride % 8)
            return fail(KR_E_SHAPE, "q_stride=%zu is not a multiple of 8, at least q_heads * head_dim", q_stride);
        if (!on(q, 16) || !on(q_out, 16)) return fail(KR_E_ALIGN, "q and q_out must be 16-byte aligned");
    }
    if (((uint64_t)tokens / kKv8Block + cache->batch) * cache->kv_heads + tokens > kMostGroups)
        return fail(KR_E_SHAPE, "too many tokens for one launch");
    Kv8AppendArgs a{};
    a.c = to_kv8(cache);
    a.step = RaggedStep{starts, lengths, cache->batch, tokens};
    if (rope) {
        a.rope = to_rope(rope);
        a.rope_units = rope_units_ok(a.rope, cache->head_dim);
    }
    a.k = k;
    a.v = v;
    a.q = q;
    a.q_out = q_out;
    a.kv_stride = kv_stride;
    a.q_stride = q_stride;
    a.q_heads = q_heads;
    return hip_status(launch_kv8_append(a, (hipStream_t)stream), "kr_kv8_append");
}

int kr_kv8_dequant(const kr_kv8_cache *cache, const uint32_t *lengths, const uint32_t *first, uint32_t count,
                   void *k_out, void *v_out, int dtype, void *stream) {
    if (int rc = check_cache(cache, "cache")) return rc;
    if (dtype != KR_DTYPE_BF16 && dtype != KR_DTYPE_F32) return fail(KR_E_INVALID, "dtype %d invalid", dtype);
    if (count > (1u << 30)) return fail(KR_E_SHAPE, "count=%u exceeds 2^30", count);
    if (count == 0 || cache->batch == 0 || (!k_out && !v_out)) return ok();
    if (!lengths) return fail(KR_E_INVALID, "lengths is NULL");
    if (!on(k_out, 16) || !on(v_out, 16)) return fail(KR_E_ALIGN, "k_out and v_out must be 16-byte aligned");
    if (!on(lengths, 4) || !on(first, 4)) return fail(KR_E_ALIGN, "lengths and first must be 4-byte aligned");
    if ((uint64_t)(count / 4 + 2) * cache->kv_heads * (cache->head_dim / 8) > 0xFFFFFF00ull)
        return fail(KR_E_SHAPE, "count=%u is too large for one launch", count);
    return hip_status(launch_kv8_dequant(to_kv8(cache), lengths, first, count, k_out, v_out, dtype == KR_DTYPE_F32,
                                         (hipStream_t)stream),
                      "kr_kv8_dequant");
}

size_t kr_kv8_attention_workspace_bytes(const kr_kv8_cache *cache, uint32_t q_heads, uint32_t tokens) {
    if (!cache || cache->kv_heads == 0 || q_heads == 0 || q_heads % cache->kv_heads || tokens == 0 || cache->batch == 0) return 0;
    const size_t n = kv8_attention_workspace_bytes(cache->batch, cache->kv_heads, q_heads / cache->kv_heads,
                                                   cache->head_dim, tokens, cache->max_ctx);
    return (n + 255) / 256 * 256;
}

int kr_kv8_attention(const kr_kv8_cache *cache, const uint16_t *q, size_t q_stride, uint32_t q_heads, uint32_t tokens,
                     const uint32_t *starts, const uint32_t *lengths, float scale, uint16_t *out, float *lse,
                     void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_cache(cache, "cache")) return rc;
    if (int rc = check_queries(cache, q, q_stride, q_heads, tokens)) return rc;
    if (!(fabsf(scale) < kMaxScale)) return fail(KR_E_INVALID, "scale must be below 2^100 in size");
    if (tokens == 0 || cache->batch == 0) return ok();
    if (int rc = check_step(cache, tokens, starts, lengths)) return rc;
    if (!out) return fail(KR_E_INVALID, "out is NULL");
    if (!on(out, 16) || !on(lse, 4)) return fail(KR_E_ALIGN, "out must be 16-byte aligned, lse 4-byte");
    if (kv8_attention_groups(cache->batch, cache->kv_heads, q_heads / cache->kv_heads, cache->head_dim, tokens, cache->max_ctx) > kMostGroups)
        return fail(KR_E_SHAPE, "tokens=%u of %u sequences and %u heads are too many for one launch", tokens, cache->batch, q_heads);
    const size_t need = kr_kv8_attention_workspace_bytes(cache, q_heads, tokens);
    if (need && (!workspace || workspace_bytes < need))
        return fail(KR_E_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
    if (!on(workspace, 16)) return fail(KR_E_ALIGN, "workspace must be 16-byte aligned");
    Kv8AttnArgs a{};
    a.c = to_kv8(cache);
    a.step = RaggedStep{starts, lengths, cache->batch, tokens};
    a.q = q;
    a.q_stride = q_stride;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.scale_log2 = scale * 1.44269504f;
    a.out = out;
    a.lse = lse;
    a.part = (float *)workspace;
    return hip_status(launch_kv8_attention(a, (hipStream_t)stream), "kr_kv8_attention");
}

size_t kr_kv8_weight_workspace_bytes(const kr_kv8_cache *cache, uint32_t q_heads, uint32_t tokens) {
    if (!cache || cache->kv_heads == 0 || q_heads == 0 || q_heads % cache->kv_heads || tokens == 0 || cache->batch == 0) return 0;
    const size_t n = kv8_weight_workspace_bytes(cache->batch, cache->kv_heads, q_heads / cache->kv_heads, tokens, cache->max_ctx);
    return (n + 255) / 256 * 256;
}

int kr_kv8_accumulate_weight(const kr_kv8_cache *cache, const uint16_t *q, size_t q_stride, uint32_t q_heads,
                             uint32_t tokens, const uint32_t *starts, const uint32_t *lengths, float scale,
                             const float *lse, float decay, float *weight, void *workspace, size_t workspace_bytes,
                             void *stream) {
    if (int rc = check_cache(cache, "cache")) return rc;
    if (int rc = check_queries(cache, q, q_stride, q_heads, tokens)) return rc;
    if (!(fabsf(scale) < kMaxScale) || !(fabsf(decay) < INFINITY))
        return fail(KR_E_INVALID, "scale must be below 2^100 in size, decay finite");
    if (tokens == 0 || cache->batch == 0) return ok();
    if (int rc = check_step(cache, tokens, starts, lengths)) return rc;
    if (!lse || !weight) return fail(KR_E_INVALID, "lse and weight must not be NULL");
    if (!on(lse, 4) || !on(weight, 4)) return fail(KR_E_ALIGN, "lse and weight must be 4-byte aligned");
    const size_t need = kr_kv8_weight_workspace_bytes(cache, q_heads, tokens);
    if (need && (!workspace || workspace_bytes < need))
        return fail(KR_E_WORKSPACE, "workspace of %zu bytes required, %zu given", need, workspace_bytes);
    if (!on(workspace, 16)) return fail(KR_E_ALIGN, "workspace must be 16-byte aligned");
    Kv8AttnArgs a{};
    a.c = to_kv8(cache);
    a.step = RaggedStep{starts, lengths, cache->batch, tokens};
    a.q = q;
    a.q_stride = q_stride;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.scale_log2 = scale * 1.44269504f;
    a.lse = const_cast<float *>(lse);
    a.decay = decay;
    a.weight = weight;
    a.part = (float *)workspace;
    return hip_status(launch_kv8_weight(a, (hipStream_t)stream), "kr_kv8_accumulate_weight");
}

int kr_kv8_evict(const kr_kv8_cache *cache, const uint32_t *lengths, const float *weight, uint32_t budget,
                 uint32_t sink, uint32_t recent, const kr_kv8_cache *to, float *to_weight, uint32_t *kept,
                 uint32_t *to_lengths, void *stream) {
    if (int rc = check_cache(cache, "cache")) return rc;
    if (int rc = check_cache(to, "to")) return rc;
    if (to->batch != cache->batch || to->kv_heads != cache->kv_heads || to->head_dim != cache->head_dim || to->format != cache->format)
        return fail(KR_E_SHAPE, "`to` must have the cache's batch, kv_heads, head_dim and format");
    if (budget == 0 || budget > to->max_ctx) return fail(KR_E_SHAPE, "budget=%u is not 1 .. to->max_ctx=%u", budget, to->max_ctx);
    if ((budget + kKv8Block - 1) / kKv8Block > kMostGroups) return fail(KR_E_SHAPE, "budget=%u is too large for one launch", budget);
    if ((uint64_t)sink + recent > budget) return fail(KR_E_SHAPE, "sink=%u + recent=%u exceeds budget=%u", sink, recent, budget);
    if (cache->batch == 0) return ok();
    if (!lengths || !weight || !to_weight || !kept) return fail(KR_E_INVALID, "NULL pointer");
    if (!on(lengths, 4) || !on(weight, 4) || !on(to_weight, 4) || !on(kept, 4) || !on(to_lengths, 4))
        return fail(KR_E_ALIGN, "lengths, weights and kept must be 4-byte aligned");
    if (to->k == cache->k || to->v == cache->v || to->k_scale == cache->k_scale || to->v_scale == cache->v_scale ||
        to->k_open == cache->k_open || to->v_open == cache->v_open || to_weight == weight || to_lengths == lengths)
        return fail(KR_E_INVALID, "`to` must not share memory with the cache");
    Kv8EvictArgs a{};
    a.from = to_kv8(cache);
    a.to = to_kv8(to);
    a.lengths = lengths;
    a.weight = weight;
    a.budget = budget;
    a.sink = sink;
    a.recent = recent;
    a.to_weight = to_weight;
    a.kept = kept;
    a.to_lengths = to_lengths;
    return hip_status(launch_kv8_evict(a, (hipStream_t)stream), "kr_kv8_evict");
}

}  // extern "C"
