// kv8_attention.hip — attention over the 8-bit key/value cache, and the attention weights of its slots.
//
// Reference semantics (grouped query heads, causal at the end of the context; its cache is bf16 pages):
//   kernels/metal/paged_gqa_and_deltanet.metal:242 and the prefill kernels beside it
//
// Mathematics.  The query rows of a sequence and kv head are r = i group + g (token i, head g of the group): every key
// and value byte is used for the whole group.  In base 2, with c_r = scale log2(e) / 2^e_r, ks and vs the scales
// of a block, q' = q 2^e_r in fp16:
//   s_rp = (q'_r . k_p) (c_r ks),   m_r = max_p s_rp,   l_r = sum_p 2^(s_rp - m_r),
//   out_r = sum_p 2^(s_rp - m_r) vs v_p / l_r
// with k_p, v_p the codes.  One pass over the slots: m_r only grows, and sums made under an older m_r are scaled down.
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_32x32x16_f16: a lane then holds one
// query row (column l & 31) and the slots 8 i + 4 (l >> 5) + j of a block, its m_r and l_r are plain registers, and after
// rounding to fp16 those probabilities are the second product's operand as they lie (see kv8.hpp for the order of v).
#include <algorithm>

#include "kv8.hpp"

namespace kr {

namespace {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

// Query row r of a tile, held as the operands of D / 16 steps: lane (column l & 31, h = l >> 5) holds for step 2 j + s
// dims 32 j + 16 h + 8 s .. + 7, the dims that a lane's 16 key bytes cover.
template <int NS>
struct QueryRow {
    f16x8_t f[2 * NS];
    float c;  // scale log2(e) 2^-e
};

// The row in fp16 times a power of two that brings its largest value to [2^14, 2^15): bf16 holds 8 bits of significand
// and fp16 11, so every value down to 2^-28 of the largest is exact, and the rest are off by 2^-39 of it at
// most.  Rows with an infinity or NaN keep them.
template <int NS>
__device__ __forceinline__ void load_query(QueryRow<NS> &q, const uint16_t *row, bool live, float scale_log2) {
    const uint32_t h = __lane_id() >> 5;
    u32x4 raw[2 * NS];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
        raw[i] = u32x4{0, 0, 0, 0};
        if (live) raw[i] = *reinterpret_cast<const u32x4 *>(row + 32 * (i / 2) + 16 * h + 8 * (i & 1));
        top = max(top, bf16_unit_max_bits(raw[i]));
    }
    top = max(top, (uint32_t)__float_as_uint(xchg32(__uint_as_float(top), __lane_id())));
    const int e = row_stage_exp(top, 14, 14, 14);
    const float up = exp2_int(e);
    q.c = scale_log2 * exp2_int(-e);
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) {
        const uint32_t W[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        f16x8_t f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            f[2 * x] = (_Float16)(__uint_as_float(W[x] << 16) * up);
            f[2 * x + 1] = (_Float16)(__uint_as_float(W[x] & 0xFFFF0000u) * up);
        }
        q.f[i] = f;
    }
}

// S^T of one block: 32 slots (rows) x 32 query rows (columns), without the scales.
template <int NS, int E4M3>
__device__ __forceinline__ f32x16 key_product(const u32x4 (&kw)[NS], const QueryRow<NS> &q) {
    f32x16 s = {};
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kv8_operand<E4M3>(kw[j].x, kw[j].y), q.f[2 * j], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kv8_operand<E4M3>(kw[j].z, kw[j].w), q.f[2 * j + 1], s, 0, 0, 0);
    }
    return s;
}

// A lane's 16-byte units of a block's keys (or values): unit j of lane l at 1024 j + 16 l.
template <int NS>
__device__ __forceinline__ void load_units(u32x4 (&w)[NS], const uint8_t *blk) {
#pragma unroll
    for (int j = 0; j < NS; ++j) w[j] = *reinterpret_cast<const u32x4 *>(blk + 1024 * j + 16 * __lane_id());
}

// Row r of sequence span s: the slots that it sees, 0 for a row past the end.
__device__ __forceinline__ uint32_t row_limit(const Kv8Span &s, uint32_t r, uint32_t group, uint32_t max_ctx) {
    const uint32_t i = r / group;
    if (i >= s.m || s.n + i + 1 <= s.m) return 0u;
    return min(s.n - s.m + i + 1, max_ctx);
}

__device__ __forceinline__ uint32_t wave_max_uniform(uint32_t v) { return wave_max_u32(v); }
__device__ __forceinline__ uint32_t wave_min_uniform(uint32_t v) { return ~wave_max_u32(~v); }

}  // namespace

// A wave per tile of 32 query rows of one kv head, over all blocks of its sequence.
template <int NS, int E4M3>
__global__ __launch_bounds__(256) void kv8_attention_kernel(Kv8AttnArgs a, uint32_t items) {
    constexpr uint32_t D = 32 * NS;
    const uint32_t lane = __lane_id(), h = lane >> 5;
    const uint32_t head = blockIdx.y, idx = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (idx >= items) return;
    uint32_t b, tile;
    if (!kv8_find(idx, a.c.batch, [&](uint32_t i) { return (kv8_span(a.step, i).m * a.group + 31) / 32; }, b, tile)) return;
    const Kv8Span s = kv8_span(a.step, b);
    const uint32_t r = 32 * tile + (lane & 31);
    const bool live = r < s.m * a.group;
    const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    QueryRow<NS> q;
    load_query<NS>(q, a.q + t * a.q_stride + (size_t)qh * D, live, a.scale_log2);
    const uint32_t limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
    const uint32_t most = wave_max_uniform(limit), least = wave_min_uniform(live ? limit : 0xFFFFFFFFu);
    const size_t bh = (size_t)b * a.c.heads + head;
    const uint8_t *k = a.c.k + bh * a.c.blocks * (size_t)(32 * D), *v = a.c.v + bh * a.c.blocks * (size_t)(32 * D);
    const float *ks = a.c.ks + bh * a.c.blocks, *vs = a.c.vs + bh * a.c.blocks;
    f32x16 o[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.0f, vref = 0.0f;
    for (uint32_t blk = 0; blk * 32 < most; ++blk) {
        u32x4 kw[NS], vw[NS];
        load_units<NS>(kw, k + (size_t)blk * (32 * D));
        load_units<NS>(vw, v + (size_t)blk * (32 * D));
        const float kscale = ks[blk], vscale = vs[blk];
        f32x16 p = key_product<NS, E4M3>(kw, q);
        const float c = q.c * kscale;
        const bool edge = blk * 32 + 32 > least;
        const uint32_t room = limit > blk * 32 ? limit - blk * 32 : 0u;  // slots of this block that the row sees
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            p[i] *= c;
            if (edge && 8 * (i >> 2) + 4 * h + (i & 3) >= room) p[i] = -INFINITY;
            top = fmaxf(top, p[i]);
        }
        top = fmaxf(top, xchg32(top, lane));
        const float m1 = fmaxf(m, top);
        const float base = m1 == -INFINITY ? 0.0f : m1;  // nothing seen yet: every 2^(-inf - 0) is 0
        float down = __builtin_amdgcn_exp2f(m - base);
        m = m1;
        // the values' scale relative to the largest so far: what enters the product in fp16 stays within [0, 1]
        float sum = 0.0f;
        l *= down;
        if (vscale > vref && vscale < INFINITY) {
            down *= vref / vscale;
            vref = vscale;
        }
        const float vrel = vref > 0.0f ? vscale / vref : (vscale == 0.0f ? 0.0f : vscale);
        f16x8_t pf[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(p[i] - base);
            sum += e;
            float w = e * vrel;
            if (edge && 8 * (i >> 2) + 4 * h + (i & 3) >= room) w = 0.0f;  // also where the block stands for NaN
            pf[(i >> 2) & 1][(i >> 3) * 4 + (i & 3)] = (_Float16)w;
        }
        l += sum;
#pragma unroll
        for (int d = 0; d < NS; ++d) {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= down;
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kv8_operand<E4M3>(vw[d].x, vw[d].y), pf[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kv8_operand<E4M3>(vw[d].z, vw[d].w), pf[1], o[d], 0, 0, 0);
        }
    }
    if (!live) return;
    l += xchg32(l, lane);
    if (a.lse && h == 0) a.lse[(size_t)t * a.q_heads + qh] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
    const float w = l == 0.0f ? 0.0f : vref / l;
    uint16_t *out = a.out + ((size_t)t * a.q_heads + qh) * D;
#pragma unroll
    for (int d = 0; d < NS; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x2 y = {pack_bf16_rne(o[d][4 * i] * w, o[d][4 * i + 1] * w),
                             pack_bf16_rne(o[d][4 * i + 2] * w, o[d][4 * i + 3] * w)};
            *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * i + 4 * h) = y;
        }
}

// A wave per block of 32 slots of one sequence and kv head: its keys stay in registers, the query rows that see it
// pass by in tiles of 32, and lane (column, h) adds up its own rows' probabilities of slots 8 i + 4 h + j; the 32
// columns are summed at the end.
template <int NS, int E4M3>
__global__ __launch_bounds__(256) void kv8_weight_kernel(Kv8AttnArgs a) {
    constexpr uint32_t D = 32 * NS;
    const uint32_t lane = __lane_id(), h = lane >> 5;
    const uint32_t head = blockIdx.y, b = blockIdx.z, blk = blockIdx.x * 4 + (threadIdx.x >> 6);
    const Kv8Span s = kv8_span(a.step, b);
    const uint32_t n = min(s.n, a.c.max_ctx), p0 = blk * 32;
    if (p0 >= n) return;
    const size_t bh = (size_t)b * a.c.heads + head;
    u32x4 kw[NS];
    load_units<NS>(kw, a.c.k + (bh * a.c.blocks + blk) * (size_t)(32 * D));
    const float kscale = a.c.ks[bh * a.c.blocks + blk];
    const uint32_t old = s.n > s.m ? s.n - s.m : 0u;  // tokens before the new ones
    float acc[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    // token i sees slots up to n - m + i: the first that sees this block
    const uint32_t i0 = p0 + s.m >= s.n ? p0 + s.m - s.n : 0u;
    const uint32_t rows = s.m * a.group;
    for (uint32_t r0 = i0 * a.group / 32 * 32; r0 < rows; r0 += 32) {
        const uint32_t r = r0 + (lane & 31);
        const bool live = r < rows;
        const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
        QueryRow<NS> q;
        load_query<NS>(q, a.q + t * a.q_stride + (size_t)qh * D, live, a.scale_log2);
        const uint32_t limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
        const uint32_t room = limit > p0 ? limit - p0 : 0u;
        const float lse = live ? a.lse[(size_t)t * a.q_heads + qh] * kLog2e : 0.0f;
        const f32x16 p = key_product<NS, E4M3>(kw, q);
        const float c = q.c * kscale;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(p[i], c, -lse));
            if (8 * (i >> 2) + 4 * h + (i & 3) < room) acc[i] += e;
        }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int x = 1; x < 32; x *= 2) acc[i] += __shfl_xor(acc[i], x);
    float *w = a.weight + bh * a.c.max_ctx;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t p = p0 + 8 * (i >> 2) + 4 * h + (i & 3);
        if ((lane & 31) == i && p < n) w[p] = (p < old ? a.decay * w[p] : 0.0f) + acc[i];
    }
}

size_t kv8_attention_workspace_bytes(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens) {
    return 0;
}

namespace {

template <class F>
hipError_t by_shape(const Kv8 &c, F &&f) {
    const auto dim = [&](auto e) -> hipError_t {
        switch (c.D) {
            case 64: return f(std::integral_constant<int, 2>{}, e);
            case 96: return f(std::integral_constant<int, 3>{}, e);
            case 128: return f(std::integral_constant<int, 4>{}, e);
            case 192: return f(std::integral_constant<int, 6>{}, e);
            default: return f(std::integral_constant<int, 8>{}, e);
        }
    };
    return c.e4m3 ? dim(std::integral_constant<int, 1>{}) : dim(std::integral_constant<int, 0>{});
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8AttnArgs &a, hipStream_t s) {
    // 32-row tiles of every sequence: at most one that is not full each
    const uint32_t items = (uint32_t)((uint64_t)a.step.tokens * a.group / 32) + std::min(a.c.batch, a.step.tokens);
    return by_shape(a.c, [&](auto ns, auto e4m3) {
        kv8_attention_kernel<decltype(ns)::value, decltype(e4m3)::value>
            <<<dim3((items + 3) / 4, a.c.heads), 256, 0, s>>>(a, items);
        return hipGetLastError();
    });
}

hipError_t launch_kv8_weight(const Kv8AttnArgs &a, hipStream_t s) {
    return by_shape(a.c, [&](auto ns, auto e4m3) {
        kv8_weight_kernel<decltype(ns)::value, decltype(e4m3)::value>
            <<<dim3((a.c.blocks + 3) / 4, a.c.heads, a.c.batch), 256, 0, s>>>(a);
        return hipGetLastError();
    });
}

}  // namespace kr
