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

// A part of a context that is split over workgroups: its blocks, and the parts in use.
struct Part {
    uint32_t first, end, parts;
};
// All parts in use but the last have the same number of blocks, a multiple of `unit`.
__device__ __forceinline__ Part part_of(uint32_t blocks, uint32_t most, uint32_t part, uint32_t unit) {
    const uint32_t per = max(((blocks + most - 1) / most + unit - 1) / unit * unit, unit);
    return Part{min(part * per, blocks), min((part + 1) * per, blocks), (blocks + per - 1) / per};
}

// Where a part's normalised O of a query row lies in the workspace, in rows; its m and l in pairs behind all of them.
__device__ __forceinline__ size_t part_at(uint32_t item, uint32_t heads, uint32_t head, uint32_t parts, uint32_t part,
                                          uint32_t tile_rows, uint32_t row) {
    return (((size_t)item * heads + head) * parts + part) * tile_rows + row;
}

constexpr uint32_t kMostParts = 512;

// A value that every lane holds, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

__device__ __forceinline__ uint32_t wave_max_uniform(uint32_t v) { return wave_max_u32(v); }
__device__ __forceinline__ uint32_t wave_min_uniform(uint32_t v) { return ~wave_max_u32(~v); }

}  // namespace

// ---- many rows: prompts and chunks
//
// A workgroup of four waves takes 128 query rows, 32 a wave, and walks the blocks that they see, kTileBlocks<NS> at a time:
// every wave turns its share of the bytes into fp16 operands in LDS once for all four (a wave unpacking for itself would
// spend more vector cycles on it than the matrix cores take), each as the 16 bytes a lane that an operand load takes.
constexpr uint32_t kManyRows = 128;
template <int NS>
constexpr int kTileBlocks = NS <= 2 ? 4 : (NS <= 4 ? 2 : 1);

template <int NS, int E4M3>
__global__ __launch_bounds__(256, NS <= 4 ? 2 : 1) void kv8_many_kernel(Kv8AttnArgs a, uint32_t items, uint32_t parts) {
    constexpr uint32_t D = 32 * NS;
    constexpr int SB = kTileBlocks<NS>, kUnits = SB * 2 * NS / 4;  // 1 KB pieces of a tile that a wave takes
    static_assert(SB * 2 * NS % 4 == 0, "whole pieces a wave");
    __shared__ u32x4 lds[SB][2][2 * NS][64];
    const uint32_t lane = __lane_id(), h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Work order: heads side by side (with eight of them each XCD's L2 keeps one), a sequence's last tiles, which see the most,
    // first; every second round of 256 workgroups reversed, so that a compute unit's workgroups add up to about the same.
    uint32_t idx = blockIdx.x;
    const uint32_t round = idx / 256;
    if (round & 1) idx = round * 256 + min(gridDim.x - round * 256, 256u) - 1 - idx % 256;
    const uint32_t head = idx % a.c.heads, rest = idx / a.c.heads, part = rest % parts, item = rest / parts;
    uint32_t b, tile;
    if (!kv8_find(item, a.c.batch, [&](uint32_t i) { return (kv8_span(a.step, i).m * a.group + kManyRows - 1) / kManyRows; }, b, tile)) return;
    const Kv8Span s = kv8_span(a.step, b);
    const uint32_t rows = s.m * a.group, tiles = (rows + kManyRows - 1) / kManyRows;
    const uint32_t tile_in_work = tile;
    tile = tiles - 1 - tile_in_work;
    const uint32_t r0 = kManyRows * tile, r = r0 + 32 * wave + (lane & 31);
    const bool live = r < rows;
    const uint32_t limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
    const uint32_t most = row_limit(s, min(r0 + kManyRows, rows) - 1, a.group, a.c.max_ctx);
    const uint32_t wave_most = wave_max_uniform(limit), wave_least = wave_min_uniform(live ? limit : 0xFFFFFFFFu);
    const Part w = part_of((most + 31) / 32, parts, part, SB);
    if (part > 0 && part >= w.parts) return;
    const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    QueryRow<NS> q;
    load_query<NS>(q, a.q + t * a.q_stride + (size_t)qh * D, live, a.scale_log2);
    const size_t bh = (size_t)b * a.c.heads + head;
    const uint8_t *k = a.c.k + bh * a.c.blocks * (size_t)(32 * D), *v = a.c.v + bh * a.c.blocks * (size_t)(32 * D);
    const float *ks = a.c.ks + bh * a.c.blocks, *vs = a.c.vs + bh * a.c.blocks;
    f32x16 o[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) o[i] = f32x16{};
    float base = -1e38f, l = 0.0f, vref = 0.0f;
    u32x4 piece[kUnits];
    float kscale[SB], vscale[SB];
    const auto fetch = [&](uint32_t blk) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const uint32_t u = wave + 4 * i, sb = u / (2 * NS), kv = u / NS % 2, j = u % NS;
            if (blk + sb < w.end)
                piece[i] = *reinterpret_cast<const u32x4 *>((kv ? v : k) + (size_t)(blk + sb) * (32 * D) + 1024 * j + 16 * lane);
        }
#pragma unroll
        for (int i = 0; i < SB; ++i) {
            const uint32_t at = min(blk + i, w.end - 1);
            kscale[i] = ks[at];
            vscale[i] = vs[at];
        }
    };
    // One block: its operands in LDS, its first slot p0.  kEdge: a row sees it in part, or it stands for NaN; then the
    // scores are masked one by one.
    const auto block = [&](auto edge, const u32x4 (*kl)[64], const u32x4 (*vl)[64], float kscale, float vscale, uint32_t p0) {
        constexpr bool kEdge = decltype(edge)::value;
        f32x16 p = {};
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j)
            p = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, kl[j][lane]), q.f[j], p, 0, 0, 0);
        float c = q.c * kscale;
        const uint32_t room = limit > p0 ? limit - p0 : 0u;  // slots of this block that the row sees
        if constexpr (kEdge) {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = 8 * (i >> 2) + 4 * h + (i & 3) < room ? p[i] * c : -INFINITY;
            c = 1.0f;
        }
        float top = fmaxf(fmaxf(p[0], p[1]), p[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) top = fmaxf(fmaxf(top, p[i]), p[i + 1]);
        top = fmaxf(top, p[15]) * c;
        top = fmaxf(top, xchg32(top, lane));
        // The base of the exponents follows the maximum only when it is passed by 2^8: the probabilities stay within fp16, and
        // O is scaled down a few times in all.  The values' scale relative to the largest so far joins the exponent: what
        // enters the second product stays in range, and l takes it out again.
        const bool finite = vscale < INFINITY;
        if (__any(top > base + 8.0f) || (finite && vscale > vref)) {
            const float base1 = fmaxf(base, top);
            float down = __builtin_amdgcn_exp2f(base - base1);
            base = base1;
            l *= down;
            if (finite && vscale > vref) {
                down *= vref / vscale;
                vref = vscale;
            }
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= down;
        }
        // a block of zeros (scale 0) has no values to keep in range; below 2^-30 of the largest the scale is held there
        const float shift = finite && vscale > 0.0f ? fmaxf(__log2f(vscale / vref), -30.0f) : 0.0f;
        const float from = base - shift;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], c, -from));
            sum += p[i];
        }
        l = fmaf(sum, __builtin_amdgcn_exp2f(-shift), l);
        if constexpr (kEdge) {
            if (!finite) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (8 * (i >> 2) + 4 * h + (i & 3) < room) p[i] = __builtin_nanf("");
            }
        }
        f16x8_t pf[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) pf[(i >> 2) & 1][(i >> 3) * 4 + (i & 3)] = (_Float16)p[i];
#pragma unroll
        for (int d = 0; d < NS; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vl[2 * d][lane]), pf[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vl[2 * d + 1][lane]), pf[1], o[d], 0, 0, 0);
        }
    };
    if (w.first < w.end) fetch(w.first);
    for (uint32_t blk = w.first; blk < w.end; blk += SB) {
        __syncthreads();  // the tile before has been read
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const uint32_t u = wave + 4 * i, sb = u / (2 * NS), kv = u / NS % 2, j = u % NS;
            lds[sb][kv][2 * j][lane] = __builtin_bit_cast(u32x4, kv8_operand<E4M3>(piece[i].x, piece[i].y));
            lds[sb][kv][2 * j + 1][lane] = __builtin_bit_cast(u32x4, kv8_operand<E4M3>(piece[i].z, piece[i].w));
        }
        float kc[SB], vc[SB];
#pragma unroll
        for (int i = 0; i < SB; ++i) {
            kc[i] = uniform(kscale[i]);
            vc[i] = uniform(vscale[i]);
        }
        __syncthreads();
        if (blk + SB < w.end) fetch(blk + SB);
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) {
            const uint32_t p0 = (blk + sb) * 32;
            if (blk + sb >= w.end || p0 >= wave_most) break;
            if (p0 + 32 > wave_least || !(vc[sb] < INFINITY))
                block(std::true_type{}, lds[sb][0], lds[sb][1], kc[sb], vc[sb], p0);
            else
                block(std::false_type{}, lds[sb][0], lds[sb][1], kc[sb], vc[sb], p0);
        }
    }
    if (!live) return;
    l += xchg32(l, lane);
    const float norm = l == 0.0f ? 0.0f : vref / l;
    if (parts == 1) {
        const size_t at = (size_t)t * a.q_heads + qh;
        if (a.lse && h == 0) a.lse[at] = l == 0.0f ? -INFINITY : (base + __log2f(l)) * kLn2;
        uint16_t *out = a.out + at * D;
#pragma unroll
        for (int d = 0; d < NS; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x2 y = {pack_bf16_rne(o[d][4 * i] * norm, o[d][4 * i + 1] * norm),
                                 pack_bf16_rne(o[d][4 * i + 2] * norm, o[d][4 * i + 3] * norm)};
                *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * i + 4 * h) = y;
            }
    } else {
        // the workspace is in the order of the tiles, not of the work
        const size_t at = part_at(item - tile_in_work + tile, a.c.heads, head, parts, part, kManyRows, r - r0);
#pragma unroll
        for (int d = 0; d < NS; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f32x4 *>(a.part + at * D + 32 * d + 8 * i + 4 * h) =
                    f32x4{o[d][4 * i] * norm, o[d][4 * i + 1] * norm, o[d][4 * i + 2] * norm, o[d][4 * i + 3] * norm};
        if (h == 0) {
            float *ml = a.part + (size_t)items * parts * a.c.heads * kManyRows * D + 2 * at;
            ml[0] = base;
            ml[1] = l;
        }
    }
}

// ---- few rows: the context split over workgroups
//
// A workgroup takes one tile of 16 query rows and one part of the sequence's blocks, its four waves every fourth block of
// the part; each wave keeps its own m, l and O, and they are joined in LDS. With more than one part the normalised
// O_s and (m_s, l_s) go to the workspace and kv8_join_kernel joins the parts in order:
//   out = sum_s 2^(m_s - M) l_s O_s / L,   L = sum_s 2^(m_s - M) l_s
// On v_mfma_f32_16x16x32_f16: lane (column l & 15, g = l >> 4) holds slots 16 t + 4 g + j after the first product, and
// needs of dim d the slots 16 s + 4 g + j for the second, eight bytes of v's order (h = g & 1, a = g >> 1).
constexpr uint32_t kFewRows = 16, kFewWaves = 4;

template <int NS>
__device__ __forceinline__ void load_query16(f16x8_t (&f)[NS], float &c, const uint16_t *row, bool live, float scale_log2) {
    const uint32_t lane = __lane_id(), g = lane >> 4;
    u32x4 raw[NS];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        raw[i] = u32x4{0, 0, 0, 0};
        // steps 2 j, 2 j + 1 cover 64 dims, 16 a lane; the last of an odd number 32, 8 a lane
        const uint32_t d = (NS & 1) && i == NS - 1 ? 32 * i + 8 * g : 64 * (i / 2) + 16 * g + 8 * (i & 1);
        if (live) raw[i] = *reinterpret_cast<const u32x4 *>(row + d);
        top = max(top, bf16_unit_max_bits(raw[i]));
    }
    top = max(top, (uint32_t)__float_as_uint(xchg32(__uint_as_float(top), lane)));
    top = max(top, (uint32_t)__float_as_uint(xchg16(__uint_as_float(top), lane)));
    const int e = row_stage_exp(top, 14, 14, 14);
    const float up = exp2_int(e);
    c = scale_log2 * exp2_int(-e);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const uint32_t W[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            f[i][2 * x] = (_Float16)(__uint_as_float(W[x] << 16) * up);
            f[i][2 * x + 1] = (_Float16)(__uint_as_float(W[x] & 0xFFFF0000u) * up);
        }
    }
}

// The bytes of one block as a wave's lanes take them.
template <int NS>
struct FewBlock {
    u32x4 k[2][NS / 2 > 0 ? NS / 2 : 1];  // [half of the slots][64 dims]
    u32x2 ke[2];                          // the last 32 dims of an odd number
    u32x2 v[2 * NS];                      // [16 dims]
    float ks, vs;
};
template <int NS>
__device__ __forceinline__ void load_few(FewBlock<NS> &f, const uint8_t *k, const uint8_t *v, const float *ks, const float *vs,
                                         uint32_t blk) {
    const uint32_t lane = __lane_id(), r = lane & 15, g = lane >> 4;
    k += (size_t)blk * (1024 * NS);
    v += (size_t)blk * (1024 * NS);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int j = 0; j < NS / 2; ++j)
            f.k[t][j] = *reinterpret_cast<const u32x4 *>(k + 512 * (4 * j + g) + 16 * (16 * t + r));
        if constexpr (NS & 1)
            f.ke[t] = *reinterpret_cast<const u32x2 *>(k + 512 * (2 * (NS - 1) + g / 2) + 16 * (16 * t + r) + 8 * (g & 1));
    }
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d)
        f.v[d] = *reinterpret_cast<const u32x2 *>(v + 1024 * (d / 2) + 512 * (g & 1) + 16 * (16 * (d & 1) + r) + 8 * (g >> 1));
    f.ks = ks[blk];
    f.vs = vs[blk];
}

template <int NS, int E4M3>
__global__ __launch_bounds__(256) void kv8_few_kernel(Kv8AttnArgs a, uint32_t parts) {
    constexpr uint32_t D = 32 * NS;
    __shared__ float sm[kFewWaves][kFewRows], sl[kFewWaves][kFewRows];
    __shared__ float so[kFewWaves][kFewRows][D + 4];
    const uint32_t lane = __lane_id(), r16 = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t head = blockIdx.y, item = blockIdx.x / parts, part = blockIdx.x % parts;
    uint32_t b, tile;
    if (!kv8_find(item, a.c.batch, [&](uint32_t i) { return (kv8_span(a.step, i).m * a.group + kFewRows - 1) / kFewRows; }, b, tile)) return;
    const Kv8Span s = kv8_span(a.step, b);
    const uint32_t rows = s.m * a.group, r = kFewRows * tile + r16;
    const bool live = r < rows;
    const uint32_t limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
    const uint32_t most = row_limit(s, min(kFewRows * tile + kFewRows, rows) - 1, a.group, a.c.max_ctx);
    const uint32_t least = row_limit(s, kFewRows * tile, a.group, a.c.max_ctx);
    const Part w = part_of((most + 31) / 32, parts, part, kFewWaves);
    if (part > 0 && part >= w.parts) return;
    const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    f16x8_t q[NS];
    float qc;
    load_query16<NS>(q, qc, a.q + t * a.q_stride + (size_t)qh * D, live, a.scale_log2);
    const size_t bh = (size_t)b * a.c.heads + head;
    const uint8_t *k = a.c.k + bh * a.c.blocks * (size_t)(32 * D), *v = a.c.v + bh * a.c.blocks * (size_t)(32 * D);
    const float *ks = a.c.ks + bh * a.c.blocks, *vs = a.c.vs + bh * a.c.blocks;
    f32x4 o[2 * NS];
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f, vref = 0.0f;
    uint32_t blk = w.first + wave;
    FewBlock<NS> f;
    if (blk < w.end) load_few<NS>(f, k, v, ks, vs, blk);
    for (; blk < w.end; blk += kFewWaves) {
        f32x4 p[2] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NS / 2; ++j) {
                p[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv8_operand<E4M3>(f.k[h][j].x, f.k[h][j].y), q[2 * j], p[h], 0, 0, 0);
                p[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv8_operand<E4M3>(f.k[h][j].z, f.k[h][j].w), q[2 * j + 1], p[h], 0, 0, 0);
            }
            if constexpr (NS & 1)
                p[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv8_operand<E4M3>(f.ke[h].x, f.ke[h].y), q[NS - 1], p[h], 0, 0, 0);
        }
        f16x8_t vf[2 * NS];
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) vf[d] = kv8_operand<E4M3>(f.v[d].x, f.v[d].y);
        const float c = qc * f.ks, vscale = f.vs;
        if (blk + kFewWaves < w.end) load_few<NS>(f, k, v, ks, vs, blk + kFewWaves);
        const bool edge = blk * 32 + 32 > least;
        const uint32_t room = limit > blk * 32 ? limit - blk * 32 : 0u;
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float x = p[i >> 2][i & 3] * c;
            if (edge && 16 * (i >> 2) + 4 * g + (i & 3) >= room) x = -INFINITY;
            p[i >> 2][i & 3] = x;
            top = fmaxf(top, x);
        }
        top = fmaxf(top, xchg32(top, lane));
        top = fmaxf(top, xchg16(top, lane));
        const float m1 = fmaxf(m, top);
        const float base = m1 == -INFINITY ? 0.0f : m1;
        float down = __builtin_amdgcn_exp2f(m - base);
        m = m1;
        l *= down;
        if (vscale > vref && vscale < INFINITY) {
            down *= vref / vscale;
            vref = vscale;
        }
        const float vrel = vref > 0.0f ? vscale / vref : (vscale == 0.0f ? 0.0f : vscale);
        f16x8_t pf;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(p[i >> 2][i & 3] - base);
            l += e;
            float x = e * vrel;
            if (edge && 16 * (i >> 2) + 4 * g + (i & 3) >= room) x = 0.0f;
            pf[i] = (_Float16)x;
        }
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][i] *= down;
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d], pf, o[d], 0, 0, 0);
        }
    }
    l += xchg32(l, lane);
    l += xchg16(l, lane);
    const float norm = l == 0.0f ? 0.0f : vref / l;
    if (g == 0) {
        sm[wave][r16] = m;
        sl[wave][r16] = l;
    }
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d)
        *reinterpret_cast<f32x4 *>(&so[wave][r16][16 * d + 4 * g]) = o[d] * norm;
    __syncthreads();
    // four dims of a row a thread
    for (uint32_t i = threadIdx.x; i < kFewRows * (D / 4); i += 256) {
        const uint32_t row = i / (D / 4), d = i % (D / 4) * 4, rr = kFewRows * tile + row;
        if (rr >= rows) continue;
        float M = sm[0][row], L = 0.0f;
#pragma unroll
        for (uint32_t x = 1; x < kFewWaves; ++x) M = fmaxf(M, sm[x][row]);
        f32x4 acc = {0, 0, 0, 0};
        bool nan = false;
#pragma unroll
        for (uint32_t x = 0; x < kFewWaves; ++x) {
            const float lx = sl[x][row];
            nan |= lx != lx;
            if (lx > 0.0f) {  // a wave that saw no slot has nothing to add
                const float wx = lx * __builtin_amdgcn_exp2f(sm[x][row] - M);
                L += wx;
                acc += wx * *reinterpret_cast<const f32x4 *>(&so[x][row][d]);
            }
        }
        if (nan) L = __builtin_nanf("");
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        acc *= inv;
        if (parts == 1) {
            const uint32_t tt = s.t0 + rr / a.group, hh = head * a.group + rr % a.group;
            const size_t at = (size_t)tt * a.q_heads + hh;
            const u32x2 y = {pack_bf16_rne(acc.x, acc.y), pack_bf16_rne(acc.z, acc.w)};
            *reinterpret_cast<u32x2 *>(a.out + at * D + d) = y;
            if (a.lse && d == 0) a.lse[at] = L == 0.0f ? -INFINITY : (M + __log2f(L)) * kLn2;
        } else {
            const size_t at = part_at(item, a.c.heads, head, parts, part, kFewRows, row);
            *reinterpret_cast<f32x4 *>(a.part + at * D + d) = acc;
            if (d == 0) {
                float *ml = a.part + (size_t)gridDim.x * a.c.heads * kFewRows * D + 2 * at;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
}

// A workgroup per query row: thread (i, j) adds up parts i, i + n, ... of four dims, then the n sums are joined.
template <int NS>
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8AttnArgs a, uint32_t items, uint32_t parts, uint32_t tile_rows,
                                                       uint32_t unit) {
    constexpr uint32_t D = 32 * NS, kQuads = D / 4, kWays = 256 / kQuads;
    __shared__ float red[4], wl[kMostParts];
    __shared__ f32x4 so[kWays][kQuads];
    const uint32_t head = blockIdx.y, item = blockIdx.x / tile_rows, row = blockIdx.x % tile_rows;
    uint32_t b, tile;
    if (!kv8_find(item, a.c.batch, [&](uint32_t i) { return (kv8_span(a.step, i).m * a.group + tile_rows - 1) / tile_rows; }, b, tile)) return;
    const Kv8Span s = kv8_span(a.step, b);
    const uint32_t rows = s.m * a.group, r = tile_rows * tile + row;
    if (r >= rows) return;
    const uint32_t most = row_limit(s, min(tile_rows * tile + tile_rows, rows) - 1, a.group, a.c.max_ctx);
    const uint32_t used = max(part_of((most + 31) / 32, parts, 0, unit).parts, 1u);
    const size_t at = part_at(item, a.c.heads, head, parts, 0, tile_rows, row);  // part p: at + p tile_rows
    const float *ml = a.part + (size_t)items * parts * a.c.heads * tile_rows * D;
    // weights of the parts, relative to the largest m
    const uint32_t tid = threadIdx.x;
    float mx = -INFINITY;
    for (uint32_t p = tid; p < used; p += 256) mx = fmaxf(mx, ml[2 * (at + (size_t)p * tile_rows)]);
    mx = wave_max(mx);
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    for (uint32_t p = tid; p < used; p += 256) {
        const float *x = ml + 2 * (at + (size_t)p * tile_rows);
        const float lx = x[1];
        wl[p] = lx == 0.0f ? 0.0f : lx * __builtin_amdgcn_exp2f(x[0] - M);  // NaN stays
    }
    __syncthreads();
    float L = 0.0f;
    for (uint32_t p = 0; p < used; ++p) L += wl[p];
    const uint32_t way = tid / kQuads, quad = tid % kQuads;
    if (way < kWays) {
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
        for (uint32_t p = way; p < used; p += kWays)
            acc += wl[p] * *reinterpret_cast<const f32x4 *>(a.part + (at + (size_t)p * tile_rows) * D + 4 * quad);
        so[way][quad] = acc;
    }
    __syncthreads();
    if (tid < kQuads) {
        f32x4 acc = so[0][tid];
#pragma unroll
        for (uint32_t i = 1; i < kWays; ++i) acc += so[i][tid];
        acc *= L == 0.0f ? 0.0f : 1.0f / L;
        const size_t to = (size_t)(s.t0 + r / a.group) * a.q_heads + head * a.group + r % a.group;
        const u32x2 y = {pack_bf16_rne(acc.x, acc.y), pack_bf16_rne(acc.z, acc.w)};
        *reinterpret_cast<u32x2 *>(a.out + to * D + 4 * tid) = y;
        if (a.lse && tid == 0) a.lse[to] = L == 0.0f ? -INFINITY : (M + __log2f(L)) * kLn2;
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

namespace {

// How a step is launched: tiles of 16 rows where the sequences have few query rows (one or two tokens of a group of
// heads), else of 128; and the parts that a context is split into, so that there are workgroups for the whole card.
struct AttnPlan {
    bool few;
    uint32_t rows, items, parts;
};
AttnPlan plan_of(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t tokens) {
    AttnPlan p;
    p.few = (uint64_t)tokens * group <= 32ull * batch;
    p.rows = p.few ? kFewRows : kManyRows;
    // tiles of every sequence: at most one that is not full each
    p.items = (uint32_t)((uint64_t)tokens * group / p.rows) + std::min(batch, tokens);
    const uint64_t tiles = (uint64_t)p.items * kv_heads, want = p.few ? 1024 : 512;
    p.parts = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(kMostParts, want / tiles));
    return p;
}

}  // namespace

size_t kv8_attention_workspace_bytes(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens) {
    const AttnPlan p = plan_of(batch, kv_heads, group, tokens);
    return p.parts == 1 ? 0 : (size_t)p.items * kv_heads * p.parts * p.rows * (D + 2) * sizeof(float);
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
    const AttnPlan p = plan_of(a.c.batch, a.c.heads, a.group, a.step.tokens);
    return by_shape(a.c, [&](auto ns, auto e4m3) -> hipError_t {
        constexpr int NS = decltype(ns)::value, E4M3 = decltype(e4m3)::value;
        if (p.few)
            kv8_few_kernel<NS, E4M3><<<dim3(p.items * p.parts, a.c.heads), 256, 0, s>>>(a, p.parts);
        else
            kv8_many_kernel<NS, E4M3><<<dim3(p.items * p.parts * a.c.heads), 256, 0, s>>>(a, p.items, p.parts);
        if (hipError_t e = hipGetLastError()) return e;
        if (p.parts == 1) return hipSuccess;
        kv8_join_kernel<NS><<<dim3(p.items * p.rows, a.c.heads), 256, 0, s>>>(a, p.items, p.parts, p.rows,
                                                                             p.few ? kFewWaves : kTileBlocks<NS>);
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
