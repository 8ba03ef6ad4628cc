// paged_attention.hip — attention over the paged key/value cache: one new token a sequence, whole prompts, and trees of drafted
// tokens.
//
// Reference semantics (grouped query heads over pages, causal at the end of the context or by a tree's mask):
//   kernels/metal/paged_gqa_and_deltanet.metal:242 and the prefill and tree kernels beside it
//
// Mathematics.  The query rows of a sequence and kv head are r = i group + g (token i, head g of the group): every key and value is
// used for the whole group.  In base 2, with c = |scale| log2(e) and the sign of scale in q:
//   s_rp = q_r . k_p,   m_r = max_p c s_rp,   l_r = sum_p 2^(c s_rp - m_r),   out_r = sum_p 2^(c s_rp - m_r) v_p / l_r
// One pass over the slots: m_r only grows, and sums made under an older one are scaled down.  The exponents are one fused
// multiply-add from the product's f32 sums, so that large scores cost no more than their own rounding.  Probabilities enter the second
// product as bf16, as the values are (the matrix cores take f32 at a fraction of the rate, and fp16 cannot hold all values); l_r sums them
// unrounded, in f32.
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a lane then holds one query row, its m_r and l_r are plain
// registers, and after rounding its probabilities are the second product's operand as they lie (paged.hpp: the order of v).
#include <algorithm>

#include "attn_work.hpp"
#include "paged.hpp"

namespace kr {

namespace {

constexpr uint32_t kAll = 0xFFFFFFFFu;
constexpr float kNoBase = -2e38f, kLowBase = -1e38f;  // of a row that has seen nothing; at least that of one that has
static_assert(kNoBase < kSeenBase && kSeenBase < kLowBase);

// The lowest `n` bits.
__device__ __forceinline__ uint32_t low_bits(uint32_t n) { return n >= 32 ? kAll : (1u << n) - 1; }

// Which slots p0 .. p0 + 31 row r of sequence span s sees, as bits.
struct Sight {
    uint32_t limit;              // causal: slots below it
    uint32_t old, cut, n;        // mask: slots of the tokens before the step (old; cut nodes have no slot), and of all
    const uint32_t *row;         // nullptr: causal
    uint32_t words;
    __device__ __forceinline__ uint32_t word(uint32_t i) const { return i < words ? row[i] : 0u; }
    __device__ __forceinline__ uint32_t bits(uint32_t p0) const {
        if (!row) return low_bits(limit > p0 ? limit - p0 : 0u);
        uint32_t seen = kAll;
        if (p0 + 32 > old) {
            const int32_t node = (int32_t)(p0 - old + cut);  // of slot p0, -31 at least
            if (node < 0) {
                seen = low_bits((uint32_t)-node) | word(0) << -node;
            } else {
                const uint32_t i = (uint32_t)node / 32, x = (uint32_t)node % 32;
                seen = word(i) >> x;
                if (x) seen |= word(i + 1) << (32 - x);
            }
        }
        return seen & low_bits(n > p0 ? n - p0 : 0u);
    }
};
__device__ __forceinline__ Sight sight_of(const PagedAttnArgs &a, const Span &s, uint32_t r, bool live) {
    Sight v{};
    v.limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
    if (a.mask) {
        v.row = a.mask + (size_t)(live ? s.t0 + r / a.group : 0u) * a.words;
        v.words = a.words;
        v.old = s.n > s.m ? s.n - s.m : 0u;
        v.cut = s.m > s.n ? s.m - s.n : 0u;
        v.n = live ? min(s.n, a.c.max_ctx) : 0u;
    }
    return v;
}
// Slots below this all rows from r0 on see.
__device__ __forceinline__ uint32_t clear_of(const PagedAttnArgs &a, const Span &s, uint32_t r0) {
    return a.mask ? min(s.n > s.m ? s.n - s.m : 0u, a.c.max_ctx) : row_limit(s, r0, a.group, a.c.max_ctx);
}

// The pages of a wave's units in the order in which it asks for them, 64 at a time and the next 64 on their way: lane l of a set
// holds the page of the unit that the wave reads l-th.
template <class F>
struct Pages {
    F load;  // the pages of set i: a value a lane
    uint32_t now, next;
    __device__ __forceinline__ explicit Pages(F f) : load(f), now(f(0)), next(f(1)) {}
    // of the i-th unit; units in rising order, each set entered at its first
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return (uint32_t)__builtin_amdgcn_readlane((int)now, (int)(i & 63)); }
    __device__ __forceinline__ void enter(uint32_t i) {
        if ((i & 63) == 0 && i) {
            now = next;
            next = load(i / 64 + 1);
        }
    }
};

// A row's running sums.
struct RowSums {
    float base = kNoBase, l = 0.0f;
};
// The base lags the maximum by up to 2^8: O is scaled down a few times in all.
constexpr float kLag = 8.0f;
__device__ __forceinline__ float row_follow(RowSums &r, float top) {
    const float base = fmaxf(r.base, top), down = __builtin_amdgcn_exp2f(r.base - base);
    r.base = base;
    r.l *= down;
    return down;
}

// ---- values that are infinite or NaN in slots that some rows do not see
//
// A product with a probability of 0 would bring them into those rows.  In a block that some row does not see whole, they are
// therefore taken out of the operand, and added to the rows that see them one slot at a time.

// Takes them out of a 16-byte piece of values; `bad` gets bit 15 and 31 of a word where its low and high value is one.
__device__ __forceinline__ void take_out(u32x4 &v, u32x4 &bad) {
    // an exponent of all ones, and no other, carries into the sign's bit; from there over its half
    const u32x4 m = ((v & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
    v &= ~((m << 1) - (m >> 15));
    bad |= m;
}
// The slots of a piece's bad words: bits 8 a + j.
__device__ __forceinline__ uint32_t bad_slots(const u32x4 &bad) {
    uint32_t s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) s |= ((bad[i] >> 15 & 1u) | (bad[i] >> 30 & 2u)) << (8 * (i >> 1) + 2 * (i & 1));
    return s;
}
__device__ __forceinline__ uint32_t wave_or(uint32_t v) {
#pragma unroll
    for (int x = 1; x < 64; x *= 2) v |= (uint32_t)__shfl_xor((int)v, x);
    return v;
}
// o plus a value that was taken out.
__device__ __forceinline__ float put_back(float o, uint16_t bits, bool seen) {
    return seen && (bits & 0x7F80u) == 0x7F80u ? o + bf16_to_f32(bits) : o;
}

// Four floats as bf16.
__device__ __forceinline__ u32x2 pack4(float x0, float x1, float x2, float x3) { return u32x2{pack_bf16_rne(x0, x1), pack_bf16_rne(x2, x3)}; }

// Query row: 8 dims, with the scale's sign.
__device__ __forceinline__ bf16x8_t query_unit(const uint16_t *p, bool live, uint32_t sign) {
    u32x4 w = {0, 0, 0, 0};
    if (live) {
        w = *reinterpret_cast<const u32x4 *>(p);
        w ^= u32x4{sign, sign, sign, sign};
    }
    return __builtin_bit_cast(bf16x8_t, w);
}
// The factor of a product's exponent: not 0, so that -infinity stays that (the smallest float takes any score below 2^-21).
__device__ __forceinline__ float score_factor(float scale) { return fmaxf(fabsf(scale), 0x1p-149f); }
__device__ __forceinline__ uint32_t query_sign(float scale) { return scale < 0.0f ? 0x80008000u : 0u; }

}  // namespace

// ---- many rows: prompts, chunks, large trees
constexpr uint32_t kManyRows = 128;

// 16 bytes a lane into LDS, past the registers: lane l's go to lds + 16 l.  lds the same in all lanes.
__device__ __forceinline__ void to_lds(const void *from, void *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

template <int NS>
__global__ __launch_bounds__(256, NS <= 4 ? 2 : 1) void paged_many_kernel(PagedAttnArgs a, Split split, uint32_t slots) {
    constexpr uint32_t D = 32 * NS;
    __shared__ u32x4 lds[2][2][2][NS][64];  // [keys, values][block & 1][unit][1 KB piece][lane]
    const uint32_t lane = __lane_id(), r32 = lane & 31, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // heads side by side: with eight of them each XCD's L2 keeps the keys and values of one
    // every second round of 256 workgroups mirrored: a compute unit's add up to about the same
    uint32_t at = blockIdx.x;
    if (at / 256 & 1) at = at / 256 * 256 + min(gridDim.x - at / 256 * 256, 256u) - 1 - at % 256;
    const uint32_t head = at % a.c.heads, idx = at / a.c.heads;
    const uint32_t share = share_of(a, split);
    uint32_t place = idx * share, left = share;
    const float c = score_factor(a.scale_log2);
    const uint32_t sign = query_sign(a.scale_log2);
    for (uint32_t odd = 0;; odd = 1) {  // the pieces of this workgroup's share
        Work w;
        uint32_t first = 0, end;
        bool whole = true;
        if (share) {
            uint32_t blocks;
            if (left == 0 || !find_place(a, split, place, w, first, blocks)) return;
            const uint32_t take = min(left, blocks - first), seen = (w.most + 31) / 32;
            left -= take;
            place += take;
            end = min(first + take, seen);
            whole = first == 0 && end == seen;
            if (first && first >= seen) continue;
            if (odd) __syncthreads();  // the last piece's blocks have been read
        } else {
            if (odd || !find_item(idx, a.c.batch, [&](uint32_t i) { return tiles_of(a, split, span_of(a.step, i)); }, w.b, w.tile)) return;
            w.tile = tiles_of(a, split, span_of(a.step, w.b)) - 1 - w.tile;  // the tiles that see the most first
            fill_work(a, split, w);
            end = (w.most + 31) / 32;
        }
        const Span &s = w.s;
        const uint32_t r0 = kManyRows * w.tile, r = r0 + 32 * wave + r32;
        const bool live = r < w.rows;
        const Sight sight = sight_of(a, s, r, live);
        const uint32_t clear = clear_of(a, s, r0 + 32 * wave);  // (rows past the end need nothing)
        const uint32_t b = w.b, t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
        bf16x8_t q[2 * NS];
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) q[i] = query_unit(a.q + t * a.q_stride + (size_t)qh * D + 16 * i + 8 * h, live, sign);
        f32x16 o[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) o[i] = f32x16{};
        RowSums sums;
        // the pages of units 2 first ..
        Pages pages([&](uint32_t set) { return page_of(a.c, b, 2 * first + 64 * set + lane); });
        // This wave's pieces of a block's keys or values, into side n & 1.
        const auto request = [&](uint32_t kind, uint32_t n, uint32_t p0, uint32_t p1) {
            const uint16_t *pool = kind ? a.c.v : a.c.k;
#pragma unroll
            for (int i = 0; i < (2 * NS + 3) / 4; ++i) {
                const uint32_t j = min(wave + 4 * i, 2u * NS - 1), unit = j / NS, piece = j % NS;  // (the same one twice where they do not divide)
                const uint32_t page = unit ? p1 : p0;
                const uint16_t *from = pool + unit_at(a.c, page < a.c.pages ? page : 0u, head, 2 * n + unit) + 512 * piece + 8 * lane;
                to_lds(from, &lds[kind][n & 1][unit][piece][0]);
            }
        };
        uint32_t pg[3][2];  // pages of blocks n, n + 1 and n + 2
        const auto pages_of = [&](uint32_t n, uint32_t (&p)[2]) {
            if (n >= end) {  // past the end: nothing reads it
                p[0] = p[1] = 0;
                return;
            }
            const uint32_t i = 2 * (n - first);
            pages.enter(i);
            p[0] = pages.at(i);
            p[1] = pages.at(i + 1);
        };
        f32x16 p;
        bool edge = false;  // the block in work is not seen whole by every row of the wave
        uint32_t seen = 0;  // its slots that the row sees, where it is
        const auto key_steps = [&](uint32_t n) {
            f32x16 x = {};
#pragma unroll
            for (int j = 0; j < 2 * NS; ++j) {
                // octet 2 j + h of slot r32: 256 bytes an octet
                const u32x4 k = lds[0][n & 1][r32 >> 4][j / 2][(j & 1) * 32 + h * 16 + (r32 & 15)];
                x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, k), q[j], x, 0, 0, 0);
            }
            return x;
        };
        const auto enter = [&](uint32_t n, const uint32_t (&pn)[2]) {
            const bool hole0 = pn[0] >= a.c.pages, hole1 = pn[1] >= a.c.pages;
            edge = 32 * n + 32 > clear || hole0 || hole1;
            if (edge) {
                seen = sight.bits(32 * n) & ~((hole0 ? 0xFFFFu : 0u) | (hole1 ? 0xFFFF0000u : 0u));
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = seen >> (8 * (i >> 2) + 4 * h + (i & 3)) & 1 ? p[i] : -INFINITY;
            }
            float top = fmaxf(fmaxf(p[0], p[1]), p[2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) top = fmaxf(fmaxf(top, p[i]), p[i + 1]);
            top = fmaxf(top, p[15]) * c;
            top = fmaxf(top, xchg32(top, lane));
            if (!edge || seen) top = fmaxf(top, kLowBase);
            if (__any(top > sums.base + kLag)) {
                const float down = row_follow(sums, top);
#pragma unroll
                for (int d = 0; d < NS; ++d) o[d] *= down;
            }
        };
        const auto body = [&](auto more, uint32_t n, const uint32_t (&pn)[2]) {
            constexpr bool kMore = decltype(more)::value;
            float sum = 0.0f;
            u32x4 pf[2];
            const bool edge_now = edge;
            const uint32_t seen_now = seen;
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const float e0 = __builtin_amdgcn_exp2f(fmaf(p[i], c, -sums.base)), e1 = __builtin_amdgcn_exp2f(fmaf(p[i + 1], c, -sums.base));
                sum += e0;
                sum += e1;
                pf[i >> 3][(i & 7) >> 1] = pack_bf16_rne(e0, e1);
            }
            sums.l += sum;
            if constexpr (kMore) p = key_steps(n + 1);
            u32x4 vf[2 * NS];
#pragma unroll
            for (int j = 0; j < 2 * NS; ++j) vf[j] = lds[1][n & 1][j & 1][j >> 1][lane];
            uint32_t bad = 0;
            if (edge_now) {
                u32x4 words[2] = {};
#pragma unroll
                for (int j = 0; j < 2 * NS; ++j) take_out(vf[j], words[j & 1]);
                bad = (bad_slots(words[0]) | bad_slots(words[1]) << 16) << (4 * h);
                if (__any(bad)) bad &= wave_or(seen_now);  // (what no row sees is left out)
            }
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[2 * d + x]),
                                                                   __builtin_bit_cast(bf16x8_t, pf[x]), o[d], 0, 0, 0);
            if (edge_now && __any(bad)) {
                for (uint32_t left = wave_or(bad); left; left &= left - 1) {
                    const uint32_t slot = (uint32_t)__builtin_ctz(left), page = slot < 16 ? pn[0] : pn[1];
                    const uint16_t *v = a.c.v + unit_at(a.c, page, head, 2 * n + slot / 16) + paged_value_at(slot % 16, 4 * h);
#pragma unroll
                    for (int d = 0; d < NS; ++d) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            o[d][i] = put_back(o[d][i], v[512 * d + 8 * (8 * (i >> 2) + (i & 3))], seen_now >> slot & 1);
                        __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
                    }
                }
            }
        };
        if (first < end) {
            // keys first and first + 1, values first
            pages_of(first, pg[0]);
            pages_of(first + 1, pg[1]);
            request(0, first, pg[0][0], pg[0][1]);
            if (first + 1 < end) request(0, first + 1, pg[1][0], pg[1][1]);
            request(1, first, pg[0][0], pg[0][1]);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            p = key_steps(first);
            enter(first, pg[0]);
            for (uint32_t n = first; n + 1 < end; ++n) {
                // what body n reads has landed, what it overwrites has been read
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();
                pages_of(n + 2, pg[2]);
                if (n + 2 < end) request(0, n + 2, pg[2][0], pg[2][1]);
                request(1, n + 1, pg[1][0], pg[1][1]);
                body(std::true_type{}, n, pg[0]);
                enter(n + 1, pg[1]);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    pg[0][x] = pg[1][x];
                    pg[1][x] = pg[2][x];
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            body(std::false_type{}, end - 1, pg[0]);
        }
        const float l = sums.l + xchg32(sums.l, lane);
        const float norm = l == 0.0f ? 0.0f : 1.0f / l;
        const bool nan = l == 0.0f && sums.base > kSeenBase;  // saw slots, all with scores of -infinity
#pragma unroll
        for (int d = 0; d < NS; ++d) o[d] *= norm;
        if (!live) {  // (a row past the sequence's)
        } else if (whole) {
            if (nan) {
#pragma unroll
                for (int d = 0; d < NS; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] = __builtin_nanf("");
            }
            const size_t to = (size_t)t * a.q_heads + qh;
            if (a.lse && h == 0) a.lse[to] = l == 0.0f ? (nan ? __builtin_nanf("") : -INFINITY) : (sums.base + __log2f(l)) * kLn2;
            uint16_t *out = a.out + to * D;
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * i + 4 * h) = pack4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
        } else {
            const size_t to = part_at(a, split, 2 * idx + odd, head, r - r0);
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4 *>(a.part + to * D + 32 * d + 8 * i + 4 * h) =
                        f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (h == 0) {
                float *ml = a.part + (size_t)slots * a.c.heads * kManyRows * D + 2 * to;
                ml[0] = sums.base;
                ml[1] = l;
            }
        }
    }
}

// ---- few rows: the context split over workgroups
//
// A workgroup takes one tile of 16 query rows and one part of the sequence's blocks of 32 slots, its four waves every fourth block of
// the part; each wave keeps its own m, l and O, and they are joined in LDS.  With more than one part the normalised O_s and (m_s, l_s)
// go to the workspace and attn_join_kernel joins the parts in order.
// On v_mfma_f32_16x16x32_bf16, keys and values straight from memory to the operands' registers, 16 bytes a lane in whole cache lines.
// Tile t of a block's keys is slots 8 t .. 8 t + 7 of both units: a lane (column l & 15, g = l >> 4) then holds after the first product
// the slots 8 t + 4 (g & 1) + j of unit g >> 1, of both tiles the 8 slots of one 16-byte piece of values.
constexpr uint32_t kFewRows = 16, kFewWaves = 4;
template <int NS>
constexpr uint32_t kFewAhead = NS <= 4 ? 2 : 1;
template <int NS>
constexpr int kFewGroups = NS <= 2 ? 3 : (NS <= 4 ? 2 : 1);  // workgroups a compute unit

// A block as a wave's lanes take it.
template <int NS>
struct FewBlock {
    u32x4 k[2][NS];  // [tile][32 dims]
    u32x4 v[NS][2];  // [32 dims][16 of them]
    uint32_t holes;  // slots without a page
};
template <int NS>
__device__ __forceinline__ void load_few(FewBlock<NS> &f, const PagedAttnArgs &a, uint32_t head, uint32_t blk, uint32_t p0, uint32_t p1) {
    const uint32_t lane = __lane_id(), r = lane & 15, g = lane >> 4;
    f.holes = (p0 < a.c.pages ? 0u : 0xFFFFu) | (p1 < a.c.pages ? 0u : 0xFFFF0000u);
    const size_t at0 = unit_at(a.c, p0 < a.c.pages ? p0 : 0u, head, 2 * blk), at1 = unit_at(a.c, p1 < a.c.pages ? p1 : 0u, head, 2 * blk + 1);
    const uint16_t *k = a.c.k + (r >> 3 ? at1 : at0) + 128 * g + 8 * (r & 7);
    const uint16_t *v = a.c.v + (g >> 1 ? at1 : at0) + 256 * (g & 1) + 8 * r;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < NS; ++j) f.k[t][j] = *reinterpret_cast<const u32x4 *>(k + 512 * j + 64 * t);
#pragma unroll
    for (int d = 0; d < NS; ++d)
#pragma unroll
        for (int x = 0; x < 2; ++x) f.v[d][x] = *reinterpret_cast<const u32x4 *>(v + 512 * d + 128 * x);
}

template <int NS>
__global__ __launch_bounds__(256, kFewGroups<NS>) void paged_few_kernel(PagedAttnArgs a, Split split) {
    constexpr uint32_t D = 32 * NS;
    __shared__ float sm[kFewWaves][kFewRows], sl[kFewWaves][kFewRows];
    __shared__ __align__(16) float so[kFewWaves][kFewRows][D + 4];
    const uint32_t lane = __lane_id(), r16 = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t head = blockIdx.y, idx = blockIdx.x;
    Work w;
    if (!find_work(a, split, idx, w)) return;
    const Span &s = w.s;
    const uint32_t r0 = kFewRows * w.tile, r = r0 + r16;
    const bool live = r < w.rows;
    const Sight sight = sight_of(a, s, r, live);
    const uint32_t clear = clear_of(a, s, r0);
    const uint32_t first = w.part * w.per, end = min(first + w.per, (w.most + 31) / 32), b = w.b;
    const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    uint32_t blk = first + wave;
    // kFewAhead<NS> blocks of a wave on their way
    constexpr uint32_t kAhead = kFewAhead<NS>;
    FewBlock<NS> f[kAhead];
    // unit i of the wave: half i % 2 of its i / 2-th block
    Pages pages([&](uint32_t set) { return page_of(a.c, b, 2 * (first + wave + kFewWaves * (32 * set + lane / 2)) + lane % 2); });
    uint32_t asked = 0;
    const auto ask = [&](FewBlock<NS> &f, uint32_t blk) {
        pages.enter(asked);
        load_few<NS>(f, a, head, blk, pages.at(asked), pages.at(asked + 1));
        asked += 2;
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (blk + i * kFewWaves < end) ask(f[i], blk + i * kFewWaves);
    const uint32_t sign = query_sign(a.scale_log2);
    const float c = score_factor(a.scale_log2);
    bf16x8_t q[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) q[i] = query_unit(a.q + t * a.q_stride + (size_t)qh * D + 32 * i + 8 * g, live, sign);
    f32x4 o[2 * NS];
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) o[d] = f32x4{0, 0, 0, 0};
    RowSums sums;
    const auto step = [&](FewBlock<NS> &f, uint32_t blk) {
        const bool edge = blk * 32 + 32 > clear || f.holes;  // some row does not see it whole
        f32x4 p[2] = {};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < NS; ++j)
                p[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f.k[t][j]), q[j], p[t], 0, 0, 0);
        uint32_t seen = kAll;  // the lane's slots of tile t: bits 16 (g >> 1) + 8 t + 4 (g & 1) + j
        if (edge) {
            seen = sight.bits(32 * blk) & ~f.holes;
            const uint32_t mine = seen >> (16 * (g >> 1) + 4 * (g & 1));
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i >> 2][i & 3] = mine >> (8 * (i >> 2) + (i & 3)) & 1 ? p[i >> 2][i & 3] : -INFINITY;
        }
        float top = p[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, p[i >> 2][i & 3]);
        top *= c;
        top = fmaxf(top, xchg32(top, lane));
        top = fmaxf(top, xchg16(top, lane));
        if (seen) top = fmaxf(top, kLowBase);
        if (__any(top > sums.base + kLag)) {
            const float down = row_follow(sums, top);
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) o[d] *= down;
        }
        float e[8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = __builtin_amdgcn_exp2f(fmaf(p[i >> 2][i & 3], c, -sums.base));
            sum += e[i];
        }
        sums.l += sum;
        const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, u32x4{pack_bf16_rne(e[0], e[1]), pack_bf16_rne(e[2], e[3]), pack_bf16_rne(e[4], e[5]),
                                                               pack_bf16_rne(e[6], e[7])});
        uint32_t bad = 0;
        if (edge) {
            u32x4 words = {};
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) take_out(f.v[d >> 1][d & 1], words);
            bad = bad_slots(words) << (16 * (g >> 1) + 4 * (g & 1));
        }
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d)
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f.v[d >> 1][d & 1]), pf, o[d], 0, 0, 0);
        if (edge && __any(bad)) {
            for (uint32_t left = wave_or(bad) & wave_or(seen); left; left &= left - 1) {  // (what no row sees is left out)
                const uint32_t slot = (uint32_t)__builtin_ctz(left), page = page_of(a.c, b, 2 * blk + slot / 16);
                const uint16_t *v = a.c.v + unit_at(a.c, page, head, 2 * blk + slot / 16) + paged_value_at(slot % 16, 4 * g);
#pragma unroll
                for (int d = 0; d < 2 * NS; ++d) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[d][i] = put_back(o[d][i], v[512 * (d >> 1) + 8 * (16 * (d & 1) + i)], seen >> slot & 1);
                    __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
                }
            }
        }
    };
    for (; blk < end; blk += kAhead * kFewWaves) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t at = blk + i * kFewWaves;
            if (at >= end) break;
            step(f[i], at);
            if (at + kAhead * kFewWaves < end) ask(f[i], at + kAhead * kFewWaves);
        }
    }
    float l = sums.l + xchg32(sums.l, lane);
    l += xchg16(l, lane);
    const float norm = l == 0.0f ? 0.0f : 1.0f / l;
    if (g == 0) {
        sm[wave][r16] = sums.base;
        sl[wave][r16] = l;
    }
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) *reinterpret_cast<f32x4 *>(&so[wave][r16][16 * d + 4 * g]) = o[d] * norm;
    __syncthreads();
    // four dims of a row a thread
    for (uint32_t i = threadIdx.x; i < kFewRows * (D / 4); i += 256) {
        const uint32_t row = i / (D / 4), d = i % (D / 4) * 4, rr = r0 + row;
        if (rr >= w.rows) continue;
        float M = sm[0][row], L = 0.0f;
#pragma unroll
        for (uint32_t x = 1; x < kFewWaves; ++x) M = fmaxf(M, sm[x][row]);
        float wx[kFewWaves];
#pragma unroll
        for (uint32_t x = 0; x < kFewWaves; ++x) {
            const float lx = sl[x][row];
            wx[x] = lx == 0.0f ? 0.0f : lx * __builtin_amdgcn_exp2f(sm[x][row] - M);  // NaN stays
            L += wx[x];
        }
        // the weights before the values, which may be near the largest float
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t x = 0; x < kFewWaves; ++x) acc += wx[x] * inv * *reinterpret_cast<const f32x4 *>(&so[x][row][d]);
        if (w.parts == 1) {
            const size_t to = (size_t)(s.t0 + rr / a.group) * a.q_heads + head * a.group + rr % a.group;
            float none = -INFINITY;
            if (L == 0.0f && M > kSeenBase) acc = f32x4{1, 1, 1, 1} * (none = __builtin_nanf(""));
            *reinterpret_cast<u32x2 *>(a.out + to * D + d) = pack4(acc.x, acc.y, acc.z, acc.w);
            if (a.lse && d == 0) a.lse[to] = L == 0.0f ? none : (M + __log2f(L)) * kLn2;
        } else {
            const size_t to = part_at(a, split, idx, head, row);
            *reinterpret_cast<f32x4 *>(a.part + to * D + d) = acc;
            if (d == 0) {
                float *ml = a.part + (size_t)gridDim.x * a.c.heads * kFewRows * D + 2 * to;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
}

namespace {

// How a step is launched: tiles of 16 rows where the sequences have few query rows, else of 128.
struct AttnPlan {
    bool few;
    Split split;
    uint32_t tiles, grid, slots;  // at most, a head; slots: of parts in the workspace
};
AttnPlan plan_of(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    AttnPlan p{};
    p.few = (uint64_t)tokens * group <= (D <= 128 ? 48ull : 32ull) * batch;
    p.split.rows = p.few ? kFewRows : kManyRows;
    // tiles of every sequence: at most one that is not full each
    p.tiles = (uint32_t)((uint64_t)tokens * group / p.split.rows) + std::min(batch, tokens);
    if (p.few) {
        p.split.unit = kFewWaves;
        // as many workgroups as the card holds at once, less the half part that a tile has more than its share on average
        const uint32_t held = (D <= 64 ? 768 : (D <= 128 ? 512 : 256)) / kv_heads;
        p.split.target = std::max(std::max(held - std::min(held, p.tiles / 2), held / 2), std::min(p.tiles, 1024u));
        p.slots = p.grid = p.split.target + p.tiles;
    } else {
        // as many workgroups as the card holds at once
        p.split.unit = D <= 128 ? 2 : 1;
        const bool split = (uint64_t)p.tiles * kv_heads < 256 && (uint64_t)p.tiles * ((max_ctx + 31) / 32) < 1ull << 31;
        p.split.target = split ? 256 * p.split.unit / kv_heads : 0;  // at least `tiles`
        p.grid = p.split.target ? p.split.target : p.tiles;
        p.slots = 2 * p.split.target;
    }
    return p;
}

}  // namespace

uint64_t paged_attention_groups(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    const AttnPlan p = plan_of(batch, kv_heads, group, D, tokens, max_ctx);
    return (uint64_t)p.grid * (p.few ? 1 : kv_heads);  // (few: heads are another dimension)
}

size_t paged_attention_workspace_bytes(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    const AttnPlan p = plan_of(batch, kv_heads, group, D, tokens, max_ctx);
    return (size_t)p.slots * kv_heads * p.split.rows * (D + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttnArgs &a, hipStream_t s) {
    const AttnPlan p = plan_of(a.c.batch, a.c.heads, a.group, a.c.D, a.step.tokens, a.c.max_ctx);
    const auto launch = [&](auto ns) -> hipError_t {
        constexpr int NS = decltype(ns)::value;
        if (p.few) paged_few_kernel<NS><<<dim3(p.grid, a.c.heads), 256, 0, s>>>(a, p.split);
        else paged_many_kernel<NS><<<dim3(p.grid * a.c.heads), 256, 0, s>>>(a, p.split, p.slots);
        if (hipError_t e = hipGetLastError()) return e;
        if (p.split.target == 0) return hipSuccess;
        if (p.few && (uint64_t)p.tiles * p.split.rows * a.c.heads <= 256) {
            attn_join_kernel<PagedAttnArgs, NS, false, true, true><<<dim3(p.tiles * p.split.rows, a.c.heads), kJoinThreads, 0, s>>>(a, p.split, p.slots, 1);
        } else {
            uint32_t per_group = kJoinRowThreads / 64;
            while (per_group < p.split.rows && (uint64_t)p.tiles * a.c.heads * (p.split.rows / per_group) > 2048) per_group *= 2;
            const dim3 grid(p.tiles * (p.split.rows / per_group), a.c.heads);
            if (p.few) attn_join_kernel<PagedAttnArgs, NS, false, false, true><<<grid, kJoinRowThreads, 0, s>>>(a, p.split, p.slots, per_group);
            else attn_join_kernel<PagedAttnArgs, NS, true, false, true><<<grid, kJoinRowThreads, 0, s>>>(a, p.split, p.slots, per_group);
        }
        return hipGetLastError();
    };
    switch (a.c.D) {
        case 64: return launch(std::integral_constant<int, 2>{});
        case 96: return launch(std::integral_constant<int, 3>{});
        case 128: return launch(std::integral_constant<int, 4>{});
        case 192: return launch(std::integral_constant<int, 6>{});
        default: return launch(std::integral_constant<int, 8>{});
    }
}

}  // namespace kr
