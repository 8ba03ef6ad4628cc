// kv8_attention.hip — attention over the 8-bit key/value cache, and the attention weights of its slots.
//
// Reference semantics (grouped query heads, causal at the end of the context; its cache is bf16 pages):
//   kernels/metal/paged_gqa_and_deltanet.metal:242 and the prefill kernels beside it
//
// Mathematics.  The query rows of a sequence and kv head are r = i group + g (token i, head g of the group): every key
// and value byte is used for the whole group.  In base 2, with c_r = scale log2(e) / 2^e_r, ks and vs the scales
// of a block, q' = q 2^e_r in fp16:
//   s_rp = (q'_r . k_p) (c_r ks),   m_r = max_p s_rp,   l_r = sum_p 2^(s_rp - m_r),
//   out_r = 2^d_r sum_p 2^(s_rp - m_r + log2 vs - d_r) v_p / l_r
// with k_p, v_p the codes.  One pass over the slots: m_r only grows, and sums made under an older m_r are scaled down.  What enters
// the second product is fp16 (the matrix cores take f32 at a fraction of its rate; half a step is 2^-11 where the bf16 output's own is
// 2^-8), so its exponent has a reference of its own for each row: d_r follows the largest product of a
// probability and its block's scale of values, so that a block of large values that a row hardly sees takes no bits from the others.
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_32x32x16_f16: a lane then holds one
// query row (column l & 31) and the slots 8 i + 4 (l >> 5) + j of a block, its m_r and l_r are plain registers, and after
// rounding to fp16 those probabilities are the second product's operand as they lie (see kv8.hpp for the order of v).
#include <algorithm>

#include "kv8.hpp"

namespace kr {

namespace {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

// The power of two that brings a row to [2^14, 2^15), from the bf16 bits of its largest |q|; 2^126 at most, which is exact too: rows
// below 2^-112 are multiples of 2^-133 and become multiples of 2^-7.
__device__ __forceinline__ int query_exp(uint32_t top) { return min(141 - (int)(top >> 7), 126); }
// The factor of a row's scores: NaN where it holds an infinity or NaN (scores that are all -infinity would look like no slot seen).
__device__ __forceinline__ float query_factor(uint32_t top, float scale) {
    return top >= 0x7F80u ? __builtin_nanf("") : __builtin_amdgcn_frexp_mantf(scale);
}

// Query row r of a tile, held as the operands of D / 16 steps: lane (column l & 31, h = l >> 5) holds for step 2 j + s
// dims 32 j + 16 h + 8 s .. + 7, the dims that a lane's 16 key bytes cover.
template <int NS>
struct QueryRow {
    f16x8_t f[2 * NS];
    float c;  // |scale| log2(e) 2^-e is c 2^x, c in [1/2, 1): times a block's scale it need be a float only
    int x;    // (the sign of scale goes into the row: a maximum stays one under c)
};
// c 2^x times a block's scale of keys.
__device__ __forceinline__ float score_scale(float c, int x, float ks) {
    return ldexpf(c * __builtin_amdgcn_frexp_mantf(ks), x + __builtin_amdgcn_frexp_expf(ks));
}

// log2 of a block's scale of values: subnormal ones too; -infinity for a block of zeros, and for one that stands for NaN.
__device__ __forceinline__ float value_scale_log2(float vs) {
    return vs < INFINITY ? (float)__builtin_amdgcn_frexp_expf(vs) + __log2f(__builtin_amdgcn_frexp_mantf(vs)) : -INFINITY;
}

// A row's running sums: base m_r (lags the maximum by up to 2^8), l_r, and d_r.  The largest product is brought to 2^kTo and may grow
// to 2^15 before d_r follows: fp16 then holds products down to 2^-21 of it in full, and half a step of the rest is 2^-32 of it.
// kLeast keeps 2^d_r a normal float; products 2^-40 below 2^8 are none in fp16, so the exponent of a block that is further down (its
// scale 2^-40 of what d_r stands for) is held there, where its probabilities still count in l_r.
struct RowSums {
    float base = -1e38f, l = 0.0f, d = 0.0f;
};
constexpr float kTo = 7.0f, kLeast = -126.0f, kFarDown = -40.0f;

// A block's exponent beside its probabilities, log2 vs - d_r.
__device__ __forceinline__ float value_shift(const RowSums &r, float vlog) { return fmaxf(vlog - r.d, kFarDown); }

// Whether a block whose largest score of the row is `top` passes what the row's base or d allow (one comparison once top is known);
// both following it, and the factor of O.
__device__ __forceinline__ bool row_passed(const RowSums &r, float top, float vlog) {
    return top - r.base > fminf(8.0f, 15.0f - (vlog - r.d));
}
__device__ __forceinline__ float row_follow(RowSums &r, float top, float vlog) {
    const float base = fmaxf(r.base, top), down = r.base - base;
    const float d = fmaxf(fmaxf(r.d + down, (top - base) + vlog - kTo), kLeast), od = down + (r.d - d);
    r.base = base;
    r.d = d;
    r.l *= __builtin_amdgcn_exp2f(down);
    return __builtin_amdgcn_exp2f(od);
}
// Whether a base is so large that in its sum with an exponent beside it that exponent is off by more than 2^-14: then the scores'
// differences from the base are taken first.  (A row that has seen no slot has no base.)
__device__ __forceinline__ bool row_far(const RowSums &r) { return fabsf(r.base) > 0x1p10f && r.base > -9e37f; }

// The row in fp16 times a power of two that brings its largest value to [2^14, 2^15): bf16 holds 8 bits of significand
// and fp16 11, so every value down to 2^-28 of the largest is exact, and the rest are off by 2^-39 of it at
// most.
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
    const int e = query_exp(top);
    const float up = copysignf(exp2_int(e), scale_log2);
    q.c = query_factor(top, fabsf(scale_log2));
    q.x = __builtin_amdgcn_frexp_expf(scale_log2) - e;
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

// A lane's 16-byte units of a block's keys (or values): unit j of lane l at 1024 j + 16 l.
template <int NS>
__device__ __forceinline__ void load_units(u32x4 (&w)[NS], const uint8_t *blk) {
#pragma unroll
    for (int j = 0; j < NS; ++j) w[j] = *reinterpret_cast<const u32x4 *>(blk + 1024 * j + 16 * __lane_id());
}

// Row r of sequence span s: the slots that it sees, 0 for a row past the end.
__device__ __forceinline__ uint32_t row_limit(const Kv8Span &s, uint32_t r, uint32_t group, uint32_t max_ctx) {
    const uint32_t i = r / group;
    if (i >= s.m || s.n < s.m - i) return 0u;
    return min(s.n - s.m + i + 1, max_ctx);
}

// ---- the work of a launch
//
// Few rows: tiles of `rows` query rows; the context of a tile is split into parts of `per` blocks, so that the workgroups have
// about the same to do whatever the lengths are: `per` is the launch's blocks, counted on the device, over the workgroups wanted.
// A sequence's tiles all have as many parts as its longest: workgroup sum_{b' < b} tiles parts + part tiles + tile, and
// those past a shorter tile's end have nothing to do.  (The tile varies first: workgroups go round the XCDs in turn, and
// with the part first one XCD would get all the empty ones.)
struct Split {
    uint32_t target;  // workgroups wanted a kv head; 0: no tile is split
    uint32_t rows;    // of a tile
    uint32_t unit;    // few rows: `per` is a multiple of it; many: workgroups that a compute unit holds
};
__device__ __forceinline__ uint32_t tiles_of(const Kv8AttnArgs &a, const Split &w, const Kv8Span &s) {
    return (s.m * a.group + w.rows - 1) / w.rows;
}
__device__ __forceinline__ uint32_t blocks_of(const Kv8AttnArgs &a, const Kv8Span &s) {
    return (min(s.n, a.c.max_ctx) + 31) / 32;
}
__device__ __forceinline__ uint32_t parts_of(uint32_t blocks, uint32_t per) { return max((blocks + per - 1) / per, 1u); }

// total / target, rounded up
__device__ __forceinline__ unsigned long long fair_share(unsigned long long total, uint32_t target) {
    return total >> 31 ? (total + target - 1) / target : ((uint32_t)total + target - 1) / target;
}

// Blocks of a part.  Every wave computes it alike.
__device__ __forceinline__ uint32_t split_per(const Kv8AttnArgs &a, const Split &w) {
    unsigned long long total = 0;
    for (uint32_t b = __lane_id(); b < a.c.batch; b += 64) {
        const Kv8Span s = kv8_span(a.step, b);
        total += (unsigned long long)tiles_of(a, w, s) * blocks_of(a, s);
    }
    const unsigned long long fair = fair_share(wave_sum_u64(total), w.target);
    return max((uint32_t)((fair + w.unit - 1) / w.unit) * w.unit, w.unit);
}

// What workgroup `idx` of a head does.
struct Work {
    Kv8Span s;
    uint32_t b, tile, part, parts, per;  // parts: of this tile, at least 1
    uint32_t rows, most;                 // query rows of the sequence; slots that the tile's last row sees
};
__device__ __forceinline__ void fill_work(const Kv8AttnArgs &a, const Split &w, Work &o) {
    o.s = kv8_span(a.step, o.b);
    o.rows = o.s.m * a.group;
    o.most = row_limit(o.s, min(w.rows * (o.tile + 1), o.rows) - 1, a.group, a.c.max_ctx);
}
__device__ __forceinline__ bool find_work(const Kv8AttnArgs &a, const Split &w, uint32_t idx, Work &o) {
    o.per = split_per(a, w);
    uint32_t item;
    const auto count = [&](uint32_t i) {
        const Kv8Span s = kv8_span(a.step, i);
        return tiles_of(a, w, s) * parts_of(blocks_of(a, s), o.per);
    };
    if (!kv8_find(idx, a.c.batch, count, o.b, item)) return false;
    const uint32_t tiles = tiles_of(a, w, kv8_span(a.step, o.b));
    o.tile = item % tiles;
    o.part = item / tiles;
    fill_work(a, w, o);
    o.parts = parts_of((o.most + 31) / 32, o.per);
    return o.part < o.parts;
}

// Many rows: where there are fewer tiles than compute units, the tiles' blocks stand in one line, tile after tile, and a workgroup
// takes an equal share of it: the end of a tile, whole ones, the beginning of the next.  (Parts of equal length, of which a whole
// number fits a tile, leave the longest workgroup a quarter more than the mean: 600 tokens over up to 12000 in four sequences,
// 10/2 heads, D 256: 124 -> 113 us.)  A tile's blocks are those that its sequence's last row sees.
// Parts cost about 14 blocks' time (O through memory, and the join), and a tile alone on a compute unit is faster than one of
// several: where the longest tile has no more blocks than 14 and the shares that a compute unit would hold, tiles stay whole
// (16/2 heads, split and whole, us.  D 128: 500 tokens 26 and 23, 1000 31 and 34, 2000 58 and 58, 200 over 1000 25 and 38;
// D 256: 1000 tokens 47 and 55; D 64: 31 and 26).
__device__ __forceinline__ uint32_t tile_blocks(const Kv8AttnArgs &a, const Kv8Span &s) {
    return max(blocks_of(a, s), 1u);  // (a tile that sees nothing is written too)
}
// A workgroup's share, in blocks; 0: a workgroup takes a tile.
__device__ __forceinline__ uint32_t share_of(const Kv8AttnArgs &a, const Split &w) {
    if (w.target == 0) return 0;
    uint32_t total = 0, most = 0;  // (the host splits no launch whose blocks pass 2^31)
    for (uint32_t b = __lane_id(); b < a.c.batch; b += 64) {
        const Kv8Span s = kv8_span(a.step, b);
        const uint32_t tiles = tiles_of(a, w, s), blocks = tile_blocks(a, s);
        total += tiles * blocks;
        if (tiles) most = max(most, blocks);
    }
    const uint32_t share = max((wave_sum_u32(total) + w.target - 1) / w.target, 1u);
    return wave_max_u32(most) <= 14 + w.unit * share ? 0 : share;
}
// The tile in which place `at` of the line falls, and where in it.
__device__ __forceinline__ bool find_place(const Kv8AttnArgs &a, const Split &w, uint32_t at, Work &o, uint32_t &block, uint32_t &blocks) {
    uint32_t item;
    const auto count = [&](uint32_t i) {
        const Kv8Span s = kv8_span(a.step, i);
        return tiles_of(a, w, s) * tile_blocks(a, s);
    };
    if (!kv8_find(at, a.c.batch, count, o.b, item)) return false;
    blocks = tile_blocks(a, kv8_span(a.step, o.b));
    o.tile = item / blocks;
    block = item % blocks;
    fill_work(a, w, o);
    return true;
}

// For the joins: the tile-th tile of all, false past the last, and where its parts lie in the workspace: slot `slot` + (part 0: `odd`) +
// part * `step`.  Of a tile that is in one part (o.parts) nothing lies there.
template <bool kMany>
__device__ __forceinline__ bool find_tile(const Kv8AttnArgs &a, const Split &w, uint32_t tile, Work &o, uint32_t &slot,
                                          uint32_t &odd, uint32_t &step) {
    if (!kv8_find(tile, a.c.batch, [&](uint32_t i) { return tiles_of(a, w, kv8_span(a.step, i)); }, o.b, o.tile)) return false;
    fill_work(a, w, o);
    uint32_t share = 0;
    if constexpr (kMany) {
        share = share_of(a, w);
        if (share == 0) {
            o.parts = 1;
            slot = odd = 0;
            step = 1;
            return true;
        }
    } else {
        o.per = split_per(a, w);
    }
    uint32_t before = 0;
    for (uint32_t i = __lane_id(); i < o.b; i += 64) {
        const Kv8Span s = kv8_span(a.step, i);
        before += tiles_of(a, w, s) * (kMany ? tile_blocks(a, s) : parts_of(blocks_of(a, s), o.per));
    }
    before = wave_sum_u32(before);
    if constexpr (kMany) {
        const uint32_t from = before + o.tile * tile_blocks(a, o.s), seen = max((o.most + 31) / 32, 1u);
        const uint32_t first = from / share, last = (from + seen - 1) / share;
        o.parts = last - first + 1;
        slot = 2 * first;  // a workgroup's first piece in the even slot, its last one in the odd
        odd = first * share < from;
        step = 2;
    } else {
        o.parts = parts_of((o.most + 31) / 32, o.per);
        slot = before + o.tile;
        odd = 0;
        step = tiles_of(a, w, o.s);
    }
    return true;
}
// parts of a tile of few rows: at most `target` and one, and target is at most 1024
constexpr uint32_t kMostParts = 1056;
// Where a part's normalised O of a row lies in the workspace, in rows; m and l of all rows lie behind them, in pairs.
__device__ __forceinline__ size_t part_at(const Kv8AttnArgs &a, const Split &w, uint32_t idx, uint32_t head, uint32_t row) {
    return ((size_t)idx * a.c.heads + head) * w.rows + row;
}

// A value that every lane holds, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

__device__ __forceinline__ uint32_t wave_min_uniform(uint32_t v) { return ~wave_max_u32(~v); }

}  // namespace

// ---- many rows: prompts and chunks
//
// A workgroup of four waves takes 128 query rows, 32 a wave, and walks the blocks that they see.  The waves turn a block's bytes
// into fp16 operands in LDS together (a wave unpacking for itself would spend more vector cycles on it than the matrix
// cores take), each as the 16 bytes a lane that an operand load takes.  Body n of the loop takes block n's softmax and second
// product and block n + 1's first; it reads keys n + 1 and values n, and writes keys n + 2 and values n + 1 into the other
// halves, so that one barrier a block is enough.  Bound by what the matrix cores and the vector unit cannot overlap: 2048 tokens
// after 14000, 32/4 heads, int8: D 128 930 TFLOP/s, D 256 875, D 64 710; a prompt of 3907 of 16/2 heads of 128 97 us (645: the
// diagonal's tiles are of unequal length).
constexpr uint32_t kManyRows = 128;

template <int NS, int E4M3>
__global__ __launch_bounds__(256, NS <= 4 ? 2 : 1) void kv8_many_kernel(Kv8AttnArgs a, Split split, uint32_t slots) {
    constexpr uint32_t D = 32 * NS;
    constexpr int kUnits = (2 * NS + 3) / 4;   // 1 KB pieces of a block's keys and values that a wave takes
    __shared__ u32x4 lds[2][2][2 * NS][64];    // [keys, values][block & 1][step][lane]
    const uint32_t lane = __lane_id(), h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // heads side by side: with eight of them each XCD's L2 keeps the bytes of one
    // every second round of 256 workgroups mirrored: a compute unit's add up to about the same
    uint32_t at = blockIdx.x;
    if (at / 256 & 1) at = at / 256 * 256 + min(gridDim.x - at / 256 * 256, 256u) - 1 - at % 256;
    const uint32_t head = at % a.c.heads, idx = at / a.c.heads;
    const uint32_t share = share_of(a, split);
    uint32_t place = idx * share, left = share;
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
            if (odd) __syncthreads();  // the last piece's bytes have been read
        } else {
            if (odd || !kv8_find(idx, a.c.batch, [&](uint32_t i) { return tiles_of(a, split, kv8_span(a.step, i)); }, w.b, w.tile)) return;
            w.tile = tiles_of(a, split, kv8_span(a.step, w.b)) - 1 - w.tile;  // the tiles that see the most first
            fill_work(a, split, w);
            end = (w.most + 31) / 32;
        }
        const Kv8Span &s = w.s;
        const uint32_t r0 = kManyRows * w.tile, r = r0 + 32 * wave + (lane & 31);
        const bool live = r < w.rows;
        const uint32_t limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
        const uint32_t least = wave_min_uniform(live ? limit : 0xFFFFFFFFu);  // the slots that all rows of the wave see
        const uint32_t b = w.b, t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
        QueryRow<NS> q;
        load_query<NS>(q, a.q + t * a.q_stride + (size_t)qh * D, live, a.scale_log2);
        const size_t bh = (size_t)b * a.c.heads + head;
        const uint8_t *k = a.c.k + bh * a.c.blocks * (size_t)(32 * D), *v = a.c.v + bh * a.c.blocks * (size_t)(32 * D);
        const float *ks = a.c.ks + bh * a.c.blocks, *vs = a.c.vs + bh * a.c.blocks;
        f32x16 o[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) o[i] = f32x16{};
        RowSums sums;
        bool far = false;     // a row of the wave is row_far
        float poison = 0.0f;  // NaN for a row that sees values that stand for NaN
        // what body n writes: this wave's pieces of keys n + 2 and values n + 1
        u32x4 piece[kUnits];
        const auto fetch = [&](uint32_t n) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                // (past the end: the last block once more, which nothing reads)
                const uint32_t u = min(wave + 4 * i, 2u * NS - 1), at = min(u < NS ? n + 2 : n + 1, end - 1), j = u < NS ? u : u - NS;
                piece[i] = *reinterpret_cast<const u32x4 *>((u < NS ? k : v) + (size_t)at * (32 * D) + 1024 * j + 16 * lane);
            }
        };
        const auto put = [&](u32x4 (*to)[64], uint32_t j, const u32x4 &w) {
            to[2 * j][lane] = __builtin_bit_cast(u32x4, kv8_operand<E4M3>(w.x, w.y));
            to[2 * j + 1][lane] = __builtin_bit_cast(u32x4, kv8_operand<E4M3>(w.z, w.w));
        };
        const auto stage = [&](uint32_t n) {
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                const uint32_t u = min(wave + 4 * i, 2u * NS - 1);  // (the same piece twice where they do not divide)
                put(u < NS ? lds[0][n & 1] : lds[1][(n + 1) & 1], u < NS ? u : u - NS, piece[i]);
            }
        };
        float ks1 = 0.0f, vs1 = 0.0f;  // scales of block n + 1, on their way
        const auto fetch_scales = [&](uint32_t n) {
            const uint32_t at = min(n + 1, end - 1);
            ks1 = ks[at];
            vs1 = vs[at];
        };
        // The scores of the block in work, times c the exponents; its row maximum has been taken into `base`.
        f32x16 p;
        float c, shift, org;  // shift: the exponent beside the probabilities; org: what the scores' exponents are taken from
        const auto key_steps = [&](f32x16 &s, const u32x4 (&kf)[2 * NS]) {
#pragma unroll
            for (int j = 0; j < 2 * NS; ++j)
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, kf[j]), q.f[j], s, 0, 0, 0);
        };
        const auto row_top = [&](const f32x16 &s) {
            float top = fmaxf(fmaxf(s[0], s[1]), s[2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) top = fmaxf(fmaxf(top, s[i]), s[i + 1]);
            return fmaxf(top, s[15]);
        };
        // What a new block's scores change: slots that a row does not see get -infinity; the row's base and reference follow only when
        // they are passed (O is scaled down a few times in all).
        const auto enter = [&](float top, float vscale, uint32_t p0) {
            float vlog = __log2f(vscale), ref = 0.0f;  // ref: what has been taken from the scores already
            const bool normal = __builtin_amdgcn_classf(vscale, 0x100);  // (log2 takes subnormal numbers for 0)
            const bool special = p0 + 32 > least || !normal || far;
            if (special) {
#pragma clang fp contract(off)  // (the same bits for the maximum and for the difference from it)
                const uint32_t room = limit > p0 ? limit - p0 : 0u;  // slots of this block that the row sees
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] = 8 * (i >> 2) + 4 * h + (i & 3) < room ? p[i] * c : -INFINITY;
                c = 1.0f;
                top = row_top(p);
                top = fmaxf(top, xchg32(top, lane));
                ref = fmaxf(sums.base, top);
#pragma unroll
                for (int i = 0; i < 16; ++i) p[i] -= ref;
                if (!(vscale < INFINITY) && room) poison = __builtin_nanf("");
                vlog = value_scale_log2(vscale);
            }
            if (__any(row_passed(sums, top, vlog))) {
                const float down = row_follow(sums, top, vlog);
#pragma unroll
                for (int d = 0; d < NS; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= down;
                far = __any(row_far(sums));
                if (far && !special) {
#pragma clang fp contract(off)
                    ref = sums.base;
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[i] = p[i] * c - ref;
                    c = 1.0f;
                }
            }
            shift = value_shift(sums, vlog);
            org = sums.base - ref;
        };
        // Body n.  One run of instructions, so that the vector unit takes the exponentials while the matrix cores multiply the
        // next keys, and the next row maximum while they multiply values.
        const auto body = [&](auto more, uint32_t n) {
            constexpr bool kMore = decltype(more)::value;
            u32x4 kf[2 * NS], vf[2 * NS];
            if constexpr (kMore) {
#pragma unroll
                for (int j = 0; j < 2 * NS; ++j) kf[j] = lds[0][(n + 1) & 1][j][lane];
                stage(n);
                fetch(n + 1);
            }
#pragma unroll
            for (int j = 0; j < 2 * NS; ++j) vf[j] = lds[1][n & 1][j][lane];
            // the values' scale joins the exponent, and l takes it out again
            const float from = org - shift;
            float sum = 0.0f;
            f16x8_t pf[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(p[i], c, -from));
                sum += e;
                pf[(i >> 2) & 1][(i >> 3) * 4 + (i & 3)] = (_Float16)e;
            }
            sums.l = fmaf(sum, __builtin_amdgcn_exp2f(-shift), sums.l);
            if constexpr (kMore) {
                p = f32x16{};
                key_steps(p, kf);
            }
#pragma unroll
            for (int d = 0; d < NS; ++d) {
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vf[2 * d]), pf[0], o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vf[2 * d + 1]), pf[1], o[d], 0, 0, 0);
            }
            if constexpr (kMore) {
                c = score_scale(q.c, q.x, uniform(ks1));
                const float vnext = uniform(vs1);
                fetch_scales(n + 1);
                float top = row_top(p) * c;
                top = fmaxf(top, xchg32(top, lane));
                enter(top, vnext, (n + 1) * 32);
            }
        };
        if (first < end) {
            // keys first and first + 1, values first
            for (uint32_t u = wave; u < 3 * NS; u += 4) {
                const uint32_t j = u % NS, at = u / NS == 1 ? first + 1 : first;
                if (at >= end) continue;
                const uint8_t *from = (u / NS == 2 ? v : k) + (size_t)at * (32 * D) + 1024 * j + 16 * lane;
                put(u / NS == 2 ? lds[1][first & 1] : lds[0][at & 1], j, *reinterpret_cast<const u32x4 *>(from));
            }
            c = score_scale(q.c, q.x, uniform(ks[first]));
            fetch(first);
            fetch_scales(first);
            __syncthreads();
            u32x4 kf[2 * NS];
#pragma unroll
            for (int j = 0; j < 2 * NS; ++j) kf[j] = lds[0][first & 1][j][lane];
            p = f32x16{};
            key_steps(p, kf);
            float top = row_top(p) * c;
            top = fmaxf(top, xchg32(top, lane));
            enter(top, uniform(vs[first]), first * 32);
            for (uint32_t n = first; n + 1 < end; ++n) {
                // a wave in its body goes before one that is still at the barrier's end: 593 -> 570 us for 2048 tokens over 14000
                // (32/4 heads, D 128); with one wave a SIMD there is none to go before
                if constexpr (NS <= 4) __builtin_amdgcn_s_setprio(0);
                __syncthreads();
                if constexpr (NS <= 4) __builtin_amdgcn_s_setprio(1);
                body(std::true_type{}, n);
            }
            __syncthreads();
            body(std::false_type{}, end - 1);
        }
        const float l = sums.l + xchg32(sums.l, lane);
        // (two factors: their product may be below the normal floats)
        const float norm = (l == 0.0f ? 0.0f : 1.0f / l) + poison, up = __builtin_amdgcn_exp2f(sums.d);
#pragma unroll
        for (int d = 0; d < NS; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * norm * up;
        if (!live) {  // (a row past the sequence's)
        } else if (whole) {
            const size_t at = (size_t)t * a.q_heads + qh;
            if (a.lse && h == 0) a.lse[at] = l == 0.0f ? -INFINITY : (sums.base + __log2f(l)) * kLn2;
            uint16_t *out = a.out + at * D;
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x2 y = {pack_bf16_rne(o[d][4 * i], o[d][4 * i + 1]), pack_bf16_rne(o[d][4 * i + 2], o[d][4 * i + 3])};
                    *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * i + 4 * h) = y;
                }
        } else {
            const size_t at = part_at(a, split, 2 * idx + odd, head, r - r0);
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f32x4 *>(a.part + at * D + 32 * d + 8 * i + 4 * h) =
                        f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (h == 0) {
                float *ml = a.part + (size_t)slots * a.c.heads * kManyRows * D + 2 * at;
                ml[0] = sums.base;
                ml[1] = l;
            }
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
// Bound by bytes: 48 sequences up to 8000, 32/8 heads of 64: 298 MB in 53 us (5.6 TB/s); 131072 slots of 2 heads of 128 16.8 us
// (4 TB/s, the start of all workgroups included).
constexpr uint32_t kFewRows = 16, kFewWaves = 4;
template <int NS>
constexpr uint32_t kFewAhead = NS <= 4 ? 2 : 1;
template <int NS>
constexpr int kFewGroups = NS <= 2 ? 4 : (NS <= 3 ? 3 : (NS <= 6 ? 2 : 1));  // workgroups a compute unit

template <int NS>
__device__ __forceinline__ void load_query16(f16x8_t (&f)[NS], float &c, int &x, const uint16_t *row, bool live, float scale_log2) {
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
    const int e = query_exp(top);
    const float up = exp2_int(e);
    c = query_factor(top, scale_log2);
    x = __builtin_amdgcn_frexp_expf(scale_log2) - e;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const uint32_t W[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            f[i][2 * y] = (_Float16)(__uint_as_float(W[y] << 16) * up);
            f[i][2 * y + 1] = (_Float16)(__uint_as_float(W[y] & 0xFFFF0000u) * up);
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
__global__ __launch_bounds__(256, kFewGroups<NS>) void kv8_few_kernel(Kv8AttnArgs a, Split split) {
    constexpr uint32_t D = 32 * NS;
    __shared__ float sm[kFewWaves][kFewRows], sl[kFewWaves][kFewRows];
    __shared__ float so[kFewWaves][kFewRows][D + 4];
    const uint32_t lane = __lane_id(), r16 = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const uint32_t head = blockIdx.y, idx = blockIdx.x;
    Work w;
    if (!find_work(a, split, idx, w)) return;
    const Kv8Span &s = w.s;
    const uint32_t r0 = kFewRows * w.tile, r = r0 + r16;
    const bool live = r < w.rows;
    const uint32_t limit = live ? row_limit(s, r, a.group, a.c.max_ctx) : 0u;
    const uint32_t least = row_limit(s, r0, a.group, a.c.max_ctx);
    const uint32_t first = w.part * w.per, end = min(first + w.per, (w.most + 31) / 32), b = w.b;
    const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    const size_t bh = (size_t)b * a.c.heads + head;
    const uint8_t *k = a.c.k + bh * a.c.blocks * (size_t)(32 * D), *v = a.c.v + bh * a.c.blocks * (size_t)(32 * D);
    const float *ks = a.c.ks + bh * a.c.blocks, *vs = a.c.vs + bh * a.c.blocks;
    uint32_t blk = first + wave;
    // kFewAhead<NS> blocks of a wave on their way: with the waves that the registers allow about 100 KB a compute unit
    constexpr uint32_t kAhead = kFewAhead<NS>;
    FewBlock<NS> f[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (blk + i * kFewWaves < end) load_few<NS>(f[i], k, v, ks, vs, blk + i * kFewWaves);
    f16x8_t q[NS];
    float qc;
    int qx;
    load_query16<NS>(q, qc, qx, a.q + t * a.q_stride + (size_t)qh * D, live, a.scale_log2);
    f32x4 o[2 * NS];
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d) o[d] = f32x4{0, 0, 0, 0};
    RowSums sums;
    bool far = false;     // a row of the wave is row_far
    float poison = 0.0f;  // NaN for a row that sees values that stand for NaN
    const auto step = [&](auto masked, const FewBlock<NS> &f, uint32_t blk) {
        constexpr bool kEdge = decltype(masked)::value;
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
        const float c = score_scale(qc, qx, f.ks), vlog = value_scale_log2(f.vs);
        const uint32_t room = limit > blk * 32 ? limit - blk * 32 : 0u;
        if (kEdge && !(f.vs < INFINITY) && room) poison = __builtin_nanf("");
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma clang fp contract(off)  // (the same bits for the maximum and for the difference from it)
            float x = p[i >> 2][i & 3] * c;
            if (kEdge && 16 * (i >> 2) + 4 * g + (i & 3) >= room) x = -INFINITY;
            p[i >> 2][i & 3] = x;
            top = fmaxf(top, x);
        }
        top = fmaxf(top, xchg32(top, lane));
        top = fmaxf(top, xchg16(top, lane));
        if (__any(row_passed(sums, top, vlog))) {
            const float down = row_follow(sums, top, vlog);
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) o[d] *= down;
            far = __any(row_far(sums));
        }
        const float shift = value_shift(sums, vlog);
        float from = sums.base - shift;
        if (far) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i >> 2][i & 3] -= sums.base;
            from = -shift;
        }
        float sum = 0.0f;
        f16x8_t pf;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float e = __builtin_amdgcn_exp2f(p[i >> 2][i & 3] - from);
            sum += e;
            pf[i] = (_Float16)e;
        }
        sums.l = fmaf(sum, __builtin_amdgcn_exp2f(-shift), sums.l);
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d)
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv8_operand<E4M3>(f.v[d].x, f.v[d].y), pf, o[d], 0, 0, 0);
    };
    for (; blk < end; blk += kAhead * kFewWaves) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t at = blk + i * kFewWaves;
            if (at >= end) break;
            f[i].ks = uniform(f[i].ks);
            f[i].vs = uniform(f[i].vs);
            if (at * 32 + 32 > least || !(f[i].vs < INFINITY)) step(std::true_type{}, f[i], at);
            else step(std::false_type{}, f[i], at);
            if (at + kAhead * kFewWaves < end) load_few<NS>(f[i], k, v, ks, vs, at + kAhead * kFewWaves);
        }
    }
    float l = sums.l + xchg32(sums.l, lane);
    l += xchg16(l, lane);
    const float norm = (l == 0.0f ? 0.0f : 1.0f / l) + poison, up = __builtin_amdgcn_exp2f(sums.d);
    if (g == 0) {
        sm[wave][r16] = sums.base;
        sl[wave][r16] = l;
    }
#pragma unroll
    for (int d = 0; d < 2 * NS; ++d)
        *reinterpret_cast<f32x4 *>(&so[wave][r16][16 * d + 4 * g]) = o[d] * norm * up;
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
            const uint32_t tt = s.t0 + rr / a.group, hh = head * a.group + rr % a.group;
            const size_t at = (size_t)tt * a.q_heads + hh;
            const u32x2 y = {pack_bf16_rne(acc.x, acc.y), pack_bf16_rne(acc.z, acc.w)};
            *reinterpret_cast<u32x2 *>(a.out + at * D + d) = y;
            if (a.lse && d == 0) a.lse[at] = L == 0.0f ? -INFINITY : (M + __log2f(L)) * kLn2;
        } else {
            const size_t at = part_at(a, split, idx, head, row);
            *reinterpret_cast<f32x4 *>(a.part + at * D + d) = acc;
            if (d == 0) {
                float *ml = a.part + (size_t)gridDim.x * a.c.heads * kFewRows * D + 2 * at;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
}

// Joins the parts of the rows that were split.  kWide: a workgroup of 16 waves a row, thread (i, j) taking parts i, i + n, ...
// of four dims, for few rows in many parts; else a wave a row, its workgroup `per_group` rows of a tile (four waves: with 16, which
// find the work once for more rows, 400 tokens over 20000 in three sequences took 110 us, not 106).  Bound by latency (work count,
// maxima, parts): 16 rows in 256 parts 6.5 us, 1536 rows in a few 8.3, 6000 rows of 256 10.3 for 34 MB.
constexpr uint32_t kJoinThreads = 1024, kJoinRowThreads = 256;
template <int NS, bool kMany, bool kWide>
__global__ __launch_bounds__(kWide ? kJoinThreads : kJoinRowThreads) void kv8_join_kernel(Kv8AttnArgs a, Split split,
                                                                                          uint32_t slots, uint32_t per_group) {
    constexpr uint32_t D = 32 * NS, kQuads = D / 4, kThreads = kWide ? kJoinThreads : 64, kWays = kThreads / kQuads;
    __shared__ f32x4 so[kWide ? kWays : 1][kQuads];
    __shared__ float ws[kWide ? kMostParts : kJoinRowThreads], red[2][kJoinThreads / 64];
    const uint32_t lane = __lane_id(), head = blockIdx.y, wave = threadIdx.x >> 6, tid = kWide ? threadIdx.x : lane;
    const uint32_t groups = split.rows / per_group;
    Work w;
    uint32_t slot, odd, slot_step;
    if (!find_tile<kMany>(a, split, blockIdx.x / groups, w, slot, odd, slot_step)) return;
    // (starts that decrease can make more parts than the launch has: none behind its last.  Counted before the exit, beside the loads
    // that it waits for: 5 sequences up to 3000 13.8 us, not 14.1)
    if (slot < slots) w.parts = min(w.parts, (slots - slot + slot_step - 1) / slot_step);
    if (w.parts == 1 || slot >= slots) return;
    const size_t slot_rows = (size_t)a.c.heads * split.rows, step = slot_step * slot_rows;  // between parts, in rows
    const auto part_row = [&](uint32_t p) { return p * step + (p == 0 ? odd * slot_rows : 0); };
    const float *all_ml = a.part + slots * slot_rows * D;
    const uint32_t way = tid / kQuads, quad = tid % kQuads, row0 = blockIdx.x % groups * per_group;
    for (uint32_t row = row0 + (kWide ? 0 : wave); row < row0 + per_group; row += kWide ? 1 : kJoinRowThreads / 64) {
        const uint32_t r = split.rows * w.tile + row;
        if (r >= w.rows) return;
        const size_t at = part_at(a, split, slot, head, row);
        const float2 *ml = reinterpret_cast<const float2 *>(all_ml) + at;
        f32x4 acc = {0, 0, 0, 0};
        float M = -INFINITY, L = 0.0f;
        for (uint32_t p = tid; p < w.parts; p += kThreads) M = fmaxf(M, ml[part_row(p)].x);
        M = wave_max(M);
        if constexpr (kWide) {
            if (lane == 0) red[0][wave] = M;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < kJoinThreads / 64; ++i) M = fmaxf(M, red[0][i]);
        }
        const float *o = a.part + at * D + 4 * quad;
        for (uint32_t p0 = 0; p0 < w.parts; p0 += kWide ? kMostParts : 64) {  // (kWide: once)
            const uint32_t n = min(w.parts - p0, kWide ? kMostParts : 64u);
            float *wl = kWide ? ws : ws + 64 * wave, sum = 0.0f;
            for (uint32_t p = tid; p < n; p += kThreads) {
                const float2 x = ml[part_row(p0 + p)];
                const float f = x.y == 0.0f ? 0.0f : x.y * __builtin_amdgcn_exp2f(x.x - M);  // NaN stays
                wl[p] = f;
                sum += f;
            }
            // the weights are divided by L before they meet values, which may be near the largest float
            sum = wave_sum(sum);
            if constexpr (kWide) {
                if (lane == 0) red[1][wave] = sum;
                __syncthreads();
                sum = red[1][0];
#pragma unroll
                for (uint32_t i = 1; i < kJoinThreads / 64; ++i) sum += red[1][i];
            } else {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
            const float before = L;
            L += sum;
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            if (p0) acc *= before * inv;
            if (way < kWays) {
#pragma unroll 8
                for (uint32_t p = way; p < n; p += kWays)
                    acc += wl[p] * inv * *reinterpret_cast<const f32x4 *>(o + part_row(p0 + p) * D);
            }
            if constexpr (!kWide) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        if constexpr (kWide) {
            if (way < kWays) so[way][quad] = acc;
            __syncthreads();
            if (tid >= kQuads) return;
            acc = so[0][tid];
#pragma unroll
            for (uint32_t i = 1; i < kWays; ++i) acc += so[i][tid];
        } else {
#pragma unroll
            for (uint32_t i = 1; i < kWays; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float other = __shfl(acc[x], (lane + i * kQuads) & 63);
                    acc[x] += lane < kQuads ? other : 0.0f;
                }
        }
        if (tid < kQuads) {
            const size_t to = (size_t)(w.s.t0 + r / a.group) * a.q_heads + head * a.group + r % a.group;
            const u32x2 y = {pack_bf16_rne(acc.x, acc.y), pack_bf16_rne(acc.z, acc.w)};
            *reinterpret_cast<u32x2 *>(a.out + to * D + 4 * tid) = y;
            if (a.lse && tid == 0) a.lse[to] = L == 0.0f ? -INFINITY : (M + __log2f(L)) * kLn2;
        }
    }
}

// ---- attention weights of the slots
//
// Column sums of the attention matrix, from K and the rows' lse alone: weight_p += sum_r 2^(c s_rp - lse_r).  The products are taken
// as S = Q K^T here: a lane holds one slot (column l & 31), the rows are summed in its registers, and their lse come from LDS.
// A workgroup takes 128 slots, 32 a wave, whose keys stay in registers, and walks the query rows that see them in tiles of 64:
// one in LDS that is multiplied, the next one on its way.  Both operands are bf16, so that a query row enters as it is and only
// the keys are converted, once a workgroup (with rows brought to fp16 as in the kernels above that took half of the vector
// instructions: 2000 tokens of 16/2 heads, D 128, 46 -> 31 us; 1000 over 8000 in two sequences 95 -> 61 us, 550 TF/s).
// Where there are many rows they are split into parts whose sums kv8_weight_join_kernel adds in order.  The workgroups loop over
// the work that the lengths turn out to be.  Short calls are bound by latency: of the 31 us about 10 are instructions.
// Few rows a sequence (one or two tokens): tiles of 32, nothing on its way, and no parts (16 decoded tokens over up to 8000 slots:
// 21 us with tiles of 64, 13.5 so: more workgroups a compute unit).
constexpr uint32_t kWeightSlots = 128, kWeightTarget = 768;
constexpr uint32_t weight_rows(bool few) { return few ? 32 : 64; }

template <bool kFew>
struct WeightSpan {
    Kv8Span s;
    uint32_t n, chunks, rows, tiles;  // slots in the cache, chunks of 128 of them; query rows, tiles of them
};
template <bool kFew>
__device__ __forceinline__ WeightSpan<kFew> weight_span(const Kv8AttnArgs &a, uint32_t b) {
    constexpr uint32_t kRows = weight_rows(kFew);
    WeightSpan<kFew> w;
    w.s = kv8_span(a.step, b);
    w.n = min(w.s.n, a.c.max_ctx);
    w.chunks = (w.n + kWeightSlots - 1) / kWeightSlots;
    w.rows = w.s.m * a.group;
    w.tiles = (w.rows + kRows - 1) / kRows;
    return w;
}
// Row tiles of a part: the launch's (chunk, tile) pairs over the workgroups wanted, at least 2 (their start costs as much).
template <bool kFew>
__device__ __forceinline__ uint32_t weight_per(const Kv8AttnArgs &a, uint32_t target) {
    if (kFew) return 1u << 27;  // more than there are
    unsigned long long total = 0;
    for (uint32_t b = __lane_id(); b < a.c.batch; b += 64) {
        const auto w = weight_span<kFew>(a, b);
        // chunks of new tokens are seen by half of the rows on average: never below half of all pairs
        const uint32_t past = w.n > w.s.m ? w.n - w.s.m : 0u;
        total += ((unsigned long long)w.chunks * w.tiles + (unsigned long long)(past / kWeightSlots) * w.tiles + 1) / 2;
    }
    total = wave_sum_u64(total);
    const unsigned long long per = total >> 31 ? (total + target - 1) / target : ((uint32_t)total + target - 1) / target;
    return max((uint32_t)per, 2u);
}
__device__ __forceinline__ uint32_t weight_parts(uint32_t tiles, uint32_t per) { return max((tiles + per - 1) / per, 1u); }
// The first row tile that sees a chunk: token i sees slots up to n - m + i.
template <bool kFew>
__device__ __forceinline__ uint32_t weight_first(const Kv8AttnArgs &a, const WeightSpan<kFew> &w, uint32_t chunk) {
    const uint32_t p0 = chunk * kWeightSlots, i0 = p0 + w.s.m > w.s.n ? p0 + w.s.m - w.s.n : 0u;
    return min(i0 * a.group / weight_rows(kFew), w.tiles);
}

// Eight codes as bf16, exact, times a power of two.
template <int E4M3>
__device__ __forceinline__ bf16x8_t weight_key(uint32_t lo, uint32_t hi, float up) {
    float y[8];
    kv8_values<E4M3>(lo, y);
    kv8_values<E4M3>(hi, y + 4);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = __builtin_amdgcn_perm(__float_as_uint(y[2 * i + 1] * up), __float_as_uint(y[2 * i] * up), 0x07060302u);
    return __builtin_bit_cast(bf16x8_t, w);
}

template <int NS, int E4M3, bool kFew>
__global__ __launch_bounds__(256, 2) void kv8_weight_kernel(Kv8AttnArgs a, uint32_t target) {
    constexpr uint32_t D = 32 * NS, kRows = weight_rows(kFew), kHalves = kRows / 32, kSides = kFew ? 1 : 2;
    __shared__ u32x4 ql[kSides][kHalves][2 * NS][64];         // [side][half of the rows][step][lane]
    __shared__ __align__(16) float cl[kSides][kRows];         // -lse_r in powers of two
    const uint32_t lane = __lane_id(), h = lane >> 5, head = blockIdx.y;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per = weight_per<kFew>(a, target);
    const auto count = [&](uint32_t i) {
        const auto w = weight_span<kFew>(a, i);
        return w.chunks * weight_parts(w.tiles, per);
    };
    for (uint32_t idx = blockIdx.x;; idx += gridDim.x) {
        uint32_t b, item;
        if (!kv8_find(idx, a.c.batch, count, b, item)) return;
        const auto w = weight_span<kFew>(a, b);
        // the chunks of every other part in reverse: late ones see fewer rows, and workgroups go round the XCDs in turn
        const uint32_t part = item / w.chunks, chunk = part & 1 ? w.chunks - 1 - item % w.chunks : item % w.chunks;
        const bool split = weight_parts(w.tiles, per) > 1;
        const uint32_t t0 = weight_first<kFew>(a, w, chunk) + part * per, t1 = min(t0 + per, w.tiles);
        if (part > 0 && t0 >= w.tiles) continue;  // part 0 writes also where no row sees the chunk
        const uint32_t p0 = chunk * kWeightSlots + 32 * wave, p = p0 + (lane & 31);
        const size_t bh = (size_t)b * a.c.heads + head;
        const uint32_t old = w.s.n > w.s.m ? w.s.n - w.s.m : 0u;  // slots before the new tokens
        float *to = a.weight + bh * a.c.max_ctx + p;
        const float had = !split && p < min(old, w.n) ? a.decay * *to : 0.0f;
        const uint32_t blk = min(p0 / 32, a.c.blocks - 1);
        u32x4 kw[NS];
        load_units<NS>(kw, a.c.k + (bh * a.c.blocks + blk) * (size_t)(32 * D));
        const float kscale = a.c.ks[bh * a.c.blocks + blk];
        bf16x8_t kf[2 * NS];
        float ck = 0.0f;  // the scale of a score
        // The query rows that see slot p are first_row .. w.rows - 1; the wave's slots are all seen from tile `clear` on.
        const auto first_row = [&](uint32_t p) { return (p + w.s.m > w.s.n ? p + w.s.m - w.s.n : 0u) * a.group; };
        const uint32_t row0 = p < w.n ? first_row(p) : w.rows, seen = w.rows - row0;
        const uint32_t clear = p0 + 32 <= w.n ? (first_row(p0 + 31) + kRows - 1) / kRows : 0xFFFFFFFFu;
        // kOfRow threads take a row's 16-byte units in turn.  Unit u = 4 j + 2 h + s goes to step 2 j + s of lane (row, h), its place
        // turned by the unit: the rows and units that are written together, and the rows read together, lie in all banks.
        constexpr uint32_t kOfRow = 256 / kRows, kUnits = (D / 8 + kOfRow - 1) / kOfRow;
        const uint32_t mine = threadIdx.x / kOfRow, first_u = threadIdx.x % kOfRow;
        const auto place = [](uint32_t lane, uint32_t u) { return lane ^ (16 / kOfRow * (u % kOfRow)); };
        u32x4 raw[kUnits];
        float lse = 0.0f;
        uint32_t row = kRows * t0 + mine, tg = row % a.group;  // what is fetched next
        const uint16_t *at = a.q + (w.s.t0 + row / a.group) * a.q_stride + (size_t)(head * a.group + tg) * D + 8 * first_u;
        const float *lse_at = a.lse + (size_t)(w.s.t0 + row / a.group) * a.q_heads + head * a.group + tg;
        const size_t next_token = a.q_stride - (size_t)a.group * D, next_tile = kRows / a.group * a.q_stride + (size_t)(kRows % a.group) * D;
        const auto fetch = [&] {
            const bool live = row < w.rows;
            const uint16_t *from = live ? at : a.q;  // (what lies past the rows is not counted)
#pragma unroll
            for (uint32_t i = 0; i < kUnits; ++i)
                if (D / 8 % kOfRow == 0 || first_u + kOfRow * i < D / 8) raw[i] = *reinterpret_cast<const u32x4 *>(from + 8 * kOfRow * i);
            lse = *(live ? lse_at : a.lse);
            row += kRows;
            at += next_tile;
            lse_at += kRows / a.group * a.q_heads + kRows % a.group;
            tg += kRows % a.group;
            if (tg >= a.group) {
                tg -= a.group;
                at += next_token;
                lse_at += a.q_heads - a.group;
            }
        };
        const auto stage = [&](uint32_t side) {
#pragma unroll
            for (uint32_t i = 0; i < kUnits; ++i) {
                const uint32_t u = first_u + kOfRow * i;
                if (D / 8 % kOfRow == 0 || u < D / 8)
                    ql[side][mine >> 5][2 * (u >> 2) + (u & 1)][place((mine & 31) + 32 * ((u >> 1) & 1), u)] = raw[i];
            }
            if (first_u == 0) cl[side][mine] = -lse * kLog2e;
        };
        float sum = 0.0f;
        const auto tile_sum = [&](uint32_t side, uint32_t tile) {
            const bool edge = tile < clear || kRows * (tile + 1) > w.rows;
#pragma unroll
            for (uint32_t x = 0; x < kHalves; ++x) {
                f32x16 s = {};
#pragma unroll
                for (int j = 0; j < 2 * NS; ++j)
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        __builtin_bit_cast(bf16x8_t, ql[side][x][j][place(lane, 4 * (j >> 1) + 2 * h + (j & 1))]), kf[j], s, 0, 0, 0);
                const auto rows = [&](auto all) {
                    const uint32_t r = kRows * tile + 32 * x + 4 * h - row0;
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 c = *reinterpret_cast<const f32x4 *>(&cl[side][32 * x + 2 * i + 4 * h]);
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const float e = __builtin_amdgcn_exp2f(fmaf(s[i + y], ck, c[y]));
                            sum += decltype(all)::value || r + 2 * i + y < seen ? e : 0.0f;
                        }
                    }
                };
                if (edge) rows(std::false_type{});
                else rows(std::true_type{});
            }
        };
        if (t0 < t1) {
            fetch();
            // The keys' operands, once the first rows are on their way too.  The codes enter times 2^-17: a sum of 256 products with
            // bf16 values stays within f32.  Scales so large that their product with 2^17 might not: they leave 2^43 of it here and
            // take the rest into the codes (scores within f32 stay there).
            ck = a.scale_log2 * (kscale * 0x1p17f);
            float kup = 0x1p-17f;
            if (!(fabsf(ck) < 0x1p60f)) {
                const int es = __builtin_amdgcn_frexp_expf(a.scale_log2) + __builtin_amdgcn_frexp_expf(kscale);
                const int kx = min(max(es - 43, -17), 100);
                ck = ldexpf(__builtin_amdgcn_frexp_mantf(a.scale_log2) * __builtin_amdgcn_frexp_mantf(kscale), es - kx);
                kup = exp2_int(kx);
            }
#pragma unroll
            for (int j = 0; j < NS; ++j) {
                kf[2 * j] = weight_key<E4M3>(kw[j].x, kw[j].y, kup);
                kf[2 * j + 1] = weight_key<E4M3>(kw[j].z, kw[j].w, kup);
            }
            stage(0);
            if (t0 + 1 < t1) fetch();
        }
        for (uint32_t tile = t0; tile < t1; ++tile) {
            const uint32_t side = kFew ? 0 : (tile - t0) & 1;
            __syncthreads();  // this tile is written, the one before has been read
            tile_sum(side, tile);
            if (tile + 1 >= t1) break;
            if constexpr (kFew) __syncthreads();
            stage(kFew ? 0 : side ^ 1);
            if (tile + 2 < t1) fetch();
        }
        sum += xchg32(sum, lane);
        if (lane < 32) {
            if (split)
                a.part[((size_t)idx * a.c.heads + head) * kWeightSlots + p - chunk * kWeightSlots] = sum;
            else if (p < w.n)
                *to = had + sum;
        }
        __syncthreads();  // LDS is free for the next work
    }
}

// Adds the parts of a chunk in order to what its slots had.  Bound by latency: 2000 slots of 2 heads 6 us.
__global__ __launch_bounds__(kWeightSlots) void kv8_weight_join_kernel(Kv8AttnArgs a, uint32_t target) {
    const uint32_t head = blockIdx.y, per = weight_per<false>(a, target);
    for (uint32_t idx = blockIdx.x;; idx += gridDim.x) {  // chunks
        uint32_t b, chunk;
        if (!kv8_find(idx, a.c.batch, [&](uint32_t i) { return weight_span<false>(a, i).chunks; }, b, chunk)) return;
        const auto w = weight_span<false>(a, b);
        const uint32_t parts = weight_parts(w.tiles, per), p = chunk * kWeightSlots + threadIdx.x;
        if (parts == 1) continue;
        uint32_t before = 0;
        for (uint32_t i = __lane_id(); i < b; i += 64) {
            const auto o = weight_span<false>(a, i);
            before += o.chunks * weight_parts(o.tiles, per);
        }
        before = wave_sum_u32(before);
        if (p >= w.n) continue;
        const uint32_t seen = w.tiles - weight_first<false>(a, w, chunk), used = weight_parts(seen, per);
        const uint32_t old = w.s.n > w.s.m ? w.s.n - w.s.m : 0u;
        float *to = a.weight + ((size_t)b * a.c.heads + head) * a.c.max_ctx + p;
        float sum = p < old ? a.decay * *to : 0.0f;
#pragma unroll 16
        for (uint32_t i = 0; i < used; ++i)
            sum += a.part[((size_t)(before + i * w.chunks + (i & 1 ? w.chunks - 1 - chunk : chunk)) * a.c.heads + head) * kWeightSlots + threadIdx.x];
        *to = sum;
    }
}

namespace {

// How a step is launched: tiles of 16 rows where the sequences have few query rows (a few tokens of a group of heads), else of
// 128.  With 40 rows a sequence, D 128, three tiles of 16 take 43 and 25 us (one sequence of 131072, eight of 8000), one of 128 48 and
// 29; with 64 they are even; at D 256, where the small tiles' operands leave one workgroup a compute unit, 64 rows take 68 and 48.
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
        // as many workgroups as the card holds at once, less the half part that a tile has more than its share on average: the few
        // that came too many would take a round of their own (four sequences of 60000, 8 heads of two: 106 -> 88 us)
        const uint32_t held = (D <= 64 ? 1024 : (D <= 96 ? 768 : (D <= 192 ? 512 : 256))) / kv_heads;
        p.split.target = std::max(std::max(held - std::min(held, p.tiles / 2), held / 2), std::min(p.tiles, 1024u));
        p.slots = p.grid = p.split.target + p.tiles;
    } else {
        // as many workgroups as the card holds at once
        p.split.unit = D <= 64 ? 3 : (D <= 128 ? 2 : 1);
        const bool split = (uint64_t)p.tiles * kv_heads < 256 && (uint64_t)p.tiles * ((max_ctx + 31) / 32) < 1ull << 31;
        p.split.target = split ? 256 * p.split.unit / kv_heads : 0;  // at least `tiles`
        p.grid = p.split.target ? p.split.target : p.tiles;
        p.slots = 2 * p.split.target;
    }
    return p;
}

}  // namespace

uint64_t kv8_attention_groups(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    const AttnPlan p = plan_of(batch, kv_heads, group, D, tokens, max_ctx);
    return (uint64_t)p.grid * (p.few ? 1 : kv_heads);  // (few: heads are another dimension)
}

size_t kv8_attention_workspace_bytes(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    const AttnPlan p = plan_of(batch, kv_heads, group, D, tokens, max_ctx);
    return (size_t)p.slots * kv_heads * p.split.rows * (D + 2) * sizeof(float);
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
    const AttnPlan p = plan_of(a.c.batch, a.c.heads, a.group, a.c.D, a.step.tokens, a.c.max_ctx);
    return by_shape(a.c, [&](auto ns, auto e4m3) -> hipError_t {
        constexpr int NS = decltype(ns)::value, E4M3 = decltype(e4m3)::value;
        if (p.few)
            kv8_few_kernel<NS, E4M3><<<dim3(p.grid, a.c.heads), 256, 0, s>>>(a, p.split);
        else
            kv8_many_kernel<NS, E4M3><<<dim3(p.grid * a.c.heads), 256, 0, s>>>(a, p.split, p.slots);
        if (hipError_t e = hipGetLastError()) return e;
        if (p.split.target == 0) return hipSuccess;
        if (p.few && (uint64_t)p.tiles * p.split.rows * a.c.heads <= 256) {
            kv8_join_kernel<NS, false, true><<<dim3(p.tiles * p.split.rows, a.c.heads), kJoinThreads, 0, s>>>(a, p.split, p.slots, 1);
        } else {
            uint32_t per_group = kJoinRowThreads / 64;
            while (per_group < p.split.rows && (uint64_t)p.tiles * a.c.heads * (p.split.rows / per_group) > 2048) per_group *= 2;
            const dim3 grid(p.tiles * (p.split.rows / per_group), a.c.heads);
            if (p.few) kv8_join_kernel<NS, false, false><<<grid, kJoinRowThreads, 0, s>>>(a, p.split, p.slots, per_group);
            else kv8_join_kernel<NS, true, false><<<grid, kJoinRowThreads, 0, s>>>(a, p.split, p.slots, per_group);
        }
        return hipGetLastError();
    });
}

// Where a sequence's rows are one tile of 32, a workgroup takes them all.
static bool few_rows(uint32_t batch, uint32_t group, uint32_t tokens) { return (uint64_t)tokens * group <= 32ull * batch; }

// Workgroups wanted a head.
static uint32_t weight_target(uint32_t kv_heads) { return std::max(kWeightTarget / kv_heads, 1u); }

size_t kv8_weight_workspace_bytes(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t tokens, uint32_t max_ctx) {
    if (few_rows(batch, group, tokens)) return 0;
    const size_t chunks = (size_t)batch * ((max_ctx + kWeightSlots - 1) / kWeightSlots);
    // at most 2 target + chunks parts a head: half of the pairs may not be counted
    return (2 * weight_target(kv_heads) + chunks) * kv_heads * kWeightSlots * sizeof(float);
}

hipError_t launch_kv8_weight(const Kv8AttnArgs &a, hipStream_t s) {
    const uint32_t target = weight_target(a.c.heads);
    const uint64_t chunks = (uint64_t)a.c.batch * ((a.c.max_ctx + kWeightSlots - 1) / kWeightSlots);
    return by_shape(a.c, [&](auto ns, auto e4m3) -> hipError_t {
        const dim3 grid((uint32_t)std::min<uint64_t>(chunks + 2 * target, std::max(2048 / a.c.heads, 1u)), a.c.heads);
        constexpr int NS = decltype(ns)::value, E4M3 = decltype(e4m3)::value;
        if (few_rows(a.c.batch, a.group, a.step.tokens)) {
            kv8_weight_kernel<NS, E4M3, true><<<grid, 256, 0, s>>>(a, target);
            return hipGetLastError();
        }
        kv8_weight_kernel<NS, E4M3, false><<<grid, 256, 0, s>>>(a, target);
        if (hipError_t e = hipGetLastError()) return e;
        const dim3 join((uint32_t)std::min<uint64_t>(chunks, std::max(2048 / a.c.heads, 1u)), a.c.heads);
        kv8_weight_join_kernel<<<join, kWeightSlots, 0, s>>>(a, target);
        return hipGetLastError();
    });
}

}  // namespace kr
