// attn_work.hpp — how attention over a cache shares a ragged step out to workgroups, and the join of tiles whose context was
// split.  A: the kernel's arguments (step, group, c.batch, c.heads, c.max_ctx, q_heads, part, out, lse).
#pragma once

#include "ragged.hpp"

namespace kr {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f;

// Row r of sequence span s: the slots that it sees, 0 for a row past the end.
template <class Group>
__device__ __forceinline__ uint32_t row_limit(const Span &s, uint32_t r, const Group &group, uint32_t max_ctx) {
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
    uint32_t rows;    // of a tile, a power of two
    uint32_t unit;    // `per` is a multiple of it (even parts: a power of two); shares: workgroups that a compute unit holds
};
// How tiles are split: as above, in at most target + tiles parts; many rows in shares of one line, below; or in even parts, few rows and
// many, at most `target` of them where there are not more tiles.
enum class Parts { few, shares, even };
template <class A>
__device__ __forceinline__ uint32_t tiles_of(const A &a, const Split &w, const Span &s) {
    return (s.m * a.group + w.rows - 1) >> __builtin_ctz(w.rows);
}
template <class A>
__device__ __forceinline__ uint32_t blocks_of(const A &a, const Span &s) {
    return (min(s.n, a.c.max_ctx) + 31) / 32;
}
__device__ __forceinline__ uint32_t parts_of(uint32_t blocks, uint32_t per) { return max((blocks + per - 1) / per, 1u); }

// total / target, rounded up
__device__ __forceinline__ unsigned long long fair_share(unsigned long long total, uint32_t target) {
    return total >> 31 ? (total + target - 1) / target : ((uint32_t)total + target - 1) / target;
}

// Even parts: the fewest blocks, in whole units, of which `target` parts are enough, so that a workgroup has one.  (Shares of one line,
// as below, are even to a block, but a second piece costs a workgroup another start and end, as much as 18 blocks of 128 rows and D 128:
// 250 tokens over up to 5000 in eight sequences, 16/2 heads of 128, took 43 us, not 33; two rounds of smaller parts won nothing
// either.)  A tile that is not split saves the way of its O through memory, about 14 blocks' time: where the longest has no more than
// that past a part, tiles stay whole.
template <class A>
__device__ __forceinline__ uint32_t even_per(const A &a, const Split &w) {
    const uint32_t lane = __lane_id();
    uint32_t tiles0 = 0, blocks0 = 0, tiles = 0, most = 0;
    float total = 0.0f;  // (where the search begins, and with some more than its error where it ends)
    for (uint32_t b = lane; b < a.c.batch; b += 64) {
        const Span s = span_of(a.step, b);
        tiles0 = tiles_of(a, w, s);
        blocks0 = blocks_of(a, s);
        tiles += tiles0;
        total += (float)tiles0 * (float)blocks0;
        if (tiles0) most = max(most, blocks0);
    }
    most = max(wave_max_u32(most), 1u);
    tiles = wave_sum_u32(tiles);
    total = wave_sum(total);
    if (tiles >= w.target) return most;
    const auto whole = [&](float per) { return ((uint32_t)fminf(per, 0x1p27f) + w.unit) & ~(w.unit - 1); };
    const uint32_t last = whole(total / (float)(w.target - tiles) * 1.0001f);  // enough: a tile has less than a part more than its share
    // (more sequences than lanes are read again for every step: longer ones)
    const uint32_t step = a.c.batch > 64 ? 4 : 16;
    for (uint32_t per = whole(total / (float)w.target);; per = min((per + max(per / step, 1u) + w.unit - 1) & ~(w.unit - 1), last)) {
        if (most <= 14 + per) return most;
        if (per >= last) return per;
        const float inv = __builtin_amdgcn_rcpf((float)per);
        // parts_of(n, per): the product is off by less than one below 2^21, and beyond there are too many
        const auto parts_by = [&](uint32_t n) {
            const uint32_t x = n + per - 1, q = (uint32_t)((float)x * inv);
            const int32_t rest = (int32_t)(x - q * per);
            return max(q + (rest >= (int32_t)per) - (rest < 0), 1u);
        };
        uint32_t parts = 0;
        if (a.c.batch <= 64) {
            parts = tiles0 * parts_by(blocks0);
        } else {
            for (uint32_t b = lane; b < a.c.batch; b += 64) {
                const Span s = span_of(a.step, b);
                parts += tiles_of(a, w, s) * parts_by(blocks_of(a, s));
            }
        }
        if (wave_sum_u32(parts) <= w.target) return per;
    }
}

// Blocks of a part.  Every wave computes it alike.
template <Parts kParts, class A>
__device__ __forceinline__ uint32_t split_per(const A &a, const Split &w) {
    if constexpr (kParts == Parts::even) {
        const uint32_t per = even_per(a, w);
        // for the join: its many small workgroups would take longer over it than over the rows
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *a.per = per;
        return per;
    }
    unsigned long long total = 0;
    for (uint32_t b = __lane_id(); b < a.c.batch; b += 64) {
        const Span s = span_of(a.step, b);
        total += (unsigned long long)tiles_of(a, w, s) * blocks_of(a, s);
    }
    const unsigned long long fair = fair_share(wave_sum_u64(total), w.target);
    return max((uint32_t)((fair + w.unit - 1) / w.unit) * w.unit, w.unit);
}

// What workgroup `idx` of a head does.
struct Work {
    Span s;
    uint32_t b, tile, part, parts, per;  // parts: of this tile, at least 1
    uint32_t rows, most;                 // query rows of the sequence; slots that the tile's last row sees (under a mask all)
};
template <class A>
__device__ __forceinline__ void fill_work(const A &a, const Split &w, Work &o) {
    o.s = span_of(a.step, o.b);
    o.rows = o.s.m * a.group;
    o.most = a.sees_all() ? min(o.s.n, a.c.max_ctx) : row_limit(o.s, min(w.rows * (o.tile + 1), o.rows) - 1, a.group, a.c.max_ctx);
}
// By o.per: the part and tile that `idx` falls to, false past the last of a launch (past the shorter tile's own last, o.part is o.parts).
template <class A>
__device__ __forceinline__ bool find_part(const A &a, const Split &w, uint32_t idx, Work &o) {
    uint32_t item;
    const auto count = [&](uint32_t i) {
        const Span s = span_of(a.step, i);
        return tiles_of(a, w, s) * parts_of(blocks_of(a, s), o.per);
    };
    if (!find_item(idx, a.c.batch, count, o.b, item)) return false;
    const uint32_t tiles = tiles_of(a, w, span_of(a.step, o.b));
    o.tile = item % tiles;
    o.part = item / tiles;
    fill_work(a, w, o);
    o.parts = parts_of((o.most + 31) / 32, o.per);
    return true;
}
template <Parts kParts, class A>
__device__ __forceinline__ bool find_work(const A &a, const Split &w, uint32_t idx, Work &o) {
    o.per = split_per<kParts>(a, w);
    return find_part(a, w, idx, o) && o.part < o.parts;
}

// Many rows: where there are fewer tiles than compute units, the tiles' blocks stand in one line, tile after tile, and a workgroup
// takes an equal share of it: the end of a tile, whole ones, the beginning of the next.  (Parts of equal length, of which a whole
// number fits a tile, leave the longest workgroup a quarter more than the mean: 600 tokens over up to 12000 in four sequences,
// 10/2 heads, D 256: 124 -> 113 us.)  A tile's blocks are those that its sequence's last row sees.
// Parts cost about 14 blocks' time (O through memory, and the join), and a tile alone on a compute unit is faster than one of
// several: where the longest tile has no more blocks than 14 and the shares that a compute unit would hold, tiles stay whole
// (16/2 heads, split and whole, us.  D 128: 500 tokens 26 and 23, 1000 31 and 34, 2000 58 and 58, 200 over 1000 25 and 38;
// D 256: 1000 tokens 47 and 55; D 64: 31 and 26).
template <class A>
__device__ __forceinline__ uint32_t tile_blocks(const A &a, const Span &s) {
    return max(blocks_of(a, s), 1u);  // (a tile that sees nothing is written too)
}
// A workgroup's share, in blocks; 0: a workgroup takes a tile.
template <class A>
__device__ __forceinline__ uint32_t share_of(const A &a, const Split &w) {
    if (w.target == 0) return 0;
    uint32_t total = 0, most = 0;  // (the host splits no launch whose blocks pass 2^31)
    for (uint32_t b = __lane_id(); b < a.c.batch; b += 64) {
        const Span s = span_of(a.step, b);
        const uint32_t tiles = tiles_of(a, w, s), blocks = tile_blocks(a, s);
        total += tiles * blocks;
        if (tiles) most = max(most, blocks);
    }
    const uint32_t share = max((wave_sum_u32(total) + w.target - 1) / w.target, 1u);
    return wave_max_u32(most) <= 14 + w.unit * share ? 0 : share;
}
// The tile in which place `at` of the line falls, and where in it.
template <class A>
__device__ __forceinline__ bool find_place(const A &a, const Split &w, uint32_t at, Work &o, uint32_t &block, uint32_t &blocks) {
    uint32_t item;
    const auto count = [&](uint32_t i) {
        const Span s = span_of(a.step, i);
        return tiles_of(a, w, s) * tile_blocks(a, s);
    };
    if (!find_item(at, a.c.batch, count, o.b, item)) return false;
    blocks = tile_blocks(a, span_of(a.step, o.b));
    o.tile = item / blocks;
    block = item % blocks;
    fill_work(a, w, o);
    return true;
}

// For the joins: the tile-th tile of all, false past the last, and where its parts lie in the workspace: slot `slot` + (part 0: `odd`) +
// part * `step`.  Of a tile that is in one part (o.parts) nothing lies there.
template <Parts kParts, class A>
__device__ __forceinline__ bool find_tile(const A &a, const Split &w, uint32_t tile, Work &o, uint32_t &slot,
                                          uint32_t &odd, uint32_t &step) {
    if (!find_item(tile, a.c.batch, [&](uint32_t i) { return tiles_of(a, w, span_of(a.step, i)); }, o.b, o.tile)) return false;
    fill_work(a, w, o);
    uint32_t share = 0;
    if constexpr (kParts == Parts::shares) {
        share = share_of(a, w);
        if (share == 0) {
            o.parts = 1;
            slot = odd = 0;
            step = 1;
            return true;
        }
    } else if constexpr (kParts == Parts::even) {
        o.per = *a.per;
    } else {
        o.per = split_per<kParts>(a, w);
    }
    uint32_t before = 0;
    for (uint32_t i = __lane_id(); i < o.b; i += 64) {
        const Span s = span_of(a.step, i);
        before += tiles_of(a, w, s) * (kParts == Parts::shares ? tile_blocks(a, s) : parts_of(blocks_of(a, s), o.per));
    }
    before = wave_sum_u32(before);
    if constexpr (kParts == Parts::shares) {
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
// parts of a tile in the wide join: at most `target` and one; that join is for so few tiles that target is at most 1024
constexpr uint32_t kMostParts = 1056;
// Where a part's normalised O of a row lies in the workspace, in rows; m and l of all rows lie behind them, in pairs.
template <class A>
__device__ __forceinline__ size_t part_at(const A &a, const Split &w, uint32_t idx, uint32_t head, uint32_t row) {
    return ((size_t)idx * a.c.heads + head) * w.rows + row;
}

// A value that every lane holds, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

__device__ __forceinline__ uint32_t wave_min_uniform(uint32_t v) { return ~wave_max_u32(~v); }

// Joins the parts of the rows that were split.  kWide: a workgroup of 16 waves a row, thread (i, j) taking parts i, i + n, ...
// of four dims, for few rows in many parts; else a wave a row, its workgroup `per_group` rows of a tile (four waves: with 16, which
// find the work once for more rows, 400 tokens over 20000 in three sequences took 110 us, not 106).  Bound by latency (work count,
// maxima, parts): 16 rows in 256 parts 6.1 us, 1536 rows in a few 7, 6000 rows of 256 9 for 34 MB.
// kNanRows: rows whose L is 0 although they saw slots (all their scores -infinity) give NaN: a base above kSeenBase says so.
constexpr float kSeenBase = -1.5e38f;
constexpr uint32_t kJoinThreads = 1024, kJoinRowThreads = 256;
template <class A, int NS, Parts kParts, bool kWide, bool kNanRows>
__global__ __launch_bounds__(kWide ? kJoinThreads : kJoinRowThreads) void attn_join_kernel(A a, Split split,
                                                                                          uint32_t slots, uint32_t per_group) {
    constexpr uint32_t D = 32 * NS, kQuads = D / 4, kThreads = kWide ? kJoinThreads : 64, kWays = kThreads / kQuads;
    // parts on their way: more take registers and so waves (6000 rows of 256, eight and two: 10.4 and 9.3 us; 1536 rows of 64 8.0 and 8.5)
    constexpr int kLoads = NS <= 2 ? 8 : 2;
    __shared__ f32x4 so[kWide ? kWays : 1][kQuads];
    __shared__ float ws[kWide ? kMostParts : kJoinRowThreads], red[2][kJoinThreads / 64];
    const uint32_t lane = __lane_id(), head = blockIdx.y, wave = threadIdx.x >> 6, tid = kWide ? threadIdx.x : lane;
    const uint32_t groups = split.rows / per_group;
    Work w;
    uint32_t slot, odd, slot_step;
    if (!find_tile<kParts>(a, split, blockIdx.x / groups, w, slot, odd, slot_step)) return;
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
#pragma unroll kLoads
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
            float none = -INFINITY;
            if (kNanRows && L == 0.0f && M > kSeenBase) acc = f32x4{1, 1, 1, 1} * (none = __builtin_nanf(""));
            const u32x2 y = {pack_bf16_rne(acc.x, acc.y), pack_bf16_rne(acc.z, acc.w)};
            *reinterpret_cast<u32x2 *>(a.out + to * D + 4 * tid) = y;
            if (a.lse && tid == 0) a.lse[to] = L == 0.0f ? none : (M + __log2f(L)) * kLn2;
        }
    }
}

}  // namespace kr
