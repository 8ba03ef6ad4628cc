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
// product as bf16, as the values are (the matrix cores take f32 at a fraction of the rate, and fp16 cannot hold all values), in tiles of
// few rows, where the matrix cores wait for bytes, as two of them; l_r sums them unrounded, in f32.
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

// Where a wave's units lie, in the order in which it asks for them, 64 at a time and the next 64's pages on their way: lane l holds
// the place, in units from the pool's start, of a set's l-th (a unit of no page: the first of the pool, and its bit in `holes`).
template <class F>
struct Units {
    F unit;  // the sequence's unit that is the i-th
    const Paged &c;
    uint32_t b, head, at_lane, ahead[2];
    unsigned long long holes_now;
    __device__ __forceinline__ uint32_t look(uint32_t set) const { return page_of(c, b, unit(64 * set + __lane_id())); }
    __device__ __forceinline__ void take(uint32_t set, uint32_t p) {
        const bool hole = p >= c.pages;
        at_lane = hole ? 0u : unit_place(c, p, head, unit(64 * set + __lane_id()));
        holes_now = __ballot(hole);
    }
    __device__ __forceinline__ Units(F f, const Paged &c, uint32_t b, uint32_t head) : unit(f), c(c), b(b), head(head) {
        ahead[0] = look(0);
        ahead[1] = look(1);
    }
    // before the first use: what is loaded between has the pages' way to come as well
    __device__ __forceinline__ void begin() { take(0, ahead[0]); }
    // ... of all once more
    __device__ __forceinline__ void restart() {
        ahead[1] = look(1);
        begin();
    }
    // of the i-th unit; units in rising order, each set entered at its first
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return (uint32_t)__builtin_amdgcn_readlane((int)at_lane, (int)(i & 63)); }
    // whether the n units from i on have no page, as bits
    __device__ __forceinline__ uint32_t holes(uint32_t i, uint32_t n) const { return (uint32_t)(holes_now >> (i & 63)) & ((1u << n) - 1); }
    __device__ __forceinline__ void enter(uint32_t i) {
        if ((i & 63) == 0 && i) {
            take(i / 64, ahead[1]);
            ahead[1] = look(i / 64 + 1);
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
// therefore taken out of the operand, and added to the rows that see them one slot at a time.  (Where probabilities are two bf16, the
// second one, of either sign or 0, would make NaN of an infinity that every row sees, too: a wave that ends with a NaN takes its blocks
// once more, all of them so.)

// Takes them out of a 16-byte piece of values; returns bit 15 and 31 of a word where its low and high value is one.
__device__ __forceinline__ u32x4 take_out(u32x4 &v) {
    // an exponent of all ones, and no other, carries into the sign's bit; from there over its half
    const u32x4 m = ((v & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
    v &= ~((m << 1) - (m >> 15));
    return m;
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
//
// A workgroup takes a tile of 128 query rows, 32 a wave, or one part of its slots, on v_mfma_f32_32x32x16_bf16.  Keys and values go from
// memory to LDS past the registers, a stage ahead, with one barrier a stage; a wave's O, queries and scores stay in registers.
// In the loop, 1040 TFLOP/s at D 128 and 980 at D 256 (a library product of 8192^3: 1151), no unit is full: the matrix cores and LDS
// (every wave reads all of a chunk) are busy half of the cycles each, the vector unit a third, and an instruction of the first keeps the
// last from issuing for 11 cycles.  So exponentials, maxima and rounding are laid between products (apart, a prompt of 3907, 16/2 heads of
// 128, took 198 us), and up to D 128 a second group of four waves, over other slots and half a stage apart, takes what the first leaves;
// above, the registers hold one wave a SIMD.  A tile's start and end are 11 us (work, pages, queries and the first stage 6, the groups'
// sums 1, the next workgroup's launch 4): that prompt takes 78 to 81 us (804 to 771 TFLOP/s, from machine to machine); 600 tokens over up to 12000 in four sequences, 10/2
// heads of 256, 97 and their join 9; 250 nodes of trees over up to 5000 in eight, 16/2 heads of 128, 26 and 7.
constexpr uint32_t kManyRows = 128;

// The n-th KB from `from` on into LDS, past the registers: 16 bytes a lane, lane l's to byte lds + 1024 n + 16 l, lds the same in all lanes
// (the instruction's offset counts on both sides).  In assembly, since the compiler would have every later read of LDS wait for it:
// whoever reads what it writes waits for vmcnt(0) and a barrier first.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is a register that the compiler uses for itself alone: that is why it is named)
template <int N>
__device__ __forceinline__ void to_lds(const uint16_t *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2"
                 ::"s"(lds + N / 4 * 4096), "v"(from + N / 4 * 2048), "n"(N % 4 * 1024) : "m0", "memory");
}
#pragma clang diagnostic pop

// All but the last N of this wave's have landed (loads end in order).
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Groups of four waves: two where the registers hold two waves a SIMD, over every other pair of blocks each.
constexpr uint32_t many_groups(uint32_t D) { return D <= 128 ? 2 : 1; }
template <int NS>
constexpr uint32_t kManyGroups = many_groups(32 * NS);

template <int NS>
__global__ __launch_bounds__(256 * kManyGroups<NS>, 1) void paged_many_kernel(PagedAttnArgs a, Split split, uint32_t slots) {
    constexpr uint32_t D = 32 * NS, G = kManyGroups<NS>;
    // A stage is G chunks of 64 slots, one a group: four units of NS pieces of 1 KB.  [keys, values][stage & 1][group][unit][piece]
    constexpr uint32_t kPiece = 1024, kUnit = NS * kPiece, kChunk = 4 * kUnit, kStage = G * kChunk, kKind = 2 * kStage;
    constexpr int kProducts = 4 * NS;  // of a chunk: of its scores, and of its values
    __shared__ __align__(16) char lds[2 * kKind];
    __shared__ float2 lds_ml[4][32];
    __shared__ uint32_t lds_bad[2][G][2];  // [stage & 1][group]: slots of values that were taken out
    const auto lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const uint32_t lane = __lane_id(), r32 = lane & 31, h = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % 4, group = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    // heads side by side: with eight of them each XCD's L2 keeps the keys and values of one
    const uint32_t head = blockIdx.x % a.c.heads, idx = blockIdx.x / a.c.heads;
    const float c = score_factor(a.scale_log2);
    const uint32_t sign = query_sign(a.scale_log2);
    Work w;
    uint32_t first = 0, end;
    bool whole = true;
    if (split.target) {
        if (!find_work<Parts::even>(a, split, idx, w)) return;
        first = w.part * w.per;
        end = min(first + w.per, (w.most + 31) / 32);
        whole = w.parts == 1;
    } else {
        if (!find_item(idx, a.c.batch, [&](uint32_t i) { return tiles_of(a, split, span_of(a.step, i)); }, w.b, w.tile)) return;
        w.tile = tiles_of(a, split, span_of(a.step, w.b)) - 1 - w.tile;  // the tiles that see the most first
        fill_work(a, split, w);
        end = (w.most + 31) / 32;
    }
    const Span &s = w.s;
    const uint32_t r0 = kManyRows * w.tile, r = r0 + 32 * wave + r32;
    const bool live = r < w.rows;
    const Sight sight = sight_of(a, s, r, live);
    const uint32_t clear = r0 + 32 * wave < w.rows ? clear_of(a, s, r0 + 32 * wave) : kAll;  // (of rows past the end nothing counts)
    const uint32_t b = w.b, t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    f32x16 o[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) o[i] = f32x16{};
    RowSums sums;
    // stage i: blocks first + 2 G i ..; the group's own two from block_of(i) on
    const uint32_t stages = first < end ? (end - first + 2 * G - 1) / (2 * G) : 0;
    const auto block_of = [&](uint32_t i) { return first + 2 * (G * i + group); };
    Units units([&](uint32_t i) { return 2 * first + i; }, a.c, b, head);
    // (a row past the sequence's takes the tile's first one's query; nothing of it is written)
    const uint32_t rq = live ? r : r0;
    const uint16_t *query = a.q + (s.t0 + rq / a.group) * a.q_stride + (size_t)(head * a.group + rq % a.group) * D + 8 * h;
    bf16x8_t q[2 * NS];
#pragma unroll
    for (int i = 0; i < 2 * NS; ++i) q[i] = *reinterpret_cast<const bf16x8_t *>(query + 16 * i);
    units.begin();
    const uint32_t clear_tile = clear_of(a, s, r0);
    // A wave brings one of the four units, its keys or its values, into LDS, NS pieces: `unit` where it lies in the pool.
    struct Request {
        const uint16_t *from;
        uint32_t to;
    };
    const auto request = [&](uint32_t kind, uint32_t unit, uint32_t to) {
        return Request{(kind ? a.c.v : a.c.k) + (size_t)unit * (kPagedUnit * D) + 8 * lane, lds_base + kind * kKind + to + group * kChunk + wave * kUnit};
    };
    const auto all_of = [&](const Request &x) { static_for<NS>([&](auto n) { to_lds<n>(x.from, x.to); }); };
    // Octet 2 j + h of slot r32 of two units, 256 bytes an octet, is the j-th operand of keys; 16 bytes of lane (dim, h) of a unit
    // and 32 dims are an operand of values.
    const char *key_at = lds + group * kChunk + (r32 >> 4) * kUnit + h * 256 + (r32 & 15) * 16;
    const char *value_at = lds + kKind + group * kChunk + lane * 16;
    // operand m of a chunk: of keys block m / 2 NS, dims 16 (m % 2 NS) ..; of values unit m / NS, 32 dims m % NS
    const auto key = [&](uint32_t from, int m) { return *reinterpret_cast<const bf16x8_t *>(key_at + from + 512 * (m % (2 * NS)) + 2 * kUnit * (m / (2 * NS))); };
    const auto value = [&](uint32_t from, int m) { return *reinterpret_cast<const u32x4 *>(value_at + from + kUnit * (m / NS) + kPiece * (m % NS)); };
    // Scores of the chunk's two blocks, the second in p[0] and the first in p[1], and the next chunk's first block's: the next second
    // block's take p[0]'s place, once its exponentials are under way, and z then p[1]'s.
    f32x16 p[2], z;
    u32x4 pf[4];       // probabilities of the four units
    uint32_t seen[2];  // the slots of the next chunk's blocks that the row sees
    float s0 = 0.0f, s1 = 0.0f;

    // The pair k of the scores, 2 elements of 32: exponentials, then their sums and rounding.
    float e[2][2];
    const auto exponent = [&](int k) {
#pragma unroll
        for (int x = 0; x < 2; ++x) e[k & 1][x] = __builtin_amdgcn_exp2f(fmaf(p[k / 8][2 * (k % 8) + x], c, -sums.base));
    };
    const auto round = [&](int k) {
        s0 += e[k & 1][0];
        s1 += e[k & 1][1];
        uint32_t both = pack_bf16_rne(e[k & 1][0], e[k & 1][1]);
        asm volatile("" : "+v"(both), "+v"(s0), "+v"(s1));  // (here: not where the compiler would put it, in one run before its use)
        pf[(k / 4 + 2) % 4][k % 4] = both;
    };
    // A look ahead of kLook operands in registers.  Between the products, `also(m)` gives the vector unit its share.
    constexpr int kLook = NS <= 4 ? 4 : 8;
    const auto scores = [&](uint32_t from, auto &&also) {
        bf16x8_t kf[kLook];
#pragma unroll
        for (int m = 0; m < kLook; ++m) kf[m] = key(from, m);
        static_for<kProducts>([&](auto at) {
            constexpr int m = at;
            f32x16 &to = m < 2 * NS ? z : p[0];
            if constexpr (m % (2 * NS) == 0) to = f32x16{};
            to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[m % kLook], q[m % (2 * NS)], to, 0, 0, 0);
            if constexpr (m + kLook < kProducts) kf[m % kLook] = key(from, m + kLook);
            also(at);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    const auto average = [&](uint32_t from, auto &&also) {
        u32x4 vf[kLook];
#pragma unroll
        for (int m = 0; m < kLook; ++m) vf[m] = value(from, m);
        static_for<kProducts>([&](auto at) {
            constexpr int m = at;
            o[m % NS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[m % kLook]), __builtin_bit_cast(bf16x8_t, pf[m / NS]),
                                                                o[m % NS], 0, 0, 0);
            if constexpr (m + kLook < kProducts) vf[m % kLook] = value(from, m + kLook);
            also(at);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // A stage that some row of the tile does not see whole, and a chunk that some row of the wave does not (n blocks, holes of their
    // units).
    const auto has_edge = [&](uint32_t from, uint32_t n, uint32_t sees, uint32_t holes) { return from + n > end || 32 * (from + n) > sees || holes; };
    const auto stage_edge = [&](uint32_t i, uint32_t holes) { return has_edge(first + 2 * G * i, 2 * G, clear_tile, holes); };
    // Takes infinities and NaN out of a stage's values in LDS, once all have landed; `clean` before that, a barrier after it.
    const auto clean = [&](uint32_t i) {
        if (threadIdx.x % 256 < 2) lds_bad[i & 1][group][threadIdx.x % 256] = 0;
    };
    const auto take_out_all = [&](uint32_t i, uint32_t from) {
        // a thread a 16-byte piece of each KB that its wave brought: all of unit `wave`, slots 8 a + 4 h + j
        u32x4 words = {};
#pragma unroll
        for (int d = 0; d < NS; ++d) {
            u32x4 *v = reinterpret_cast<u32x4 *>(lds + kKind + from + group * kChunk + wave * kUnit + kPiece * d) + lane;
            u32x4 x = *v;
            words |= take_out(x);
            *v = x;
        }
        const uint32_t bad = bad_slots(words) << (16 * (wave & 1) + 4 * h);
        if (bad) atomicOr(&lds_bad[i & 1][group][wave >> 1], bad);
    };
    // ... and gives them to the rows that see them; seen_by: the chunk's slots that the row sees.
    const auto put_back_all = [&](uint32_t i, const uint32_t (&seen_by)[2]) {
#pragma unroll 1
        for (uint32_t y = 0; y < 2; ++y) {
            const uint32_t sees = y ? seen_by[1] : seen_by[0];
            uint32_t rest = lds_bad[i & 1][group][y];
            if (rest) rest &= wave_or(sees);  // (what no row sees is left out)
            for (rest = __builtin_amdgcn_readfirstlane(rest); rest; rest &= rest - 1) {
                const uint32_t slot = (uint32_t)__builtin_ctz(rest), unit = 2 * (block_of(i) + y) + slot / 16;
                const uint16_t *v = a.c.v + unit_at(a.c, page_of(a.c, b, unit), head, unit) + paged_value_at(slot % 16, 4 * h);
#pragma unroll
                for (int d = 0; d < NS; ++d) {
#pragma unroll
                    for (int x = 0; x < 16; ++x) o[d][x] = put_back(o[d][x], v[512 * d + 8 * (8 * (x >> 2) + (x & 3))], sees >> slot & 1);
                    __builtin_amdgcn_sched_barrier(0);  // (one at a time: registers)
                }
            }
        }
    };
    // Of the next stage's scores: slots that a row does not see get -infinity.
    const auto hide = [&](uint32_t i, uint32_t holes) {
        const uint32_t n = block_of(i);
        holes = holes >> (4 * group) & 15;
        seen[0] = seen[1] = kAll;
        if (!has_edge(n, 2, clear, holes)) return;
        static_for<2>([&](auto at) {
            constexpr uint32_t k = at;
            f32x16 &y = k ? p[0] : p[1];
            const uint32_t none = (holes >> (2 * k) & 1 ? 0xFFFFu : 0u) | (holes >> (2 * k) & 2 ? 0xFFFF0000u : 0u);
            seen[k] = n + k < end ? sight.bits(32 * (n + k)) & ~none : 0u;
#pragma unroll
            for (int x = 0; x < 16; ++x) y[x] = seen[k] >> (8 * (x >> 2) + 4 * h + (x & 3)) & 1 ? y[x] : -INFINITY;
        });
    };
    // Their maximum, in eight steps of two; the row's base follows where it is passed.
    float top[2];
    const auto highest = [&](int k) {
        if (k == 0) top[0] = top[1] = -INFINITY;
#pragma unroll
        for (int x = 0; x < 2; ++x) top[x] = fmaxf(fmaxf(top[x], p[x][2 * k]), p[x][2 * k + 1]);
    };
    const auto follow = [&] {
        float m = fmaxf(top[0], top[1]) * c;
        m = fmaxf(m, xchg32(m, lane));
        if (seen[0] | seen[1]) m = fmaxf(m, kLowBase);
        if (__any(m > sums.base + kLag)) {
            const float down = row_follow(sums, m);
            s0 *= down;
            s1 *= down;
#pragma unroll
            for (int d = 0; d < NS; ++d) o[d] *= down;
        }
    };
    if (stages) {
        // The loop of a wave: next scores beside exponentials, values' products beside the next maxima.  Of a SIMD's two waves the
        // second group's is half a stage ahead: one is at the exponentials, which take the vector unit longer than the matrix
        // cores take the products beside them, while the other one's products want little else.  Its keys come a stage earlier.
        constexpr uint32_t kOfStage = 4 * G;
        const auto unit_of = [&](uint32_t i) { return units.at(kOfStage * i + 4 * group + wave); };
        const auto holes_of = [&](uint32_t i) { return units.holes(kOfStage * i, kOfStage); };
        const auto next_scores = [&](uint32_t from, auto &&also) {
            scores(from, [&](auto at) {
                constexpr int m = at;
                static_for<16 * (m + 1) / kProducts - 16 * m / kProducts>([&](auto x) {
                    constexpr int k = 16 * m / kProducts + x;
                    exponent(k);
                    if constexpr (k > 0) round(k - 1);
                });
                also(at);
            });
            round(15);
            p[1] = z;
        };
        // keys of stages 0 and 1, values of 0
        uint32_t u0 = unit_of(0), u1 = unit_of(1), u2 = unit_of(2), h0 = holes_of(0), h1 = holes_of(1), h2 = holes_of(2);
        all_of(request(0, u0, 0));
        all_of(request(1, u0, 0));
        all_of(request(0, u1, kStage));  // (past the last stage: a unit that nothing reads)
        bool edge = stage_edge(0, h0);
        if (edge) clean(0);
        landed<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2 * NS; ++i) q[i] = __builtin_bit_cast(bf16x8_t, __builtin_bit_cast(u32x4, q[i]) ^ u32x4{sign, sign, sign, sign});
        scores(0, [](auto) {});
        p[1] = z;
        hide(0, h0);
#pragma unroll
        for (int k = 0; k < 8; ++k) highest(k);
        follow();
        if constexpr (G == 2) {
            __syncthreads();  // keys 0 have been read
            if (group == 1) {
                all_of(request(0, u2, 0));
                next_scores(kStage, [](auto) {});
            }
        }
        uint32_t now = 0;  // the buffers of stage i
        for (uint32_t i = 0; i + 1 < stages; ++i) {
            // what this stage reads has landed, and what is overwritten has been read
            landed<0>();
            __syncthreads();
            if (edge) {
                take_out_all(i, now);
                __syncthreads();
            }
            const uint32_t other = now ^ kStage;
            units.enter(kOfStage * (i + 3));
            const uint32_t u3 = unit_of(i + 3), h3 = holes_of(i + 3);
            const Request values = request(1, u1, other), keys = group ? request(0, u3, other) : request(0, u2, now);
            // a KB for the stages after with every few products
            if (group == 0) {
                next_scores(other, [&](auto at) {
                    if constexpr (at % 4 == 1) to_lds<at / 4>(values.from, values.to);
                });
            }
            const uint32_t seen_now[2] = {seen[0], seen[1]};
            hide(i + 1, h1);
            average(now, [&](auto at) {
                constexpr int m = at;
                static_for<8 * (m + 1) / kProducts - 8 * m / kProducts>([&](auto x) { highest(8 * m / kProducts + x); });
                if constexpr (m % 4 == 1) to_lds<m / 4>(keys.from, keys.to);
            });
            if (edge) put_back_all(i, seen_now);
            follow();
            if (G == 2 && group == 1) {
                next_scores(now, [&](auto at) {
                    if constexpr (at % 4 == 1) to_lds<at / 4>(values.from, values.to);
                });
            }
            edge = stage_edge(i + 1, h1);
            if (edge) clean(i + 1);
            u1 = u2;
            u2 = u3;
            h1 = h2;
            h2 = h3;
            now = other;
        }
        if (group == 0) {
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                exponent(k);
                round(k);
            }
        }
        landed<0>();
        __syncthreads();
        if (edge) {
            take_out_all(stages - 1, now);
            __syncthreads();
        }
        average(now, [](auto) {});
        if (edge) put_back_all(stages - 1, seen);
    }
    sums.l = s0 + s1;
    float l = sums.l + xchg32(sums.l, lane);
    if constexpr (G == 2) {  // the second group's sums join the first's
        __syncthreads();
            f32x4 *other = reinterpret_cast<f32x4 *>(lds) + wave * (4 * NS * 64) + lane;
        if (group == 1) {
            if (h == 0) lds_ml[wave][r32] = make_float2(sums.base, l);
#pragma unroll
            for (int d = 0; d < NS; ++d)
#pragma unroll
                for (int x = 0; x < 4; ++x) other[(4 * d + x) * 64] = f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
        }
        __syncthreads();
        if (group == 1) return;
        const float2 ml = lds_ml[wave][r32];
        const float base = fmaxf(sums.base, ml.x), f0 = __builtin_amdgcn_exp2f(sums.base - base), f1 = __builtin_amdgcn_exp2f(ml.x - base);
        sums.base = base;
        l = l * f0 + ml.y * f1;
#pragma unroll
        for (int d = 0; d < NS; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 y = other[(4 * d + x) * 64];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[d][4 * x + k] = fmaf(o[d][4 * x + k], f0, y[k] * f1);
            }
    }
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
                for (int x = 0; x < 16; ++x) o[d][x] = __builtin_nanf("");
        }
        const size_t to = (size_t)t * a.q_heads + qh;
        if (a.lse && h == 0) a.lse[to] = l == 0.0f ? (nan ? __builtin_nanf("") : -INFINITY) : (sums.base + __log2f(l)) * kLn2;
        uint16_t *out = a.out + to * D;
#pragma unroll
        for (int d = 0; d < NS; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<u32x2 *>(out + 32 * d + 8 * x + 4 * h) = pack4(o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]);
    } else {
        const size_t to = part_at(a, split, idx, head, r - r0);
#pragma unroll
        for (int d = 0; d < NS; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4 *>(a.part + to * D + 32 * d + 8 * x + 4 * h) =
                    f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
        if (h == 0) {
            float *ml = a.part + (size_t)slots * a.c.heads * kManyRows * D + 2 * to;
            ml[0] = sums.base;
            ml[1] = l;
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
// Bound by bytes: 48 sequences up to 8000, 32/8 heads of 64, 103 us for 595 MB, 5.8 TB/s (a copy 5.2, a plain read 7.0); one of 131072,
// 16/2 heads of 128, 25 us for 134 MB; by latency where there are few: five sequences up to 3000 8.4 us.
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
// Units at u0 and u1.
template <int NS, bool kOnce>
__device__ __forceinline__ void load_few(FewBlock<NS> &f, const Paged &c, uint32_t u0, uint32_t u1, uint32_t holes) {
    const auto load16 = [](const u32x4 *p) { return kOnce ? __builtin_nontemporal_load(p) : *p; };
    constexpr size_t kSize = kPagedUnit * 32 * NS;
    const uint32_t lane = __lane_id(), r = lane & 15, g = lane >> 4;
    f.holes = (holes & 1 ? 0xFFFFu : 0u) | (holes & 2 ? 0xFFFF0000u : 0u);
    const uint16_t *k = c.k + (r >> 3 ? u1 : u0) * kSize + 128 * g + 8 * (r & 7);
    const uint16_t *v = c.v + (g >> 1 ? u1 : u0) * kSize + 256 * (g & 1) + 8 * r;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < NS; ++j) f.k[t][j] = load16(reinterpret_cast<const u32x4 *>(k + 512 * j + 64 * t));
#pragma unroll
    for (int d = 0; d < NS; ++d)
#pragma unroll
        for (int x = 0; x < 2; ++x) f.v[d][x] = load16(reinterpret_cast<const u32x4 *>(v + 512 * d + 128 * x));
}

// kOnce: what is read is read once: past the caches (nontemporal).
template <int NS, bool kOnce>
__global__ __launch_bounds__(256, kFewGroups<NS>) void paged_few_kernel(PagedAttnArgs a, Split split) {
    constexpr uint32_t D = 32 * NS;
    __shared__ float sm[kFewWaves][kFewRows], sl[kFewWaves][kFewRows];
    __shared__ __align__(16) float so[kFewWaves][kFewRows][D + 4];
    const uint32_t lane = __lane_id(), r16 = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t head = blockIdx.y, idx = blockIdx.x;
    Work w;
    if (!find_work<Parts::even>(a, split, idx, w)) return;
    const Span &s = w.s;
    const uint32_t r0 = kFewRows * w.tile, r = r0 + r16;
    const bool live = r < w.rows;
    const Sight sight = sight_of(a, s, r, live);
    uint32_t clear = clear_of(a, s, r0);
    const uint32_t first = w.part * w.per, end = min(first + w.per, (w.most + 31) / 32), b = w.b;
    const uint32_t t = s.t0 + r / a.group, qh = head * a.group + r % a.group;
    uint32_t blk = first + wave;
    // kFewAhead<NS> blocks of a wave on their way
    constexpr uint32_t kAhead = kFewAhead<NS>;
    FewBlock<NS> f[kAhead];
    // unit i of the wave: half i % 2 of its i / 2-th block
    Units units([&](uint32_t i) { return 2 * (first + wave + kFewWaves * (i / 2)) + i % 2; }, a.c, b, head);
    units.begin();
    uint32_t asked = 0;
    const auto ask = [&](FewBlock<NS> &f) {
        units.enter(asked);
        load_few<NS, kOnce>(f, a.c, units.at(asked), units.at(asked + 1), units.holes(asked, 2));
        asked += 2;
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (blk + i * kFewWaves < end) ask(f[i]);
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
        // in two bf16 each, the second what the first leaves: to 2^-17 of them (one alone is off by as much as the result's own rounding)
        u32x4 high, low;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            high[i] = pack_bf16_rne(e[2 * i], e[2 * i + 1]);
            low[i] = pack_bf16_rne(e[2 * i] - __uint_as_float(high[i] << 16), e[2 * i + 1] - __uint_as_float(high[i] & 0xFFFF0000u));
        }
        uint32_t bad = 0;
        if (edge) {
            u32x4 words = {};
#pragma unroll
            for (int d = 0; d < 2 * NS; ++d) words |= take_out(f.v[d >> 1][d & 1]);
            bad = bad_slots(words) << (16 * (g >> 1) + 4 * (g & 1));
        }
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) {
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f.v[d >> 1][d & 1]), __builtin_bit_cast(bf16x8_t, high), o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f.v[d >> 1][d & 1]), __builtin_bit_cast(bf16x8_t, low), o[d], 0, 0, 0);
        }
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
    for (;;) {
        for (; blk < end; blk += kAhead * kFewWaves) {
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                const uint32_t at = blk + i * kFewWaves;
                if (at >= end) break;
                step(f[i], at);
                if (at + kAhead * kFewWaves < end) ask(f[i]);
            }
        }
        float nan = 0.0f;
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) nan += (o[d][0] + o[d][1]) + (o[d][2] + o[d][3]);
        if (__builtin_expect(clear == 0 || !__any(nan != nan), 1)) break;
        clear = 0;  // every block as one that some row does not see whole
        sums = RowSums{};
#pragma unroll
        for (int d = 0; d < 2 * NS; ++d) o[d] = f32x4{0, 0, 0, 0};
        blk = first + wave;
        asked = 0;
        units.restart();
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
            if (blk + i * kFewWaves < end) ask(f[i]);
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
        } else if (idx < split.target) {  // (where the tiles are `target` and more, none is split: only `target` parts have a place)
            const size_t to = part_at(a, split, idx, head, row);
            *reinterpret_cast<f32x4 *>(a.part + to * D + d) = acc;
            if (d == 0) {
                float *ml = a.part + (size_t)split.target * a.c.heads * kFewRows * D + 2 * to;
                ml[0] = M;
                ml[1] = L;
            }
        }
    }
}

namespace {

// How a step is launched: tiles of 16 rows where the sequences have few query rows, else of 128.
struct AttnPlan {
    bool few, once;
    Split split;
    uint32_t tiles, grid, slots;  // at most, a head; slots: of parts in the workspace
};
AttnPlan plan_of(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    AttnPlan p{};
    const uint64_t rows = (uint64_t)tokens * group;
    // Few rows: one tile of 16 a sequence, or all the rows there are over so few slots that their latency counts (us, few and many.
    // D 128, 2 heads: 16 tokens of 8 rows over 3000 14.9 and 18.4, 8 over 100000 69 and 35, 8 sequences of 8 over 300 12.6 and 16.9, over
    // 3000 25.7 and 22.0; D 64, 8 heads: 8 sequences of 4 tokens of 4 rows 19.2 and 25.1, 32 of 8 tokens 68 and 41).
    p.few = rows <= 16ull * batch || rows * kv_heads * max_ctx <= 3u << 19;
    p.split.rows = p.few ? kFewRows : kManyRows;
    // tiles of every sequence: at most one that is not full each
    p.tiles = (uint32_t)(rows / p.split.rows) + std::min(batch, tokens);
    if (p.few) {
        // Keys and values that one tile reads in the mean, and more of them than may still be in the caches from the last call (a chunk among
        // decoded tokens reads its own once a tile all the same: 63 and one of 193, 32/8 heads of 64, contexts of 4000 to 8000, 259 us, in two
        // calls 174.  us, with and without,
        // over changing layers: 48 sequences up to 8000, 32/8 heads of 64, 110 and 122; 4 of 4000, 16/2 heads of 128, 16.0 and 16.3, one
        // 14.4 and 13.6; 8 of 32 rows over 300 16.7 and 14.1).
        p.once = rows <= 16ull * batch && (uint64_t)batch * max_ctx * kv_heads * D * 4 >= 1u << 24;
        p.split.unit = kFewWaves;
        // as many workgroups as the card holds at once, or where the tiles are as many already, twice that (64 sequences up to 3000,
        // 32/8 heads of 128, 89 us -> 81; below, a second round costs more: 40 of 4000 119 -> 125)
        const uint32_t held = (D <= 64 ? 768 : (D <= 128 ? 512 : 256)) / kv_heads;
        p.split.target = p.tiles < held ? held : std::max(2 * held, std::min(p.tiles, 1024u));
        p.grid = std::max(p.split.target, p.tiles);
        p.slots = p.split.target;
    } else {
        p.split.unit = D <= 128 ? 4 : 2;  // a stage
        // Contexts that a table can hold in so few blocks are not split: the join's launch takes longer (split and whole, us, D 128, 2 heads:
        // 1000 tokens 30 and 25, 200 over 1000 24 and 27; D 256: 500 tokens 29 and 26, 100 over 800 33 and 39).
        const uint32_t longest = (max_ctx + 31) / 32;
        const bool split = (uint64_t)p.tiles * kv_heads < 256 && longest > 4096 / D;
        p.split.target = split ? 256 / kv_heads : 0;  // as many workgroups as the card holds at once: at least `tiles`
        p.grid = p.split.target ? p.split.target : p.tiles;
        p.slots = p.split.target;
    }
    return p;
}

size_t part_floats(const AttnPlan &p, uint32_t kv_heads, uint32_t D) { return (size_t)p.slots * kv_heads * p.split.rows * (D + 2); }

}  // namespace

uint64_t paged_attention_groups(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    const AttnPlan p = plan_of(batch, kv_heads, group, D, tokens, max_ctx);
    return (uint64_t)p.grid * (p.few ? 1 : kv_heads * many_groups(D));  // (few: heads are another dimension)
}

size_t paged_attention_workspace_bytes(uint32_t batch, uint32_t kv_heads, uint32_t group, uint32_t D, uint32_t tokens, uint32_t max_ctx) {
    const AttnPlan p = plan_of(batch, kv_heads, group, D, tokens, max_ctx);
    return p.slots ? part_floats(p, kv_heads, D) * sizeof(float) + 16 : 0;
}

hipError_t launch_paged_attention(const PagedAttnArgs &args, hipStream_t s) {
    PagedAttnArgs a = args;
    const AttnPlan p = plan_of(a.c.batch, a.c.heads, a.group, a.c.D, a.step.tokens, a.c.max_ctx);
    a.per = reinterpret_cast<uint32_t *>(a.part + part_floats(p, a.c.heads, a.c.D));
    const auto launch = [&](auto ns) -> hipError_t {
        constexpr int NS = decltype(ns)::value;
        if (p.few && p.once) paged_few_kernel<NS, true><<<dim3(p.grid, a.c.heads), 256, 0, s>>>(a, p.split);
        else if (p.few) paged_few_kernel<NS, false><<<dim3(p.grid, a.c.heads), 256, 0, s>>>(a, p.split);
        else paged_many_kernel<NS><<<dim3(p.grid * a.c.heads), 256 * kManyGroups<NS>, 0, s>>>(a, p.split, p.slots);
        if (hipError_t e = hipGetLastError()) return e;
        if (p.split.target == 0) return hipSuccess;
        if (p.few && (uint64_t)p.tiles * p.split.rows * a.c.heads <= 256) {
            attn_join_kernel<PagedAttnArgs, NS, Parts::even, true, true><<<dim3(p.tiles * p.split.rows, a.c.heads), kJoinThreads, 0, s>>>(a, p.split, p.slots, 1);
        } else {
            uint32_t per_group = kJoinRowThreads / 64;
            while (per_group < p.split.rows && (uint64_t)p.tiles * a.c.heads * (p.split.rows / per_group) > 2048) per_group *= 2;
            const dim3 grid(p.tiles * (p.split.rows / per_group), a.c.heads);
            attn_join_kernel<PagedAttnArgs, NS, Parts::even, false, true><<<grid, kJoinRowThreads, 0, s>>>(a, p.split, p.slots, per_group);
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
