// paged_cache.hip — the paged key/value cache: appending (with the heads' norm and the rotation), and reading back.
//
// Reference semantics of the append (norm, rotation, order):
//   kernels/metal/paged_gqa_and_deltanet.metal:115-222
#include <algorithm>

#include "paged.hpp"
#include "rope.hpp"

namespace kr {

namespace {

// The units that sequence b's new tokens fall into: `first` .. first + items - 1 (slots n0 .. end - 1 are new).
struct UnitSpan {
    Span s;
    uint32_t n0, end, first, items;
};
__device__ __forceinline__ UnitSpan unit_span(const PagedAppendArgs &a, uint32_t b) {
    UnitSpan r;
    r.s = span_of(a.step, b);
    r.n0 = r.s.n > r.s.m ? r.s.n - r.s.m : 0u;
    r.end = min(r.s.n, a.c.max_ctx);
    r.first = r.n0 / kPagedUnit;
    r.items = r.end > r.n0 ? (r.end - 1) / kPagedUnit - r.first + 1 : 0u;
    return r;
}

// Heads of a unit that a workgroup takes: as many as make about 512 dims.
__host__ __device__ constexpr uint32_t chunk_heads(uint32_t D) { return 512 / D; }
// Threads of a row, each with two pieces of 8 dims: the power of two from D / 16 on.
__host__ __device__ constexpr uint32_t row_threads(uint32_t D) { return D <= 64 ? 4 : (D <= 128 ? 8 : 16); }

enum RopeKind : int { kNone, kHalf, kNeighbours, kAny };  // kHalf, kNeighbours: rotary_dim a multiple of 16

// Dim d's partner in its pair, whether d is the pair's first, and its place in the table's row.
struct Pair {
    uint32_t other, at;
    bool first;
};
__device__ __forceinline__ Pair pair_of(const RopeArgs &r, uint32_t d) {
    if (r.interleaved) return Pair{d ^ 1, d / 2, d % 2 == 0};
    const uint32_t half = r.rotary_dim / 2;
    return d < half ? Pair{d + half, d, true} : Pair{d - half, d - half, false};
}

}  // namespace

// Workgroups: values of (unit, chunk of kv heads), keys of the same, then query rows.
// Values come through LDS: a thread then collects the 8 slots of a dim that lie together.  16-byte pieces whose slots are not all new
// are written slot by slot: the others hold older tokens.
// Keys and queries: row_threads(D) threads a row, each with the two pieces of 8 dims that its rotation pairs (neighbouring ones
// without), so that norm, rotation and rounding stay in registers; the row's sum of squares goes over its lanes.  kAny pairs dims that
// lie anywhere: their partners are read one by one.
// Bound by latency where tokens are few (16 tokens, 2 heads of 128, 16 queries: 4.0 us: lengths, rows and table, pages, stores) and by
// bytes where they are many (3907 tokens, 8 heads of 64, 32 queries, norm and rotation: 12.6 us for 49 MB, 3.9 TB/s; rows that went
// through LDS took 39).
template <uint32_t D, int kRope>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, uint32_t items) {
    constexpr uint32_t kUnits = D / 8, kChunk = chunk_heads(D), kLanes = row_threads(D), kRowsAtOnce = 256 / kLanes;
    __shared__ __align__(16) uint16_t vs[kPagedUnit][kChunk * D];
    const uint32_t chunks = (a.c.heads + kChunk - 1) / kChunk, groups = items * chunks;
    const bool query = blockIdx.x >= 2 * groups;
    UnitSpan s{};
    uint32_t u = 0, h0 = 0, heads = 0, from = 0, count = 0, t0 = 0, r0 = 0;  // slots `from` .., count of them; tokens t0 ..; r0: in the unit
    size_t base = 0, head_step = 0;
    if (!query) {
        const uint32_t i = blockIdx.x % groups;
        uint32_t b, item;
        if (!find_item(i / chunks, a.c.batch, [&](uint32_t x) { return unit_span(a, x).items; }, b, item)) return;
        s = unit_span(a, b);
        u = s.first + item;
        const uint32_t page = page_of(a.c, b, u);
        if (page >= a.c.pages) return;
        h0 = i % chunks * kChunk;
        heads = min(kChunk, a.c.heads - h0);
        from = max(s.n0, u * kPagedUnit);
        count = min(s.end, (u + 1) * kPagedUnit) - from;
        r0 = from % kPagedUnit;
        t0 = s.s.t0 + (from + s.s.m - s.s.n);
        base = unit_at(a.c, page, h0, u);
        head_step = (size_t)(kPagedUnit << a.c.shift) * D;
    }
    if (blockIdx.x < groups) {
        const uint32_t width = heads * kUnits;  // pieces of a token
        const uint16_t *src = a.v + t0 * a.kv_stride + (size_t)h0 * D;
        for (uint32_t i = threadIdx.x; i < count * width; i += 256) {
            const uint32_t r = i / width, x = i % width;
            *reinterpret_cast<u32x4 *>(&vs[r0 + r][8 * x]) = *reinterpret_cast<const u32x4 *>(src + r * a.kv_stride + 8 * x);
        }
        __syncthreads();
        // piece i of a head: dims i / 64 32 + i % 32, half h = i / 32 % 2: slots 4 h + j and 8 + 4 h + j
        for (uint32_t i = threadIdx.x; i < heads * 2 * D; i += 256) {
            const uint32_t head = i / (2 * D), p = i % (2 * D), h = p / 32 % 2, d = head * D + p / 64 * 32 + p % 32;
            uint16_t *to = a.c.v + base + head * head_step + 8 * p;
            uint32_t e[8];
#pragma unroll
            for (uint32_t x = 0; x < 8; ++x) e[x] = vs[x / 4 * 8 + 4 * h + x % 4][d];
            if (count == kPagedUnit) {
                *reinterpret_cast<u32x4 *>(to) = u32x4{e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16};
            } else {
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x)
                    if (x / 4 * 8 + 4 * h + x % 4 - r0 < count) to[x] = (uint16_t)e[x];
            }
        }
        return;
    }
    // rows: (slot, head) of a unit's keys, or (token, head) of the queries
    const uint32_t of = query ? a.q_heads : heads;  // rows of a token
    uint32_t row = threadIdx.x / kLanes, end = count * heads;
    size_t first_row = 0;
    if (query) {
        first_row = (size_t)(blockIdx.x - 2 * groups) * kRowsAtOnce;
        const size_t rows = (size_t)a.step.tokens * a.q_heads;
        end = (uint32_t)min((size_t)kRowsAtOnce, rows - first_row);
    }
    const uint16_t *weight = query ? a.q_norm : a.k_norm;
    const uint32_t p = threadIdx.x % kLanes, R = a.rope.rotary_dim;
    // the thread's pieces
    uint32_t u0 = 2 * p, u1 = 2 * p + 1;
    bool turns = kRope == kNeighbours ? 16 * p < R : false;
    if constexpr (kRope == kHalf) {
        turns = 16 * p < R;
        u0 = turns ? p : 2 * p;
        u1 = turns ? p + R / 16 : 2 * p + 1;
    }
    const bool mine = 16 * p < D;
    for (; row < (end + kRowsAtOnce - 1) / kRowsAtOnce * kRowsAtOnce; row += kRowsAtOnce) {
        const bool live = row < end && mine;
        const size_t at = first_row + min(row, end - 1);
        const uint32_t t = query ? (uint32_t)(at / of) : t0 + (uint32_t)at / of, head = (uint32_t)(at % of);
        const bool nobody = query && a.step.starts && (t < a.step.starts[0] || t >= a.step.starts[a.c.batch]);
        const uint16_t *src = query ? a.q + t * a.q_stride + (size_t)head * D : a.k + t * a.kv_stride + (size_t)(h0 + head) * D;
        float lo[8], hi[8];
        load8(src + (mine ? 8 * u0 : 0u), lo);
        load8(src + (mine ? 8 * u1 : 0u), hi);
        float f = 1.0f;
        if (weight) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], sum));
            if (!mine) sum = 0.0f;
#pragma unroll
            for (uint32_t x = 1; x < kLanes; x *= 2) sum += __shfl_xor(sum, (int)x);
            f = rsqrtf(sum * (1.0f / D) + a.eps);
            float w0[8], w1[8];
            load8_at(weight + (mine ? 8 * u0 : 0u), w0);
            load8_at(weight + (mine ? 8 * u1 : 0u), w1);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                lo[e] = lo[e] * f * w0[e];
                hi[e] = hi[e] * f * w1[e];
            }
        }
        if constexpr (kRope != kNone) {
            const uint32_t pos = a.rope.positions[t];
            const float *cs = a.rope.cos_sin + (size_t)(pos < a.rope.rows ? pos : 0u) * R;
            if constexpr (kRope == kAny) {
                if (pos < a.rope.rows) {
                    const auto turn = [&](float (&y)[8], uint32_t u) {
#pragma unroll
                        for (uint32_t e = 0; e < 8; ++e) {
                            const uint32_t d = 8 * u + e;
                            if (d >= R || !mine) continue;
                            const Pair x = pair_of(a.rope, d);
                            float other = bf16_to_f32(src[x.other]), y0, y1;
                            if (weight) other = other * f * bf16_to_f32(weight[x.other]);
                            rope_pair(x.first ? y[e] : other, x.first ? other : y[e], cs[2 * x.at], cs[2 * x.at + 1], y0, y1);
                            y[e] = x.first ? y0 : y1;
                        }
                    };
                    turn(lo, u0);
                    turn(hi, u1);
                }
            } else {
                // 16 numbers of the table either way: dims 16 p .. of a row are pairs 8 p .. of its first half
                float c[16];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    *reinterpret_cast<f32x4 *>(c + 4 * x) = *reinterpret_cast<const f32x4 *>(cs + (turns ? 16 * p + 4 * x : 0));
                if (turns && pos < a.rope.rows) {
                    if constexpr (kRope == kHalf) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) rope_pair(lo[e], hi[e], c[2 * e], c[2 * e + 1], lo[e], hi[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            rope_pair(lo[e], lo[e + 1], c[e], c[e + 1], lo[e], lo[e + 1]);
                            rope_pair(hi[e], hi[e + 1], c[8 + e], c[9 + e], hi[e], hi[e + 1]);
                        }
                    }
                }
            }
        }
        if (!live || nobody) continue;
        if (query) {
            uint16_t *to = a.q_out + t * a.q_stride + (size_t)head * D;
            store8(to + 8 * u0, lo);
            store8(to + 8 * u1, hi);
        } else {
            uint16_t *to = a.c.k + base + head * head_step;
            store8(to + paged_key_at(r0 + row / of, 8 * u0), lo);
            store8(to + paged_key_at(r0 + row / of, 8 * u1), hi);
        }
    }
}

// Units that the new tokens fall into: at most two more a sequence than whole ones.
static uint64_t append_items(const PagedAppendArgs &a) {
    return a.step.starts ? (uint64_t)a.step.tokens / kPagedUnit + 2ull * std::min(a.c.batch, a.step.tokens) : a.c.batch;
}
uint64_t paged_append_groups(const PagedAppendArgs &a) {
    const uint32_t chunk = chunk_heads(a.c.D), rows = 256 / row_threads(a.c.D);
    return 2 * append_items(a) * ((a.c.heads + chunk - 1) / chunk) + (a.q ? ((uint64_t)a.step.tokens * a.q_heads + rows - 1) / rows : 0);
}
hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t s) {
    const dim3 grid((uint32_t)paged_append_groups(a));
    const auto items = (uint32_t)append_items(a);
    const int kind = !a.rope.cos_sin ? kNone : !rope_units_ok(a.rope, a.c.D) ? kAny : a.rope.interleaved ? kNeighbours : kHalf;
    const auto launch = [&](auto d) {
        constexpr uint32_t D = decltype(d)::value;
        switch (kind) {
            case kNone: paged_append_kernel<D, kNone><<<grid, 256, 0, s>>>(a, items); break;
            case kHalf: paged_append_kernel<D, kHalf><<<grid, 256, 0, s>>>(a, items); break;
            case kNeighbours: paged_append_kernel<D, kNeighbours><<<grid, 256, 0, s>>>(a, items); break;
            default: paged_append_kernel<D, kAny><<<grid, 256, 0, s>>>(a, items); break;
        }
    };
    switch (a.c.D) {
        case 64: launch(std::integral_constant<uint32_t, 64>{}); break;
        case 96: launch(std::integral_constant<uint32_t, 96>{}); break;
        case 128: launch(std::integral_constant<uint32_t, 128>{}); break;
        case 192: launch(std::integral_constant<uint32_t, 192>{}); break;
        default: launch(std::integral_constant<uint32_t, 256>{}); break;
    }
    return hipGetLastError();
}

// A thread takes 8 dims of a slot: 16 bytes of its keys, and of its values, whose slots lie together, 8 times 2.  Bound by those, and by
// lines that several of a unit's slots ask for (40000 slots of 2 heads of 128 in bf16 26 us for 82 MB, 3.2 TB/s; 64000 of 8 heads 202 for
// 524; 16 slots 5.1): a way to look at a cache and to move it, which no step takes.
template <class T>
__global__ __launch_bounds__(256) void paged_read_kernel(Paged c, RaggedStep step, const uint32_t *first, uint32_t count, T *k_out,
                                                         T *v_out) {
    const uint32_t units = c.D / 8, b = blockIdx.y;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t u8 = i % units, head = i / units % c.heads;
    const size_t at = i / units / c.heads;
    if (at >= count) return;
    const size_t slot = (first ? first[b] : 0u) + at;
    const bool there = slot < min(step.lengths[b], c.max_ctx);
    const uint32_t u = there ? (uint32_t)slot / kPagedUnit : 0u, r = slot % kPagedUnit, page = there ? page_of(c, b, u) : 0xFFFFFFFFu;
    float k[8] = {}, v[8] = {};
    if (page < c.pages) {
        const size_t from = unit_at(c, page, head, u);
        load8(c.k + from + paged_key_at(r, 8 * u8), k);
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[e] = bf16_to_f32(c.v[from + paged_value_at(r, 8 * u8 + e)]);
    }
    const size_t to = (((size_t)b * count + at) * c.heads + head) * c.D + 8 * u8;
    if (k_out) store8(k_out + to, k);
    if (v_out) store8(v_out + to, v);
}

hipError_t launch_paged_read(const Paged &c, const RaggedStep &step, const uint32_t *first, uint32_t count, void *k_out,
                             void *v_out, int f32, hipStream_t s) {
    const dim3 grid((uint32_t)(((uint64_t)count * c.heads * (c.D / 8) + 255) / 256), c.batch);
    if (f32) paged_read_kernel<float><<<grid, 256, 0, s>>>(c, step, first, count, (float *)k_out, (float *)v_out);
    else paged_read_kernel<uint16_t><<<grid, 256, 0, s>>>(c, step, first, count, (uint16_t *)k_out, (uint16_t *)v_out);
    return hipGetLastError();
}

}  // namespace kr
