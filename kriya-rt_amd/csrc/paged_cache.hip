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

constexpr uint32_t kRows = kPagedUnit, kMaxDim = 256;

}  // namespace

// Workgroups: (unit, kv head, keys or values), then (token, 16 query heads).  Each stages its up to 16 rows in LDS.  Keys and queries:
// as f32, with the rows' sums of squares, then every thread normalises and turns 8 dims of a row, whatever the pairing, and
// rounds them once.  Values: as they are, then every thread collects the 8 slots of a dim that lie together.  16-byte pieces whose
// slots are not all new are written slot by slot: the others hold older tokens.
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, uint32_t items) {
    __shared__ __align__(16) float xs[kRows][kMaxDim];
    __shared__ float squares[kRows][kMaxDim / 8];
    const uint32_t D = a.c.D, units = D / 8;
    const uint32_t kv_groups = items * a.c.heads * 2;
    const uint16_t *src, *weight;
    size_t stride;             // between rows
    uint32_t rows, t0, t_step; // row i is of token t0 + i t_step
    uint32_t r0 = 0;           // slot of row 0 in its unit
    uint16_t *dst;
    bool values = false, query = blockIdx.x >= kv_groups;
    if (query) {
        const uint32_t chunks = (a.q_heads + kRows - 1) / kRows, i = blockIdx.x - kv_groups, h0 = i % chunks * kRows;
        t0 = i / chunks;
        t_step = 0;
        if (a.step.starts && (t0 < a.step.starts[0] || t0 >= a.step.starts[a.c.batch])) return;  // nobody's row
        src = a.q + t0 * a.q_stride + (size_t)h0 * D;
        dst = a.q_out + t0 * a.q_stride + (size_t)h0 * D;
        stride = D;
        rows = min(kRows, a.q_heads - h0);
        weight = a.q_norm;
    } else {
        values = blockIdx.x & 1;
        const uint32_t head = blockIdx.x / 2 % a.c.heads;
        uint32_t b, item;
        if (!find_item(blockIdx.x / 2 / a.c.heads, a.c.batch, [&](uint32_t i) { return unit_span(a, i).items; }, b, item)) return;
        const UnitSpan s = unit_span(a, b);
        const uint32_t u = s.first + item, page = page_of(a.c, b, u);
        if (page >= a.c.pages) return;
        const uint32_t from = max(s.n0, u * kPagedUnit), to = min(s.end, (u + 1) * kPagedUnit);
        r0 = from % kPagedUnit;
        rows = to - from;
        t0 = s.s.t0 + (from + s.s.m - s.s.n);
        t_step = 1;
        stride = a.kv_stride;
        src = (values ? a.v : a.k) + t0 * a.kv_stride + (size_t)head * D;
        dst = (values ? a.c.v : a.c.k) + unit_at(a.c, page, head, u);
        weight = a.k_norm;
    }
    if (values) {
        uint16_t *vs = reinterpret_cast<uint16_t *>(&xs[0][0]);
        for (uint32_t i = threadIdx.x; i < rows * units; i += 256) {
            const uint32_t r = i / units, c = i % units;
            *reinterpret_cast<u32x4 *>(vs + (r0 + r) * D + 8 * c) = *reinterpret_cast<const u32x4 *>(src + r * stride + 8 * c);
        }
        __syncthreads();
        // piece i: dims i / 64 32 + i % 32, half h = i / 32 % 2: slots 4 h + j and 8 + 4 h + j
        for (uint32_t i = threadIdx.x; i < 2 * D; i += 256) {
            const uint32_t h = i / 32 % 2, d = i / 64 * 32 + i % 32;
            uint16_t e[8];
            bool all = true;
#pragma unroll
            for (uint32_t x = 0; x < 8; ++x) {
                const uint32_t r = x / 4 * 8 + 4 * h + x % 4;
                const bool fresh = r - r0 < rows;
                all = all && fresh;
                e[x] = vs[r * D + d];
                if (!fresh) e[x] = 0;
            }
            uint16_t *to = dst + 8 * i;
            if (all) {
                *reinterpret_cast<u32x4 *>(to) = u32x4{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16,
                                                       e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16};
            } else {
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x)
                    if (x / 4 * 8 + 4 * h + x % 4 - r0 < rows) to[x] = e[x];
            }
        }
        return;
    }
    const bool turn = a.rope.cos_sin != nullptr;
    if (!turn && !weight) {  // as they are
        for (uint32_t i = threadIdx.x; i < rows * units; i += 256) {
            const uint32_t r = i / units, c = i % units;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(src + r * stride + 8 * c);
            *reinterpret_cast<u32x4 *>(query ? dst + r * stride + 8 * c : dst + paged_key_at(r0 + r, 8 * c)) = v;
        }
        return;
    }
    for (uint32_t i = threadIdx.x; i < rows * units; i += 256) {
        const uint32_t r = i / units, c = i % units;
        float v[8], sum = 0.0f;
        load8(src + r * stride + 8 * c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
        store8(&xs[r][8 * c], v);
        squares[r][c] = sum;
    }
    __syncthreads();
    const uint32_t R = turn ? a.rope.rotary_dim : 0u, half = R / 2;
    for (uint32_t i = threadIdx.x; i < rows * units; i += 256) {
        const uint32_t r = i / units, c = i % units;
        float f = 1.0f;
        if (weight) {
            float sum = 0.0f;
            for (uint32_t x = 0; x < units; ++x) sum += squares[r][x];
            f = rsqrtf(sum / (float)D + a.eps);
        }
        const auto at = [&](uint32_t d) {
            const float x = xs[r][d];
            return weight ? x * f * bf16_to_f32(weight[d]) : x;
        };
        const uint32_t pos = turn ? a.rope.positions[t0 + r * t_step] : 0u;
        const float *cs = pos < a.rope.rows ? a.rope.cos_sin + (size_t)pos * R : nullptr;
        float y[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const uint32_t d = 8 * c + e;
            y[e] = at(d);
            if (cs && d < R) {
                const bool low = a.rope.interleaved ? d % 2 == 0 : d < half;
                const uint32_t p = a.rope.interleaved ? d / 2 : (low ? d : d - half);
                const float other = at(a.rope.interleaved ? d ^ 1 : (low ? d + half : d - half));
                float y0, y1;
                rope_pair(low ? y[e] : other, low ? other : y[e], cs[2 * p], cs[2 * p + 1], y0, y1);
                y[e] = low ? y0 : y1;
            }
        }
        store8(query ? dst + r * stride + 8 * c : dst + paged_key_at(r0 + r, 8 * c), y);
    }
}

// Units that the new tokens fall into: at most two more a sequence than whole ones.
static uint64_t append_items(const PagedAppendArgs &a) {
    return a.step.starts ? (uint64_t)a.step.tokens / kPagedUnit + 2ull * std::min(a.c.batch, a.step.tokens) : a.c.batch;
}
uint64_t paged_append_groups(const PagedAppendArgs &a) {
    const uint64_t chunks = a.q ? (a.q_heads + kRows - 1) / kRows : 0;
    return append_items(a) * a.c.heads * 2 + a.step.tokens * chunks;
}
hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t s) {
    paged_append_kernel<<<dim3((uint32_t)paged_append_groups(a)), 256, 0, s>>>(a, (uint32_t)append_items(a));
    return hipGetLastError();
}

// A thread takes 8 dims of a slot.
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
