// kv8_cache.hip — the 8-bit key/value cache: appending (with the rotation), reading back, and eviction.
//
// Reference semantics of the append (rotation, order, contiguous slots; its cache is bf16):
//   kernels/metal/paged_gqa_and_deltanet.metal:115-222
#include <algorithm>

#include "kv8.hpp"
#include "rope.hpp"

namespace kr {

namespace {

// Codes a block from 32 x D values held as groups of 4 slots x 8 dims: group i of 128 threads is slots 4 (i / (D/8)) ..
// + 3, dims 8 (i % (D/8)) .. + 7.  D <= 256: at most two groups a thread.
constexpr uint32_t kGroups = 2;

struct GroupAt {
    uint32_t g, u;  // 4 g: first slot; 8 u: first dim
};
__device__ __forceinline__ GroupAt group_at(uint32_t i, uint32_t units) { return GroupAt{i / units, i % units}; }

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// max |x| of the block over the 128 threads of a side (0 keys, 1 values), as bits: magnitudes order as integers, and
// an infinity or NaN comes out on top.  All 256 threads call it.
__device__ __forceinline__ float side_amax(uint32_t bits, uint32_t (&red)[4]) {
    bits = wave_max_u32(bits);
    const uint32_t w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[w] = bits;
    __syncthreads();
    return __uint_as_float(max(red[w & 2], red[(w & 2) + 1]));
}

__device__ __forceinline__ void store_codes(uint8_t *blk, bool values, GroupAt at, const float (&x)[4][8], float scale,
                                            int e4m3) {
    uint32_t code[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) code[j][e] = kv8_code(x[j][e], scale, e4m3);
    if (values) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint32_t *>(blk + kv8_value_at(at.g, 8 * at.u + e)) =
                code[0][e] | code[1][e] << 8 | code[2][e] << 16 | code[3][e] << 24;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x2 w = {code[j][0] | code[j][1] << 8 | code[j][2] << 16 | code[j][3] << 24,
                             code[j][4] | code[j][5] << 8 | code[j][6] << 16 | code[j][7] << 24};
            *reinterpret_cast<u32x2 *>(blk + kv8_key_at(4 * at.g + j, 8 * at.u)) = w;
        }
    }
}

// The blocks that sequence b's new tokens fall into: `first` .. `last` (slots n0 .. end - 1 are new).
struct AppendSpan {
    Kv8Span s;
    uint32_t n0, end, first, last, items;
};
__device__ __forceinline__ AppendSpan append_span(const Kv8AppendArgs &a, uint32_t b) {
    AppendSpan r;
    r.s = kv8_span(a.step, b);
    r.n0 = r.s.n > r.s.m ? r.s.n - r.s.m : 0u;
    r.end = min(r.s.n, a.c.max_ctx);
    r.items = 0;
    if (r.end > r.n0) {
        r.first = r.n0 / kKv8Block;
        r.last = (r.end - 1) / kKv8Block;
        // the first block reads the raw rows that the last one replaces: one workgroup takes both, in that order
        r.items = max(r.last - r.first, 1u);
    }
    return r;
}

}  // namespace

// Workgroups 0 .. items * heads - 1: one block each (keys by threads 0 .. 127, values by the others), then one for
// every token's q.  A block that already holds tokens is coded again from its raw rows (at most 32 rows; all of a
// decoded token's traffic is 24 KB a head, well under a microsecond of HBM), so its codes are those of the whole
// block coded at once.  Bound by latency at one token a sequence: one round of loads, one reduction, one of stores.
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a, uint32_t items) {
    __shared__ uint32_t red[4];
    const uint32_t D = a.c.D, units = D / 8;
    if (blockIdx.x >= items * a.c.heads) {
        const uint32_t t = blockIdx.x - items * a.c.heads;
        const uint16_t *src = a.q + t * a.q_stride;
        uint16_t *dst = a.q_out + t * a.q_stride;
        if (a.rope_units)
            rope_token<uint16_t, true>(a.rope, t, src, dst, a.q_heads, D);
        else
            rope_token<uint16_t, false>(a.rope, t, src, dst, a.q_heads, D);
        return;
    }
    const uint32_t head = blockIdx.x % a.c.heads;
    uint32_t b, item;
    if (!kv8_find(blockIdx.x / a.c.heads, a.c.batch, [&](uint32_t i) { return append_span(a, i).items; }, b, item)) return;
    const AppendSpan s = append_span(a, b);
    const bool values = threadIdx.x >= 128;
    const uint32_t tid = threadIdx.x & 127;
    const size_t bh = (size_t)b * a.c.heads + head;
    uint16_t *open = (values ? a.c.vo : a.c.ko) + bh * kKv8Block * D;
    const uint16_t *fresh = (values ? a.v : a.k) + (size_t)head * D;
    for (uint32_t blk = s.first + item;; blk = s.last) {
        float x[kGroups][4][8];
        uint32_t top = 0;
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
            if (tid + 128 * i >= D) continue;
            const GroupAt at = group_at(tid + 128 * i, units);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t slot = blk * kKv8Block + 4 * at.g + j;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][j][e] = 0.0f;
                if (slot >= s.end) continue;
                if (slot < s.n0) {
                    load8(open + (4 * at.g + j) * D + 8 * at.u, x[i][j]);
                } else {
                    const uint32_t t = s.s.t0 + (slot + s.s.m - s.s.n);
                    const uint16_t *row = fresh + t * a.kv_stride;
                    const uint32_t pos = values || !a.rope.cos_sin ? 0xFFFFFFFFu : a.rope.positions[t];
                    if (!values && a.rope.cos_sin && pos < a.rope.rows) {
                        rope_unit(row, at.u, a.rope.cos_sin + (size_t)pos * a.rope.rotary_dim, a.rope.rotary_dim,
                                  a.rope.interleaved, x[i][j]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[i][j][e] = bf16_to_f32(pack_bf16_rne(x[i][j][e], 0.0f) & 0xFFFFu);
                    } else {
                        load8(row + 8 * at.u, x[i][j]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[i][j][e]));
            }
        }
        const float scale = side_amax(top, red) / kv8_largest(a.c.e4m3);
        uint8_t *bytes = (values ? a.c.v : a.c.k) + (bh * a.c.blocks + blk) * (size_t)(kKv8Block * D);
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
            if (tid + 128 * i >= D) continue;
            const GroupAt at = group_at(tid + 128 * i, units);
            store_codes(bytes, values, at, x[i], scale, a.c.e4m3);
            if (blk != s.last) continue;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t slot = blk * kKv8Block + 4 * at.g + j;
                if (slot >= s.n0 && slot < s.end) store8(open + (4 * at.g + j) * D + 8 * at.u, x[i][j]);
            }
        }
        if (tid == 0) (values ? a.c.vs : a.c.ks)[bh * a.c.blocks + blk] = scale;
        if (item != 0 || blk == s.last) return;
    }
}

hipError_t launch_kv8_append(const Kv8AppendArgs &a, hipStream_t s) {
    // at most one block a token, and 31 others a full block: the sequences' blocks are counted on the device
    const uint64_t items = a.step.starts ? a.step.tokens / kKv8Block + std::min(a.c.batch, a.step.tokens) : a.c.batch;
    const uint32_t q_blocks = a.q ? a.step.tokens : 0;
    kv8_append_kernel<<<dim3((uint32_t)(items * a.c.heads) + q_blocks), 256, 0, s>>>(a, (uint32_t)items);
    return hipGetLastError();
}

// ---- reading back

// A thread takes 4 slots (aligned to the cache's groups of 4) x 8 dims of one head.
template <class T>
__global__ __launch_bounds__(256) void kv8_dequant_kernel(Kv8 c, const uint32_t *lengths, const uint32_t *first,
                                                          uint32_t count, uint32_t groups, T *k_out, T *v_out) {
    const uint32_t units = c.D / 8, b = blockIdx.z;
    const uint32_t w = blockIdx.x * 256 + threadIdx.x;
    const uint32_t u = w % units, h = w / units % c.heads, gi = w / units / c.heads;
    if (gi >= groups) return;
    const uint32_t f = first ? first[b] : 0u;
    const uint32_t n = min(lengths[b], c.max_ctx);
    const bool values = blockIdx.y == 1;
    T *out = values ? v_out : k_out;
    if (!out) return;
    const uint64_t slot0 = ((uint64_t)(f / 4) + gi) * 4;
    float x[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = 0.0f;
    if (slot0 < n) {
        const uint32_t blk = (uint32_t)(slot0 / kKv8Block), g = (uint32_t)(slot0 % kKv8Block) / 4;
        const size_t at = ((size_t)b * c.heads + h) * c.blocks + blk;
        const uint8_t *bytes = (values ? c.v : c.k) + at * (kKv8Block * c.D);
        const float scale = (values ? c.vs : c.ks)[at];
        if (values) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t v = *reinterpret_cast<const uint32_t *>(bytes + kv8_value_at(g, 8 * u + e));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j][e] = kv8_value(v, j, c.e4m3) * scale;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u32x2 v = *reinterpret_cast<const u32x2 *>(bytes + kv8_key_at(4 * g + j, 8 * u));
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] = kv8_value(e < 4 ? v.x : v.y, e & 3, c.e4m3) * scale;
            }
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        const uint64_t slot = slot0 + j;
        if (slot < f || slot - f >= count) continue;
        if (slot >= n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[j][e] = 0.0f;
        }
        store8(out + (((size_t)b * count + (slot - f)) * c.heads + h) * c.D + 8 * u, x[j]);
    }
}

hipError_t launch_kv8_dequant(const Kv8 &c, const uint32_t *lengths, const uint32_t *first, uint32_t count, void *k_out,
                              void *v_out, int f32, hipStream_t s) {
    const uint32_t groups = (count + 3) / 4 + (first ? 1 : 0);
    const uint64_t threads = (uint64_t)groups * c.heads * (c.D / 8);
    const dim3 grid((uint32_t)((threads + 255) / 256), 2, c.batch);
    if (f32)
        kv8_dequant_kernel<float><<<grid, 256, 0, s>>>(c, lengths, first, count, groups, (float *)k_out, (float *)v_out);
    else
        kv8_dequant_kernel<uint16_t><<<grid, 256, 0, s>>>(c, lengths, first, count, groups, (uint16_t *)k_out,
                                                          (uint16_t *)v_out);
    return hipGetLastError();
}

// ---- eviction

namespace {

// A weight as an unsigned number of the same order: -0 as 0, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

}  // namespace

// A workgroup per (sequence, head): the kept slots in order.  Of the middle (slots sink .. n - recent - 1) the `want`
// largest keys: the smallest of them is found eight bits a pass by histograms, ties are taken from the lowest
// slot.  Then every wave counts its run of slots, and writes the kept ones behind those of the waves before it.
__global__ __launch_bounds__(kSelectThreads) void kv8_select_kernel(Kv8EvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t found[2];                          // the digit, and how many keys of larger digits
    __shared__ uint32_t kept_of[kSelectWaves], ties_of[kSelectWaves];
    const uint32_t head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const size_t bh = (size_t)b * a.from.heads + head;
    const float *w = a.weight + bh * a.from.max_ctx;
    float *to_w = a.to_weight + bh * a.to.max_ctx;
    uint32_t *kept = a.kept + bh * a.budget;
    const uint32_t n = min(a.lengths[b], a.from.max_ctx);
    if (a.to_lengths && head == 0 && tid == 0) a.to_lengths[b] = min(n, a.budget);
    if (n <= a.budget) {
        for (uint32_t p = tid; p < n; p += kSelectThreads) {
            kept[p] = p;
            to_w[p] = w[p];
        }
        return;
    }
    const uint32_t lo = a.sink, hi = n - a.recent;  // sink + recent <= budget < n
    uint32_t want = a.budget - a.sink - a.recent;
    uint32_t prefix = 0, mask = 0;
    if (want) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (uint32_t p = lo + tid; p < hi; p += kSelectThreads) {
                const uint32_t key = weight_key(w[p]);
                if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (wave == 0) {  // the digit in which the want-th largest falls: lane l holds digits 4 l .. 4 l + 3
                uint32_t c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += c[i] = hist[4 * lane + i];
                uint32_t above = sum;  // keys in this lane's digits and those of the lanes above
#pragma unroll
                for (uint32_t o = 1; o < 64; o *= 2) {
                    const uint32_t down = __shfl_down(above, o);
                    if (lane + o < 64) above += down;
                }
                above -= sum;
                if (above < want && above + sum >= want) {
#pragma unroll
                    for (int i = 3; i >= 0; --i) {
                        if (above < want && above + c[i] >= want) {
                            found[0] = 4 * lane + i;
                            found[1] = above;
                        }
                        above += c[i];
                    }
                }
            }
            __syncthreads();
            want -= found[1];
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            __syncthreads();
        }
    }
    // keys above `prefix` stay, and the first `want` that equal it
    const bool any = a.budget > a.sink + a.recent;
    const uint32_t run = (n + kSelectThreads - 1) / kSelectThreads * 64;  // slots of a wave
    const uint32_t p0 = wave * run, p1 = min(p0 + run, n);
    uint32_t sure = 0, ties = 0;
    for (uint32_t p = p0 + lane; p < p0 + run; p += 64) {
        bool s = false, t = false;
        if (p < p1) {
            const uint32_t key = any ? weight_key(w[p]) : 0u;
            const bool middle = p >= lo && p < hi;
            s = !middle || (any && key > prefix);
            t = middle && any && key == prefix;
        }
        sure += (uint32_t)__builtin_popcountll(__ballot(s));
        ties += (uint32_t)__builtin_popcountll(__ballot(t));
    }
    if (lane == 0) {
        kept_of[wave] = sure;
        ties_of[wave] = ties;
    }
    __syncthreads();
    uint32_t at = 0, tied = 0;  // kept and tied ones before this wave
    for (uint32_t i = 0; i < wave; ++i) {
        at += kept_of[i] + min(ties_of[i], want - min(tied, want));
        tied += ties_of[i];
    }
    for (uint32_t p = p0 + lane; p < p0 + run; p += 64) {
        bool s = false, t = false;
        float wp = 0.0f;
        if (p < p1) {
            wp = w[p];
            const uint32_t key = any ? weight_key(wp) : 0u;
            const bool middle = p >= lo && p < hi;
            s = !middle || (any && key > prefix);
            t = middle && any && key == prefix;
        }
        const uint64_t tm = __ballot(t), below = (1ull << lane) - 1;
        t = t && tied + (uint32_t)__builtin_popcountll(tm & below) < want;
        tied += (uint32_t)__builtin_popcountll(tm);
        const uint64_t km = __ballot(s || t);
        if (s || t) {
            const uint32_t i = at + (uint32_t)__builtin_popcountll(km & below);
            kept[i] = p;
            to_w[i] = wp;
        }
        at += (uint32_t)__builtin_popcountll(km);
    }
}

// A workgroup per new block: keys by threads 0 .. 127, values by the others, as in the append.  The slots behind the
// new length are given code 0.
__global__ __launch_bounds__(256) void kv8_gather_kernel(Kv8EvictArgs a) {
    __shared__ uint32_t red[4];
    __shared__ uint32_t from[kKv8Block];
    const uint32_t blk = blockIdx.x, head = blockIdx.y, b = blockIdx.z, D = a.from.D, units = D / 8;
    const uint32_t n = min(a.lengths[b], a.from.max_ctx), left = min(n, a.budget);
    const uint32_t base = blk * kKv8Block;
    if (base >= left) return;
    const size_t bh = (size_t)b * a.from.heads + head;
    const uint32_t mine = min(left - base, kKv8Block), last = (left - 1) / kKv8Block, old_last = (n - 1) / kKv8Block;
    const bool values = threadIdx.x >= 128, fits = n <= a.budget;
    const uint32_t tid = threadIdx.x & 127;
    if (threadIdx.x < kKv8Block) from[threadIdx.x] = threadIdx.x < mine ? a.kept[bh * a.budget + base + threadIdx.x] : 0u;
    __syncthreads();
    const size_t block_bytes = (size_t)kKv8Block * D;
    const uint8_t *src = (values ? a.from.v : a.from.k) + bh * a.from.blocks * block_bytes;
    uint8_t *dst = (values ? a.to.v : a.to.k) + (bh * a.to.blocks + blk) * block_bytes;
    const float *ss = (values ? a.from.vs : a.from.ks) + bh * a.from.blocks;
    float *ds = (values ? a.to.vs : a.to.ks) + bh * a.to.blocks + blk;
    const uint16_t *open = (values ? a.from.vo : a.from.ko) + bh * block_bytes;
    uint16_t *to_open = (values ? a.to.vo : a.to.ko) + bh * block_bytes;
    if (fits || (blk != last && from[kKv8Block - 1] == base + kKv8Block - 1)) {  // in their places: slots only move down
        for (uint32_t i = tid; i < block_bytes / 16; i += 128)
            reinterpret_cast<u32x4 *>(dst)[i] = reinterpret_cast<const u32x4 *>(src + blk * block_bytes)[i];
        if (blk == last)
            for (uint32_t i = tid; i < block_bytes / 8; i += 128)
                reinterpret_cast<u32x4 *>(to_open)[i] = reinterpret_cast<const u32x4 *>(open)[i];
        if (tid == 0) *ds = ss[blk];
        return;
    }
    float x[kGroups][4][8];
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < kGroups; ++i) {
        if (tid + 128 * i >= D) continue;
        const GroupAt at = group_at(tid + 128 * i, units);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t r = 4 * at.g + j;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][j][e] = 0.0f;
            if (r >= mine) continue;
            const uint32_t p = from[r], pb = p / kKv8Block, pr = p % kKv8Block;
            if (pb == old_last) {
                load8(open + pr * D + 8 * at.u, x[i][j]);
            } else {
                const uint8_t *bytes = src + pb * block_bytes;
                const float scale = ss[pb];
                if (values) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[i][j][e] = kv8_value(bytes[kv8_value_at(pr / 4, 8 * at.u + e) + pr % 4], 0, a.from.e4m3) * scale;
                } else {
                    const u32x2 v = *reinterpret_cast<const u32x2 *>(bytes + kv8_key_at(pr, 8 * at.u));
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][j][e] = kv8_value(e < 4 ? v.x : v.y, e & 3, a.from.e4m3) * scale;
                }
            }
            if (blk == last) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][j][e] = bf16_to_f32(pack_bf16_rne(x[i][j][e], 0.0f) & 0xFFFFu);
                store8(to_open + r * D + 8 * at.u, x[i][j]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[i][j][e]));
        }
    }
    const float scale = side_amax(top, red) / kv8_largest(a.from.e4m3);
#pragma unroll
    for (uint32_t i = 0; i < kGroups; ++i) {
        if (tid + 128 * i >= D) continue;
        store_codes(dst, values, group_at(tid + 128 * i, units), x[i], scale, a.from.e4m3);
    }
    if (tid == 0) *ds = scale;
}

hipError_t launch_kv8_evict(const Kv8EvictArgs &a, hipStream_t s) {
    kv8_select_kernel<<<dim3(a.from.heads, a.from.batch), kSelectThreads, 0, s>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    const uint32_t blocks = (a.budget + kKv8Block - 1) / kKv8Block;
    kv8_gather_kernel<<<dim3(blocks, a.from.heads, a.from.batch), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace kr
