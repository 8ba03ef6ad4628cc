// kv8_cache.hip — the 8-bit key/value cache: appending (with the rotation), reading back, and eviction.
//
// Reference semantics of the append (rotation, order, contiguous slots; its cache is bf16):
//   kernels/metal/paged_gqa_and_deltanet.metal:115-222
#include <algorithm>

#include "kv8.hpp"
#include "rope.hpp"

namespace kr {

namespace {

// A block is coded by two sides of 64 or 128 threads, keys and values.  A thread holds groups of 4 slots x 8 dims: group i is
// slots 4 (i / (D / 8)) .. + 3, dims 8 (i % (D / 8)) .. + 7; D > 128 makes two groups a thread.
__host__ __device__ constexpr uint32_t side_threads(uint32_t D) { return D <= 64 ? 64 : 128; }

struct GroupAt {
    uint32_t g, u;  // 4 g: first slot; 8 u: first dim
};
__device__ __forceinline__ GroupAt group_at(uint32_t i, uint32_t units) { return GroupAt{i / units, i % units}; }

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// max |x| of the block over the waves of a side, as bits: magnitudes order as integers, and an infinity or NaN comes out on
// top.  All threads of the workgroup call it.
__device__ __forceinline__ float side_amax(uint32_t bits, uint32_t (&red)[4], uint32_t per_side) {
    bits = wave_max_u32(bits);
    const uint32_t w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[w] = bits;
    __syncthreads();
    return __uint_as_float(per_side == 64 ? red[w] : max(red[w & 2], red[(w & 2) + 1]));
}

// The codes of a group into the block's bytes in LDS, in the cache's order (straight to memory the values' words would be
// spread 16 bytes apart: 64 lines an instruction).
template <int E4M3, bool kPlain>
__device__ __forceinline__ void put_codes(uint8_t *blk, bool values, GroupAt at, const float (&x)[4][8], const Kv8Coder &c) {
    if (values) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint32_t *>(blk + kv8_value_at(at.g, 8 * at.u + e)) =
                kv8_codes<E4M3, kPlain>(c, x[0][e], x[1][e], x[2][e], x[3][e]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x2 w = {kv8_codes<E4M3, kPlain>(c, x[j][0], x[j][1], x[j][2], x[j][3]),
                             kv8_codes<E4M3, kPlain>(c, x[j][4], x[j][5], x[j][6], x[j][7])};
            *reinterpret_cast<u32x2 *>(blk + kv8_key_at(4 * at.g + j, 8 * at.u)) = w;
        }
    }
}

// The blocks that sequence b's new tokens fall into: `first` .. `last` (slots n0 .. end - 1 are new).
struct AppendSpan {
    Span s;
    uint32_t n0, end, first, last, items;
};
__device__ __forceinline__ AppendSpan append_span(const Kv8AppendArgs &a, uint32_t b) {
    AppendSpan r;
    r.s = span_of(a.step, b);
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

// Workgroups 0 .. items * heads - 1: one block each (keys by the first side of threads, values by the second), then one for
// every token's q.  A block that already holds tokens is coded again from its raw rows (at most 32 rows; all of a
// decoded token's traffic is 24 KB a head, well under a microsecond of HBM), so its codes are those of the whole
// block coded at once.  Bound by latency at one token a sequence: all rows are loaded in one round (from clamped addresses, what
// does not count is zeroed after), with rotation after a round for positions and one for the table.
// kRope: 0 none, 1 in 8-dim units, 2 any rotary_dim.  16 tokens of 2 heads of 128, rotated, with 16 heads of q: 6.7 us; 3907 of 8
// heads of 64 in five sequences, not rotated: 8.5 us.
template <int E4M3, int kGroups, int kRope>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8AppendArgs a, uint32_t items) {
    __shared__ uint32_t red[4];
    __shared__ __align__(16) uint8_t codes[2][kKv8Block * 128 * kGroups];
    const uint32_t D = a.c.D, units = D / 8, per_side = blockDim.x / 2;
    if (blockIdx.x >= items * a.c.heads) {
        if constexpr (kRope != 0) {
            const uint32_t t = blockIdx.x - items * a.c.heads;
            if (a.step.starts && (t < a.step.starts[0] || t >= a.step.starts[a.c.batch])) return;  // nobody's row
            rope_token<uint16_t, kRope == 1>(a.rope, t, a.q + t * a.q_stride, a.q_out + t * a.q_stride, a.q_heads, D);
        }
        return;
    }
    const uint32_t head = blockIdx.x % a.c.heads;
    uint32_t b, item;
    if (!find_item(blockIdx.x / a.c.heads, a.c.batch, [&](uint32_t i) { return append_span(a, i).items; }, b, item)) return;
    const AppendSpan s = append_span(a, b);
    const bool values = __builtin_amdgcn_readfirstlane(threadIdx.x >= per_side);
    const uint32_t tid = values ? threadIdx.x - per_side : threadIdx.x;
    const size_t bh = (size_t)b * a.c.heads + head;
    uint16_t *open = (values ? a.c.vo : a.c.ko) + bh * kKv8Block * D;
    const uint16_t *fresh = (values ? a.v : a.k) + (size_t)head * D;
    for (uint32_t blk = s.first + item;; blk = s.last) {
        float x[kGroups][4][8];
        uint32_t top = 0;
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
            const GroupAt at = group_at(min(tid + per_side * i, D - 1), units);  // (threads past D repeat the last group)
            const uint16_t *row[4];
            const float *cs[4];
            bool turn[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t slot = min(blk * kKv8Block + 4 * at.g + j, s.end - 1);
                const uint32_t t = s.s.t0 + (max(slot, s.n0) + s.s.m - s.s.n);
                row[j] = slot < s.n0 ? open + (slot % kKv8Block) * D : fresh + t * a.kv_stride;
                if constexpr (kRope != 0) {
                    const uint32_t pos = a.rope.positions[t];
                    turn[j] = !values && slot >= s.n0 && pos < a.rope.rows && 8 * at.u < a.rope.rotary_dim;
                    cs[j] = a.rope.cos_sin + (size_t)(turn[j] ? pos : 0u) * a.rope.rotary_dim;
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) load8(row[j] + 8 * at.u, x[i][j]);
            if constexpr (kRope == 1) {
                const uint32_t half = a.rope.rotary_dim / 2;
                const bool low = 8 * at.u < half;
                const uint32_t turned = 8 * at.u < a.rope.rotary_dim ? at.u : 0u;  // a unit whose pairs are in the table
                if (a.rope.interleaved) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        float c[8];
                        load8(cs[j] + 8 * turned, c);
                        if (turn[j]) {
#pragma unroll
                            for (int e = 0; e < 8; e += 2) rope_pair(x[i][j][e], x[i][j][e + 1], c[e], c[e + 1], x[i][j][e], x[i][j][e + 1]);
                        }
                    }
                } else {
                    const uint32_t other = turned == 0 || low ? turned + half / 8 : turned - half / 8;
                    const uint32_t pair = turned < half / 8 ? turned : turned - half / 8;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        float o[8], c[16];
                        load8(row[j] + 8 * other, o);
                        load8(cs[j] + 16 * pair, *reinterpret_cast<float(*)[8]>(&c[0]));
                        load8(cs[j] + 16 * pair + 8, *reinterpret_cast<float(*)[8]>(&c[8]));
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float y0, y1;
                            rope_pair(low ? x[i][j][e] : o[e], low ? o[e] : x[i][j][e], c[2 * e], c[2 * e + 1], y0, y1);
                            if (turn[j]) x[i][j][e] = low ? y0 : y1;
                        }
                    }
                }
            }
            if constexpr (kRope == 2) {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (turn[j]) rope_unit(row[j], at.u, cs[j], a.rope.rotary_dim, a.rope.interleaved, x[i][j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                if constexpr (kRope != 0) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][j][e] = bf16_to_f32(pack_bf16_rne(x[i][j][e], 0.0f) & 0xFFFFu);
                }
                if (blk * kKv8Block + 4 * at.g + j >= s.end) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][j][e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, abs_bits(x[i][j][e]));
            }
        }
        const float scale = side_amax(top, red, per_side) / kv8_largest(E4M3);
        const Kv8Coder coder = kv8_coder(scale);
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
            if (tid + per_side * i >= D) continue;
            const GroupAt at = group_at(tid + per_side * i, units);
            if (coder.plain) put_codes<E4M3, true>(codes[values], values, at, x[i], coder);
            else put_codes<E4M3, false>(codes[values], values, at, x[i], coder);
            if (blk != s.last) continue;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t slot = blk * kKv8Block + 4 * at.g + j;
                if (slot >= s.n0 && slot < s.end) store8(open + (4 * at.g + j) * D + 8 * at.u, x[i][j]);
            }
        }
        if (tid == 0) (values ? a.c.vs : a.c.ks)[bh * a.c.blocks + blk] = scale;
        __syncthreads();
        u32x4 *bytes = reinterpret_cast<u32x4 *>((values ? a.c.v : a.c.k) + (bh * a.c.blocks + blk) * (size_t)(kKv8Block * D));
        for (uint32_t i = tid; i < kKv8Block * D / 16; i += per_side) bytes[i] = reinterpret_cast<const u32x4 *>(codes[values])[i];
        if (item != 0 || blk == s.last) return;
        __syncthreads();
    }
}

hipError_t launch_kv8_append(const Kv8AppendArgs &a, hipStream_t s) {
    // at most one block a token, and 31 others a full block: the sequences' blocks are counted on the device
    const uint64_t items = a.step.starts ? a.step.tokens / kKv8Block + std::min(a.c.batch, a.step.tokens) : a.c.batch;
    const dim3 grid((uint32_t)(items * a.c.heads) + (a.q ? a.step.tokens : 0));
    const uint32_t threads = 2 * side_threads(a.c.D);
    const auto go = [&](auto rope) {
        constexpr int kRope = decltype(rope)::value;
        const uint32_t n = (uint32_t)items;
        if (a.c.D <= 128) {
            if (a.c.e4m3) kv8_append_kernel<1, 1, kRope><<<grid, threads, 0, s>>>(a, n);
            else kv8_append_kernel<0, 1, kRope><<<grid, threads, 0, s>>>(a, n);
        } else {
            if (a.c.e4m3) kv8_append_kernel<1, 2, kRope><<<grid, threads, 0, s>>>(a, n);
            else kv8_append_kernel<0, 2, kRope><<<grid, threads, 0, s>>>(a, n);
        }
    };
    if (!a.rope.cos_sin) go(std::integral_constant<int, 0>{});
    else if (a.rope_units) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
    return hipGetLastError();
}

// ---- reading back

// A thread takes 4 slots (aligned to the cache's groups of 4) x 8 dims of one head.  Bound by bytes: 8 sequences of 4000 tokens,
// 2 heads of 128, to bf16: 48 MB in 12.4 us (3.9 TB/s).
template <int E4M3, class T>
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
                float y[4];
                kv8_values<E4M3>(v, y);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j][e] = y[j] * scale;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const u32x2 v = *reinterpret_cast<const u32x2 *>(bytes + kv8_key_at(4 * g + j, 8 * u));
                kv8_values<E4M3>(v.x, x[j]);
                kv8_values<E4M3>(v.y, x[j] + 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[j][e] *= scale;
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
    const auto go = [&](auto e4m3, auto *k, auto *v) {
        kv8_dequant_kernel<decltype(e4m3)::value><<<grid, 256, 0, s>>>(c, lengths, first, count, groups, k, v);
    };
    const auto of = [&](auto *k, auto *v) {
        if (c.e4m3) go(std::integral_constant<int, 1>{}, k, v);
        else go(std::integral_constant<int, 0>{}, k, v);
    };
    if (f32) of((float *)k_out, (float *)v_out);
    else of((uint16_t *)k_out, (uint16_t *)v_out);
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
constexpr uint32_t kSelectHeld = 16;    // weights a thread holds in registers: contexts up to 16384
constexpr uint32_t kSelectCopies = 8;   // of the histogram: the lanes of a wave share a few exponents, and take turns at a word

// The slots of a wave: run consecutive ones, 64 an index.
struct SelectRun {
    const float *w;
    uint32_t p0, run, n;
};

// kHeld: run <= 64 kSelectHeld, the weights read once; else from memory (the caches) each time.
template <bool kHeld>
__device__ void select_slots(const Kv8EvictArgs &a, const SelectRun &s, float *to_w, uint32_t *kept,
                             uint32_t (&hist)[256][kSelectCopies + 1], uint32_t (&found)[2], uint32_t (&kept_of)[kSelectWaves],
                             uint32_t (&ties_of)[kSelectWaves]) {
    const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    float held[kSelectHeld];
    const auto slot = [&](uint32_t i) { return s.p0 + 64 * i + lane; };
    const auto hold = [&](uint32_t first) {
#pragma unroll
        for (uint32_t i = 0; i < kSelectHeld; ++i) held[i] = s.w[min(slot(first + i), s.n - 1)];
    };
    if constexpr (kHeld) hold(0);
    // f(slot, weight) for the wave's slots, 64 at a time, all lanes together
    const auto each = [&](auto &&f) {
        for (uint32_t first = 0; first < (kHeld ? 1 : s.run / 64); first += kSelectHeld) {
            if constexpr (!kHeld) hold(first);
#pragma unroll
            for (uint32_t i = 0; i < kSelectHeld; ++i)
                if (64 * (first + i) < s.run) f(slot(first + i), held[i]);
        }
    };
    const uint32_t lo = a.sink, hi = s.n - a.recent;  // sink + recent <= budget < n
    uint32_t want = a.budget - a.sink - a.recent;
    uint32_t prefix = 0, mask = 0;
    const bool any = want > 0;
    if (any) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256 * (kSelectCopies + 1); i += kSelectThreads) (&hist[0][0])[i] = 0;
            __syncthreads();
            each([&](uint32_t p, float w) {
                const uint32_t key = weight_key(w);
                if (p >= lo && p < hi && (key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u][lane % kSelectCopies], 1u);
            });
            __syncthreads();
            if (wave == 0) {  // the digit in which the want-th largest falls: lane l holds digits 4 l .. 4 l + 3
                uint32_t c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[i] = 0;
#pragma unroll
                    for (uint32_t x = 0; x < kSelectCopies; ++x) c[i] += hist[4 * lane + i][x];
                    sum += c[i];
                }
                const uint32_t upto = wave_scan_u32(sum);
                uint32_t above = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63) - upto;  // keys in the digits of the lanes above
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
        }
    }
    // keys above `prefix` stay, and the first `want` that equal it
    const auto sure = [&](uint32_t p, uint32_t key) { return p < s.n && (p < lo || p >= hi || (any && key > prefix)); };
    const auto tie = [&](uint32_t p, uint32_t key) { return p >= lo && p < hi && any && key == prefix; };
    uint32_t sures = 0, ties = 0;
    each([&](uint32_t p, float w) {
        const uint32_t key = weight_key(w);
        sures += (uint32_t)__builtin_popcountll(__ballot(sure(p, key)));
        ties += (uint32_t)__builtin_popcountll(__ballot(tie(p, key)));
    });
    if (lane == 0) {
        kept_of[wave] = sures;
        ties_of[wave] = ties;
    }
    __syncthreads();
    uint32_t at = 0, tied = 0;  // kept and tied ones before this wave
    for (uint32_t i = 0; i < wave; ++i) {
        at += kept_of[i] + min(ties_of[i], want - min(tied, want));
        tied += ties_of[i];
    }
    each([&](uint32_t p, float w) {
        const uint32_t key = weight_key(w);
        const uint64_t below = (1ull << lane) - 1, tm = __ballot(tie(p, key));
        const bool keep = sure(p, key) || (tie(p, key) && tied + (uint32_t)__builtin_popcountll(tm & below) < want);
        tied += (uint32_t)__builtin_popcountll(tm);
        const uint64_t km = __ballot(keep);
        if (keep) {
            const uint32_t i = at + (uint32_t)__builtin_popcountll(km & below);
            kept[i] = p;
            to_w[i] = w;
        }
        at += (uint32_t)__builtin_popcountll(km);
    });
}

}  // namespace

// A workgroup per (sequence, head): the kept slots in order.  Of the middle (slots sink .. n - recent - 1) the `want`
// largest keys: the smallest of them is found eight bits a pass by histograms, ties are taken from the lowest
// slot.  Then every wave counts its run of slots, and writes the kept ones behind those of the waves before it.
// Bound by latency (four passes with three barriers each): 16 workgroups of up to 8100 slots 12.5 us.
__global__ __launch_bounds__(kSelectThreads) void kv8_select_kernel(Kv8EvictArgs a) {
    __shared__ uint32_t hist[256][kSelectCopies + 1];  // (one word more: the digits' first words in different banks)
    __shared__ uint32_t found[2];                      // the digit, and how many keys of larger digits
    __shared__ uint32_t kept_of[kSelectWaves], ties_of[kSelectWaves];
    const uint32_t head = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
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
    const uint32_t run = (n + kSelectThreads - 1) / kSelectThreads * 64;
    const SelectRun s{w, (tid >> 6) * run, run, n};
    if (run <= 64 * kSelectHeld) select_slots<true>(a, s, to_w, kept, hist, found, kept_of, ties_of);
    else select_slots<false>(a, s, to_w, kept, hist, found, kept_of, ties_of);
}

// A workgroup per new block: keys by the first side of threads, 16 dims of a slot each (the kept slots of 32 lanes lie side by side
// but for the gaps), values by the second, a dim each with all 32 slots: its bytes lie 16 apart in the old blocks, so a wave's loads
// of one slot cover whole lines.  Both sides' new bytes are 16-byte units.  The slots behind the new length are given code 0.
// Where the kept slots come from a few old blocks (four: every other token kept needs two or three), a thread loads its dim's
// bytes of those whole, 16 a load, and picks from them in LDS; else byte by byte.  8 sequences of 8100 cut to 4000, 2 heads, D 128:
// 25 -> 22 us, of which the bytes (every old line holds some that stay: 50 MB) take 10 at a copy's rate.
constexpr uint32_t kGatherSpan = 4;  // old blocks that go through LDS (16 or 32 KB)
template <int E4M3, int kGroups>
__global__ __launch_bounds__(256) void kv8_gather_kernel(Kv8EvictArgs a) {
    __shared__ uint32_t red[4];
    __shared__ uint32_t from[kKv8Block];
    constexpr uint32_t kDims = 128 * kGroups;
    __shared__ u32x4 units[kGatherSpan][2][kDims];  // [old block][h][dim]
    const uint32_t blk = blockIdx.x, head = blockIdx.y, b = blockIdx.z, D = a.from.D, per_side = blockDim.x / 2;
    const uint32_t n = min(a.lengths[b], a.from.max_ctx), left = min(n, a.budget);
    const uint32_t base = blk * kKv8Block;
    if (base >= left) return;
    const size_t bh = (size_t)b * a.from.heads + head;
    const uint32_t mine = min(left - base, kKv8Block), last = (left - 1) / kKv8Block, old_last = (n - 1) / kKv8Block;
    const bool values = __builtin_amdgcn_readfirstlane(threadIdx.x >= per_side), fits = n <= a.budget;
    const uint32_t tid = values ? threadIdx.x - per_side : threadIdx.x;
    if (threadIdx.x < kKv8Block) from[threadIdx.x] = a.kept[bh * a.budget + base + min(threadIdx.x, mine - 1)];
    __syncthreads();
    const size_t block_bytes = (size_t)kKv8Block * D;
    const uint8_t *src = (values ? a.from.v : a.from.k) + bh * a.from.blocks * block_bytes;
    uint8_t *dst = (values ? a.to.v : a.to.k) + (bh * a.to.blocks + blk) * block_bytes;
    const float *ss = (values ? a.from.vs : a.from.ks) + bh * a.from.blocks;
    float *ds = (values ? a.to.vs : a.to.ks) + bh * a.to.blocks + blk;
    const uint16_t *open = (values ? a.from.vo : a.from.ko) + bh * block_bytes;
    uint16_t *to_open = (values ? a.to.vo : a.to.ko) + bh * block_bytes;
    if (fits || (blk != last && from[kKv8Block - 1] == base + kKv8Block - 1)) {  // in their places: slots only move down
        for (uint32_t i = tid; i < block_bytes / 16; i += per_side)
            reinterpret_cast<u32x4 *>(dst)[i] = reinterpret_cast<const u32x4 *>(src + blk * block_bytes)[i];
        if (blk == last)
            for (uint32_t i = tid; i < block_bytes / 8; i += per_side)
                reinterpret_cast<u32x4 *>(to_open)[i] = reinterpret_cast<const u32x4 *>(open)[i];
        if (tid == 0) *ds = ss[blk];
        return;
    }
    // 32 elements a thread and group: x[i][r] is slot r of dim tid (values), x[i][16 j + e] slot tid % 32 of dim 16 c + e (keys)
    const uint32_t mine_r = tid % kKv8Block, mine_p = from[mine_r], mine_b = mine_p / kKv8Block;  // lane r: slot r comes from here
    const float mine_scale = ss[mine_b];
    const uint32_t first_b = __builtin_amdgcn_readfirstlane(from[0] / kKv8Block), last_b = __builtin_amdgcn_readfirstlane(from[mine - 1] / kKv8Block);
    const auto chunk_at = [&](uint32_t i, uint32_t j) { return tid / kKv8Block + per_side / kKv8Block * (2 * i + j); };  // c
    float x[kGroups][32];
    uint32_t top = 0;
    const bool raw_rows = from[mine - 1] / kKv8Block == old_last;  // the block takes some of the old last block's
#pragma unroll
    for (uint32_t i = 0; i < kGroups; ++i) {
        const uint32_t d = min(tid + per_side * i, D - 1);  // (threads past D repeat the last)
        if (values && last_b - first_b < kGatherSpan) {
            // the dim's bytes of the old blocks, and those of the kept slots out of LDS (each thread reads what it wrote)
            u32x4 w[kGatherSpan][2];
#pragma unroll
            for (uint32_t q = 0; q < kGatherSpan; ++q)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
                    w[q][h] = *reinterpret_cast<const u32x4 *>(src + min(first_b + q, last_b) * block_bytes + kv8_value_at(h, d));
#pragma unroll
            for (uint32_t q = 0; q < kGatherSpan; ++q)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) units[q][h][tid + per_side * i] = w[q][h];
            const uint32_t g = mine_p % kKv8Block / 4;
            const uint32_t at = ((mine_b - first_b) * 2 + (g & 1)) * (kDims * 16) + kv8_value_at(g & ~1u, 0) + mine_p % 4;
            const uint8_t *bytes = reinterpret_cast<const uint8_t *>(&units[0][0][tid + per_side * i]);
#pragma unroll
            for (uint32_t r = 0; r < kKv8Block; ++r) {
                const float scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine_scale), r));
                x[i][r] = kv8_value<E4M3>(bytes[__builtin_amdgcn_readlane(at, r)]) * scale;
            }
        } else if (values) {
            const uint64_t at = mine_b * block_bytes + kv8_value_at(mine_p % kKv8Block / 4, 0) + mine_p % 4;
#pragma unroll
            for (uint32_t r = 0; r < kKv8Block; ++r) {
                // the slot is the whole wave's: its part of the address and its scale go through scalar registers
                const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)at, r), hi = __builtin_amdgcn_readlane((uint32_t)(at >> 32), r);
                const uint8_t *slot = src + ((uint64_t)hi << 32 | lo);
                const float scale = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine_scale), r));
                x[i][r] = kv8_value<E4M3>(slot[kv8_value_at(0, d)]) * scale;
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                const uint32_t c = min(chunk_at(i, j), D / 16 - 1);
                const u32x4 v = *reinterpret_cast<const u32x4 *>(src + mine_b * block_bytes + kv8_key_at(mine_p % kKv8Block, 16 * c));
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) kv8_values<E4M3>(v[y], &x[i][16 * j + 4 * y]);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[i][16 * j + e] *= mine_scale;
            }
        }
        if (raw_rows || blk == last) {
#pragma unroll
            for (uint32_t y = 0; y < 32; ++y) {
                const uint32_t r = values ? y : mine_r, c = chunk_at(i, y / 16), p = from[r];
                const uint32_t dim = values ? d : 16 * min(c, D / 16 - 1) + y % 16;
                if (p / kKv8Block == old_last) x[i][y] = bf16_to_f32(open[(p % kKv8Block) * D + dim]);
                if (blk == last) {
                    const uint32_t bits = pack_bf16_rne(x[i][y], 0.0f) & 0xFFFFu;
                    x[i][y] = bf16_to_f32(bits);
                    if (r < mine && (values ? tid + per_side * i < D : c < D / 16)) to_open[r * D + dim] = (uint16_t)bits;
                }
            }
        }
        if (mine < kKv8Block) {
#pragma unroll
            for (uint32_t y = 0; y < 32; ++y) x[i][y] = (values ? y : mine_r) < mine ? x[i][y] : 0.0f;
        }
#pragma unroll
        for (uint32_t y = 0; y < 32; ++y) top = max(top, abs_bits(x[i][y]));
    }
    const float scale = side_amax(top, red, per_side) / kv8_largest(E4M3);
    const Kv8Coder coder = kv8_coder(scale);
    const auto put = [&](auto plain) {
#pragma unroll
        for (uint32_t i = 0; i < kGroups; ++i) {
            const uint32_t d = tid + per_side * i;
            if (values) {
                if (d >= D) continue;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    u32x4 w;
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) {  // slots 16 s + 8 a + 4 h + j, y = 2 a + s
                        const uint32_t r = 16 * (y & 1) + 8 * (y >> 1) + 4 * h;
                        w[y] = kv8_codes<E4M3, decltype(plain)::value>(coder, x[i][r], x[i][r + 1], x[i][r + 2], x[i][r + 3]);
                    }
                    *reinterpret_cast<u32x4 *>(dst + kv8_value_at(h, d)) = w;
                }
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    const uint32_t c = chunk_at(i, j);
                    if (c >= D / 16) continue;
                    u32x4 w;
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) {
                        const float *v = &x[i][16 * j + 4 * y];
                        w[y] = kv8_codes<E4M3, decltype(plain)::value>(coder, v[0], v[1], v[2], v[3]);
                    }
                    *reinterpret_cast<u32x4 *>(dst + kv8_key_at(mine_r, 16 * c)) = w;
                }
            }
        }
    };
    if (coder.plain) put(std::true_type{});
    else put(std::false_type{});
    if (tid == 0) *ds = scale;
}

hipError_t launch_kv8_evict(const Kv8EvictArgs &a, hipStream_t s) {
    kv8_select_kernel<<<dim3(a.from.heads, a.from.batch), kSelectThreads, 0, s>>>(a);
    if (hipError_t e = hipGetLastError()) return e;
    const uint32_t blocks = (a.budget + kKv8Block - 1) / kKv8Block;
    const dim3 grid(blocks, a.from.heads, a.from.batch);
    const uint32_t threads = 2 * side_threads(a.from.D);
    if (a.from.D <= 128) {
        if (a.from.e4m3) kv8_gather_kernel<1, 1><<<grid, threads, 0, s>>>(a);
        else kv8_gather_kernel<0, 1><<<grid, threads, 0, s>>>(a);
    } else {
        if (a.from.e4m3) kv8_gather_kernel<1, 2><<<grid, threads, 0, s>>>(a);
        else kv8_gather_kernel<0, 2><<<grid, threads, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace kr
