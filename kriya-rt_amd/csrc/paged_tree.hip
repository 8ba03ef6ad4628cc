// paged_tree.hip — trees of drafted tokens: their plan (ancestor masks and positions) and the commit of an accepted path.
//
// Reference semantics (tree verification by masks, greedy acceptance):
//   kernels/metal/paged_gqa_and_deltanet.metal:1536-1620, crates/kriya-speculate/src/eagle_medusa.rs:186-717
#include "paged.hpp"

namespace kr {

namespace {

constexpr int32_t kNone = -1;

// Node i's parent: a node before it, or none.
__device__ __forceinline__ int32_t parent_of(const int32_t *parents, uint32_t i) {
    const int32_t p = parents[i];
    return p >= 0 && (uint32_t)p < i ? p : kNone;
}

// lane l: the largest of lanes 0 .. l
__device__ __forceinline__ uint32_t wave_scan_max(uint32_t v) {
    const uint32_t lane = __lane_id();
#pragma unroll
    for (uint32_t x = 1; x < 64; x *= 2) {
        const uint32_t o = __shfl_up(v, x);
        if (lane >= x) v = max(v, o);
    }
    return v;
}

}  // namespace

// A workgroup a sequence, a thread a node.  A node's ancestors are found from it upwards, in order of falling place, so its
// words are complete one after the other and written once.  Nodes whose parent is the node before them form runs: a run's bits are
// set at once, so that a chain (a prompt given as a tree) takes a few steps and not its length.
// Bound by latency: one tree of 24 nodes 2.8 us, 64 of up to some hundred 6.1.
__global__ __launch_bounds__(256) void tree_plan_kernel(const int32_t *parents, RaggedStep step, uint32_t words, uint32_t *mask,
                                                        uint32_t *positions) {
    __shared__ int32_t par[kTreeNodes];
    __shared__ uint16_t run[kTreeNodes];  // where a node's run begins
    const Span s = span_of(step, blockIdx.x);
    const uint32_t known = min(s.m, 32 * words), old = s.n > s.m ? s.n - s.m : 0u;
    for (uint32_t i = threadIdx.x; i < known; i += 256) par[i] = parent_of(parents + s.t0, i);
    __syncthreads();
    if (threadIdx.x < 64) {
        uint32_t carry = 0;
        for (uint32_t i0 = 0; i0 < known; i0 += 64) {
            const uint32_t i = i0 + threadIdx.x;
            const bool begins = i < known && (i == 0 || par[i] != (int32_t)i - 1);
            const uint32_t v = max(wave_scan_max(begins ? i : 0u), carry);
            if (i < known) run[i] = (uint16_t)v;
            carry = __shfl(v, 63);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < s.m; i += 256) {
        uint32_t *row = mask + (size_t)(s.t0 + i) * words;
        uint32_t depth = 1;
        if (i < known) {
            depth = 0;
            uint32_t at = words, bits = 0;  // words from `at` on are written; bits: of word at - 1
            const auto down_to = [&](uint32_t w) {  // makes word w the next one to be written
                while (at > w + 1) {
                    row[--at] = bits;
                    bits = 0;
                }
            };
            for (int32_t hi = (int32_t)i; hi >= 0;) {
                const uint32_t lo = run[hi];
                depth += (uint32_t)hi - lo + 1;
                down_to((uint32_t)hi / 32);
                for (;;) {
                    const uint32_t w = at - 1, from = lo > 32 * w ? lo - 32 * w : 0u, to = min((uint32_t)hi - 32 * w, 31u);
                    bits |= (0xFFFFFFFFu >> (31 - to)) & (0xFFFFFFFFu << from);
                    if (lo >= 32 * w) break;
                    down_to(w - 1);
                }
                hi = par[lo];
            }
            while (at > 0) {
                row[--at] = bits;
                bits = 0;
            }
        } else {
            for (uint32_t w = 0; w < words; ++w) row[w] = 0;
        }
        positions[s.t0 + i] = old + depth - 1;
    }
}

hipError_t launch_tree_plan(const int32_t *parents, const RaggedStep &step, uint32_t words, uint32_t *mask, uint32_t *positions,
                            hipStream_t s) {
    tree_plan_kernel<<<dim3(step.batch), 256, 0, s>>>(parents, step, words, mask, positions);
    return hipGetLastError();
}

// Workgroup (layer, sequence).  Each finds the path for itself (a few hundred bytes from the L2; a launch of its own would cost more
// than the walks), the first layer's writes it out.  A node is the next one of the path if its parent is the last one and its token the
// choice there: for every node that is looked up at once, and the walk then searches LDS.  A thread moves columns, 8 dims of a head's
// keys or one dim of its values, over the nodes that change places, 64 of the path at a time: path[i] >= i and rising, so the rows of
// later nodes are never where an earlier one goes, and within eight nodes all are loaded before one is stored.  No thread touches
// another's column.
// Bound by latency (lengths; nodes; the walk, a step of LDS a node; pages; rows) and by lines: a slot's values are 2 of each 16 bytes.
// 4 sequences, 36 layers of 2 heads of 128: 6 us; 48 of about 60 nodes, 24 layers of 8 heads of 64: 13.7 for 14 MB (512 threads, of
// which a compute unit holds four workgroups, 14.0; 640 16.3).  One lookup a node and LDS walks took it from 160.
constexpr uint32_t kCommitThreads = 320, kNoNode = 0xFFFFu;
__global__ __launch_bounds__(kCommitThreads) void paged_commit_kernel(PagedCommitArgs a) {
    __shared__ uint16_t follows[kTreeNodes], path[kTreeNodes];
    __shared__ uint32_t found, moved;
    __shared__ uint32_t from_page[64], to_page[64], from_slot[64], to_slot[64];  // places in a page
    const uint32_t b = blockIdx.y, lane = threadIdx.x & 63, D = a.c.D;
    const Span s = span_of(a.step, b);
    const uint32_t m = min(s.m, kTreeNodes), old = s.n > s.m ? s.n - s.m : 0u;
    for (uint32_t i = threadIdx.x; i < m; i += kCommitThreads) {
        const int32_t p = parent_of(a.parents + s.t0, i);
        follows[i] = (uint16_t)(p >= 0 && a.drafted[s.t0 + i] == a.targets[s.t0 + (uint32_t)max(p, 0)] ? (uint32_t)p : kNoNode);
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        uint32_t at = 0, n = 0;
        if (m) {
            if (lane == 0) path[0] = 0;
            n = 1;
            while (n < a.max_path) {
                uint32_t next = kNoNode;
                for (uint32_t i0 = (at + 1) & ~63u; i0 < m; i0 += 64) {
                    const unsigned long long hit = __ballot(i0 + lane < m && follows[i0 + lane] == at);
                    if (hit) {
                        next = i0 + (uint32_t)__builtin_ctzll(hit);
                        break;
                    }
                }
                if (next == kNoNode) break;
                if (lane == 0) path[n] = (uint16_t)next;
                ++n;
                at = next;
            }
        }
        if (lane == 0) found = n;
        if (blockIdx.x == 0 && lane == 0) {
            a.counts[b] = n;
            a.new_lengths[b] = m ? (s.n + n > s.m ? s.n + n - s.m : 0u) : s.n;
            if (m) a.next[b] = a.targets[s.t0 + at];
        }
    }
    __syncthreads();
    const uint32_t n = found;
    if (blockIdx.x == 0)
        for (uint32_t i = threadIdx.x; i < a.max_path; i += kCommitThreads) a.path[(size_t)b * a.max_path + i] = i < n ? path[i] : 0u;
    if (s.n < s.m) return;  // (a length that was cut off: its nodes have no slots)
    const size_t page_size = (size_t)a.c.heads * (kPagedUnit << a.c.shift) * D, layer = (size_t)blockIdx.x * a.c.pages * page_size;
    const uint32_t slots = kPagedUnit << a.c.shift, key_columns = a.c.heads * (D / 8), columns = key_columns + a.c.heads * D;
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        if (threadIdx.x < 64) {
            const uint32_t i = i0 + lane, node = i < n ? path[i] : i, from = old + node, to = old + i;
            uint32_t pf = 0, pt = 0;
            bool moves = node != i && from < a.c.max_ctx;  // (to < from)
            if (moves) {
                pf = page_of(a.c, b, from / kPagedUnit);
                pt = page_of(a.c, b, to / kPagedUnit);
                moves = pf < a.c.pages && pt < a.c.pages;
            }
            const unsigned long long all = __ballot(moves);
            if (moves) {
                const uint32_t x = (uint32_t)__popcll(all & ((1ull << lane) - 1));
                from_page[x] = pf;
                to_page[x] = pt;
                from_slot[x] = from & (slots - 1);
                to_slot[x] = to & (slots - 1);
            }
            if (lane == 0) moved = (uint32_t)__popcll(all);
        }
        __syncthreads();
        const uint32_t count = moved;
        for (uint32_t c = threadIdx.x; c < columns; c += kCommitThreads) {
            const bool values = c >= key_columns;
            const uint32_t x = values ? c - key_columns : c, per = values ? D : D / 8, head = x / per, d = values ? x % per : x % per * 8;
            const size_t column = layer + (size_t)head * slots * D;
            const auto place = [&](uint32_t page, uint32_t slot) {
                const uint32_t r = slot % kPagedUnit;
                return column + page * page_size + (size_t)(slot / kPagedUnit) * (kPagedUnit * D) + (values ? paged_value_at(r, d) : paged_key_at(r, d));
            };
            for (uint32_t k = 0; k < count; k += 8) {
                // (past the last one: the last one again, which is not stored)
                if (values) {
                    uint16_t v[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) v[i] = a.c.v[place(from_page[min(k + i, count - 1)], from_slot[min(k + i, count - 1)])];
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        if (k + i < count) a.c.v[place(to_page[k + i], to_slot[k + i])] = v[i];
                } else {
                    u32x4 v[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        v[i] = *reinterpret_cast<const u32x4 *>(a.c.k + place(from_page[min(k + i, count - 1)], from_slot[min(k + i, count - 1)]));
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i)
                        if (k + i < count) *reinterpret_cast<u32x4 *>(a.c.k + place(to_page[k + i], to_slot[k + i])) = v[i];
                }
            }
        }
        __syncthreads();
    }
}

hipError_t launch_paged_commit(const PagedCommitArgs &a, hipStream_t s) {
    paged_commit_kernel<<<dim3(a.layers, a.c.batch), kCommitThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace kr
