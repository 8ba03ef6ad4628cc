// ragged.hpp — the sequences of a ragged step on the device, and the item of them that a workgroup takes.
#pragma once

#include "kr_internal.hpp"

namespace kr {

struct Span {
    uint32_t t0, m;   // its new tokens: rows t0 .. t0 + m - 1
    uint32_t n;       // its tokens, the new ones included
};
// `starts` and `lengths` come from device memory: rows are cut to the step's tokens.
__device__ __forceinline__ Span span_of(const RaggedStep &s, uint32_t b) {
    Span r;
    r.n = s.lengths[b];
    if (!s.starts) {
        r.t0 = b;
        r.m = 1;
    } else {
        r.t0 = min(s.starts[b], s.tokens);
        r.m = min(max(s.starts[b + 1], r.t0), s.tokens) - r.t0;
    }
    return r;
}

// Sums over the lanes by DPP (a shuffle through LDS takes several times as long, and every workgroup starts with these):
// lane l gets lanes 0 .. l, the last lane all.
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);   // row_shr 1, 2, 4, 8: zeros come in
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // lane 15 of a row to the next one
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // lane 31 to the upper half
    return v;
}
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(v), 63);
}
// (each lane's value below 2^52, so that 24-bit pieces of 64 of them stay within a word)
__device__ __forceinline__ unsigned long long wave_sum_u64(unsigned long long v) {
    return wave_sum_u32((uint32_t)v & 0xFFFFFFu) + ((unsigned long long)wave_sum_u32((uint32_t)(v >> 24) & 0xFFFFFFu) << 24) +
           ((unsigned long long)wave_sum_u32((uint32_t)(v >> 48)) << 48);
}

// The item-th of the items of sequence b that idx falls to, where sequence b has count(b) items; false past the last.
// Wave-uniform: every wave finds it for itself, 64 sequences a step.
template <class F>
__device__ __forceinline__ bool find_item(uint32_t idx, uint32_t batch, F &&count, uint32_t &b, uint32_t &item) {
    const uint32_t lane = __lane_id();
    for (uint32_t base = 0; base < batch; base += 64) {
        const uint32_t c = base + lane < batch ? count(base + lane) : 0u;
        const uint32_t sum = wave_scan_u32(c), total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        if (idx < total) {
            const uint32_t l = (uint32_t)__builtin_ctzll(__ballot(sum > idx));
            b = base + l;
            item = idx - (uint32_t)__builtin_amdgcn_readlane((int)(sum - c), (int)l);
            return true;
        }
        idx -= total;
    }
    return false;
}

}  // namespace kr
