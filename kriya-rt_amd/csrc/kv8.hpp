// kv8.hpp — the 8-bit key/value cache on the device: where the bytes of a block lie, its codes, and the sequences of
// a ragged step.
//
// A block is 32 slots of one sequence and kv head, D dims.  Its bytes stand as the matrix instructions want them:
//   keys    byte of (slot r, dim d) at (d / 16) 512 + 16 r + d % 16: a lane's 16 bytes are 16 dims of one slot, the
//           lanes of a load side by side (an instruction reads whole cache lines and no lane moves a byte);
//   values  byte of (slot r = 16 s + 8 a + 4 h + j, dim d) at (d / 32) 1024 + 512 h + 16 (d % 32) + 8 a + 4 s + j:
//           a lane's 16 bytes are the 16 slots whose probabilities the same lane already holds after the first
//           product (a C fragment's rows 8 i + 4 h + j), so the probabilities never leave their registers.
#pragma once

#include "kr_internal.hpp"

namespace kr {

__host__ __device__ constexpr uint32_t kv8_key_at(uint32_t r, uint32_t d) { return d / 16 * 512 + 16 * r + d % 16; }
// the four slots 4 g .. 4 g + 3 of dim d, g = r / 4
__host__ __device__ constexpr uint32_t kv8_value_at(uint32_t g, uint32_t d) {
    return d / 32 * 1024 + 512 * (g & 1) + 16 * (d % 32) + 8 * ((g >> 1) & 1) + 4 * (g >> 2);
}

// ---- codes
__host__ __device__ constexpr float kv8_largest(int e4m3) { return e4m3 ? 448.0f : 127.0f; }

// Four bytes to four halves (lo: bytes 0 and 1), exact.  int8: byte ^ 0x80 under the pattern of 1024.0 (ulp 1), less
// 1152; three instructions a pair.  e4m3: one conversion a pair.
template <int E4M3>
__device__ __forceinline__ void kv8_halves(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (E4M3) {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
    } else {
        const uint32_t u = w ^ 0x80808080u;
        const f16x2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const f16x2_t a = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
        const f16x2_t b = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
        lo = __builtin_bit_cast(uint32_t, a);
        hi = __builtin_bit_cast(uint32_t, b);
    }
}
// Eight bytes to a matrix operand.
template <int E4M3>
__device__ __forceinline__ f16x8_t kv8_operand(uint32_t w0, uint32_t w1) {
    u32x4 o;
    uint32_t a, b;
    kv8_halves<E4M3>(w0, a, b);
    o.x = a;
    o.y = b;
    kv8_halves<E4M3>(w1, a, b);
    o.z = a;
    o.w = b;
    return __builtin_bit_cast(f16x8_t, o);
}

// The value of byte j of w.
__device__ __forceinline__ float kv8_value(uint32_t w, int j, int e4m3) {
    if (!e4m3) return (float)(int8_t)(w >> (8 * j));
    const int b = (int)((w >> (8 * j)) & 0xFFu);
    return __builtin_amdgcn_cvt_f32_fp8(b, 0);
}

// The code byte of x in a block of this scale.  The quotient is IEEE (a tie between two codes is the definition's); it
// is at most M up to rounding, and NaN only where the scale is infinite or NaN, which is stored as code 0 (times
// that scale: NaN).
__device__ __forceinline__ uint32_t kv8_code(float x, float scale, int e4m3) {
    const float m = kv8_largest(e4m3);
    float q = scale > 0.0f ? x / scale : 0.0f;
    q = q == q ? fminf(fmaxf(q, -m), m) : 0.0f;
    if (e4m3) return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, 0.0f, 0, false) & 0xFFu;
    return (uint32_t)(int)rintf(q) & 0xFFu;
}

// ---- the sequences of a step
struct Kv8Span {
    uint32_t t0, m;   // its new tokens: rows t0 .. t0 + m - 1
    uint32_t n;       // its tokens, the new ones included
};
// `starts` and `lengths` come from device memory: rows are cut to the step's tokens.
__device__ __forceinline__ Kv8Span kv8_span(const Kv8Step &s, uint32_t b) {
    Kv8Span r;
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

// The item-th of the items of sequence b that idx falls to, where sequence b has count(b) items; false past the last.
// Wave-uniform: every wave finds it for itself, 64 sequences a step.
template <class F>
__device__ __forceinline__ bool kv8_find(uint32_t idx, uint32_t batch, F &&count, uint32_t &b, uint32_t &item) {
    const uint32_t lane = __lane_id();
    for (uint32_t base = 0; base < batch; base += 64) {
        const uint32_t c = base + lane < batch ? count(base + lane) : 0u;
        uint32_t sum = c;
#pragma unroll
        for (uint32_t o = 1; o < 64; o *= 2) {
            const uint32_t up = __shfl_up(sum, o);
            if (lane >= o) sum += up;
        }
        const uint32_t total = __builtin_amdgcn_readlane(sum, 63);
        if (idx < total) {
            const uint32_t l = (uint32_t)__builtin_ctzll(__ballot(sum > idx));
            b = base + l;
            item = idx - __builtin_amdgcn_readlane(sum - c, l);
            return true;
        }
        idx -= total;
    }
    return false;
}

}  // namespace kr
