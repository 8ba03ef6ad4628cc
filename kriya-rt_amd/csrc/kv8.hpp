// kv8.hpp — the 8-bit key/value cache on the device: where the bytes of a block lie, and its codes.
//
// A block is 32 slots of one sequence and kv head, D dims.  Its bytes stand as the matrix instructions want them:
//   keys    byte of (slot r, dim d) at (d / 16) 512 + 16 r + d % 16: a lane's 16 bytes are 16 dims of one slot, the
//           lanes of a load side by side (an instruction reads whole cache lines and no lane moves a byte);
//   values  byte of (slot r = 16 s + 8 a + 4 h + j, dim d) at (d / 32) 1024 + 512 h + 16 (d % 32) + 8 a + 4 s + j:
//           a lane's 16 bytes are the 16 slots whose probabilities the same lane already holds after the first
//           product (a C fragment's rows 8 i + 4 h + j), so the probabilities never leave their registers.
#pragma once

#include "kr_internal.hpp"
#include "ragged.hpp"

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

// The values of the four bytes of w, and of one byte.
template <int E4M3>
__device__ __forceinline__ void kv8_values(uint32_t w, float *v) {
    if constexpr (E4M3) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v[0] = lo[0];
        v[1] = lo[1];
        v[2] = hi[0];
        v[3] = hi[1];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)(int8_t)(w >> (8 * j));
    }
}
template <int E4M3>
__device__ __forceinline__ float kv8_value(uint8_t b) {
    if constexpr (E4M3) return __builtin_amdgcn_cvt_f32_fp8((int)b, 0);
    return (float)(int8_t)b;
}

// Codes of a block.  A code is the rounding of the IEEE quotient x / scale, so that ties are the definition's.  With y the rounded
// reciprocal of the scale and q = x y, one step q + (x - q scale) y, the bracket exact in a fused multiply-add, is that
// quotient (Markstein's theorem) as long as nothing underflows: three instructions instead of a division's ten; scales
// outside 2^-70 .. 2^100 (a block of zeros, one that stands for NaN) take the division.
struct Kv8Coder {
    float scale, inv;
    bool plain;  // in a scalar register (else the compiler takes both ways and selects: 500 instructions more for 32 codes)
};
// scale: the same in all lanes
__device__ __forceinline__ Kv8Coder kv8_coder(float scale) {
    return Kv8Coder{scale, 1.0f / scale, __builtin_amdgcn_readfirstlane(scale >= 0x1p-70f && scale <= 0x1p100f) != 0};
}
// Four codes in a word.  The quotients are at most M up to rounding, NaN only where the scale is infinite or NaN, which
// is stored as code 0 (times that scale: NaN).
template <int E4M3, bool kPlain>
__device__ __forceinline__ uint32_t kv8_codes(const Kv8Coder &c, float x0, float x1, float x2, float x3) {
    float x[4] = {x0, x1, x2, x3};
    if constexpr (kPlain) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float q = x[j] * c.inv;
            x[j] = fmaf(fmaf(-q, c.scale, x[j]), c.inv, q);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float m = kv8_largest(E4M3), q = c.scale > 0.0f ? x[j] / c.scale : 0.0f;
            x[j] = q == q ? fminf(fmaxf(q, -m), m) : 0.0f;
        }
    }
    if constexpr (E4M3) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
        return (uint32_t)w;
    } else {
        uint32_t u[4];  // 1.5 * 2^23 added: rounded to even, the low byte is the code
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __float_as_uint(x[j] + 12582912.0f);
        const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000C0Cu);
        return lo | hi;
    }
}

}  // namespace kr
