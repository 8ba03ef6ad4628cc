// rope.hpp — the rotation of a pair, shared by the kernels that turn q and k.
#pragma once

#include "kr_internal.hpp"

namespace kr {

// (x0 c - x1 s, x0 s + x1 c), the arithmetic of rope_kv_append_kernel.
__device__ __forceinline__ void rope_pair(float x0, float x1, float c, float s, float &y0, float &y1) {
    y0 = fmaf(x0, c, -x1 * s);
    y1 = fmaf(x0, s, x1 * c);
}

// Eight consecutive dims as floats, and back (bf16 rounded to nearest even).
__device__ __forceinline__ void load8(const uint16_t *p, float (&v)[8]) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
    const uint32_t W[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(W[e] << 16);
        v[2 * e + 1] = __uint_as_float(W[e] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
    }
}
__device__ __forceinline__ void store8(uint16_t *p, const float (&v)[8]) {
    const u32x4 w = {pack_bf16_rne(v[0], v[1]), pack_bf16_rne(v[2], v[3]), pack_bf16_rne(v[4], v[5]),
                     pack_bf16_rne(v[6], v[7])};
    *reinterpret_cast<u32x4 *>(p) = w;
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    reinterpret_cast<f32x4 *>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4 *>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
}

// The heads of token t, one workgroup: its threads walk the heads' items.  kUnits: items are the 8-dim units of a head
// (half layout: a unit and its partner half / 8 units on), else single pairs and single passed-through dims.  A thread
// owns both elements of every pair that it turns, so y may be x.
template <class T, bool kUnits>
__device__ __forceinline__ void rope_token(const RopeArgs &a, uint32_t t, const T *xt, T *yt, uint32_t heads,
                                           uint32_t D) {
    const uint32_t R = a.rotary_dim, half = R / 2;
    const uint32_t pos = a.positions[t];
    const bool turn = pos < a.rows, in_place = xt == yt;
    const float *cs = a.cos_sin + (size_t)(turn ? pos : 0) * R;
    const float sign = a.inverse ? -1.0f : 1.0f;
    const uint32_t turned = kUnits ? (a.interleaved ? R / 8 : R / 16) : half;
    const uint32_t passed = in_place ? 0 : (kUnits ? (D - R) / 8 : D - R);
    if (!turn && in_place) return;
    const uint32_t items = turned + passed;
    for (uint32_t w = threadIdx.x; w < heads * items; w += blockDim.x) {
        const uint32_t h = w / items, i = w % items;
        const T *xh = xt + (size_t)h * D;
        T *yh = yt + (size_t)h * D;
        if constexpr (kUnits) {
            if (i >= turned) {
                float v[8];
                load8(xh + R + 8 * (i - turned), v);
                store8(yh + R + 8 * (i - turned), v);
            } else if (a.interleaved) {
                float v[8];
                load8(xh + 8 * i, v);
                if (turn) {
                    float cv[8];
                    load8(cs + 8 * i, cv);
#pragma unroll
                    for (int e = 0; e < 8; e += 2) rope_pair(v[e], v[e + 1], cv[e], sign * cv[e + 1], v[e], v[e + 1]);
                }
                store8(yh + 8 * i, v);
            } else {
                float lo[8], hi[8];
                load8(xh + 8 * i, lo);
                load8(xh + half + 8 * i, hi);
                if (turn) {
                    float cv[8], cw[8];
                    load8(cs + 16 * i, cv);
                    load8(cs + 16 * i + 8, cw);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float c = e < 4 ? cv[2 * e] : cw[2 * e - 8], s = e < 4 ? cv[2 * e + 1] : cw[2 * e - 7];
                        rope_pair(lo[e], hi[e], c, sign * s, lo[e], hi[e]);
                    }
                }
                store8(yh + 8 * i, lo);
                store8(yh + half + 8 * i, hi);
            }
        } else {
            if (i >= turned) {
                yh[R + i - turned] = xh[R + i - turned];
                continue;
            }
            const uint32_t d0 = a.interleaved ? 2 * i : i, d1 = a.interleaved ? 2 * i + 1 : i + half;
            const T a0 = xh[d0], a1 = xh[d1];
            if (!turn) {
                yh[d0] = a0;
                yh[d1] = a1;
                continue;
            }
            float y0, y1;
            if constexpr (sizeof(T) == 2) {
                rope_pair(bf16_to_f32(a0), bf16_to_f32(a1), cs[2 * i], sign * cs[2 * i + 1], y0, y1);
                yh[d0] = (T)(pack_bf16_rne(y0, y0) & 0xFFFFu);
                yh[d1] = (T)(pack_bf16_rne(y1, y1) & 0xFFFFu);
            } else {
                rope_pair(a0, a1, cs[2 * i], sign * cs[2 * i + 1], y0, y1);
                yh[d0] = y0;
                yh[d1] = y1;
            }
        }
    }
}

// Dims 8 u .. 8 u + 7 of a head turned by its table row cs [R / 2, 2] (R even): `x` the head's dims.  Pairs may lie
// anywhere, so the partners are read one by one where R / 2 is no multiple of 8.
__device__ __forceinline__ void rope_unit(const uint16_t *x, uint32_t u, const float *cs, uint32_t R, int interleaved,
                                          float (&v)[8]) {
    load8(x + 8 * u, v);
    if (8 * u >= R) return;
    const uint32_t half = R / 2;
    if (interleaved) {
#pragma unroll
        for (uint32_t e = 0; e < 8; e += 2) {
            const uint32_t i = 4 * u + e / 2;
            if (i < half) {
                const float c = cs[2 * i], s = cs[2 * i + 1];
                rope_pair(v[e], v[e + 1], c, s, v[e], v[e + 1]);
            }
        }
        return;
    }
    if (half % 8 == 0) {
        const bool low = 8 * u < half;
        float o[8];
        load8(x + (low ? 8 * u + half : 8 * u - half), o);
        const uint32_t i = low ? 8 * u : 8 * u - half;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            const float c = cs[2 * (i + e)], s = cs[2 * (i + e) + 1];
            float y0, y1;
            rope_pair(low ? v[e] : o[e], low ? o[e] : v[e], c, s, y0, y1);
            v[e] = low ? y0 : y1;
        }
        return;
    }
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) {
        const uint32_t d = 8 * u + e;
        if (d < R) {
            const bool low = d < half;
            const uint32_t i = low ? d : d - half;
            const float o = bf16_to_f32(x[low ? d + half : d - half]), c = cs[2 * i], s = cs[2 * i + 1];
            float y0, y1;
            rope_pair(low ? v[e] : o, low ? o : v[e], c, s, y0, y1);
            v[e] = low ? y0 : y1;
        }
    }
}

}  // namespace kr
