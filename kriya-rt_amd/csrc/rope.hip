// rope.hip — rotary positions in general form: tables of (cos, sin) for stretched contexts, and the rotation of
// whole or partial heads in either pairing.
//
// Reference semantics (RoPE table and rotation, whole heads, pairs of halves):
//   crates/kriya-backend-metal/src/encoder.rs:1940-1950
//   kernels/metal/paged_gqa_and_deltanet.metal:115-222
#include <math.h>

#include "rope.hpp"

namespace kr {

// The angle of position p at f turns a position is p f turns, of which only the fraction counts.  p f is taken in 64
// bits (an error of 2^-53 p f turns: 1e-11 at a million), the fraction by rint; its sine and cosine are 64 bits too, so a table holds
// the f32 nearest to them.  Bound by its launch: 3907 rows of 16 pairs 2.2 us.
__global__ __launch_bounds__(256) void rope_table_kernel(RopeTurns f, uint32_t half, uint32_t first, uint32_t count,
                                                         double gain, float *cos_sin) {
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t r = (uint32_t)(at / half), i = (uint32_t)(at % half);
    if (r >= count) return;
    const double turns = ((double)first + (double)r) * f.turns[i];
    double s, c;
    sincospi(2.0 * (turns - rint(turns)), &s, &c);
    reinterpret_cast<float2 *>(cos_sin)[at] = make_float2((float)(gain * c), (float)(gain * s));
}

hipError_t launch_rope_table(const RopeTurns &f, uint32_t half, uint32_t first, uint32_t count, double gain,
                             float *cos_sin, hipStream_t s) {
    const uint64_t blocks = ((uint64_t)count * half + 255) / 256;
    rope_table_kernel<<<dim3((uint32_t)blocks), 256, 0, s>>>(f, half, first, count, gain, cos_sin);
    return hipGetLastError();
}

// A workgroup a token: its table row is loaded once for all heads.  Bound by bytes where there are many: 3907 tokens of 16 heads of
// 128 in f32, a quarter turned, 64 MB in 13.6 us (4.7 TB/s); 16 tokens of 18 heads 3 us, a launch and two dependent loads.
template <class T, bool kUnits>
__global__ __launch_bounds__(256) void rope_apply_kernel(RopeArgs a, const T *x, size_t xs, T *y, size_t ys,
                                                         uint32_t heads, uint32_t D) {
    rope_token<T, kUnits>(a, blockIdx.x, x + blockIdx.x * xs, y + blockIdx.x * ys, heads, D);
}

template <class T>
static hipError_t launch_rope_apply_t(const RopeArgs &a, const T *x, size_t xs, T *y, size_t ys, uint32_t tokens,
                                      uint32_t heads, uint32_t D, hipStream_t s) {
    const size_t unit = 16 / sizeof(T);  // elements of a 16-byte piece
    const bool units = rope_units_ok(a, D) && (uintptr_t)x % 16 == 0 && (uintptr_t)y % 16 == 0 && xs % unit == 0 &&
                       ys % unit == 0;
    const uint32_t items = heads * (units ? D / 8 : D);
    const uint32_t threads = items >= 256 ? 256 : (items + 63) / 64 * 64;
    if (units)
        rope_apply_kernel<T, true><<<tokens, threads, 0, s>>>(a, x, xs, y, ys, heads, D);
    else
        rope_apply_kernel<T, false><<<tokens, threads, 0, s>>>(a, x, xs, y, ys, heads, D);
    return hipGetLastError();
}

hipError_t launch_rope_apply(const RopeArgs &a, const void *x, size_t xs, void *y, size_t ys, int f32, uint32_t tokens,
                             uint32_t heads, uint32_t D, hipStream_t s) {
    if (f32) return launch_rope_apply_t(a, (const float *)x, xs, (float *)y, ys, tokens, heads, D, s);
    return launch_rope_apply_t(a, (const uint16_t *)x, xs, (uint16_t *)y, ys, tokens, heads, D, s);
}

}  // namespace kr
