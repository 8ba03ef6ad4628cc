// api_checks.hpp — checks that the entry points of the caches share.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "kriya_kv8.h"
#include "kr_internal.hpp"

namespace kr {

// A launch has fewer than 2^32 threads in a dimension: this many workgroups of 256.
constexpr uint64_t kMostGroups = 0xFFFFFFFFull / 256;

inline bool on(const void *p, size_t a) { return (uintptr_t)p % a == 0; }

// Memory of a call: what one argument points to, `bytes` of it, or of each of `rows` rows, `stride` bytes from one to the next.
struct Range {
    const char *name;
    const void *at;
    size_t bytes, rows = 1, stride = 0;
    size_t whole() const { return (rows - 1) * stride + bytes; }
};
// Whether any byte is in both.
inline bool meet(const Range &x, const Range &y) {
    const auto a = (uintptr_t)x.at, b = (uintptr_t)y.at;
    if (!x.at || !y.at || !x.bytes || !y.bytes || !x.rows || !y.rows || a >= b + y.whole() || b >= a + x.whole()) return false;
    if (x.rows == 1 && y.rows == 1) return true;
    if (x.rows > 1 && y.rows > 1 && x.stride != y.stride) {  // row by row
        if (x.rows > y.rows) return meet(y, x);
        for (size_t i = 0; i < x.rows; ++i)
            if (meet(Range{x.name, (const char *)x.at + i * x.stride, x.bytes}, y)) return true;
        return false;
    }
    // row i of x and row j of y meet where (i - j) stride lies between b - a - x.bytes and b - a + y.bytes
    const auto step = (int64_t)(x.rows > 1 ? x.stride : y.stride), low = (int64_t)(b - a) - (int64_t)x.bytes, high = (int64_t)(b - a) + (int64_t)y.bytes;
    const auto below = [&](int64_t v) { return v / step - (v % step < 0); };  // v / step, rounded down
    return std::max(below(low) + 1, 1 - (int64_t)y.rows) <= std::min(-below(-high) - 1, (int64_t)x.rows - 1);
}
// Written memory must not be that of any other argument.
inline int check_apart(std::initializer_list<Range> written, std::initializer_list<Range> read) {
    for (auto x = written.begin(); x != written.end(); ++x) {
        for (auto y = written.begin(); y != x; ++y)
            if (meet(*x, *y)) return fail(KR_E_INVALID, "%s and %s overlap", y->name, x->name);
        for (const Range &y : read)
            if (meet(*x, y)) return fail(KR_E_INVALID, "%s overlaps %s", x->name, y.name);
    }
    return KR_OK;
}

inline int check_rope(const kr_rope *r, uint32_t head_dim) {
    if (!r->cos_sin || !r->positions) return fail(KR_E_INVALID, "rope: NULL pointer");
    if (r->layout != KR_ROPE_HALF && r->layout != KR_ROPE_INTERLEAVED) return fail(KR_E_INVALID, "rope: layout %d", r->layout);
    if (r->inverse != 0 && r->inverse != 1) return fail(KR_E_INVALID, "rope: inverse must be 0 or 1");
    if (r->rows == 0) return fail(KR_E_SHAPE, "rope: the table has no rows");
    if (r->rotary_dim == 0 || r->rotary_dim % 2 || r->rotary_dim > head_dim)
        return fail(KR_E_SHAPE, "rope: rotary_dim=%u is not even, 2 .. head_dim=%u", r->rotary_dim, head_dim);
    if (!on(r->cos_sin, 8) || !on(r->positions, 4)) return fail(KR_E_ALIGN, "rope: cos_sin must be 8-byte aligned");
    return KR_OK;
}

inline RopeArgs to_rope(const kr_rope *r) {
    return RopeArgs{r->cos_sin, r->positions, r->rows, r->rotary_dim, r->layout == KR_ROPE_INTERLEAVED, r->inverse};
}

constexpr float kMaxScale = 0x1p100f;  // times log2(e) a float

}  // namespace kr
