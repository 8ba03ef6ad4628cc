// api_checks.hpp — checks that the entry points of the caches share.
#pragma once

#include <initializer_list>

#include "kriya_kv8.h"
#include "kr_internal.hpp"

namespace kr {

// A launch has fewer than 2^32 threads in a dimension: this many workgroups of 256.
constexpr uint64_t kMostGroups = 0xFFFFFFFFull / 256;

inline bool on(const void *p, size_t a) { return (uintptr_t)p % a == 0; }

// Memory of a call: what one argument points to.
struct Range {
    const char *name;
    const void *at;
    size_t bytes;
};
// Written memory must not be that of any other argument.
inline int check_apart(std::initializer_list<Range> written, std::initializer_list<Range> read) {
    const auto meet = [](const Range &x, const Range &y) {
        const auto a = (uintptr_t)x.at, b = (uintptr_t)y.at;
        return x.at && y.at && a < b + y.bytes && b < a + x.bytes;
    };
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
