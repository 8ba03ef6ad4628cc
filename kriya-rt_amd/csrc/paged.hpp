// paged.hpp — where a slot of the paged cache lies.
//
// A unit is 16 slots of one page and kv head, D dims, bf16 in the order of the matrix instructions' operands:
//   keys    (slot r, dim d) at d / 8 128 + 8 r + d % 8: a lane's 16 bytes are 8 dims of one slot, those of 16 slots side by side;
//   values  (slot r = 8 a + 4 h + j, dim d) at d / 32 512 + 256 h + 8 (d % 32) + 4 a + j: a lane's 16 bytes are 8 slots of one dim,
//           those whose probabilities the same lane holds after the first product, so that no probability changes lanes.
#pragma once

#include "ragged.hpp"

namespace kr {

// elements within a unit
__host__ __device__ constexpr uint32_t paged_key_at(uint32_t r, uint32_t d) { return d / 8 * 128 + 8 * r + d % 8; }
__host__ __device__ constexpr uint32_t paged_value_at(uint32_t r, uint32_t d) {
    return d / 32 * 512 + r / 4 % 2 * 256 + d % 32 * 8 + r / 8 * 4 + r % 4;
}

// The page that holds unit u (slots 16 u ..) of sequence b; c.pages or more: none.
__device__ __forceinline__ uint32_t page_of(const Paged &c, uint32_t b, uint32_t u) {
    const uint32_t p = u >> c.shift;
    return p < c.max_pages ? c.table[(size_t)b * c.max_pages + p] : 0xFFFFFFFFu;
}
// Where unit u lies: units from the pool's start (below 2^32), and elements.
__device__ __forceinline__ uint32_t unit_place(const Paged &c, uint32_t page, uint32_t head, uint32_t u) {
    return ((page * c.heads + head) << c.shift) + (u & ((1u << c.shift) - 1));
}
__device__ __forceinline__ size_t unit_at(const Paged &c, uint32_t page, uint32_t head, uint32_t u) {
    return (size_t)unit_place(c, page, head, u) * (kPagedUnit * c.D);
}

}  // namespace kr
