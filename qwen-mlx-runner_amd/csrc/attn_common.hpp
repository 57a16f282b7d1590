// Device code shared by the kernels that write the paged cache
// (rope_append.hip) and those that read it (attn_paged.hip): places in a
// page, and the cache's 16-bit types.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.hpp"

namespace qmr {
namespace attn {

constexpr uint32_t kBlock = 32;             // keys of a block
constexpr uint32_t kKeyChunk = kBlock * 8;  // halves between a key's successive 8 dims

// Rounded to nearest, ties to even; past the type's range to infinity.
template <bool BF16>
__device__ __forceinline__ uint16_t half_bits(float x) {
    if constexpr (BF16) {
        return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
    } else {
        return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
    }
}

// First half of block `block` of a page's head, in 64 bits: pools pass 2^32
// halves.
__device__ __forceinline__ size_t block_at(const PagedCache &c, uint32_t page, uint32_t head, uint32_t block) {
    return (size_t(page) * c.kv_heads + head) * (size_t(c.page) * c.dim) + size_t(block) * (kBlock * c.dim);
}

// A key's first half; its dims 8i..8i+7 are kKeyChunk * i further.
__device__ __forceinline__ size_t key_row(const PagedCache &c, uint32_t page, uint32_t head, uint32_t slot) {
    const uint32_t k = slot % kBlock;
    return block_at(c, page, head, slot / kBlock) + (16 * (k / 4 % 2) + 4 * (k / 8) + k % 4) * 8;
}

// The chunk of eight slots that a value is in, for dim 0; dim d is 8d further.
__device__ __forceinline__ size_t value_chunk(const PagedCache &c, uint32_t page, uint32_t head, uint32_t slot) {
    return block_at(c, page, head, slot / kBlock) + size_t(slot % kBlock / 8) * c.dim * 8;
}

}  // namespace attn
}  // namespace qmr
