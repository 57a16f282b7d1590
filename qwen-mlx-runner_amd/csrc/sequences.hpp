// Device code shared by the operators that keep a state for each sequence
// (conv_causal.hip, attn_linear.hip): where sequences stand among the tokens,
// and which slot of the pool is a sequence's own.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.hpp"

namespace qmr {
namespace seq {

constexpr uint32_t kFresh = 0x80000000u;  // of a slot word: the state is taken as zeros
constexpr uint32_t kNoSlot = 0xffffffffu;

// First token and number of tokens of sequence s, inside the rows whatever the
// starts hold.
__device__ __forceinline__ void tokens_of(const Sequences &q, uint32_t s, uint32_t &first, uint32_t &count) {
    first = min(q.starts[s], q.tokens);
    const uint32_t end = min(q.starts[s + 1], q.tokens);
    count = end > first ? min(end - first, q.most) : 0;
}

// A sequence's slot and whether it is read. A slot past the pool, or one that
// an earlier sequence names, is no slot: of two sequences that share one the
// first has it, so that no two write the same state. For whole waves.
__device__ __forceinline__ uint32_t slot_of(const Sequences &q, uint32_t s, bool &read) {
    const uint32_t word = q.slots[s], slot = word & ~kFresh, l = threadIdx.x % 64;
    read = false;
    if (slot >= q.pool) return kNoSlot;
    for (uint32_t base = 0; base < s; base += 64)
        if (__ballot(base + l < s && (q.slots[min(base + l, s)] & ~kFresh) == slot)) return kNoSlot;
    read = !(word & kFresh);
    return slot;
}

// Which part of which sequence is number `id`, where a sequence has a part for
// every `size` tokens begun: false past the last. For whole waves.
__device__ __forceinline__ bool part_of(const Sequences &q, uint32_t id, uint32_t size, uint32_t &s, uint32_t &part) {
    const uint32_t l = threadIdx.x % 64;
    for (uint32_t base = 0; base < q.seqs; base += 64) {
        uint32_t first = 0, count = 0;
        if (base + l < q.seqs) tokens_of(q, base + l, first, count);
        const uint32_t own = (count + size - 1) / size;
        uint32_t up_to = own;
        for (uint32_t d = 1; d < 64; d *= 2) {
            const uint32_t before = __shfl_up(up_to, d);
            if (l >= d) up_to += before;
        }
        const uint64_t past = __ballot(up_to > id);
        if (past) {
            const uint32_t at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            s = base + at;
            part = id - (__builtin_amdgcn_readlane(up_to, at) - __builtin_amdgcn_readlane(own, at));
            return true;
        }
        id -= __builtin_amdgcn_readlane(up_to, 63);
    }
    return false;
}

// The number that sequence s's first part has. For whole waves.
__device__ __forceinline__ uint32_t parts_before(const Sequences &q, uint32_t s, uint32_t size) {
    const uint32_t l = threadIdx.x % 64;
    uint32_t sum = 0;
    for (uint32_t base = 0; base < s; base += 64) {
        uint32_t first = 0, count = 0;
        if (base + l < s) tokens_of(q, base + l, first, count);
        sum += (count + size - 1) / size;
    }
    for (uint32_t d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    return __builtin_amdgcn_readfirstlane(sum);
}

}  // namespace seq
}  // namespace qmr
