// Device code shared by the kernels that feed the matrix cores through LDS
// (attn_paged.hip, attn_linear_chunks.hip): FP32 values as f16 terms, loads
// from memory straight to LDS, barriers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace qmr {
namespace wave {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kRsrcWord3 = 0x00020000u;

// x - the low (0) or high (1) f16 of h, in one instruction.
template <int HIGH>
__device__ __forceinline__ float less_half(float x, uint32_t h) {
    float r;
    if constexpr (HIGH) {
        asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    } else {
        asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    }
    return r;
}

// Two f16 in a word, to nearest.
__device__ __forceinline__ uint32_t two_halves(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), h2));
}

// A wave's 64 chunks of 16 bytes from memory straight to LDS, chunk after chunk
// from byte `to`; `rsrc`: a buffer's four words. The compiler does not see that
// they are on their way: wait_dma is the wait. The idle cycles are those a load has to keep from a
// vector instruction that wrote its scalar operands, and from m0's own write.
// (m0 is a register that the compiler allots to nothing, and it warns of the
// name; its own writes of m0 are merged across what does not say that it is written.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(u4 rsrc, uint32_t offset, uint32_t more, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(more))
                 : "memory", "m0");
}

// The same of 64 words.
__device__ __forceinline__ void dma4(u4 rsrc, uint32_t offset, uint32_t more, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(offset), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(more))
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Until at most LATER of this wave's loads are on their way.
template <int LATER>
__device__ __forceinline__ void wait_dma() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LATER) : "memory");
}

// A barrier that orders LDS alone: loads stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// LDS written by some lanes of a wave and read by others of the same wave.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

}  // namespace wave
}  // namespace qmr
