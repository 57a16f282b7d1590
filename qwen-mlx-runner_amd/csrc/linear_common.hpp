// Device code shared by the kernels of linear attention (attn_linear.hip,
// attn_linear_chunks.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels.hpp"

namespace qmr {
namespace linear {

// Four FP32 of a row, which need not lie on 16 bytes.
struct Quad {
    float x[4];
};

__device__ __forceinline__ Quad quad_at(const float *p, bool there) {
    return there ? *reinterpret_cast<const Quad *>(p) : Quad{};
}

// The log of a decay, from its row's value and what the gates make of it.
__device__ __forceinline__ float log_decay(bool gates, float x, float a_log, float dt_bias) {
    if (!gates) return x;
    const float y = x + dt_bias;
    // Past 20, log(1 + e^y) is y to 2^-33 of it.
    return -expf(a_log) * (y > 20.f ? y : log1pf(expf(y)));
}

// That of value head h at token t.
__device__ __forceinline__ float log_decay(const LinearArgs &a, size_t t, uint32_t h) {
    return log_decay(a.gates, a.a[t * a.a_stride + h], a.gates ? a.a_log[h] : 0.f, a.gates ? a.dt_bias[h] : 0.f);
}

__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// What the output norm multiplies an element of its head by, apart from 1 / rms.
__device__ __forceinline__ float gate_of(float z, float norm) { return norm * z * sigmoid(z); }

}  // namespace linear
}  // namespace qmr
