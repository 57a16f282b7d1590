// Linear attention with a state and a decay for each head. For value head h,
// whose queries and keys are those of key head h / (v_heads / k_heads), and a
// state S of dk x dv:
//
//   S_t = e^g S_{t-1} + k (beta (v - (e^g S_{t-1})^T k))^T    the delta rule, or
//   S_t = e^g S_{t-1} + k v^T
//   o_t = scale S_t^T q_t
//
// g is given, or -exp(a_log) softplus(a + dt_bias); beta = sigmoid(b). Queries
// and keys may be divided by their length first (x / sqrt(sum x^2 + eps)); the
// output may get an RMS norm of the head, its weights and silu(z).
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "linear_common.hpp"
#include "sequences.hpp"
#include "wave_ops.hpp"

namespace qmr {
namespace {

using linear::gate_of;
using linear::log_decay;
using linear::Quad;
using linear::quad_at;
using linear::sigmoid;
using wave::f4;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;

// v and another value, the sum of each over two halves of a wave: v's in the
// lanes whose bit is clear, the other's where it is set.
template <int LANES>
__device__ __forceinline__ float both_halves(float v, float other) {
    const uint32_t a = __float_as_uint(v), b = __float_as_uint(other);
    if constexpr (LANES == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
}

// Token after token, a workgroup a sequence and value head: for single tokens
// and a few. A thread has R rows of four columns of the state in registers; a
// wave has 32 columns of 8R rows, eight lanes a row, and the waves are CB blocks
// of columns by 8 / CB of rows. One sum over the rows a token, of 11 numbers a
// lane: k and q meet the old state together, since
//
//   S_t^T q = e^g S_{t-1}^T q + (k . q) u,  u what the token adds along k,
//
// and k.k, q.q and q.k give the lengths. In a wave the sum is halved and dealt at
// once, 12 numbers to six to three a lane, so that 12 swaps and 12 adds do what
// 33 exchanges would. Rows of q, k, v and z come to LDS two tokens ahead.
//
// With many sequences the states bound it: 32 tokens of as many sequences, 48
// heads of 128 x 128, are 201 MB read and written in 36 us (5.6 TB/s, in part
// from the last-level cache). A single one takes 5.9 us, a launch and its chain
// of loads, sums and barriers, and each further token 1.3 us: 400 instructions a
// wave, two waves a SIMD. (With a gate's exponentials, the decay's and three
// roots with their quotients in every token and wave it was 2.1.)
template <int CB, int R>
__global__ __launch_bounds__(kThreads) void attn_linear_tokens_kernel(LinearArgs a) {
    constexpr int RB = kWaves / CB, kKeys = R * 8 * RB, kValues = CB * 32;  // row blocks; dimensions there is room for
    constexpr int kRow = 2 * (kKeys + kValues), kEach = (kRow + kThreads - 1) / kThreads;
    __shared__ __align__(16) float rows[3][kRow];          // q, k, v, what z and the norm's weights make of an output
    __shared__ __align__(16) float sums[2][kWaves][8][12]; // of a wave's eight column groups
    __shared__ float decays[2][64], betas[2][64];  // of 64 tokens at once, a lane a token
    __shared__ float squares[2][CB];
    const uint32_t s = blockIdx.x / a.v_heads, h = blockIdx.x % a.v_heads;
    uint32_t first, count;
    seq::tokens_of(a.seq, s, first, count);
    if (count == 0) return;
    bool read;
    const uint32_t slot = seq::slot_of(a.seq, s, read);

    const uint32_t tid = threadIdx.x, wave = tid / 64, l = tid % 64;
    const uint32_t cb = wave % CB, rb = wave / CB, group = l % 8;
    const uint32_t col = cb * 32 + group * 4, row = rb * (8 * R) + l / 8 * R;
    const uint32_t dk = a.dk, dv = a.dv, kh = h / (a.v_heads / a.k_heads);
    const bool has = col < dv;
    float *state = a.state + (size_t(slot == seq::kNoSlot ? 0 : slot) * a.v_heads + h) * dk * dv;
    Quad S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = quad_at(state + size_t(row + i) * dv + col, read && has && row + i < dk);

    // What this thread brings of a token's rows.
    const float *from[kEach];
    float norm[kEach] = {};
    uint32_t step[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const uint32_t i = tid + e * kThreads;
        const bool of_q = i < kKeys, of_k = !of_q && i < 2 * kKeys, of_z = i >= 2 * kKeys + kValues;
        const uint32_t d = of_q ? i : of_k ? i - kKeys : i - 2 * kKeys - of_z * kValues;
        const float *p = of_q   ? a.q + size_t(first) * a.q_stride + size_t(kh) * dk
                         : of_k ? a.k + size_t(first) * a.k_stride + size_t(kh) * dk
                         : of_z ? a.z + size_t(first) * a.z_stride + size_t(h) * dv
                                : a.v + size_t(first) * a.v_stride + size_t(h) * dv;
        step[e] = of_q ? a.q_stride : of_k ? a.k_stride : of_z ? a.z_stride : a.v_stride;
        from[e] = i < kRow && d < (of_q || of_k ? dk : dv) && (!of_z || a.out_eps > 0.f) ? p + d : nullptr;
        if (of_z && from[e]) norm[e] = a.norm[d];
    }
    float next[kEach];
    auto load = [&](uint32_t t) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) next[e] = from[e] ? from[e][size_t(t) * step[e]] : 0.f;
    };
    auto keep = [&](uint32_t t) {
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (const uint32_t i = tid + e * kThreads; i < kRow)
                rows[t % 3][i] = i < 2 * kKeys + kValues ? next[e] : gate_of(next[e], norm[e]);
    };
    auto gates = [&](uint32_t t) {
        const size_t token = size_t(first) + t + l;
        const bool any = t + l < count;
        if (wave == 0) decays[t / 64 % 2][l] = any ? expf(log_decay(a, token, h)) : 1.f;
        if (wave == 1) betas[t / 64 % 2][l] = any && a.delta ? sigmoid(a.b[token * a.b_stride + h]) : 1.f;
    };
    load(0);
    keep(0);
    gates(0);
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the state is here, and no wait for it below waits for the loads ahead
    if (count > 1) load(1);
    wave::lds_barrier();
    for (uint32_t t = 0; t < count; ++t) {
        if (t && t % 64 == 0) gates(t);
        if (t + 1 < count) keep(t + 1);
        if (t + 2 < count) load(t + 2);
        const float *now = rows[t % 3];
        float sum[12] = {};  // S^T k, S^T q, k.k, q.q, q.k
        Quad k[R / 4];
#pragma unroll
        for (int j = 0; j < R / 4; ++j) {
            const Quad q = *reinterpret_cast<const Quad *>(now + row + 4 * j);
            k[j] = *reinterpret_cast<const Quad *>(now + kKeys + row + 4 * j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ki = k[j].x[i], qi = q.x[i];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    sum[c] = fmaf(S[4 * j + i].x[c], ki, sum[c]);
                    sum[4 + c] = fmaf(S[4 * j + i].x[c], qi, sum[4 + c]);
                }
                sum[8] = fmaf(ki, ki, sum[8]);
                sum[9] = fmaf(qi, qi, sum[9]);
                sum[10] = fmaf(qi, ki, sum[10]);
            }
        }
        // Lanes with bit 5 have the last six, of those lanes with bit 4 the last three.
#pragma unroll
        for (int i = 0; i < 6; ++i) sum[i] = both_halves<32>(sum[i], sum[6 + i]);
#pragma unroll
        for (int i = 0; i < 3; ++i) sum[i] = both_halves<16>(sum[i], sum[3 + i]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
            sum[i] += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(sum[i]), 0x128, 0xf, 0xf, true));  // row_ror:8
        const uint32_t at = t % 2;  // the other one may still be read
        if (!(l & 8)) {
#pragma unroll
            for (int i = 0; i < 3; ++i) sums[at][wave][group][l / 32 * 6 + l / 16 % 2 * 3 + i] = sum[i];
        }
        wave::lds_barrier();
        f4 sk{}, sq{}, dots{};
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const f4 *p = reinterpret_cast<const f4 *>(sums[at][b * CB + cb][group]);
            sk += p[0];
            sq += p[1];
            dots += p[2];
        }
        const float decay = decays[t / 64 % 2][t % 64], beta = betas[t / 64 % 2][t % 64];
        const Quad v = *reinterpret_cast<const Quad *>(now + 2 * kKeys + col);
        const float fk = a.qk_eps > 0.f ? rsqrtf(dots[0] + a.qk_eps) : 1.f;
        const float fq = (a.qk_eps > 0.f ? rsqrtf(dots[1] + a.qk_eps) : 1.f) * a.scale;
        Quad u, o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u.x[j] = a.delta ? beta * (v.x[j] - decay * (sk[j] * fk)) : v.x[j];
            o.x[j] = fq * (decay * sq[j] + dots[2] * fk * u.x[j]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float ki = k[i / 4].x[i % 4] * fk;
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i].x[j] = fmaf(ki, u.x[j], decay * S[i].x[j]);
        }
        if (a.out_eps > 0.f) {
            float sum_sq = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum_sq = fmaf(o.x[j], o.x[j], sum_sq);  // columns past dv are zero
#pragma unroll
            for (int d = 1; d < 8; d *= 2) sum_sq += __shfl_xor(sum_sq, d);
            if constexpr (CB > 1) {
                if (rb == 0 && l == 0) squares[at][cb] = sum_sq;
                wave::lds_barrier();
                sum_sq = 0.f;
#pragma unroll
                for (int b = 0; b < CB; ++b) sum_sq += squares[at][b];
            }
            const Quad gate = *reinterpret_cast<const Quad *>(now + 2 * kKeys + kValues + col);
            const float f = rsqrtf(sum_sq / float(dv) + a.out_eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) o.x[j] = o.x[j] * f * gate.x[j];
        }
        if (rb == 0 && l < 8 && has)  // the waves of the first rows write the outputs
            *reinterpret_cast<Quad *>(a.out + (size_t(first) + t) * a.out_stride + size_t(h) * dv + col) = o;
    }
    if (!a.keep || slot == seq::kNoSlot) return;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (has && row + i < dk) *reinterpret_cast<Quad *>(state + size_t(row + i) * dv + col) = S[i];
}

template <int CB>
void go_tokens(const LinearArgs &a, hipStream_t stream) {
    const uint32_t blocks = a.seq.seqs * a.v_heads, rows = (a.dk + 64 / CB - 1) / (64 / CB);  // of a thread
    if (rows <= 4) {
        attn_linear_tokens_kernel<CB, 4><<<blocks, kThreads, 0, stream>>>(a);
    } else if constexpr (CB >= 2) {
        if (rows <= 8) {
            attn_linear_tokens_kernel<CB, 8><<<blocks, kThreads, 0, stream>>>(a);
        } else if constexpr (CB >= 4) {
            if (rows <= 16) {
                attn_linear_tokens_kernel<CB, 16><<<blocks, kThreads, 0, stream>>>(a);
            } else if constexpr (CB >= 8) {
                attn_linear_tokens_kernel<CB, 32><<<blocks, kThreads, 0, stream>>>(a);
            }
        }
    }
}

}  // namespace

hipError_t launch_attn_linear(const LinearArgs &a, const LinearPlan &pl, void *workspace, hipStream_t stream) {
    if (pl.chunks) return launch_linear_chunks(a, pl, workspace, stream);
    if (a.dv <= 32) {
        go_tokens<1>(a, stream);
    } else if (a.dv <= 64) {
        go_tokens<2>(a, stream);
    } else if (a.dv <= 128) {
        go_tokens<4>(a, stream);
    } else {
        go_tokens<8>(a, stream);
    }
    return hipGetLastError();
}

const char *linear_kernel_name(const LinearPlan &pl) {
    return pl.chunks ? "linear_scan_kernel" : "attn_linear_tokens_kernel";
}

}  // namespace qmr
