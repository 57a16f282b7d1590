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

namespace qmr {
namespace {

using linear::gate_of;
using linear::log_decay;
using linear::Quad;
using linear::quad_at;
using linear::sigmoid;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;

// Token after token, a workgroup a sequence and value head. A thread has R rows
// of four columns of the state in registers, CG threads a row. One sum over
// the rows a token: k and q meet the old state together, since
//
//   S_t^T q = e^g S_{t-1}^T q + (k . q) u,  u what the token adds along k.
template <int CG, int R>
__global__ __launch_bounds__(kThreads) void attn_linear_tokens_kernel(LinearArgs a) {
    __shared__ Quad sums[2][kWaves][2][CG];
    __shared__ float dots[2][kWaves][3];
    const uint32_t s = blockIdx.x / a.v_heads, h = blockIdx.x % a.v_heads;
    uint32_t first, count;
    seq::tokens_of(a.seq, s, first, count);
    if (count == 0) return;
    bool read;
    const uint32_t slot = seq::slot_of(a.seq, s, read);

    const uint32_t wave = threadIdx.x / 64, l = threadIdx.x % 64;
    const uint32_t col = threadIdx.x % CG * 4, row = threadIdx.x / CG * R;
    const uint32_t dk = a.dk, dv = a.dv, kh = h / (a.v_heads / a.k_heads);
    const bool has = col < dv;
    float *state = a.state + (size_t(slot == seq::kNoSlot ? 0 : slot) * a.v_heads + h) * dk * dv;
    Quad S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = quad_at(state + size_t(row + i) * dv + col, read && has && row + i < dk);

    const float *qp = a.q + size_t(first) * a.q_stride + size_t(kh) * dk + row;
    const float *kp = a.k + size_t(first) * a.k_stride + size_t(kh) * dk + row;
    const float *vp = a.v + size_t(first) * a.v_stride + size_t(h) * dv + col;
    Quad q[R / 4], k[R / 4], v;
    auto load = [&](uint32_t t) {
#pragma unroll
        for (int i = 0; i < R / 4; ++i) {
            q[i] = quad_at(qp + size_t(t) * a.q_stride + 4 * i, row + 4 * i < dk);
            k[i] = quad_at(kp + size_t(t) * a.k_stride + 4 * i, row + 4 * i < dk);
        }
        v = quad_at(vp + size_t(t) * a.v_stride, has);
    };
    load(0);
    for (uint32_t t = 0; t < count; ++t) {
        Quad sk{}, sq{};
        float kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float ki = k[i / 4].x[i % 4], qi = q[i / 4].x[i % 4];
            kk = fmaf(ki, ki, kk);
            qq = fmaf(qi, qi, qq);
            qk = fmaf(qi, ki, qk);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk.x[j] = fmaf(S[i].x[j], ki, sk.x[j]);
                sq.x[j] = fmaf(S[i].x[j], qi, sq.x[j]);
            }
        }
#pragma unroll
        for (int d = CG; d < 64; d *= 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk.x[j] += __shfl_xor(sk.x[j], d);
                sq.x[j] += __shfl_xor(sq.x[j], d);
            }
            kk += __shfl_xor(kk, d);
            qq += __shfl_xor(qq, d);
            qk += __shfl_xor(qk, d);
        }
        const uint32_t at = t % 2;  // the other one may still be read
        if (l < CG) {
            sums[at][wave][0][l] = sk;
            sums[at][wave][1][l] = sq;
        }
        if (l == 0) {
            dots[at][wave][0] = kk;
            dots[at][wave][1] = qq;
            dots[at][wave][2] = qk;
        }
        const size_t token = size_t(first) + t;
        const float decay = expf(log_decay(a, token, h));
        const float beta = a.delta ? sigmoid(a.b[token * a.b_stride + h]) : 1.f;
        __syncthreads();
        sk = Quad{};
        sq = Quad{};
        kk = qq = qk = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk.x[j] += sums[at][w][0][l % CG].x[j];
                sq.x[j] += sums[at][w][1][l % CG].x[j];
            }
            kk += dots[at][w][0];
            qq += dots[at][w][1];
            qk += dots[at][w][2];
        }
        const float fk = a.qk_eps > 0.f ? 1.f / sqrtf(kk + a.qk_eps) : 1.f;
        const float fq = (a.qk_eps > 0.f ? 1.f / sqrtf(qq + a.qk_eps) : 1.f) * a.scale;
        Quad u, o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u.x[j] = a.delta ? beta * (v.x[j] - decay * (sk.x[j] * fk)) : v.x[j];
            o.x[j] = fq * (decay * sq.x[j] + qk * fk * u.x[j]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float ki = k[i / 4].x[i % 4] * fk;
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i].x[j] = fmaf(ki, u.x[j], decay * S[i].x[j]);
        }
        if (t + 1 < count) load(t + 1);
        if (wave == 0) {
            if (a.out_eps > 0.f) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) sum += o.x[j] * o.x[j];  // columns past dv are zero
#pragma unroll
                for (int d = 1; d < CG; d *= 2) sum += __shfl_xor(sum, d);
                const float f = 1.f / sqrtf(sum / float(dv) + a.out_eps);
                const Quad z = quad_at(a.z + token * a.z_stride + size_t(h) * dv + col, has);
                const Quad n = quad_at(a.norm + col, has);
#pragma unroll
                for (int j = 0; j < 4; ++j) o.x[j] = o.x[j] * f * gate_of(z.x[j], n.x[j]);
            }
            if (l < CG && has)
                *reinterpret_cast<Quad *>(a.out + token * a.out_stride + size_t(h) * dv + col) = o;
        }
    }
    if (!a.keep || slot == seq::kNoSlot) return;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (has && row + i < dk) *reinterpret_cast<Quad *>(state + size_t(row + i) * dv + col) = S[i];
}

template <int CG>
void go_tokens(const LinearArgs &a, hipStream_t stream) {
    const uint32_t blocks = a.seq.seqs * a.v_heads, rows = (a.dk + kThreads / CG - 1) / (kThreads / CG);
    if (rows <= 4) {
        attn_linear_tokens_kernel<CG, 4><<<blocks, kThreads, 0, stream>>>(a);
    } else if constexpr (CG >= 16) {
        if (rows <= 8) {
            attn_linear_tokens_kernel<CG, 8><<<blocks, kThreads, 0, stream>>>(a);
        } else if constexpr (CG >= 32) {
            if (rows <= 16) {
                attn_linear_tokens_kernel<CG, 16><<<blocks, kThreads, 0, stream>>>(a);
            } else if constexpr (CG >= 64) {
                attn_linear_tokens_kernel<CG, 32><<<blocks, kThreads, 0, stream>>>(a);
            }
        }
    }
}

}  // namespace

hipError_t launch_attn_linear(const LinearArgs &a, const LinearPlan &pl, void *workspace, hipStream_t stream) {
    if (pl.chunks) return launch_linear_chunks(a, pl, workspace, stream);
    if (a.dv <= 32) {
        go_tokens<8>(a, stream);
    } else if (a.dv <= 64) {
        go_tokens<16>(a, stream);
    } else if (a.dv <= 128) {
        go_tokens<32>(a, stream);
    } else {
        go_tokens<64>(a, stream);
    }
    return hipGetLastError();
}

const char *linear_kernel_name(const LinearPlan &pl) {
    return pl.chunks ? "linear_scan_kernel" : "attn_linear_tokens_kernel";
}

}  // namespace qmr
