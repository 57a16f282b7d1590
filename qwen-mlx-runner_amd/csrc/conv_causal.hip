// The short causal convolution of a linear-attention layer, one filter a
// channel, over the new tokens of several sequences:
//
//   y[t][c] = act(bias[c] + sum_j w[c][j] x[t - (width - 1) + j][c])
//
// Inputs before a sequence's first new token come from its state, the last
// width - 1 inputs that it had; the last ones of state and new tokens together
// are its next state.
//
// Memory bounds it: every input is read once and every output written once
// (10240 channels, 12000 tokens: 209 us, 4.7 TB/s, a large copy's rate; one token:
// 3.9 us, a launch and two loads one after the other).
// A thread has four channels of `span` successive tokens of one sequence and
// keeps the window in registers, so that of its inputs only the width - 1
// before its first are read again. Spans begin where their sequence begins
// (not at multiples of all tokens): with a span of at least width - 1 tokens
// only the first one of a sequence looks at the state, and that one replaces
// it, having read it first.
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "sequences.hpp"

namespace qmr {
namespace {

constexpr int kThreads = 64;
constexpr int kAhead = 8;  // tokens whose loads are under way together

// V FP32 of a row, which need not lie on more than 4 bytes.
template <int V>
struct Vec {
    float x[V];
};

template <int V>
__device__ __forceinline__ Vec<V> load(const float *p) {
    return *reinterpret_cast<const Vec<V> *>(p);
}

template <int V, int W>
__global__ __launch_bounds__(kThreads) void conv_causal_kernel(ConvArgs a, uint32_t span) {
    const Sequences &q = a.seq;
    uint32_t s, part, first, count;
    if (!seq::part_of(q, blockIdx.x, span, s, part)) return;
    seq::tokens_of(q, s, first, count);
    bool read = false;
    uint32_t slot = seq::kNoSlot;
    if (part == 0) slot = seq::slot_of(q, s, read);
    const uint32_t c = (blockIdx.y * kThreads + threadIdx.x) * V;
    if (c >= a.channels) return;

    const size_t xs = a.x_stride, ys = a.y_stride;
    const float *x = a.x + size_t(first) * xs + c;
    float *y = a.y + size_t(first) * ys + c;
    float *state = a.state + size_t(slot == seq::kNoSlot ? 0 : slot) * (W - 1) * a.channels + c;
    const uint32_t t0 = part * span, t1 = min(t0 + span, count);

    Vec<V> window[W - 1];  // the inputs before the next token, oldest first
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
        if (part > 0) {
            window[j] = load<V>(x + size_t(t0 - (W - 1) + j) * xs);
        } else if (read) {
            window[j] = load<V>(state + size_t(j) * a.channels);
        } else {
            window[j] = Vec<V>{};
        }
    }
    float w[V][W], bias[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = a.bias ? a.bias[c + v] : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[v][j] = a.w[size_t(c + v) * W + j];
    }
    if (slot != seq::kNoSlot && a.keep) {
        // Input i of the next state stands at token count - (W - 1) + i, or
        // still in the window that the state gave.
        Vec<V> next[W - 1];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int64_t t = int64_t(count) - (W - 1) + i;
            next[i] = Vec<V>{};
            if (t >= 0) {
                next[i] = load<V>(x + size_t(t) * xs);
            } else {
#pragma unroll
                for (int j = 0; j < W - 1; ++j)
                    if (j == t + (W - 1)) next[i] = window[j];
            }
        }
#pragma unroll
        for (int i = 0; i < W - 1; ++i) *reinterpret_cast<Vec<V> *>(state + size_t(i) * a.channels) = next[i];
    }
    for (uint32_t t = t0; t < t1; t += kAhead) {
        Vec<V> in[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (t + k < t1) in[k] = load<V>(x + size_t(t + k) * xs);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (t + k >= t1) break;
            Vec<V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float sum = bias[v];
#pragma unroll
                for (int j = 0; j < W - 1; ++j) sum = fmaf(w[v][j], window[j].x[v], sum);
                sum = fmaf(w[v][W - 1], in[k].x[v], sum);
                out.x[v] = a.silu ? sum / (1.f + expf(-sum)) : sum;
            }
            *reinterpret_cast<Vec<V> *>(y + size_t(t + k) * ys) = out;
#pragma unroll
            for (int j = 0; j + 1 < W - 1; ++j) window[j] = window[j + 1];
            window[W - 2] = in[k];
        }
    }
}

}  // namespace

hipError_t launch_conv_causal(const ConvArgs &a, const DeviceLimits &lim, hipStream_t stream) {
    const Sequences &q = a.seq;
    const uint32_t v = a.channels % 4 == 0 ? 4 : 1;
    const uint32_t columns = (a.channels / v + kThreads - 1) / kThreads;
    // The longest span of which there are still eight waves for every CU. With
    // two and with 32 in place of eight, 10240 channels in us: 200 tokens 9.4 and
    // 6.6 (6.6), 600 17.7 and 12.5 (13.4), 1400 23.3 and 23.0 (21.5), 6000 109 and
    // 104 (108).
    uint32_t span = 32;
    while (span > 4 && uint64_t(q.tokens / span + 1) * columns < uint64_t(lim.num_cus) * 8) span /= 2;
    const uint32_t parts = uint32_t(std::min<uint64_t>(q.tokens, uint64_t(q.tokens) / span + q.seqs));
    const dim3 grid(parts, columns);
    auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, stream>>>(a, span); };
    switch (a.width * 2 + (v == 4)) {
        case 4: go(conv_causal_kernel<1, 2>); break;
        case 5: go(conv_causal_kernel<4, 2>); break;
        case 6: go(conv_causal_kernel<1, 3>); break;
        case 7: go(conv_causal_kernel<4, 3>); break;
        case 8: go(conv_causal_kernel<1, 4>); break;
        default: go(conv_causal_kernel<4, 4>); break;
    }
    return hipGetLastError();
}

}  // namespace qmr
