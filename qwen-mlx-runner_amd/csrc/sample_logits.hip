// A token from each row of logits, drawn with a given random number. With
// weights w_i = exp((x_i - max) / temperature) the tokens kept are
//
//   top k     the first k by logit, equal logits by index
//   top p     of those, in that order, each one before which less than p of
//             their weight stands (so the first always)
//   min p     of those, the ones with w_i >= min_p
//
// and the token is the first by index up to which more than uniform * (weight
// kept) is kept. NaN and -infinity are never kept; of infinite logits each
// weighs 1 and the others nothing. A temperature that is not above 0 takes the
// first largest logit.
//
// Weights are whole numbers, w_i * 2^shift rounded, the shift such that a row's
// sum stays below 2^62: sums are exact in any order, so a token does not depend
// on how the row was split, and a weight is off by 2^-45 at most at 248320
// tokens. They are worked out in 64 bits: with weights of 32, one draw in a
// hundred of a broad row would fall on the other side of a border.
//
// Nothing is sorted. The borders of top k and top p are a logit and a number of
// ties at it, found digit by digit: a histogram of the next eight bits of those
// that agree in the bits before, counts for top k, weights for top p.
#include <hip/hip_runtime.h>

#include "kernels.hpp"

namespace qmr {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
using u64 = unsigned long long;

constexpr uint32_t kNone = 0xffffffffu;

// Ordered as the logits are; NaN and -infinity are 0. Both zeros are one logit.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// n weights of at most 2^shift add up to 2^62 at most.
__host__ __device__ constexpr uint32_t shift_of(uint32_t n) {
    uint32_t bits = 10;
    while ((uint64_t(1) << bits) < n) ++bits;
    return 62 - bits;
}

// What a row's weights are made with.
struct Weights {
    float max;
    double temperature;
    double one;  // 2^shift

    __device__ double plain(uint32_t key) const {
        const float x = logit_of(key);
        if (x == max) return 1.0;
        if (max == INFINITY) return 0.0;
        return exp((double(x) - double(max)) / temperature);
    }
    __device__ u64 whole(uint32_t key) const { return u64(__double2ll_rn(plain(key) * one)); }
};

template <typename T>
__device__ __forceinline__ T block_sum(T v, T *room) {
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    __syncthreads();
    if (threadIdx.x % 64 == 0) room[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kWaves; ++w) v += room[w];
    return v;
}

// The sums up to and with each thread's v.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *room) {
    for (int d = 1; d < 64; d *= 2) {
        const T before = __shfl_up(v, d);
        if (int(threadIdx.x % 64) >= d) v += before;
    }
    __syncthreads();
    if (threadIdx.x % 64 == 63) room[threadIdx.x / 64] = v;
    __syncthreads();
    for (int w = 0; w < int(threadIdx.x / 64); ++w) v += room[w];
    return v;
}

// A border: keys above `key` are kept, and of those at it the first `ties` by
// index.
struct Border {
    uint32_t key = 0;
    uint32_t ties = 0;
};

// A workgroup a row.
__global__ __launch_bounds__(kThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ u64 bins[256];
    __shared__ u64 room[kWaves];
    __shared__ u64 found[2];
    const uint32_t row = blockIdx.x, n = a.vocab, tid = threadIdx.x;
    const float *x = a.logits + size_t(row) * a.stride;

    uint32_t top = 0;
    u64 valid = 0;
    for (uint32_t i = tid; i < n; i += kThreads) {
        const uint32_t key = key_of(x[i]);
        top = max(top, key);
        valid += key != 0;
    }
    for (int d = 1; d < 64; d *= 2) top = max(top, uint32_t(__shfl_xor(top, d)));
    if (tid % 64 == 0) room[tid / 64] = top;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) top = max(top, uint32_t(room[w]));
    valid = block_sum(valid, room);
    if (top == 0) {
        if (tid == 0) a.tokens[row] = kNone, a.probs[row] = 0.f;
        return;
    }

    const float temperature = a.temperature[row];
    const Weights weights{logit_of(top), double(temperature), double(u64(1) << shift_of(n))};
    const bool greedy = !(temperature > 0.f);

    // Walks the keys from the largest down to where `before(sum)` no longer
    // holds, sums of amount(key) over the keys of `in`; `sum` is then that of
    // the keys above the border.
    auto descend = [&](auto in, auto amount, auto inside, u64 &above) {
        uint32_t prefix = 0;
        above = 0;
        for (int digit = 3; digit >= 0; --digit) {
            const int low = 8 * digit;
            __syncthreads();
            if (tid < 256) bins[tid] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < n; i += kThreads) {
                const uint32_t key = key_of(x[i]);
                if (key == 0 || !in(key, i)) continue;
                if (digit < 3 && (key >> (low + 8)) != (prefix >> (low + 8))) continue;
                atomicAdd(&bins[(key >> low) & 255], amount(key));
            }
            __syncthreads();
            if (tid == 0) {
                // The last bin, from above, whose first key may still be inside.
                u64 sum = above;
                uint32_t at = 0, some = 0;
                u64 up_to = above;
                for (int b = 255; b >= 0; --b) {
                    if (bins[b] == 0) continue;
                    if (some && !inside(sum)) break;
                    at = b;
                    up_to = sum;
                    some = 1;
                    sum += bins[b];
                }
                found[0] = at;
                found[1] = up_to;
            }
            __syncthreads();
            prefix |= uint32_t(found[0]) << low;
            above = found[1];
        }
        return prefix;
    };

    // Top k.
    Border k{0, kNone};
    const uint32_t most = a.top_k[row];
    if (greedy) {
        k = {top, 1};
    } else if (most > 0 && most < valid) {
        u64 above;
        k.key = descend([](uint32_t, uint32_t) { return true; }, [](uint32_t) { return u64(1); },
                        [&](u64 sum) { return sum < most; }, above);
        k.ties = uint32_t(most - above);
    }
    // The index of the last tie that a border keeps.
    auto last_tie = [&](const Border &b, u64 ties) -> uint32_t {
        if (b.key == 0 || ties >= n) return n;
        u64 before = 0;
        for (uint32_t base = 0; base < n; base += kThreads) {
            const uint32_t i = base + tid;
            const u64 tie = i < n && key_of(x[i]) == b.key;
            const u64 up_to = before + block_scan(tie, room);
            __syncthreads();
            if (tie && up_to == ties) found[0] = i;
            if (tid == kThreads - 1) room[0] = up_to;
            __syncthreads();
            before = room[0];
            const bool done = before >= ties;
            const uint32_t at = uint32_t(found[0]);
            __syncthreads();
            if (done) return at;
        }
        return n;
    };
    uint32_t k_last = last_tie(k, k.ties);
    auto in_k = [&](uint32_t key, uint32_t i) { return key > k.key || (key == k.key && i <= k_last); };

    // Top p.
    Border p{0, kNone};
    const float part = a.top_p[row];
    uint32_t p_last = n;
    if (!greedy && part < 1.f) {
        u64 all = 0;
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t key = key_of(x[i]);
            if (key && in_k(key, i)) all += weights.whole(key);
        }
        const double target = fmax(double(part), 0.0) * double(block_sum(all, room));
        u64 above;
        p.key = descend(in_k, [&](uint32_t key) { return weights.whole(key); },
                        [&](u64 sum) { return double(sum) < target; }, above);
        // Ties: the one before which `above` and j of their weight stand.
        const u64 w = weights.whole(p.key);
        p.ties = 1;
        if (w == 0) {
            p.ties = double(above) < target || above == 0 ? kNone : 1;
        } else {
            u64 j = target > double(above) ? u64((target - double(above)) / double(w)) : 0;
            while (j > 0 && double(above + (j - 1) * w) >= target) --j;
            while (double(above + j * w) < target) ++j;
            p.ties = uint32_t(max(j, u64(1)));
        }
        p_last = last_tie(p, p.ties);
    }
    const float min_p = a.min_p[row];
    auto kept = [&](uint32_t i) -> uint32_t {
        const uint32_t key = i < n ? key_of(x[i]) : 0;
        if (key == 0 || !in_k(key, i)) return 0;
        if (key < p.key || (key == p.key && i > p_last)) return 0;
        if (key != top && min_p > 0.f && weights.plain(key) < double(min_p)) return 0;
        return key;
    };

    u64 total = 0;
    for (uint32_t i = tid; i < n; i += kThreads) {
        const uint32_t key = kept(i);
        if (key) total += weights.whole(key);
    }
    total = block_sum(total, room);
    const double u = fmin(fmax(double(a.uniform[row]), 0.0), 1.0);
    const u64 target = min(u64(u * double(total)), total - 1);
    u64 before = 0;
    for (uint32_t base = 0; base < n; base += kThreads) {
        const uint32_t key = kept(base + tid);
        const u64 w = key ? weights.whole(key) : 0;
        const u64 up_to = before + block_scan(w, room);
        if (w && up_to > target && up_to - w <= target) {
            a.tokens[row] = base + tid;
            a.probs[row] = float(double(w) / double(total));
        }
        __syncthreads();
        if (tid == kThreads - 1) room[0] = up_to;
        __syncthreads();
        before = room[0];
        __syncthreads();
        if (before > target) return;
    }
}

}  // namespace

hipError_t launch_sample_logits(const SampleArgs &a, const DeviceLimits &, hipStream_t stream) {
    sample_row_kernel<<<a.rows, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace qmr
