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
// tokens (2^-46 where there are fewer). They are worked out in 64 bits: with weights of 32, one draw in a
// hundred of a broad row would fall on the other side of a border.
//
// Nothing is sorted. A token's place is one number, its logit's bits above its
// index's, so that every border is a place and there are no ties. Rows go over
// the chip in slices, and what decides is narrowed down in four launches:
//
//   sample_max     the largest and smallest logit of each slice
//   sample_bins    tokens and weight by bins of logits, at most a 16th of the
//                  temperature wide, of each slice and of the row
//   sample_gather  from the row's bins, those that a border may fall into; the
//                  tokens in them, and each slice's weight above them
//   sample_pick    a workgroup a row: the borders among those tokens, the slice
//                  that the number falls into, and the token there (one of
//                  them, without a look at slices, if there are few)
//
// A row that fits sample_pick's LDS needs that launch alone. One that has too
// many tokens in its bins (many equal logits, or a temperature so far above most
// of them that they share a few bins, beside an outlier that widens those) is
// worked on by sample_pick alone, which reads it once a digit of the borders: 0.9
// to 1.7 ms for 248320 logits with top k or top p, where 35 to 44 us are usual.
//
// One row of 248320 takes 3.6, 7.4, 7.0 and 5.6 us: launches, and each kernel's
// chain of loads, scans and barriers. 48 rows take 13, 26, 22 and 25: reading them
// (48 MB, 3.6 TB/s at first, then from the caches), the weights' 15 operations of
// 64 bits and LDS sums in the second, a workgroup a row in the last.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.hpp"

namespace qmr {
namespace {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kBins = kThreads;     // a thread a bin; the last: weights that round to nothing
constexpr uint32_t kPerNat = 16;         // bins of a temperature: 511 of them reach below 2^-46
constexpr uint32_t kCandidates = 8192;   // of a row, at most
constexpr uint32_t kSliceStep = 4096;
constexpr uint32_t kFew = 64;            // candidates that a wave has in its lanes
constexpr uint32_t kNone = 0xffffffffu;
constexpr int kSteps = 64;  // of an octave, in the table of powers

// Ordered as the logits are; NaN and -infinity are 0. Both zeros are one logit.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A token's place, larger for those kept first.
__device__ __forceinline__ u64 place_of(uint32_t key, uint32_t i) { return u64(key) << 32 | uint32_t(~i); }
__device__ __forceinline__ uint32_t key_at(u64 place) { return uint32_t(place >> 32); }
__device__ __forceinline__ uint32_t index_at(u64 place) { return ~uint32_t(place); }

// n weights of at most 2^shift add up to 2^62 at most; a weight and 2^52 are a
// double's whole number. Rows in bins: 2^45 at most, so that a weight of the last
// bin, below 2^-46 of the greatest, is nothing wherever it is worked out.
__host__ __device__ constexpr uint32_t shift_of(uint32_t n) {
    uint32_t bits = 12;
    while ((uint64_t(1) << bits) < n) ++bits;
    return n > kCandidates && bits < 17 ? 45 : 62 - bits;
}

// A row's, read before anything is waited for.
struct Settings {
    float temperature, min_p, top_p;
    uint32_t top_k;
    __device__ Settings(const SampleArgs &a, uint32_t row)
        : temperature(a.temperature[row]), min_p(a.min_p[row]), top_p(a.top_p[row]), top_k(a.top_k[row]) {}
};

// A row's weights and bins, from its largest and smallest logit.
struct Weights {
    uint32_t top;
    float max, half_max, per_bin;  // bins: half the distance from the largest, times per_bin
    double temperature, per_step;  // per_step: kSteps log2(e) / temperature
    const double *powers;          // 2^(i / kSteps)
    int shift;
    float min_p;

    __device__ Weights(const SampleArgs &a, const Settings &set, uint32_t top_, uint32_t least, const double *powers_)
        : top(top_), max(logit_of(top_)), temperature(set.temperature), powers(powers_), shift(shift_of(a.vocab)),
          min_p(set.min_p) {
        per_step = 1.4426950408889634 * kSteps / temperature;
        half_max = 0.5f * max;
        const float width = half_max - 0.5f * logit_of(least);
        // Narrow rows take all bins but the last, which then is empty.
        per_bin = fminf(fmaxf(2.f * kPerNat / set.temperature, width > 0.f ? float(kBins - 2) / width : 0.f), 1e38f);
    }
    __device__ bool greedy() const { return !(temperature > 0); }
    __device__ double plain(uint32_t key) const {
        if (key == top) return 1.0;
        if (max == INFINITY) return 0.0;
        return exp((double(logit_of(key)) - double(max)) / temperature);
    }
    // 2^t = 2^(n / 64) e^y, |y| <= ln 2 / 128, from a table and the exponential's
    // series: the term after the last is below 2^-54. Added to 2^52 the weight is
    // rounded to a whole number and stands in the mantissa's low bits.
    __device__ u64 whole(uint32_t key) const {
        const double t = (double(logit_of(key)) - double(max)) * per_step;
        if (!(t > -64.0 * kSteps)) return key == top ? u64(1) << shift : 0;  // also where both are infinite
        const double n = rint(t), y = (t - n) * (0.6931471805599453 / kSteps);
        const int steps = int(n);
        double e = 1.0 / 120;
        e = fma(e, y, 1.0 / 24);
        e = fma(e, y, 1.0 / 6);
        e = fma(e, y, 0.5);
        e = fma(e, y, 1.0);
        e = fma(e, y, 1.0);
        e *= powers[steps & (kSteps - 1)];
        return u64(__double_as_longlong(ldexp(e, (steps >> 6) + shift) + 0x1p52)) & ((u64(1) << 52) - 1);
    }
    __device__ bool likely(uint32_t key) const { return key == top || !(min_p > 0.f) || plain(key) >= double(min_p); }
    // Never smaller for a smaller logit, whatever rounds.
    __device__ uint32_t bin(uint32_t key) const {
        if (key == top) return 0;
        const float z = (half_max - 0.5f * logit_of(key)) * per_bin;
        return z < float(kBins - 1) ? uint32_t(z) : kBins - 1;
    }
};

// For whole workgroups, which wait before they look at it.
__device__ __forceinline__ void fill_powers(double *powers) {
    if (threadIdx.x < kSteps) powers[threadIdx.x] = exp2(double(threadIdx.x) / kSteps);
}

// The value of the lane that CTRL names in the rows of ROWS, 0 where there is
// none: steps of scans that stay in registers. Through LDS the four launches of
// a row of 248320 took 34.7 us, so 31.9: they have some 30 such scans.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 from_lane(u64 v) {
    const uint32_t low = __builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, ROWS, 0xf, false);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, ROWS, 0xf, false);
    return u64(high) << 32 | low;
}

// Each lane's join of all lanes up to it; 0 changes nothing.
template <typename Join>
__device__ __forceinline__ u64 wave_scan(u64 v, Join join) {
    v = join(v, from_lane<0x111, 0xf>(v));  // row_shr:1
    v = join(v, from_lane<0x112, 0xf>(v));
    v = join(v, from_lane<0x114, 0xf>(v));
    v = join(v, from_lane<0x118, 0xf>(v));
    v = join(v, from_lane<0x142, 0xa>(v));  // row_bcast:15
    return join(v, from_lane<0x143, 0xc>(v));  // row_bcast:31
}

struct Add {
    __device__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max {
    __device__ u64 operator()(u64 a, u64 b) const { return a > b ? a : b; }
};

// Of both values, the join over the workgroup.
template <typename Join>
__device__ __forceinline__ void block_all(u64 &a, u64 &b, u64 *room, Join join) {
    a = wave_scan(a, join);
    b = wave_scan(b, join);
    __syncthreads();
    if (threadIdx.x % 64 == 63) room[threadIdx.x / 64] = a, room[kWaves + threadIdx.x / 64] = b;
    __syncthreads();
    a = room[0], b = room[kWaves];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) a = join(a, room[w]), b = join(b, room[kWaves + w]);
}

__device__ __forceinline__ u64 block_sum(u64 v, u64 *room) {
    u64 none = 0;
    block_all(v, none, room, Add{});
    return v;
}

// Of both values, the sums up to and with each thread's.
__device__ __forceinline__ void block_scan(u64 &a, u64 &b, u64 *room) {
    a = wave_scan(a, Add{});
    b = wave_scan(b, Add{});
    __syncthreads();
    if (threadIdx.x % 64 == 63) room[threadIdx.x / 64] = a, room[kWaves + threadIdx.x / 64] = b;
    __syncthreads();
    const int wave = threadIdx.x / 64;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w) a += w < wave ? room[w] : 0, b += w < wave ? room[kWaves + w] : 0;
}

__device__ __forceinline__ u64 block_scan(u64 v, u64 *room) {
    u64 none = 0;
    block_scan(v, none, room);
    return v;
}

// Which bins the borders may fall into.
struct Bounds {
    uint32_t first, last;  // between them tokens may be kept or not; all above are
    uint32_t k_bin;        // where top k ends; kNone: it keeps all
    uint32_t k_rank;       // so many of k_bin are kept by top k
    u64 above;             // weight above `first`
    u64 above_k;           // weight above k_bin, or of all
};

// What the launches leave for each other, a row.
struct Work {
    Bounds *bounds;    // [rows]
    u64 *best;         // [rows][slices] a slice's first place
    uint32_t *least;   // [rows][slices] its smallest key, of those kept at all
    uint32_t *count;   // [rows][kBins]
    u64 *weight;       // [rows][kBins]
    uint32_t *found;   // [rows] candidates
    u64 *of_slice;     // [rows][slices][kBins] weight
    u64 *sure;         // [rows][slices] weight above the bins of the candidates
    u64 *candidates;   // [rows][kCandidates]
    uint32_t slices, slice;
};

// A row's largest and smallest key from its slices'.
__device__ __forceinline__ void extremes(const Work &w, uint32_t row, u64 &best, uint32_t &least, u64 *room) {
    best = 0;
    u64 low = 0;  // upside down
    for (uint32_t i = threadIdx.x; i < w.slices; i += kThreads) {
        best = max(best, w.best[size_t(row) * w.slices + i]);
        low = max(low, u64(~w.least[size_t(row) * w.slices + i]));
    }
    block_all(best, low, room, Max{});
    least = ~uint32_t(low);
}

// Eight logits of a thread, two runs of four (which need not lie on more than 4
// bytes) that are a workgroup's width apart; -infinity past the end. (By single
// ones the three launches that read 48 rows took 14, 28 and 23 us, so 13, 26, 22.)
constexpr uint32_t kAhead = 8;
struct Four {
    float x[4];
};
struct Ahead {
    float x[kAhead];
    static __device__ __forceinline__ uint32_t first() { return threadIdx.x * 4; }
    static __device__ __forceinline__ uint32_t at(uint32_t i, uint32_t j) { return i + j / 4 * (4 * kThreads) + j % 4; }
    __device__ __forceinline__ void load(const float *p, uint32_t i, uint32_t end) {
#pragma unroll
        for (uint32_t r = 0; r < kAhead; r += 4) {
            const uint32_t k = at(i, r);
            Four v{{-INFINITY, -INFINITY, -INFINITY, -INFINITY}};
            if (k + 4 <= end) {
                v = *reinterpret_cast<const Four *>(p + k);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j)
                    if (k + j < end) v.x[j] = p[k + j];
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) x[r + j] = v.x[j];
        }
    }
};

__global__ __launch_bounds__(kThreads) void sample_max_kernel(SampleArgs a, Work w) {
    __shared__ u64 room[2 * kWaves];
    const uint32_t row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const float *x = a.logits + size_t(row) * a.stride;
    for (uint32_t i = slice * kThreads + tid; i < kBins; i += w.slices * kThreads) {
        w.count[size_t(row) * kBins + i] = 0;
        w.weight[size_t(row) * kBins + i] = 0;
    }
    if (slice == 0 && tid == 0) w.found[row] = 0;
    u64 best = 0, low = 0;
    const uint32_t end = min((slice + 1) * w.slice, a.vocab);
    Ahead ahead;
    const uint32_t begin = slice * w.slice + Ahead::first();
    ahead.load(x, begin, end);
    for (uint32_t i = begin; i < end; i += kAhead * kThreads) {
        const Ahead now = ahead;
        ahead.load(x, i + kAhead * kThreads, end);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t key = key_of(now.x[j]);
            if (key == 0) continue;
            best = max(best, place_of(key, Ahead::at(i, j)));
            low = max(low, u64(~key));
        }
    }
    block_all(best, low, room, Max{});
    if (tid == 0) {
        w.best[size_t(row) * w.slices + slice] = best;
        w.least[size_t(row) * w.slices + slice] = ~uint32_t(low);
    }
}

__global__ __launch_bounds__(kThreads) void sample_bins_kernel(SampleArgs a, Work w) {
    __shared__ u64 room[2 * kWaves], weight[kBins];
    __shared__ double powers[kSteps];
    __shared__ uint32_t count[kBins];
    const uint32_t row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const float *x = a.logits + size_t(row) * a.stride;
    const uint32_t begin = slice * w.slice + Ahead::first(), end = min((slice + 1) * w.slice, a.vocab);
    Ahead ahead;
    ahead.load(x, begin, end);  // on their way while the slices' largest is found
    const Settings set(a, row);
    fill_powers(powers);
    u64 best;
    uint32_t least;
    extremes(w, row, best, least, room);
    const Weights of(a, set, key_at(best), least, powers);
    if (best == 0 || of.greedy()) return;
    weight[tid] = 0;
    count[tid] = 0;
    __syncthreads();
    for (uint32_t i = begin; i < end; i += kAhead * kThreads) {
        const Ahead now = ahead;
        ahead.load(x, i + kAhead * kThreads, end);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t key = key_of(now.x[j]);
            const uint32_t bin = key ? of.bin(key) : kBins - 1;
            if (bin == kBins - 1) continue;
            atomicAdd(&count[bin], 1u);
            atomicAdd(&weight[bin], of.whole(key));
        }
    }
    __syncthreads();
    const uint32_t n = count[tid];
    const u64 sum = weight[tid];
    w.of_slice[(size_t(row) * w.slices + slice) * kBins + tid] = sum;
    if (n) {
        atomicAdd(&w.count[size_t(row) * kBins + tid], n);
        atomicAdd(&w.weight[size_t(row) * kBins + tid], sum);
    }
}

// n, sum: tokens and weight of this thread's bin.
__device__ Bounds bounds_of(const Settings &set, const Weights &of, uint32_t n, u64 sum, u64 *room, u64 *found) {
    const uint32_t tid = threadIdx.x, k = set.top_k;
    const float p = set.top_p;
    u64 tokens = n, weight = sum;
    block_scan(tokens, weight, room);
    Bounds b;
    if (tid < 4) found[tid] = kNone;
    __syncthreads();
    // A border past the last bin but one is none: what is there weighs nothing.
    if (k > 0 && tokens >= k && tokens - n < k) found[0] = tid;
    if (tid == kBins - 1) found[1] = weight;
    __syncthreads();
    b.k_bin = uint32_t(found[0]);
    u64 most = found[1], least = most;
    __syncthreads();
    if (b.k_bin != kNone) {
        if (tid == b.k_bin) {
            found[1] = weight;
            found[2] = weight - sum;
            found[3] = k - (tokens - n);
        }
        __syncthreads();
        most = found[1];
        least = found[2];
        b.k_rank = uint32_t(found[3]);
        __syncthreads();
    } else {
        b.k_rank = 0;
    }
    b.above_k = least;
    b.first = b.k_bin;
    b.last = b.k_bin;
    if (p < 1.f) {
        // The first bin up to which the weight that top p asks for stands, with
        // the least and with the most that top k may keep.
        const double lo = fmax(double(p), 0.0) * double(least) * (1 - 1e-12), hi = fmax(double(p), 0.0) * double(most) * (1 + 1e-12);
        const bool in_lo = double(weight) >= lo, in_hi = double(weight) >= hi;
        const bool was_lo = tid > 0 && double(weight - sum) >= lo, was_hi = tid > 0 && double(weight - sum) >= hi;
        if (tid < 2) found[tid] = kBins - 1;
        __syncthreads();
        if (in_lo && !was_lo) found[0] = tid;
        if (in_hi && !was_hi) found[1] = tid;
        __syncthreads();
        b.first = min(b.first, uint32_t(found[0]));
        b.last = min(b.last, uint32_t(found[1]));
        __syncthreads();
    }
    if (of.min_p > 0.f) {
        // Where the weight min_p stands, give or take what the weights round to in 64
        // bits (at a temperature far above the logits that is many bins) and a bin for
        // what else rounds.
        const double nats = -log(double(fminf(of.min_p, 1.f))), off = 1e-14 * (1 + nats);
        const double bins = 0.5 * of.temperature * double(of.per_bin);
        auto bin_at = [&](double n) { return n > 0 ? n * bins < double(kBins) ? uint32_t(n * bins) : kBins : 0u; };
        const uint32_t from = bin_at(nats - off);
        b.first = min(b.first, from > 0 ? from - 1 : 0);
        b.last = min(b.last, bin_at(nats + off) + 1);
    }
    if (b.first == kNone) b.first = kBins;  // no border: all is kept
    // Few tokens down to the last border: they are all candidates.
    if (tid == 0) found[1] = kNone;
    __syncthreads();
    if (tid == b.last) found[1] = tokens;
    __syncthreads();
    if (found[1] <= kFew) b.first = 0;
    if (tid == 0) found[0] = 0;
    __syncthreads();
    if (b.first > 0 && tid == min(b.first, kBins) - 1) found[0] = weight;
    __syncthreads();
    b.above = found[0];
    __syncthreads();
    return b;
}

__global__ __launch_bounds__(kThreads) void sample_gather_kernel(SampleArgs a, Work w) {
    constexpr uint32_t kRoom = 2048;
    __shared__ u64 room[2 * kWaves], found[4], places[kRoom];
    __shared__ uint32_t here, first;
    const uint32_t row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x;
    const float *x = a.logits + size_t(row) * a.stride;
    const uint32_t begin = slice * w.slice + Ahead::first(), end = min((slice + 1) * w.slice, a.vocab);
    Ahead ahead;
    ahead.load(x, begin, end);
    const Settings set(a, row);
    const u64 own = w.of_slice[(size_t(row) * w.slices + slice) * kBins + tid], sum = w.weight[size_t(row) * kBins + tid];
    const uint32_t count = w.count[size_t(row) * kBins + tid];
    u64 best;
    uint32_t least;
    extremes(w, row, best, least, room);
    const Weights of(a, set, key_at(best), least, nullptr);  // bins alone
    if (best == 0 || of.greedy()) return;
    if (tid == 0) here = 0;
    const Bounds b = bounds_of(set, of, count, sum, room, found);
    const u64 sure = block_sum(tid < b.first ? own : u64(0), room);
    if (tid == 0) w.sure[size_t(row) * w.slices + slice] = sure;
    if (slice == 0 && tid == 0) w.bounds[row] = b;
    if (b.first == kBins) return;
    for (uint32_t i = begin; i < end; i += kAhead * kThreads) {
        const Ahead now = ahead;
        ahead.load(x, i + kAhead * kThreads, end);
#pragma unroll
        for (uint32_t j = 0; j < kAhead; ++j) {
            const uint32_t key = key_of(now.x[j]);
            const uint32_t bin = key ? of.bin(key) : kBins - 1;
            if (bin == kBins - 1 || ((bin < b.first || bin > b.last) && bin != b.k_bin)) continue;
            const uint32_t at = atomicAdd(&here, 1u);
            const u64 place = place_of(key, Ahead::at(i, j));
            if (at < kRoom) {
                places[at] = place;
            } else {
                const uint32_t to = atomicAdd(&w.found[row], 1u);
                if (to < kCandidates) w.candidates[size_t(row) * kCandidates + to] = place;
            }
        }
    }
    __syncthreads();
    const uint32_t n = min(here, kRoom);
    if (tid == 0 && n) first = atomicAdd(&w.found[row], n);
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kThreads)
        if (first + i < kCandidates) w.candidates[size_t(row) * kCandidates + first + i] = places[i];
}

// A workgroup a row from here on. Both the row and its candidates are given as
// each(f): f(place, key) for all of them, spread over the threads.
struct PickLds {
    u64 amounts[256];
    u64 some[256];       // a place of each bin
    uint32_t counts[256];
    u64 room[2 * kWaves];
    u64 found[4];
    u64 inside[4], there[4];  // of the bins, a bit each
};

// The last place, from the first one down, before which `inside(sum)` holds,
// sums of amount(key) over the places that each() gives and `in` takes, from
// `above` on (the first if it holds nowhere, 0 if there are none): a histogram
// of the first eight bits in which they differ, then of the next eight of those
// in the border's bin, until that has one.
template <typename Each, typename In, typename Amount, typename Inside>
__device__ u64 border_of(PickLds &lds, Each each, In in, Amount amount, Inside inside, u64 above) {
    const uint32_t tid = threadIdx.x;
    u64 top = 0, rest = 0;  // rest: the smallest, upside down
    each([&](u64 place) {
        if (in(place)) top = max(top, place), rest = max(rest, ~place);
    });
    block_all(top, rest, lds.room, Max{});
    rest = ~rest;
    if (top == 0) return 0;
    if (top == rest) return top;
    // The window's bits, and those above it.
    const int high = 64 - __clzll(static_cast<long long>(top ^ rest));
    int width = min(8, high), low = high - width;
    u64 prefix = high < 64 ? top >> high : 0;
    for (;;) {
        __syncthreads();
        if (tid < 256) lds.amounts[tid] = 0, lds.some[tid] = 0, lds.counts[tid] = 0;
        __syncthreads();
        each([&](u64 place) {
            if (!in(place) || place >> low >> width != prefix) return;
            const uint32_t bin = 255 - uint32_t(place >> low & ((1u << width) - 1));  // the largest first
            atomicAdd(&lds.amounts[bin], amount(key_at(place)));
            atomicAdd(&lds.counts[bin], 1u);
            lds.some[bin] = place;
        });
        __syncthreads();
        const u64 sum = tid < 256 ? lds.amounts[tid] : 0, before = above + block_scan(sum, lds.room) - sum;
        // inside() holds up to some of the bins, of which the last is taken.
        if (tid < 256) {
            const bool there = lds.counts[tid] != 0;
            const u64 all = __ballot(there), some = __ballot(there && inside(before));
            if (tid % 64 == 0) lds.there[tid / 64] = all, lds.inside[tid / 64] = some;
            lds.amounts[tid] = before;
        }
        __syncthreads();
        uint32_t at = 0;
#pragma unroll
        for (int w = 3; w >= 0; --w)
            if (lds.there[w]) at = 64 * w + __ffsll(lds.there[w]) - 1;  // the first, if it holds for none
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (lds.inside[w]) at = 64 * w + 63 - __clzll(lds.inside[w]);
        if (lds.counts[at] == 1) return lds.some[at];
        above = lds.amounts[at];
        prefix = prefix << width | (255 - at);
        width = min(8, low);
        low -= width;
    }
}

__device__ __forceinline__ u64 target_of(const SampleArgs &a, uint32_t row, u64 total) {
    const double u = fmin(fmax(double(a.uniform[row]), 0.0), 1.0);
    return min(u64(u * double(total)), total - 1);
}

__device__ __forceinline__ u64 lane_of(u64 v, uint32_t l) {
    return u64(__builtin_amdgcn_readlane(uint32_t(v >> 32), l)) << 32 | uint32_t(__builtin_amdgcn_readlane(uint32_t(v), l));
}

// border_of for places of a wave's first n lanes, `in` and amount theirs: each
// lane adds up what stands before it.
template <typename Inside>
__device__ __forceinline__ u64 border_of_few(uint32_t n, u64 place, bool in, u64 amount, Inside inside, u64 above) {
    const u64 own = in ? place : 0, weight = in ? amount : 0;
    u64 before = above, top = 0;
    for (uint32_t j = 0; j < n; ++j) {
        const u64 other = lane_of(own, j);
        before += other > place ? lane_of(weight, j) : 0;
        top = max(top, other);
    }
    const u64 last = lane_of(wave_scan(in && inside(before) ? ~place : 0, Max{}), 63);
    return last ? ~last : top;
}

// Draws from what tokens begin..end-1 keep: weight(i), 0 if it is not
// kept; `before` of the weight stands before them, and `target` falls into them.
template <typename Weight>
__device__ void draw(const SampleArgs &a, uint32_t row, PickLds &lds, uint32_t begin, uint32_t end, Weight weight, u64 before, u64 target,
                     u64 total) {
    constexpr uint32_t kEach = 8;  // of a thread, in sequence
    for (uint32_t base = begin; base < end; base += kEach * kThreads) {
        const uint32_t first = base + threadIdx.x * kEach;
        u64 own[kEach], sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            own[j] = first + j < end ? weight(first + j) : 0;
            sum += own[j];
        }
        u64 up_to = before + block_scan(sum, lds.room);
        if (threadIdx.x == kThreads - 1) lds.found[3] = up_to;
        if (up_to > target && up_to - sum <= target) {
            up_to -= sum;
#pragma unroll
            for (uint32_t j = 0; j < kEach; ++j) {
                up_to += own[j];
                if (up_to > target && up_to - own[j] <= target) {
                    a.tokens[row] = first + j;
                    a.probs[row] = float(double(own[j]) / double(total));
                }
            }
        }
        __syncthreads();
        before = lds.found[3];
        if (before > target) return;
        __syncthreads();
    }
}

// `whole`: rows that fit the candidates' LDS, with no launch before this one.
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a, Work w, bool whole) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    u64 *places = reinterpret_cast<u64 *>(dynamic);            // [kCandidates]
    u64 *of_slices = places + (whole ? a.vocab : kCandidates);  // [slices]
    __shared__ PickLds lds;
    __shared__ double powers[kSteps];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float *x = a.logits + size_t(row) * a.stride;
    const Settings set(a, row);
    Bounds b{};  // not there for rows that return below
    uint32_t found = 0;
    if (!whole) {
        b = w.bounds[row];
        found = w.found[row];
    }
    fill_powers(powers);
    u64 best = 0;
    uint32_t least = 0, n = 0;
    if (whole) {
        n = a.vocab;
        u64 low = 0;
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t key = key_of(x[i]);
            const u64 place = key ? place_of(key, i) : 0;
            places[i] = place;
            best = max(best, place);
            if (key) low = max(low, u64(~key));
        }
        block_all(best, low, lds.room, Max{});
        least = ~uint32_t(low);
    } else {
        extremes(w, row, best, least, lds.room);
    }
    const Weights of(a, set, key_at(best), least, powers);
    if (best == 0 || of.greedy()) {
        if (tid == 0) {
            a.tokens[row] = best ? index_at(best) : kNone;
            a.probs[row] = best ? 1.f : 0.f;
        }
        return;
    }
    if (!whole) n = b.first < kBins ? found : 0;
    const bool listed = whole || n <= kCandidates;
    // Few candidates (top k, or a narrow row): every wave has them in its lanes,
    // and no border takes a barrier. Three of a row of 248320, none above them: this
    // launch takes 5.6 us, where it took 10.7.
    const bool few = !whole && n <= kFew;
    if (!whole && listed && !few) {
        for (uint32_t i = tid; i < n; i += kThreads) places[i] = w.candidates[size_t(row) * kCandidates + i];
    }
    __syncthreads();
    auto each = [&](auto f) {
        if (listed) {
            for (uint32_t i = tid; i < n; i += kThreads)
                if (places[i]) f(places[i]);
        } else {
            for (uint32_t i = tid; i < a.vocab; i += kThreads) {
                const uint32_t key = key_of(x[i]);
                if (key) f(place_of(key, i));
            }
        }
    };
    const bool bins = listed && !whole;  // the places are those of some bins

    const uint32_t k = set.top_k;
    const float p = set.top_p;
    u64 k_border = 0, p_border = 0, kept_by_k = 0, few_place = 0, few_weight = 0;
    if (few) {
        const uint32_t l = tid % 64;
        const u64 place = l < n ? w.candidates[size_t(row) * kCandidates + l] : 0;
        const uint32_t key = key_at(place), bin = place ? of.bin(key) : kNone;
        const u64 amount = place ? of.whole(key) : 0;
        if (b.k_bin != kNone) {
            k_border = border_of_few(n, place, bin == b.k_bin, 1, [&](u64 before) { return before < b.k_rank; }, 0);
            kept_by_k = lane_of(wave_scan(bin == b.k_bin && place >= k_border ? amount : 0, Add{}), 63);
        }
        if (p < 1.f) {
            const double target = fmax(double(p), 0.0) * double(kept_by_k + b.above_k);
            p_border = border_of_few(n, place, place >= k_border && bin <= b.last, amount,
                                     [&](u64 before) { return double(before) < target; }, b.above);
        }
        const bool kept = place && place >= max(k_border, p_border) && bin >= b.first && bin <= b.last && of.likely(key);
        few_place = place;
        few_weight = kept ? amount : 0;
        if (b.first == 0) {  // no other token is kept
            const u64 total = lane_of(wave_scan(few_weight, Add{}), 63), target = target_of(a, row, total);
            u64 before = 0;
            for (uint32_t j = 0; j < n; ++j)
                before += index_at(lane_of(few_place, j)) < index_at(place) ? lane_of(few_weight, j) : 0;
            if (tid < 64 && kept && before <= target && before + few_weight > target) {
                a.tokens[row] = index_at(place);
                a.probs[row] = float(double(few_weight) / double(total));
            }
            return;
        }
    }
    // Top k.
    if (!few && (bins ? b.k_bin != kNone : k > 0 && k < a.vocab)) {
        const u64 rank = bins ? b.k_rank : k;
        k_border = border_of(
            lds, each, [&](u64 place) { return !bins || of.bin(key_at(place)) == b.k_bin; }, [](uint32_t) { return u64(1); },
            [&](u64 before) { return before < rank; }, 0);
    }
    // Top p, of what top k keeps.
    if (!few && p < 1.f) {
        u64 sum = 0;
        if (!bins || b.k_bin != kNone)
            each([&](u64 place) {
                if (place >= k_border && (!bins || of.bin(key_at(place)) == b.k_bin)) sum += of.whole(key_at(place));
            });
        kept_by_k = block_sum(sum, lds.room) + (bins ? b.above_k : 0);
        const double target = fmax(double(p), 0.0) * double(kept_by_k);
        p_border = border_of(
            lds, each, [&](u64 place) { return place >= k_border && (!bins || of.bin(key_at(place)) <= b.last); },
            [&](uint32_t key) { return of.whole(key); }, [&](u64 before) { return double(before) < target; }, bins ? b.above : 0);
    }
    const u64 border = max(k_border, p_border);
    auto weight = [&](uint32_t i) -> u64 {
        const uint32_t key = key_of(x[i]);
        return key && place_of(key, i) >= border && of.likely(key) ? of.whole(key) : 0;
    };
    if (!bins) {
        u64 sum = 0;
        each([&](u64 place) {
            if (place >= border && of.likely(key_at(place))) sum += of.whole(key_at(place));
        });
        const u64 total = block_sum(sum, lds.room);
        draw(a, row, lds, 0, a.vocab, weight, 0, target_of(a, row, total), total);
        return;
    }
    // The slice that the number falls into.
    for (uint32_t s = tid; s < w.slices; s += kThreads) of_slices[s] = w.sure[size_t(row) * w.slices + s];
    __syncthreads();
    if (few) {
        if (tid < 64 && few_weight) atomicAdd(&of_slices[index_at(few_place) / w.slice], few_weight);
    } else {
        each([&](u64 place) {
            const uint32_t key = key_at(place), bin = of.bin(key);
            if (place >= border && bin >= b.first && bin <= b.last && of.likely(key))
                atomicAdd(&of_slices[index_at(place) / w.slice], of.whole(key));
        });
    }
    __syncthreads();
    u64 sum = 0;
    for (uint32_t s = tid; s < w.slices; s += kThreads) sum += of_slices[s];
    const u64 total = block_sum(sum, lds.room), target = target_of(a, row, total);
    u64 before = 0;
    for (uint32_t base = 0; base < w.slices; base += kThreads) {
        const u64 own = base + tid < w.slices ? of_slices[base + tid] : 0, up_to = before + block_scan(own, lds.room);
        if (own && up_to > target && up_to - own <= target) {
            lds.found[0] = base + tid;
            lds.found[1] = up_to - own;
        }
        if (tid == kThreads - 1) lds.found[2] = up_to;
        __syncthreads();
        before = lds.found[2];
        if (before > target) break;
        __syncthreads();
    }
    const uint32_t slice = uint32_t(lds.found[0]);
    before = lds.found[1];
    __syncthreads();
    draw(a, row, lds, slice * w.slice, min((slice + 1) * w.slice, a.vocab), weight, before, target, total);
}

size_t row_bytes(uint32_t slices) {
    return size_t(slices) * (8 + 4 + 8 + kBins * 8) + kBins * 12 + 4 + size_t(kCandidates) * 8 + sizeof(Bounds) + 64;
}

}  // namespace

// Slices of at least 4096 logits, eight a thread, and more where there are rows
// enough to fill the chip four times over. A row of 248320 in slices of 2048 and
// 1024 took 36 and 39 us where it took 35 (its bins are added up across slices); 48
// rows that may fill it twice and eight times 118 and 94 us for 94.
SamplePlan plan_sample(const SampleArgs &a, const DeviceLimits &lim, size_t limit) {
    SamplePlan pl;
    pl.whole = a.vocab <= kCandidates;
    pl.rows = a.rows;
    if (pl.whole) return pl;
    pl.slice = kSliceStep;
    const uint64_t most = uint64_t(lim.num_cus) * 4;
    while (uint64_t(a.rows) * ((a.vocab + pl.slice - 1) / pl.slice) > most && pl.slice < a.vocab) pl.slice += kSliceStep;
    limit = std::min(limit, size_t(64) << 20);
    while (row_bytes((a.vocab + pl.slice - 1) / pl.slice) > limit) pl.slice *= 2;
    pl.slices = (a.vocab + pl.slice - 1) / pl.slice;
    pl.rows = uint32_t(std::min<uint64_t>(a.rows, limit / row_bytes(pl.slices)));
    pl.workspace = pl.rows * row_bytes(pl.slices);
    return pl;
}

hipError_t launch_sample_logits(const SampleArgs &all, const SamplePlan &pl, void *workspace, hipStream_t stream) {
    SampleArgs a = all;
    for (uint32_t row = 0; row < all.rows; row += pl.rows) {
        const uint32_t n = std::min(pl.rows, all.rows - row);
        a.logits = all.logits + size_t(row) * all.stride;
        a.temperature = all.temperature + row;
        a.top_k = all.top_k + row;
        a.top_p = all.top_p + row;
        a.min_p = all.min_p + row;
        a.uniform = all.uniform + row;
        a.tokens = all.tokens + row;
        a.probs = all.probs + row;
        a.rows = n;
        Work w{};
        w.slices = pl.slices;
        w.slice = pl.slice;
        uint32_t lds = all.vocab * 8;
        if (!pl.whole) {
            unsigned char *at = static_cast<unsigned char *>(workspace);
            auto take = [&](size_t bytes) {
                unsigned char *p = at;
                at += (bytes + 7) / 8 * 8;
                return p;
            };
            const size_t slices = size_t(n) * pl.slices;
            w.bounds = reinterpret_cast<Bounds *>(take(n * sizeof(Bounds)));
            w.best = reinterpret_cast<u64 *>(take(slices * 8));
            w.weight = reinterpret_cast<u64 *>(take(size_t(n) * kBins * 8));
            w.of_slice = reinterpret_cast<u64 *>(take(slices * kBins * 8));
            w.sure = reinterpret_cast<u64 *>(take(slices * 8));
            w.candidates = reinterpret_cast<u64 *>(take(size_t(n) * kCandidates * 8));
            w.least = reinterpret_cast<uint32_t *>(take(slices * 4));
            w.count = reinterpret_cast<uint32_t *>(take(size_t(n) * kBins * 4));
            w.found = reinterpret_cast<uint32_t *>(take(size_t(n) * 4));
            lds = kCandidates * 8 + pl.slices * 8;
            const dim3 grid(pl.slices, n);
            sample_max_kernel<<<grid, kThreads, 0, stream>>>(a, w);
            sample_bins_kernel<<<grid, kThreads, 0, stream>>>(a, w);
            sample_gather_kernel<<<grid, kThreads, 0, stream>>>(a, w);
        }
        const hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(sample_pick_kernel), lds);
        if (e != hipSuccess) return e;
        sample_pick_kernel<<<n, kThreads, lds, stream>>>(a, w, pl.whole);
    }
    return hipGetLastError();
}

}  // namespace qmr
