// Linear attention over chunks of 32 tokens, on the matrix cores (attn_linear.hip
// says what is computed). In a chunk, with G the running sum of the log decays
// in it, S the state before it and c the factor that normalises a row:
//
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j  (j < i)          T = (I + A)^-1
//   R_i  = beta_i (v_i - e^(G_i) S^T k_i)                    U = T R
//   M_ij = scale e^(G_i - G_j) q_i . k_j  (j <= i)
//   o_i  = scale e^(G_i) S^T q_i + (M U)_i
//   S'   = e^(G_32) S + sum_j e^(G_32 - G_j) k_j U_j^T
//
// (without the delta rule U = V). Exponents are differences that are never
// positive where decays do not grow, so nothing overflows on the way.
//
// Three launches. linear_prepare_kernel has a workgroup a chunk and key head:
// everything that does not depend on the state, all chunks at once, left in the
// workspace as the operands that the matrix instructions take (4100 tokens of 16
// key and 48 value heads of 128: 53 us, 68 MB read and 122 MB written, 3.6 TB/s,
// bound by memory and the splits' vector work alike). linear_scan_kernel
// goes through a sequence's chunks: a workgroup has some 16-column tiles of a
// value head's state, a wave one, in its accumulators; the next chunk's operands
// come to LDS meanwhile (bound by a chunk's chain of products and splits: 1.7 us
// a chunk, 219 us for those tokens, of which 84 matrix instructions are a third).
// linear_norm_kernel norms the outputs, whose rows the workgroups of a head share
// (49 us for those: 302 MB at 6.2 TB/s, much of it from the last-level cache).
//
// Columns of the state do not meet until the output norm, so a wave needs
// nothing of another one, and S, R and U need not leave its registers: a product
// leaves column n of its 16x16 tiles in lanes n, n + 16, n + 32 and n + 48, four
// rows each, and that is where the next product takes its operand from if its
// left side counts the rows in the same order (slot 8g + 4h + i of 32 is row
// 16h + 4g + i). The operands in the workspace do.
//
// Precision: FP32 values are two f16 terms, the second what the first leaves
// (22 bits), a product three matrix instructions (the product of the two second
// terms, 2^-22 of it, is left out); sums are FP32. One FP32 matrix instruction
// would take 5.3 times as long as those three. Rows of q and k are scaled by
// powers of two to 2^3..2^4, a column of S, R and U to at most 2^15, so that the
// terms stay among the normal f16 numbers as far as they matter: an element of R
// and U is off by 2^-30 of the largest of its column and chunk where that is more
// than its own 22 bits, one of S by 2^-30 of its column's, and one of M by 2^-29
// of scale |q_i| |k|, k the longest key up to i as far as it is not yet forgotten.
//
// The chunk's algebra has products of tokens with later ones, by zero: a value
// that is not finite would reach tokens before it. A chunk that has some, or
// whose T is not small (keys longer than 1, where the recurrence itself is not
// stable), or, with the delta rule, that has a key longer than kLongest, is done
// token after token by the same waves.
#include <hip/hip_runtime.h>

#include <algorithm>

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
using wave::dma16;
using wave::dma4;
using wave::f2;
using wave::f4;
using wave::h2;
using wave::h8;
using wave::kRsrcWord3;
using wave::lds_barrier;
using wave::two_halves;
using wave::u4;
using wave::wait_dma;
using wave::wave_lds_sync;

constexpr uint32_t kChunk = 32;
constexpr uint32_t kTile = 1024;         // bytes of one f16 operand of 16 x 32
constexpr uint32_t kOut = 0x80000000u;   // buffer offset past every range
constexpr float kForget = -1000.f;       // e^-1000 is 0 in FP32 whatever it meets
constexpr int kScore = 2;                // M's entries are products of scaled rows by 2^-kScore, and a row's own power
constexpr int kSolve = 4;                // T's entries are by 2^kSolve
constexpr int kRoom = 16;                // products with S and U, of scaled rows, are by 2^-kRoom: S and U may be near FP32's largest

// A chunk's operands. Of a key head: Q [2 tiles of 16 tokens][blocks][2 terms],
// and K. Of a value head: M [2][2 terms], scalars, T as M (delta rule).
constexpr uint32_t kScalars = 4 * kTile;  // where they stand
enum Scalar : uint32_t { kBeta = 0, kX = 32, kQ = 64, kM = 96, kU = 128, kWhole = 160, kMost = 161, kWild = 162 };

__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Under the delta rule R has S^T k: a key of this length takes as much from the
// other tokens' part in R as a value that many times the state.
constexpr float kLongest = 16.f;

// Two terms of each side.
__device__ __forceinline__ f4 mfma3(u4 ah, u4 al, u4 bh, u4 bl, f4 c) {
    c = mfma(al, bh, c);
    c = mfma(ah, bl, c);
    return mfma(ah, bh, c);
}

// Eight values as terms, to nearest both. `minus`: -1 that the compiler does
// not see through, for the instruction that multiplies an f16 into FP32.
__device__ __forceinline__ void terms(const float (&x)[8], float minus, u4 &hi, u4 &lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 h = __builtin_convertvector((f2{x[2 * i], x[2 * i + 1]}), h2);
        hi[i] = __builtin_bit_cast(uint32_t, h);
        lo[i] = two_halves(__builtin_fmaf(float(h[0]), minus, x[2 * i]), __builtin_fmaf(float(h[1]), minus, x[2 * i + 1]));
    }
}

// So many times: a matrix instruction, then others that may run beside it.
template <int TIMES, int VALU, int LDS>
__device__ __forceinline__ void in_turn() {
#pragma unroll
    for (int i = 0; i < TIMES; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (LDS > 0) __builtin_amdgcn_sched_group_barrier(0x100, LDS, 0);
        if constexpr (VALU > 0) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
    }
}

// The largest of a column's four lanes.
__device__ __forceinline__ float column_max(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float column_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

__device__ __forceinline__ int exponent(float x) {  // |x| < 2^it; 0 for what is not finite
    return __builtin_amdgcn_frexp_expf(x);
}

__device__ __forceinline__ u4 rsrc_of(const void *p, uint32_t bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    return u4{uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(at))),
              uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(at >> 32) & 0xFFFFu)),
              uint32_t(__builtin_amdgcn_readfirstlane(bytes)), kRsrcWord3};
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const float *p, uint32_t bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    const uint64_t same = uint64_t(__builtin_amdgcn_readfirstlane(uint32_t(at >> 32))) << 32 | uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(at)));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<float *>(same), 0, __builtin_amdgcn_readfirstlane(int(bytes)), kRsrcWord3);
}

// Which chunks a pass has, and where their operands are.
struct Pass {
    unsigned char *operands;  // [chunk][k_heads * k_bytes + v_heads * v_bytes]
    float *from, *to;         // a state [v_heads][dk][dv] and its scales that the last pass left, or this one leaves; the last one leaves none
    uint32_t first, last;
    uint32_t k_bytes, v_bytes;
    uint32_t columns;         // workgroups of a head

    __device__ unsigned char *of_key(const LinearArgs &a, uint32_t chunk, uint32_t h) const {
        return operands + size_t(chunk - first) * (size_t(a.k_heads) * k_bytes + size_t(a.v_heads) * v_bytes) + size_t(h) * k_bytes;
    }
    __device__ unsigned char *of_value(const LinearArgs &a, uint32_t chunk, uint32_t h) const {
        return of_key(a, chunk, a.k_heads) + size_t(h) * v_bytes;
    }
};

constexpr int kPrepare = 256;

template <int KB>
struct PrepareLds {
    static constexpr uint32_t kPitch = 36;                      // floats of a row of 32
    static constexpr uint32_t kSquare = 32 * kPitch * 4;
    static constexpr uint32_t kRows = 0;                        // [4][32] FP32 of rows
    static constexpr uint32_t kRest = kRows + 4 * 32 * 4;       // terms of q and k, then what follows
    static constexpr uint32_t kTerms = 4 * kTile * KB;          // of q, or of k
    static constexpr uint32_t kGram = kRest;                    // q k, k k
    static constexpr uint32_t kWaves = kGram + 2 * kSquare;     // each wave's own
    static constexpr uint32_t kG = kSquare, kWave = kG + 32 * 8 + 2 * 32 * 4;
    static constexpr uint32_t kEnd = kWaves + 4 * kWave;
    static constexpr uint32_t kBytes = kRest + 2 * kTerms > kEnd ? kRest + 2 * kTerms : kEnd;
};

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// T = (I + A)^-1 in the place of A [32][pitch], a wave's: two blocks of
// 16 on the diagonal, a lane a column, then T21 = -T22 (A21 T11) in FP32
// matrix instructions. (A lane a column of all 32 takes 496 products in place
// of 120, and each row waits for the one before it.)
template <uint32_t PITCH>
__device__ __forceinline__ void invert(float *A) {
    const uint32_t l = threadIdx.x % 64, g = l / 16, m = l % 16, at = l / 16 % 2 * 16;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float even = uint32_t(i) == m ? 1.f : 0.f, odd = 0.f;
#pragma unroll
        for (int c = 0; c < i; ++c) {
            const float v = A[(at + i) * PITCH + at + c];
            if (c % 2) odd = fmaf(-v, x[c], odd);
            else even = fmaf(-v, x[c], even);
        }
        x[i] = even + odd;
    }
    float *T = A;
    if (l < 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) T[(at + i) * PITCH + at + m] = x[i];
    }
    wave_lds_sync();
    // Step s has columns 4g + s of the left side and those rows of the right.
    const f4 a21 = *reinterpret_cast<const f4 *>(A + (16 + m) * PITCH + 4 * g);
    const f4 t22 = *reinterpret_cast<const f4 *>(T + (16 + m) * PITCH + 16 + 4 * g);
    f4 y{}, z{};
#pragma unroll
    for (int s = 0; s < 4; ++s) y = mfma4(a21[s], T[(4 * g + s) * PITCH + m], y);
#pragma unroll
    for (int s = 0; s < 4; ++s) z = mfma4(t22[s], y[s], z);
#pragma unroll
    for (int i = 0; i < 4; ++i) T[(16 + 4 * g + i) * PITCH + m] = -z[i];
    wave_lds_sync();
}

template <int KB, bool DELTA>
__global__ __launch_bounds__(kPrepare) void linear_prepare_kernel(LinearArgs a, Pass pass) {
    extern __shared__ __align__(16) unsigned char lds[];
    using L = PrepareLds<KB>;
    float *gram = reinterpret_cast<float *>(lds + L::kGram);
    float *rows = reinterpret_cast<float *>(lds + L::kRows);  // c of k, c of q, bad
    unsigned char *rest = lds + L::kRest;

    const uint32_t chunk = pass.first + blockIdx.x, kh = blockIdx.y, tid = threadIdx.x;
    const uint32_t l = tid % 64, w = __builtin_amdgcn_readfirstlane(tid / 64), g = l / 16, m = l % 16;
    uint32_t s, part, first, count;
    if (!seq::part_of(a.seq, chunk, kChunk, s, part)) return;
    seq::tokens_of(a.seq, s, first, count);
    const uint32_t t0 = part * kChunk, n = min(kChunk, count - t0);
    const size_t token0 = size_t(first) + t0;
    unsigned char *out = pass.of_key(a, chunk, kh);

    // Eight lanes a token: 4-dim pieces seg, seg + 8, ..
    {
        const uint32_t i = tid / 8, seg = tid % 8;
        const bool real = i < n;
        const float *qr = a.q + (token0 + i) * a.q_stride + size_t(kh) * a.dk;
        const float *kr = a.k + (token0 + i) * a.k_stride + size_t(kh) * a.dk;
        Quad x[2][KB];
#pragma unroll
        for (int u = 0; u < KB; ++u) {
            const uint32_t d = (seg + 8 * u) * 4;
            x[0][u] = quad_at(qr + d, real && d < a.dk);
            x[1][u] = quad_at(kr + d, real && d < a.dk);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = 0.f, sum = 0.f;
#pragma unroll
            for (int u = 0; u < KB; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    top = fmaxf(top, fabsf(x[r][u].x[j]));
                    sum = fmaf(x[r][u].x[j], x[r][u].x[j], sum);
                }
#pragma unroll
            for (int d = 1; d < 8; d *= 2) {
                top = fmaxf(top, __shfl_xor(top, d));
                sum += __shfl_xor(sum, d);
            }
            const int p = top > 0.f ? min(4 - exponent(top), 120) : 0;  // the largest to 2^3..2^4
            const float f = a.qk_eps > 0.f ? 1.f / sqrtf(sum + a.qk_eps) : 1.f;
            if (seg == 0) {
                rows[32 * (1 - r) + i] = top > 0.f ? ldexpf(f, -p) : 0.f;
                // (finite, and with the delta rule keys of up to kLongest)
                rows[64 + 32 * r + i] = sum * f * f < (DELTA && r == 1 ? kLongest * kLongest : INFINITY) ? 0.f : 1.f;
            }
            const float by = ldexpf(1.f, p);
#pragma unroll
            for (int u = 0; u < KB; ++u) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float b0 = x[r][u].x[2 * j] * by, b1 = x[r][u].x[2 * j + 1] * by;
                    const h2 h = __builtin_convertvector((f2{b0, b1}), h2);
                    hi[j] = __builtin_bit_cast(uint32_t, h);
                    lo[j] = two_halves(b0 - float(h[0]), b1 - float(h[1]));
                }
                const uint32_t at = ((i / 16 * KB + u) * 2) * kTile + (seg % 4 * 16 + i % 16) * 16 + seg / 4 * 8;
                unsigned char *to = rest + r * L::kTerms + at;
                *reinterpret_cast<uint2 *>(to) = uint2{hi[0], hi[1]};
                *reinterpret_cast<uint2 *>(to + kTile) = uint2{lo[0], lo[1]};
                to = out + r * L::kTerms + at;
                *reinterpret_cast<uint2 *>(to) = uint2{hi[0], hi[1]};
                *reinterpret_cast<uint2 *>(to + kTile) = uint2{lo[0], lo[1]};
            }
        }
    }
    __syncthreads();

    // Products of rows: tiles (0, 0), (1, 0), (1, 1).
    const uint32_t rt = w > 0, ct = w == 2;
    f4 qk{}, kk{};
    if (w < 3) {
        auto term = [&](uint32_t r, uint32_t tile, uint32_t kb, uint32_t hl) {
            return *reinterpret_cast<const u4 *>(rest + r * L::kTerms + ((tile * KB + kb) * 2 + hl) * kTile + l * 16);
        };
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const u4 bh = term(1, ct, kb, 0), bl = term(1, ct, kb, 1);
            qk = mfma3(term(0, rt, kb, 0), term(0, rt, kb, 1), bh, bl, qk);
            if constexpr (DELTA) kk = mfma3(term(1, rt, kb, 0), term(1, rt, kb, 1), bh, bl, kk);
        }
    }
    __syncthreads();  // the terms give way to the products
    if (w < 3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gram[(rt * 16 + 4 * g + i) * L::kPitch + ct * 16 + m] = qk[i];
            if constexpr (DELTA) gram[(32 + rt * 16 + 4 * g + i) * L::kPitch + ct * 16 + m] = kk[i];
        }
    }
    __syncthreads();

    // A wave a value head of this key head. Lanes have a token each (twice), and
    // then of rows m and 16 + m the columns 4g.. and 16 + 4g.., as operands do.
    unsigned char *own = lds + L::kWaves + w * L::kWave;
    float *A = reinterpret_cast<float *>(own);  // then T
    double *Gs = reinterpret_cast<double *>(own + L::kG);
    float *by_row = reinterpret_cast<float *>(own + L::kG + 32 * 8);
    int *long_row = reinterpret_cast<int *>(by_row + 32);
    const uint32_t group = a.v_heads / a.k_heads, j = l % 32;
    const float ck = rows[j], cq = rows[32 + j];
    const bool bad_rows = rows[64 + j] + rows[96 + j] > 0.f;
    // Up to its token, a row's longest key as an exponent.
    const float length = ck > 0.f ? float(exponent(ck)) : -INFINITY;
    float longest = length;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const float before = __shfl_up(longest, d, 32);
        if (j >= uint32_t(d)) longest = fmaxf(longest, before);
    }
    f4 cks[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) cks[half] = *reinterpret_cast<const f4 *>(rows + 16 * half + 4 * g);
    for (uint32_t vh = w; vh < group; vh += kPrepare / 64) {
        const uint32_t h = kh * group + vh;
        const bool real = j < n;
        float step = real ? log_decay(a, token0 + j, h) : 0.f;
        step = step < kForget ? kForget : step;
        const float beta = DELTA ? (real ? sigmoid(a.b[(token0 + j) * a.b_stride + h]) : 0.f) : 1.f;
        double G = step;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const double before = __shfl_up(G, d, 32);
            if (j >= uint32_t(d)) G += before;
        }
        const double all = __shfl(G, 31, 32);
        // M's rows are by 2^-p: no key up to theirs, decayed as far as they see it,
        // is longer than 2^p. A later key has no part in it, nor one that is forgotten,
        // down to 2^-96 of the longest (where e^(G_i - G_j) leaves FP32's normal numbers).
        const float nats = float(G) * 1.4426950408889634f;
        float seen = length - nats;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const float before = __shfl_up(seen, d, 32);
            if (j >= uint32_t(d)) seen = fmaxf(seen, before);
        }
        const int p = longest > -INFINITY ? int(fmaxf(ceilf(seen + nats), longest - 96.f)) : 0;
        Gs[j] = G;
        by_row[j] = beta * ck;
        long_row[j] = p;
        wave_lds_sync();
        unsigned char *to = pass.of_value(a, chunk, h);
        bool bad = bad_rows;
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {  // rows
            const uint32_t i = 16 * half + m;
            const double Gi = Gs[i];
            const float of_row = by_row[i];
            const int p_row = long_row[i];
            float M[8];
#pragma unroll
            for (uint32_t c = 0; c < 2; ++c) {  // columns
                const uint32_t j0 = 16 * c + 4 * g;
                f4 below{};
#pragma unroll
                for (uint32_t q = 0; q < 4; ++q) M[4 * c + q] = 0.f;
                if (c <= half) {
                    const f4 qk = *reinterpret_cast<const f4 *>(gram + i * L::kPitch + j0);
                    f4 kk{};
                    if constexpr (DELTA) kk = *reinterpret_cast<const f4 *>(gram + (32 + i) * L::kPitch + j0);
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) {
                        const float e = i >= j0 + q ? expf(float(Gi - Gs[j0 + q])) : 0.f;
                        M[4 * c + q] = i >= j0 + q ? qk[q] * ldexpf(cks[c][q], -kScore - p_row) * e : 0.f;
                        below[q] = i > j0 + q ? of_row * cks[c][q] * kk[q] * e : 0.f;
                        bad |= !(fabsf(M[4 * c + q]) < 60000.f);
                    }
                }
                if constexpr (DELTA) *reinterpret_cast<f4 *>(A + i * L::kPitch + j0) = below;
            }
            u4 hi, lo;
            terms(M, -1.f, hi, lo);
            *reinterpret_cast<u4 *>(to + 2 * half * kTile + l * 16) = hi;
            *reinterpret_cast<u4 *>(to + (2 * half + 1) * kTile + l * 16) = lo;
        }
        float rows_of_t = 1.f;
        if constexpr (DELTA) {
            wave_lds_sync();
            invert<L::kPitch>(A);
            rows_of_t = 0.f;
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                const uint32_t i = 16 * half + m;
                float x[8], sum = 0.f;
#pragma unroll
                for (uint32_t c = 0; c < 2; ++c) {
                    const f4 t = c <= half ? *reinterpret_cast<const f4 *>(A + i * L::kPitch + 16 * c + 4 * g) : f4{};
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) {
                        bad |= !(fabsf(t[q]) < 2.f);
                        sum += fabsf(t[q]);
                        x[4 * c + q] = ldexpf(t[q], kSolve);
                    }
                }
                rows_of_t = fmaxf(rows_of_t, column_sum(sum));
                u4 hi, lo;
                terms(x, -1.f, hi, lo);
                unsigned char *t = to + kScalars + kTile + 2 * half * kTile + l * 16;
                *reinterpret_cast<u4 *>(t) = hi;
                *reinterpret_cast<u4 *>(t + kTile) = lo;
            }
#pragma unroll
            for (int d = 1; d < 16; d *= 2) rows_of_t = fmaxf(rows_of_t, __shfl_xor(rows_of_t, d));
        }
        const float grown = expf(float(G)), left = expf(float(all - G)), whole = expf(float(all));
        const float of_q = ldexpf(a.scale * grown * cq, kRoom), of_x = beta * grown * ck, of_u = left * ck;
        const float of_m = ldexpf(a.scale * cq, kScore + p + kRoom);
        bad |= !(fabsf(of_q) < INFINITY) || !(fabsf(of_x) < INFINITY) || !(of_u < INFINITY) || !(fabsf(of_m) < INFINITY) ||
               !(whole < INFINITY);
        float most = of_u;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        const bool wild = __ballot(bad) != 0;
        float *scalars = reinterpret_cast<float *>(to + kScalars);
        if (l < 32) {
            scalars[kBeta + j] = beta;
            scalars[kX + j] = of_x;
            scalars[kQ + j] = of_q;
            scalars[kM + j] = of_m;
            scalars[kU + j] = of_u;
        }
        if (l == 0) {
            scalars[kWhole] = whole;
            // What a chunk adds to a column of the state, at most, by the largest
            // of R (32 tokens, dims up to 2^4).
            scalars[kMost] = ldexpf(most * rows_of_t, 9);
            reinterpret_cast<uint32_t *>(scalars)[kWild] = wild;
        }
        wave_lds_sync();
    }
}

// One wave's columns of a chunk, token after token, for chunks whose algebra
// would not hold. S: the state itself, tile t's lane has rows 16t + 4g + i.
template <int TD>
__device__ __forceinline__ void tokens_of_chunk(const LinearArgs &a, size_t token0, uint32_t n, uint32_t h, uint32_t col, f4 (&S)[TD]) {
    const uint32_t g = threadIdx.x % 64 / 16, kh = h / (a.v_heads / a.k_heads);
    const bool has = col < a.dv;
    for (uint32_t t = 0; t < n; ++t) {
        const size_t token = token0 + t;
        const float *qr = a.q + token * a.q_stride + size_t(kh) * a.dk, *kr = a.k + token * a.k_stride + size_t(kh) * a.dk;
        float kk = 0.f, qq = 0.f, qk = 0.f, sk = 0.f, sq = 0.f;
#pragma unroll
        for (int td = 0; td < TD; ++td) {
            const uint32_t d = 16 * td + 4 * g;
            const Quad q = quad_at(qr + d, d < a.dk), k = quad_at(kr + d, d < a.dk);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                kk = fmaf(k.x[i], k.x[i], kk);
                qq = fmaf(q.x[i], q.x[i], qq);
                qk = fmaf(q.x[i], k.x[i], qk);
                sk = fmaf(S[td][i], k.x[i], sk);
                sq = fmaf(S[td][i], q.x[i], sq);
            }
        }
        kk = column_sum(kk);
        qq = column_sum(qq);
        qk = column_sum(qk);
        sk = column_sum(sk);
        sq = column_sum(sq);
        const float decay = expf(log_decay(a, token, h));
        const float v = has ? a.v[token * a.v_stride + size_t(h) * a.dv + col] : 0.f;
        const float fk = a.qk_eps > 0.f ? 1.f / sqrtf(kk + a.qk_eps) : 1.f;
        const float fq = (a.qk_eps > 0.f ? 1.f / sqrtf(qq + a.qk_eps) : 1.f) * a.scale;
        const float u = a.delta ? sigmoid(a.b[token * a.b_stride + h]) * (v - decay * (sk * fk)) : v;
        if (g == 0 && has)
            a.out[token * a.out_stride + size_t(h) * a.dv + col] = fq * (decay * sq + qk * fk * u);
#pragma unroll
        for (int td = 0; td < TD; ++td) {
            const uint32_t d = 16 * td + 4 * g;
            const Quad k = quad_at(kr + d, d < a.dk);
#pragma unroll
            for (int i = 0; i < 4; ++i) S[td][i] = fmaf(k.x[i] * fk, u, decay * S[td][i]);
        }
    }
}

// How a workgroup's waves share the work: NC have a 16-column tile each, NL load.
template <int KB, int NC, int NL, bool DELTA>
struct Scan {
    static constexpr int kThreads = (NC + NL) * 64;
    static constexpr uint32_t kTerms = 4 * kTile * KB;  // of Q, or of K
    static constexpr uint32_t kKey = 2 * kTerms, kValue = (DELTA ? 9 : 5) * kTile;
    static constexpr uint32_t kV = kChunk * NC * 16 * 4;  // the workgroup's columns of the values
    static constexpr uint32_t kStage = kKey + kValue + kV;
    static constexpr uint32_t kBytes = 2 * kStage;
    static_assert(kBytes <= 160 * 1024, "two stages fit LDS");
};

template <int KB, int NC, int NL, bool DELTA>
__global__ __launch_bounds__((NC + NL) * 64, KB < 8 ? 2 : 1) void linear_scan_kernel(LinearArgs a, Pass pass) {
    extern __shared__ __align__(16) unsigned char lds[];
    using L = Scan<KB, NC, NL, DELTA>;
    constexpr int TD = 2 * KB;
    const uint32_t l = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), g = l / 16, m = l % 16;

    // Workgroups go to the eight dies in turn: all those of a key head to one,
    // whose cache then has its operands once.
    const uint32_t group = a.v_heads / a.k_heads, of_unit = group * pass.columns;
    const uint32_t unit = blockIdx.x % 8 + blockIdx.x / 8 / of_unit * 8, in_unit = blockIdx.x / 8 % of_unit;
    if (unit >= a.seq.seqs * a.k_heads) return;
    const uint32_t s = unit / a.k_heads, kh = unit % a.k_heads, h = kh * group + in_unit / pass.columns;

    uint32_t first, count;
    seq::tokens_of(a.seq, s, first, count);
    if (count == 0) return;
    const uint32_t begin = seq::parts_before(a.seq, s, kChunk), end = begin + (count + kChunk - 1) / kChunk;
    const uint32_t c0 = max(begin, pass.first), c1 = min(end, pass.last);
    if (c0 >= c1) return;

    const uint32_t lds0 = uint32_t(uintptr_t((__attribute__((address_space(3))) unsigned char *)lds));
    auto stage_of = [&](uint32_t c) { return (c - c0) % 2 * L::kStage; };
    if (w >= NC) {
        // A chunk ahead of the others: every barrier says that a chunk is there
        // and that the one before is no longer read.
        constexpr uint32_t kAt = NC * 16;  // columns of the workgroup
        const uint32_t col0 = in_unit % pass.columns * kAt + l % kAt;
        const uint32_t values_at = col0 < a.dv ? (l / kAt * a.v_stride + col0) * 4 : kOut;
        const uint32_t own = w - NC;
        for (uint32_t c = c0; c < c1; ++c) {
            const uint32_t to = lds0 + stage_of(c), t0 = (c - begin) * kChunk, n = min(kChunk, count - t0);
            const u4 keys = rsrc_of(pass.of_key(a, c, kh), L::kKey), values = rsrc_of(pass.of_value(a, c, h), L::kValue);
            const u4 v = rsrc_of(a.v + (size_t(first) + t0) * a.v_stride + size_t(h) * a.dv, ((n - 1) * a.v_stride + a.dv) * 4);
            uint32_t piece = own * 256, row = own * (64 / kAt) * a.v_stride * 4;
            asm volatile("" : "+s"(piece), "+s"(row));  // counted here, not kept in registers for every piece
#pragma unroll
            for (uint32_t p = 0; p < L::kV; p += NL * 256, piece += NL * 256, row += NL * (64 / kAt) * a.v_stride * 4)
                dma4(v, values_at + row, 0, to + L::kKey + L::kValue + piece);  // past the rows, zeros
            piece = own * kTile;
            asm volatile("" : "+s"(piece));
#pragma unroll
            for (uint32_t p = 0; p < L::kKey + L::kValue; p += NL * kTile, piece += NL * kTile) {
                if (p + NL * kTile <= L::kKey || piece < L::kKey) {
                    dma16(keys, l * 16, piece, to + piece);
                } else if (p + NL * kTile <= L::kKey + L::kValue || piece < L::kKey + L::kValue) {
                    dma16(values, l * 16, piece - L::kKey, to + piece);
                }
            }
            wait_dma<0>();
            lds_barrier();
        }
        return;
    }

    const bool starts = c0 == begin, ends = c1 == end;
    bool read;
    const uint32_t slot = seq::slot_of(a.seq, s, read);
    const uint32_t tile = in_unit % pass.columns * NC + w, col = tile * 16 + m, state_bytes = a.dk * a.dv * 4;
    const bool has = col < a.dv, idle = tile * 16 >= a.dv;
    float *pool = a.state + (size_t(slot == seq::kNoSlot ? 0 : slot) * a.v_heads + h) * a.dk * a.dv;
    const float *from = starts ? pool : pass.from + size_t(h) * a.dk * a.dv;
    // Of a buffer's rows these lanes have 4g + i of every 16; what is past the
    // head's dimensions or the sequence's tokens is past the buffer.
    uint32_t state_at = has ? (4 * g * a.dv + col) * 4 : kOut;
    const uint32_t out_at = has ? (4 * g * a.out_stride + col) * 4 : kOut;
    f4 S[TD];
    {
        const auto r = buffer_of(from, !starts || read ? state_bytes : 0);
#pragma unroll
        for (int t = 0; t < TD; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                S[t][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, int(state_at + (16 * t + i) * a.dv * 4), 0, 0));
    }
    float minus = -1.f;
    asm volatile("" : "+v"(minus));

    // S is kept by 2^scale, a column's own.
    int scale = 0;
    auto biggest = [&] {
        float top = 0.f;
#pragma unroll
        for (int t = 0; t < TD; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(S[t][i]));
        return column_max(top);
    };
    auto rescale = [&](int to) {
#pragma unroll
        for (int t = 0; t < TD; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[t][i] = ldexpf(S[t][i], to - scale);
        scale = to;
    };
    // A column of zeros has room for values of any size; one with an infinity is
    // kept as it is.
    auto fitting = [](float top) { return top > 0.f && top < INFINITY ? max(-113, min(15 - exponent(top), 110)) : 0; };
    // A state that the last pass left is kept as it was there, its columns'
    // scales behind it: no result depends on where passes end.
    const size_t scale_at = size_t(a.v_heads) * a.dk * a.dv + size_t(h) * a.dv + col;
    if (!starts && has) scale = __float_as_int(pass.from[scale_at]);
    // An infinity fits no scale: with one in its state a wave goes token after token.
    uint32_t infinite;  // whether there is one
    auto fit = [&](bool anew) {
        const float top = biggest();
        infinite = __ballot(top == INFINITY) != 0;
        rescale(anew ? fitting(top) : scale);
    };
    fit(starts);

    uint32_t c = c0;
    if (idle) {
        for (; c < c1; ++c) lds_barrier();
    }
    // Two loops, so that a chunk that is done token after token costs the others
    // no register moves where the paths would meet.
    while (c < c1) {
        bool slow = false;
        do {
            lds_barrier();  // the chunk's operands are there
            // This lane's places in the stage, each a register and constants from there.
            const uint32_t stage = stage_of(c);
            uint32_t own = stage + l * 16, rows_at = stage + L::kKey + kScalars + g * 16;
            uint32_t across_at = stage + L::kTerms + (m % 4 * 16 + 4 * g + m / 4) * 16;
            uint32_t v_at = stage + L::kKey + L::kValue + (4 * g * NC * 16 + w * 16 + m) * 4;
            asm volatile("" : "+v"(own), "+v"(rows_at), "+v"(across_at), "+v"(v_at));
            const float *scalars = reinterpret_cast<const float *>(lds + stage + L::kKey + kScalars);
            // LDS answers late: operands are asked for well before the matrix
            // instructions that take them, into registers that the last ones left.
            struct Terms {
                u4 hi, lo;
            };
            auto at = [&](uint32_t p) {
                return Terms{*reinterpret_cast<const u4 *>(lds + own + p), *reinterpret_cast<const u4 *>(lds + own + (p + kTile))};
            };
            // A tile of K^T: rows of four dims of four tokens, read across.
            auto across = [&](int t, int term) {
                u4 r;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    typedef short s4 __attribute__((ext_vector_type(4)));
                    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
                    const unsigned char *p = lds + across_at + (((half * KB + t / 2) * 2 + term) * kTile + t % 2 * 8);
                    const u2 x = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p));
                    r[2 * half] = x[0];
                    r[2 * half + 1] = x[1];
                }
                return r;
            };
            // A sum waits for the matrix instruction before it some time longer than
            // that one keeps the others: as many sums as there are go on in turn.
            auto step = [&](int which, const Terms &x, u4 hi, u4 lo, f4 &c) {
                c = mfma(which == 0 ? x.lo : x.hi, which == 1 ? lo : hi, c);
            };
            auto of_rows = [&](uint32_t which, int half) { return *reinterpret_cast<const f4 *>(lds + rows_at + (which + 16 * half) * 4); };
            const float whole = scalars[kWhole], most = scalars[kMost];
            const uint32_t wild = reinterpret_cast<const uint32_t *>(scalars)[kWild];
            const uint32_t t0 = (c - begin) * kChunk, n = min(kChunk, count - t0);
            float v[8];  // tokens 16h + 4g + i at 4h + i
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = *reinterpret_cast<const float *>(lds + v_at + (16 * (e / 4) + e % 4) * (NC * 16) * 4);
            f4 beta[2], of_x[2], of_u[2];
            Terms tk[2][KB], tq[2][KB], tt[2], tu[TD];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                beta[half] = of_rows(kBeta, half);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
                    if constexpr (DELTA) tk[half][kb] = at(L::kTerms + (half * KB + kb) * 2 * kTile);
            }
            __builtin_amdgcn_sched_barrier(0);
            u4 sh[KB], sl[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                float both[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) both[e] = S[2 * kb + e / 4][e % 4];
                terms(both, minus, sh[kb], sl[kb]);
            }
            __builtin_amdgcn_sched_barrier(0);
            // S^T k; meanwhile R's part that does not wait for it, all by 2^scale.
            constexpr int PAR = KB > 1 ? 2 : 1;  // sums of blocks 0, 2, .. and 1, 3, ..
            f4 x2[2][PAR] = {}, o2[2][PAR] = {}, x[2], o[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                of_x[half] = of_rows(kX, half);
                if constexpr (DELTA) tt[half] = at(L::kKey + kScalars + kTile + half * 2 * kTile);
            }
#pragma unroll
            for (int kb = 0; kb < KB; kb += PAR) {
                if constexpr (DELTA) {
#pragma unroll
                    for (int i = 0; i < 6 * PAR; ++i)
                        step(i / (2 * PAR), tk[i % 2][kb + i / 2 % PAR], sh[kb + i / 2 % PAR], sl[kb + i / 2 % PAR], x2[i % 2][i / 2 % PAR]);
                }
#pragma unroll
                for (int i = 0; i < 2 * PAR; ++i) tq[i % 2][kb + i / 2] = at((i % 2 * KB + kb + i / 2) * 2 * kTile);
            }
            float r[8];
            {
                const float by = ldexpf(1.f, scale);
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = v[e] * (DELTA ? beta[e / 4][e % 4] * by : by);
            }
            // Values that are not finite, or so far above the state that they leave the
            // exponents that `up` can take back (2^116).
            float odd = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) odd = fmaf(r[e] * 0x1p12f, 0.f, odd);
            const float top = biggest();
            if constexpr (DELTA) in_turn<6 * KB, 2, 1>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int half = 0; half < 2; ++half) x[half] = PAR > 1 ? x2[half][0] + x2[half][PAR - 1] : x2[half][0];
            slow = (__builtin_amdgcn_readfirstlane(wild) | infinite) != 0 || __ballot(odd != 0.f) != 0;
            if (slow) break;
            // S^T q; meanwhile R and its terms, by 2^up more; the next state's scale:
            // below 2^15 whatever the chunk adds.
#pragma unroll
            for (int half = 0; half < 2; ++half) of_u[half] = of_rows(kU, half);
#pragma unroll
            for (int kb = 0; kb < KB; kb += PAR) {
#pragma unroll
                for (int i = 0; i < 6 * PAR; ++i)
                    step(i / (2 * PAR), tq[i % 2][kb + i / 2 % PAR], sh[kb + i / 2 % PAR], sl[kb + i / 2 % PAR], o2[i % 2][i / 2 % PAR]);
#pragma unroll
                for (int t = 2 * kb; t < 2 * kb + 2 * PAR; ++t) tu[t] = Terms{across(t, 0), across(t, 1)};
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) o[half] = PAR > 1 ? o2[half][0] + o2[half][PAR - 1] : o2[half][0];
            if constexpr (DELTA) {
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = fmaf(-of_x[e / 4][e % 4], x[e / 4][e % 4], r[e]);
            }
            float r_top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) r_top = fmaxf(r_top, fabsf(r[e]));
            r_top = column_max(r_top);
            const int up = max(-113, min((DELTA ? 5 : 13) - exponent(r_top), 110));
            // In 64 bits: the product of long keys' part and large values may be past
            // FP32's range where the sum they bound is not.
            const double next = fma(double(most), double(r_top), double(whole) * double(top));
            int to = next > 0.0 ? min(scale + 15 - __builtin_amdgcn_frexp_exp(next), scale + 100) : 0;  // as fitting()
            to = max(-113, min(to, 110));
            u4 uh, ul;
            {
                const float by = ldexpf(1.f, up);
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] *= by;
            }
            terms(r, minus, uh, ul);
            in_turn<6 * KB, 3, 1>();
            __builtin_amdgcn_sched_barrier(0);
            // U, by 2^(scale + up + kSolve): below 2^15 while rows of T add up to 2^6.
            float u[8];
            if constexpr (DELTA) {
                f4 y[2] = {};
#pragma unroll
                for (int i = 0; i < 6; ++i) step(i / 2, tt[i % 2], uh, ul, y[i % 2]);
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = y[e / 4][e % 4];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) u[e] = r[e];
            }
            Terms tm[2];
            f4 of_q[2], of_m[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                tm[half] = at(L::kKey + half * 2 * kTile);
                of_q[half] = of_rows(kQ, half);
                of_m[half] = of_rows(kM, half);
            }
            {
                const float keep = ldexpf(whole, to - scale);
#pragma unroll
                for (int t = 0; t < TD; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) S[t][i] *= keep;
                // Each by itself: where keys are zero and the state has shrunk, the
                // power of two alone may be past FP32's.
                const int by = to - scale - up - (DELTA ? kSolve : 0);
#pragma unroll
                for (int e = 0; e < 8; ++e) of_u[e / 4][e % 4] = ldexpf(of_u[e / 4][e % 4], by);
            }
            if constexpr (DELTA) in_turn<6, 6, 1>();
            __builtin_amdgcn_sched_barrier(0);
            u4 wh, wl;
            {
                float left[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) left[e] = u[e] * of_u[e / 4][e % 4];
                terms(left, minus, wh, wl);
                if constexpr (DELTA) terms(u, minus, uh, ul);
            }
            __builtin_amdgcn_sched_barrier(0);
            // The next state, M U and the outputs.
            f4 y[2] = {};
#pragma unroll
            for (int i = 0; i < 6; ++i) step(i / 2, tm[i % 2], uh, ul, y[i % 2]);
#pragma unroll
            for (int i = 0; i < 3 * TD; ++i) step(i / TD, tu[i % TD], wh, wl, S[i % TD]);
            const float one = ldexpf(1.f, -scale - kRoom), of_y = ldexpf(1.f, (DELTA ? -kSolve : 0) - up - scale - kRoom);
            const auto rows = buffer_of(a.out + (size_t(first) + t0) * a.out_stride + size_t(h) * a.dv, ((n - 1) * a.out_stride + a.dv) * 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float out = of_q[e / 4][e % 4] * (o[e / 4][e % 4] * one) + of_m[e / 4][e % 4] * (y[e / 4][e % 4] * of_y);
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(out), rows,
                                                      int(out_at + (16 * (e / 4) + e % 4) * a.out_stride * 4), 0, 0);
            }
            scale = to;
#pragma unroll
            for (int t = 0; t < TD; ++t) asm volatile("" : "+v"(S[t]));  // in the registers it came in
        } while (++c < c1);
        if (!slow) break;
        const uint32_t t0 = (c - begin) * kChunk;
        rescale(0);
        tokens_of_chunk<TD>(a, size_t(first) + t0, min(kChunk, count - t0), h, col, S);
        fit(true);
        ++c;
    }
    if (idle || (ends ? !a.keep || slot == seq::kNoSlot : pass.to == nullptr)) return;
    if (!ends && has && g == 0) pass.to[scale_at] = __int_as_float(scale);
    rescale(ends ? 0 : scale);
    const auto r = buffer_of(ends ? pool : pass.to + size_t(h) * a.dk * a.dv, state_bytes);
    asm volatile("" : "+v"(state_at));  // or all of the addresses wait in registers for this
#pragma unroll
    for (int t = 0; t < TD; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[t][i]), r, int(state_at + (16 * t + i) * a.dv * 4), 0, 0);
}

constexpr int kNorm = 256;

// The RMS norm and gate of the outputs, where they are: LANES lanes a head's row
// of a token, a workgroup a chunk's tokens of one head, all of whose loads are
// under way at once.
template <int LANES>
__global__ __launch_bounds__(kNorm) void linear_norm_kernel(LinearArgs a) {
    constexpr int kSlots = kNorm / LANES, kEach = kSlots < 32 ? 32 / kSlots : 1;
    uint32_t s, part, first, count;
    if (!seq::part_of(a.seq, blockIdx.x, kChunk, s, part)) return;
    seq::tokens_of(a.seq, s, first, count);
    const uint32_t t0 = part * kChunk, n = min(kChunk, count - t0), h = blockIdx.y;
    const uint32_t col = threadIdx.x % LANES * 4, slot = threadIdx.x / LANES;
    const bool has = col < a.dv;
    const Quad norm = quad_at(a.norm + col, has);
    float *out = a.out + (size_t(first) + t0 + slot) * a.out_stride + size_t(h) * a.dv + col;
    const float *gate = a.z + (size_t(first) + t0 + slot) * a.z_stride + size_t(h) * a.dv + col;
    Quad o[kEach], z[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const bool there = has && slot + k * kSlots < n;
        o[k] = quad_at(out + size_t(k) * kSlots * a.out_stride, there);
        z[k] = quad_at(gate + size_t(k) * kSlots * a.z_stride, there);
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fmaf(o[k].x[i], o[k].x[i], sum);
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) sum += __shfl_xor(sum, d);
        const float f = 1.f / sqrtf(sum / float(a.dv) + a.out_eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[k].x[i] = o[k].x[i] * f * gate_of(z[k].x[i], norm.x[i]);
        if (has && slot + k * kSlots < n) *reinterpret_cast<Quad *>(out + size_t(k) * kSlots * a.out_stride) = o[k];
    }
}

template <int KB, bool DELTA>
hipError_t go_prepare(const LinearArgs &a, const Pass &pass, hipStream_t stream) {
    const auto kernel = linear_prepare_kernel<KB, DELTA>;
    constexpr uint32_t lds = PrepareLds<KB>::kBytes;
    const hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kernel), lds);
    if (e != hipSuccess) return e;
    kernel<<<dim3(pass.last - pass.first, a.k_heads), kPrepare, lds, stream>>>(a, pass);
    return hipGetLastError();
}

template <int KB, int NC, int NL, bool DELTA>
hipError_t go_scan(const LinearArgs &a, const Pass &pass, hipStream_t stream) {
    const auto kernel = linear_scan_kernel<KB, NC, NL, DELTA>;
    using L = Scan<KB, NC, NL, DELTA>;
    const hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kernel), L::kBytes);
    if (e != hipSuccess) return e;
    const uint32_t units = (a.seq.seqs * a.k_heads + 7) / 8 * 8;
    kernel<<<units * (a.v_heads / a.k_heads) * pass.columns, L::kThreads, L::kBytes, stream>>>(a, pass);
    return hipGetLastError();
}

template <int KB, bool DELTA>
hipError_t go_pass(const LinearArgs &a, const LinearPlan &pl, const Pass &pass, hipStream_t stream) {
    const hipError_t e = go_prepare<KB, DELTA>(a, pass, stream);
    if (e != hipSuccess) return e;
    if constexpr (KB == 8) {
        return go_scan<KB, 2, 2, DELTA>(a, pass, stream);  // two states' worth of registers a wave
    } else {
        return pl.columns == 2 ? go_scan<KB, 2, 2, DELTA>(a, pass, stream) : go_scan<KB, 4, 4, DELTA>(a, pass, stream);
    }
}

}  // namespace

LinearPlan plan_linear(const LinearArgs &a, const DeviceLimits &lim, size_t limit, uint32_t form, uint32_t columns) {
    LinearPlan pl;
    const Sequences &q = a.seq;
    const uint32_t longest = std::min(q.most, q.tokens);
    // Token after token up to eight, whatever the dimensions. Both forms in us, 48
    // heads of 128 x 128: one sequence of 4, 8, 12 and 16 tokens 12/21, 17/21, 23/21
    // and 28/22; eight sequences of 8 and 12 29/38 and 38/39; 32 of 8 and 12 77/95 and
    // 102/97. Eight heads of 64 x 64, one sequence of 8 and 12: 16/17 and 21/18. Three
    // heads of 256 x 192 would do with fewer (8 and 12: 30/26 and 42/27); a rule for
    // them alone would save those 4 us.
    if (form == 1 || (form == 0 && longest <= 8)) return pl;
    // Rows that a buffer's 32-bit offsets reach over a chunk.
    if (a.v_stride > 1u << 22 || a.out_stride > 1u << 22) return pl;
    if (columns != 2 && columns != 4) columns = 0;
    const uint32_t tiles = (a.dv + 15) / 16;
    pl.blocks = a.dk <= 64 ? 2 : a.dk <= 128 ? 4 : 8;
    pl.columns = columns && pl.blocks < 8 ? columns : 2;
    pl.parts = uint32_t(std::min<uint64_t>(q.tokens, uint64_t(q.tokens) / kChunk + q.seqs));
    pl.k_bytes = size_t(8) * kTile * pl.blocks;
    pl.v_bytes = size_t(a.delta ? 9 : 5) * kTile;
    // Four tiles a workgroup read a chunk's operands half as often, two are twice
    // as many workgroups: as long as those have a CU each. 48 heads of 128 x 128,
    // 512 tokens a sequence, two tiles / four in us: one sequence 59/61, two 96/74,
    // four 144/125, 16 572/449; 64 heads of 64 x 64: 47/49, 54/56, 76/70, 280/265.
    if (columns == 0 && pl.blocks < 8)
        while (pl.columns < 4 && uint64_t(std::min(q.seqs, pl.parts)) * a.v_heads * ((tiles + pl.columns - 1) / pl.columns) >
                                     uint64_t(lim.num_cus))
            pl.columns *= 2;
    const size_t each = a.k_heads * pl.k_bytes + a.v_heads * pl.v_bytes;
    limit = std::min(limit, size_t(256) << 20);
    pl.per_pass = pl.parts;
    if (each * pl.parts > limit) {
        pl.carry_bytes = (size_t(a.v_heads) * (a.dk + 1) * a.dv * 4 + 255) / 256 * 256;
        if (limit < 2 * pl.carry_bytes + each) return LinearPlan{};
        pl.per_pass = uint32_t((limit - 2 * pl.carry_bytes) / each);
    }
    pl.workspace = 2 * pl.carry_bytes + each * pl.per_pass;
    pl.chunks = true;
    return pl;
}

// The workspace holds the operands of so many chunks; more go in passes, and
// the state of a sequence that a pass leaves unfinished goes from one to the
// next.
hipError_t launch_linear_chunks(const LinearArgs &a, const LinearPlan &pl, void *workspace, hipStream_t stream) {
    Pass pass{};
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    pass.operands = ws + 2 * pl.carry_bytes;
    pass.k_bytes = uint32_t(pl.k_bytes);
    pass.v_bytes = uint32_t(pl.v_bytes);
    pass.columns = ((a.dv + 15) / 16 + pl.columns - 1) / pl.columns;
    hipError_t e = hipSuccess;
    uint32_t turn = 0;
    for (uint32_t c = 0; c < pl.parts && e == hipSuccess; c += pl.per_pass, ++turn) {
        pass.first = c;
        pass.last = std::min(pl.parts, c + pl.per_pass);
        pass.from = reinterpret_cast<float *>(ws + (turn % 2) * pl.carry_bytes);
        pass.to = pass.last < pl.parts ? reinterpret_cast<float *>(ws + (1 - turn % 2) * pl.carry_bytes) : nullptr;
        switch (pl.blocks * 2 + a.delta) {
            case 4: e = go_pass<2, false>(a, pl, pass, stream); break;
            case 5: e = go_pass<2, true>(a, pl, pass, stream); break;
            case 8: e = go_pass<4, false>(a, pl, pass, stream); break;
            case 9: e = go_pass<4, true>(a, pl, pass, stream); break;
            case 16: e = go_pass<8, false>(a, pl, pass, stream); break;
            default: e = go_pass<8, true>(a, pl, pass, stream); break;
        }
    }
    if (e != hipSuccess || !(a.out_eps > 0.f)) return e;
    const dim3 grid(pl.parts, a.v_heads);
    if (a.dv <= 32) linear_norm_kernel<8><<<grid, kNorm, 0, stream>>>(a);
    else if (a.dv <= 64) linear_norm_kernel<16><<<grid, kNorm, 0, stream>>>(a);
    else if (a.dv <= 128) linear_norm_kernel<32><<<grid, kNorm, 0, stream>>>(a);
    else linear_norm_kernel<64><<<grid, kNorm, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace qmr
