// Attention of new tokens over a paged key-value cache (layouts:
// rope_append.hip), for one token a sequence as for whole prompts.
//
//   o_r = sum_j p_rj v_j,  p_r = softmax_j(scale q_r . k_j)
//
// over the keys j that row r (a token's query head) may see. One pass over the
// keys with the running maximum m and sum l of each row, in 32 bits, in powers
// of two (q carries scale * log2 e).
//
// Products run on the matrix cores in the cache's own 16-bit type: an FP32
// operand is the sum of two f16 terms (22 bits) or three bf16 terms (24 bits).
// That is two or three times the matrix work, which a call of few rows has to
// spare, and an error near 32-bit arithmetic's own, as every product of this
// library has. f16 spans 40 powers of two: queries are scaled by a power of two
// a row, so that an element is off by 2^-39 of the row's largest where that is
// more than its own 22 bits; weights are off by 2^-36 of the largest (kTop).
//
// Operand placement (v_mfma_f32_16x16x32: A row and B column lane % 16, K
// chunk lane / 16; D[i][j] in lane j + 16 (i / 4), element i % 4): S^T = K Q^T
// with the 32 keys of a block dealt to two instructions so that lane (n, g)
// ends with the scores of row n and keys 8g..8g+7, which is where P^T has to
// be as the B operand of O^T = V^T P^T. Scores never leave their lane.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace qmr {
namespace {

using attn::kBlock;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef f4 f4u __attribute__((aligned(4)));  // rows of FP32 need no more

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr uint32_t kMaxSplits = 512;  // key ranges of a tile, at most
constexpr uint32_t kFewSplits = 16;   // that a wave joins alone, at most
constexpr uint32_t kRsrcWord3 = 0x00020000u;
constexpr uint32_t kNone = 0xFFFFFFFFu;

// Terms of an FP32 operand in the cache's type.
template <bool BF16>
constexpr int kTerms = BF16 ? 3 : 2;

template <bool BF16>
__device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
    if constexpr (BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
}

template <bool BF16>
__device__ __forceinline__ f16v mfma32(u4 a, u4 b, f16v c) {
    if constexpr (BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
}

__device__ __forceinline__ uint32_t high_halves(uint32_t lo, uint32_t hi) {  // lo >> 16 | hi & 0xFFFF0000
    return __builtin_amdgcn_perm(hi, lo, 0x07060302u);
}

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

// Eight FP32 values as kTerms vectors of eight halves that add up to them, each
// term exact in what the ones before leave: bf16 ones truncated, f16 ones to
// nearest (the second rounds at 2^-23).
template <bool BF16>
__device__ __forceinline__ void split8(const float (&x)[8], u4 (&t)[kTerms<BF16>]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = x[2 * i], b = x[2 * i + 1];
        if constexpr (BF16) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
                t[k][i] = high_halves(ua, ub);
                a -= __uint_as_float(ua & 0xFFFF0000u);
                b -= __uint_as_float(ub & 0xFFFF0000u);
            }
        } else {
            t[0][i] = two_halves(a, b);
            t[1][i] = two_halves(less_half<0>(a, t[0][i]), less_half<1>(b, t[0][i]));
        }
    }
}

// The power of two that brings a row's queries, `most` at most, to 2^14..2^15. Not
// below FP32's normal numbers: as a factor of 0 it would make NaN of the minus
// infinity of a key that is not seen.
__device__ __forceinline__ int query_exponent(float most) {
    int e;
    frexpf(most, &e);
    return max(e - 15, -126);
}

// A block of keys or values as a buffer of its own bytes: loads past it give
// zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_rsrc(const uint16_t *pool, size_t at, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t *>(pool + at), 0, int(bytes), kRsrcWord3);
}

__device__ __forceinline__ u4 load16(__amdgpu_buffer_rsrc_t r, uint32_t offset, uint32_t more) {
    return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(r, int(offset), int(more), 0));
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

// What a workgroup works on: a tile of query rows of one sequence and key
// head. Row r of the sequence is token r / group, head r % group.
struct Tile {
    uint32_t seq, first_token, row0, rows;  // rows: of the whole sequence
    int length, context;                    // cache length; position of the sequence's first new token
};

// Tile number `tile` among all sequences' (ceil(rows / R) of each), found by
// a wave's prefix sum over 64 sequences at a time; false past the last.
__device__ __forceinline__ bool find_tile(const PagedCache &c, uint32_t group, uint32_t R, uint32_t tile, Tile &t) {
    const uint32_t l = threadIdx.x % 64;
    for (uint32_t base = 0; base < c.seqs; base += 64) {
        const uint32_t s = base + l;
        uint32_t from = 0, end = 0, length = 0;
        if (s < c.seqs) {
            from = c.starts[s];
            end = c.starts[s + 1];
            length = c.lengths[s];
        }
        const uint32_t to = min(end, c.tokens), count = to > from ? to - from : 0;
        const uint32_t own = (count * group + R - 1) / R;
        uint32_t sum = own;
        if (__ballot(own > 1) == 0) {  // decode: bits to count
            const uint64_t some = __ballot(own != 0);
            sum += __builtin_amdgcn_mbcnt_hi(uint32_t(some >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(some), 0));
        } else {
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const uint32_t o = __shfl_up(sum, d);
                if (l >= uint32_t(d)) sum += o;
            }
        }
        const uint32_t total = __builtin_amdgcn_readlane(sum, 63);
        if (tile >= total) {
            tile -= total;
            continue;
        }
        const int at = __ffsll(__ballot(sum > tile)) - 1;
        t.seq = base + at;
        t.first_token = __builtin_amdgcn_readlane(from, at);
        t.rows = __builtin_amdgcn_readlane(count, at) * group;
        t.row0 = (tile - __builtin_amdgcn_readlane(sum - own, at)) * R;
        t.length = int(min(uint32_t(__builtin_amdgcn_readlane(length, at)), 0x7FFFFFFFu));
        t.context = t.length - int(__builtin_amdgcn_readlane(end, at) - t.first_token);
        return true;
    }
    return false;
}

// Keys [lo, hi) that a new token of the sequence may see.
__device__ __forceinline__ void visible(const AttendArgs &a, const Tile &t, uint32_t token, int &lo, int &hi) {
    const int pos = t.context + int(token);
    hi = a.causal ? min(pos + 1, t.length) : t.length;
    hi = max(min(hi, int(a.max_keys)), 0);
    // pos - window is taken where it is not negative: a window may be as long as
    // INT32_MAX, and a sequence's first new tokens may stand before position 0.
    lo = a.window && pos >= int(a.window) ? pos - int(a.window) + 1 : 0;
}

// The order of a range's blocks: those that some row sees in part first (the
// ones before and after what every row sees), then the others, so that the
// loop over these has no masks.
struct Order {
    int first, lead, whole, after, edges, count;
    __device__ __forceinline__ Order(int from, int to, int lo_most, int hi_least) {
        const int b = int(kBlock), end = (to + b - 1) / b;
        first = from / b;
        whole = min(max((lo_most + b - 1) / b, first), end);
        after = min(max(hi_least / b, whole), end);
        lead = whole - first;
        edges = lead + end - after;
        count = end - first;
    }
    // First key of the i-th block; of the last one past them.
    __device__ __forceinline__ int key(int i) const {
        i = min(i, count - 1);
        return (i < lead ? first + i : i < edges ? after + i - lead : whole + i - edges) * int(kBlock);
    }
};

// Results of key ranges, to be joined: for each (tile, head, range) R rows of
// DM floats, and their m and l; for each (tile, head) its rows' places in the
// output (kNone: nothing to join).
struct Partial {
    float *o;
    float2 *ml;
    uint32_t *place;
};

typedef uint16_t us2 __attribute__((ext_vector_type(2)));
typedef int16_t is2 __attribute__((ext_vector_type(2)));

// The exponent of the type's infinity and NaNs, and its 1.0, in both halves.
template <bool BF16>
constexpr uint32_t kInf = BF16 ? 0x7F807F80u : 0x7C007C00u;
template <bool BF16>
constexpr uint32_t kOne = BF16 ? 0x3F803F80u : 0x3C003C00u;

// The halves' sizes, the larger of each.
__device__ __forceinline__ us2 larger(us2 a, uint32_t v) {
    return __builtin_elementwise_max(a, __builtin_bit_cast(us2, v & 0x7FFF7FFFu));
}

template <bool BF16>
__device__ __forceinline__ bool has_not_finite(us2 largest) {
    constexpr uint16_t inf = kInf<BF16> & 0xFFFF;
    return largest[0] >= inf || largest[1] >= inf;
}

// Ones in the halves that are not finite.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite(uint32_t v) {
    const us2 over = __builtin_bit_cast(us2, v & 0x7FFF7FFFu) + __builtin_bit_cast(us2, 0x80008000u - kInf<BF16>);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(is2, over) >> 15);
}

// Ones in the halves of the keys first..first+7 that lie in [lo, hi).
__device__ __forceinline__ u4 halves_of(int first, int lo, int hi) {
    u4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = first + 2 * i;
        m[i] = (k >= lo && k < hi ? 0x0000FFFFu : 0u) | (k + 1 >= lo && k + 1 < hi ? 0xFFFF0000u : 0u);
    }
    return m;
}

// 1.0 in those halves.
template <bool BF16>
__device__ __forceinline__ u4 ones_of(int first, int lo, int hi) {
    return halves_of(first, lo, hi) & kOne<BF16>;
}

// Whether one of a block's keys lo..hi-1 (counted from its first) is not finite.
// An infinite key can give a score of minus infinity, which has no weight and
// leaves no mark on its row; a wave that has met such a score looks at the keys
// of all its blocks once more.
template <bool BF16>
__device__ __forceinline__ bool sees_bad_key(__amdgpu_buffer_rsrc_t block, uint32_t dim, int lo, int hi) {
    const uint32_t l = threadIdx.x % 64, place = 16 * (l / 4 % 2) + 4 * (l / 8 % 4) + l % 4;  // of slot l % 32
    uint32_t bad = 0;
#pragma unroll 1
    for (uint32_t ch = l / 32; ch < dim / 8; ch += 2) {
        const u4 x = load16(block, (ch * kBlock + place) * 16, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= not_finite<BF16>(x[i]);
    }
    const uint64_t some = __ballot(bad != 0);
    auto below = [](int n) { return n >= 32 ? 0xFFFFFFFFu : (1u << max(n, 0)) - 1; };
    return ((uint32_t(some) | uint32_t(some >> 32)) & below(hi) & ~below(lo)) != 0;
}

// Few rows: 16 rows a workgroup, every wave all of them over its own blocks of
// the range (block w, w + 4, ..), straight from memory into operand registers,
// whole lines at a time; nothing is shared but the queries, which wait in LDS
// as operands. The waves' m, l and O are joined through LDS at the end. A wave
// holds a block of keys and one of values (32 KB at 256 dims), a CU two
// workgroups: 256 KB on their way, more than HBM needs. 32 rows a workgroup
// spilled registers.
// Memory bounds it: 32 sequences of 8 heads of 128 over up to 8001 keys (521
// MB) 105 us, 5.0 TB/s (repeated, so in part from the last-level cache; a large
// copy reaches 4.8); one token of 24/4 heads of 256 over 32768 (134 MB) 28 us
// with the join, 4.8 TB/s, and 34.9 over one of four caches in turn, which the
// last-level cache does not hold; over 1001 keys (4 MB) 10.5 us, of which the
// join takes 3 and the first workgroup's chain of dependent steps (its sequence, its
// page, keys and queries, products, waves joined) the rest.
template <bool BF16, int DM>
__global__ __launch_bounds__(kThreads, 2) void attn_rows_kernel(AttendArgs a, AttendPlan pl, Partial ws) {
    constexpr int R = 16, T = kTerms<BF16>, KS = DM / 32, VT = DM / 16;
    // The maximum lags by at most 2^kLag. f16 weights reach from 2^kTop to 2^15, as
    // far from the type's smallest step as it allows: their second term rounds at
    // 2^-25, 2^-36 of the row's largest. That counts where the row's weight is on a
    // key whose value is near zero (the first position of many a sequence) and its
    // output is what small weights make of the others. Of 4096 keys 14 nats below
    // such a key 2.8e-4 were lost with a top of 2^7, a lag of 2^8 and truncated
    // terms, and 4e-6, the scores' own rounding, are now; the shorter lag takes
    // 0.3% of a prompt, one of 2^2 2%.
    constexpr float kTop = BF16 ? 0.f : 11.f, kLag = BF16 ? 8.f : 4.f;
    constexpr int kPitch = DM + 4;  // LDS pitch of a joined row: 16 rows on different banks
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ float row_scale[R];
    __shared__ float wave_m[kWaves][R], wave_l[kWaves][R];
    const PagedCache &c = a.cache;
    const uint32_t l = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = l % 16, g = l / 16;
    const uint32_t split = blockIdx.x % pl.splits, unit = blockIdx.x / pl.splits;  // unit: tile and key head
    const uint32_t head = unit % c.kv_heads, tile = unit / c.kv_heads;
    const uint32_t group = a.heads / c.kv_heads, dim = c.dim;
    Tile t;
    if (!find_tile(c, group, R, tile, t)) {
        if (pl.splits > 1 && split == 0 && threadIdx.x < R) ws.place[size_t(unit) * R + threadIdx.x] = kNone;
        return;
    }
    const uint32_t in_tile = min(uint32_t(R), t.rows - t.row0);

    int lo_first, hi_first, lo_last, hi_last;
    visible(a, t, t.row0 / group, lo_first, hi_first);
    visible(a, t, (t.row0 + in_tile - 1) / group, lo_last, hi_last);
    const int base = lo_first / int(kBlock) * int(kBlock);
    const bool one_range = base + int64_t(pl.keys) >= hi_last;
    const int64_t from64 = base + int64_t(split) * pl.keys;
    const bool some = from64 < hi_last;
    const int from = some ? int(from64) : 0;
    const int to = some ? int(min(from64 + int64_t(pl.keys), int64_t(hi_last))) : 0;

    // Blocks w, w + 4, .. of the order. A block's keys are loaded while the
    // block before is weighed, its values while its scores are worked out, the
    // first ones while the queries are; the page after next is named by then.
    // Pages are read as constants (scalar loads), whose wait does not wait for
    // the blocks in flight. A page past the pool, or a block past the last,
    // reads as zeros: no memory is touched.
    const Order order(from, to, lo_last, hi_first);
    const auto *table = (const __attribute__((address_space(4))) uint32_t *)(c.table + size_t(t.seq) * c.columns);
    const uint32_t page_shift = __builtin_ctz(c.page);
    auto page_of = [&](int key0) { return table[uint32_t(key0) >> page_shift]; };
    auto rsrc_of = [&](const uint16_t *pool, uint32_t named, int key0, bool real) {
        const bool held = real && named < c.pages;
        const size_t at = attn::block_at(c, held ? named : 0, head, (uint32_t(key0) & (c.page - 1)) / kBlock);
        return block_rsrc(pool, at, held ? dim * kBlock * 2 : 0);
    };
    int at = int(w), key0 = 0, next_key = 0;
    uint32_t named = 0, next = 0;
    if (at < order.count) {
        key0 = order.key(at);
        next_key = order.key(at + kWaves);
        named = page_of(key0);
        next = page_of(next_key);
    }

    // The queries' loads go out before the blocks': thread (row % 16, p) has
    // chunks p and p + 16 of 8 dims.
    constexpr int CH = (DM / 8 + 15) / 16;
    const uint32_t qn = threadIdx.x / 16, qp = threadIdx.x % 16;
    float x[CH][8];
    const uint32_t q_row = t.row0 + min(qn, in_tile - 1);
    const float *q_own = a.q + size_t(t.first_token + q_row / group) * a.q_stride + size_t(head * group + q_row % group) * dim;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const uint32_t ch = qp + 16 * k;
        const f4 none = {0.f, 0.f, 0.f, 0.f};
        const bool in = qn < in_tile && ch * 8 < dim;
        const float *at = q_own + (ch * 8 < dim ? ch * 8 : 0);
        const f4 x0 = *reinterpret_cast<const f4u *>(at), x1 = *reinterpret_cast<const f4u *>(at + 4);
        *reinterpret_cast<f4 *>(x[k]) = in ? x0 : none;
        *reinterpret_cast<f4 *>(x[k] + 4) = in ? x1 : none;
    }

    u4 k[KS][2];
    auto load_keys = [&](uint32_t named, int key0, bool real) {
        const auto r = rsrc_of(c.k, named, key0, real);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int i = 0; i < 2; ++i) k[s][i] = load16(r, (g * 32 + n) * 16, s * 2048 + i * 256);
        }
    };
    // Dims past the head's own take other values or zeros, and are not kept.
    u4 v[VT];
    auto load_values = [&](uint32_t named, int key0, bool real) {
        const auto r = rsrc_of(c.v, named, key0, real);
#pragma unroll
        for (int d = 0; d < VT; ++d) v[d] = load16(r, (g * dim + n) * 16, d * 256);
    };
    if (at < order.count) {
        load_keys(named, key0, true);
        load_values(named, key0, true);
    }

    // The queries, as operands.
    u4 *qs = reinterpret_cast<u4 *>(lds);  // [KS][T][64 lanes]
    float q_most = 0.f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[k][j] *= a.scale * kLog2e;
            q_most = fmaxf(q_most, fabsf(x[k][j]));
        }
    }
    int e = 0;
    if constexpr (!BF16) {
#pragma unroll
        for (int d = 1; d < 16; d *= 2) q_most = fmaxf(q_most, __shfl_xor(q_most, d));
        if (q_most > 0.f && q_most < INFINITY) e = query_exponent(q_most);
    }
    if (qp == 0) row_scale[qn] = ldexpf(1.f, e);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const uint32_t ch = qp + 16 * k;
        if (ch >= DM / 8) continue;
        if constexpr (!BF16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[k][j] = ldexpf(x[k][j], -e);
        }
        u4 terms[T];
        split8<BF16>(x[k], terms);
#pragma unroll
        for (int i = 0; i < T; ++i) qs[(ch / 4 * T + i) * 64 + (ch % 4) * 16 + qn] = terms[i];
    }
    __syncthreads();

    // What the lane's row may see.
    int lo, hi;
    visible(a, t, (t.row0 + min(n, in_tile - 1)) / group, lo, hi);
    const float rs = row_scale[n];
    float m = -INFINITY, off = kTop, sum = 0.f;  // off: kTop - m
    bool deep = false, gap = false;              // the wave has met a score of minus infinity, a page past the pool
    // Of a lane's outputs, those that saw a value that is not finite.
    uint32_t poison[(VT + 7) / 8] = {};
    f4 o[VT];
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = f4{0.f, 0.f, 0.f, 0.f};

    auto block = [&](auto edge) {
        const bool held = named < c.pages;
        // The queries' operands come from LDS for every block where they and
        // the block do not fit the registers together.
        uint32_t ql = l;
        if constexpr (DM == 256) asm volatile("" : "+v"(ql));
        f4 scores[2] = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int i = 0; i < T; ++i) {
                const u4 q = qs[(s * T + i) * 64 + ql];
#pragma unroll
                for (int j = 0; j < 2; ++j) scores[j] = mfma16<BF16>(k[s][j], q, scores[j]);
            }
            // Not all of them on their way at once, which would not fit.
            if (DM == 256 && s % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
        const bool more = at + kWaves < order.count;
        const int key_now = key0;
        if constexpr (edge()) {
            // Values that no row sees may be anything: zero them.
            const u4 kept = halves_of(key_now + 8 * int(g), lo_first, hi_last);
#pragma unroll
            for (int d = 0; d < VT; ++d) v[d] &= kept;
            if (lo_first != lo_last || hi_first != hi_last) {
                // One that is not finite and that only some rows see must not
                // even meet the others' zero weights: it is taken out, and the
                // rows that see it (by a product of its place and what they
                // see) become NaN.
                us2 largest = {0, 0};
#pragma unroll
                for (int d = 0; d < VT; ++d) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) largest = larger(largest, v[d][i]);
                }
                if (__ballot(has_not_finite<BF16>(largest)) != 0) {
#pragma unroll
                    for (int d = 0; d < VT; ++d) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[d][i] &= ~not_finite<BF16>(v[d][i]);
                    }
                    const auto again = rsrc_of(c.v, named, key_now, true);
                    const u4 seen = ones_of<BF16>(key_now + 8 * int(g), lo, hi);
#pragma unroll
                    for (int d8 = 0; d8 < VT; d8 += 8) {
#pragma unroll 1
                        for (int d = 0; d < 8 && d8 + d < VT; ++d) {
                            u4 bad = load16(again, (g * dim + n) * 16, (d8 + d) * 256) & kept;
#pragma unroll
                            for (int i = 0; i < 4; ++i) bad[i] = not_finite<BF16>(bad[i]) & kOne<BF16>;
                            const f4 count = mfma16<BF16>(bad, seen, f4{0.f, 0.f, 0.f, 0.f});
                            uint32_t bits = 0;
#pragma unroll
                            for (int i = 0; i < 4; ++i) bits |= count[i] > 0.f ? 1u << i : 0u;
                            poison[d8 / 8] |= bits << (4 * d);
                        }
                    }
                }
            }
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = scores[0][i], p[4 + i] = scores[1][i];
        // Of the keys that are seen the least score: minus infinity for some infinite
        // keys.
        float least = INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int key = key_now + 8 * int(g) + e;
            const bool seen = !edge() || (key >= lo && key < hi);
            least = fminf(least, seen ? p[e] : INFINITY);
            if (!seen) p[e] = -INFINITY;
        }
        float most = p[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) most = fmaxf(most, p[e]);
        most *= rs;
        auto small = [&] { return least == -INFINITY; };
        if (held & (__ballot((most > m + kLag) | small()) != 0)) {
            if (__ballot(most > m + kLag) != 0) {
                most = fmaxf(most, __shfl_xor(most, 16));
                most = fmaxf(most, __shfl_xor(most, 32));
                const float up = fmaxf(m, most);
                const float f = up > m ? exp2f(m - up) : 1.f;
                m = up;
                off = kTop - (m == -INFINITY ? 0.f : m);
                sum *= f;
#pragma unroll
                for (int d = 0; d < VT; ++d) o[d] *= f;
            }
            deep |= __ballot(small()) != 0;
        }
        // A page past the pool has no weight.
        const float less = held ? off : -INFINITY;
        gap |= !held;
        load_keys(next, next_key, more);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(p[e], rs, less));
            sum += p[e];
        }
        u4 pt[T];
        split8<BF16>(p, pt);
#pragma unroll
        for (int d = 0; d < VT; ++d) {
#pragma unroll
            for (int i = 0; i < T; ++i) o[d] = mfma16<BF16>(v[d], pt[i], o[d]);
        }
        load_values(next, next_key, more);
        at += kWaves;
        key0 = next_key;
        named = next;
        next_key = order.key(at + kWaves);
        next = page_of(next_key);
    };
    while (at < order.edges) block(std::true_type{});
    while (at < order.count) block(std::false_type{});
    // A query that is not finite gives the blocks of pages past the pool weights of
    // NaN: a row that sees no key is zero all the same.
    if (gap && __ballot(sum != sum) != 0) {
        bool sees = false;
        for (int i = int(w); i < order.count; i += kWaves) {
            const int key = order.key(i);
            sees |= page_of(key) < c.pages && max(lo, key) < min(hi, key + int(kBlock));
        }
        if (!sees) {
            m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int d = 0; d < VT; ++d) o[d] = f4{0.f, 0.f, 0.f, 0.f};
        }
    }
    if (deep) {
        for (int i = int(w); i < order.count; i += kWaves) {
            const int key = order.key(i);
            if (sees_bad_key<BF16>(rsrc_of(c.k, page_of(key), key, true), dim, lo - key, hi - key)) sum = __builtin_nanf("");
        }
    }

    // Join the waves. (What a thread is in the workgroup is worked out again:
    // the loop needs the registers.)
    uint32_t thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const uint32_t jl = thread % 64, jn = jl % 16, jg = jl / 16, rn = thread / 16, rp = thread % 16;
    float *os = reinterpret_cast<float *>(lds);  // [kWaves][16][kPitch]
    float all = sum;
    all += __shfl_xor(all, 16);
    all += __shfl_xor(all, 32);
    __syncthreads();
    uint32_t poisoned = poison[0];
#pragma unroll
    for (int d = 8; d < VT; d += 8) poisoned |= poison[d / 8];
    if (__ballot(poisoned != 0) != 0) {
#pragma unroll
        for (int d = 0; d < VT; ++d) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (poison[d / 8] >> (d % 8 * 4 + i) & 1) o[d][i] = __builtin_nanf("");
        }
    }
#pragma unroll
    for (int d = 0; d < VT; ++d) *reinterpret_cast<f4 *>(os + (w * 16 + jn) * kPitch + 16 * d + 4 * jg) = o[d];
    if (jg == 0) {
        wave_m[w][jn] = m;
        wave_l[w][jn] = all;
    }
    __syncthreads();
    // Sixteen threads a row, four dims at a time.
    const bool real = rn < in_tile;
    const uint32_t row = t.row0 + rn, token = t.first_token + row / group, qh = head * group + row % group;
    if (pl.splits > 1 && split == 0 && rp == 0)
        ws.place[size_t(unit) * R + rn] = one_range || !real ? kNone : token * a.heads + qh;
    if (!real || (one_range && split > 0)) return;
    float top = wave_m[0][rn], f[kWaves], joined = 0.f;
#pragma unroll
    for (int k = 1; k < kWaves; ++k) top = fmaxf(top, wave_m[k][rn]);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        const float mk = wave_m[k][rn], lk = wave_l[k][rn];
        f[k] = mk == -INFINITY ? (lk == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mk - top);
        joined += f[k] * lk;
    }
    const size_t part = (size_t(unit) * pl.splits + split) * R + rn;
    const float over = joined == 0.f ? 0.f : 1.f / joined;
    float *y = one_range ? a.out + size_t(token) * a.out_stride + size_t(qh) * dim : ws.o + part * DM;
#pragma unroll
    for (uint32_t d = rp * 4; d < DM; d += 64) {
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kWaves; ++k) acc += f[k] * *reinterpret_cast<const f4 *>(os + (k * 16 + rn) * kPitch + d);
        if (!one_range) {
            if (joined != 0.f) *reinterpret_cast<f4 *>(y + d) = acc;
        } else if (d < dim) {
            *reinterpret_cast<f4u *>(y + d) = acc * over;
        }
    }
    if (!one_range && rp == 0) ws.ml[part] = make_float2(top, joined);
}

// Many rows: 128 rows a workgroup, 32 a wave, which keeps its queries' operands
// and its O in registers; blocks of 32 keys come through LDS, each read by all
// four waves. v_mfma_f32_32x32x16 (A row and B column lane % 32, K chunk
// lane / 32; D[i][j] in lane j + 32 (i / 4 % 2), element i % 4 + 4 (i / 8)), keys
// dealt so that lane (n, g) ends with row n's scores of keys 16s + 8g + 0..7, as
// P^T has to stand for step s of O^T = V^T P^T.
//
// The scores of block i + 1 are worked out while block i's are weighed: matrix
// and vector instructions that do not wait for each other, and that stand in
// the order in which they should issue, a step's operands read from LDS kAhead
// steps before (scheduling barriers keep it). Blocks go from memory straight to
// a ring of three in LDS, two iterations ahead of their use, with one barrier
// a block.
//
// The matrix cores bound it, at the card's power: their clock falls as they
// fill. A prompt of 4100 tokens of 32/8 heads of 128 (f16) takes 278 us, 495
// TFLOP/s of the formula and 990 of the instructions, as each operand of FP32
// is two terms; 512 tokens of 24/4 heads of 256 over 16513 keys (bf16, three
// terms) 529 us, 387 and 1160. A large matrix product reaches 1166 in f16 and
// 1227 in bf16.
template <bool BF16, int DM>
__global__ __launch_bounds__(kThreads, DM == 256 ? 1 : 2) void attn_tile_kernel(AttendArgs a, AttendPlan pl, Partial ws) {
    constexpr int R = 32 * kWaves, T = kTerms<BF16>, KS = DM / 16, VT = DM / 32;
    constexpr float kTop = BF16 ? 0.f : 11.f, kLag = BF16 ? 8.f : 4.f;
    constexpr int kChunks = DM * 4;             // 16-byte chunks of a block
    constexpr int kEach = kChunks / kThreads;   // a thread's
    constexpr uint32_t kBytes = kChunks * 16;
    constexpr int kAhead = 4;
    // Of a query's terms two stay in registers; the third of bf16 would not fit
    // beside O and waits in LDS, but for the last steps of the largest heads,
    // for which LDS is too small.
    constexpr int kLow = T < 3 ? 0 : DM == 256 ? KS - 2 : KS;
    extern __shared__ __align__(16) unsigned char lds[];  // three blocks of keys, three of values, kLow steps a wave
    u4 *ql = reinterpret_cast<u4 *>(lds + 6 * kBytes) + (threadIdx.x / 64) * (kLow * 64);
    __shared__ int apart;
    const PagedCache &c = a.cache;
    const uint32_t l = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t n = l % 32, g = l / 32;
    const uint32_t split = blockIdx.x % pl.splits, unit = blockIdx.x / pl.splits;  // unit: tile and key head
    const uint32_t head = unit % c.kv_heads, tile = unit / c.kv_heads;
    const uint32_t group = a.heads / c.kv_heads, dim = c.dim;
    Tile t;
    // The last tiles first: they see the most keys.
    if (!find_tile(c, group, R, pl.tiles - 1 - tile, t)) {
        if (pl.splits > 1 && split == 0 && threadIdx.x < R) ws.place[size_t(unit) * R + threadIdx.x] = kNone;
        return;
    }
    const uint32_t in_tile = min(uint32_t(R), t.rows - t.row0);
    // Keys that some row of the tile sees, and that all do.
    int lo_tile, hi_tile, lo_most, hi_least;
    visible(a, t, t.row0 / group, lo_tile, hi_least);
    visible(a, t, (t.row0 + in_tile - 1) / group, lo_most, hi_tile);
    const int base = lo_tile / int(kBlock) * int(kBlock);
    const bool one_range = base + int64_t(pl.keys) >= hi_tile;
    const int64_t from64 = base + int64_t(split) * pl.keys;
    const bool some = from64 < hi_tile;
    const int from = some ? int(from64) : 0;
    const int to = some ? int(min(from64 + int64_t(pl.keys), int64_t(hi_tile))) : 0;

    // This wave's rows.
    const uint32_t r0 = 32 * w, r = r0 + n;
    int lo, hi;
    visible(a, t, (t.row0 + min(r, in_tile - 1)) / group, lo, hi);
    if (threadIdx.x == 0) apart = -1;

    const Order order(from, to, lo_most, hi_least);
    // A page's name: 64 of them wait in a register, so that no scalar load's
    // wait falls among those for LDS.
    const uint32_t *table = c.table + size_t(t.seq) * c.columns;
    const uint32_t page_shift = __builtin_ctz(c.page);
    uint32_t names = 0, names_at = 0x80000000u;
    auto page_of = [&](int key0) {
        const uint32_t column = uint32_t(key0) >> page_shift;
        if (column - names_at >= 64) {
            names_at = column;
            names = table[min(column + l, c.columns - 1)];
            asm volatile("s_waitcnt vmcnt(0)" : "+v"(names));  // here, not at each use
        }
        return uint32_t(__builtin_amdgcn_readlane(names, column - names_at));
    };
    const uint32_t lds0 = uint32_t(uintptr_t((__attribute__((address_space(3))) unsigned char *)lds));
    // The number of the order's i-th block in either pool, kNone for one of a
    // page past the pool.
    const uint32_t block_bytes = dim * kBlock * 2, page_blocks = c.page / kBlock;
    auto place_of = [&](int i) {
        const int key = order.key(i);
        const uint32_t named = page_of(key), in_page = (uint32_t(key) & (c.page - 1)) / kBlock;
        return named < c.pages ? (named * c.kv_heads + head) * page_blocks + in_page : kNone;
    };
    auto words_of = [&](const uint16_t *pool, uint32_t at) {
        const bool held = at != kNone;
        const uint64_t p = reinterpret_cast<uint64_t>(pool) + uint64_t(held ? at : 0) * block_bytes;
        return u4{uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(p))),
                  uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(p >> 32) & 0xFFFFu)), held ? block_bytes : 0, kRsrcWord3};
    };
    // That block to the ring's slot at byte `to`; zeros from nowhere.
    const uint32_t own_bytes = l * 16 + w * 1024, lds_own = lds0 + w * 1024;
    auto fetch = [&](const uint16_t *pool, uint32_t at, uint32_t to) {
        const u4 words = words_of(pool, at);
#pragma unroll
        for (int i = 0; i < kEach; ++i) dma16(words, own_bytes, i * kWaves * 1024, lds_own + to + i * kWaves * 1024);
    };
    // Values that no row of the tile sees may be anything: zeros. Those that are
    // not finite in a block that some rows see in part are zeros too, and
    // `apart` says that there are some.
    auto clean_values = [&](uint32_t at, int key0) {
        u4 *vb = reinterpret_cast<u4 *>(lds + at);
        uint32_t some_bad = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const uint32_t ch = threadIdx.x + i * kThreads;
            u4 v = vb[ch] & halves_of(key0 + 8 * int(ch / dim), lo_tile, hi_tile);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t bad = not_finite<BF16>(v[j]);
                v[j] &= ~bad;
                some_bad |= bad;
            }
            vb[ch] = v;
        }
        if (some_bad) apart = key0;
    };

    // Blocks, by their place in the order: this one and the three after; the
    // ring's slots of keys and of values in the order of their use.
    uint32_t at0 = kNone, at1 = kNone, at2 = kNone, at3 = kNone;
    uint32_t k0 = 0, k1 = kBytes, k2 = 2 * kBytes, v0 = 3 * kBytes, v1 = 4 * kBytes, v2 = 5 * kBytes;
    // What no load writes (dims past the head's) is zero.
    if (dim < DM)
        for (uint32_t i = threadIdx.x; i < 6 * kChunks; i += kThreads) reinterpret_cast<u4 *>(lds)[i] = u4{0, 0, 0, 0};
    lds_barrier();
    if (order.count > 0) {
        at0 = place_of(0), at1 = place_of(1), at2 = place_of(2), at3 = place_of(3);
        fetch(c.k, at0, k0);
        fetch(c.k, at1, k1);
        fetch(c.v, at0, v0);
        fetch(c.k, at2, k2);
        fetch(c.v, at1, v1);
    }

    // Queries.
    u4 q[KS][2], q_last[2];
    float rs = 1.f;
    {
        const uint32_t row = t.row0 + min(r, in_tile - 1);
        const float *src = a.q + size_t(t.first_token + row / group) * a.q_stride + size_t(head * group + row % group) * dim;
        f4 x[KS][2];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int i = 0; i < 2; ++i) x[s][i] = *reinterpret_cast<const f4u *>(src + min(16 * s + 8 * g, dim - 8) + 4 * i);
        }
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const float f = 16 * s + 8 * g < dim ? a.scale * kLog2e : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[s][i] = f == 0.f ? f4{0.f, 0.f, 0.f, 0.f} : x[s][i] * f;
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fmaxf(most, fabsf(x[s][i][j]));
            }
        }
        int e = 0;
        if constexpr (!BF16) {
            most = fmaxf(most, __shfl_xor(most, 32));
            if (most > 0.f && most < INFINITY) e = query_exponent(most);
            rs = ldexpf(1.f, e);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = BF16 ? x[s][j / 4][j % 4] : ldexpf(x[s][j / 4][j % 4], -e);
            u4 terms[T];
            split8<BF16>(y, terms);
            q[s][0] = terms[0];
            q[s][1] = terms[1];
            if (s < kLow) ql[s * 64 + l] = terms[T - 1];
            if (T == 3 && s >= kLow) q_last[T == 3 ? s - kLow : 0] = terms[T - 1];
        }
    }
    f16v o[VT];
#pragma unroll
    for (int d = 0; d < VT; ++d) o[d] = f16v{};
    float m = -INFINITY, sum = 0.f;
    uint32_t poison[(VT + 1) / 2] = {};  // of a lane's outputs, those that saw a value that is not finite

    const uint32_t key_at = g * 32 + (n & 7) + 2 * (n & 8) + (n & 16) / 2;  // where A's row n is in a key chunk pair
    auto key_operand = [&](uint32_t at, int s) { return reinterpret_cast<const u4 *>(lds + at)[s * 64 + key_at]; };
    auto value_operand = [&](uint32_t at, int i) {
        return reinterpret_cast<const u4 *>(lds + at)[(i / VT * 2 + g) * dim + 32 * (i % VT) + n];
    };
    auto low_operand = [&](int s) { return s < kLow ? ql[s * 64 + l] : q_last[s < kLow ? 0 : s - kLow]; };
    // A matrix instruction that adds to the one before it waits half as long
    // again: two sums in turn where there are registers for it (of 128 dims
    // there are not, but two waves on a SIMD).
    constexpr int SUMS = DM == 128 ? 1 : 2;
    auto score_step = [&](f16v (&x)[SUMS], int s, u4 k, u4 low) {
#pragma unroll
        for (int i = 0; i < T; ++i) {
            f16v &sum = x[(s * T + i) % SUMS];
            sum = mfma32<BF16>(k, i == 2 ? low : q[s][i == 2 ? 0 : i], sum);
        }
    };
    auto total = [](const f16v (&x)[SUMS]) { return SUMS == 2 ? x[0] + x[SUMS - 1] : x[0]; };

    auto largest = [](f16v x) {
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, x[i]);
        return most;
    };
    f16v next = {};
    float next_most = 0.f;
    float least_to = 0.f;            // the least exponent of a weight, but for those of the masked blocks
    bool deep = false, gap = false;  // the wave has met a score of minus infinity in these, a page past the pool
    if (order.count > 0) {
        wait_dma<4 * kEach>();
        lds_barrier();
        f16v first[SUMS] = {};
#pragma unroll
        for (int s = 0; s < KS; ++s) score_step(first, s, key_operand(k0, s), low_operand(s));
        next = total(first);
        next_most = largest(next);
    }
    // Of the largest heads, O has its place in the accumulation registers: left
    // to itself the compiler moves it to the others and back for every block.
    auto stays = [](f16v &x) {
        if constexpr (DM == 256) asm volatile("" : "+a"(x));
    };
    int at = 0;
    auto block = [&](auto edge) {
        f16v p = next;
#pragma unroll
        for (int d = 0; d < VT; ++d) stays(o[d]);
        wait_dma<2 * kEach>();  // the next keys and these values are there
        lds_barrier();
        const bool held = at0 != kNone;
        gap |= !held;
        float most = next_most;
        int key0 = 0;
        if constexpr (edge()) {
            key0 = order.key(at);
            clean_values(v0, key0);
            float least = INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = key0 + 16 * (i / 8) + 8 * int(g) + i % 8;
                const bool seen = key >= lo && key < hi;
                least = fminf(least, seen ? p[i] : INFINITY);
                if (!seen) p[i] = -INFINITY;
            }
            deep |= __ballot(least == -INFINITY) != 0;
            most = largest(p);
        }
        most = held ? most * rs : -INFINITY;
        if (__ballot(most > m + kLag) != 0) {
            most = fmaxf(most, __shfl_xor(most, 32));
            const float up = fmaxf(m, most);
            const float f = up > m ? exp2f(m - up) : 1.f;
            m = up;
            sum *= f;
#pragma unroll
            for (int d = 0; d < VT; ++d) {
                o[d] *= f;
                stays(o[d]);
            }
        }
        const float off = held ? kTop - (m == -INFINITY ? 0.f : m) : -INFINITY;
        if constexpr (edge()) lds_barrier();

        // The next block's scores, and this one's weights between them; then
        // the weights times the values, two tiles of dims in turn.
        u4 ring[kAhead], low[2];
        auto operand = [&](int i) { return i < KS ? key_operand(k1, i) : value_operand(v0, i - KS); };
        auto take = [&](int i) {
            const u4 x = ring[i % kAhead];
            if (i + kAhead < KS + 2 * VT) ring[i % kAhead] = operand(i + kAhead);
            return x;
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i) ring[i] = operand(i);
        if constexpr (T == 3) low[0] = low_operand(0), low[1] = low_operand(1);
        __builtin_amdgcn_sched_barrier(0);
        f16v ahead[SUMS] = {};
        uint32_t at4 = kNone;
        u4 pt[2][T];
        float x[8];
        auto weigh = [&](int j) {
            const float to = fmaf(p[j], rs, off);
            x[j % 8] = __builtin_amdgcn_exp2f(to);
            if constexpr (!edge()) least_to = fminf(least_to, to);
            sum += x[j % 8];
            if (j % 8 == 7) split8<BF16>(x, pt[j / 8]);
        };
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            score_step(ahead, i, take(i), low[i % 2]);
            if constexpr (T == 3)
                if (i + 2 < KS) low[i % 2] = low_operand(i + 2);
            // The first half of the weights here, the other one while the first
            // meets its values.
#pragma unroll
            for (int j = i * 8 / KS; j < (i + 1) * 8 / KS; ++j) weigh(j);
            if (KS < 8 && i == 0) fetch(c.k, at3, k0);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 2 * VT; i += 2) {
            const int s = i / VT, d = i % VT;
            const u4 va = take(KS + i), vb = take(KS + i + 1);
#pragma unroll
            for (int j = 0; j < T; ++j) {
                o[d] = mfma32<BF16>(va, pt[s][j], o[d]);
                o[d + 1] = mfma32<BF16>(vb, pt[s][j], o[d + 1]);
            }
            if (s == 0) {
#pragma unroll
                for (int j = 8 + d * 8 / VT; j < 8 + (d + 2) * 8 / VT; ++j) weigh(j);
            }
            if (KS >= 8 && i == 0) fetch(c.k, at3, k0);
            if (i == VT) next = total(ahead);
            if (i == VT) fetch(c.v, at2, v2);
            if (i == 2 * VT - 2) {
                at4 = place_of(at + 4);
                next_most = largest(next);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (edge()) {
            if (apart == key0) {
                // The rows that see one of the values left out become NaN.
                const auto again = block_rsrc(c.v, size_t(at0) * (dim * kBlock), block_bytes);
#pragma unroll
                for (int d2 = 0; d2 < VT; d2 += 2) {
#pragma unroll 1
                    for (int d = 0; d < 2; ++d) {
                        f16v count = {};
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            u4 bad = load16(again, ((2 * s + g) * dim + n) * 16, (d2 + d) * 512);
#pragma unroll
                            for (int i = 0; i < 4; ++i) bad[i] = not_finite<BF16>(bad[i]) & kOne<BF16>;
                            count = mfma32<BF16>(bad, ones_of<BF16>(key0 + 16 * s + 8 * int(g), lo, hi), count);
                        }
                        uint32_t bits = 0;
#pragma unroll
                        for (int i = 0; i < 16; ++i) bits |= count[i] > 0.f ? 1u << i : 0u;
                        poison[d2 / 2] |= bits << (16 * d);
                    }
                }
            }
        }
        at0 = at1, at1 = at2, at2 = at3, at3 = at4;
        const uint32_t used_k = k0, used_v = v0;
        k0 = k1, k1 = k2, k2 = used_k;
        v0 = v1, v1 = v2, v2 = used_v;
        ++at;
    };
    while (at < order.edges) block(std::true_type{});
    while (at < order.count) block(std::false_type{});
    wait_dma<0>();  // LDS is given back
    // As in the rows kernel: rows that see no key, and infinite keys.
    if (gap && __ballot(sum != sum) != 0) {
        bool sees = false;
        for (int i = 0; i < order.count; ++i) {
            const int key = order.key(i);
            sees |= place_of(i) != kNone && max(lo, key) < min(hi, key + int(kBlock));
        }
        if (!sees) {
            m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int d = 0; d < VT; ++d) o[d] = f16v{};
        }
    }
    if (deep || __ballot(least_to == -INFINITY) != 0) {
        for (int i = 0; i < order.count; ++i) {
            const int key = order.key(i);
            const uint32_t named = place_of(i);
            if (named == kNone) continue;
            if (sees_bad_key<BF16>(block_rsrc(c.k, size_t(named) * (dim * kBlock), block_bytes), dim, lo - key, hi - key))
                sum = __builtin_nanf("");
        }
    }

#pragma unroll
    for (int d = 0; d < VT; ++d) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (poison[d / 2] >> (d % 2 * 16 + i) & 1) o[d][i] = __builtin_nanf("");
    }
    float all = sum + __shfl_xor(sum, 32);
    const bool real = r < in_tile;
    const uint32_t row = t.row0 + min(r, in_tile - 1), token = t.first_token + row / group, qh = head * group + row % group;
    if (one_range) {
        if (split == 0 && real) {
            const float f = all == 0.f ? 0.f : 1.f / all;
            float *y = a.out + size_t(token) * a.out_stride + size_t(qh) * dim;
#pragma unroll
            for (int d = 0; d < VT; ++d) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t at = 32 * d + 8 * i + 4 * g;
                    if (at >= dim) continue;
                    const f4 x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                    *reinterpret_cast<f4u *>(y + at) = x * f;
                }
            }
        }
    } else if (real) {
        const size_t part = (size_t(unit) * pl.splits + split) * R + r;
        if (all != 0.f) {
#pragma unroll
            for (int d = 0; d < VT; ++d) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f4 *>(ws.o + part * DM + 32 * d + 8 * i + 4 * g) =
                        f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            }
        }
        if (g == 0) ws.ml[part] = make_float2(m, all);
    }
    if (pl.splits > 1 && split == 0 && g == 0) ws.place[size_t(unit) * R + r] = one_range || !real ? kNone : token * a.heads + qh;
}

// Adds the ranges of a row up. WIDE: a workgroup a row, every wave a quarter of
// the ranges, whose loads depend on nothing and are all in flight at once. For
// few ranges a wave a row (one token of 24/4 heads of 256 over 2001 keys, 4, 8 and
// 16 ranges, rows kernel and join: 16.2, 13.5 and 12.2 us, as WIDE 16.2, 13.0 and
// 11.4; 12288 rows of 256 dims in 5 ranges, the join alone: 15.8, as WIDE 18.6).
// Of its 3 us with few rows most is one more launch.
template <int DM, bool WIDE>
__global__ __launch_bounds__(kThreads) void attn_join_kernel(AttendArgs a, AttendPlan pl, Partial ws, uint32_t rows) {
    constexpr int E = DM / 64, kFirst = 8;
    typedef float fe __attribute__((ext_vector_type(E)));
    __shared__ float weight[kWaves][WIDE ? kMaxSplits : kFewSplits], part_o[kWaves][WIDE ? DM : 1];
    const uint32_t l = threadIdx.x % 64, w = threadIdx.x / 64;
    const uint32_t at_row = WIDE ? blockIdx.x : blockIdx.x * kWaves + w;
    if (at_row >= rows) return;
    const uint32_t unit = at_row / pl.rows, r = at_row % pl.rows;
    const size_t first = size_t(unit) * pl.splits * pl.rows + r;
    // What the wave adds first is loaded before its weights are known.
    const uint32_t from = WIDE ? w : 0, by = WIDE ? kWaves : 1;
    const fe *o = reinterpret_cast<const fe *>(ws.o + first * DM) + l;
    auto part_of = [&](uint32_t s) { return o[size_t(s) * pl.rows * (DM / E)]; };
    auto ml_of = [&](uint32_t s) { return ws.ml[first + size_t(s) * pl.rows]; };
    const uint32_t place = ws.place[at_row];
    const float2 own = l < pl.splits ? ml_of(l) : make_float2(-INFINITY, 0.f);
    fe ahead[kFirst];
#pragma unroll
    for (uint32_t i = 0; i < kFirst; ++i) ahead[i] = part_of(min(from + i * by, pl.splits - 1));

    float top = own.x, all = 0.f;
    for (uint32_t s = l + 64; s < pl.splits; s += 64) top = fmaxf(top, ml_of(s).x);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    // A range that saw nothing (its sum is 0) left no row.
    auto weigh = [&](uint32_t s, float2 ml) {
        const float f = ml.y == 0.f ? 0.f : ml.x == -INFINITY ? 1.f : exp2f(ml.x - top);
        weight[w][s] = ml.y == 0.f ? -1.f : f;
        all += f * ml.y;
    };
    if (l < pl.splits) weigh(l, own);
    for (uint32_t s = l + 64; s < pl.splits; s += 64) weigh(s, ml_of(s));
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    fe acc = {};
    auto add = [&](uint32_t s, fe x) {
        const float f = weight[w][s];
        if (f >= 0.f || f != f) acc += f * x;
    };
#pragma unroll
    for (uint32_t i = 0; i < kFirst; ++i)
        if (from + i * by < pl.splits) add(from + i * by, ahead[i]);
#pragma unroll 8
    for (uint32_t s = from + kFirst * by; s < pl.splits; s += by) add(s, part_of(s));
    const float f = all == 0.f ? 0.f : 1.f / all;
    if constexpr (WIDE) {
        *reinterpret_cast<fe *>(&part_o[w][l * E]) = acc;
        __syncthreads();
    }
    if (place == kNone) return;
    float *y = a.out + size_t(place / a.heads) * a.out_stride + size_t(place % a.heads) * a.cache.dim;
    if constexpr (WIDE) {
        const uint32_t d = threadIdx.x;
        if (d < a.cache.dim) y[d] = (part_o[0][d] + part_o[1][d] + part_o[2][d] + part_o[3][d]) * f;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (l * E + e < a.cache.dim) y[l * E + e] = acc[e] * f;
    }
}

uint32_t wide_dim(uint32_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

Partial parts(const AttendArgs &a, const AttendPlan &pl, void *ws) {
    const size_t rows = size_t(pl.tiles) * a.cache.kv_heads * pl.splits * pl.rows;
    Partial p;
    p.o = static_cast<float *>(ws);
    p.ml = reinterpret_cast<float2 *>(p.o + rows * wide_dim(a.cache.dim));
    p.place = reinterpret_cast<uint32_t *>(p.ml + rows);
    return p;
}

size_t workspace_of(const AttendArgs &a, const AttendPlan &pl) {
    if (pl.splits == 1) return 0;
    const size_t units = size_t(pl.tiles) * a.cache.kv_heads;
    return units * pl.rows * (size_t(pl.splits) * (wide_dim(a.cache.dim) + 2) + 1) * 4;
}

template <bool BF16, int DM>
hipError_t launch_rows(const AttendArgs &a, const AttendPlan &pl, const Partial &ws, hipStream_t stream) {
    const size_t queries = size_t(DM / 32) * kTerms<BF16> * 1024;
    const size_t joined = size_t(kWaves) * 16 * (DM + 4) * 4;
    const size_t lds = queries > joined ? queries : joined;
    const auto kernel = attn_rows_kernel<BF16, DM>;
    if (lds > 65536 - 2048) {
        const hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kernel), lds);
        if (e != hipSuccess) return e;
    }
    kernel<<<pl.tiles * a.cache.kv_heads * pl.splits, kThreads, lds, stream>>>(a, pl, ws);
    return hipGetLastError();
}

template <bool BF16, int DM>
hipError_t launch_dim(const AttendArgs &a, const AttendPlan &pl, const Partial &ws, hipStream_t stream) {
    hipError_t e;
    if (pl.rows == 16) {
        e = launch_rows<BF16, DM>(a, pl, ws, stream);
    } else {
        // Three blocks of keys and of values, and bf16's third query terms.
        constexpr size_t lds = 6 * DM * 64 + (BF16 ? kWaves * (DM == 256 ? DM - 32 : DM) * 64 : 0);
        const auto kernel = attn_tile_kernel<BF16, DM>;
        if (lds > 65536 - 2048) {
            e = raise_lds_limit(reinterpret_cast<const void *>(kernel), lds);
            if (e != hipSuccess) return e;
        }
        kernel<<<pl.tiles * a.cache.kv_heads * pl.splits, kThreads, lds, stream>>>(a, pl, ws);
        e = hipGetLastError();
    }
    if (e != hipSuccess || pl.splits == 1) return e;
    const uint32_t rows = pl.tiles * a.cache.kv_heads * pl.rows;
    if (pl.splits <= 4 || (pl.splits <= kFewSplits && rows >= 4096)) {
        attn_join_kernel<DM, false><<<(rows + kWaves - 1) / kWaves, kThreads, 0, stream>>>(a, pl, ws, rows);
    } else {
        attn_join_kernel<DM, true><<<rows, kThreads, 0, stream>>>(a, pl, ws, rows);
    }
    return hipGetLastError();
}

template <bool BF16>
hipError_t launch_type(const AttendArgs &a, const AttendPlan &pl, const Partial &ws, hipStream_t stream) {
    switch (wide_dim(a.cache.dim)) {
        case 64: return launch_dim<BF16, 64>(a, pl, ws, stream);
        case 128: return launch_dim<BF16, 128>(a, pl, ws, stream);
        default: return launch_dim<BF16, 256>(a, pl, ws, stream);
    }
}

}  // namespace

// The plan is the cheapest of an estimate over both kernels and their numbers
// of key ranges, from sizes alone. Fitted to MI355X timings (us), per dims 64,
// 128 and 256, bf16 and f16:
//   rows kernel  a workgroup takes `start`, `chain` for each round of its four
//                waves' blocks, and less by `fewer` where waves have none, as a
//                CU's cache then brings less; a CU works a tile of 16 rows
//                against a block off in `each` whatever is resident, and starts
//                a tile in 2; keys and values come in at 5.3 TB/s from 128
//                workgroups on, at half that from 37
//   tile kernel  10 for start and end, `chain` a block alone, `each` a block of
//                128 rows when the CU's two workgroups (one of 256 dims) overlap
//   join         3, and each range's rows written and read once
// Both sides where it decides, rows / tile kernel in its best number of ranges:
// 64 tokens of 24 heads of 256 over 4064 keys (bf16) 34 / 42 us, 150 over 4150 58
// / 69, 512 over 16512 569 / 540; one prompt of 32 heads of 128 (f16), 500 tokens
// 19 / 25, 1000 40 / 41, 2000 114 / 85, 4100 375 / 280.
// Ranges, in the rows kernel (four caches in turn): one token of 24/4 heads of 256
// over 32768 keys in 8, 16, 32, 64 and 128: 83, 50, 35, 33.5 and 35.5 us; over 4001
// in 16, 32 and 64: 13.9, 13.3 and 15.2; over 1001 in 1, 8, 16 and 32 (of one
// block): 17.6, 11.1, 10.6 and 10.5; over 101 in 1 and 4: 7.7 and 9.8; 32 sequences
// of 8 heads of 128 over up to 8001 in 1, 2 and 4: 106, 109 and 117.
AttendPlan plan_attend(const AttendArgs &a, const DeviceLimits &lim, size_t workspace_limit, uint32_t force_rows,
                       uint32_t force_splits) {
    const PagedCache &c = a.cache;
    const uint64_t group = a.heads / c.kv_heads;
    // Sequences with a row: at most n. Each takes whole tiles.
    const uint64_t n = c.seqs < c.tokens ? c.seqs : c.tokens;
    const int wide = wide_dim(c.dim) == 64 ? 0 : wide_dim(c.dim) == 128 ? 1 : 2;
    static constexpr double kRowsStart[3] = {4.5, 5.1, 6.3}, kRowsChain[3] = {0.39, 0.65, 1.45}, kRowsFewer[3] = {0.03, 0.07, 0.17};
    static constexpr double kTileChain[2][3] = {{0.95, 1.2, 2.0}, {1.0, 1.4, 2.4}};
    static constexpr double kRowsEach[2][3] = {{0.07, 0.19, 0.33}, {0.09, 0.21, 0.42}};
    static constexpr double kTileEach[2][3] = {{1.1, 1.05, 2.1}, {1.2, 1.45, 2.6}};
    const double cus = lim.num_cus;
    // Of the keys before a sequence's end, those that its average row sees.
    const double share = a.causal ? 1 - std::min(1.0, double(c.tokens) / n / a.max_keys) / 2 : 1;
    AttendPlan best;
    double least = 0;
    for (const uint32_t rows : {16u, 128u}) {
        if ((force_rows == 16 || force_rows == 128) && rows != force_rows) continue;
        AttendPlan pl;
        pl.rows = rows;
        const uint64_t by_rows = n + (c.tokens * group - n) / rows;
        const uint64_t by_token = c.tokens * ((group + rows - 1) / rows);
        pl.tiles = uint32_t(by_rows < by_token ? by_rows : by_token);
        // The keys that a tile's rows see, at most: with a window those of its
        // first row to those of its last.
        const uint64_t across = (rows + group - 1) / group + kBlock;
        const uint64_t keys = a.window && a.window + across < a.max_keys ? a.window + across : a.max_keys;
        // A range is a block for each wave, or several; in the rows kernel also
        // one or two blocks, which come through a CU's own cache the sooner.
        const uint64_t units = uint64_t(pl.tiles) * c.kv_heads, step = kWaves * kBlock;
        const uint64_t least_keys = rows == 16 ? kBlock : step;
        const uint64_t most = std::min<uint64_t>((keys + least_keys - 1) / least_keys, kMaxSplits);
        // Workgroups go to the eight XCDs in turn: tiles that read the same keys
        // share one's L2 if their distance is a multiple of eight (six tokens
        // of 24/4 heads over 16006 keys in 16, 18, 20 and 21 ranges: 23.8, 22.9,
        // 22.9 and 28.7 us; four sequences of four tokens over 6004 in 6, 7 and
        // 8: 33.3, 38.3 and 29.9).
        const bool shared = rows == 16 && c.tokens * group > n * rows;
        uint64_t before = 0;
        const uint64_t first = force_splits == 0 ? 1 : std::min<uint64_t>(force_splits, most);
        for (uint64_t s = first; s <= (force_splits == 0 ? most : first); s += s < 32 ? 1 : s / 8) {
            const uint64_t even = (keys + s - 1) / s;
            pl.keys = uint32_t(rows == 16 && even <= kBlock       ? kBlock
                               : rows == 16 && even <= 2 * kBlock ? 2 * kBlock
                                                                  : (even + step - 1) / step * step);
            pl.splits = uint32_t((keys + pl.keys - 1) / pl.keys);
            if (pl.splits == before) continue;
            const uint64_t streams = pl.splits * uint64_t(c.kv_heads);
            if (shared && force_splits == 0 && pl.splits > 1 && streams > 8 && streams % 8 != 0) continue;
            before = pl.splits;
            pl.workspace = workspace_of(a, pl);
            if (pl.workspace > workspace_limit && pl.splits > 1) break;
            const double blocks = pl.keys / kBlock, work = double(units) * pl.splits * blocks * share / cus;
            const double rounds = std::ceil(double(units) * pl.splits / (rows == 128 && wide < 2 ? 2 * cus : cus));
            double us;
            if (rows == 16) {
                const double moved = double(n) * c.kv_heads * keys * c.dim * 4 / 5.3e6;
                const double fed = std::max(1.0, 0.6 + 51 / (double(units) * pl.splits));
                const double idle = std::max(0.0, kWaves - blocks);
                const double alone = kRowsStart[wide] + std::ceil(blocks / kWaves) * kRowsChain[wide] - idle * idle * kRowsFewer[wide];
                us = std::max({alone * (1 + 0.8 * (rounds - 1) * share), work * kRowsEach[c.bf16][wide] + 2 * double(units) * pl.splits / cus, moved * fed});
            } else {
                us = std::max({10 + blocks * kTileChain[c.bf16][wide], rounds * (10 + blocks * share * kTileChain[c.bf16][wide]),
                               10 * rounds + work * kTileEach[c.bf16][wide]});
            }
            if (pl.splits > 1) {
                const double joined = double(c.tokens) * a.heads * pl.splits * wide_dim(c.dim) * 8;
                us += 3 + joined / 4.0e6 + 0.02 * pl.splits;
            }
            if (best.rows == 0 || us < least) {
                best = pl;
                least = us;
            }
        }
    }
    // A forced number of ranges whose workspace is too large.
    if (best.rows == 0) return plan_attend(a, lim, workspace_limit, force_rows, 1);
    return best;
}

const char *attend_kernel_name(const AttendPlan &pl) { return pl.rows == 16 ? "attn_rows_kernel" : "attn_tile_kernel"; }

hipError_t launch_attn_paged(const AttendArgs &a, const AttendPlan &pl, void *workspace, hipStream_t stream) {
    const Partial ws = pl.splits > 1 ? parts(a, pl, workspace) : Partial{};
    return a.cache.bf16 ? launch_type<true>(a, pl, ws, stream) : launch_type<false>(a, pl, ws, stream);
}

}  // namespace qmr
