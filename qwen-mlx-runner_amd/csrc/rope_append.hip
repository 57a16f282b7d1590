// Rotary positions with several axes, and appending to a paged key-value cache.
//
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * freqs[i]
//
// for pair i of a head's first `rotary` dimensions; the position is that of
// the pair's axis (time, height, width, ..). An optional RMS norm of the head
// comes first: x / sqrt(mean(x^2) + eps) * w.
//
// The angle is taken in turns: position * (freqs[i] / 2 pi) in 64 bits, its
// fraction of a turn rounded to 32 bits. A product in 32 bits is off by half
// an ulp of the angle, 0.03 rad at a position of a million; the fraction is off
// by 2^-26 turns at every position. One 64-bit product a pair and token costs
// nothing beside the rows it serves.
//
// Cache layout. A page holds, for each key-value head, its keys as blocks of
// 32 keys, and so its values; both in the order that the matrix instructions
// of the attention kernels take their operands, so that a wave's loads of a
// block are whole lines and need no transposition:
//   key block    [dim / 8][key order 32][8 dims]; slot 8a + 4b + c of a block
//                is at key order 16b + 4a + c (a < 4, b < 2, c < 4)
//   value block  [slot / 8][dim][8 slots]
// A key row goes out as 8- or 16-byte pieces. A value chunk (8 slots of one
// dim) is 16 bytes: the wave that owns the chunk's first new token gathers up
// to eight tokens and writes each chunk with one store; chunks that the new
// tokens fill in part take 2-byte stores and keep their other slots.
#include <hip/hip_runtime.h>

#include "attn_common.hpp"
#include "kernels.hpp"

namespace qmr {
namespace {

constexpr int kThreads = 256;

// Four FP32 of a row, which need not lie on 16 bytes.
struct Quad {
    float x[4];
};

// What pair i turns by, for token t.
__device__ __forceinline__ void turn_of(const RopeSpec &r, uint32_t tokens, uint32_t t, uint32_t i, float &c, float &s) {
    uint32_t axis = 0;
    if (r.dealt) {
        const uint32_t at = i % r.axes;
        if (at != 0 && i < r.axes * r.sections[at]) axis = at;
    } else {
        uint32_t end = r.sections[0];
        while (axis + 1 < r.axes && i >= end) end += r.sections[++axis];
    }
    const double per = double(r.freqs[i]) * 0.15915494309189533577;  // 1 / (2 pi)
    const double turns = double(r.positions[size_t(axis) * tokens + t]) * per;
    sincospif(2.f * float(turns - rint(turns)), &s, &c);
}

// One lane's part of a head: IT units of V pairs. A unit's 2V elements are
// V at `first` and V at `second` of the row (halves), or 2V in sequence.
template <int V, int IT>
struct Part {
    float a[IT][V], b[IT][V];
};

// What those pairs turn by.
template <int V, int IT>
struct Turns {
    float c[IT][V], s[IT][V];
};

template <int V>
__device__ __forceinline__ void load_unit(const float *x, uint32_t u, const RopeSpec &r, float (&a)[V], float (&b)[V]) {
    const uint32_t half = r.rotary / 2, turning = half / V;
    const bool halves = u < turning && !r.adjacent;
    const float *pa = x + (u < turning ? (halves ? V * u : 2 * V * u) : r.rotary + 2 * V * (u - turning));
    const float *pb = halves ? pa + half : pa + V;
    float e[2 * V];
    if constexpr (V == 4) {
        *reinterpret_cast<Quad *>(e) = *reinterpret_cast<const Quad *>(pa);
        *reinterpret_cast<Quad *>(e + V) = *reinterpret_cast<const Quad *>(pb);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = pa[k], e[V + k] = pb[k];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        a[k] = halves ? e[k] : e[2 * k];
        b[k] = halves ? e[V + k] : e[2 * k + 1];
    }
}

// Where a unit's 2V results go: f(offset in the row, V values) twice.
template <int V, typename F>
__device__ __forceinline__ void store_unit(uint32_t u, const RopeSpec &r, const float (&a)[V], const float (&b)[V], F &&f) {
    const uint32_t half = r.rotary / 2, turning = half / V;
    const bool halves = u < turning && !r.adjacent;
    const uint32_t at = u < turning ? (halves ? V * u : 2 * V * u) : r.rotary + 2 * V * (u - turning);
    float e[2 * V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if (halves) {
            e[k] = a[k];
            e[V + k] = b[k];
        } else {
            e[2 * k] = a[k];
            e[2 * k + 1] = b[k];
        }
    }
    f(at, e);
    f(halves ? at + half : at + V, e + V);
}

// One head row for a group of `lanes` lanes.
template <int V, int IT>
__device__ __forceinline__ void load_row(const float *x, const RopeSpec &r, uint32_t lane, uint32_t lanes, uint32_t units,
                                         Part<V, IT> &p) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const uint32_t u = lane + k * lanes;
#pragma unroll
        for (int j = 0; j < V; ++j) p.a[k][j] = p.b[k][j] = 0.f;
        if (u < units) load_unit<V>(x, u, r, p.a[k], p.b[k]);
    }
}

// Its RMS norm, with the weights of the lane's own elements.
template <int V, int IT>
__device__ __forceinline__ void norm_row(const Part<V, IT> &weights, float eps, uint32_t dim, uint32_t lanes, Part<V, IT> &p) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < IT; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum += p.a[k][j] * p.a[k][j] + p.b[k][j] * p.b[k][j];
    }
    for (uint32_t d = 1; d < lanes; d *= 2) sum += __shfl_xor(sum, d);
    const float f = 1.f / sqrtf(sum / float(dim) + eps);
#pragma unroll
    for (int k = 0; k < IT; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            p.a[k][j] = p.a[k][j] * f * weights.a[k][j];
            p.b[k][j] = p.b[k][j] * f * weights.b[k][j];
        }
    }
}

template <int V, int IT>
__device__ __forceinline__ void turn_row(const RopeSpec &r, uint32_t lane, uint32_t lanes, const Turns<V, IT> &turns,
                                         Part<V, IT> &p) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        if ((lane + k * lanes) * V >= r.rotary / 2) continue;  // passes as it is, infinities too
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float a = p.a[k][j], b = p.b[k][j];
            p.a[k][j] = a * turns.c[k][j] - b * turns.s[k][j];
            p.b[k][j] = b * turns.c[k][j] + a * turns.s[k][j];
        }
    }
}

template <int V, int IT>
__device__ __forceinline__ void turns_of(const RopeSpec &r, uint32_t tokens, uint32_t t, uint32_t lane, uint32_t lanes,
                                         Turns<V, IT> &turns) {
#pragma unroll
    for (int k = 0; k < IT; ++k) {
        const uint32_t u = lane + k * lanes;
#pragma unroll
        for (int j = 0; j < V; ++j) turns.c[k][j] = 1.f, turns.s[k][j] = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (u * V < r.rotary / 2) turn_of(r, tokens, t, u * V + j, turns.c[k][j], turns.s[k][j]);
    }
}

template <int V>
__device__ __forceinline__ void store_f32(float *y, uint32_t at, const float *e) {
    if constexpr (V == 4) {
        *reinterpret_cast<Quad *>(y + at) = *reinterpret_cast<const Quad *>(e);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) y[at + k] = e[k];
    }
}

// How rows are spread: `lanes` lanes for a head, 64 / lanes heads of one token
// a wave at a time, `heads_each` heads a group before it ends. The angles of a
// token are worked out once a group.
struct Spread {
    uint32_t lanes, units, heads_each, slices;  // slices: waves of one token
    uint32_t span = 1;                          // tokens of a wave of values
};

// Memory bounds it: 4352 tokens of 16 heads of 72 (40 MB) 8.7 us, 4.6 TB/s, as
// near as a large copy comes (4.8); a single token is a launch, 3.5 us.
template <int V, int IT>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(RopeArgs a, Spread sp) {
    const uint32_t wave = blockIdx.x * (kThreads / 64) + threadIdx.x / 64, l = threadIdx.x % 64;
    const uint32_t t = wave / sp.slices;
    if (t >= a.tokens) return;
    const uint32_t group = l / sp.lanes, lane = l % sp.lanes, groups = 64 / sp.lanes;
    Turns<V, IT> turns;
    turns_of<V, IT>(a.rope, a.tokens, t, lane, sp.lanes, turns);
    const uint32_t h0 = (wave % sp.slices) * sp.heads_each * groups + group;
    for (uint32_t k = 0; k < sp.heads_each; ++k) {
        const uint32_t h = h0 + k * groups;
        if (h >= a.heads) break;
        Part<V, IT> p;
        load_row<V, IT>(a.x + size_t(t) * a.x_stride + size_t(h) * a.dim, a.rope, lane, sp.lanes, sp.units, p);
        turn_row<V, IT>(a.rope, lane, sp.lanes, turns, p);
        float *y = a.y + size_t(t) * a.y_stride + size_t(h) * a.dim;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const uint32_t u = lane + i * sp.lanes;
            if (u < sp.units)
                store_unit<V>(u, a.rope, p.a[i], p.b[i], [&](uint32_t at, const float *e) { store_f32<V>(y, at, e); });
        }
    }
}

// The sequence of token t and its position there, the same for a whole wave;
// position -1 where the token has none.
__device__ __forceinline__ void place_of(const PagedCache &c, uint32_t t, uint32_t &seq, int64_t &pos, uint32_t &end) {
    const uint32_t l = threadIdx.x % 64;
    seq = 0;
    for (uint32_t base = 0; base < c.seqs; base += 64) {
        const bool before = base + l < c.seqs && c.starts[base + l + 1] <= t;
        const uint32_t n = __popcll(__ballot(before));
        seq += n;
        if (n < 64) break;
    }
    pos = -1;
    end = t + 1;
    if (seq >= c.seqs || c.starts[seq] > t) return;
    end = max(min(c.starts[seq + 1], c.tokens), t + 1);  // past t whatever the starts hold
    pos = int64_t(c.lengths[seq]) - int64_t(c.starts[seq + 1] - t);
}

// The page slot of a position: false where nothing is kept.
__device__ __forceinline__ bool slot_of(const PagedCache &c, uint32_t seq, int64_t pos, uint32_t &page, uint32_t &slot) {
    if (pos < 0 || uint64_t(pos) >= uint64_t(c.columns) * c.page) return false;
    page = c.table[size_t(seq) * c.columns + uint32_t(uint64_t(pos) / c.page)];
    slot = uint32_t(uint64_t(pos) % c.page);
    return page < c.pages;
}

// Slots first..first+n-1 of the value chunks at `to` from tokens t..t+n-1.
template <bool BF16>
__device__ __forceinline__ void append_values(const AppendArgs &a, uint16_t *to, uint32_t first, uint32_t t, uint32_t h, uint32_t n) {
    const uint32_t dim = a.cache.dim;
    const float *x = a.v + size_t(t) * a.v_stride + size_t(h) * dim;
    for (uint32_t d0 = threadIdx.x % 64 * 4; d0 < dim; d0 += 256) {
        float e[8][4];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (i >= n) continue;
            *reinterpret_cast<Quad *>(e[i]) = *reinterpret_cast<const Quad *>(x + size_t(i) * a.v_stride + d0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint16_t *chunk = to + size_t(d0 + j) * 8;
            if (n == 8) {
                uint4 w;
                w.x = attn::half_bits<BF16>(e[0][j]) | uint32_t(attn::half_bits<BF16>(e[1][j])) << 16;
                w.y = attn::half_bits<BF16>(e[2][j]) | uint32_t(attn::half_bits<BF16>(e[3][j])) << 16;
                w.z = attn::half_bits<BF16>(e[4][j]) | uint32_t(attn::half_bits<BF16>(e[5][j])) << 16;
                w.w = attn::half_bits<BF16>(e[6][j]) | uint32_t(attn::half_bits<BF16>(e[7][j])) << 16;
                *reinterpret_cast<uint4 *>(chunk) = w;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    if (i < n) chunk[first + i] = attn::half_bits<BF16>(e[i][j]);
            }
        }
    }
}

// Waves [0, tokens * slices): query and key heads, turned. The others: values,
// one wave `span` tokens and a head.
//
// 2011 tokens of 24/4 heads of 256 with norms (124 MB) 36 us, 3.4 TB/s, and 26
// from the last-level cache; a large copy reaches 4.8 and the rotation alone 4.3
// at this size: angles, norms and layouts take vector instructions beside the
// stream (7.1 million of a wave, 12 us of four SIMDs a CU). With the norms'
// weights loaded for each row 41 us, a wave of values a token 38, a row loaded
// before the last one is turned 41. One token 5.4 us, 48 of 32/8 heads of 128 4.2:
// a launch and its chain of loads (the token's sequence, its length, its page).
template <int V, int IT, bool BF16>
__global__ __launch_bounds__(kThreads) void kv_append_rope_kernel(AppendArgs a, Spread sp) {
    const uint32_t wave = blockIdx.x * (kThreads / 64) + threadIdx.x / 64, l = threadIdx.x % 64;
    const PagedCache &c = a.cache;
    const uint32_t tokens = c.tokens, dim = c.dim;
    uint32_t seq, end, page = 0, slot = 0;
    int64_t pos;
    if (wave < tokens * sp.slices) {
        const uint32_t t = wave / sp.slices;
        const uint32_t group = l / sp.lanes, lane = l % sp.lanes, groups = 64 / sp.lanes;
        const uint32_t h0 = (wave % sp.slices) * sp.heads_each * groups + group, heads = a.heads + c.kv_heads;
        Part<V, IT> q_norm, k_norm;
        if (a.eps > 0.f) {
            if (a.heads > 0) load_row<V, IT>(a.q_norm, a.rope, lane, sp.lanes, sp.units, q_norm);  // else no view
            load_row<V, IT>(a.k_norm, a.rope, lane, sp.lanes, sp.units, k_norm);
        }
        place_of(c, t, seq, pos, end);
        const bool kept = slot_of(c, seq, pos, page, slot);
        Turns<V, IT> turns;
        turns_of<V, IT>(a.rope, tokens, t, lane, sp.lanes, turns);
        for (uint32_t k = 0; k < sp.heads_each; ++k) {
            const uint32_t h = h0 + k * groups;
            if (h >= heads) break;
            const bool key = h >= a.heads;
            const uint32_t kh = h - a.heads;
            Part<V, IT> p;
            load_row<V, IT>(key ? a.k + size_t(t) * a.k_stride + size_t(kh) * dim : a.q + size_t(t) * a.q_stride + size_t(h) * dim,
                            a.rope, lane, sp.lanes, sp.units, p);
            if (a.eps > 0.f) norm_row<V, IT>(key ? k_norm : q_norm, a.eps, dim, sp.lanes, p);
            turn_row<V, IT>(a.rope, lane, sp.lanes, turns, p);
            float *y = a.q_out + size_t(t) * a.out_stride + size_t(h) * dim;
            uint16_t *row = c.k + attn::key_row(c, page, kh, slot);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const uint32_t u = lane + i * sp.lanes;
                if (u >= sp.units) continue;
                store_unit<V>(u, a.rope, p.a[i], p.b[i], [&](uint32_t at, const float *e) {
                    if (!key) {
                        store_f32<V>(y, at, e);
                    } else if (kept) {
                        uint16_t *to = row + (at / 8) * attn::kKeyChunk + at % 8;
                        if constexpr (V == 4) {
                            uint2 w;
                            w.x = attn::half_bits<BF16>(e[0]) | uint32_t(attn::half_bits<BF16>(e[1])) << 16;
                            w.y = attn::half_bits<BF16>(e[2]) | uint32_t(attn::half_bits<BF16>(e[3])) << 16;
                            *reinterpret_cast<uint2 *>(to) = w;
                        } else {
#pragma unroll
                            for (int j = 0; j < V; ++j) to[j] = attn::half_bits<BF16>(e[j]);
                        }
                    }
                });
            }
        }
        return;
    }
    const uint32_t at = wave - tokens * sp.slices, h = at % c.kv_heads;
    uint32_t t = at / c.kv_heads * sp.span;
    const uint32_t last = min(t + sp.span, tokens);
    while (t < last) {
        place_of(c, t, seq, pos, end);
        const uint32_t in_chunk = uint32_t(pos) % 8;
        // A chunk's first slot leads it, or the first new token.
        if (pos >= 0 && (in_chunk == 0 || t == c.starts[seq]) && slot_of(c, seq, pos, page, slot))
            append_values<BF16>(a, c.v + attn::value_chunk(c, page, h, slot), slot % 8, t, h, min(8 - in_chunk, end - t));
        t = pos < 0 ? t + 1 : min(t + 8 - in_chunk, end);
    }
}

// Lanes, units and slices for rows of `heads` heads. A token's heads go to as
// few waves as still give every CU eight, since each wave works out the
// token's angles again (2011 tokens as above with four, eight and 16: 34.6, 35.9
// and 36.3 us: four make one wave a token, eight two of 13 and one step, which
// is what they lose by; the rotation of 4352 of 16 heads of 72 8.7 with each, 10.2
// with 32).
Spread spread_of(uint32_t dim, uint32_t v, uint32_t tokens, uint32_t heads, const DeviceLimits &lim) {
    Spread s;
    s.units = dim / (2 * v);
    s.lanes = 1;
    while (s.lanes < s.units && s.lanes < 64) s.lanes *= 2;
    const uint32_t groups = 64 / s.lanes, steps = (heads + groups - 1) / groups;
    const uint64_t want = uint64_t(lim.num_cus) * 8;
    s.heads_each = steps;
    while (s.heads_each > 1 && uint64_t(tokens) * ((steps + s.heads_each - 1) / s.heads_each) < want) --s.heads_each;
    s.slices = (steps + s.heads_each - 1) / s.heads_each;
    return s;
}

}  // namespace

hipError_t launch_rope_axes(const RopeArgs &a, const DeviceLimits &lim, hipStream_t stream) {
    const bool wide = a.dim % 8 == 0 && a.rope.rotary % 8 == 0;
    const Spread sp = spread_of(a.dim, wide ? 4 : 1, a.tokens, a.heads, lim);
    const uint64_t waves = uint64_t(a.tokens) * sp.slices;
    const uint32_t blocks = uint32_t((waves + kThreads / 64 - 1) / (kThreads / 64));
    if (wide) {
        rope_axes_kernel<4, 1><<<blocks, kThreads, 0, stream>>>(a, sp);
    } else {
        rope_axes_kernel<1, 2><<<blocks, kThreads, 0, stream>>>(a, sp);
    }
    return hipGetLastError();
}

hipError_t launch_kv_append_rope(const AppendArgs &a, const DeviceLimits &lim, hipStream_t stream) {
    const PagedCache &c = a.cache;
    const bool wide = a.rope.rotary % 8 == 0;
    Spread sp = spread_of(c.dim, wide ? 4 : 1, c.tokens, a.heads + c.kv_heads, lim);
    // One token of eight leads a chunk where sequences have many.
    sp.span = c.tokens / 8 >= c.seqs ? 8 : 1;
    const uint64_t waves = uint64_t(c.tokens) * sp.slices + uint64_t((c.tokens + sp.span - 1) / sp.span) * c.kv_heads;
    const uint32_t blocks = uint32_t((waves + kThreads / 64 - 1) / (kThreads / 64));
    if (wide && c.bf16) {
        kv_append_rope_kernel<4, 1, true><<<blocks, kThreads, 0, stream>>>(a, sp);
    } else if (wide) {
        kv_append_rope_kernel<4, 1, false><<<blocks, kThreads, 0, stream>>>(a, sp);
    } else if (c.bf16) {
        kv_append_rope_kernel<1, 2, true><<<blocks, kThreads, 0, stream>>>(a, sp);
    } else {
        kv_append_rope_kernel<1, 2, false><<<blocks, kThreads, 0, stream>>>(a, sp);
    }
    return hipGetLastError();
}

}  // namespace qmr
