// Launch interface between the host runtime (runtime.cpp) and the HIP
// kernels (affine_rows.hip, affine_mfma.hip, affine_gemv.hip, affine_tile.hip,
// dense_mfma.hip, misc_kernels.hip, wide_mfma.hip, rope_append.hip,
// attn_paged.hip, conv_causal.hip, attn_linear.hip, sample_logits.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "contract.hpp"

namespace qmr {

// One packed-affine product: y[t][r] = sum_c (q*s + b) * x[t][c] for
// t < batch (token-major x [batch][cols], y [batch][rows]).
struct AffineArgs {
    const uint32_t *w;  // [rows][cols*bits/32] packed codes, little-endian fields
    const void *s;      // [rows][cols/group] metadata (F32 or 16-bit patterns)
    const void *b;
    const float *x;
    float *y;
    uint32_t rows, cols, bits, group, batch;
    Meta meta;
    // Fused forms (null when unused).
    //  - residual: y = residual + W x, added in the final store (may alias y).
    //  - MLP (up_w set): w/s/b are the gate matrix and up_w/up_s/up_b the up
    //    matrix of the same shape and format; x[t] is RMS-normalised with the
    //    `norm` weights and `eps`, and y[t] = silu(gate x) * (up x).
    const float *residual = nullptr;
    const uint32_t *up_w = nullptr;
    const void *up_s = nullptr;
    const void *up_b = nullptr;
    const float *norm = nullptr;
    float eps = 0.f;
};

// Tiling of the GEMV/block kernel. A workgroup has 8 half-wave row slots;
// `ks` slots share a row group and split its K rounds, each slot owns `rr`
// rows. rr/ks = 0 lets the planner choose.
struct GemvPlan {
    int rr = 0;
    int ks = 0;
};

// Raises a kernel's dynamic-LDS limit on the current device to `bytes`
// (launches above 64 KB need it): once per kernel, device and larger size,
// under a lock, so that device handles used from different threads do not
// race on it.
hipError_t raise_lds_limit(const void *kernel, size_t bytes);

struct DeviceLimits {
    size_t max_lds_per_block;  // bytes of LDS one workgroup may allocate
    int num_cus;
};

// VALU GEMV / small-block kernel (batch 1..4, group 32/64/128, Q4/Q8).
hipError_t launch_affine_gemv(const AffineArgs &a, GemvPlan plan, const DeviceLimits &lim,
                              hipStream_t stream);
// Reference-arithmetic kernel for any group size (also reference mode).
hipError_t launch_affine_generic(const AffineArgs &a, hipStream_t stream);
// Row dequantisation y[c] = q*s + b (bit-exact RN32).
hipError_t launch_embed_affine(const uint32_t *w, const void *s, const void *b, Meta meta,
                               uint32_t row, uint32_t cols, uint32_t bits, uint32_t group,
                               float *y, hipStream_t stream);
// Dense F16 weights: matvec / block and embedding row.
hipError_t launch_dense_f16(const uint16_t *w, const float *x, float *y, uint32_t rows,
                            uint32_t cols, uint32_t batch, hipStream_t stream);
hipError_t launch_embed_f16(const uint16_t *w, uint32_t row, uint32_t cols, float *y,
                            hipStream_t stream);
// y[i] = x[i] for i < n (x == y allowed only as the identical view).
hipError_t launch_copy_f32(const float *x, float *y, uint32_t n, int num_cus, hipStream_t stream);
// p[i] = 0 for i < n (a fill kernel: safe to capture into a graph).
hipError_t launch_zero_u32(uint32_t *p, uint32_t n, hipStream_t stream);
// One wave that returns after `ticks` of the device's real-time counter.
hipError_t launch_delay(unsigned long long ticks, hipStream_t stream);
// Geometry of read_checksum: workgroups of 256 threads (0 = about 48 KB per
// workgroup), 16-byte loads per thread in flight (1, 2, 4 or 8; 0 = 4),
// non-temporal loads (1), plain (0) or the default (-1: non-temporal).
struct ReadPlan {
    uint32_t workgroups = 0;
    uint32_t unroll = 0;
    int nt = -1;
};
// One streaming read of three views (byte sizes, multiples of 4); out holds
// kChecksumSlots u32 whose XOR is the XOR of every word read.
hipError_t launch_read_checksum(const void *a, uint32_t na, const void *b, uint32_t nb, const void *c, uint32_t nc,
                                uint32_t *out, const ReadPlan &plan, hipStream_t stream);
// A last arriver's wait on the other K splits' {value, epoch} slots (the
// row-band, split-K and dense kernels).
struct TileWait {
    // Device-visible word that a last arriver which gives up sets to
    // 0x80000000 | band (row-band kernel: its band's workgroups were not all
    // resident), 0xC0000000 | band (split-K kernel) or 0xA0000000 | band
    // (dense kernel); null: no report (the outputs are NaN either way).
    uint32_t *status = nullptr;
    // The last arriver clears each slot it took (row-band: plain and residual
    // forms; split-K and dense: every form), so that a workspace that was
    // zero stays zero and the next launch may reuse the same epoch.
    bool reset_slots = false;
    // Testing: the last arriver waits for a tag no split publishes and gives
    // up after a short bound; every workgroup still exits.
    bool force_give_up = false;
};

// Streaming GEMV / small block on the matrix cores (batch 1..4; Q4/Q8;
// group 32/64/128 with 2*batch <= 16*group/128). See affine_mfma.hip.
struct MfmaPlan {
    uint32_t rt = 0;      // waves (16-row tiles) per workgroup; 0 = unsupported
    uint32_t nbands = 0;  // row bands
    uint32_t ns = 0;      // K splits across workgroups
    uint32_t tiles = 0;   // 128-column K tiles
    uint32_t tps = 0;     // K tiles per split
    bool pairs = false;   // 16-bit metadata staged with 32-bit loads
    size_t lds = 0;       // dynamic LDS bytes per workgroup
    uint32_t rounds = 0;  // rounds of resident workgroups the grid takes
};
bool affine_mfma_supported(const AffineArgs &a);
// force_ns > 0 (tuning hook) keeps only that number of K splits.
MfmaPlan plan_affine_mfma(const AffineArgs &a, const DeviceLimits &lim, uint32_t force_ns = 0);
// Workspace bytes the plan needs for cross-workgroup partial sums (0 if none).
size_t affine_mfma_workspace(const MfmaPlan &pl, const AffineArgs &a);
// `slots` holds affine_mfma_workspace bytes (64-bit slots: a partial counts
// only when its epoch matches); `epoch` must differ from the previous
// launch's that used the same slots, unless those slots were cleared;
// `counters` holds pl.nbands zeroed u32 (the kernel returns them to zero).
hipError_t launch_affine_mfma(const AffineArgs &a, const MfmaPlan &pl, unsigned long long *slots,
                              uint32_t *counters, uint32_t epoch, const TileWait &wait, hipStream_t stream);

// Dense F16 matvec / block (batch 1..4) on the matrix cores: row bands of
// 16-row tiles, K in ns splits whose epoch-tagged sums an elected finisher
// adds. See dense_mfma.hip.
struct DensePlan {
    uint32_t rt = 0;      // 16-row tiles per workgroup; 0 = unsupported
    uint32_t kw = 0;      // waves per tile (contiguous K runs of the split)
    uint32_t ring = 0;    // 128-byte entries in flight per wave (4 or 8)
    uint32_t nbands = 0;  // row bands
    uint32_t ns = 0;      // K splits across workgroups
    uint32_t tiles = 0;   // 128-column K tiles
    uint32_t tps = 0;     // K tiles per split
    uint32_t xi = 0;      // x items staged per thread
    size_t lds = 0;       // dynamic LDS bytes per workgroup
    double cost_us = 0;   // the planner's time estimate
};
// Fields the tuning hook pins (0 = the planner's choice).
struct DenseForce {
    uint32_t ring = 0, kw = 0, rt = 0, ns = 0;
};
// 16-byte aligned weights, cols % 32 == 0, 1..4 RHS, views below 2 GiB.
bool dense_mfma_supported(const uint16_t *w, uint32_t rows, uint32_t cols, uint32_t batch);
// Pinned fields that no feasible plan has fall back to the planner's plan.
// The planner scores every feasible plan with a cost model fitted to MI355X
// timings and keeps the cheapest.
DensePlan plan_dense_mfma(uint32_t rows, uint32_t cols, uint32_t batch, const DeviceLimits &lim,
                          const DenseForce &force = DenseForce{});
size_t dense_mfma_workspace(const DensePlan &pl, uint32_t rows, uint32_t batch);
// Estimated time (us) of the vector-ALU dense kernels on the same product,
// for the choice between the two.
double dense_valu_cost(uint32_t rows, uint32_t cols, uint32_t batch);
// `slots` (dense_mfma_workspace bytes) and `counters` (pl.nbands zeroed u32)
// as for launch_affine_mfma; both may be null when pl.ns == 1.
hipError_t launch_dense_mfma(const uint16_t *w, const float *x, float *y, uint32_t rows, uint32_t cols,
                             uint32_t batch, const DensePlan &pl, unsigned long long *slots, uint32_t *counters,
                             uint32_t epoch, const TileWait &wait, hipStream_t stream);

// Streaming GEMV / small block on the matrix cores with every workgroup
// owning whole rows (no cross-workgroup reduction). See affine_rows.hip.
struct RowsPlan {
    uint32_t rt = 0;         // 16-row tiles per workgroup; 0 = unsupported
    uint32_t kw = 0;         // K waves per tile
    uint32_t j = 0;          // entries per wave per staged chunk
    uint32_t nbands = 0;     // workgroups
    uint32_t n_entries = 0;  // 128-byte entries per row
    uint32_t n_chunks = 0;   // ceil(n_entries / (kw * j))
    bool pairs = false;      // 16-bit metadata staged with 32-bit loads
    size_t stage_bytes = 0;  // one LDS staging buffer
    size_t lds = 0;          // dynamic LDS bytes per workgroup
};
bool affine_rows_supported(const AffineArgs &a);
// force_rt/force_kw (both nonzero) pin the workgroup shape and force_j the
// chunk depth; zeros leave the choice to the planner.
// The MLP form's tiling: gate and up tiles of the same rows in one workgroup
// (even rt, the first rt/2 tiles from the gate matrix).
RowsPlan plan_affine_mlp(const AffineArgs &a, const DeviceLimits &lim, uint32_t force_rt = 0,
                         uint32_t force_kw = 0, uint32_t force_j = 0);
RowsPlan plan_affine_rows(const AffineArgs &a, const DeviceLimits &lim, uint32_t force_rt = 0,
                          uint32_t force_kw = 0, uint32_t force_j = 0);
hipError_t launch_affine_rows(const AffineArgs &a, const RowsPlan &pl, hipStream_t stream);

// Streaming GEMV / small block on the matrix cores over row bands of 16-row
// tiles: each band's K range in ns long splits across workgroups and KW
// contiguous per-wave runs inside one; the band's last split adds the
// others' epoch-tagged partial sums. See affine_tile.hip.
struct TilePlan {
    uint32_t kw = 0;          // waves per row tile; 0 = unsupported
    uint32_t tr = 0;          // row tiles per band (workgroup)
    uint32_t ns = 0;          // K splits across workgroups
    uint32_t nbands = 0;      // row bands
    uint32_t n_entries = 0;   // 128-byte entries per row
    uint32_t tiles = 0;       // 128-column K tiles
    uint32_t gp = 0;          // LDS pitch of a row's metadata
    uint32_t meta_bytes = 0;  // LDS bytes of the staged metadata
    uint32_t img_bytes = 0;   // LDS bytes of the staged x images
    uint32_t xi = 0;          // x items staged per thread
    uint32_t ring = 0;        // code entries in flight per wave (2 or 3)
    size_t lds = 0;           // dynamic LDS bytes per workgroup
    bool elect = false;       // every split publishes; an arrival counter elects each band's finisher
    uint32_t phases = 1;      // 2: x images staged in two halves (single split, one wave per tile)
    uint32_t phase_entry = 0; // with phases == 2: the first entry of the second half
};
bool affine_tile_supported(const AffineArgs &a);
// Zeros leave the choice to the planner; force_phases 1 keeps one phase of
// x staging, 2 takes two where the plan allows it.
TilePlan plan_affine_tile(const AffineArgs &a, const DeviceLimits &lim, uint32_t force_kw = 0,
                          uint32_t force_tr = 0, uint32_t force_ns = 0, uint32_t force_ring = 0,
                          uint32_t force_phases = 0);
// Workspace bytes for the partial-sum slots (0 when ns == 1).
size_t affine_tile_workspace(const TilePlan &pl, const AffineArgs &a);
// `partial` holds affine_tile_workspace bytes (64-bit slots: a slot counts
// only when its epoch matches); `epoch` must differ from the previous
// launch's that used the same slots, unless those slots were cleared.
// `counters` holds pl.nbands zeroed u32 when pl.elect (the kernel returns
// them to zero); otherwise it may be null.
hipError_t launch_affine_tile(const AffineArgs &a, const TilePlan &pl, unsigned long long *partial,
                              uint32_t *counters, uint32_t epoch, const TileWait &wait, hipStream_t stream);

// Wide block on MFMA (Q4/Q8, group 32/64/128, F32 or BF16 metadata, batch up to
// 256; F16 metadata in group 32 up to 16 RHS): a prep launch converts x into
// images in `workspace` (wide_mfma_workspace bytes), the contraction, and with
// K splits the sum of their planes. See wide_mfma.hip.
struct WidePlan {
    uint32_t rt = 0;   // 16-row tiles per workgroup; 0 = no plan
    uint32_t ct = 0;   // 16-RHS tiles per workgroup
    uint32_t nw = 0;   // waves (K classes) per workgroup, 4 or 8
    uint32_t ns = 0;   // K splits across workgroups
    uint32_t ups = 0;  // 128-column units per split (a multiple of nw)
};
bool wide_mfma_supported(const AffineArgs &a);
// Non-zero fields of `force` (tuning hook) are kept.
WidePlan plan_wide(const AffineArgs &a, const DeviceLimits &lim, const WidePlan &force = WidePlan{});
size_t wide_mfma_workspace(const AffineArgs &a, const WidePlan &pl);
size_t wide_mfma_image_bytes(const AffineArgs &a);  // of 32 RHS; a plan without K splits needs these alone
hipError_t launch_wide_mfma(const AffineArgs &a, const WidePlan &pl, unsigned char *workspace, hipStream_t stream);
bool wide_instance(const WidePlan &pl);  // rt, ct and nw are a compiled instance's
// Host-side walk of every code, image and metadata load the wide contraction
// kernel issues under a plan (its ns: the splits asked for): the largest end
// (offset + size) of the in-range loads in each view, beside the views'
// extents, and whether a metadata load missed an element that it is for.
struct WideExtent {
    uint64_t code_end, code_extent, image_end, image_extent, meta_end, meta_extent, meta_short;
};
WideExtent wide_address_extent(const AffineArgs &a, WidePlan pl);

// Rotary positions: the first `rotary` dimensions of a head turn in pairs, pair
// i by the position of its axis times freqs[i]. See rope_append.hip.
struct RopeSpec {
    const int32_t *positions;  // [axes][tokens]
    const float *freqs;        // [rotary / 2]
    uint32_t rotary;           // 0: nothing turns
    uint32_t adjacent;         // pairs (2i, 2i + 1) instead of (i, i + rotary/2)
    uint32_t dealt;            // axes dealt to the pairs in turn, not section by section
    uint32_t axes;
    uint32_t sections[4];      // pairs of each axis
};
struct RopeArgs {
    const float *x;
    float *y;
    uint32_t tokens, heads, dim, x_stride, y_stride;  // strides: floats from token to token
    RopeSpec rope;
};
hipError_t launch_rope_axes(const RopeArgs &a, const DeviceLimits &lim, hipStream_t stream);

// A paged key-value cache and the sequences that read and extend it. Sequence
// s has the new tokens starts[s]..starts[s+1]-1, the last `new` of its
// lengths[s] positions; position p is slot p % page of page table[s][p / page].
// A page past the pool holds nothing. Block layouts: rope_append.hip.
struct PagedCache {
    const uint32_t *starts;   // [seqs + 1]
    const uint32_t *lengths;  // [seqs]
    const uint32_t *table;    // [seqs][columns]
    uint16_t *k;              // [pages][kv_heads][page / 32] key blocks
    uint16_t *v;              // [pages][kv_heads][page / 32] value blocks
    uint32_t seqs, tokens, kv_heads, dim, page, pages, columns;
    bool bf16;
};
struct AppendArgs {
    const float *q, *k, *v;       // rows of one token each
    const float *q_norm, *k_norm; // [dim], used when eps > 0
    float *q_out;
    uint32_t heads, q_stride, k_stride, v_stride, out_stride;
    float eps;                    // 0: no normalisation
    RopeSpec rope;
    PagedCache cache;
};
hipError_t launch_kv_append_rope(const AppendArgs &a, const DeviceLimits &lim, hipStream_t stream);

// Attention of the new tokens over the cache. See attn_paged.hip.
struct AttendArgs {
    const float *q;  // [tokens] rows of heads * dim
    float *out;
    uint32_t heads, q_stride, out_stride;
    uint32_t max_keys;  // no key at or past this position is read
    uint32_t causal, window;
    float scale;
    PagedCache cache;
};
// What a launch does, from sizes alone: the lengths are on the device.
struct AttendPlan {
    uint32_t rows = 0;      // query rows of one tile
    uint32_t tiles = 0;     // tiles of all sequences, at most
    uint32_t splits = 1;    // key ranges of a tile
    uint32_t keys = 0;      // keys of one range
    size_t workspace = 0;   // bytes of the ranges' partial results
};
// force_rows (16 or 128) and force_splits (tuning hook) are kept where they can
// be; zeros leave the choice to the planner.
AttendPlan plan_attend(const AttendArgs &a, const DeviceLimits &lim, size_t workspace_limit, uint32_t force_rows = 0,
                       uint32_t force_splits = 0);
hipError_t launch_attn_paged(const AttendArgs &a, const AttendPlan &pl, void *workspace, hipStream_t stream);
const char *attend_kernel_name(const AttendPlan &pl);

// New tokens of some sequences, each of which has a state in a slot of a pool:
// sequence s has the tokens starts[s]..starts[s+1]-1, at most the first `most`
// of them, and the slot slots[s], whose bit 31 says that its state is taken as
// zeros. Slots past the pool and slots that an earlier sequence names keep
// nothing. See sequences.hpp.
struct Sequences {
    const uint32_t *starts;  // [seqs + 1]
    const uint32_t *slots;   // [seqs]
    uint32_t seqs, tokens, most, pool;
};

// Causal convolution, a filter a channel. See conv_causal.hip.
struct ConvArgs {
    const float *x;     // [tokens] rows of channels
    const float *w;     // [channels][width]
    const float *bias;  // [channels] or null
    float *state;       // [pool][width - 1][channels]
    float *y;
    uint32_t channels, width, x_stride, y_stride;
    bool silu, keep;    // keep: states are replaced
    Sequences seq;
};
hipError_t launch_conv_causal(const ConvArgs &a, const DeviceLimits &lim, hipStream_t stream);

// Linear attention with a state and a decay for each value head. See
// attn_linear.hip.
struct LinearArgs {
    const float *q, *k, *v;       // rows of k_heads * dk, k_heads * dk and v_heads * dv
    const float *a, *b;           // rows of v_heads: decays, and the delta rule's factors
    const float *a_log, *dt_bias; // [v_heads], used when gates
    const float *z, *norm;        // rows of v_heads * dv and [dv], used when out_eps > 0
    float *state;                 // [pool][v_heads][dk][dv]
    float *out;                   // rows of v_heads * dv
    uint32_t k_heads, v_heads, dk, dv;
    uint32_t q_stride, k_stride, v_stride, a_stride, b_stride, z_stride, out_stride;
    bool gates, delta, keep;
    float scale, qk_eps, out_eps;  // eps 0: no norm
    Sequences seq;
};
// What a launch does, from sizes alone: where the sequences are is known on the
// device.
struct LinearPlan {
    bool chunks = false;      // chunks of 32 tokens on the matrix cores; else token after token
    uint32_t blocks = 0;      // 32-wide blocks of the key dimension, 2, 4 or 8
    uint32_t columns = 0;     // 16-column tiles of a workgroup
    uint32_t parts = 0;       // chunks of all sequences, at most
    uint32_t per_pass = 0;    // chunks whose operands the workspace holds
    size_t k_bytes = 0, v_bytes = 0;  // operands of a chunk, of one key and one value head
    size_t carry_bytes = 0;   // a state between passes
    size_t workspace = 0;
};
// `form` (tuning hook): 1 token after token, 2 chunks where they are possible, 0
// the planner's choice; `columns` 2 or 4, or 0.
LinearPlan plan_linear(const LinearArgs &a, const DeviceLimits &lim, size_t workspace_limit, uint32_t form = 0,
                       uint32_t columns = 0);
hipError_t launch_attn_linear(const LinearArgs &a, const LinearPlan &pl, void *workspace, hipStream_t stream);
hipError_t launch_linear_chunks(const LinearArgs &a, const LinearPlan &pl, void *workspace, hipStream_t stream);
const char *linear_kernel_name(const LinearPlan &pl);

// A token from each row of logits. See sample_logits.hip.
struct SampleArgs {
    const float *logits;  // [rows] of vocab, one every `stride` floats
    const float *temperature;
    const uint32_t *top_k;
    const float *top_p, *min_p, *uniform;
    uint32_t *tokens;
    float *probs;
    uint32_t rows, vocab, stride;
};
struct SamplePlan {
    bool whole = false;       // a row fits a workgroup's LDS
    uint32_t slice = 0, slices = 0;  // logits of a slice, slices of a row
    uint32_t rows = 0;        // rows at a time
    size_t workspace = 0;
};
SamplePlan plan_sample(const SampleArgs &a, const DeviceLimits &lim, size_t workspace_limit);
hipError_t launch_sample_logits(const SampleArgs &a, const SamplePlan &pl, void *workspace, hipStream_t stream);

// The plan the GEMV launcher would use (for tests and tuning reports).
GemvPlan plan_affine_gemv(const AffineArgs &a, GemvPlan forced, const DeviceLimits &lim);

}  // namespace qmr
