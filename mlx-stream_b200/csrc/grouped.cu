// Products grouped by expert over 16-bit weights: y[p] = W_g x[p] for offsets[g] <= p < offsets[g + 1], or SwiGLU of a gate and an up product of the
// same rows.  Weights row-major, outputs or inputs first, nothing laid out anew; rows may be gathered and scattered on the way.  Two kernels, by
// the call's rows alone (the groups' sizes are on the device):
//   * up to 16 rows: grouped_few_kernel streams the weights through mma.sync (bound: HBM);
//   * more: grouped_tile_kernel, tcgen05 tiles over CTA pairs.  Many rows per group are bound by the tensor pipe under the power cap, few by HBM:
//     512 rows over 256 groups (K 2304, N 5120, f32) 0.76 ms = 6.6 TB/s, 1.01 of the measured copy rate, with the same tiles.
// 17 rows over 64 groups (K 5120, 2 x 2304 outputs): 121 us with the tiles (5.9 TB/s); 16 rows: 105 us streamed (6.3 TB/s) against 126 with the tiles.
#include "common.cuh"
#include "kernels.h"
#include "tensor_map.cuh"
#include "umma_pair.cuh"

namespace mlxs {

// EXACT: the exponential's own function (f32 outputs); without it the product with log2(e) rounds once more, 2^-24 of the exponent,
// far inside a 16-bit output's half step
template <bool EXACT>
__device__ __forceinline__ float gp_swiglu(float g, float u, float limit) {
    if (limit > 0.f) {   // comparisons keep a NaN
        g = g > limit ? limit : g;
        u = u > limit ? limit : (u < -limit ? -limit : u);
    }
    return __fdividef(g, 1.f + (EXACT ? expf(-g) : __expf(-g))) * u;
}

// The rows [r0, r1) of group g, cut to the call's rows; false where the offsets had to be cut
__device__ __forceinline__ bool gp_range(const GroupedArgs& a, uint32_t g, uint32_t& r0, uint32_t& r1) {
    if (!a.offsets) { r0 = 0; r1 = a.rows; return true; }   // one group
    const uint32_t o0 = a.offsets[g], o1 = a.offsets[g + 1];
    r0 = min(o0, a.rows);
    r1 = max(min(o1, a.rows), r0);
    return o0 <= o1 && o1 <= a.rows;
}

// ------------------------------------------------------------------------------------------------------------
// few rows
// ------------------------------------------------------------------------------------------------------------
// Calls of up to 16 rows (a token's or two tokens' experts): the weights' bytes are everything, and tiles of 512 outputs would leave most SMs
// without work.  A CTA takes 32 rows of a group's matrix (inputs first: 64) and all the group's rows; its eight warps split the inputs and stream
// the weights from memory straight into mma fragments, 16 bytes per lane, four blocks ahead.  The warps' sums meet in shared memory, in order.
// The matrix instruction truncates where it adds to its accumulator, so after GN_CHAIN products a warp's accumulators move on to f32 sums in shared memory
// (f32 outputs against 64 bits with one chain to a warp: K 5120 6.0e-7, gate and up 1.2e-6, 65,536 same-signed inputs 2.5e-5).
// Bound by HBM: one token's eight experts (K 5120, gate and up of 2304) 63 us = 6.0 TB/s, 0.92 of the measured copy rate (82 with the tiles);
// inputs first 66 us (64-byte runs of a row per warp instead of 64 bytes of eight rows).  One row alone: 14.7 us, latency.
constexpr uint32_t GN_ROWS = 16, GN_WARPS = 8, GN_AHEAD = 4, GN_CHAIN = 16;

__device__ __forceinline__ uint4 gn_stream16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 gn_ld16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 gn_ld8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
template <bool BF16>
__device__ __forceinline__ void gn_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const uint32_t a[4] = {a0, a1, a2, a3};
    if (BF16) mma_bf16(d, a, b0, b1);
    else mma_f16(d, a, b0, b1);
}

// the accumulators to the warp's sums, row(m, h) and column n of them; they begin anew
template <int MT, int NT, class Row>
__device__ __forceinline__ void gn_move(float (&acc)[MT][NT][4], float* out, bool first, Row row) {
    const uint32_t t = threadIdx.x & 3u;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float2* const o = reinterpret_cast<float2*>(out + row(m, h) * GN_ROWS + n * 8 + 2 * t);
                float2 v = make_float2(acc[m][n][2 * h], acc[m][n][2 * h + 1]);
                if (!first) { const float2 s = *o; v.x += s.x; v.y += s.y; }
                *o = v;
                acc[m][n][2 * h] = acc[m][n][2 * h + 1] = 0.f;
            }
}

// Outputs first.  W row r of the CTA's 32 (r < 16: m-tile 0) is w + row_of(r) ld_w.  A lane's eight consecutive inputs stand for the k positions 2t,
// 2t+1, 2t+8, 2t+9 of two products, the same for both operands.
template <bool BF16, int NT, class RowOf>
__device__ __forceinline__ void gn_out_in(const GroupedArgs& a, const uint16_t* w, RowOf row_of, const uint32_t* xrow, uint32_t n_rows, float* out) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint16_t *wp[4], *xp[NT];
#pragma unroll
    for (int r = 0; r < 4; ++r) wp[r] = w + (size_t)row_of(r * 8 + g) * a.ld_w + t * 8;
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = static_cast<const uint16_t*>(a.x) + (size_t)xrow[n * 8 + g < n_rows ? n * 8 + g : 0] * a.ld_x + t * 8;
    float acc[2][NT][4] = {};
    struct Block { uint4 w[4], x[NT]; } b[GN_AHEAD];
    const uint32_t n_kb = (a.K + 31) / 32;
    auto ask = [&](Block& to, uint32_t kb) {
        const bool in = kb < n_kb && kb * 32 + t * 8 < a.K;
#pragma unroll
        for (int r = 0; r < 4; ++r) to.w[r] = in ? gn_stream16(wp[r] + kb * 32) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n) to.x[n] = in ? gn_ld16(xp[n] + kb * 32) : zero;
    };
#pragma unroll
    for (uint32_t i = 0; i < GN_AHEAD; ++i) ask(b[i], warp + i * GN_WARPS);
    // [row of W][row of x], eight columns to a fragment
    const auto row = [&](int m, int h) { return m * 16 + h * 8 + g; };
    uint32_t chain = 0;
    bool first = true;
#pragma unroll 1
    for (uint32_t kb = warp; kb < n_kb; kb += GN_AHEAD * GN_WARPS) {
        if (chain == GN_CHAIN) { gn_move<2, NT>(acc, out, first, row); first = false; chain = 0; }
        chain += 2 * GN_AHEAD;
#pragma unroll
        for (uint32_t i = 0; i < GN_AHEAD; ++i) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 lo = b[i].w[2 * m], hi = b[i].w[2 * m + 1], x = b[i].x[n];
                    gn_mma<BF16>(acc[m][n], lo.x, hi.x, lo.y, hi.y, x.x, x.y);
                    gn_mma<BF16>(acc[m][n], lo.z, hi.z, lo.w, hi.w, x.z, x.w);
                }
            ask(b[i], kb + (GN_AHEAD + i) * GN_WARPS);
        }
    }
    gn_move<2, NT>(acc, out, first, row);
}

// Inputs first: a lane takes eight outputs (lane / 4) of the inputs 4t .. 4t + 3 of a block of 16, which stand for the k positions 2t, 2t+1, 2t+8,
// 2t+9; two inputs' words are permuted into pairs along k.  Row i of m-tile j is output (i % 8) 8 + 2 j + i / 8.
template <bool BF16, int NT>
__device__ __forceinline__ void gn_in_out(const GroupedArgs& a, const uint16_t* w8, const uint32_t* xrow, uint32_t n_rows, float* out) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint16_t* xp[NT];
    w8 += (size_t)(t * 4) * a.ld_w;
#pragma unroll
    for (int n = 0; n < NT; ++n) xp[n] = static_cast<const uint16_t*>(a.x) + (size_t)xrow[n * 8 + g < n_rows ? n * 8 + g : 0] * a.ld_x + t * 4;
    float acc[4][NT][4] = {};
    struct Block { uint4 w[4]; uint2 x[NT]; } b[GN_AHEAD];
    const uint32_t n_kb = (a.K + 15) / 16;
    auto ask = [&](Block& to, uint32_t kb) {
        const bool in = kb < n_kb && kb * 16 + t * 4 < a.K;
#pragma unroll
        for (int r = 0; r < 4; ++r) to.w[r] = in ? gn_stream16(w8 + (size_t)(kb * 16 + r) * a.ld_w) : zero;
#pragma unroll
        for (int n = 0; n < NT; ++n) to.x[n] = in ? gn_ld8(xp[n] + kb * 16) : make_uint2(0, 0);
    };
#pragma unroll
    for (uint32_t i = 0; i < GN_AHEAD; ++i) ask(b[i], warp + i * GN_WARPS);
    const auto row = [&](int m, int h) { return g * 8 + 2 * m + h; };
    uint32_t chain = 0;
    bool first = true;
#pragma unroll 1
    for (uint32_t kb = warp; kb < n_kb; kb += GN_AHEAD * GN_WARPS) {
        if (chain == GN_CHAIN) { gn_move<4, NT>(acc, out, first, row); first = false; chain = 0; }
        chain += GN_AHEAD;
#pragma unroll
        for (uint32_t i = 0; i < GN_AHEAD; ++i) {
            const uint32_t r0[4] = {b[i].w[0].x, b[i].w[0].y, b[i].w[0].z, b[i].w[0].w}, r1[4] = {b[i].w[1].x, b[i].w[1].y, b[i].w[1].z, b[i].w[1].w};
            const uint32_t r2[4] = {b[i].w[2].x, b[i].w[2].y, b[i].w[2].z, b[i].w[2].w}, r3[4] = {b[i].w[3].x, b[i].w[3].y, b[i].w[3].z, b[i].w[3].w};
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    gn_mma<BF16>(acc[m][n], __byte_perm(r0[m], r1[m], 0x5410), __byte_perm(r0[m], r1[m], 0x7632), __byte_perm(r2[m], r3[m], 0x5410),
                                 __byte_perm(r2[m], r3[m], 0x7632), b[i].x[n].x, b[i].x[n].y);
            ask(b[i], kb + (GN_AHEAD + i) * GN_WARPS);
        }
    }
    gn_move<4, NT>(acc, out, first, row);
}

__device__ __forceinline__ void gn_put(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void gn_put(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void gn_put(float v, float* o) { *o = v; }

template <bool BF16, bool IN_OUT, bool SWIGLU, class O>
__global__ void __launch_bounds__(GN_WARPS * 32, 2) grouped_few_kernel(const GroupedArgs a) {
    constexpr uint32_t W_ROWS = IN_OUT ? 64 : 32, OUTS = SWIGLU ? W_ROWS / 2 : W_ROWS;
    __shared__ __align__(16) float sums[GN_WARPS][W_ROWS * GN_ROWS];
    __shared__ uint32_t s_xrow[GN_ROWS], s_yrow[GN_ROWS], s_group;
    const uint32_t tid = threadIdx.x, p0 = blockIdx.y, f0 = blockIdx.x * OUTS;
    // the group whose rows begin at p0, if one does
    if (tid == 0) s_group = 0xFFFFFFFFu;
    grid_dep_wait();
    grid_dep_launch();
    __syncthreads();
    for (uint32_t g = tid; g < a.G; g += GN_WARPS * 32) {
        uint32_t r0, r1;
        const bool ok = gp_range(a, g, r0, r1);
        if (!ok && blockIdx.x == 0 && p0 == 0) atomicMax(a.status, ST_BAD_OFFSETS);
        if (r0 == p0 && r1 > p0) atomicMin(&s_group, g);
    }
    __syncthreads();
    const uint32_t g = s_group;
    if (g == 0xFFFFFFFFu) return;
    uint32_t r0, r1;
    gp_range(a, g, r0, r1);
    const uint32_t n_rows = r1 - r0;                                  // at most the call's rows: 16
    if (tid < n_rows) {
        const uint32_t p = p0 + tid, o = a.order ? a.order[p] : p;
        uint32_t xr = a.gather ? o / a.x_div : p, yr = a.scatter ? o : p;
        if (xr >= a.x_rows || yr >= a.y_rows) { xr = 0; yr = 0xFFFFFFFFu; atomicMax(a.status, ST_BAD_ROW); }
        s_xrow[tid] = xr; s_yrow[tid] = yr;
    }
    __syncthreads();
    const uint16_t* w = static_cast<const uint16_t*>(a.w) + (size_t)g * a.w_stride;
    float* const mine = sums[tid >> 5];
    if (IN_OUT) {
        // this lane's eight outputs; behind the last: the last eight
        const uint32_t lane8 = (tid & 31u) >> 2, f = f0 + (SWIGLU ? lane8 % 4 : lane8) * 8;
        const uint16_t* w8 = w + (SWIGLU && lane8 >= 4 ? a.N : 0) + (f < a.N ? f : a.N - 8);
        if (n_rows <= 8) gn_in_out<BF16, 1>(a, w8, s_xrow, n_rows, mine);
        else gn_in_out<BF16, 2>(a, w8, s_xrow, n_rows, mine);
    } else {
        const auto row_of = [&](uint32_t r) {
            const uint32_t f = f0 + (SWIGLU ? r % 16 : r), c = f < a.N ? f : a.N - 1;
            return SWIGLU && r >= 16 ? a.N + c : c;
        };
        if (n_rows <= 8) gn_out_in<BF16, 1>(a, w, row_of, s_xrow, n_rows, mine);
        else gn_out_in<BF16, 2>(a, w, row_of, s_xrow, n_rows, mine);
    }
    __syncthreads();
    for (uint32_t i = tid; i < OUTS * n_rows; i += GN_WARPS * 32) {
        const uint32_t f = i % OUTS, r = i / OUTS;
        float v = sums[0][f * GN_ROWS + r], u = 0.f;
        for (uint32_t k = 1; k < GN_WARPS; ++k) v += sums[k][f * GN_ROWS + r];
        if (SWIGLU) {
            u = sums[0][(OUTS + f) * GN_ROWS + r];
            for (uint32_t k = 1; k < GN_WARPS; ++k) u += sums[k][(OUTS + f) * GN_ROWS + r];
            v = gp_swiglu<sizeof(O) == 4>(v, u, a.limit);
        }
        const uint32_t yr = s_yrow[r];
        if (yr != 0xFFFFFFFFu && f0 + f < a.N) gn_put(v, static_cast<O*>(a.y) + (size_t)yr * a.ld_y + f0 + f);
    }
}

template <bool BF16, bool IN_OUT, bool SWIGLU, class O>
static cudaError_t few_launch(const GroupedArgs& a, cudaStream_t st) {
    constexpr uint32_t OUTS = (IN_OUT ? 64 : 32) / (SWIGLU ? 2 : 1);
    return launch_dependent(true, grouped_few_kernel<BF16, IN_OUT, SWIGLU, O>, dim3((a.N + OUTS - 1) / OUTS, a.rows), dim3(GN_WARPS * 32), 0, st, a);
}

// ------------------------------------------------------------------------------------------------------------
// tensor-core tiles
// ------------------------------------------------------------------------------------------------------------
// An item is 512 outputs (activation: 256 and their gates) of up to 256 rows of a group, D[outputs][rows] = W x^T: the weights are the MMA's A operand, so
// that a ragged last tile pads rows only to 32.  Two CTAs share it (cta_group::2, M = 256): each holds half of the outputs, as two accumulators of 128, and half
// of the rows' operand.  Per stage of 64 inputs a CTA takes in 48 KB for eight MMAs of 128 cycles: 48 bytes a cycle, where 256 outputs would take 64 and
// came out 6 % slower at K 8192.  Copies are few and large (one box of weights, one of rows): a stage in six boxes took 398 ns without any MMA, in two 284.
//   * gate and up are one accumulator each, so a thread has both of an output; the weights' box is gate rows behind up rows (a four-dimensional map);
//   * weights with the inputs first are M-major operands: boxes of 64 outputs x 64 inputs, the same stage;
//   * gathered rows come by cp.async into a ring of their own, two warps to a stage.  Tensor-map gathers (four rows to a copy) take 97 cycles each: 32768 rows 3.0 ms against
//     1.29 to 1.32 now (gate and up of 2048, groups as routed; in sorted order and groups of 512 each 0.86 to 0.94); one arrival per copying thread on the slot's barrier took longer than the stage (2400 rows 720 us against 390);
//   * the epilogue packs two rows to a word and turns 16 x 32 outputs through shared memory: 8-byte stores, 64 bytes of a row per warp.
// Sorted rows, 64 groups of 512, K 4096, gate and up of 2048: 0.86 - 0.94 ms = 1,170 - 1,280 TFLOP/s, the tensor pipe busy 81 - 84 % of the cycles at 1.57 GHz (power
// cap); one product of 8192^3 0.73 - 0.83 ms where the library's took 0.68 - 0.70.  What is left: a 256-row item has no second accumulator buffer (512 columns are full),
// so its epilogue (2 - 5 us of 60) stands alone, and 512 rows of a group are often three tiles of 192.
// Every wait is bounded; on a give-up the CTA sets the status word, tells its cluster and still meets the others at the end; what the wait was for is not stored.
constexpr uint32_t GT_KS = 64;                                   // inputs per stage: 128 bytes, one swizzle row
constexpr uint32_t GT_STAGES = 4;
constexpr uint32_t GT_A_HALF = 128 * GT_KS * 2;                  // 128 outputs of a stage
constexpr uint32_t GT_A_BYTES = 2 * GT_A_HALF;                   // a CTA's outputs of a stage: one half per accumulator
constexpr uint32_t GT_B_BYTES = 128 * GT_KS * 2;                 // at most: a CTA's half of 256 rows
constexpr uint32_t GT_STAGE = GT_A_BYTES + GT_B_BYTES;
constexpr uint32_t GT_MAX_G = 1024;
constexpr uint32_t GT_EPI_WARPS = 8, GT_SLOT_WARPS = 2, GT_GATHER_WARPS = GT_SLOT_WARPS * GT_STAGES;   // gathered rows: two warps to a stage, four stages at once
constexpr uint32_t GT_X_SLOTS = 8;                                // at most: gathered rows have a ring of their own
constexpr uint32_t GT_X = GT_STAGES * GT_A_BYTES;                // the rows' operand, behind the weights' ring
constexpr uint32_t GT_THREADS = 64 + (GT_EPI_WARPS + GT_GATHER_WARPS) * 32;
constexpr uint32_t GT_TURN = 8 * 32 * 4;                         // an epilogue warp's turn of 16 rows x 32 outputs, two rows to a word
constexpr uint32_t GT_SMEM = GT_STAGES * GT_STAGE + GT_EPI_WARPS * 2 * GT_TURN + 1024;

constexpr uint32_t GT_PARTS = 4;                                  // most parts of a reduction: a cluster of eight CTAs
// The accumulator's additions truncate (1.7e-8 of the sum for each product of 16 inputs: 2.4e-6 after 2304 inputs; inputs of one sign, 65,536 of them
// in f16: 1e-4, near f16's half step), so for f32 outputs and for long sums of 16-bit ones the sums move on after as many stages as this: the epilogue
// warps add them, rounding, to running sums in the tensor memory's second half
// (bf16; products of f16 have 22 bits, of which more is cut: about one and a half times the error).  f32 outputs, K 512 to 6144, gate and up, random signs:
// bf16 9.6e-7 off 64 bits with eight stages, f16 1.3e-6, 6.9e-7 with four.  16384 rows of 32 groups, 2048 -> 6144: 569 us with eight, 677 with four.
constexpr uint32_t GT_CHAIN_BF16 = 7, GT_CHAIN_F16 = 4;
// 16-bit outputs: inputs from which on their sums move on, where a sum of one sign may drift by a sixteenth of the type's half step
constexpr uint32_t GT_LONG_F16 = 8192, GT_LONG_BF16 = 65536;
constexpr uint32_t GT_RUN = 256;                                 // first column of the running sums
constexpr uint32_t GT_BOXES = 5;
__host__ __device__ constexpr uint32_t gt_box_rows(uint32_t i) { return i < 3 ? 16u << i : 32 * i; }   // 16 32 64 96 128

struct TileParams {
    CUtensorMap w, x[GT_BOXES];   // x by box height
    GroupedArgs a;
    uint32_t n_ft, n_ks;          // output tiles of a row tile, stages
    uint32_t cap;                 // most rows of a tile: 64 (running sums), 128, 160, 192 or 256
    uint32_t w_loads;             // copies that a stage of weights takes
    uint32_t fmt;
    uint32_t parts;               // parts of the reduction, a CTA pair of the item's cluster to each (1: no cluster, pairs walk the items)
    uint32_t chain;               // running sums: stages after which an accumulator moves on
};

struct GtItem { uint32_t g, p0, rows, n; };   // group, first position, rows, MMA N (a multiple of 32)
// walks the call's row tiles: tile number -> group and rows.  A group's rows are cut into as few tiles as hold them, all alike.
struct GtWalk {
    const uint32_t *off, *tiles;   // [G][first, end], [G + 1] first row tile
    uint32_t G, g = 0;
    __device__ GtItem at(uint32_t tile) {
        if (tiles[g + 1] <= tile) {
            uint32_t lo = g + 1, hi = G;                   // tiles[lo] <= tile < tiles[hi]
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (tiles[mid] <= tile) lo = mid; else hi = mid;
            }
            g = lo;
        }
        const uint32_t r0 = off[2 * g], len = off[2 * g + 1] - r0, nt = tiles[g + 1] - tiles[g];
        const uint32_t per = ((len + nt - 1) / nt + 31) / 32 * 32, i = tile - tiles[g];
        GtItem it;
        it.g = g; it.p0 = r0 + i * per; it.rows = min(per, len - i * per); it.n = (it.rows + 31) / 32 * 32;
        return it;
    }
};

__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
        "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 bytes, or zeros where there is nothing to read.  No clobber of memory: the compiler may load the next rows' numbers meanwhile; the wait for the
// copies has one.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u));
}
__device__ __forceinline__ void st_shared4(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster16(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <bool SWIGLU, class O, bool SUMS>
__global__ void __launch_bounds__(GT_THREADS, 1) grouped_tile_kernel(const __grid_constant__ TileParams P) {
    extern __shared__ uint8_t smem_any[];
    __shared__ __align__(8) uint64_t full_bar[GT_STAGES], empty_bar[GT_STAGES], acc_full[2], acc_empty[2], x_full[GT_X_SLOTS], x_empty[GT_X_SLOTS];
    __shared__ uint32_t s_tmem, s_off[2 * GT_MAX_G], s_tiles[GT_MAX_G + 1], s_row[GT_GATHER_WARPS][128 / GT_SLOT_WARPS];
    __shared__ volatile int s_abort;
    const GroupedArgs& a = P.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    // the pair's even CTA leads; in a cluster of several pairs each takes a part of the reduction
    const uint32_t cl_rank = cluster_rank(), rank = cl_rank & 1u, leader = cl_rank & ~1u, part = cl_rank >> 1;
    const uint16_t pair_mask = (uint16_t)(3u << leader);
    const uint32_t ring = (smem_u32(smem_any) + 1023u) & ~1023u;
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < GT_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (uint32_t s = 0; s < GT_X_SLOTS; ++s) { mbar_init(&x_full[s], 2 * GT_SLOT_WARPS); mbar_init(&x_empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * GT_EPI_WARPS); }
        s_abort = 0;
        mbar_fence_init();
        tma_prefetch_map(&P.w);
    }
    // What came before on the stream is complete from here on; what follows may start its own beginning.  Tensor memory is taken only now: a CTA that
    // held it while it waited could keep it from the grid that it waits for.
    grid_dep_wait();
    grid_dep_launch();
    if (warp == 1) tmem_alloc_pair(&s_tmem, 512);
    // the groups' positions and row tiles
    for (uint32_t g = threadIdx.x; g < a.G; g += blockDim.x) {
        uint32_t r0, r1;
        if (!gp_range(a, g, r0, r1) && blockIdx.x == 0) atomicMax(a.status, ST_BAD_OFFSETS);
        s_off[2 * g] = r0; s_off[2 * g + 1] = r1;
    }
    __syncthreads();
    if (warp == 0) {
        const uint32_t per = (a.G + 31) / 32, g0 = min(lane * per, a.G), g1 = min(g0 + per, a.G);
        uint32_t mine = 0;
        for (uint32_t g = g0; g < g1; ++g) mine += (s_off[2 * g + 1] - s_off[2 * g] + P.cap - 1) / P.cap;
        uint32_t sum = mine;
        for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, o); if (lane >= o) sum += v; }
        uint32_t at = sum - mine;
        for (uint32_t g = g0; g < g1; ++g) { s_tiles[g] = at; at += (s_off[2 * g + 1] - s_off[2 * g] + P.cap - 1) / P.cap; }
        if (lane == 31) s_tiles[a.G] = sum;
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = s_tmem, n_items = s_tiles[a.G] * P.n_ft, pair = blockIdx.x / (2 * P.parts);
    // pairs walk the items; a cluster of several pairs takes one
    const uint32_t n_pairs = P.parts == 1 ? gridDim.x / 2 : max(n_items, 1u);
    const uint32_t ks0 = part * P.n_ks / P.parts, ks1 = (part + 1) * P.n_ks / P.parts;
    constexpr uint32_t FT = SWIGLU ? 256 : 512;                  // outputs of an item: half of them this CTA's
    // tensor memory: buffers of two accumulators of `cap` columns (with running sums: in the first half, those in the second)
    const uint32_t n_buf = (SUMS ? 128 : 256) / P.cap, n_chains = SUMS ? (ks1 - ks0 + P.chain - 1) / P.chain : 1;
    auto give_up = [&](uint32_t code) { if (!s_abort) atomicMax(a.status, code); s_abort = 1; };
    GtWalk walk{s_off, s_tiles, a.G};
    // gathered rows: as many slots as tiles of at most cap rows leave room for
    const uint32_t x_slot = P.cap * 64, x_slots = min(GT_STAGES * GT_B_BYTES / x_slot, GT_X_SLOTS);

    if (warp == 0) {
        // ---------------- producer: this CTA's outputs' weights, and its half of the tile's rows where they lie in order ----------------
        const bool gather = a.gather;
        uint32_t s = 0, ph = 0, n_stage = 0;
        bool ok = true;
        for (uint32_t i = pair; i < n_items && ok; i += n_pairs) {
            const GtItem it = walk.at(i / P.n_ft);
            const int32_t f0 = (int32_t)((i % P.n_ft) * FT + rank * (FT / 2)), g = (int32_t)it.g;
            const uint32_t hb = it.n / 2, b0 = it.p0 + rank * hb, bi = hb <= 16 ? 0 : hb <= 32 ? 1 : (hb + 31) / 32;
            const uint32_t bytes = 2 * (GT_A_BYTES + (gather ? 0 : gt_box_rows(bi) * GT_KS * 2));   // both CTAs' copies
            for (uint32_t ks = ks0; ks < ks1; ++ks) {
                if (!mbar_wait_warp_at(smem_u32(&empty_bar[s]), ph ^ 1u, &s_abort, a.poll_limit)) { give_up(ST_WAIT_EMPTY); ok = false; break; }
                if (lane == 0 && (!a.withhold || ++n_stage != a.withhold)) {
                    const uint32_t full = map_to_rank(smem_u32(&full_bar[s]), leader), sa = ring + s * GT_A_BYTES;
                    const int32_t k = (int32_t)(ks * GT_KS);
                    if (rank == 0) mbar_expect_tx(&full_bar[s], bytes);
                    if (!a.in_out) {
                        tma_load_4d(sa, &P.w, k, f0, 0, g, full);
                    } else if (SWIGLU) {
                        // 64 outputs, 64 inputs, gate and up: the halves of one accumulator's tile lie 16 KB apart in the box's order
                        tma_load_4d(sa, &P.w, f0, k, 0, g, full);
                        tma_load_4d(sa + GT_A_HALF, &P.w, f0 + 64, k, 0, g, full);
                    } else if (P.w_loads == 1) {
                        tma_load_4d(sa, &P.w, 0, k, f0 / 64, g, full);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) tma_load_4d(sa + j * (GT_A_HALF / 2), &P.w, f0 + j * 64, k, 0, g, full);
                    }
                    if (!gather) tma_load_2d(ring + GT_X + s * GT_B_BYTES, &P.x[bi], k, (int32_t)b0, full);
                }
                __syncwarp();
                if (++s == GT_STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: the even CTA's, for both ----------------
        if (rank == 0) {
            uint32_t s = 0, ph = 0, xs = 0, x_ph = 0, n_done = 0;
            bool ok = true;
            // K-major: 16 inputs are 32 bytes of every row; M-major: 16 rows of 128 bytes.  M-major 64-output tiles of one accumulator:
            // 8 KB apart, but for the activation's boxes (gate and up of 64 outputs) 16 KB
            const uint32_t a_step = a.in_out ? 2048u : 32u, a_lbo = !a.in_out ? 16u : SWIGLU ? GT_A_HALF : GT_A_HALF / 2;
            const uint32_t a_next = a.in_out && SWIGLU ? GT_A_HALF / 2 : GT_A_HALF;   // to the second accumulator's tile
            for (uint32_t i = pair; i < n_items && ok; i += n_pairs) {
                const GtItem it = walk.at(i / P.n_ft);
                const uint32_t idesc = umma_idesc_pair(P.fmt, it.n, a.in_out);
                for (uint32_t chain = 0; chain < n_chains && ok; ++chain) {
                    const uint32_t buf = n_done % n_buf, acc = tmem + buf * 2 * P.cap;
                    const uint32_t k0 = SUMS ? ks0 + chain * P.chain : ks0, k1 = SUMS ? min(k0 + P.chain, ks1) : ks1;
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(smem_u32(&acc_empty[buf]), (n_done / n_buf & 1u) ^ 1u, &s_abort, a.poll_limit));
                    if (!ok) { give_up(ST_WAIT_EMPTY); break; }
                    tc_fence_after();
                    for (uint32_t ks = k0; ks < k1; ++ks) {
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(smem_u32(&full_bar[s]), ph, &s_abort, a.poll_limit));
                        if (ok && a.gather) ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(smem_u32(&x_full[xs]), x_ph, &s_abort, a.poll_limit));
                        if (!ok) { give_up(ST_WAIT_FULL); break; }
                        tc_fence_after();
                        const uint32_t sa = ring + s * GT_A_BYTES, sb = ring + GT_X + (a.gather ? xs * x_slot : s * GT_B_BYTES);
                        if (elect_one()) {
#pragma unroll
                            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                                for (uint32_t j = 0; j < GT_KS / 16; ++j)
                                    umma_f16_pair(acc + h * P.cap, umma_desc_sw128(sa + h * a_next + j * a_step, a_lbo, 1024),
                                                  umma_desc_sw128(sb + j * 32, 16, 1024), idesc, ks != k0 || j ? 1u : 0u);
                            umma_commit_pair(smem_u32(&empty_bar[s]), pair_mask);
                            if (a.gather) umma_commit_pair(smem_u32(&x_empty[xs]), pair_mask);
                        }
                        __syncwarp();
                        if (++s == GT_STAGES) { s = 0; ph ^= 1u; }
                        if (++xs == x_slots) { xs = 0; x_ph ^= 1u; }
                    }
                    if (!ok) break;
                    if (elect_one()) umma_commit_pair(smem_u32(&acc_full[buf]), pair_mask);
                    __syncwarp();
                    ++n_done;
                }
            }
        }
    } else if (warp < 2 + GT_EPI_WARPS) {
        // ---------------- epilogue: a thread owns a lane (output) of both accumulators; a warp every other 16 rows of the tile ----------------
        const uint32_t q = warp & 3u, half = (warp - 2) >> 2;
        uint32_t n_done = 0;
        O* y = static_cast<O*>(a.y);
        const uint32_t turn = ring + GT_STAGES * GT_STAGE + (warp - 2) * 2 * GT_TURN;
        for (uint32_t i = pair; i < n_items; i += n_pairs) {
            const GtItem it = walk.at(i / P.n_ft);
            const uint32_t f = (i % P.n_ft) * FT + rank * (FT / 2) + q * 32 + lane;
            bool ok = true;
            for (uint32_t chain = 0; chain < n_chains; ++chain) {
            const uint32_t buf = n_done % n_buf, lanes = (q * 32u) << 16;
            const bool last = !SUMS || chain + 1 == n_chains;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(smem_u32(&acc_full[buf]), n_done / n_buf & 1u, &s_abort, a.poll_limit));
            if (!ok) { give_up(ST_WAIT_FULL); break; }
            tc_fence_after();
            for (uint32_t c = half * 16; c < it.rows; c += 32) {
                uint32_t v0[16], v1[16];
                tmem_ld16_nowait(tmem + buf * 2 * P.cap + c + lanes, v0);
                tmem_ld16_nowait(tmem + buf * 2 * P.cap + P.cap + c + lanes, v1);
                if (SUMS && chain) {
                    uint32_t r0[16], r1[16];
                    tmem_ld16_nowait(tmem + GT_RUN + c + lanes, r0);
                    tmem_ld16_nowait(tmem + GT_RUN + P.cap + c + lanes, r1);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        v0[j] = __float_as_uint(__uint_as_float(r0[j]) + __uint_as_float(v0[j]));
                        v1[j] = __float_as_uint(__uint_as_float(r1[j]) + __uint_as_float(v1[j]));
                    }
                }
                if (!last) {
                    tmem_wait_ld();
                    tmem_st16(tmem + GT_RUN + c + lanes, v0);
                    tmem_st16(tmem + GT_RUN + P.cap + c + lanes, v1);
                    continue;
                }
                if (P.parts > 1) {
                    // a part's sums, where the ring was (its copies have landed, the products have read them): [accumulator][row][128 outputs]
                    tmem_wait_ld();
                    const uint32_t z = ring + (c * 128 + q * 32 + lane) * 4;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        st_shared4(z + j * 512, v0[j]);
                        st_shared4(z + (P.cap + j) * 512, v1[j]);
                    }
                    continue;
                }
                // lane j < 16: where row c + j of the tile goes
                uint32_t yr = 0xFFFFFFFFu;
                if (lane < 16 && c + lane < it.rows) {
                    const uint32_t p = it.p0 + c + lane, o = a.order ? a.order[p] : p;
                    yr = a.scatter ? o : p;
                    if ((a.gather && o / a.x_div >= a.x_rows) || yr >= a.y_rows) { yr = 0xFFFFFFFFu; atomicMax(a.status, ST_BAD_ROW); }
                }
                tmem_wait_ld();
                if constexpr (sizeof(O) == 4) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint32_t row = __shfl_sync(0xFFFFFFFFu, yr, j);
                        if (row == 0xFFFFFFFFu) continue;
                        float* o = reinterpret_cast<float*>(y) + (size_t)row * a.ld_y + f;
                        if (SWIGLU) {
                            if (f < a.N) *o = gp_swiglu<true>(__uint_as_float(v0[j]), __uint_as_float(v1[j]), a.limit);
                        } else {
                            if (f < a.N) *o = __uint_as_float(v0[j]);
                            if (f + 128 < a.N) o[128] = __uint_as_float(v1[j]);
                        }
                    }
                } else {
                    // two rows to a word, turned through shared memory: a lane then stores four outputs (8 bytes) of a row, a warp
                    // instruction four rows
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float x0 = __uint_as_float(v0[2 * k]), x1 = __uint_as_float(v0[2 * k + 1]);
                        const float z0 = __uint_as_float(v1[2 * k]), z1 = __uint_as_float(v1[2 * k + 1]);
                        if (SWIGLU) {
                            st_shared4(turn + (k * 32 + lane) * 4, pack2(gp_swiglu<false>(x0, z0, a.limit), gp_swiglu<false>(x1, z1, a.limit), O()));
                        } else {
                            st_shared4(turn + (k * 32 + lane) * 4, pack2(x0, x1, O()));
                            st_shared4(turn + GT_TURN + (k * 32 + lane) * 4, pack2(z0, z1, O()));
                        }
                    }
                    __syncwarp();
                    const uint32_t fq = f - lane + (lane & 7u) * 4;
                    constexpr uint32_t HALVES = SWIGLU ? 1 : 2;
                    uint4 w[2][HALVES];                  // all read before the first is used
#pragma unroll
                    for (uint32_t i2 = 0; i2 < 2; ++i2)
#pragma unroll
                        for (uint32_t h = 0; h < HALVES; ++h) w[i2][h] = ld_shared16(turn + h * GT_TURN + ((lane >> 3) + 4 * i2) * 128 + (lane & 7u) * 16);
#pragma unroll
                    for (uint32_t i2 = 0; i2 < 2; ++i2) {
                        const uint32_t k = (lane >> 3) + 4 * i2;
                        const uint32_t ra = __shfl_sync(0xFFFFFFFFu, yr, 2 * k), rb = __shfl_sync(0xFFFFFFFFu, yr, 2 * k + 1);
                        O *oa = y + (size_t)ra * a.ld_y + fq, *ob = y + (size_t)rb * a.ld_y + fq;
#pragma unroll
                        for (uint32_t h = 0; h < HALVES; ++h) {
                            const uint4 v = w[i2][h];
                            if (fq + h * 128 < a.N) {
                                if (ra != 0xFFFFFFFFu) *reinterpret_cast<uint2*>(oa + h * 128) = make_uint2(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.z, v.w, 0x5410));
                                if (rb != 0xFFFFFFFFu) *reinterpret_cast<uint2*>(ob + h * 128) = make_uint2(__byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x7632));
                            }
                        }
                    }
                }
            }
            if (!last) tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[buf]), leader));
            ++n_done;
            }
            if (!ok) break;
        }
    } else if (a.gather) {
        // ---------------- gathered rows: two warps to every fourth stage, so that waiting for its copies keeps nobody; eight lanes copy 128 bytes of a row ----------------
        // (one arrival per warp and stage: with one per thread, posted by the copies themselves, the arrivals took longer than the stage).  Their ring is
        // their own and as deep as the tile's rows allow, so that they are there before the weights: a weights slot that waited for its rows
        // stood idle meanwhile (K 4096, 2 x 2048 outputs: 2400 Zipf rows of 64
        // groups 377 us with the rows in the weights' slots, 360 now, 338 in sorted order; 512 rows of 64, K 5120, 490 and 462).
        const uint32_t gw = warp - 2 - GT_EPI_WARPS, turn = gw % GT_STAGES, share = gw / GT_STAGES, r_in = lane >> 3, chunk = lane & 7u;
        uint32_t slot = turn, ph = 0, base = 0;                   // base: stages of the items before, modulo the turns
        bool ok = true;
        // this CTA's rows of an item's tile (what the columns behind the tile's last row hold is not stored), and how many of them are this warp's: every second
        const auto rows_of = [&](uint32_t i, uint32_t& p0) {
            const GtItem it = walk.at(i / P.n_ft);
            const uint32_t hb = it.n / 2, t0 = rank * hb, valid = it.rows > t0 ? min(hb, it.rows - t0) : 0;
            p0 = it.p0 + t0 + share;
            return (valid + GT_SLOT_WARPS - 1 - share) / GT_SLOT_WARPS;
        };
        uint32_t next[128 / GT_SLOT_WARPS / 32], mine = 0;       // the next item's rows: asked for an item ahead
        const auto ask_rows = [&](uint32_t i) {
            if (i >= n_items) return 0u;
            uint32_t p0;
            const uint32_t n = rows_of(i, p0);
#pragma unroll
            for (uint32_t k = 0; k < 128 / GT_SLOT_WARPS / 32; ++k) next[k] = lane + k * 32 < n ? a.order[p0 + (lane + k * 32) * GT_SLOT_WARPS] : 0;
            return n;
        };
        uint32_t n_next = ask_rows(pair);
        for (uint32_t i = pair; i < n_items && ok; i += n_pairs) {
            __syncwarp();
            mine = n_next;
#pragma unroll
            for (uint32_t k = 0; k < 128 / GT_SLOT_WARPS / 32; ++k) {
                const uint32_t xr = next[k] / a.x_div;
                s_row[gw][lane + k * 32] = xr < a.x_rows ? xr : 0;    // out of range: reads row 0, the epilogue skips it
            }
            __syncwarp();
            n_next = ask_rows(i + n_pairs);
            for (uint32_t ks = ks0 + (turn + GT_STAGES - base) % GT_STAGES; ks < ks1; ks += GT_STAGES) {
                const uint32_t sb = ring + GT_X + slot * x_slot;
                if (!mbar_wait_warp_at(smem_u32(&x_empty[slot]), ph ^ 1u, &s_abort, a.poll_limit)) { give_up(ST_WAIT_EMPTY); ok = false; break; }
                const uint32_t k = ks * GT_KS + chunk * 8;
                const bool there = k < a.K;                       // K is a multiple of 8
                const uint16_t* x = static_cast<const uint16_t*>(a.x) + (there ? k : 0);
#pragma unroll 8
                for (uint32_t i = r_in; i < mine; i += 4) {
                    const uint32_t r = i * GT_SLOT_WARPS + share;
                    cp_async16(sb + r * 128 + ((chunk ^ (r & 7u)) << 4), x + (size_t)s_row[gw][i] * a.ld_x, there);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&x_full[slot]), leader));
                slot += GT_STAGES;                                // at most as many as the ring has
                if (slot >= x_slots) { slot -= x_slots; ph ^= 1u; }
            }
            base = (base + ks1 - ks0) % GT_STAGES;
        }
    }
    // every thread comes here, also after a give-up
    if (s_abort) cluster_abort(&s_abort, 2 * P.parts);
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    const bool gave_up = s_abort != 0;                  // in every CTA of the cluster alike: a part of the sums may be missing
    if (gave_up) abort_drain();
    if (P.parts > 1 && pair < n_items && !gave_up) {
        // the parts of a share of the rows, in order, over distributed shared memory: a thread four outputs of a row, of both accumulators
        GtWalk w{s_off, s_tiles, a.G};
        const GtItem it = w.at(pair / P.n_ft);
        const uint32_t c0 = part * it.rows / P.parts, c1 = (part + 1) * it.rows / P.parts, f0 = (pair % P.n_ft) * FT + rank * (FT / 2);
        for (uint32_t i = threadIdx.x; i < (c1 - c0) * 32; i += GT_THREADS) {
            const uint32_t c = c0 + i / 32, f = f0 + i % 32 * 4, p = it.p0 + c, o = a.order ? a.order[p] : p, yr = a.scatter ? o : p;
            if ((a.gather && o / a.x_div >= a.x_rows) || yr >= a.y_rows) { atomicMax(a.status, ST_BAD_ROW); continue; }
            float4 w4[GT_PARTS][2], v[2];
#pragma unroll
            for (uint32_t s = 0; s < GT_PARTS; ++s)          // all on their way before the first is added
                if (s < P.parts) {
                    const uint32_t z = map_to_rank(ring + (c * 128 + i % 32 * 4) * 4, 2 * s + rank);
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) w4[s][h] = ld_cluster16(z + h * P.cap * 512);
                }
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                v[h] = w4[0][h];
#pragma unroll
                for (uint32_t s = 1; s < GT_PARTS; ++s)
                    if (s < P.parts) v[h] = make_float4(v[h].x + w4[s][h].x, v[h].y + w4[s][h].y, v[h].z + w4[s][h].z, v[h].w + w4[s][h].w);
            }
            if (SWIGLU)
                v[0] = make_float4(gp_swiglu<sizeof(O) == 4>(v[0].x, v[1].x, a.limit), gp_swiglu<sizeof(O) == 4>(v[0].y, v[1].y, a.limit),
                                   gp_swiglu<sizeof(O) == 4>(v[0].z, v[1].z, a.limit), gp_swiglu<sizeof(O) == 4>(v[0].w, v[1].w, a.limit));
            O* y = static_cast<O*>(a.y) + (size_t)yr * a.ld_y + f;
#pragma unroll
            for (uint32_t h = 0; h < (SWIGLU ? 1u : 2u); ++h) {
                if (f + h * 128 >= a.N) continue;
                if constexpr (sizeof(O) == 4) *reinterpret_cast<float4*>(y + h * 128) = v[h];
                else *reinterpret_cast<uint2*>(y + h * 128) = make_uint2(pack2(v[h].x, v[h].y, O()), pack2(v[h].z, v[h].w, O()));
            }
        }
    }
    if (P.parts > 1) { __syncwarp(); cluster_sync_all(); }   // nobody's shared memory goes away under a reader
    tc_fence_after();
    if (warp == 1) tmem_free_pair(tmem, 512);
}

// clusters of 1 .. 4 CTA pairs that the device holds at once
struct GtClusters { uint32_t n[GT_PARTS + 1]; };
static GtClusters gt_clusters(const void* kernel, int sm_count) {
    GtClusters c{};
    for (uint32_t parts = 1; parts <= GT_PARTS; ++parts) {
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2 * parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2 * parts * 74); cfg.blockDim = dim3(GT_THREADS); cfg.dynamicSmemBytes = GT_SMEM; cfg.attrs = &attr; cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = sm_count / (int)(2 * parts); }
        c.n[parts] = n > 0 ? (uint32_t)n : 1u;
    }
    return c;
}
// How a call is cut: rows of a tile at most (128: two accumulator buffers; more: one; the parts' sums fit where the ring was up to 192) and parts of
// the reduction (one group, K 5120, N 2304: 300 rows 31 us in one part, 22 in two, 18 in four; 777 rows in tiles of 160 38 and 28; 1500 rows in tiles
// of 128 35 and 45).  The groups' sizes are on the device; the estimate takes them as equal.  A stage costs its products (4.4 cycles a row) or its
// bytes (62 a cycle), whichever is longer; joining parts costs 50 cycles a row, and what has parts starts anew with each wave of clusters.  Returns the
// row tiles that the call can have at most.
// sums: 64 rows and two buffers beside the running sums, or 128 and one that the products wait for
static uint32_t gt_cut(const GroupedArgs& a, bool sums, uint32_t n_ft, uint32_t n_ks, const GtClusters& room, uint32_t* cap, uint32_t* parts) {
    const uint32_t groups = a.G < a.rows ? a.G : a.rows, per = (a.rows + groups - 1) / groups;
    double best = 0;
    for (const uint32_t c : {64u, 128u, 160u, 192u, 256u})
        for (uint32_t s = 1; s <= (c <= 192 ? GT_PARTS : 1u) && s <= n_ks; ++s) {
            if (sums ? c > 128 : c == 64) continue;
            const uint32_t tiles = (per + c - 1) / c, n = ((per + tiles - 1) / tiles + 31) / 32 * 32;
            const uint64_t items = (uint64_t)groups * tiles * n_ft, waves = (items + room.n[s] - 1) / room.n[s];
            const double stage = 4.4 * n > (32768 + n * 64) / 62.0 ? 4.4 * n : (32768 + n * 64) / 62.0;
            const double wave = (n_ks + s - 1) / s * stage * (sums && c == 128 ? 1.2 : 1.0) + (s > 1 ? 50.0 * n : c > 128 ? 3000 : 0);
            const double t = waves * wave + (s > 1 ? (waves - 1) * 6000.0 : 0);
            if (best == 0 || t < best) { best = t; *cap = c; *parts = s; }
        }
    return a.rows / *cap + groups;
}

template <bool SWIGLU, class O, bool SUMS>
static cudaError_t tile_launch(const GroupedArgs& a, cudaStream_t st) {
    TileParams P;
    P.a = a;
    P.n_ft = (a.N + (SWIGLU ? 255 : 511)) / (SWIGLU ? 256 : 512);
    P.n_ks = (a.K + GT_KS - 1) / GT_KS;
    P.fmt = a.dtype == DT_BF16 ? UMMA_BF16 : UMMA_F16;
    P.w_loads = 1;
    const auto kernel = grouped_tile_kernel<SWIGLU, O, SUMS>;
    cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GT_SMEM);
    if (set != cudaSuccess) return set;
    static const GtClusters room = gt_clusters(reinterpret_cast<const void*>(kernel), a.sm_count);
    const uint32_t most_tiles = gt_cut(a, SUMS, P.n_ft, P.n_ks, room, &P.cap, &P.parts);
    // a part's stages in as few chains as hold them, all alike
    const uint32_t part_ks = (P.n_ks + P.parts - 1) / P.parts, most_chain = a.dtype == DT_BF16 ? GT_CHAIN_BF16 : GT_CHAIN_F16;
    const uint32_t chains = (part_ks + most_chain - 1) / most_chain;
    P.chain = (part_ks + chains - 1) / chains;
    cudaError_t e;
    const uint64_t N = a.N, K = a.K, G = a.G, ld = a.ld_w, gs = a.w_stride;
    // A box is one CTA's weights of a stage.  Activation: gate rows, then up rows (outputs first), or 64 outputs' gate and up
    // (inputs first).  Plain, inputs first: four blocks of 64 outputs, by one copy where the outputs are a multiple of 64
    if (!a.in_out)
        e = SWIGLU ? encode_map<4>(&P.w, a.dtype, a.w, {K, N, 2, G}, {ld, N * ld, gs}, {64, 128, 2, 1})
                   : encode_map<4>(&P.w, a.dtype, a.w, {K, N, 1, G}, {ld, ld, gs}, {64, 256, 1, 1});
    else if (SWIGLU)
        e = encode_map<4>(&P.w, a.dtype, a.w, {N, K, 2, G}, {ld, N, gs}, {64, 64, 2, 1});
    else if (N % 64 == 0)
        e = encode_map<4>(&P.w, a.dtype, a.w, {64, K, N / 64, G}, {ld, 64, gs}, {64, 64, 4, 1});
    else {
        P.w_loads = 4;
        e = encode_map<4>(&P.w, a.dtype, a.w, {N, K, 1, G}, {ld, ld, gs}, {64, 64, 1, 1});
    }
    for (uint32_t i = 0; i < GT_BOXES && !a.gather && e == cudaSuccess; ++i)
        e = encode_map<2>(&P.x[i], a.dtype, a.x, {K, a.x_rows}, {a.ld_x}, {64, gt_box_rows(i)});
    if (e != cudaSuccess) return e;
    const uint32_t clusters = P.parts == 1 ? (uint32_t)a.sm_count / 2 : most_tiles * P.n_ft;
    return launch_dependent_clusters(kernel, 2 * P.parts, clusters, GT_THREADS, GT_SMEM, st, P);
}
template <bool BF16, class O>
static cudaError_t grouped_out(const GroupedArgs& a, cudaStream_t st) {
    if (a.rows <= GN_ROWS) {
        if (a.in_out) return a.swiglu ? few_launch<BF16, true, true, O>(a, st) : few_launch<BF16, true, false, O>(a, st);
        return a.swiglu ? few_launch<BF16, false, true, O>(a, st) : few_launch<BF16, false, false, O>(a, st);
    }
    if (sizeof(O) == 4 || a.K > (BF16 ? GT_LONG_BF16 : GT_LONG_F16)) return a.swiglu ? tile_launch<true, O, true>(a, st) : tile_launch<false, O, true>(a, st);
    return a.swiglu ? tile_launch<true, O, sizeof(O) == 4>(a, st) : tile_launch<false, O, sizeof(O) == 4>(a, st);
}
cudaError_t launch_grouped(const GroupedArgs& a, cudaStream_t st) {
    if (a.dtype == DT_BF16) return a.out_dtype == DT_F32 ? grouped_out<true, float>(a, st) : grouped_out<true, __nv_bfloat16>(a, st);
    return a.out_dtype == DT_F32 ? grouped_out<false, float>(a, st) : grouped_out<false, __half>(a, st);
}

__global__ void __launch_bounds__(256) gate_up_act_kernel(const float* __restrict__ gate_up, uint32_t T, uint32_t I, float limit, __nv_bfloat16* __restrict__ h) {
    const size_t n = (size_t)T * (I / 4);                   // four outputs to a thread
    grid_dep_wait();
    grid_dep_launch();
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t t = i / (I / 4), f = i % (I / 4) * 4;
        const float4 g = *reinterpret_cast<const float4*>(gate_up + t * 2 * I + f), u = *reinterpret_cast<const float4*>(gate_up + t * 2 * I + I + f);
        *reinterpret_cast<uint2*>(h + t * I + f) =
            make_uint2(pack2(gp_swiglu<true>(g.x, u.x, limit), gp_swiglu<true>(g.y, u.y, limit), __nv_bfloat16()),
                       pack2(gp_swiglu<true>(g.z, u.z, limit), gp_swiglu<true>(g.w, u.w, limit), __nv_bfloat16()));
    }
}
cudaError_t launch_gate_up_act(const float* gate_up, uint32_t T, uint32_t I, float limit, __nv_bfloat16* h, cudaStream_t st) {
    const size_t blocks = ((size_t)T * (I / 4) + 255) / 256;
    return launch_dependent(true, gate_up_act_kernel, dim3((uint32_t)(blocks < 2368 ? blocks : 2368)), dim3(256), 0, st, gate_up, T, I, limit, h);
}

}  // namespace mlxs
