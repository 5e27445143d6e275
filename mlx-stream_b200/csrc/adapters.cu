// Low-rank adapters of many requests beside a shared projection: y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t].
//
// Both factors are thin (rank <= 256 of thousands), so the work is bytes and, for few tokens, latency: x, base and y once, an adapter's A and B once per unit
// of up to 64 tokens that use it.  A cluster of C CTAs takes a unit: every CTA sums a C-th of the inputs, the sums meet over distributed shared memory
// (always in the same order, no atomics: a call repeats itself), every CTA then makes a C-th of the outputs.  C is as large as the units leave SMs for.
//   * Up to 64 tokens (of 512 adapters and more: up to 511), or 2048 adapters and more: adapters_tile_kernel, a tile of 64 tokens, whose distinct adapters
//     are dealt out over `slots` clusters.
//   * More tokens (or more than 16 that have 14 per adapter): every CTA sorts the ids of a segment of up to 2048 tokens by itself, so that an adapter's
//     tokens, wherever they lie, share its units (999 mixed tokens of 24 adapters: 318 us by tiles, 145 sorted).  From 16 tokens per unit on, and ranks
//     40 to 128 where there is enough work, adapters_tensor_kernel (tcgen05); otherwise adapters_sorted_kernel (mma.sync).
//   * u = A x is kept as 16-bit parts, each the rounding of what the ones before it leave: two, 16 (bf16) or 22 (f16) bits, so that what is lost between the
//     factors is far inside an output's rounding; three of bf16, 24 bits, where outputs are f32 (rank 64, 5120 inputs, no base: two parts 2.5e-6 off 64 bits,
//     f32 2.3e-7).  f16 parts are scaled by the row's largest power of two, since A x may pass f16's range where y does not.
//   * base is added in f32, one rounding.
// Measured (GPU time, other inputs every call): one token of rank 16, 5120 -> 2304: 7.3 us, a chain of two cluster barriers and three cold loads; 64 tokens of 48
// adapters, rank 32: 10.3 us (floor 1.7), f32 outputs 11.2; 4000 of eight, rank 32: 38.5 us (floor 12.5), f32 outputs 44; 8192 tokens of six, rank 64, 4096 -> 2048: 56.5 us (floor
// 19.7), f32 outputs 68; 999 of 24, rank 128, f16, f32 outputs: 37 us (floor 10.3); 8192 of six, rank 256 (mma.sync): 290 us (floor 23), f32 outputs 382.
// The mma.sync kernels take operands straight from global memory as fragments, 16 bytes per lane: a lane's eight consecutive inputs stand for the k
// positions 2t, 2t+1, 2t+8, 2t+9 of two products, the same for both operands.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tensor_map.cuh"
#include "umma_pair.cuh"

namespace mlxs {

constexpr uint32_t AD_TT = 64;          // tokens of a tile
constexpr uint32_t AD_WARPS = 8;
constexpr uint32_t AD_MR = 64;          // rank rows of a pass
constexpr uint32_t AD_KS = 64, AD_STAGES = 4;   // inputs of a stage, stages of the ring (more than 16 tokens)
constexpr uint32_t AD_ROW = AD_KS * 2;          // bytes of a row of a stage
// The matrix instruction truncates where it adds.  How the sums are kept: in one accumulator; the inner product's in chains of ad_chain products of 16
// inputs, added with rounding (f32 outputs: 4000 f16 tokens of rank 16, 5120 inputs, in one accumulator 9.0e-7 off 64 bits, of one sign 3.2e-6; f32 sums 3.9e-7);
// the outer product's too, 32 rank columns by themselves (f32 outputs above rank 128: up to 48 products, 1.03e-6 in one accumulator).  Kernels of their
// own: beside one another their registers cost every call.
enum AdSums { AD_PLAIN, AD_CHAINED, AD_ROUNDED };
template <class O, AdSums SUMS>
constexpr uint32_t ad_chain = SUMS == AD_PLAIN ? 0 : sizeof(O) == 4 ? 16 : 64;
constexpr uint32_t AD_LONG = 16384;              // 16-bit outputs: one accumulator to so many inputs (512 products at most)

__device__ __forceinline__ uint4 ad_ld16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// not volatile: the compiler may put operand loads between the products
template <class T>
__device__ __forceinline__ void ad_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ad_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ad_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float ad_f32(float v) { return v; }
__device__ __forceinline__ void ad_round(float v, float& o) { o = v; }
__device__ __forceinline__ void ad_round(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void ad_round(float v, __half& o) { o = __float2half_rn(v); }
// 16-bit parts of the inner product
template <class T, class O>
constexpr int AD_PARTS = std::is_same<T, __nv_bfloat16>::value && sizeof(O) == 4 ? 3 : 2;
// two values as NP 16-bit parts each, packed, the largest first
template <class T, int NP>
__device__ __forceinline__ void ad_split(float x, float y, uint32_t (&parts)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        T h[2];
        ad_round(x, h[0]); ad_round(y, h[1]);
        parts[p] = *reinterpret_cast<uint32_t*>(h);
        // an infinity has no remainder
        x = isinf(ad_f32(h[0])) ? 0.f : x - ad_f32(h[0]);
        y = isinf(ad_f32(h[1])) ? 0.f : y - ad_f32(h[1]);
    }
}
// eight 16-bit values of which the first n count
__device__ __forceinline__ uint4 ad_first(uint4 v, int n) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = n >= 2 * i + 2 ? w[i] : n == 2 * i + 1 ? w[i] & 0xFFFFu : 0u;
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ float2 ad_ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void ad_st_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

struct AdSmem {                          // dynamic shared memory, byte offsets
    // rp: rank rows that a pass writes; u: the 16-bit parts, u_part bytes each; pitch: bytes of a token in one, 64 modulo 128 (rows on other banks)
    uint32_t part, u, u_part, bytes, r16, rp, pitch, stage;
};
__host__ __device__ inline AdSmem ad_smem(uint32_t R, uint32_t tokens, uint32_t n_parts) {
    AdSmem s;
    s.r16 = (R + 15) / 16 * 16;
    s.rp = R <= 16 ? 16 : R <= 32 ? 32 : AD_MR;
    s.pitch = (R + 31) / 32 * 64;
    if (s.pitch % 128 == 0) s.pitch += 64;
    // one after the other: the ring of operands, the warps' sums, the 16-bit parts
    s.u = 0;
    s.u_part = AD_TT * s.pitch;
    s.stage = (AD_TT + s.rp) * AD_ROW;
    const uint32_t warps = AD_WARPS * 16 * (s.rp + 4) * 4, ring = tokens > 16 ? AD_STAGES * s.stage : 0;
    s.part = n_parts * s.u_part > warps ? n_parts * s.u_part : warps;
    if (ring > s.part) s.part = ring;
    s.bytes = s.part + s.r16 * AD_TT * 4;
    return s;
}

// The sums of a warp, one token's rank rows side by side, rows of rp + 4 floats: a fragment's stores and the reads along the rank meet no bank twice.
// `more`: added to what is there.
template <int MT, int NT>
__device__ __forceinline__ void ad_put_sums(const float (&acc)[MT][NT][4], float* out, uint32_t rp, uint32_t m0, bool more = false) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float* const o = out + (n * 8 + 2 * t + (e & 1)) * (rp + 4) + (m0 + m) * 16 + g + (e >> 1) * 8;
                *o = more ? *o + acc[m][n][e] : acc[m][n][e];
            }
}

// One warp's share of the inner products of MT x 16 rank rows from r0 on and NT x 8 tokens: k blocks of 32 from kb on, every `step`-th.
// The next block's operands are asked for before a block's products run.  Rows behind the last token, and rank rows behind the last, read the
// first: what their products are is not looked at.
// CHAIN: products after which the accumulators move on to the warp's sums, or 0.
template <class T, int MT, int NT, uint32_t CHAIN>
__device__ __forceinline__ void ad_inner(const AdaptersArgs& a, const T* A, uint32_t R, uint32_t r0, const uint32_t* rows, uint32_t n_rows, uint32_t t0,
                                         uint32_t kb, uint32_t kb_end, uint32_t step, float* out, uint32_t rp) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float acc[MT][NT][4] = {};
    const T *xr[NT], *ar[MT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) xr[n] = static_cast<const T*>(a.x) + (size_t)(t0 + rows[n * 8 + g < n_rows ? n * 8 + g : 0]) * a.ld_x + t * 8;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) ar[m][h] = A + (size_t)(r0 + m * 16 + h * 8 + g < R ? r0 + m * 16 + h * 8 + g : r0) * a.K + t * 8;
    struct Block { uint4 x[NT], w[MT][2]; } b0, b1;
    auto ask = [&](Block& b, uint32_t at) {
        const uint32_t k = at * 32;
        const bool in = at < kb_end && k + t * 8 < a.K;
#pragma unroll
        for (int n = 0; n < NT; ++n) b.x[n] = in ? ad_ld16(xr[n] + k) : zero;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) b.w[m][h] = in ? ad_ld16(ar[m][h] + k) : zero;
    };
    auto multiply = [&](const Block& b) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                ad_mma<T>(acc[m][n], b.w[m][0].x, b.w[m][1].x, b.w[m][0].y, b.w[m][1].y, b.x[n].x, b.x[n].y);
                ad_mma<T>(acc[m][n], b.w[m][0].z, b.w[m][1].z, b.w[m][0].w, b.w[m][1].w, b.x[n].z, b.x[n].w);
            }
    };
    ask(b0, kb);
    uint32_t chain = 0;
    bool more = false;
#pragma unroll 1
    for (; kb < kb_end; kb += 2 * step) {
        if (CHAIN && chain == CHAIN) {
            ad_put_sums<MT, NT>(acc, out, rp, 0, more);
#pragma unroll
            for (int i = 0; i < MT * NT * 4; ++i) acc[i / (NT * 4)][i / 4 % NT][i % 4] = 0.f;
            more = true; chain = 0;
        }
        chain += 4;
        ask(b1, kb + step);
        multiply(b0);
        ask(b0, kb + 2 * step);
        multiply(b1);
    }
    ad_put_sums<MT, NT>(acc, out, rp, 0, more);
}

__device__ __forceinline__ void ad_copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ uint4 ad_lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
// 17 .. 64 tokens: the rows of x and A go through a ring of stages of 64 inputs in shared memory (fragment loads straight from memory keep too few
// bytes in flight: 2 TB/s over the GPU).  In a stage 16-byte chunk c of row r lies at c ^ (4 (r odd)): the eight lanes of a load phase (two rows,
// four chunks) meet no bank twice.  A warp takes 16 NH tokens from row n0 on, block kq of the stage's two blocks of 32 inputs, and MT of the pass'
// m-tiles from m0 on.  Rows that were not copied give products that are not looked at.  CHAIN: products after which the accumulators move on to
// sums in registers, or 0.
template <class T, int MT, int NT, uint32_t CHAIN>
__device__ __forceinline__ void ad_inner_ring(const AdaptersArgs& a, const AdSmem& L, const T* A, uint32_t r0, uint32_t rr, const uint32_t* rows,
                                              uint32_t n_rows, uint32_t t0, uint32_t k0, uint32_t k1, uint32_t smem, uint32_t n0, uint32_t kq, uint32_t m0,
                                              float* out) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t n_st = (k1 - k0 + AD_KS - 1) / AD_KS, chunk = tid & 7u, row0 = tid >> 3;      // eight threads to a row, 32 rows at a time
    const uint32_t a_at = AD_TT * AD_ROW, to0 = smem + row0 * AD_ROW + ((chunk ^ ((row0 & 1u) << 2)) << 4);
    const T *xs[2], *as[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = row0 + i * 32;
        xs[i] = r < n_rows ? static_cast<const T*>(a.x) + (size_t)(t0 + rows[r]) * a.ld_x + k0 + chunk * 8 : nullptr;
        as[i] = r < rr ? A + (size_t)(r0 + r) * a.K + k0 + chunk * 8 : nullptr;
    }
    float acc[MT][NT][4] = {}, sum[MT][NT][4] = {};
    uint32_t ask_slot = 0, ask_st = 0, chain = 0;
    auto ask = [&]() {
        if (ask_st < n_st) {
            const uint32_t to = to0 + ask_slot * L.stage, k = ask_st * AD_KS;
            const bool in = k0 + k + chunk * 8 < k1;          // else: zeros, from the row's first bytes
            const uint32_t from = in ? k : 0;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                if (xs[i]) ad_copy16(to + i * 32 * AD_ROW, (in ? xs[i] : xs[i] - chunk * 8) + from, in);
                if (as[i]) ad_copy16(to + a_at + i * 32 * AD_ROW, (in ? as[i] : as[i] - chunk * 8) + from, in);
            }
        }
        ask_slot = ask_slot + 1 == AD_STAGES ? 0 : ask_slot + 1;
        ++ask_st;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (uint32_t st = 0; st + 1 < AD_STAGES; ++st) ask();
    const uint32_t frag = smem + g * AD_ROW + (((kq * 4 + t) ^ ((g & 1u) << 2)) << 4);     // rows g and g + 8 have the same parity
    const uint32_t x_frag = frag + n0 * AD_ROW, a_frag = frag + a_at + m0 * 16 * AD_ROW;
    uint32_t slot = 0;
#pragma unroll 1
    for (uint32_t st = 0; st < n_st; ++st) {
        asm volatile("cp.async.wait_group %0;" ::"n"(AD_STAGES - 2) : "memory");
        __syncthreads();
        ask();
        const uint32_t xa = x_frag + slot * L.stage, aa = a_frag + slot * L.stage;
        slot = slot + 1 == AD_STAGES ? 0 : slot + 1;
        uint4 x[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n] = ad_lds16(xa + n * 8 * AD_ROW);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint4 lo = ad_lds16(aa + m * 16 * AD_ROW), hi = ad_lds16(aa + (m * 16 + 8) * AD_ROW);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                ad_mma<T>(acc[m][n], lo.x, hi.x, lo.y, hi.y, x[n].x, x[n].y);
                ad_mma<T>(acc[m][n], lo.z, hi.z, lo.w, hi.w, x[n].z, x[n].w);
            }
        }
        if (CHAIN && ((chain += 2) == CHAIN || st + 1 == n_st)) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) { sum[m][n][e] += acc[m][n][e]; acc[m][n][e] = 0.f; }
            chain = 0;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                     // the warps' sums lie where the ring was
    ad_put_sums<MT, NT>(CHAIN ? sum : acc, out, L.rp, m0);
}

// two 16-bit values to f32
__device__ __forceinline__ float2 ad_unpack(uint32_t v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
__device__ __forceinline__ float2 ad_unpack(uint32_t v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ uint32_t ad_pack(float x, float y, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t ad_pack(float x, float y, __half) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Up to MT x 16 tokens times the outputs of blocks of 32 from fb on, every eighth block.  Column c of product j stands for output
// (c / 2) 8 + 2 j + c % 2 of the block, so that a lane ends up with eight consecutive outputs of a token.  The next 32 rank columns of B are
// asked for before a product, 16-bit bases a block ahead.  The parts' rows behind the last token hold anything, those of rank columns behind
// the last hold zeros.
// ROUNDED: 32 rank columns are summed by themselves, the small parts first, and added with rounding.
template <class T, class O, int MT, bool ROUNDED>
__device__ __forceinline__ void ad_outer(const AdaptersArgs& a, const T* B, uint32_t R, uint32_t fb, uint32_t fb_end, const uint32_t* rows, uint32_t n_rows,
                                         uint32_t t0, uint32_t u, uint32_t u_part, uint32_t pitch, const float* row_scale) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    constexpr int V = sizeof(O) / 2;                      // 16-byte words of eight outputs
    constexpr bool AHEAD = sizeof(O) == 2;
    if (fb >= fb_end) return;
    O* y[MT][2];
    const O* base[MT][2];
    float scale[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t i = m * 16 + h * 8 + g;
            y[m][h] = nullptr; base[m][h] = nullptr; scale[m][h] = 1.f;
            if (i < n_rows) {
                const size_t row = t0 + rows[i];
                y[m][h] = static_cast<O*>(a.y) + row * a.ld_y + t * 8;
                if (a.base) base[m][h] = static_cast<const O*>(a.base) + row * a.ld_base + t * 8;
                if (std::is_same<T, __half>::value) scale[m][h] = row_scale[i];
            }
        }
    const uint32_t u0 = u + g * pitch + t * 16, k_end = (R + 31) / 32 * 32;
    uint4 bv[2][4], bs[MT][2][V];
    auto ask = [&](uint4 (&b)[4], uint32_t block, uint32_t k) {
        // outputs behind the last read the last one's row (their products go nowhere), rank columns behind the last are zeros
        const int left = (int)R - (int)(k + t * 8);
        const bool in = block < fb_end && left > 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t o = block * 32 + (g >> 1) * 8 + 2 * j + (g & 1u);
            b[j] = in ? ad_ld16(B + (size_t)(o < a.N ? o : a.N - 1) * a.R + k + t * 8) : zero;
        }
        if (in && left < 8)
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = ad_first(b[j], left);
    };
    auto ask_base = [&](uint4 (&to)[MT][2][V], uint32_t block) {
        const bool in = block < fb_end && block * 32 + t * 8 < a.N;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int v = 0; v < V; ++v)    // plain loads: in place, y's own rows are read here
                    to[m][h][v] = in && base[m][h] ? *reinterpret_cast<const uint4*>(base[m][h] + block * 32 + v * (8 / V)) : zero;
    };
    ask(bv[0], fb, 0);
    if (AHEAD) ask_base(bs, fb);
#pragma unroll 1
    for (; fb < fb_end; fb += AD_WARPS) {
        float acc[MT][4][4] = {};
        auto multiply = [&](const uint4 (&b)[4], uint32_t k) {
            constexpr int NP = AD_PARTS<T, O>;
            if constexpr (ROUNDED) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    uint4 lo[NP], hi[NP];
#pragma unroll
                    for (int part = 0; part < NP; ++part) {
                        const uint32_t at = u0 + part * u_part + m * 16 * pitch + k * 2;
                        lo[part] = ad_lds16(at); hi[part] = ad_lds16(at + 8 * pitch);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float s[4] = {};
#pragma unroll
                        for (int part = NP - 1; part >= 0; --part) {
                            ad_mma<T>(s, lo[part].x, hi[part].x, lo[part].y, hi[part].y, b[j].x, b[j].y);
                            ad_mma<T>(s, lo[part].z, hi[part].z, lo[part].w, hi[part].w, b[j].z, b[j].w);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[m][j][e] += s[e];
                    }
                }
                return;
            }
#pragma unroll
            for (int part = 0; part < NP; ++part)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint32_t at = u0 + part * u_part + m * 16 * pitch + k * 2;
                    const uint4 lo = ad_lds16(at), hi = ad_lds16(at + 8 * pitch);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        ad_mma<T>(acc[m][j], lo.x, hi.x, lo.y, hi.y, b[j].x, b[j].y);
                        ad_mma<T>(acc[m][j], lo.z, hi.z, lo.w, hi.w, b[j].z, b[j].w);
                    }
                }
        };
        if (!AHEAD) ask_base(bs, fb);
#pragma unroll 1
        for (uint32_t k = 0; k < k_end; k += 64) {
            const bool more = k + 32 < k_end;
            ask(bv[1], more ? fb : fb + AD_WARPS, more ? k + 32 : 0);
            multiply(bv[0], k);
            if (more) {
                const bool last = k + 64 >= k_end;
                ask(bv[0], last ? fb + AD_WARPS : fb, last ? 0 : k + 64);
                multiply(bv[1], k + 32);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) bv[0][j] = bv[1][j];
            }
        }
        if (fb * 32 + t * 8 < a.N) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!y[m][h]) continue;
                    const float s = scale[m][h];
                    if constexpr (sizeof(O) == 4) {
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            const uint4 b = bs[m][h][v];
                            *reinterpret_cast<float4*>(y[m][h] + fb * 32 + v * 4) =
                                make_float4(fmaf(acc[m][2 * v][2 * h], s, __uint_as_float(b.x)), fmaf(acc[m][2 * v][2 * h + 1], s, __uint_as_float(b.y)),
                                            fmaf(acc[m][2 * v + 1][2 * h], s, __uint_as_float(b.z)), fmaf(acc[m][2 * v + 1][2 * h + 1], s, __uint_as_float(b.w)));
                        }
                    } else {
                        const uint32_t b[4] = {bs[m][h][0].x, bs[m][h][0].y, bs[m][h][0].z, bs[m][h][0].w};
                        uint32_t o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 f = ad_unpack(b[j], O());
                            o[j] = ad_pack(fmaf(acc[m][j][2 * h], s, f.x), fmaf(acc[m][j][2 * h + 1], s, f.y), O());
                        }
                        *reinterpret_cast<uint4*>(y[m][h] + fb * 32) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                }
        }
        if (AHEAD) ask_base(bs, fb + AD_WARPS);
    }
}

struct AdShared {
    __align__(16) int32_t id[AD_TT];
    int32_t adapter[AD_TT];
    uint32_t rows[AD_TT], bare[AD_TT], n[4];                        // n: distinct adapters, rows of this one, bare rows, distinct of the first 32 tokens
    float scale[AD_TT];
};

// y = base for n tokens without an adapter: this CTA's outputs, a warp to a row
template <class O, class Row>
__device__ __forceinline__ void ad_copy(const AdaptersArgs& a, const Row* rows, uint32_t n_rows, uint32_t t0, uint32_t C, uint32_t rank) {
    if (a.base == a.y) return;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    constexpr uint32_t VEC = 16 / sizeof(O);
    const uint32_t c0 = (uint32_t)((uint64_t)rank * (a.N / 8) / C) * (8 / VEC), c1 = (uint32_t)((uint64_t)(rank + 1) * (a.N / 8) / C) * (8 / VEC);   // 16-byte words
    for (uint32_t i = warp; i < n_rows; i += AD_WARPS) {
        const size_t row = t0 + rows[i];
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const O*>(a.base) + row * a.ld_base);
        uint4* to = reinterpret_cast<uint4*>(static_cast<O*>(a.y) + row * a.ld_y);
        for (uint32_t c = c0 + lane; c < c1; c += 128) {
            uint4 w[4] = {};
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (a.base && c + k * 32 < c1) w[k] = from[c + k * 32];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (c + k * 32 < c1) to[c + k * 32] = w[k];
        }
    }
}

// where the 16-bit parts of rank columns r, r + 1 (r even) of a token go
struct AdParts {                         // rows of `pitch` bytes
    uint32_t u, u_part, pitch;
    __device__ uint32_t at(uint32_t p, uint32_t i, uint32_t r) const { return u + p * u_part + i * pitch + r * 2; }
};
// The CTAs' sums in order (part: f32 [tokens][r16], in every CTA at the same place), a warp to a token; the parts, and a power of two that the outputs
// are multiplied by, go to every CTA.  Eight warps.
// NJ: 64 rank columns at most, NI: tokens of a warp whose reads are under way together.
template <class T, int NP, int NJ, int NI, class Parts>
__device__ __forceinline__ void ad_fold(const AdaptersArgs& a, uint32_t C, uint32_t rank, int32_t id, uint32_t R, uint32_t n_rows, uint32_t warp,
                                        uint32_t part, uint32_t r16, uint32_t scales, const Parts& parts) {
    const uint32_t lane = threadIdx.x & 31u, step = C * AD_WARPS;
    const float scale = a.scales ? a.scales[id] : 1.f;
    for (uint32_t i0 = rank + C * warp; i0 < n_rows; i0 += NI * step) {
        float v[NI][NJ][2] = {};
        for (uint32_t c = 0; c < C; ++c) {
            float2 p[NI][NJ];
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const uint32_t r = j * 64 + lane * 2, i = i0 + n * step;
                    p[n][j] = make_float2(0.f, 0.f);
                    if (r < R && i < n_rows) p[n][j] = ad_ld_cluster2(map_to_rank(part + (i * r16 + r) * 4, c));
                }
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int j = 0; j < NJ; ++j) { v[n][j][0] += p[n][j].x; v[n][j][1] += p[n][j].y; }
        }
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const uint32_t i = i0 + n * step;
            if (i >= n_rows) break;
            float most = 0.f, down = 1.f, up = 1.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t r = j * 64 + lane * 2;
                v[n][j][0] = r < R ? v[n][j][0] * scale : 0.f;       // zeros behind the rank whatever the scale
                v[n][j][1] = r + 1 < R ? v[n][j][1] * scale : 0.f;
                most = fmaxf(most, fmaxf(fabsf(v[n][j][0]), fabsf(v[n][j][1])));
            }
            if (std::is_same<T, __half>::value) {
                for (uint32_t o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
                // a power of two next to the row's largest: the parts lie in (-2, 2); rows of zeros, and of infinities, as they are
                const uint32_t e = __float_as_uint(most) & 0x7F800000u;
                if (e >= 0x00800000u && e <= 0x7E800000u) { up = __uint_as_float(e); down = __uint_as_float(0x7F000000u - e); }
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t r = j * 64 + lane * 2;
                if (r >= (R + 31) / 32 * 32) continue;               // zeros behind the last rank column
                uint32_t split[NP];
                ad_split<T, NP>(v[n][j][0] * down, v[n][j][1] * down, split);
                for (uint32_t c = 0; c < C; ++c)
#pragma unroll
                    for (int p = 0; p < NP; ++p) ad_st_cluster(map_to_rank(parts.at(p, i, r), c), split[p]);
            }
            if (std::is_same<T, __half>::value && lane < C) ad_st_cluster(map_to_rank(scales + i * 4, lane), __float_as_uint(up));
        }
    }
}

// One adapter's n_rows <= 16 n_q tokens t0 + sh.rows[..], by the whole cluster, n_q = 1, 2 or 4.
template <class T, class O, AdSums SUMS>
__device__ __forceinline__ void ad_unit(const AdaptersArgs& a, const AdSmem& L, uint8_t* smem, AdShared& sh, uint32_t C, uint32_t rank, int32_t id,
                                        uint32_t n_rows, uint32_t n_q, uint32_t t0) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, base_s = smem_u32(smem);
    float* const warp_part = reinterpret_cast<float*>(smem);
    float* const part = reinterpret_cast<float*>(smem + L.part);
    const uint32_t n_kb = (a.K + 31) / 32, kb0 = (uint32_t)((uint64_t)rank * n_kb / C), kb1 = (uint32_t)((uint64_t)(rank + 1) * n_kb / C);
    const uint32_t n_fb = (a.N + 31) / 32, fb0 = (uint32_t)((uint64_t)rank * n_fb / C), fb1 = (uint32_t)((uint64_t)(rank + 1) * n_fb / C);
    const int32_t given = a.ranks ? a.ranks[id] : (int32_t)a.R;
    const uint32_t R = given < 0 ? 0u : min((uint32_t)given, a.R);
    const T* A = static_cast<const T*>(a.a) + (size_t)id * a.a_stride;
    const T* B = static_cast<const T*>(a.b) + (size_t)id * a.b_stride;

    // ---- inner product: this CTA's inputs ----
    constexpr uint32_t CHAIN = ad_chain<O, SUMS>;
    for (uint32_t r0 = 0; r0 < R; r0 += AD_MR) {
        const uint32_t rr = min(R - r0, AD_MR);                      // rank rows of the pass
        uint32_t n_sums;                                             // partial sums of a value, one after the other n_next floats apart
        const uint32_t region = 16 * (L.rp + 4);                     // floats of a warp's sums
        if (n_q == 1) {
            float* const mine = warp_part + warp * region;
            n_sums = AD_WARPS;
            if (n_rows <= 8) {
                if (rr <= 16) ad_inner<T, 1, 1, CHAIN>(a, A, R, r0, sh.rows, n_rows, t0, kb0 + warp, kb1, AD_WARPS, mine, L.rp);
                else if (rr <= 32) ad_inner<T, 2, 1, CHAIN>(a, A, R, r0, sh.rows, n_rows, t0, kb0 + warp, kb1, AD_WARPS, mine, L.rp);
                else ad_inner<T, 4, 1, CHAIN>(a, A, R, r0, sh.rows, n_rows, t0, kb0 + warp, kb1, AD_WARPS, mine, L.rp);
            } else {
                if (rr <= 16) ad_inner<T, 1, 2, CHAIN>(a, A, R, r0, sh.rows, n_rows, t0, kb0 + warp, kb1, AD_WARPS, mine, L.rp);
                else if (rr <= 32) ad_inner<T, 2, 2, CHAIN>(a, A, R, r0, sh.rows, n_rows, t0, kb0 + warp, kb1, AD_WARPS, mine, L.rp);
                else ad_inner<T, 4, 2, CHAIN>(a, A, R, r0, sh.rows, n_rows, t0, kb0 + warp, kb1, AD_WARPS, mine, L.rp);
            }
        } else {
            // warp = (tokens, inputs, m-tiles): 4 x 2 x 1, or 2 x 2 x 2 (where there is one m-tile, both halves take it)
            const uint32_t q = n_q == 4 ? warp >> 1 : warp >> 2, kq = warp & 1u, mh = warp >> 1 & 1u, k_end = min(kb1 * 32, a.K);
            float* const mine = warp_part + (q * 2 + kq) * region;
            n_sums = 2;
            if (n_q == 4) {
                if (L.rp == 16) ad_inner_ring<T, 1, 2, CHAIN>(a, L, A, r0, rr, sh.rows, n_rows, t0, kb0 * 32, k_end, base_s, q * 16, kq, 0, mine);
                else if (L.rp == 32) ad_inner_ring<T, 2, 2, CHAIN>(a, L, A, r0, rr, sh.rows, n_rows, t0, kb0 * 32, k_end, base_s, q * 16, kq, 0, mine);
                else ad_inner_ring<T, 4, 2, CHAIN>(a, L, A, r0, rr, sh.rows, n_rows, t0, kb0 * 32, k_end, base_s, q * 16, kq, 0, mine);
            } else {
                if (L.rp <= 32) ad_inner_ring<T, 1, 2, CHAIN>(a, L, A, r0, rr, sh.rows, n_rows, t0, kb0 * 32, k_end, base_s, q * 16, kq, L.rp == 16 ? 0 : mh, mine);
                else ad_inner_ring<T, 2, 2, CHAIN>(a, L, A, r0, rr, sh.rows, n_rows, t0, kb0 * 32, k_end, base_s, q * 16, kq, mh * 2, mine);
            }
        }
        __syncthreads();
        // the warps' sums in order, a warp to a token
        for (uint32_t c = warp; c < n_rows; c += AD_WARPS) {
            const float* p = warp_part + c / 16 * n_sums * region + c % 16 * (L.rp + 4);
            for (uint32_t r = lane; r < rr; r += 32) {
                float s = p[r];
                for (uint32_t w = 1; w < n_sums; ++w) s += p[w * region + r];
                part[c * L.r16 + r0 + r] = s;
            }
        }
        __syncthreads();
    }
    cluster_sync_all();
    const AdParts parts{base_s + L.u, L.u_part, L.pitch};
    ad_fold<T, AD_PARTS<T, O>, 4, 1>(a, C, rank, id, R, n_rows, warp, base_s + L.part, L.r16, smem_u32(sh.scale), parts);
    cluster_sync_all();
    // ---- outer product: this CTA's outputs ----
    constexpr bool ROUNDED = SUMS == AD_ROUNDED;
    if (n_rows <= 16)
        ad_outer<T, O, 1, ROUNDED>(a, B, R, fb0 + warp, fb1, sh.rows, n_rows, t0, base_s + L.u, L.u_part, L.pitch, sh.scale);
    else
        for (uint32_t h = 0; h < n_rows; h += 32)
            if (n_rows - h <= 16)
                ad_outer<T, O, 1, ROUNDED>(a, B, R, fb0 + warp, fb1, sh.rows + h, n_rows - h, t0, base_s + L.u + h * L.pitch, L.u_part, L.pitch, sh.scale + h);
            else
                ad_outer<T, O, 2, ROUNDED>(a, B, R, fb0 + warp, fb1, sh.rows + h, min(n_rows - h, 32u), t0, base_s + L.u + h * L.pitch, L.u_part, L.pitch,
                                           sh.scale + h);
    __syncthreads();
}

// an id's place: its adapter, or n_adapters for none
__device__ __forceinline__ uint32_t ad_place(const AdaptersArgs& a, uint32_t t, bool report) {
    const int32_t id = a.ids[t];
    if (id >= 0 && (uint32_t)id >= a.n_adapters && report) atomicMax(a.status, ST_BAD_ADAPTER);
    return id < 0 || (uint32_t)id >= a.n_adapters ? a.n_adapters : (uint32_t)id;
}

// Up to 64 tokens, or more adapters than the sorting form counts: tile by tile
template <class T, class O, AdSums SUMS>
__global__ void __launch_bounds__(AD_WARPS * 32, 2) adapters_tile_kernel(const AdaptersArgs a, const uint32_t C, const uint32_t slots) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ AdShared sh;
    const AdSmem L = ad_smem(a.R, a.T, AD_PARTS<T, O>);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = cluster_rank();
    const uint32_t unit = blockIdx.x / C, tile = unit / slots, slot = unit % slots, t0 = tile * AD_TT;

    grid_dep_wait();
    grid_dep_launch();
    // the tile's ids and its distinct adapters, in order of their first token
    if (warp < 2) {
        const uint32_t place = t0 + tid < a.T ? ad_place(a, t0 + tid, slot == 0 && rank == 0) : a.n_adapters;
        sh.id[tid] = place == a.n_adapters ? -1 : (int32_t)place;
    }
    __syncthreads();
    if (warp < 2) {
        const int32_t id = sh.id[tid];
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, id);
        bool first = id >= 0 && (same & ((1u << lane) - 1)) == 0;
        if (warp == 1)
            for (uint32_t j = 0; j < 32; j += 4) {
                const int4 v = *reinterpret_cast<const int4*>(sh.id + j);
                first = first && v.x != id && v.y != id && v.z != id && v.w != id;
            }
        const uint32_t firsts = __ballot_sync(0xFFFFFFFFu, first), before = __popc(firsts & ((1u << lane) - 1));
        if (warp == 0) {
            if (first) sh.adapter[before] = id;
            if (lane == 0) sh.n[3] = __popc(firsts);
        }
        asm volatile("bar.sync 1, 64;" ::: "memory");
        if (warp == 1) {
            if (first) sh.adapter[sh.n[3] + before] = id;
            if (lane == 0) sh.n[0] = sh.n[3] + __popc(firsts);
        }
    } else if (warp == 2) {
        uint32_t n = 0;
        for (uint32_t h = 0; h < 2; ++h) {
            const bool bare = sh.id[h * 32 + lane] < 0 && t0 + h * 32 + lane < a.T;
            const uint32_t m = __ballot_sync(0xFFFFFFFFu, bare);
            if (bare) sh.bare[n + __popc(m & ((1u << lane) - 1))] = h * 32 + lane;
            n += __popc(m);
        }
        if (lane == 0) sh.n[2] = n;
    }
    __syncthreads();
    const uint32_t n_adapters = sh.n[0];
    if (slot == 0) ad_copy<O>(a, sh.bare, sh.n[2], t0, C, rank);
    for (uint32_t d = slot; d < n_adapters; d += slots) {
        const int32_t id = sh.adapter[d];
        if (warp == 0) {
            uint32_t n = 0;
            for (uint32_t h = 0; h < 2; ++h) {
                const bool mine = sh.id[h * 32 + lane] == id;
                const uint32_t m = __ballot_sync(0xFFFFFFFFu, mine);
                if (mine) sh.rows[n + __popc(m & ((1u << lane) - 1))] = h * 32 + lane;
                n += __popc(m);
            }
            if (lane == 0) sh.n[1] = n;
        }
        __syncthreads();
        ad_unit<T, O, SUMS>(a, L, smem, sh, C, rank, id, sh.n[1], sh.n[1] <= 16 ? 1 : sh.n[1] <= 32 ? 2 : 4, t0);
    }
}

// More tokens: every CTA sorts the ids of a segment of up to 2048 tokens in its own shared memory (stable, so that all CTAs have the same order),
// then the segment's clusters take units of one adapter and up to 64 of its tokens, wherever they lie.
constexpr uint32_t AD_SEG = 2048, AD_FEW = 512, AD_MANY = 2048;      // tokens of a segment; adapters that are counted, and none
template <uint32_t PLACES>
struct AdSort {                          // dynamic shared memory behind AdSmem
    uint32_t first[PLACES + 1];          // first token in the order (low half), first unit (high half)
    uint16_t cursor[AD_WARPS][PLACES];
    uint16_t order[AD_SEG];
};
// the lanes that hold the same place, by one ballot per bit of the largest (a match of whole words took 700 cycles)
__device__ __forceinline__ uint32_t ad_same(uint32_t place, uint32_t bits, bool in) {
    uint32_t same = __ballot_sync(0xFFFFFFFFu, in);
    for (uint32_t b = 0; b < bits; ++b) {
        const bool one = place >> b & 1u;
        const uint32_t m = __ballot_sync(0xFFFFFFFFu, one);
        same &= one ? m : ~m;
    }
    return same;
}
// `scratch`: 2 x AD_SEG x 2 bytes, free again afterwards.  All threads of the CTA (AD_WARPS warps or more; the first AD_WARPS work).
template <uint32_t PLACES>
__device__ __forceinline__ void ad_sort(const AdaptersArgs& a, AdSort<PLACES>& so, uint16_t* scratch, uint32_t* s_scan, uint32_t t0, uint32_t n_tok, uint32_t tt, bool report) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    // a warp counts the places of its run of tokens, then the runs of a place follow one another
    const uint32_t run_len = (n_tok + AD_WARPS * 32 - 1) / (AD_WARPS * 32) * 32, run0 = warp < AD_WARPS ? warp * run_len : n_tok, run1 = min(run0 + run_len, n_tok);
    for (uint32_t i = tid; i < AD_WARPS * PLACES / 2; i += blockDim.x) reinterpret_cast<uint32_t*>(so.cursor)[i] = 0;
    __syncthreads();
    // a token's place, and its number among the run's tokens of that place
    uint16_t* const place_of = scratch;
    uint16_t* const number_of = place_of + AD_SEG;
    const uint32_t bits = 32 - __clz(a.n_adapters);
#pragma unroll 4
    for (uint32_t i = run0 + lane; i < run1; i += 32) place_of[i] = (uint16_t)ad_place(a, t0 + i, report);
    __syncwarp();
#pragma unroll 1
    for (uint32_t i = run0 + lane; i < run0 + run_len && i - lane < run1; i += 32) {
        const bool in = i < run1;
        const uint32_t place = in ? place_of[i] : 0u, same = ad_same(place, bits, in), before = __popc(same & ((1u << lane) - 1));
        const uint32_t at = in ? so.cursor[warp][place] : 0;
        __syncwarp();
        if (in) number_of[i] = (uint16_t)(at + before);
        if (in && before == 0) so.cursor[warp][place] = (uint16_t)(at + __popc(same));
        __syncwarp();
    }
    __syncthreads();
    // a run of places to a thread: counts and units (up to tt tokens) summed side by side
    constexpr uint32_t MINE = PLACES / (AD_WARPS * 32);
    uint32_t v[MINE] = {}, sum = 0, run = 0;
    if (warp < AD_WARPS) {
#pragma unroll
        for (uint32_t j = 0; j < MINE; ++j) {
            const uint32_t p = tid * MINE + j;
            uint32_t n = 0;
            for (uint32_t w = 0; w < AD_WARPS; ++w) n += so.cursor[w][p];
            v[j] = n | ((n + tt - 1) / tt) << 16;
            sum += v[j];
        }
        run = sum;
        for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t w = __shfl_up_sync(0xFFFFFFFFu, run, o); if (lane >= o) run += w; }
        if (lane == 31) s_scan[warp] = run;
    }
    __syncthreads();
    if (warp < AD_WARPS) {
        uint32_t at = run - sum;
        for (uint32_t w = 0; w < warp; ++w) at += s_scan[w];
#pragma unroll
        for (uint32_t j = 0; j < MINE; ++j) {
            const uint32_t p = tid * MINE + j;
            so.first[p] = at;
            uint32_t pos = at & 0xFFFFu;
            for (uint32_t w = 0; w < AD_WARPS; ++w) {
                const uint32_t n = so.cursor[w][p];
                so.cursor[w][p] = (uint16_t)pos;
                pos += n;
            }
            at += v[j];
            if (p == PLACES - 1) so.first[PLACES] = at;
        }
    }
    __syncthreads();
    for (uint32_t i = run0 + lane; i < run1; i += 32) so.order[so.cursor[warp][place_of[i]] + number_of[i]] = (uint16_t)i;
    __syncthreads();
}
// unit u of the sorted segment: its place (n_adapters: no adapter), its tokens so.order[at .. at + rows), and the most tokens that a unit of its place has
struct AdUnit { uint32_t place, at, rows, per; };
template <uint32_t PLACES>
__device__ __forceinline__ AdUnit ad_find(const AdSort<PLACES>& so, uint32_t n_places, uint32_t tt, uint32_t u) {
    uint32_t lo = 0, hi = n_places;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (so.first[mid] >> 16 <= u) lo = mid; else hi = mid;
    }
    const uint32_t at = so.first[lo] & 0xFFFFu, n = (so.first[lo + 1] & 0xFFFFu) - at, n_chunks = (n + tt - 1) / tt;
    AdUnit r;
    r.place = lo;
    r.per = (n + n_chunks - 1) / n_chunks;
    const uint32_t c0 = (u - (so.first[lo] >> 16)) * r.per;
    r.at = at + c0;
    r.rows = min(r.per, n - c0);
    return r;
}

template <class T, class O, AdSums SUMS, uint32_t PLACES>
__global__ void __launch_bounds__(AD_WARPS * 32, 2) adapters_sorted_kernel(const AdaptersArgs a, const uint32_t C, const uint32_t per_seg, const uint32_t seg_len, const uint32_t tt) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ AdShared sh;
    __shared__ uint32_t s_scan[AD_WARPS];
    const AdSmem L = ad_smem(a.R, a.T, AD_PARTS<T, O>);
    const uint32_t tid = threadIdx.x, rank = cluster_rank();
    const uint32_t cl = blockIdx.x / C, seg = cl / per_seg, t0 = seg * seg_len, n_tok = min(seg_len, a.T - t0), n_places = a.n_adapters + 1;
    AdSort<PLACES>& so = *reinterpret_cast<AdSort<PLACES>*>(smem + L.bytes);
    grid_dep_wait();
    grid_dep_launch();
    ad_sort(a, so, reinterpret_cast<uint16_t*>(smem), s_scan, t0, n_tok, tt, cl % per_seg == 0 && rank == 0);
    const uint32_t n_units = so.first[n_places] >> 16;
    for (uint32_t u = cl % per_seg; u < n_units; u += per_seg) {
        const AdUnit un = ad_find(so, n_places, tt, u);
        if (tid < un.rows) sh.rows[tid] = so.order[un.at + tid];
        __syncthreads();
        if (un.place == a.n_adapters) {
            ad_copy<O>(a, sh.rows, un.rows, t0, C, rank);
            __syncthreads();
        } else {
            ad_unit<T, O, SUMS>(a, L, smem, sh, C, rank, (int32_t)un.place, un.rows, un.per <= 16 ? 1 : un.per <= 32 ? 2 : 4, t0);   // one split for all units of an adapter
        }
    }
}

// ------------------------------------------------------------------------------------------------------------
// many tokens per adapter: the same cut, both products on the tensor cores
// ------------------------------------------------------------------------------------------------------------
// For units of 16 tokens and more mma.sync's operands, read from shared memory by every warp again, take longer than the bytes.  Here a
// unit's inner product is D1[rank 128][tokens 64] = A x^T and its outer product, per block of 128 outputs, D2[outputs 128][tokens 64] = B u^T (the parts of u, one after
// the other, into one accumulator): tcgen05.mma with M = 128, N = 64, accumulators in tensor memory.  A ring of stages: 64 inputs of A (a tensor-map copy)
// and of the unit's x rows (asynchronous copies, eight lanes to a row), later 64 rank columns of a block of B (asynchronous copies, which zero what lies behind
// the adapter's rank).  A warp to a ring slot, one that issues the products, eight that read accumulators: inner sums -> shared memory -> the cluster's fold ->
// parts of u as operand rows; outputs -> turned through shared memory -> + base -> y.  The fold's steps are joined by mbarriers between the CTAs, so the
// ring runs on underneath.  Every wait is bounded: a give-up sets the status word, and everybody still meets at the end.
// 8192 tokens of six adapters, rank 64, 4096 -> 2048, in cycles (with one buffer of accumulators; with two the call takes 1 us more): sort 8,500, start 3,500,
// inner 35,000 (the issuer: 400 for a stage's four small MMAs), fold 7,000, outer 40,000 (16 blocks of 128 outputs; each a chain of tensor-memory read, turn, base
// and store over eight warps): 56.5 us against 71 with mma.sync.  Measured and not kept: base through the ring (52 -> 51 us, rank 128 with f32 outputs 36 -> 51), prefetches of x and base into L2 (their issue
// takes what they save), 64-byte pieces of base one block further ahead.
// The accumulators truncate (see the grouped products).  The inner product's stages go in order to accumulators of a few stages each, three to a buffer of two;
// the epilogue warps add a buffer's, rounding, to sums in shared memory while the next one fills, so an inner product of any length has chains of
// ab_chain stages.  (Six accumulators that shared all of a CTA's stages: 8192 f16 tokens of six, rank 64, 5120 inputs, f32 outputs, 1.27e-6 off 64 bits; 9000
// of two, 65,536 inputs of one sign, 6.8e-5.)  Of u's parts the small ones are multiplied first, under the large one's truncations.
constexpr uint32_t AB_CHAINS = 3, AB_D2 = 2 * AB_CHAINS * 64;        // accumulators of 64 columns to a buffer, the outputs' first column
template <class T, class O>
constexpr uint32_t ab_chain = sizeof(O) == 2 ? 32 : std::is_same<T, __half>::value ? 4 : 8;   // stages: f16 products lose about twice as much
constexpr uint32_t AB_MOST_SLOTS = 9, AB_MAX_R = 128, AB_MIN_ROWS = 16;   // ranks to, tokens per unit from
constexpr uint32_t AB_LITTLE = 12000;                                // tokens x rank that mma.sync does sooner
constexpr uint32_t AB_U_BYTES = 64 * 128;                            // one part of 64 rank columns of the unit's tokens
constexpr uint32_t AB_TURN = 16 * 32 * 4;                            // an epilogue warp's turn of 16 tokens x 32 outputs
constexpr uint32_t AB_MOST_SMEM = 227 * 1024 - 512;                  // beside the barriers
struct AbSmem {
    uint32_t slots, slot, x;                                         // ring slots, their bytes, x rows behind R rows of A (the products read 128: what is there)
    uint32_t u, part, turn, sort, bytes;                             // behind the ring, offsets from its 1024-byte boundary
    __host__ __device__ uint32_t threads() const { return (1 + AD_WARPS + slots) * 32; }
};
__host__ __device__ inline AbSmem ab_smem(uint32_t R, uint32_t n_parts) {
    AbSmem s;
    const uint32_t u_bytes = (R + 63) / 64 * n_parts * AB_U_BYTES, part_bytes = (R + 15) / 16 * 16 * 64 * 4;
    const uint32_t rest = u_bytes + part_bytes + AD_WARPS * AB_TURN + (uint32_t)sizeof(AdSort<AD_FEW>) + 1024;
    s.x = R * 128;                                                   // a multiple of 1024
    s.slot = R <= 64 ? 128 * 128 : s.x + 64 * 128;                   // a block of 128 outputs' B fits too
    s.slots = R <= 64 ? AB_MOST_SLOTS : 5;
    if (s.slots * s.slot + rest > AB_MOST_SMEM) s.slots = 4;        // three parts at ranks above 120
    s.u = s.slots * s.slot;
    s.part = s.u + u_bytes;
    s.turn = s.part + part_bytes;
    s.sort = s.turn + AD_WARPS * AB_TURN;
    s.bytes = s.slots * s.slot + rest;
    return s;
}
// operand rows of 64 rank columns, 128 bytes, 16-byte chunks swizzled by the row: [64-column chunk][part][64 tokens]
template <int NP>
struct AbParts {
    uint32_t u;
    __device__ uint32_t at(uint32_t p, uint32_t i, uint32_t r) const {
        return u + ((r >> 6) * NP + p) * AB_U_BYTES + i * 128 + ((((r & 63u) >> 3) ^ (i & 7u)) << 4) + (r & 7u) * 2;
    }
};
struct AbParams {
    CUtensorMap a;                       // [n_adapters][R][K], boxes of R rows x 64 inputs
    AdaptersArgs p;
    uint32_t C, per_seg, seg_len;
};
__device__ __forceinline__ void ab_tma_3d(uint32_t dst, const CUtensorMap* map, int32_t c0, int32_t c1, int32_t c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(c0),
                 "r"(c1), "r"(c2), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void ab_expect(uint32_t bar, uint32_t bytes) {   // bytes to wait for, no arrival
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// The first n bytes of 16, zeros behind.  No clobber of memory: the compiler may load the next rows' numbers meanwhile (a load between every two
// copies made a stage's 16 copies 1600 cycles); the wait for the copies has one.
__device__ __forceinline__ void ab_copy(uint32_t dst, const void* src, uint32_t n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n));
}
template <class T, class O>
__global__ void __launch_bounds__((1 + AD_WARPS + AB_MOST_SLOTS) * 32, 1) adapters_tensor_kernel(const __grid_constant__ AbParams P) {
    extern __shared__ uint8_t smem_any[];
    __shared__ __align__(8) uint64_t full_bar[AB_MOST_SLOTS], empty_bar[AB_MOST_SLOTS], d1_full[2], d1_empty[2], d2_full[2], d2_empty[2], part_ready, u_ready, u_go;
    __shared__ uint32_t s_tmem, s_scan[AD_WARPS];
    __shared__ float s_scale[AD_TT];
    __shared__ volatile int s_abort;
    const AdaptersArgs& a = P.p;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = cluster_rank(), C = P.C;
    const uint32_t ring = (smem_u32(smem_any) + 1023u) & ~1023u;
    uint8_t* const ring_p = smem_any + (ring - smem_u32(smem_any));
    constexpr int NP = AD_PARTS<T, O>;
    const AbSmem L = ab_smem(a.R, NP);
    const uint32_t cl = blockIdx.x / C, seg = cl / P.per_seg, t0 = seg * P.seg_len, n_tok = min(P.seg_len, a.T - t0), n_places = a.n_adapters + 1;
    AdSort<AD_FEW>& so = *reinterpret_cast<AdSort<AD_FEW>*>(ring_p + L.sort);
    if (tid == 0) {
        for (uint32_t s = 0; s < L.slots; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&d1_full[b], 1); mbar_init(&d1_empty[b], AD_WARPS); mbar_init(&d2_full[b], 1); mbar_init(&d2_empty[b], AD_WARPS); }
        mbar_init(&part_ready, C); mbar_init(&u_ready, C); mbar_init(&u_go, 1);
        s_abort = 0;
        mbar_fence_init();
        tma_prefetch_map(&P.a);
    }
    grid_dep_wait();                                                  // before tensor memory is taken, see the grouped products
    grid_dep_launch();
    if (warp == AD_WARPS) tmem_alloc(&s_tmem, 512);                   // the issuer's warp
    ad_sort(a, so, reinterpret_cast<uint16_t*>(ring_p), s_scan, t0, n_tok, AD_TT, cl % P.per_seg == 0 && rank == 0);
    fence_async_smem();                                               // the sort's scratch was where copies land
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = s_tmem, n_units = so.first[n_places] >> 16;
    const uint32_t n_ks = (a.K + 63) / 64, ks0 = rank * n_ks / C, ks1 = (rank + 1) * n_ks / C;
    const uint32_t n_fb = (a.N + 127) / 128, fb0 = rank * n_fb / C, fb1 = (rank + 1) * n_fb / C;
    constexpr uint32_t CHAIN = ab_chain<T, O>, ROUND = AB_CHAINS * CHAIN;
    auto give_up = [&](uint32_t code) { if (!s_abort) atomicMax(a.status, code); s_abort = 1; };
    auto rank_of = [&](uint32_t place) {
        const int32_t given = a.ranks ? a.ranks[place] : (int32_t)a.R;
        return given < 0 ? 0u : min((uint32_t)given, a.R);
    };

    if (warp > AD_WARPS) {
        // ---------------- a ring slot's warp: every L.slots-th stage ----------------
        const uint32_t slot = warp - AD_WARPS - 1, full = smem_u32(&full_bar[slot]), empty = smem_u32(&empty_bar[slot]), at = ring + slot * L.slot;
        const uint32_t chunk = lane & 7u, row0 = lane >> 3;
        uint32_t ph = 0, base = 0, before = 0;                        // base: stages of the units before, modulo the ring
        bool ok = true;
        for (uint32_t u = cl % P.per_seg; u < n_units && ok; u += P.per_seg) {
            const AdUnit un = ad_find(so, n_places, AD_TT, u);
            if (un.place == a.n_adapters) continue;
            const uint32_t R = rank_of(un.place), chunks = (R + 63) / 64, n_in = R ? ks1 - ks0 : 0, n_st = n_in + (fb1 - fb0) * chunks;
            const T* const B = static_cast<const T*>(a.b) + (size_t)un.place * a.b_stride;
            const T* xr[AD_TT / 4];
#pragma unroll
            for (uint32_t i = 0; i < AD_TT / 4; ++i) xr[i] = static_cast<const T*>(a.x) + (size_t)(t0 + so.order[un.at + min(row0 + i * 4, un.rows - 1)]) * a.ld_x;
            for (uint32_t st = (slot + L.slots - base) % L.slots; st < n_st; st += L.slots) {
                if (!mbar_wait_warp_at(empty, ph ^ 1u, &s_abort, a.poll_limit)) { give_up(ST_WAIT_EMPTY); ok = false; break; }
                if (a.withhold && before + st + 1 == a.withhold) { ph ^= 1u; continue; }
                if (st < n_in) {
                    const uint32_t k = (ks0 + st) * 64;
                    if (lane == 0) {
                        ab_expect(full, a.R * 128);
                        ab_tma_3d(at, &P.a, (int32_t)k, 0, (int32_t)un.place, full);
                    }
                    const bool in = k + chunk * 8 < a.K;
                    const uint32_t from = in ? k + chunk * 8 : 0, n = in ? 16 : 0;
#pragma unroll
                    for (uint32_t i = 0; i < AD_TT / 4; ++i) {
                        const uint32_t r = row0 + i * 4;
                        if (r < un.rows) ab_copy(at + L.x + r * 128 + ((chunk ^ (r & 7u)) << 4), xr[i] + from, n);
                    }
                } else {
                    const uint32_t i = st - n_in, f0 = (fb0 + i / chunks) * 128, r = (i % chunks) * 64 + chunk * 8;
                    const uint32_t n = r >= R ? 0 : R - r < 8 ? (R - r) * 2 : 16;       // bytes of this lane's eight rank columns that count
                    const T* b = B + (n ? r : 0);
                    const uint32_t n_f = min(a.N - f0, 128u);
#pragma unroll 4
                    for (uint32_t f = row0; f < n_f; f += 4) ab_copy(at + f * 128 + ((chunk ^ (f & 7u)) << 4), b + (size_t)(f0 + f) * a.R, n);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_at(full);
                ph ^= 1u;
            }
            base = (base + n_st) % L.slots;
            before += n_st;
        }
    } else if (warp == AD_WARPS) {
        // ---------------- issuer ----------------
        const uint32_t fmt = std::is_same<T, __half>::value ? UMMA_F16 : UMMA_BF16, idesc = umma_idesc(fmt, 64);
        uint32_t s = 0, ph = 0, n_done = 0, n_rounds = 0, n_blocks = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t code) {
            if (!ok) return;
            ok = mbar_wait_warp_at(smem_u32(bar), parity, &s_abort, a.poll_limit);
            if (!ok) give_up(code);
            tc_fence_after();
        };
        auto next = [&]() { if (++s == L.slots) { s = 0; ph ^= 1u; } };
        for (uint32_t u = cl % P.per_seg; u < n_units && ok; u += P.per_seg) {
            const AdUnit un = ad_find(so, n_places, AD_TT, u);
            if (un.place == a.n_adapters) continue;
            const uint32_t R = rank_of(un.place), chunks = (R + 63) / 64;
            for (uint32_t k0 = ks0, chain = 0; k0 < ks1 && ok && R; k0 += CHAIN) {
                const uint32_t buf = n_rounds & 1u, k1 = min(k0 + CHAIN, ks1);
                if (chain == 0) wait(&d1_empty[buf], (n_rounds >> 1 & 1u) ^ 1u, ST_WAIT_EMPTY);
                const uint32_t d1 = __shfl_sync(0xFFFFFFFFu, tmem + (buf * AB_CHAINS + chain) * 64, 0);
                for (uint32_t ks = k0; ks < k1 && ok; ++ks) {
                    wait(&full_bar[s], ph, ST_WAIT_FULL);
                    if (!ok) break;
                    const uint32_t at = __shfl_sync(0xFFFFFFFFu, (ring + s * L.slot) >> 4, 0) | 1u << 16, x_at = at + (L.x >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) umma_f16_lo(d1, at + j * 2, x_at + j * 2, UMMA_SW128_HI, idesc, ks != k0 || j ? 1u : 0u);
                        umma_commit(&empty_bar[s]);
                    }
                    __syncwarp();
                    next();
                }
                if (!ok) break;
                if (++chain == AB_CHAINS || k1 == ks1) {
                    if (elect_one()) umma_commit(&d1_full[buf]);
                    __syncwarp();
                    chain = 0;
                    ++n_rounds;
                }
            }
            if (!ok) break;
            // the parts of u are there (a unit without a rank has none: its outputs are base)
            if (R) wait(&u_go, n_done & 1u, ST_WAIT_FULL);
            for (uint32_t fb = fb0; fb < fb1 && ok && R; ++fb, ++n_blocks) {
                const uint32_t buf = n_blocks & 1u, acc = tmem + AB_D2 + buf * 64;
                wait(&d2_empty[buf], (n_blocks >> 1 & 1u) ^ 1u, ST_WAIT_EMPTY);
                uint32_t first = 0, first_b = 0;                       // of two chunks the first one's slot, whose large part comes last
                const uint32_t u_at = __shfl_sync(0xFFFFFFFFu, (ring + L.u) >> 4, 0) | 1u << 16;
                const auto multiply = [&](uint32_t at, uint32_t c, uint32_t part) {
                    const uint32_t ua = u_at + (c * NP + part) * (AB_U_BYTES >> 4), steps = (min(R - c * 64, 64u) + 15) / 16;
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        if (j < steps) umma_f16_lo(acc, at + j * 2, ua + j * 2, UMMA_SW128_HI, idesc, c || part + 1 < NP || j ? 1u : 0u);
                };
                for (uint32_t c = 0; c < chunks && ok; ++c) {
                    wait(&full_bar[s], ph, ST_WAIT_FULL);
                    if (!ok) break;
                    const uint32_t at = __shfl_sync(0xFFFFFFFFu, (ring + s * L.slot) >> 4, 0) | 1u << 16;
                    const bool last = c + 1 == chunks;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t part = NP - 1; part; --part) multiply(at, c, part);
                        if (last) {
                            multiply(at, c, 0);
                            umma_commit(&empty_bar[s]);
                            if (c) { multiply(first_b, 0, 0); umma_commit(&empty_bar[first]); }
                        }
                    }
                    __syncwarp();
                    first = s; first_b = at;
                    next();
                }
                if (!ok) break;
                if (elect_one()) umma_commit(&d2_full[buf]);
                __syncwarp();
            }
            if (R) ++n_done;
        }
    } else {
        // ---------------- accumulators: warp = (lanes 32 q .. 32 q + 31, tokens 32 half .. 32 half + 31) ----------------
        const uint32_t q = warp & 3u, half = warp >> 2, etid = tid;   // warps 0 .. 7
        float* const part = reinterpret_cast<float*>(ring_p + L.part);
        const uint32_t r16 = (a.R + 15) / 16 * 16, turn = ring + L.turn + warp * AB_TURN;
        const AbParts<NP> parts{ring + L.u};
        uint32_t n_done = 0, n_rounds = 0, n_blocks = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(smem_u32(bar), parity, &s_abort, a.poll_limit));
            if (!ok) give_up(ST_WAIT_FULL);
            return ok;
        };
        // all eight warps go on, or give up, together: they meet at named barriers
        auto together = [&]() {
            uint32_t r;
            asm volatile("{\n\t.reg .pred p, r;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred r, 1, 256, p;\n\tselp.u32 %0, 1, 0, r;\n\t}" : "=r"(r) : "r"((uint32_t)ok) : "memory");
            ok = r != 0;
            return ok;
        };
        for (uint32_t u = cl % P.per_seg; u < n_units && ok; u += P.per_seg) {
            const AdUnit un = ad_find(so, n_places, AD_TT, u);
            if (un.place == a.n_adapters) { ad_copy<O>(a, so.order + un.at, un.rows, t0, C, rank); continue; }
            const uint32_t R = rank_of(un.place);
            if (!R) {   // outputs are base
                ad_copy<O>(a, so.order + un.at, un.rows, t0, C, rank);
                continue;
            }
            // inner sums of this CTA's inputs, a buffer of accumulators at a time
            for (uint32_t k0 = ks0; k0 < ks1; k0 += ROUND, ++n_rounds) {
                const uint32_t buf = n_rounds & 1u, n_chains = (min(ROUND, ks1 - k0) + CHAIN - 1) / CHAIN;
                if (!wait(&d1_full[buf], n_rounds >> 1 & 1u)) break;
                tc_fence_after();
                if (q * 32 < R)
                    for (uint32_t c = half * 32; c < half * 32 + 32 && c < un.rows; c += 16) {
                        float sum[16];
                        const bool mine = q * 32 + lane < r16;
                        float* const o = part + c * r16 + q * 32 + lane;
                        if (k0 != ks0 && mine)                       // all on their way before the accumulators are read
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) sum[j] = o[j * r16];
                        for (uint32_t chain = 0; chain < n_chains; ++chain) {
                            uint32_t v[16];
                            tmem_ld16(tmem + (buf * AB_CHAINS + chain) * 64 + c + ((q * 32u) << 16), v);
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) sum[j] = chain || k0 != ks0 ? sum[j] + __uint_as_float(v[j]) : __uint_as_float(v[j]);
                        }
                        if (mine)
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) o[j * r16] = sum[j];
                    }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d1_empty[buf]);
            }
            if (!together()) break;
            if (etid < C) mbar_arrive_cluster(map_to_rank(smem_u32(&part_ready), etid));
            wait(&part_ready, n_done & 1u);
            if (!together()) break;
            ad_fold<T, NP, AB_MAX_R / 64, 4>(a, C, rank, (int32_t)un.place, R, un.rows, warp, ring + L.part, r16, smem_u32(s_scale), parts);
            together();
            if (etid < C) mbar_arrive_cluster(map_to_rank(smem_u32(&u_ready), etid));
            wait(&u_ready, n_done & 1u);
            fence_async_smem();
            if (!together()) break;
            if (etid == 0) mbar_arrive(&u_go);
            ++n_done;
            // outputs: a lane eight of a token, four lanes a token's 32, a warp eight tokens at a time
            constexpr int V = sizeof(O) / 2;                          // 16-byte words of eight outputs
            const uint32_t i0 = half * 32 + (lane >> 2), f8 = q * 32 + (lane & 3u) * 8;
            uint32_t rows[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) rows[k] = t0 + so.order[un.at + min(i0 + k * 8, un.rows - 1)];
            uint4 b[4][V];
            auto ask_base = [&](uint32_t fb) {
                const uint32_t f = fb * 128 + f8;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        b[k][v] = make_uint4(0, 0, 0, 0);
                        if (a.base && fb < fb1 && f < a.N && i0 + k * 8 < un.rows)
                            b[k][v] = *reinterpret_cast<const uint4*>(static_cast<const O*>(a.base) + (size_t)rows[k] * a.ld_base + f + v * (8 / V));
                    }
            };
            ask_base(fb0);
            for (uint32_t fb = fb0; fb < fb1 && ok; ++fb, ++n_blocks) {
                const uint32_t buf = n_blocks & 1u, f = fb * 128 + f8;
                const bool in = f < a.N;
                if (!wait(&d2_full[buf], n_blocks >> 1 & 1u)) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    if (half * 32 + h * 16 >= un.rows) break;
                    uint32_t v[16];
                    tmem_ld16(tmem + AB_D2 + buf * 64 + half * 32 + h * 16 + ((q * 32u) << 16), v);
                    __syncwarp();
#pragma unroll
                    for (uint32_t j = 0; j < 16; ++j) asm volatile("st.shared.u32 [%0], %1;" ::"r"(turn + (j * 32 + lane) * 4), "r"(v[j]) : "memory");
                    __syncwarp();
                    uint4 turned[2][2];                  // all read before the first is used
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) turned[j][k] = ad_lds16(turn + ((lane >> 2) + j * 8) * 128 + (lane & 3u) * 32 + k * 16);
#pragma unroll
                    for (uint32_t j = 0; j < 2; ++j) {
                        const uint32_t i = i0 + h * 16 + j * 8;
                        if (!in || i >= un.rows) continue;
                        const float s = std::is_same<T, __half>::value ? s_scale[i] : 1.f;
                        const uint4 w0 = turned[j][0], w1 = turned[j][1];
                        uint4* y = reinterpret_cast<uint4*>(static_cast<O*>(a.y) + (size_t)rows[h * 2 + j] * a.ld_y + f);
                        if constexpr (sizeof(O) == 4) {
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint4 w = k ? w1 : w0, c = b[h * 2 + j][k];
                                y[k] = make_uint4(__float_as_uint(fmaf(__uint_as_float(w.x), s, __uint_as_float(c.x))), __float_as_uint(fmaf(__uint_as_float(w.y), s, __uint_as_float(c.y))),
                                                  __float_as_uint(fmaf(__uint_as_float(w.z), s, __uint_as_float(c.z))), __float_as_uint(fmaf(__uint_as_float(w.w), s, __uint_as_float(c.w))));
                            }
                        } else {
                            const uint4 c = b[h * 2 + j][0];
                            const float2 c0 = ad_unpack(c.x, O()), c1 = ad_unpack(c.y, O()), c2 = ad_unpack(c.z, O()), c3 = ad_unpack(c.w, O());
                            *y = make_uint4(ad_pack(fmaf(__uint_as_float(w0.x), s, c0.x), fmaf(__uint_as_float(w0.y), s, c0.y), O()),
                                            ad_pack(fmaf(__uint_as_float(w0.z), s, c1.x), fmaf(__uint_as_float(w0.w), s, c1.y), O()),
                                            ad_pack(fmaf(__uint_as_float(w1.x), s, c2.x), fmaf(__uint_as_float(w1.y), s, c2.y), O()),
                                            ad_pack(fmaf(__uint_as_float(w1.z), s, c3.x), fmaf(__uint_as_float(w1.w), s, c3.y), O()));
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d2_empty[buf]);
                ask_base(fb + 1);                        // under the next block's products
            }
            together();
        }
    }
    // every thread comes here, also after a give-up
    if (s_abort) cluster_abort(&s_abort, C);
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    if (s_abort) abort_drain();                         // in every CTA of the cluster alike
    tc_fence_after();
    if (warp == AD_WARPS) tmem_free(tmem, 512);
}

template <class... Params, class... Args>
static cudaError_t ad_launch(void (*kernel)(Params...), uint32_t C, uint32_t clusters, uint32_t threads, size_t smem, cudaStream_t st, const Args&... args) {
    const cudaError_t e = allow_shared(kernel);
    return e == cudaSuccess ? launch_dependent_clusters(kernel, C, clusters, threads, smem, st, args...) : e;
}
// clusters of 1, 2, 4, 8 CTAs of the tensor-core kernel that the device holds at once
struct AbClusters { uint32_t n[9]; };
static AbClusters ab_clusters(const void* kernel, uint32_t n_parts, int sm_count) {
    AbClusters c{};
    const AbSmem L = ab_smem(AB_MAX_R, n_parts);
    if (allow_shared(kernel) != cudaSuccess) cudaGetLastError();
    for (uint32_t C = 1; C <= 8; C *= 2) {
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = C; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(C * 148); cfg.blockDim = dim3(L.threads()); cfg.dynamicSmemBytes = L.bytes; cfg.attrs = &attr; cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = sm_count / (int)C; }
        c.n[C] = n > 0 ? (uint32_t)n : 1u;
    }
    return c;
}
template <class T, class O, AdSums SUMS>
static cudaError_t adapters_launch(const AdaptersArgs& a, cudaStream_t st) {
    const AdSmem L = ad_smem(a.R, a.T, AD_PARTS<T, O>);
    const uint32_t sms = (uint32_t)a.sm_count;
    // CTAs of the mma.sync kernels that run at once: two to an SM (ranks to 128) where their shared memory and the 1 KB
    // that each costs besides fit twice into 228 KB
    const bool few = a.n_adapters < AD_FEW;
    const uint32_t sort = few ? sizeof(AdSort<AD_FEW>) : sizeof(AdSort<AD_MANY>);
    const uint32_t room = L.bytes + sort + sizeof(AdShared) + 1024 + 64 <= 114 * 1024 ? 2 * sms : sms;
    // a cluster is as large as the units leave SMs for
    const auto spread = [](uint64_t units, uint32_t ctas, uint32_t least) { uint32_t C = 8; while (C > least && units * C > ctas) C /= 2; return C; };
    // 5120 -> 2304, tiles against sorted: 64 tokens, rank 16 or 32: of one adapter 15.3 and 9.1 us, of four 11.1 and 9.6, of 16 8.3 and 10.6; 40 of three 9.1 both.
    // 600 adapters, 4096 -> 2048: 200 tokens, rank 16, 24 and 29, rank 64 46 and 65; 999: 86 and 59, 158 and 144; 8192: 720 and 181, 1320 and 488
    if (a.T <= 16 || (a.T <= AD_TT && a.T < 14 * (uint64_t)a.n_adapters) || (!few && a.T < 512) || a.n_adapters >= AD_MANY) {
        const uint32_t tiles = (a.T + AD_TT - 1) / AD_TT, most = a.T < a.n_adapters ? a.T : a.n_adapters, distinct = most < AD_TT ? most : AD_TT;
        const uint32_t C = spread((uint64_t)tiles * distinct, room, 2);
        uint32_t slots = room / (C * tiles);
        slots = slots < 1 ? 1 : slots > distinct ? distinct : slots;
        return ad_launch(adapters_tile_kernel<T, O, SUMS>, C, slots * tiles, AD_WARPS * 32, L.bytes, st, a, C, slots);
    }
    const uint32_t segs = (a.T + AD_SEG - 1) / AD_SEG, tokens = (a.T + segs - 1) / segs;   // segments all alike
    // a segment's units: about as many as it has adapters, or 64 tokens
    const uint32_t units = tokens / AD_TT > a.n_adapters ? tokens / AD_TT : a.n_adapters < tokens ? a.n_adapters : tokens;
    // mma.sync against tensor cores, 5120 -> 2304: rank 32: 1000 tokens of 32 adapters 27 and 24 us, 4000 of 8 38 and 39; rank 64: 1000 of 32 34 and 25, 4000
    // of 8 57 and 39; rank 128: 56 and 29, 115 and 42.  Eight tokens per unit, rank 32: 16 and 22 (256 of 32), 55 and 93 (4000 of 64).  Little work: 105 tokens
    // of three, 2048 -> 4584: rank 64 12.3 and 14.9, rank 96 15.9 and 17.0, rank 128 19.0 and 17.0; 256 of four, rank 64, 15.1 and 15.9, rank 96 24 and 18.
    if (a.R > 32 && (uint64_t)a.T * a.R > AB_LITTLE && a.R <= AB_MAX_R && tokens >= AB_MIN_ROWS * units && few) {
        AbParams P;
        P.p = a;
        cudaError_t e = encode_map<3>(&P.a, a.dtype, a.a, {a.K, a.R, a.n_adapters}, {a.K, a.a_stride}, {64, a.R, 1});
        if (e != cudaSuccess) return e;
        static const AbClusters room1 = ab_clusters(reinterpret_cast<const void*>(adapters_tensor_kernel<T, O>), AD_PARTS<T, O>, a.sm_count);   // an SM holds one CTA
        P.C = 8;
        P.seg_len = tokens;
        while (P.C > 1 && ((uint64_t)units * segs > room1.n[P.C] || P.C > (a.K + 63) / 64)) P.C /= 2;   // every CTA has inputs to sum
        P.per_seg = room1.n[P.C] / segs;
        P.per_seg = P.per_seg < 1 ? 1 : P.per_seg > units + tokens / AD_TT + 1 ? units + tokens / AD_TT + 1 : P.per_seg;
        const AbSmem S = ab_smem(a.R, AD_PARTS<T, O>);
        return ad_launch(adapters_tensor_kernel<T, O>, P.C, P.per_seg * segs, S.threads(), S.bytes, st, P);
    }
    // Tokens of a unit at most, and CTAs of its cluster: by waves of clusters, each a start (us: 6, or 9 with the ring) and the unit's outputs and
    // inputs over its CTAs; a unit of up to 16 tokens takes about as long per token as a larger one (longer at high ranks: A and B are read once per
    // unit), and more of them fill the SMs (units of 64 against the choice: 431 tokens of one adapter, rank 8, 872 -> 5120, 20 and 12.6 us; 648 of four, rank 8, 4096 -> 5120, 28 and 19; 4465 of 58, rank 8,
    // 2304 -> 5120, 92 and 79; 4000 of eight, rank 32, 5120 -> 2304, 48 and 38; 4000 of 64 stays at 64: 55, with 16 62;
    // rank 256: 200 of two, 4096 -> 4096, 72 and 32).
    uint32_t tt = AD_TT, C = 8, cut = units;
    const uint32_t n = a.n_adapters < tokens ? a.n_adapters : tokens;
    const double one = (3.0 * a.K + 28.0 * a.N) / 5120;
    double best = 0;
    for (const uint32_t t : {16u, 32u, 64u}) {
        const uint32_t most = tokens / t + n / 2 > n ? tokens / t + n / 2 : n;
        const double rows = (double)tokens / most;
        for (uint32_t c = 1; c <= 8; c *= 2) {
            const uint32_t at_once = room / (c * segs);              // of a segment's clusters
            const double waves = at_once ? (most + at_once - 1) / at_once : (double)most * c * segs / room;
            const double us = waves * ((t > 16 && rows > 8 ? 9 : 6) + one * (rows > 16 ? rows / (13 + a.R / 32.0) : 1.0) / c);
            if (best == 0 || us < best) { best = us; tt = t; C = c; cut = most; }
        }
    }
    uint32_t per_seg = room / (C * segs);
    per_seg = per_seg < 1 ? 1 : per_seg > cut + tokens / tt + 1 ? cut + tokens / tt + 1 : per_seg;
    return ad_launch(few ? adapters_sorted_kernel<T, O, SUMS, AD_FEW> : adapters_sorted_kernel<T, O, SUMS, AD_MANY>, C, per_seg * segs, AD_WARPS * 32, L.bytes + sort, st, a, C,
                     per_seg, tokens, tt);
}
template <class T>
static cudaError_t adapters_out(const AdaptersArgs& a, cudaStream_t st) {
    if (a.out_dtype == DT_F32) return a.R > 128 ? adapters_launch<T, float, AD_ROUNDED>(a, st) : adapters_launch<T, float, AD_CHAINED>(a, st);
    return a.K > AD_LONG ? adapters_launch<T, T, AD_CHAINED>(a, st) : adapters_launch<T, T, AD_PLAIN>(a, st);
}
cudaError_t launch_adapters(const AdaptersArgs& a, cudaStream_t st) {
    return a.dtype == DT_BF16 ? adapters_out<__nv_bfloat16>(a, st) : adapters_out<__half>(a, st);
}

}  // namespace mlxs
