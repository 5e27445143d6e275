// Low-rank adapters of many requests beside a shared projection: y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t].
//
// Both factors are thin (rank <= 256 of thousands), so the work is bytes: x, base and y once, an adapter's A and B once per 64 tokens that
// use it; the products themselves (2 R (K + N) per token) are small enough for mma.sync.
//   * A cluster of C CTAs takes a tile of 64 tokens and, one after the other, the adapters that occur in it (its share of them where few tiles
//     leave SMs free: the tile's distinct adapters are dealt out over `slots` clusters).  Nothing is sorted and no workspace is held: the
//     cluster finds an adapter's rows in the tile's 64 ids.
//   * Inner product u = A x: every CTA sums a C-th of the inputs; its warps split that share again.  The partial sums meet over distributed
//     shared memory, warps first, then CTAs, always in the same order (no atomics: a call repeats itself, and a row's sums do not depend on
//     which other rows are there beyond the split of the warps by the adapter's row count, 32 or fewer or more).
//   * u is kept as two 16-bit parts, hi = round(u), lo = round(u - hi): 16 (bf16) or 22 (f16) bits, so what is lost between the factors is far
//     inside an output's rounding.  f16 parts are scaled by the row's largest power of two, since A x may pass f16's range where y does not.
//   * Outer product y = base + u B^T: every CTA a C-th of the outputs, base added in f32, one rounding.
// Operands come straight from global memory as mma fragments, 16 bytes per lane: a lane's eight consecutive inputs stand for the k positions
// 2t, 2t+1, 2t+8, 2t+9 of two products, the same for both operands.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "umma_pair.cuh"

namespace mlxs {

constexpr uint32_t AD_TT = 64;          // tokens of a tile
constexpr uint32_t AD_WARPS = 8;
constexpr uint32_t AD_MR = 64;          // rank rows of a pass

__device__ __forceinline__ uint4 ad_ld16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <class T>
__device__ __forceinline__ void ad_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void ad_mma<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const uint32_t a[4] = {a0, a1, a2, a3};
    mma_bf16(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void ad_mma<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    const uint32_t a[4] = {a0, a1, a2, a3};
    mma_f16(d, a, b0, b1);
}
__device__ __forceinline__ float ad_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ad_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void ad_round(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void ad_round(float v, __half& o) { o = __float2half_rn(v); }
// two values as two 16-bit parts each, packed
template <class T>
__device__ __forceinline__ void ad_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    T h[2], l[2];
    ad_round(x, h[0]); ad_round(y, h[1]);
    // an infinity has no remainder
    const float dx = x - ad_f32(h[0]), dy = y - ad_f32(h[1]);
    ad_round(isinf(ad_f32(h[0])) ? 0.f : dx, l[0]); ad_round(isinf(ad_f32(h[1])) ? 0.f : dy, l[1]);
    hi = *reinterpret_cast<uint32_t*>(h);
    lo = *reinterpret_cast<uint32_t*>(l);
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

// eight outputs of a row: base (or nothing) + v, rounded once
__device__ __forceinline__ void ad_put8(float* y, const float* base, const float (&v)[8]) {
    float4 lo = make_float4(v[0], v[1], v[2], v[3]), hi = make_float4(v[4], v[5], v[6], v[7]);
    if (base) {
        const float4 b0 = *reinterpret_cast<const float4*>(base), b1 = *reinterpret_cast<const float4*>(base + 4);
        lo.x += b0.x; lo.y += b0.y; lo.z += b0.z; lo.w += b0.w;
        hi.x += b1.x; hi.y += b1.y; hi.z += b1.z; hi.w += b1.w;
    }
    *reinterpret_cast<float4*>(y) = lo;
    *reinterpret_cast<float4*>(y + 4) = hi;
}
template <class T>
__device__ __forceinline__ void ad_put8(T* y, const T* base, const float (&v)[8]) {
    uint4 b = make_uint4(0, 0, 0, 0);
    if (base) b = *reinterpret_cast<const uint4*>(base);
    const T* bt = reinterpret_cast<const T*>(&b);
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) ad_round(base ? ad_f32(bt[i]) + v[i] : v[i], o[i]);
    *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(o);
}

struct AdSmem {                          // dynamic shared memory, byte offsets
    uint32_t warp_part, part, u_hi, u_lo, bytes, r16, rp, pitch;   // rp: rank rows that a pass writes; pitch: bytes of a token's parts, 64 modulo 128 (rows on other banks)
};
__host__ __device__ inline AdSmem ad_smem(uint32_t R) {
    AdSmem s;
    s.r16 = (R + 15) / 16 * 16;
    s.rp = R <= 16 ? 16 : R <= 32 ? 32 : AD_MR;
    s.pitch = (R + 31) / 32 * 64;
    if (s.pitch % 128 == 0) s.pitch += 64;
    s.warp_part = 0;
    s.part = AD_WARPS * s.rp * 32 * 4;
    s.u_hi = s.part + s.r16 * AD_TT * 4;
    s.u_lo = s.u_hi + AD_TT * s.pitch;
    s.bytes = s.u_lo + AD_TT * s.pitch;
    return s;
}

// One warp's share of the inner products of MT x 16 rank rows from r0 on and NT x 8 tokens: k blocks of 32 from kb on, every `step`-th
template <class T, int MT, int NT>
__device__ __forceinline__ void ad_inner(const AdaptersArgs& a, const T* A, uint32_t R, uint32_t r0, const uint32_t* rows, uint32_t n_rows, uint32_t t0,
                                         uint32_t kb, uint32_t kb_end, uint32_t step, float* out) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    float acc[MT][NT][4] = {};
    const T* xr[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xr[n] = n * 8 + g < n_rows ? static_cast<const T*>(a.x) + (size_t)(t0 + rows[n * 8 + g]) * a.ld_x + t * 8 : nullptr;
    const T* ar = A + (size_t)(r0 + g) * a.K + t * 8;
#pragma unroll 2
    for (; kb < kb_end; kb += step) {
        const uint32_t k = kb * 32;
        const bool in = k + t * 8 < a.K;
        uint4 xv[NT], av[MT][2];
        const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NT; ++n) xv[n] = xr[n] && in ? ad_ld16(xr[n] + k) : zero;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) av[m][h] = r0 + m * 16 + h * 8 + g < R && in ? ad_ld16(ar + (size_t)(m * 16 + h * 8) * a.K + k) : zero;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                ad_mma<T>(acc[m][n], av[m][0].x, av[m][1].x, av[m][0].y, av[m][1].y, xv[n].x, xv[n].y);
                ad_mma<T>(acc[m][n], av[m][0].z, av[m][1].z, av[m][0].w, av[m][1].w, xv[n].z, xv[n].w);
            }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float* o = out + (m * 16 + g) * 32 + n * 8 + 2 * t;
            *reinterpret_cast<float2*>(o) = make_float2(acc[m][n][0], acc[m][n][1]);
            *reinterpret_cast<float2*>(o + 8 * 32) = make_float2(acc[m][n][2], acc[m][n][3]);
        }
}

// MT x 16 tokens times 32 outputs from f0 on.  Column c of product j stands for output (c / 2) 8 + 2 j + c % 2, so that a lane ends up
// with eight consecutive outputs of a token.
template <class T, class O, int MT>
__device__ __forceinline__ void ad_outer(const AdaptersArgs& a, const T* B, uint32_t R, uint32_t f0, const uint32_t* rows, uint32_t n_rows, uint32_t t0,
                                         uint32_t u_hi, uint32_t u_lo, uint32_t pitch, const float* row_scale) {
    const uint32_t lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    float acc[MT][4][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (uint32_t k = 0; k < R; k += 32) {
        const int left = (int)R - (int)(k + t * 8);       // of this lane's eight rank rows, those that count
        uint4 bv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t f = f0 + (g >> 1) * 8 + 2 * j + (g & 1u);
            bv[j] = f < a.N && left > 0 ? ad_first(ad_ld16(B + (size_t)f * a.R + k + t * 8), left) : zero;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const uint32_t at = (part ? u_lo : u_hi) + (m * 16 + g) * pitch + k * 2 + t * 16;
                uint4 lo = zero, hi = zero;
                if (left > 0 && m * 16 + g < n_rows) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w) : "r"(at));
                if (left > 0 && m * 16 + g + 8 < n_rows) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w) : "r"(at + 8 * pitch));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ad_mma<T>(acc[m][j], lo.x, hi.x, lo.y, hi.y, bv[j].x, bv[j].y);
                    ad_mma<T>(acc[m][j], lo.z, hi.z, lo.w, hi.w, bv[j].z, bv[j].w);
                }
            }
    }
    const uint32_t f = f0 + t * 8;
    if (f >= a.N) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t i = m * 16 + h * 8 + g;
            if (i >= n_rows) continue;
            const float s = row_scale[i];
            const float v[8] = {acc[m][0][2 * h] * s, acc[m][0][2 * h + 1] * s, acc[m][1][2 * h] * s, acc[m][1][2 * h + 1] * s,
                                acc[m][2][2 * h] * s, acc[m][2][2 * h + 1] * s, acc[m][3][2 * h] * s, acc[m][3][2 * h + 1] * s};
            const size_t row = t0 + rows[i];
            ad_put8(static_cast<O*>(a.y) + row * a.ld_y + f, a.base ? static_cast<const O*>(a.base) + row * a.ld_base + f : nullptr, v);
        }
}

template <class T, class O>
__global__ void __launch_bounds__(AD_WARPS * 32) adapters_kernel(const AdaptersArgs a, const uint32_t C, const uint32_t slots) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(16) int32_t s_id[AD_TT], s_adapter[AD_TT];
    __shared__ uint32_t s_rows[AD_TT], s_bare[AD_TT], s_n[4];       // s_n: distinct adapters, rows of this one, bare rows, distinct of the first 32 tokens
    __shared__ float s_scale[AD_TT];
    const AdSmem L = ad_smem(a.R);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, rank = cluster_rank();
    const uint32_t unit = blockIdx.x / C, tile = unit / slots, slot = unit % slots, t0 = tile * AD_TT;
    float* const warp_part = reinterpret_cast<float*>(smem + L.warp_part);
    float* const part = reinterpret_cast<float*>(smem + L.part);
    const uint32_t base_s = smem_u32(smem);

    // the tile's ids and its distinct adapters, in order of their first token
    if (warp < 2) {
        int32_t id = -1;
        if (t0 + tid < a.T) {
            id = a.ids[t0 + tid];
            if (id >= 0 && (uint32_t)id >= a.n_adapters) {
                if (slot == 0 && rank == 0) atomicMax(a.status, ST_BAD_ADAPTER);
                id = -1;
            }
        }
        s_id[tid] = id;
    }
    __syncthreads();
    if (warp < 2) {
        const int32_t id = s_id[tid];
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, id);
        bool first = id >= 0 && (same & ((1u << lane) - 1)) == 0;
        if (warp == 1)
            for (uint32_t j = 0; j < 32; j += 4) {
                const int4 v = *reinterpret_cast<const int4*>(s_id + j);
                first = first && v.x != id && v.y != id && v.z != id && v.w != id;
            }
        const uint32_t firsts = __ballot_sync(0xFFFFFFFFu, first), before = __popc(firsts & ((1u << lane) - 1));
        if (warp == 0) {
            if (first) s_adapter[before] = id;
            if (lane == 0) s_n[3] = __popc(firsts);
        }
        asm volatile("bar.sync 1, 64;" ::: "memory");
        if (warp == 1) {
            if (first) s_adapter[s_n[3] + before] = id;
            if (lane == 0) s_n[0] = s_n[3] + __popc(firsts);
        }
    } else if (warp == 2) {
        uint32_t n = 0;
        for (uint32_t h = 0; h < 2; ++h) {
            const bool bare = s_id[h * 32 + lane] < 0 && t0 + h * 32 + lane < a.T;
            const uint32_t m = __ballot_sync(0xFFFFFFFFu, bare);
            if (bare) s_bare[n + __popc(m & ((1u << lane) - 1))] = h * 32 + lane;
            n += __popc(m);
        }
        if (lane == 0) s_n[2] = n;
    }
    __syncthreads();
    const uint32_t n_adapters = s_n[0];

    // tokens without an adapter: y = base
    if (slot == 0 && a.base != a.y) {
        const uint32_t c0 = (uint32_t)((uint64_t)rank * (a.N / 8) / C), c1 = (uint32_t)((uint64_t)(rank + 1) * (a.N / 8) / C), n = s_n[2] * (c1 - c0);
        constexpr uint32_t VEC = 16 / sizeof(O);
        for (uint32_t i = tid; i < n; i += AD_WARPS * 32) {
            const size_t row = t0 + s_bare[i / (c1 - c0)], f = (size_t)(c0 + i % (c1 - c0)) * 8;
#pragma unroll
            for (uint32_t v = 0; v < 8 / VEC; ++v) {
                uint4 w = make_uint4(0, 0, 0, 0);
                if (a.base) w = *reinterpret_cast<const uint4*>(static_cast<const O*>(a.base) + row * a.ld_base + f + v * VEC);
                *reinterpret_cast<uint4*>(static_cast<O*>(a.y) + row * a.ld_y + f + v * VEC) = w;
            }
        }
    }

    const uint32_t n_kb = (a.K + 31) / 32, kb0 = (uint32_t)((uint64_t)rank * n_kb / C), kb1 = (uint32_t)((uint64_t)(rank + 1) * n_kb / C);
    const uint32_t n_fb = (a.N + 31) / 32, fb0 = (uint32_t)((uint64_t)rank * n_fb / C), fb1 = (uint32_t)((uint64_t)(rank + 1) * n_fb / C);
    for (uint32_t d = slot; d < n_adapters; d += slots) {
        const int32_t id = s_adapter[d];
        if (warp == 0) {
            uint32_t n = 0;
            for (uint32_t h = 0; h < 2; ++h) {
                const bool mine = s_id[h * 32 + lane] == id;
                const uint32_t m = __ballot_sync(0xFFFFFFFFu, mine);
                if (mine) s_rows[n + __popc(m & ((1u << lane) - 1))] = h * 32 + lane;
                n += __popc(m);
            }
            if (lane == 0) s_n[1] = n;
        }
        __syncthreads();
        const uint32_t n_rows = s_n[1];
        const int32_t given = a.ranks ? a.ranks[id] : (int32_t)a.R;
        const uint32_t R = given < 0 ? 0u : min((uint32_t)given, a.R);
        const T* A = static_cast<const T*>(a.a) + (size_t)id * a.a_stride;
        const T* B = static_cast<const T*>(a.b) + (size_t)id * a.b_stride;

        // ---- inner product: this CTA's inputs; warps split them by 8, or by 4 for each half of more than 32 tokens ----
        const uint32_t n_split = n_rows > 32 ? 4 : 8, half = n_rows > 32 ? warp >> 2 : 0, split = n_rows > 32 ? warp & 3u : warp;
        const uint32_t h_rows = half ? n_rows - 32 : min(n_rows, 32u);
        for (uint32_t r0 = 0; r0 < R; r0 += AD_MR) {
            const uint32_t rr = min(R - r0, AD_MR);                      // rank rows of the pass
            float* const mine = warp_part + warp * L.rp * 32;
            const uint32_t kb = kb0 + split;
            if (h_rows <= 8) {
                if (rr <= 16) ad_inner<T, 1, 1>(a, A, R, r0, s_rows + half * 32, h_rows, t0, kb, kb1, n_split, mine);
                else if (rr <= 32) ad_inner<T, 2, 1>(a, A, R, r0, s_rows + half * 32, h_rows, t0, kb, kb1, n_split, mine);
                else ad_inner<T, 4, 1>(a, A, R, r0, s_rows + half * 32, h_rows, t0, kb, kb1, n_split, mine);
            } else {
                if (rr <= 16) ad_inner<T, 1, 4>(a, A, R, r0, s_rows + half * 32, h_rows, t0, kb, kb1, n_split, mine);
                else if (rr <= 32) ad_inner<T, 2, 4>(a, A, R, r0, s_rows + half * 32, h_rows, t0, kb, kb1, n_split, mine);
                else ad_inner<T, 4, 4>(a, A, R, r0, s_rows + half * 32, h_rows, t0, kb, kb1, n_split, mine);
            }
            __syncthreads();
            // the warps' sums in order, tokens side by side
            for (uint32_t i = tid; i < rr * 64; i += AD_WARPS * 32) {
                const uint32_t r = i / 64, c = i % 64, hf = c / 32;
                if (c >= n_rows) continue;
                const float* p = warp_part + (hf * 4) * L.rp * 32 + r * 32 + c % 32;
                float s = p[0];
                for (uint32_t w = 1; w < n_split; ++w) s += p[w * L.rp * 32];
                part[c * L.r16 + r0 + r] = s;
            }
            __syncthreads();
        }
        cluster_sync_all();
        // ---- the CTAs' sums in order, a warp to a token; the parts go to every CTA ----
        for (uint32_t i = rank + C * warp; i < n_rows; i += C * AD_WARPS) {
            const float scale = a.scales ? a.scales[id] : 1.f;
            float v[4][2];
            float most = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t r = j * 64 + lane * 2;
                v[j][0] = v[j][1] = 0.f;
                if (r >= R) continue;
                const uint32_t at = base_s + L.part + (i * L.r16 + r) * 4;
                for (uint32_t c = 0; c < C; ++c) {
                    const float2 p = ad_ld_cluster2(map_to_rank(at, c));
                    v[j][0] += p.x;
                    v[j][1] += p.y;
                }
                v[j][0] *= scale;
                v[j][1] = r + 1 < R ? v[j][1] * scale : 0.f;
                most = fmaxf(most, fmaxf(fabsf(v[j][0]), fabsf(v[j][1])));
            }
            float down = 1.f, up = 1.f;
            if (std::is_same<T, __half>::value) {
                for (uint32_t o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
                // a power of two next to the row's largest: the parts lie in (-2, 2); rows of zeros, and of infinities, as they are
                const uint32_t e = __float_as_uint(most) & 0x7F800000u;
                if (e >= 0x00800000u && e <= 0x7E800000u) { up = __uint_as_float(e); down = __uint_as_float(0x7F000000u - e); }
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t r = j * 64 + lane * 2;
                if (r >= a.R) continue;
                uint32_t hi, lo;
                ad_split<T>(v[j][0] * down, v[j][1] * down, hi, lo);
                for (uint32_t c = 0; c < C; ++c) {
                    const uint32_t to = map_to_rank(base_s + L.u_hi + i * L.pitch + r * 2, c);
                    ad_st_cluster(to, hi);
                    ad_st_cluster(to + (L.u_lo - L.u_hi), lo);
                }
            }
            if (lane < C) ad_st_cluster(map_to_rank(smem_u32(&s_scale[i]), lane), __float_as_uint(up));
        }
        cluster_sync_all();
        // ---- outer product: this CTA's outputs ----
        for (uint32_t fb = fb0 + warp; fb < fb1; fb += AD_WARPS) {
            if (n_rows <= 16) ad_outer<T, O, 1>(a, B, R, fb * 32, s_rows, n_rows, t0, base_s + L.u_hi, base_s + L.u_lo, L.pitch, s_scale);
            else if (n_rows <= 32) ad_outer<T, O, 2>(a, B, R, fb * 32, s_rows, n_rows, t0, base_s + L.u_hi, base_s + L.u_lo, L.pitch, s_scale);
            else ad_outer<T, O, 4>(a, B, R, fb * 32, s_rows, n_rows, t0, base_s + L.u_hi, base_s + L.u_lo, L.pitch, s_scale);
        }
        __syncthreads();
    }
}

template <class T, class O>
static cudaError_t adapters_launch(const AdaptersArgs& a, cudaStream_t st) {
    const uint32_t tiles = (a.T + AD_TT - 1) / AD_TT, most = a.T < a.n_adapters ? a.T : a.n_adapters, distinct = most < AD_TT ? most : AD_TT;
    const uint64_t work = (uint64_t)tiles * distinct;              // (tile, adapter) pairs at most
    const uint32_t C = work <= 32 ? 8 : 4;
    uint32_t slots = (uint32_t)a.sm_count * 2 / (C * tiles);
    slots = slots < 1 ? 1 : slots > distinct ? distinct : slots;
    const AdSmem L = ad_smem(a.R);
    const auto kernel = adapters_kernel<T, O>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L.bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = C; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C * slots * tiles); cfg.blockDim = dim3(AD_WARPS * 32); cfg.dynamicSmemBytes = L.bytes; cfg.stream = st; cfg.attrs = &attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, C, slots);
}
cudaError_t launch_adapters(const AdaptersArgs& a, cudaStream_t st) {
    if (a.dtype == DT_BF16) return a.out_dtype == DT_F32 ? adapters_launch<__nv_bfloat16, float>(a, st) : adapters_launch<__nv_bfloat16, __nv_bfloat16>(a, st);
    return a.out_dtype == DT_F32 ? adapters_launch<__half, float>(a, st) : adapters_launch<__half, __half>(a, st);
}

}  // namespace mlxs
