// Products grouped by expert over 16-bit weights: y[p] = W_g x[p] for offsets[g] <= p < offsets[g + 1], or SwiGLU of a
// gate and an up product of the same rows.
#include "common.cuh"
#include "kernels.h"
#include "umma_pair.cuh"

namespace mlxs {

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, float* o) { *o = v; }

__device__ __forceinline__ float gp_swiglu(float g, float u, float limit) {
    if (limit > 0.f) {   // comparisons keep a NaN
        g = g > limit ? limit : g;
        u = u > limit ? limit : (u < -limit ? -limit : u);
    }
    return __fdividef(g, 1.f + expf(-g)) * u;
}

// The rows [r0, r1) of group g, cut to the call's rows; false where the offsets had to be cut
__device__ __forceinline__ bool gp_range(const GroupedArgs& a, uint32_t g, uint32_t& r0, uint32_t& r1) {
    const uint32_t o0 = a.offsets[g], o1 = a.offsets[g + 1];
    r0 = min(o0, a.rows);
    r1 = max(min(o1, a.rows), r0);
    return o0 <= o1 && o1 <= a.rows;
}

// ------------------------------------------------------------------------------------------------------------
// tensor-core tiles
// ------------------------------------------------------------------------------------------------------------
constexpr uint32_t GT_KS = 64;                                   // inputs per stage: 128 bytes, one swizzle row
constexpr uint32_t GT_NT = 256;                                  // most rows of a tile (MMA N)
constexpr uint32_t GT_STAGES = 6;
constexpr uint32_t GT_A_BYTES = 128 * GT_KS * 2;                 // a CTA's 128 outputs of a stage
constexpr uint32_t GT_B_BYTES = 128 * GT_KS * 2;                 // at most: a CTA's half of 256 rows
constexpr uint32_t GT_STAGE = GT_A_BYTES + GT_B_BYTES;
constexpr uint32_t GT_SWAP_BYTES = 2 * 4 * 2 * 8 * 32 * 4;       // gate / up swap: [buffer][warp pair][side][8 rows][32 outputs] f32
constexpr uint32_t GT_SMEM = GT_STAGES * GT_STAGE + GT_SWAP_BYTES + 1024;
constexpr uint32_t GT_MAX_G = 1024;
constexpr uint32_t GT_EPI_WARPS = 8;

struct TileParams {
    CUtensorMap w, x;
    GroupedArgs a;
    uint32_t n_ft, n_ks;     // output tiles of a row tile, stages
    uint32_t fmt, poll_limit;
};

struct GtItem { uint32_t g, p0, rows, n; };   // group, first position, rows, MMA N (a multiple of 32)
// walks the call's row tiles: tile number -> group and rows.  A group's rows are cut into as few tiles as hold them, all alike.
struct GtWalk {
    const uint32_t *off, *tiles;   // [G + 1] positions, [G + 1] first row tile
    uint32_t g = 0;
    __device__ GtItem at(uint32_t tile) {
        while (tiles[g + 1] <= tile) ++g;
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
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// true where all 64 threads of a named barrier say so
__device__ __forceinline__ bool both_warps(uint32_t id, bool ok) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, r;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.and.pred r, %1, 64, p;\n\tselp.u32 %0, 1, 0, r;\n\t}" : "=r"(r) : "r"(id), "r"((uint32_t)ok) : "memory");
    return r != 0;
}

template <bool SWIGLU, class O>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(64 + GT_EPI_WARPS * 32, 1) grouped_tile_kernel(const __grid_constant__ TileParams P) {
    extern __shared__ uint8_t smem_any[];
    __shared__ __align__(8) uint64_t full_bar[GT_STAGES], empty_bar[GT_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t s_tmem, s_off[2 * GT_MAX_G], s_tiles[GT_MAX_G + 1];
    __shared__ volatile int s_abort;
    const GroupedArgs& a = P.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, rank = cluster_rank();
    const uint32_t ring = (smem_u32(smem_any) + 1023u) & ~1023u;
    float* swap = reinterpret_cast<float*>(smem_any + (ring - smem_u32(smem_any)) + GT_STAGES * GT_STAGE);
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < GT_STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * GT_EPI_WARPS); }
        s_abort = 0;
        mbar_fence_init();
        tma_prefetch_map(&P.w);
        tma_prefetch_map(&P.x);
    }
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
        for (uint32_t g = g0; g < g1; ++g) mine += (s_off[2 * g + 1] - s_off[2 * g] + GT_NT - 1) / GT_NT;
        uint32_t sum = mine;
        for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, o); if (lane >= o) sum += v; }
        uint32_t at = sum - mine;
        for (uint32_t g = g0; g < g1; ++g) { s_tiles[g] = at; at += (s_off[2 * g + 1] - s_off[2 * g] + GT_NT - 1) / GT_NT; }
        if (lane == 31) s_tiles[a.G] = sum;
    } else if (warp == 1) {
        tmem_alloc_pair(&s_tmem, 512);
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = s_tmem, n_items = s_tiles[a.G] * P.n_ft, n_pairs = gridDim.x / 2, pair = blockIdx.x / 2;
    constexpr uint32_t FT = SWIGLU ? 128 : 256;                  // outputs of an item
    auto give_up = [&](uint32_t code) { if (!s_abort) atomicMax(a.status, code); s_abort = 1; };
    GtWalk walk{s_off, s_tiles};

    if (warp == 0) {
        // ---------------- producer: this CTA's half of A's rows and of B's ----------------
        const bool gather = a.gather;
        uint32_t s = 0, ph = 0;
        bool ok = true;
        for (uint32_t i = pair; i < n_items && ok; i += n_pairs) {
            const GtItem it = walk.at(i / P.n_ft);
            const uint32_t f0 = (i % P.n_ft) * FT + rank * (FT / 2), hb = it.n / 2, b0 = it.p0 + rank * hb;
            const uint32_t nb = (hb + 31) / 32, b_bytes = gather ? hb * GT_KS * 2 : nb * 32 * GT_KS * 2;
            const uint32_t both = 2 * (GT_A_BYTES + b_bytes);
            // rows of W behind this CTA's two halves of 64 outputs: one after the other, or the gate's and the up's
            const uint32_t o0 = f0, o1 = SWIGLU ? a.N + f0 : f0 + 64;
            int32_t r[4] = {0, 0, 0, 0};
            if (gather && lane < hb / 4)
                for (int j = 0; j < 4; ++j) {
                    // a position behind the tile's last repeats it, an index out of range reads row 0: neither is stored
                    const uint32_t p = min(b0 + lane * 4 + j, it.p0 + it.rows - 1), xr = a.order[p] / a.x_div;
                    r[j] = xr < a.x_rows ? (int32_t)xr : 0;
                }
            for (uint32_t ks = 0; ks < P.n_ks; ++ks) {
                if (!mbar_wait_warp_at(smem_u32(&empty_bar[s]), ph ^ 1u, &s_abort)) { give_up(ST_WAIT_EMPTY); ok = false; break; }
                const uint32_t full = map_to_rank(smem_u32(&full_bar[s]), 0), sa = ring + s * GT_STAGE, sb = sa + GT_A_BYTES;
                const int32_t k = (int32_t)(ks * GT_KS);
                if (lane == 0) {
                    if (rank == 0) mbar_expect_tx(&full_bar[s], both);
                    if (a.in_out) {
                        tma_load_3d(sa, &P.w, (int32_t)o0, k, (int32_t)it.g, full);
                        tma_load_3d(sa + GT_A_BYTES / 2, &P.w, (int32_t)o1, k, (int32_t)it.g, full);
                    } else {
                        tma_load_3d(sa, &P.w, k, (int32_t)o0, (int32_t)it.g, full);
                        tma_load_3d(sa + GT_A_BYTES / 2, &P.w, k, (int32_t)o1, (int32_t)it.g, full);
                    }
                }
                if (gather) {
                    if (lane < hb / 4) tma_gather4(sb + lane * 4 * 128, &P.x, k, r[0], r[1], r[2], r[3], full);
                } else if (lane < nb) {
                    tma_load_2d(sb + lane * 32 * 128, &P.x, k, (int32_t)(b0 + lane * 32), full);
                }
                if (++s == GT_STAGES) { s = 0; ph ^= 1u; }
            }
        }
        if (s_abort) for (int i = 0; i < 2000; ++i) __nanosleep(1000);   // copies in flight land before the memory goes
    } else if (warp == 1) {
        // ---------------- MMA issuer: the even CTA's, for both ----------------
        if (rank == 0) {
            uint32_t s = 0, ph = 0, n_done = 0;
            bool ok = true;
            for (uint32_t i = pair; i < n_items && ok; i += n_pairs) {
                const GtItem it = walk.at(i / P.n_ft);
                const uint32_t idesc = umma_idesc_pair(P.fmt, it.n, a.in_out), buf = n_done & 1u, acc = tmem + buf * 256;
                if (!mbar_wait_cluster(smem_u32(&acc_empty[buf]), (n_done >> 1 & 1u) ^ 1u, &s_abort)) { give_up(ST_WAIT_EMPTY); ok = false; }
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                tc_fence_after();
                for (uint32_t ks = 0; ks < P.n_ks; ++ks) {
                    if (!mbar_wait_cluster(smem_u32(&full_bar[s]), ph, &s_abort)) { give_up(ST_WAIT_FULL); ok = false; }
                    ok = __all_sync(0xFFFFFFFFu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = ring + s * GT_STAGE, sb = sa + GT_A_BYTES;
                    // K-major: 16 inputs are 32 bytes of every row; M-major: 16 rows of 128 bytes
                    const uint32_t a_step = a.in_out ? 2048u : 32u;
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t j = 0; j < GT_KS / 16; ++j)
                            umma_f16_pair(acc, umma_desc_sw128(sa + j * a_step, a.in_out ? GT_A_BYTES / 2 : 16, 1024),
                                          umma_desc_sw128(sb + j * 32, 16, 1024), idesc, ks | j ? 1u : 0u);
                        umma_commit_pair(smem_u32(&empty_bar[s]), 3);
                    }
                    __syncwarp();
                    if (++s == GT_STAGES) { s = 0; ph ^= 1u; }
                }
                if (ok && elect_one()) umma_commit_pair(smem_u32(&acc_full[buf]), 3);
                __syncwarp();
                ++n_done;
            }
        }
    } else {
        // ---------------- epilogue: a thread owns one lane (output) of the accumulator; a warp half of the tile's rows ----------------
        const uint32_t q = warp & 3u, half = (warp - 2) >> 2;
        uint32_t n_done = 0, swaps = 0;
        O* y = static_cast<O*>(a.y);
        for (uint32_t i = pair; i < n_items; i += n_pairs) {
            const GtItem it = walk.at(i / P.n_ft);
            const uint32_t buf = n_done & 1u, f0 = (i % P.n_ft) * FT + rank * (FT / 2);
            bool got = __all_sync(0xFFFFFFFFu, mbar_wait_cluster(smem_u32(&acc_full[buf]), n_done >> 1 & 1u, &s_abort));
            if (SWIGLU) got = both_warps(1 + half * 2 + (q & 1u), got);   // the two warps of a swap go on, or give up, together
            if (!got) { give_up(ST_WAIT_FULL); break; }
            tc_fence_after();
            const uint32_t f = f0 + (SWIGLU ? (q & 1u) * 32 : q * 32) + lane;
            for (uint32_t c = half * 16; c < it.n; c += 32) {
                uint32_t v[16];
                tmem_ld16_nowait(tmem + buf * 256 + c + ((q * 32u) << 16), v);
                // lane j < 16: where row c + j of the tile goes
                uint32_t yr = 0xFFFFFFFFu;
                if (lane < 16 && c + lane < it.rows) {
                    const uint32_t p = it.p0 + c + lane, o = a.order ? a.order[p] : p;
                    yr = a.scatter ? o : p;
                    if ((a.gather && o / a.x_div >= a.x_rows) || yr >= a.y_rows) { yr = 0xFFFFFFFFu; atomicMax(a.status, ST_BAD_ROW); }
                }
                tmem_wait_ld();
                if (SWIGLU) {
                    // Warps q and q + 2 hold gate and up of the same outputs: the first takes rows 0 .. 7 of the chunk, the second
                    // 8 .. 15, and each gives the other what it needs.
                    const uint32_t pr = half * 2 + (q & 1u), up = q >> 1;
                    float* b = swap + ((swaps & 1u) * 4 + pr) * 512;
#pragma unroll
                    for (int j = 0; j < 8; ++j) b[(up * 8 + j) * 32 + lane] = __uint_as_float(up ? v[j] : v[8 + j]);
                    asm volatile("bar.sync %0, 64;" ::"r"(1 + pr) : "memory");
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float other = b[((up ^ 1u) * 8 + j) * 32 + lane], mine = __uint_as_float(up ? v[8 + j] : v[j]);
                        const uint32_t row = __shfl_sync(0xFFFFFFFFu, yr, up * 8 + j);
                        const float z = up ? gp_swiglu(other, mine, a.limit) : gp_swiglu(mine, other, a.limit);
                        if (row != 0xFFFFFFFFu && f < a.N) from_f32(z, y + (size_t)row * a.ld_y + f);
                    }
                    ++swaps;
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint32_t row = __shfl_sync(0xFFFFFFFFu, yr, j);
                        if (row != 0xFFFFFFFFu && f < a.N) from_f32(__uint_as_float(v[j]), y + (size_t)row * a.ld_y + f);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_rank(smem_u32(&acc_empty[buf]), 0));
            ++n_done;
        }
    }
    // every thread comes here, also after a give-up
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    if (warp == 1) tmem_free_pair(tmem, 512);
}

// cuTensorMapEncodeTiled through the runtime, so that the library needs no link to the driver
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}
// a matrix (rank 2) or a stack of matrices (3) of 16-bit elements: boxes of 64 inner elements, rows swizzled over 128 bytes
static cudaError_t encode_map(CUtensorMap* map, int dtype, int rank, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t ld, uint64_t stride,
                              uint32_t box1) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {d0, d1, d2}, strides[2] = {ld * 2, stride * 2};
    const cuuint32_t box[3] = {64, box1, 1}, step[3] = {1, 1, 1};
    const CUresult r = fn(map, dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
                          dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <bool SWIGLU, class O>
static cudaError_t tile_launch(const GroupedArgs& a, cudaStream_t st) {
    TileParams P;
    P.a = a;
    P.n_ft = (a.N + (SWIGLU ? 127 : 255)) / (SWIGLU ? 128 : 256);
    P.n_ks = (a.K + GT_KS - 1) / GT_KS;
    P.fmt = a.dtype == DT_BF16 ? UMMA_BF16 : UMMA_F16;
    cudaError_t e = a.in_out ? encode_map(&P.w, a.dtype, 3, a.w, a.n_w(), a.K, a.G, a.ld_w, a.w_stride, 64)
                             : encode_map(&P.w, a.dtype, 3, a.w, a.K, a.n_w(), a.G, a.ld_w, a.w_stride, 64);
    if (e == cudaSuccess) e = encode_map(&P.x, a.dtype, 2, a.x, a.K, a.x_rows, 1, a.ld_x, 0, a.gather ? 1 : 32);
    if (e != cudaSuccess) return e;
    const auto kernel = grouped_tile_kernel<SWIGLU, O>;
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GT_SMEM)) != cudaSuccess) return e;
    kernel<<<a.sm_count / 2 * 2, 64 + GT_EPI_WARPS * 32, GT_SMEM, st>>>(P);
    return cudaGetLastError();
}
template <class O>
static cudaError_t grouped_out(const GroupedArgs& a, cudaStream_t st) {
    return a.swiglu ? tile_launch<true, O>(a, st) : tile_launch<false, O>(a, st);
}
cudaError_t launch_grouped(const GroupedArgs& a, cudaStream_t st) {
    if (a.out_dtype == DT_F32) return grouped_out<float>(a, st);
    return a.dtype == DT_BF16 ? grouped_out<__nv_bfloat16>(a, st) : grouped_out<__half>(a, st);
}

}  // namespace mlxs
