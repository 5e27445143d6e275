// Products grouped by expert over 16-bit weights: y[p] = W_g x[p] for offsets[g] <= p < offsets[g + 1], or SwiGLU of a
// gate and an up product of the same rows.
#include "common.cuh"
#include "kernels.h"

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

// One CTA: 64 rows of a group x 64 outputs, operands through shared memory in slices of 32 inputs, a thread 4 x 4 sums.
template <class T, class O>
__global__ void __launch_bounds__(256) grouped_kernel(const GroupedArgs a) {
    __shared__ float xs[32][68], ws[2][32][68];
    __shared__ uint32_t xrow[64], yrow[64];
    const uint32_t g = blockIdx.z, n0 = blockIdx.x * 64, tid = threadIdx.x;
    uint32_t r0, r1;
    if (!gp_range(a, g, r0, r1) && tid == 0) atomicMax(a.status, ST_BAD_OFFSETS);
    const uint32_t parts = a.swiglu ? 2 : 1, tx = tid % 16, ty = tid / 16;
    const T* w = static_cast<const T*>(a.w) + (size_t)g * a.w_stride;
    for (uint32_t p0 = r0 + blockIdx.y * 64; p0 < r1; p0 += gridDim.y * 64) {
        if (tid < 64) {
            const uint32_t p = p0 + tid;
            uint32_t xr = 0xFFFFFFFFu, yr = 0xFFFFFFFFu;
            if (p < r1) {
                xr = a.gather ? a.order[p] / a.x_div : p;
                yr = a.scatter ? a.order[p] : p;
                if (xr >= a.x_rows || yr >= a.y_rows) { xr = yr = 0xFFFFFFFFu; atomicMax(a.status, ST_BAD_ROW); }
            }
            xrow[tid] = xr; yrow[tid] = yr;
        }
        float acc[2][4][4] = {};
        __syncthreads();
        for (uint32_t k0 = 0; k0 < a.K; k0 += 32) {
            for (uint32_t i = tid; i < 64 * 32; i += 256) {
                const uint32_t r = i / 32, k = i % 32;
                xs[k][r] = xrow[r] != 0xFFFFFFFFu && k0 + k < a.K ? to_f32(static_cast<const T*>(a.x)[(size_t)xrow[r] * a.ld_x + k0 + k]) : 0.f;
            }
            for (uint32_t part = 0; part < parts; ++part)
                for (uint32_t i = tid; i < 64 * 32; i += 256) {
                    const uint32_t n = a.in_out ? i % 64 : i / 32, k = a.in_out ? i / 64 : i % 32;
                    const size_t o = part * a.N + n0 + n;
                    ws[part][k][n] = n0 + n < a.N && k0 + k < a.K ? to_f32(w[a.in_out ? (size_t)(k0 + k) * a.ld_w + o : o * a.ld_w + k0 + k]) : 0.f;
                }
            __syncthreads();
            for (uint32_t k = 0; k < 32; ++k)
                for (uint32_t part = 0; part < parts; ++part)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[part][i][j] = fmaf(xs[k][ty * 4 + i], ws[part][k][tx * 4 + j], acc[part][i][j]);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t n = n0 + tx * 4 + j, yr = yrow[ty * 4 + i];
                if (n < a.N && yr != 0xFFFFFFFFu)
                    from_f32(a.swiglu ? gp_swiglu(acc[0][i][j], acc[1][i][j], a.limit) : acc[0][i][j], static_cast<O*>(a.y) + (size_t)yr * a.ld_y + n);
            }
        __syncthreads();
    }
}

template <class T, class O>
static cudaError_t grouped_launch(const GroupedArgs& a, cudaStream_t st) {
    const uint32_t tiles = (a.rows + 63) / 64;
    grouped_kernel<T, O><<<dim3((a.N + 63) / 64, tiles < 64 ? tiles : 64, a.G), 256, 0, st>>>(a);
    return cudaGetLastError();
}
cudaError_t launch_grouped(const GroupedArgs& a, cudaStream_t st) {
    if (a.dtype == DT_BF16) return a.out_dtype == DT_F32 ? grouped_launch<__nv_bfloat16, float>(a, st) : grouped_launch<__nv_bfloat16, __nv_bfloat16>(a, st);
    return a.out_dtype == DT_F32 ? grouped_launch<__half, float>(a, st) : grouped_launch<__half, __half>(a, st);
}

}  // namespace mlxs
