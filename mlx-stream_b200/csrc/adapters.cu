// Low-rank adapters of many requests: y[t] = base[t] + scale_a B_a (A_a x[t]), a = ids[t].
#include "common.cuh"
#include "kernels.h"

namespace mlxs {

__device__ __forceinline__ float ad_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float ad_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float ad_f32(float v) { return v; }
__device__ __forceinline__ void ad_put(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void ad_put(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void ad_put(float v, float* o) { *o = v; }

// One CTA per token: the inner product's rows by warps, then the outputs by threads.
template <class T, class O>
__global__ void __launch_bounds__(256) adapters_kernel(const AdaptersArgs a) {
    __shared__ float u[256];
    const uint32_t t = blockIdx.x, tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const int32_t id = a.ids[t];
    const bool bad = id >= 0 && (uint32_t)id >= a.n_adapters, on = id >= 0 && !bad;
    if (bad && tid == 0) atomicMax(a.status, ST_BAD_ADAPTER);
    uint32_t R = 0;
    if (on) {
        const int32_t r = a.ranks ? a.ranks[id] : (int32_t)a.R;
        R = r < 0 ? 0u : min((uint32_t)r, a.R);
        const float scale = a.scales ? a.scales[id] : 1.f;
        const T* x = static_cast<const T*>(a.x) + (size_t)t * a.ld_x;
        for (uint32_t i = warp; i < R; i += 8) {
            const T* A = static_cast<const T*>(a.a) + (size_t)id * a.a_stride + (size_t)i * a.K;
            float s = 0.f;
            for (uint32_t k = lane; k < a.K; k += 32) s = fmaf(ad_f32(x[k]), ad_f32(A[k]), s);
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (lane == 0) u[i] = s * scale;
        }
    }
    __syncthreads();
    for (uint32_t n = tid; n < a.N; n += 256) {
        float s = 0.f;
        if (on) {
            const T* B = static_cast<const T*>(a.b) + (size_t)id * a.b_stride + (size_t)n * a.R;
            for (uint32_t i = 0; i < R; ++i) s = fmaf(u[i], ad_f32(B[i]), s);
        }
        const float v = a.base ? ad_f32(static_cast<const O*>(a.base)[(size_t)t * a.ld_base + n]) + s : s;
        ad_put(v, static_cast<O*>(a.y) + (size_t)t * a.ld_y + n);
    }
}

template <class T, class O>
static cudaError_t adapters_launch(const AdaptersArgs& a, cudaStream_t st) {
    adapters_kernel<T, O><<<a.T, 256, 0, st>>>(a);
    return cudaGetLastError();
}
cudaError_t launch_adapters(const AdaptersArgs& a, cudaStream_t st) {
    if (a.dtype == DT_BF16) return a.out_dtype == DT_F32 ? adapters_launch<__nv_bfloat16, float>(a, st) : adapters_launch<__nv_bfloat16, __nv_bfloat16>(a, st);
    return a.out_dtype == DT_F32 ? adapters_launch<__half, float>(a, st) : adapters_launch<__half, __half>(a, st);
}

}  // namespace mlxs
