// Tensor maps for the copies into swizzled operand tiles (host side).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "kernels.h"

namespace mlxs {

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
// 16-bit elements, boxes of 64 inner elements, rows swizzled over 128 bytes; dims, strides (in elements, from the second dimension on) and
// box from the innermost out; what lies outside reads as zero
template <int RANK>
static cudaError_t encode_map(CUtensorMap* map, int dtype, const void* base, const uint64_t (&dims)[RANK], const uint64_t (&strides)[RANK - 1],
                              const uint32_t (&box)[RANK]) {
    const EncodeTiled fn = encode_tiled();
    if (!fn) return cudaErrorNotSupported;
    cuuint64_t d[RANK], s[RANK - 1];
    cuuint32_t b[RANK], step[RANK];
    for (int i = 0; i < RANK; ++i) { d[i] = dims[i]; b[i] = box[i]; step[i] = 1; }
    for (int i = 0; i < RANK - 1; ++i) s[i] = strides[i] * 2;
    const CUresult r = fn(map, dtype == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)RANK, const_cast<void*>(base),
                          d, s, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

}  // namespace mlxs
