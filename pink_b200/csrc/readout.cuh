// Shared pieces of the read-out operators (route.cu, read_out.cu, product.cu): element types, argument checks, reductions.
#pragma once
#include "../../include/pink_b200.h"
#include "kernels.cuh"

#include <cfloat>
#include <cstdio>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace pinkb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, loaded and stored as one word of VEC * sizeof(T) bytes (the caller has checked the alignment).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

inline size_t element_size(uint32_t type) { return type == PINK_B200_F32 ? 4 : 2; }

// Calls fn with a value of the element type that `type` names.
template <typename Fn>
cudaError_t with_type(uint32_t type, Fn fn)
{
    if (type == PINK_B200_F32) return fn(float());
    if (type == PINK_B200_BF16) return fn(__nv_bfloat16());
    return fn(__half());
}

// Largest power of two of elements (at most `most`) that every listed row start is aligned to.
struct RowAlign
{
    uint64_t bits = 0;
    RowAlign& add(const void* p, uint64_t ld, size_t size)
    {
        if (p) bits |= reinterpret_cast<uintptr_t>(p) | ld * size;
        return *this;
    }
    uint32_t elements(size_t size, uint32_t most) const
    {
        uint32_t v = most;
        while (v > 1 && bits % (v * size)) v >>= 1;
        return v;
    }
};

constexpr uint32_t kNoNeuron = 0xFFFFFFFFu;

inline int launch_status(cudaError_t e, const char* what)
{
    if (e == cudaSuccess) return PINK_B200_OK;
    cudaGetLastError();
    char msg[256];
    std::snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
    return report_error(PINK_B200_ECUDA, msg);
}

// Maximum and sum over a warp; every lane gets the result.  The sum's order is fixed.
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

} // namespace pinkb
